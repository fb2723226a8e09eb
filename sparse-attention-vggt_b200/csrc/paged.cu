// Host checks shared by the paged-cache entry points.
#include "paged.cuh"

#include "kernels.h"
#include "tc05.cuh"

namespace vggt {

int check_pool(int dtype, int64_t n_pages, int kv_heads, int page, int dim, int64_t page_stride,
               int64_t head_stride, int64_t row_stride, int64_t table_width, int64_t seqs,
               int64_t total, Pool* pool) {
  if (dtype != VGGT_DTYPE_BF16 && dtype != VGGT_DTYPE_FP16)
    return api_fail("the paged cache requires BF16 or FP16 (dtype code %d)", dtype);
  if (dim != 64 && dim != 128) return api_fail("head dim %d unsupported (64 or 128)", dim);
  if (page < 16 || page > 1024 || (page & (page - 1)))
    return api_fail("page size %d unsupported (a power of two from 16 to 1024)", page);
  if (n_pages < 0 || table_width < 0 || seqs < 0 || total < 0)
    return api_fail("negative size argument");
  if (kv_heads < 1 || kv_heads > 65535) return api_fail("kv_heads %d outside [1, 65535]", kv_heads);
  if (n_pages > 0x7fffffffLL || seqs > 65535 || total > 0x7fffffffLL ||
      table_width > 0x7fffffffLL / page)
    return api_fail("size argument too large (pages, tokens and slots stay below 2^31, seqs below "
                    "65536)");
  if (page_stride < 0 || head_stride < 0 || row_stride < dim || page_stride % 8 ||
      head_stride % 8 || row_stride % 8)
    return api_fail("pool strides must be multiples of 8 elements, rows at least dim apart");
  *pool = Pool{n_pages, page_stride, head_stride, row_stride, kv_heads, page,
               __builtin_ctz((unsigned)page), dim};
  return 0;
}

bool encode_pool_tmap(CUtensorMap* map, const void* pages, int dtype, const Pool& pool,
                      uint32_t rows) {
  const uint64_t dims[4] = {(uint64_t)pool.dim, (uint64_t)pool.page, (uint64_t)pool.kv_heads,
                            (uint64_t)pool.n_pages};
  const uint64_t strides[3] = {(uint64_t)pool.row_stride * 2, (uint64_t)pool.head_stride * 2,
                               (uint64_t)pool.page_stride * 2};
  const uint32_t box[4] = {64, rows, 1, 1};
  return encode_tmap_sw128(map, pages, dtype, 4, dims, strides, box);
}

}  // namespace vggt
