// Attention over the paged cache: argument checks and choice of the kernel.
#include <cmath>

#include "kernels.h"
#include "paged.cuh"

using namespace vggt;

namespace {

// Up to 16 rows per sequence and key head go to the warp-level kernel, more to
// the tcgen05 one.  32 sequences over 32,768 keys of 128, in us, warp-level
// against tcgen05: 4 rows 473 / 578, 20 rows 559 / 563, 32 rows 548 / 514, 64
// rows 974 / 530 (the warp-level kernel with tiles of 32 and 64 rows).
bool few_rows(int64_t max_new, int group) { return max_new * group <= 16; }

PagedPlan plan_of(int64_t total, int64_t seqs, int kv_heads, int group, int dim, int64_t max_new,
                  int64_t max_len) {
  return few_rows(max_new, group)
             ? paged_rows_plan(total, seqs, kv_heads, group, dim, max_len)
             : paged_tc05_plan(total, seqs, kv_heads, group, dim, max_len);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

extern "C" size_t vggt_paged_attention_workspace_size(int64_t total, int64_t seqs, int kv_heads,
                                                      int group, int dim, int64_t max_new,
                                                      int64_t max_len) {
  if (total <= 0 || seqs <= 0 || kv_heads < 1 || group < 1 || max_new < 1 || max_len < 0 ||
      (dim != 64 && dim != 128))
    return 0;
  clamp_expected(total, max_new, max_len);
  return (size_t)kMaxCounters * 4 +
         plan_of(total, seqs, kv_heads, group, dim, max_new, max_len).partial_bytes;
}

extern "C" int vggt_paged_attention(
    const void* q, int dtype, int64_t total, int64_t q_token_stride, int64_t q_head_stride,
    const void* k_pages, const void* v_pages, int64_t n_pages, int kv_heads, int page, int dim,
    int64_t page_stride, int64_t head_stride, int64_t row_stride, const int32_t* table,
    int64_t table_width, int64_t seqs, const int32_t* lengths, const int32_t* starts, int group,
    int causal, float scale, int64_t max_new, int64_t max_len, void* out,
    int64_t out_token_stride, int64_t out_head_stride, float* lse, int32_t* status,
    void* workspace, size_t workspace_bytes, void* stream) {
  PagedAttnArgs a{};
  if (int rc = check_pool(dtype, n_pages, kv_heads, page, dim, page_stride, head_stride,
                          row_stride, table_width, seqs, total, &a.pool))
    return rc;
  if (group < 1 || (int64_t)kv_heads * group > 65535 || total * group > 0x7fffffffLL)
    return api_fail("group %d: kv_heads * group must lie in [1, 65535], tokens * group below 2^31",
                    group);
  if (!std::isfinite(scale) || scale <= 0.f) return api_fail("scale must be positive and finite");
  if (max_new < 1 || max_len < 0) return api_fail("max_new must be positive, max_len not negative");
  if (total == 0 || seqs == 0) return api_fail(nullptr);
  if (!q || !out || !lengths || !starts || !table || !workspace)
    return api_fail("q, out, lengths, starts, table and workspace must be non-NULL");
  if (!k_pages || !v_pages || n_pages < 1) return api_fail("the pools are empty");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_pages) || !aligned16(v_pages) ||
      !aligned16(workspace))
    return api_fail("q, out, the pools and the workspace must be 16-byte aligned");
  if (q_token_stride % 8 || q_head_stride % 8 || out_token_stride % 8 || out_head_stride % 8)
    return api_fail("strides of q and out must be multiples of 8 elements");
  clamp_expected(total, max_new, max_len);
  const PagedPlan plan = plan_of(total, seqs, kv_heads, group, dim, max_new, max_len);
  const size_t need = (size_t)kMaxCounters * 4 + plan.partial_bytes;
  if (workspace_bytes < need)
    return api_fail("workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (plan.tiles * kv_heads * plan.splits > 0x7fffffffLL)
    return api_fail("too many query rows (%lld tokens)", (long long)total);
  a.q = q;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.t = {table, lengths, starts, table_width, seqs, total, status};
  a.group = group;
  a.causal = causal != 0;
  a.dtype = dtype;
  a.scale = scale;
  a.out = out;
  a.o_token = out_token_stride;
  a.o_head = out_head_stride;
  a.lse = lse;
  a.workspace = workspace;
  a.wait_ns = api_wait_ns();
  a.wait_selftest = api_wait_selftest();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return api_cuda(few_rows(max_new, group) ? launch_paged_rows(a, plan, st)
                                           : launch_paged_tc05(a, plan, st));
}
