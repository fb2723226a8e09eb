// The TMA producer of the weights of few rows, which streams 64-key tiles of K
// through a ring.
#pragma once

#include <type_traits>

#include "paged.cuh"
#include "tc05.cuh"

namespace vggt {

// Run by one full warp.  Tile t of the run that starts at slot `first_slot`
// (a multiple of 64) goes to stage t % kStages as kHalves blocks of 64 rows x
// 128 bytes (swizzled), one box per page or per 64 slots of a larger page.  Slots at or past `keys` (counted from
// first_slot) are not loaded where a whole box of them can be left out; page
// numbers that may not be used read as zeros.  full / empty: the first of
// kStages barriers each.  Returns when no copy is in flight.
//
// Page numbers are read 32 boxes ahead and the rest is 32-bit arithmetic on
// constants of the box count: with 64-bit counters and divisions by the box
// size a tile took this warp 1,400 clocks, longer than the copies.
template <int kHalves, int kStages>
__device__ __forceinline__ void produce_tiles(const PageTable& table, const Pool& pool,
                                              int64_t seq, int head, int64_t first_slot, int keys,
                                              int tiles, const CUtensorMap* map, uint32_t ring,
                                              uint32_t full, uint32_t empty,
                                              volatile int* abort_flag, uint64_t wait_ns) {
  constexpr uint32_t kBlock = 64 * 128, kStage = kHalves * kBlock;
  const int lane = threadIdx.x & 31;
  const int32_t* row_of_table = table.table + seq * table.width;
  const int in_page = (int)first_slot & (pool.page - 1), page_mask = pool.page - 1;
  auto run = [&](auto boxes_) {
    constexpr int kBoxes = decltype(boxes_)::value;  // per tile and block
    constexpr int kBox = 64 / kBoxes, kAhead = 32 / kBoxes;
    int page = 0, stage = 0, issued = 0;
    uint32_t phase = 1;
    for (int t = 0; t < tiles; ++t) {
      const int key0 = t * 64, turn = t & (kAhead - 1);
      if (turn == 0) {
        const int key = key0 + lane * kBox;
        page = (int)pool.n_pages;  // past the pool: reads as zeros
        if (key < keys && key < tiles * 64) {
          const int got = __ldg(row_of_table + ((first_slot + key) >> pool.page_shift));
          if (got >= 0 && got < pool.n_pages)
            page = got;
          else
            raise_status(table.status, VGGT_STATUS_BAD_PAGE);
        }
      }
      int pages[kBoxes];
#pragma unroll
      for (int b = 0; b < kBoxes; ++b)
        pages[b] = __shfl_sync(0xffffffffu, page, turn * kBoxes + b);
      int live = (keys - key0 + kBox - 1) / kBox;
      live = live < kBoxes ? live : kBoxes;
      if (t >= kStages && !tc::warp_wait(empty + 8u * stage, phase, abort_flag, wait_ns)) break;
      if (tc::elect_one()) {
        const uint32_t bar = full + 8u * stage, dst = ring + stage * kStage;
        const int row = (in_page + key0) & page_mask;
        tc::mbar_expect_tx(bar, (uint32_t)(live * kBox) * kHalves * 128u);
#pragma unroll
        for (int b = 0; b < kBoxes; ++b)
          if (b < live)
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
              tc::tma_load_4d(dst + h * kBlock + b * kBox * 128, map, bar, h * 64,
                              (row + b * kBox) & page_mask, head, pages[b]);
      }
      __syncwarp();
      ++issued;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    for (int t = issued > kStages ? issued - kStages : 0; t < issued; ++t)
      tc::mbar_wait_drain(full + 8u * (t % kStages), (uint32_t)((t / kStages) & 1), 1000000000ull);
  };
  if (pool.page >= 64)
    run(std::integral_constant<int, 1>{});
  else if (pool.page == 32)
    run(std::integral_constant<int, 2>{});
  else
    run(std::integral_constant<int, 4>{});
}

}  // namespace vggt
