// What the kernels of attention over shared prefixes have in common (attn_shared.cu says what they compute).
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace mfq {

constexpr float kSharedNeg = -1e30f;

struct SharedAttnArgs {
  const __nv_bfloat16* q;  // [B * q_len, Hq, D]
  const uint8_t *k, *v;    // pages
  const float *k_scale, *v_scale;
  const int *table, *seq_lens;         // [B, max_pages], [B]
  const int *group_starts, *prefix_lens, *members;  // [groups + 1] places, [groups], [B] batch row of each place (null: its number)
  float *part_o, *part_ml;             // of the prefixes: [B * q_len * Hq, slots, D], [.., slots, 2]
  __nv_bfloat16* out;
  int* status;
  int B, Hq, Hk, max_pages, pages, groups, q_len, slots, prefix_splits, tail_splits;  // slots: partials of a query row and head over its prefix
  float scale_log2;
};

__device__ __forceinline__ void shared_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// Behind a wait that ran out (the status says so, results are invalid): copies and products that were started may still be on their way to memory that is
// about to be used again or given back.
__device__ __forceinline__ void let_started_work_end() {
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 2000000ull) {
  }
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t v) {  // two codes to fp16
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(v)));
  return r;
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_half(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 2^e that brings a positive number to [2^at, 2^(at + 1)); zeros, infinities and NaN: as if they were 1
__device__ __forceinline__ float power_to(float x, int at) {
  const int e = int(__float_as_uint(x) >> 23 & 0xff);
  return e == 0 || e == 255 ? 1.f : __uint_as_float(uint32_t(min(max(254 + at - e, 1), 254)) << 23);
}
// The x-th of the groups' tiles of `per_tile` query rows, all groups in order (whole warp): its group and number, false behind the last one.
__device__ __forceinline__ bool find_tile(const SharedAttnArgs& a, int x, int per_tile, int per_seq, int& group, int& tile) {
  int before = 0;
  for (int g = 0; g < a.groups; g += 32) {
    const int i = g + int(lane_id());
    int n = 0;
    if (i < a.groups) {
      const int lo = min(max(a.group_starts[i], 0), a.B), hi = min(max(a.group_starts[i + 1], lo), a.B);
      n = ((hi - lo) * per_seq + per_tile - 1) / per_tile;
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (int(lane_id()) >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + upto > x);
    if (past) {
      const int at = __ffs(past) - 1;
      group = g + at;
      tile = x - before - (__shfl_sync(0xffffffffu, upto, at) - __shfl_sync(0xffffffffu, n, at));
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}
// The group of a place (whole warp): how many groups end at it or before; a.groups behind the last one.
__device__ __forceinline__ int group_of(const SharedAttnArgs& a, int place) {
  int n = 0;
  for (int g = 0; g < a.groups; g += 32) {
    const int i = g + int(lane_id());
    n += __popc(__ballot_sync(0xffffffffu, i < a.groups && a.group_starts[i + 1] <= place));
  }
  return n;
}
__device__ __forceinline__ int member_row(const SharedAttnArgs& a, int place) {  // -1: none
  const int row = a.members ? a.members[place] : place;
  return row >= 0 && row < a.B ? row : -1;
}
// A group of n rows has (n - 1) / per_tile + 1 tiles, so that g groups of n in all have at most this, whatever the groups are.
inline int tiles_at_most(const SharedAttnArgs& a, int per_tile) {
  const int rows = a.B * (a.Hq / a.Hk) * a.q_len;
  return (rows - a.groups) / per_tile + a.groups;
}

}  // namespace mfq
