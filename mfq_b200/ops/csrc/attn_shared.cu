// Decode / verify attention over FP8 pages for sequences that share their first pages in groups: a group's prefix is read once for all
// of its sequences, every sequence's own tail once for itself, and the two are joined by the running maximum and sum of the softmax:
//
//   m = max(m_a, m_b),  l = l_a 2^(m_a - m) + l_b 2^(m_b - m),  o = (o_a 2^(m_a - m) + o_b 2^(m_b - m)) / l      (scores times log2 e)
//
// A unit of work is a run of pages of one table row with the query rows that go over it: a group with its prefix, or one sequence with its
// tail.  Query rows are (sequence, query token, head of the group of heads that share a KV head); a CTA takes a tile of them, one KV head
// and one split of the pages, and leaves (m, l, o) in fp32 for the merge.
// The page layout is that of attn_decode.cu, which says how its fragments are single shared-memory loads.
//
// Numbers: a row of q is scaled by a power of two to 2^13 <= max |q| < 2^14, so that fp16 holds its bf16 values exactly unless they are 2^-27 of
// the largest; E4M3 is exact in fp16; a page's multipliers meet the scores in fp32.  P times the V multiplier is rounded to fp16 (2^-12) after a power of
// two, kept for the rows of a warp, that brings the multipliers near 2^4 and is raised, the sums with it, where a page has larger ones.
// The reference reads shared prefixes once per row (mfq/kernels/cuda/paged_kv.cu).
#include "attn_shared.cuh"

namespace mfq {

template <int D, int WR>
struct SharedTile {
  static constexpr int kLanes = 4 / WR;  // groups of warps that take alternate pages
  static constexpr int kStages = WR == 1 ? 3 : WR == 2 ? 4 : 8;
  static constexpr int kPage = 16 * D, kStage = 2 * kPage + 128;
  static constexpr int kRing = kLanes * kStages * kStage;
  static constexpr int kSmem = kRing + 2 * kLanes * kStages * 8 + 16;
  static_assert(kRing >= 4 * (16 * D + 32) * 4, "the ring is the merge's scratch too");
};

// kPrefix: blockIdx.x = one of the groups' tiles of 16 WR rows; else blockIdx.x = place.  blockIdx.z = split.
template <int D, int WR, bool kPrefix>
__global__ void __launch_bounds__(128, D <= 128 ? 3 : 1)
shared_attn_kernel(const SharedAttnArgs a) {
  using L = SharedTile<D, WR>;
  constexpr int KSTEPS = D / 16, NBD = D / 8, kStages = L::kStages, kLanes = L::kLanes;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
  const int tile16 = warp % WR, page_lane = warp / WR;
  uint8_t* ring = smem + page_lane * kStages * L::kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kRing) + page_lane * kStages;
  uint64_t* empty = reinterpret_cast<uint64_t*>(smem + L::kRing) + (kLanes + page_lane) * kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kRing + 2 * kLanes * kStages * 8);
  pdl_trigger();
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0 && tile16 == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], WR); }
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();

  const int kvh = blockIdx.y, G = a.Hq / a.Hk, per_seq = G * a.q_len;
  const int splits = kPrefix ? a.prefix_splits : a.tail_splits, split = blockIdx.z;
  int first, count, slot, tile = 0;  // places of the unit, where its partial goes
  int page_lo, page_hi;
  if constexpr (kPrefix) {
    int g;
    if (!find_tile(a, blockIdx.x, 16 * WR, per_seq, g, tile)) return;
    first = min(max(a.group_starts[g], 0), a.B);
    count = min(max(a.group_starts[g + 1], first), a.B) - first;
    page_lo = 0;
    page_hi = min(max(a.prefix_lens[g], 0) >> 4, a.max_pages);
    slot = split;
  } else {
    first = blockIdx.x;
    const int g = group_of(a, first);
    count = g < a.groups && first >= a.group_starts[0] ? 1 : 0;
    const int row = count ? member_row(a, first) : -1;
    page_lo = count ? min(max(a.prefix_lens[g], 0) >> 4, a.max_pages) : 0;
    page_hi = row >= 0 ? min((max(a.seq_lens[row], 0) + 15) >> 4, a.max_pages) : 0;
    slot = a.slots - a.tail_splits + split;
  }
  if (count == 0) return;
  const int table_row = member_row(a, first);
  if (table_row < 0) { page_hi = page_lo; }
  {
    const int n = max(page_hi - page_lo, 0), per = (n + splits - 1) / splits;
    page_lo += split * per;
    page_hi = min(page_hi, page_lo + per);
  }
  const int my_pages = page_hi > page_lo + page_lane ? (page_hi - page_lo - page_lane + kLanes - 1) / kLanes : 0;
  const int* bt = a.table + size_t(max(table_row, 0)) * a.max_pages;
  const int rows = count * per_seq;
  bool ok = true;

  auto issue = [&](int i) {  // one thread of the lane: start the copies of its i-th page
    const int s = i % kStages;
    int page = bt[page_lo + page_lane + kLanes * i];
    if (page < 0 || page >= a.pages) {
      atomicCAS(a.status, 0, kStatusBadArgument);
      page = 0;
    }
    const size_t ph = size_t(page) * a.Hk + kvh;
    uint8_t* st = ring + s * L::kStage;
    mbar_expect_tx(&full[s], L::kStage);
    shared_bulk_load(st, a.k + ph * L::kPage, L::kPage, &full[s]);
    shared_bulk_load(st + L::kPage, a.v + ph * L::kPage, L::kPage, &full[s]);
    shared_bulk_load(st + 2 * L::kPage, a.k_scale + ph * 16, 64, &full[s]);
    shared_bulk_load(st + 2 * L::kPage + 64, a.v_scale + ph * 16, 64, &full[s]);
  };
  if (lane == 0 && tile16 == 0)
    for (int i = 0; i < min(my_pages, kStages); ++i) issue(i);

  // ---- this thread's two rows: their place, causal length and part of q ----
  uint32_t qa[KSTEPS][4];
  int row_len[2];
  size_t hq[2];
  bool live[2];
  float to_log2[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = (tile * WR + tile16) * 16 + g8 + 8 * half;
    const int place = first + r / per_seq, in = r % per_seq, qr = in / G;
    const int row = r < rows ? member_row(a, place) : -1;
    live[half] = row >= 0;
    hq[half] = live[half] ? (size_t(row) * a.q_len + qr) * a.Hq + kvh * G + in % G : 0;
    // a row that is not there has a zero query and is never stored: unmasked, it leaves `whole` below to the others
    row_len[half] = live[half] ? a.seq_lens[row] - (a.q_len - 1 - qr) : 0x7fffffff;
    const __nv_bfloat16* qp = a.q + hq[half] * D;
    float x[KSTEPS][4], top = 0.f;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      const int d0 = 64 * (s >> 2) + 16 * c + 4 * (s & 3);
      uint2 raw = make_uint2(0, 0);
      if (live[half]) raw = *reinterpret_cast<const uint2*>(qp + d0);
      const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(&raw);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[s][e] = __bfloat162float(b[e]);
        top = fmaxf(top, fabsf(x[s][e]));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float up = power_to(top, 13);
    to_log2[half] = a.scale_log2 / up;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      qa[s][half] = half_pair(x[s][0] * up, x[s][1] * up);
      qa[s][2 + half] = half_pair(x[s][2] * up, x[s][3] * up);
    }
  }
  const int low = __reduce_min_sync(0xffffffffu, min(row_len[0], row_len[1]));
  int most = max(live[0] ? row_len[0] : 0, live[1] ? row_len[1] : 0);
  most = __reduce_max_sync(0xffffffffu, most);

  float o[NBD][4];
#pragma unroll
  for (int j = 0; j < NBD; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m_run[2] = {kSharedNeg, kSharedNeg}, l_run[2] = {0.f, 0.f};
  float v_up = 0.f;  // power of two on the V multipliers; 0: none chosen yet

  for (int i = 0; i < my_pages; ++i) {
    const int s = i % kStages;
    ok = mbar_wait(&full[s], (i / kStages) & 1, abort_flag, a.status, kStatusTimeoutEpilogue);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    const uint8_t *sK = ring + s * L::kStage, *sV = sK + L::kPage;
    const float* sKs = reinterpret_cast<const float*>(sV + L::kPage);
    const float* sVs = sKs + 16;
    const int tok0 = (page_lo + page_lane + kLanes * i) << 4;
    float sc[2][4];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.f;
#pragma unroll
      for (int ch = 0; ch < D / 64; ++ch) {
        const uint4 kw = *reinterpret_cast<const uint4*>(sK + ch * 1024 + (nb * 8 + g8) * 64 + c * 16);
        const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) mma_half(sc[nb], qa[ch * 4 + sub], e4m3_pair(w[sub]), e4m3_pair(w[sub] >> 16));
      }
    }
    const bool whole = tok0 + 16 <= low;  // all rows see all of the page
    float mx[2] = {kSharedNeg, kSharedNeg};
    float2 vs[2];
    bool raise = false;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int tk = nb * 8 + 2 * c;
      const float2 ks = *reinterpret_cast<const float2*>(sKs + tk);
      vs[nb] = *reinterpret_cast<const float2*>(sVs + tk);
      if (!whole) {  // what nobody sees may hold anything
        if (tok0 + tk >= most) vs[nb].x = 0.f;
        if (tok0 + tk + 1 >= most) vs[nb].y = 0.f;
      }
      const float big = fmaxf(fabsf(vs[nb].x), fabsf(vs[nb].y));
      raise |= big * v_up > 1024.f || (v_up == 0.f && big > 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int half = e >> 1;
        sc[nb][e] *= ((e & 1) ? ks.y : ks.x) * to_log2[half];
        if (!whole && tok0 + tk + (e & 1) >= row_len[half]) sc[nb][e] = kSharedNeg;
        mx[half] = fmaxf(mx[half], sc[nb][e]);
      }
    }
    float corr[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
      mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
      const float mn = fmaxf(m_run[half], mx[half]);
      corr[half] = exp2f(m_run[half] - mn);
      m_run[half] = mn;
    }
    float o_corr[2] = {corr[0], corr[1]};
    if (__any_sync(0xffffffffu, raise)) {
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(fabsf(vs[0].x), fabsf(vs[0].y)), fmaxf(fabsf(vs[1].x), fabsf(vs[1].y))))));
      const float up = power_to(top, 4);
      if (v_up != 0.f) { o_corr[0] *= up / v_up; o_corr[1] *= up / v_up; }
      v_up = up;
    }
    float psum[2] = {0.f, 0.f}, p[2][4];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int half = e >> 1;
        // a masked score is kSharedNeg: exp2 gives 0 unless the whole row is still empty, hence the test (true for NaN)
        const float pe = !(sc[nb][e] <= 0.5f * kSharedNeg) ? exp2f(sc[nb][e] - m_run[half]) : 0.f;
        psum[half] += pe;
        p[nb][e] = pe * (((e & 1) ? vs[nb].y : vs[nb].x) * v_up);
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) l_run[half] = l_run[half] * corr[half] + psum[half];
    const uint32_t pa[4] = {half_pair(p[0][0], p[0][1]), half_pair(p[0][2], p[0][3]), half_pair(p[1][0], p[1][1]), half_pair(p[1][2], p[1][3])};
    if (__any_sync(0xffffffffu, o_corr[0] != 1.f || o_corr[1] != 1.f)) {
#pragma unroll
      for (int j = 0; j < NBD; ++j) { o[j][0] *= o_corr[0]; o[j][1] *= o_corr[0]; o[j][2] *= o_corr[1]; o[j][3] *= o_corr[1]; }
    }
    // codes of tokens that no row sees are left out: 0 times a NaN would be one
    uint32_t keep = 0xffffffffu;
    if (!whole) {
      keep = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (tok0 + 2 * c + (e & 1) + 8 * (e >> 1) < most) keep |= 0xffu << (8 * e);
    }
#pragma unroll
    for (int j = 0; j < NBD; ++j) {
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(sV + (8 * j + g8) * 16 + 4 * c) & keep;
      mma_half(o[j], pa, e4m3_pair(vw), e4m3_pair(vw >> 16));
    }
    __syncwarp();
    if constexpr (WR == 1) {
      if (lane == 0 && i + kStages < my_pages) issue(i + kStages);
    } else {
      if (lane == 0) mbar_arrive(&empty[s]);
      if (tile16 == 0 && lane == 0 && i >= 1 && i - 1 + kStages < my_pages) {  // the stage of the page before: its other readers are done by now, or nearly
        const int e = (i - 1) % kStages;
        if (mbar_wait(&empty[e], ((i - 1) / kStages) & 1, abort_flag, a.status, kStatusTimeoutProducer)) issue(i - 1 + kStages);
      }
      __syncwarp();
    }
  }
  // ---- merge: the lanes of a row, then the warps that took other pages of it ----
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    l_run[half] += __shfl_xor_sync(0xffffffffu, l_run[half], 1);
    l_run[half] += __shfl_xor_sync(0xffffffffu, l_run[half], 2);
  }
  __syncthreads();
  float* w_o = reinterpret_cast<float*>(smem) + warp * (16 * D + 32);  // [16][D], then (m, l) of each row
  const float down = v_up != 0.f ? 1.f / v_up : 0.f;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = g8 + 8 * half;
#pragma unroll
    for (int j = 0; j < NBD; ++j)
      *reinterpret_cast<float2*>(w_o + r * D + 8 * j + 2 * c) = make_float2(o[j][2 * half] * down, o[j][2 * half + 1] * down);
    if (c == 0) { w_o[16 * D + 2 * r] = m_run[half]; w_o[16 * D + 2 * r + 1] = l_run[half]; }
  }
  __syncthreads();
  if (!ok || *abort_flag) return;
  for (int idx = threadIdx.x; idx < 16 * WR * D; idx += 128) {
    const int t = idx / (16 * D), r = idx / D % 16, d = idx % D;
    const int global = (tile * WR + t) * 16 + r;
    if (global >= rows) continue;
    const int row = member_row(a, first + global / per_seq), in = global % per_seq;
    if (row < 0) continue;
    const float* base = reinterpret_cast<const float*>(smem) + t * (16 * D + 32);
    float mm = kSharedNeg, ll = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kLanes; ++w) mm = fmaxf(mm, base[w * WR * (16 * D + 32) + 16 * D + 2 * r]);
#pragma unroll
    for (int w = 0; w < kLanes; ++w) {
      const float* wo = base + w * WR * (16 * D + 32);
      const float cw = exp2f(wo[16 * D + 2 * r] - mm);
      ll += wo[16 * D + 2 * r + 1] * cw;
      acc += wo[r * D + d] * cw;
    }
    const size_t part = ((size_t(row) * a.q_len + in / G) * a.Hq + kvh * G + in % G) * a.slots + slot;
    a.part_o[part * D + d] = acc;
    if (d == 0) { a.part_ml[2 * part] = mm; a.part_ml[2 * part + 1] = ll; }
  }
}

// A warp per query row and head: o = sum of the partials' o 2^(m - max) / sum of their l 2^(m - max).
template <int D>
__global__ void __launch_bounds__(256)
shared_attn_merge_kernel(const SharedAttnArgs a) {
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x * 8 + warp, per_seq = a.q_len * a.Hq, place = item / per_seq;
  if (place >= a.B || place < a.group_starts[0] || place >= a.group_starts[a.groups]) return;
  const int row = member_row(a, place);
  if (row < 0) return;
  const size_t hq = size_t(row) * per_seq + item % per_seq;
  const float* ml = a.part_ml + hq * a.slots * 2;
  const float* po = a.part_o + hq * a.slots * D;
  float mm = kSharedNeg;
  for (int s = lane; s < a.slots; s += 32) mm = fmaxf(mm, ml[2 * s + 1] > 0.f || isnan(ml[2 * s + 1]) ? ml[2 * s] : kSharedNeg);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  float ll = 0.f, acc[D / 32] = {};
  for (int s = 0; s < a.slots; ++s) {
    const float l = ml[2 * s + 1];
    if (l == 0.f) continue;  // nothing seen there
    const float w = exp2f(ml[2 * s] - mm);
    ll += l * w;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const float2 x = *reinterpret_cast<const float2*>(po + s * D + 64 * j + 2 * lane);
      acc[2 * j] += x.x * w;
      acc[2 * j + 1] += x.y * w;
    }
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
    *reinterpret_cast<__nv_bfloat162*>(a.out + hq * D + 64 * j + 2 * lane) = __floats2bfloat162_rn(acc[2 * j] * inv, acc[2 * j + 1] * inv);
}

template <int D, int WR, bool kPrefix>
static int launch_shared_units(const SharedAttnArgs& a, dim3 grid, cudaStream_t stream) {
  using L = SharedTile<D, WR>;
  auto kernel = &shared_attn_kernel<D, WR, kPrefix>;
  static bool attr[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -6;
  if (!attr[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess) return -6;
    attr[dev] = true;
  }
  launch_kernel(kernel, grid, dim3(128), L::kSmem, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}

int launch_shared_prefix_tc(const SharedAttnArgs& a, int dim, bool two_tiles, cudaStream_t stream);  // attn_shared_tc.cu

template <int D>
static int launch_shared(const SharedAttnArgs& a, int tile, cudaStream_t stream) {
  const dim3 grid(tiles_at_most(a, tile), a.Hk, a.prefix_splits);
  const int rc = tile == 16   ? launch_shared_units<D, 1, true>(a, grid, stream)
                 : tile == 32 ? launch_shared_units<D, 2, true>(a, grid, stream)
                 : tile == 64 ? launch_shared_units<D, 4, true>(a, grid, stream)
                              : launch_shared_prefix_tc(a, D, tile == 256, stream);
  if (rc) return rc;
  if (const int rc = launch_shared_units<D, 1, false>(a, dim3(a.B, a.Hk, a.tail_splits), stream)) return rc;
  launch_kernel(shared_attn_merge_kernel<D>, dim3((a.B * a.q_len * a.Hq + 7) / 8), dim3(256), 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}

}  // namespace mfq

// q, out: [B * q_len, Hq, D] bf16; pages of the FP8 pool, `pages` of them; group_starts [groups + 1], prefix_lens [groups], members [B] or null; tile: query rows of a
// prefix CTA, 16, 32, 64 or for heads of 64 and 128 also 128, 256; partials [B * q_len * Hq * (prefix_splits (twice for a tile of 128) + tail_splits)] x D and x 2 floats.  (Hq / Hk) * q_len <= 16.  Rows in no group are not written.
extern "C" int mfq_paged_attn_decode_shared(const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale, const int* table,
                                            const int* seq_lens, const int* group_starts, const int* prefix_lens, const int* members, void* out,
                                            float* part_o, float* part_ml, int B, int Hq, int Hk, int D, int max_pages, int pages, int groups, int q_len,
                                            int tile, int prefix_splits, int tail_splits, float sm_scale, int* status, cudaStream_t stream) {
  using namespace mfq;
  if (B <= 0 || B > 65535 || Hk <= 0 || Hq % Hk || q_len < 1 || (Hq / Hk) * q_len > 16 || groups < 1 || groups > B || (tile != 16 && tile != 32 && tile != 64 && (D > 128 || (tile != 128 && tile != 256))) || prefix_splits < 1 ||
      tail_splits < 1 || pages < 1 || max_pages < 1 || Hk > 65535 || prefix_splits > 65535 || tail_splits > 65535)
    return -1;
  const SharedAttnArgs a{static_cast<const __nv_bfloat16*>(q), static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), k_scale, v_scale, table, seq_lens,
                         group_starts, prefix_lens, members, part_o, part_ml, static_cast<__nv_bfloat16*>(out), status, B, Hq, Hk, max_pages, pages, groups,
                         q_len, prefix_splits * (tile == 128 ? 2 : 1) + tail_splits, prefix_splits, tail_splits, sm_scale * 1.4426950408889634f};
  if (D == 128) return launch_shared<128>(a, tile, stream);
  if (D == 256) return launch_shared<256>(a, tile, stream);
  if (D == 64) return launch_shared<64>(a, tile, stream);
  return -1;
}
