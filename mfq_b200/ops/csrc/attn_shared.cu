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
// Numbers: a row of q is scaled by a power of two to 2^13 <= max |q| < 2^14, so that fp16 holds its bf16 values exactly down to 2^-30 of
// the largest; E4M3 is exact in fp16; a page's multipliers meet the scores in fp32.  P times the V multiplier is rounded to fp16 (2^-12) after a power of
// two, kept for the rows of a warp, that brings the multipliers near 2^4 and is raised, the sums with it, where a page has larger ones.
// The reference reads shared prefixes once per row (mfq/kernels/cuda/paged_kv.cu).
#include "attn_shared.cuh"
#include "pair.cuh"

#include <initializer_list>

namespace mfq {

template <int D>
struct SharedRing {  // four warps take alternate pages, each through a ring of its own
  static constexpr int kStages = 3, kPage = 16 * D, kStage = 2 * kPage + 128, kRing = 4 * kStages * kStage;
  static constexpr int kSmem = kRing + 4 * kStages * 8 + 16;
};
// What the four warps of a unit have, in floats where the rings were: parts [16 rows][kStride], then (m, l) of each row.  The columns behind D bring the rows
// of a fragment to different banks.  The first part becomes the unit's; its (m, l) are behind the four.
template <int D, bool kNarrow>
struct UnitParts {
  static constexpr int kStride = D + (kNarrow ? 4 : 8), kPart = 16 * kStride + 32, kMl = 4 * kPart, kEnd = kMl + 32;
};

__device__ __forceinline__ uint32_t transposed_pairs(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float4 load_peer(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float2 load_peer2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}

// What a warp has of a unit: the running maximum and sum of its rows and their outputs, in one of two forms.
//   wide   (up to 16 query rows): rows are the rows of the products, lane parts (g8, c) of m16n8k16 fragments
//   narrow (up to 8): the page's 16 tokens are the rows and the query rows the columns, S^T = K Q^T and O^T += V^T P, which halves the
//          products and the softmax (attn_decode.cu); a lane has the columns 2c and 2c + 1, of tokens (dims) g8 and g8 + 8
template <int D, bool kNarrow>
struct UnitRows {
  static constexpr int kSteps = D / 16, kOut = kNarrow ? D / 16 : D / 8, kQ = kNarrow ? 2 : 4;
  uint32_t q[kSteps][kQ];
  float o[kOut][4], m[2], l[2], to_log2[2], v_up;
  int len[2], low, most;

  // row_of(r): where row r's q is, in rows of D (negative: there is none); len_of(r): the keys that it sees
  template <typename RowOf, typename LenOf>
  __device__ __forceinline__ void load(const SharedAttnArgs& a, RowOf row_of, LenOf len_of, int g8, int c) {
    constexpr int kHalves = kNarrow ? 1 : 2;
    float up[kHalves];
    uint2 raw[kHalves][kSteps];
#pragma unroll
    for (int half = 0; half < kHalves; ++half) {  // all requested before the first is used
      const long long row = row_of(g8 + 8 * half);
      const __nv_bfloat16* qp = a.q + row * D;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        raw[half][s] = make_uint2(0, 0);
        if (row >= 0) raw[half][s] = *reinterpret_cast<const uint2*>(qp + 64 * (s >> 2) + 16 * c + 4 * (s & 3));
      }
    }
    bool there[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = kNarrow ? 2 * c + e : g8 + 8 * e;
      there[e] = row_of(r) >= 0;
      // a row that is not there has a zero query and is never stored: unmasked, it leaves `whole` below to the others
      len[e] = there[e] ? len_of(r) : 0x7fffffff;
    }
#pragma unroll
    for (int half = 0; half < kHalves; ++half) {
      float top = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(&raw[half][s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(__bfloat162float(b[e])));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      up[half] = power_to(top, 13);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(&raw[half][s]);
        q[s][half] = half_pair(__bfloat162float(b[0]) * up[half], __bfloat162float(b[1]) * up[half]);
        q[s][kNarrow ? 1 : 2 + half] = half_pair(__bfloat162float(b[2]) * up[half], __bfloat162float(b[3]) * up[half]);
      }
    }
    int lo = 0x7fffffff, hi = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float of = kNarrow ? __shfl_sync(0xffffffffu, up[0], (2 * c + e) * 4) : up[e % kHalves];
      to_log2[e] = a.scale_log2 / of;
      lo = min(lo, len[e]);
      hi = max(hi, there[e] ? len[e] : 0);
      m[e] = kSharedNeg;
      l[e] = 0.f;
    }
    low = __reduce_min_sync(0xffffffffu, lo);
    most = __reduce_max_sync(0xffffffffu, hi);
    v_up = 0.f;  // power of two on the V multipliers; 0: none chosen yet
#pragma unroll
    for (int j = 0; j < kOut; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  }

  // the V multipliers of this lane's tokens, near 2^4 or less after a power of two that the warp keeps; what nobody sees may hold anything
  __device__ __forceinline__ bool raises(float a, float b) const {
    const float big = fmaxf(fabsf(a), fabsf(b));
    return big * v_up > 1024.f || (v_up == 0.f && big > 0.f);
  }
  __device__ __forceinline__ void raise(float big, float (&o_corr)[2]) {
    const float up = power_to(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big))), 4);
    if (v_up != 0.f) { o_corr[0] *= up / v_up; o_corr[1] *= up / v_up; }
    v_up = up;
  }

  __device__ __forceinline__ void page(const uint8_t* sK, int tok0, int g8, int c) {
    const uint8_t* sV = sK + 16 * D;
    const float *sKs = reinterpret_cast<const float*>(sV + 16 * D), *sVs = sKs + 16;
    const bool whole = tok0 + 16 <= low;  // all rows see all of the page
    uint32_t keep = 0xffffffffu;  // codes of tokens that no row sees are left out: 0 times a NaN would be one
    if (!whole) {
      keep = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (tok0 + 2 * c + (e & 1) + 8 * (e >> 1) < most) keep |= 0xffu << (8 * e);
    }
    if constexpr (kNarrow) {
      float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ch = 0; ch < D / 64; ++ch) {
        const uint4 k0 = *reinterpret_cast<const uint4*>(sK + ch * 1024 + g8 * 64 + c * 16);
        const uint4 k1 = *reinterpret_cast<const uint4*>(sK + ch * 1024 + (8 + g8) * 64 + c * 16);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
          const uint32_t f[4] = {e4m3_pair(w0[sub]), e4m3_pair(w1[sub]), e4m3_pair(w0[sub] >> 16), e4m3_pair(w1[sub] >> 16)};
          mma_half(sc, f, q[ch * 4 + sub][0], q[ch * 4 + sub][1]);
        }
      }
      const float ks0 = sKs[g8], ks1 = sKs[g8 + 8];
      float vs0 = sVs[g8], vs1 = sVs[g8 + 8];
#pragma unroll
      for (int x = 0; x < 4; ++x) sc[x] *= (x < 2 ? ks0 : ks1) * to_log2[x & 1];
      if (!whole) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (tok0 + g8 + 8 * (x >> 1) >= len[x & 1]) sc[x] = kSharedNeg;
        if (tok0 + g8 >= most) vs0 = 0.f;
        if (tok0 + g8 + 8 >= most) vs1 = 0.f;
      }
      float corr[2], o_corr[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(sc[e], sc[2 + e]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[e], mx);
        o_corr[e] = corr[e] = exp2f(m[e] - mn);
        m[e] = mn;
      }
      if (__any_sync(0xffffffffu, raises(vs0, vs1))) raise(fmaxf(fabsf(vs0), fabsf(vs1)), o_corr);
      float p[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int e = x & 1;
        // a masked score is kSharedNeg: exp2 gives 0 unless the whole row is still empty, hence the test (true for NaN)
        const float pe = !(sc[x] <= 0.5f * kSharedNeg) ? exp2f(sc[x] - m[e]) : 0.f;
        l[e] = (x < 2 ? l[e] * corr[e] : l[e]) + pe;
        p[x] = pe * ((x < 2 ? vs0 : vs1) * v_up);
      }
      const uint32_t pb0 = transposed_pairs(half_pair(p[0], p[1])), pb1 = transposed_pairs(half_pair(p[2], p[3]));
      if (__any_sync(0xffffffffu, o_corr[0] != 1.f || o_corr[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < kOut; ++j) { o[j][0] *= o_corr[0]; o[j][1] *= o_corr[1]; o[j][2] *= o_corr[0]; o[j][3] *= o_corr[1]; }
      }
#pragma unroll
      for (int j = 0; j < kOut; ++j) {
        const uint32_t v0 = *reinterpret_cast<const uint32_t*>(sV + (16 * j + g8) * 16 + 4 * c) & keep;
        const uint32_t v1 = *reinterpret_cast<const uint32_t*>(sV + (16 * j + 8 + g8) * 16 + 4 * c) & keep;
        const uint32_t f[4] = {e4m3_pair(v0), e4m3_pair(v1), e4m3_pair(v0 >> 16), e4m3_pair(v1 >> 16)};
        mma_half(o[j], f, pb0, pb1);
      }
    } else {
      float sc[2][4], mx[2] = {kSharedNeg, kSharedNeg};
      float2 vs[2];
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.f;
#pragma unroll
        for (int ch = 0; ch < D / 64; ++ch) {
          const uint4 kw = *reinterpret_cast<const uint4*>(sK + ch * 1024 + (nb * 8 + g8) * 64 + c * 16);
          const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
          for (int sub = 0; sub < 4; ++sub) mma_half(sc[nb], q[ch * 4 + sub], e4m3_pair(w[sub]), e4m3_pair(w[sub] >> 16));
        }
      }
      bool up = false;
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        const int tk = nb * 8 + 2 * c;
        const float2 ks = *reinterpret_cast<const float2*>(sKs + tk);
        vs[nb] = *reinterpret_cast<const float2*>(sVs + tk);
        if (!whole) {
          if (tok0 + tk >= most) vs[nb].x = 0.f;
          if (tok0 + tk + 1 >= most) vs[nb].y = 0.f;
        }
        up |= raises(vs[nb].x, vs[nb].y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int half = e >> 1;
          sc[nb][e] *= ((e & 1) ? ks.y : ks.x) * to_log2[half];
          if (!whole && tok0 + tk + (e & 1) >= len[half]) sc[nb][e] = kSharedNeg;
          mx[half] = fmaxf(mx[half], sc[nb][e]);
        }
      }
      float corr[2], o_corr[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
        mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
        const float mn = fmaxf(m[half], mx[half]);
        o_corr[half] = corr[half] = exp2f(m[half] - mn);
        m[half] = mn;
      }
      if (__any_sync(0xffffffffu, up)) raise(fmaxf(fmaxf(fabsf(vs[0].x), fabsf(vs[0].y)), fmaxf(fabsf(vs[1].x), fabsf(vs[1].y))), o_corr);
      float psum[2] = {0.f, 0.f}, p[2][4];
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int half = e >> 1;
          const float pe = !(sc[nb][e] <= 0.5f * kSharedNeg) ? exp2f(sc[nb][e] - m[half]) : 0.f;
          psum[half] += pe;
          p[nb][e] = pe * (((e & 1) ? vs[nb].y : vs[nb].x) * v_up);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) l[half] = l[half] * corr[half] + psum[half];
      const uint32_t pa[4] = {half_pair(p[0][0], p[0][1]), half_pair(p[0][2], p[0][3]), half_pair(p[1][0], p[1][1]), half_pair(p[1][2], p[1][3])};
      if (__any_sync(0xffffffffu, o_corr[0] != 1.f || o_corr[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < kOut; ++j) { o[j][0] *= o_corr[0]; o[j][1] *= o_corr[0]; o[j][2] *= o_corr[1]; o[j][3] *= o_corr[1]; }
      }
#pragma unroll
      for (int j = 0; j < kOut; ++j) {
        const uint32_t vw = *reinterpret_cast<const uint32_t*>(sV + (8 * j + g8) * 16 + 4 * c) & keep;
        mma_half(o[j], pa, e4m3_pair(vw), e4m3_pair(vw >> 16));
      }
    }
  }

  __device__ __forceinline__ void put(float* to, int g8, int c) {
    constexpr int kStride = UnitParts<D, kNarrow>::kStride;
    const float down = v_up != 0.f ? 1.f / v_up : 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = kNarrow ? 2 * c + e : g8 + 8 * e;
      if constexpr (kNarrow) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 4);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 8);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 16);
#pragma unroll
        for (int j = 0; j < kOut; ++j) {
          to[r * kStride + 16 * j + g8] = o[j][e] * down;
          to[r * kStride + 16 * j + 8 + g8] = o[j][2 + e] * down;
        }
      } else {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
#pragma unroll
        for (int j = 0; j < kOut; ++j) *reinterpret_cast<float2*>(to + r * kStride + 8 * j + 2 * c) = make_float2(o[j][2 * e] * down, o[j][2 * e + 1] * down);
      }
      if ((kNarrow ? g8 : c) == 0) *reinterpret_cast<float2*>(to + 16 * kStride + 2 * r) = make_float2(m[e], l[e]);
    }
  }
};

// The pages page_lo .. page_hi - 1 of a table row by four warps in turn, through their rings (barriers initialised), into one part (UnitParts;
// all of it behind a block barrier).  `load` fills a UnitRows; what it reads is requested behind the first pages.
template <int D, bool kNarrow, typename Load>
__device__ __forceinline__ void unit_part(const SharedAttnArgs& a, uint8_t* smem, const int* bt, int kvh, int page_lo, int page_hi, int rows, Load load) {
  using L = SharedRing<D>;
  using P = UnitParts<D, kNarrow>;
  constexpr int kStages = L::kStages, kPart = P::kPart;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * kStages * L::kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kRing) + warp * kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kRing + 4 * kStages * 8);
  const int my_pages = page_hi > page_lo + warp ? (page_hi - page_lo - warp + 3) / 4 : 0;
  int next = lane == 0 && my_pages > 0 ? bt[page_lo + warp] : 0;
  const auto issue = [&](int i) {  // lane 0: start the copies of this warp's i-th page; its id was fetched a page ahead
    const int s = i % kStages;
    int page = next;
    if (i + 1 < my_pages) next = bt[page_lo + warp + 4 * (i + 1)];
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
  if (lane == 0)
    for (int i = 0; i < min(my_pages, kStages); ++i) issue(i);
  UnitRows<D, kNarrow> t;
  load(t, g8, c);
  for (int i = 0; i < my_pages; ++i) {
    const int s = i % kStages;
    if (!mbar_wait_warp(&full[s], (i / kStages) & 1, abort_flag, a.status, kStatusTimeoutEpilogue)) {
      let_started_work_end();
      break;
    }
    t.page(ring + s * L::kStage, (page_lo + warp + 4 * i) << 4, g8, c);
    __syncwarp();
    if (lane == 0 && i + kStages < my_pages) issue(i + kStages);
  }
  float* parts = reinterpret_cast<float*>(smem);  // the rings have been read
  __syncthreads();
  t.put(parts + warp * kPart, g8, c);
  __syncthreads();
  const int d = threadIdx.x % (D / 4) * 4;
#pragma unroll 4
  for (int r = threadIdx.x / (D / 4); r < rows; r += 512 / D) {
    float2 ml[4];
    float4 v[4], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      ml[w] = *reinterpret_cast<const float2*>(parts + w * kPart + 16 * P::kStride + 2 * r);
      v[w] = *reinterpret_cast<const float4*>(parts + w * kPart + r * P::kStride + d);
    }
    const float mm = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
    float ll = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float by = exp2f(ml[w].x - mm);
      ll += ml[w].y * by;
      acc.x += v[w].x * by; acc.y += v[w].y * by; acc.z += v[w].z * by; acc.w += v[w].w * by;
    }
    *reinterpret_cast<float4*>(parts + r * P::kStride + d) = acc;
    if (d == 0) *reinterpret_cast<float2*>(parts + P::kMl + 2 * r) = make_float2(mm, ll);
  }
}
template <int D>
__device__ __forceinline__ void unit_barriers(uint8_t* smem) {
  using L = SharedRing<D>;
  if (threadIdx.x == 0) *reinterpret_cast<volatile int*>(smem + L::kRing + 4 * L::kStages * 8) = 0;
  if ((threadIdx.x & 31) == 0) {
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kRing) + (threadIdx.x >> 5) * L::kStages;
    for (int s = 0; s < L::kStages; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
  }
  __syncthreads();
}

// The prefixes of groups with few query rows: blockIdx.x = one of the groups' tiles of 16 query rows (8, narrow), blockIdx.z = split.  Bound by a warp's
// chain of a page (products, maximum, exponentials, products), 0.5 to 1 us with three or four CTAs on an SM; up to some 32 query rows its tiles, which share an SM
// with tails, are ahead of one of 128 rows that needs an SM to itself (48 sequences in 5 groups with two heads of 64: 20.4 us against 25.2), with more behind it
// (16 sequences of four heads behind 5000 tokens: 35.6 against 21.3).
template <int D, bool kNarrow>
__global__ void __launch_bounds__(128, kNarrow ? 4 : 3)
shared_prefix_kernel(const SharedAttnArgs a) {
  using L = SharedRing<D>;
  constexpr int kTile = kNarrow ? 8 : 16;
  using P = UnitParts<D, kNarrow>;
  static_assert(L::kRing >= P::kEnd * 4, "the rings are the merge's scratch too");
  extern __shared__ __align__(128) uint8_t smem[];
  unit_barriers<D>(smem);
  pdl_wait();
  pdl_trigger();  // behind the wait: the tails, which may start now, read what this kernel's predecessors wrote
  const int kvh = blockIdx.y, G = a.Hq / a.Hk, per_seq = G * a.q_len, split = blockIdx.z;
  int group, tile;
  if (!find_tile(a, blockIdx.x, kTile, per_seq, group, tile)) return;
  const int first = min(max(a.group_starts[group], 0), a.B), rows = (min(max(a.group_starts[group + 1], first), a.B) - first) * per_seq;
  const int prefix = a.prefix_lens[group], table_row = member_row(a, first);  // (a group with a tile has a first row)
  int page_lo = 0, page_hi = 0;
  if (table_row >= 0) {
    const int n = min(max(prefix, 0) >> 4, a.max_pages), per = (n + a.prefix_splits - 1) / a.prefix_splits;
    page_lo = min(split * per, n);
    page_hi = min(n, page_lo + per);
  }
  const auto row_of = [&](int r) -> long long {
    const int i = tile * kTile + r, in = i % per_seq;
    const int row = r < kTile && i < rows ? member_row(a, first + i / per_seq) : -1;
    return row < 0 ? -1 : (static_cast<long long>(row) * a.q_len + in / G) * a.Hq + kvh * G + in % G;
  };
  const auto len_of = [&](int r) {
    const int i = tile * kTile + r;
    return a.seq_lens[member_row(a, first + i / per_seq)] - (a.q_len - 1 - i % per_seq / G);
  };
  const float* mine = reinterpret_cast<const float*>(smem);
  unit_part<D, kNarrow>(a, smem, a.table + size_t(max(table_row, 0)) * a.max_pages, kvh, page_lo, page_hi, kTile,
                        [&](UnitRows<D, kNarrow>& t, int g8, int c) { t.load(a, row_of, len_of, g8, c); });
  __syncthreads();
  for (int i = threadIdx.x; i < kTile * (D / 4); i += 128) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const long long row = row_of(r);
    if (row < 0) continue;
    const size_t part = row * a.slots + split;
    *reinterpret_cast<float4*>(a.part_o + part * D + d) = *reinterpret_cast<const float4*>(mine + r * P::kStride + d);
    if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = *reinterpret_cast<const float2*>(mine + P::kMl + 2 * r);
  }
}

constexpr int kMostSlots = 64, kMostRanks = 8;

// The tails (without prefix splits: whole sequences, each through its own table), and what comes of them and of the prefixes' partials: blockIdx.x = place,
// blockIdx.z = split of its pages; the splits of a place are one cluster.  Starts beside the prefixes (behind their wait) and waits for them with its own
// part done: as a kernel behind them, with another for the merge, the step that brought this took 64 sequences of 512 tokens behind 8192 from 77 to 51 us
// on a B200 (44 now).  They are at 0.9 of the rate of a copy while they read; whole sequences from L2 by the page's chain, 16 windows of heads of 256 and 3000 tokens 21.6 us.
template <int D, bool kNarrow>
__global__ void __launch_bounds__(128, D <= 128 ? (kNarrow ? 4 : 3) : (kNarrow ? 2 : 1))
shared_tail_kernel(const SharedAttnArgs a) {
  using L = SharedRing<D>;
  using P = UnitParts<D, kNarrow>;
  static_assert(L::kRing >= (P::kEnd + 16 * (kMostRanks + kMostSlots) + 16) * 4, "the rings are the merge's scratch too");
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_trigger();
  unit_barriers<D>(smem);
  if (a.prefix_splits == 0) pdl_wait();  // no prefixes' kernel has waited for what is read here
  const int place = blockIdx.x, kvh = blockIdx.y, ranks = gridDim.z, rank = blockIdx.z;
  const int G = a.Hq / a.Hk, rows = G * a.q_len;
  // requested side by side: the row and its length, the group and its prefix
  const int row = member_row(a, place), seq_len = a.seq_lens[max(row, 0)], group = group_of(a, place), grouped_from = a.group_starts[0];
  const bool grouped = group < a.groups && place >= grouped_from;
  if (row < 0 || !grouped) {  // the whole cluster alike
    if (grouped && threadIdx.x == 0) atomicCAS(a.status, 0, kStatusBadArgument);  // a member that is no row
    pdl_wait();  // this grid ends behind the prefixes' in any case
    return;
  }
  const int front = a.prefix_splits ? min(max(a.prefix_lens[group], 0) >> 4, a.max_pages) : 0;
  const int all = max(min(int((unsigned(max(seq_len, 0)) + 15u) >> 4), a.max_pages) - front, 0), per = (all + ranks - 1) / ranks;
  const int page_lo = front + min(all, rank * per), page_hi = front + min(all, (rank + 1) * per);
  float *mine = reinterpret_cast<float*>(smem), *weights = mine + P::kEnd, *inverse = weights + 16 * (kMostRanks + kMostSlots);
  const auto row_of = [&](int r) -> long long { return r < rows ? (static_cast<long long>(row) * a.q_len + r / G) * a.Hq + kvh * G + r % G : -1; };
  const auto len_of = [&](int r) { return seq_len - (a.q_len - 1 - r / G); };
  unit_part<D, kNarrow>(a, smem, a.table + size_t(row) * a.max_pages, kvh, page_lo, page_hi, rows,
                        [&](UnitRows<D, kNarrow>& t, int g8, int c) { t.load(a, row_of, len_of, g8, c); });
  if (ranks > 1) cluster_sync_all();
  else __syncthreads();
  pdl_wait();  // the prefixes' partials
  {  // weights of the ranks' parts and of the prefix's: eight threads to a row, all of its (m, l) requested before the first is used
    const int r = threadIdx.x >> 3, e8 = threadIdx.x & 7;
    constexpr int kEntries = 1 + kMostSlots / 8;  // a rank's, then slots'
    static_assert(kMostRanks == 8 && kMostSlots % 8 == 0);
    float2 ml[kEntries];
#pragma unroll
    for (int x = 0; x < kEntries; ++x) ml[x] = make_float2(kSharedNeg, 0.f);
    if (r < rows) {
      const float* prefix_ml = a.part_ml + 2 * (size_t(row_of(r)) * a.slots + e8);
      if (e8 < ranks) ml[0] = load_peer2(map_to_cta(mine + P::kMl + 2 * r, e8));
#pragma unroll
      for (int x = 1; x < kEntries; ++x)
        if (8 * (x - 1) + e8 < a.slots) ml[x] = *reinterpret_cast<const float2*>(prefix_ml + 16 * (x - 1));
    }
    float mm = kSharedNeg, sum = 0.f;
#pragma unroll
    for (int x = 0; x < kEntries; ++x)
      if (ml[x].y != 0.f) mm = fmaxf(mm, ml[x].x);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
#pragma unroll
    for (int x = 0; x < kEntries; ++x) {
      const float by = ml[x].y != 0.f ? exp2f(ml[x].x - mm) : 0.f;  // a part that saw nothing may hold anything
      sum += ml[x].y * by;
      if (r < rows && (x == 0 || 8 * (x - 1) + e8 < a.slots)) weights[r * (kMostRanks + kMostSlots) + 8 * x + e8] = by;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (r < rows && e8 == 0) inverse[r] = sum != 0.f ? 1.f / sum : 0.f;
  }
  __syncthreads();
  for (int i = rank * 128 + threadIdx.x; i < rows * (D / 4); i += ranks * 128) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const size_t hq = row_of(r);
    const float* by = weights + r * (kMostRanks + kMostSlots);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](const float4& v, float w) {
      if (w != 0.f) { acc.x += v.x * w; acc.y += v.y * w; acc.z += v.z * w; acc.w += v.w * w; }
    };
    float4 theirs[kMostRanks];
#pragma unroll
    for (int e = 0; e < kMostRanks; ++e)
      if (e < ranks) theirs[e] = load_peer(map_to_cta(mine + r * P::kStride + d, e));
#pragma unroll
    for (int e = 0; e < kMostRanks; ++e)
      if (e < ranks) add(theirs[e], by[e]);
    const float4* src = reinterpret_cast<const float4*>(a.part_o + hq * a.slots * D + d);  // (no slots: not read)
    for (int e = 0; e < a.slots; e += 8) {  // eight requested before the first is used; behind the last one the last again, for nothing
      float4 v[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] = __ldcg(src + min(e + x, a.slots - 1) * (D / 4));
#pragma unroll
      for (int x = 0; x < 8; ++x) add(v[x], e + x < a.slots ? by[kMostRanks + e + x] : 0.f);
    }
    const float n = inverse[r];
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(acc.x * n, acc.y * n), __floats2bfloat162_rn(acc.z * n, acc.w * n)};
    *reinterpret_cast<uint2*>(a.out + hq * D + d) = *reinterpret_cast<const uint2*>(h);
  }
  if (ranks > 1) cluster_sync_all();  // parts are read until here
}

template <typename K>
static bool set_smem(K kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (!done[dev] && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  return done[dev] = true;
}
template <int D, bool kNarrow>
static int launch_shared_prefix(const SharedAttnArgs& a, cudaStream_t stream) {
  static bool done[64] = {};
  if (!set_smem(shared_prefix_kernel<D, kNarrow>, SharedRing<D>::kSmem, done)) return -6;
  launch_kernel(shared_prefix_kernel<D, kNarrow>, dim3(tiles_at_most(a, kNarrow ? 8 : 16), a.Hk, a.prefix_splits), dim3(128), SharedRing<D>::kSmem, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}
template <int D, bool kNarrow>
static int launch_shared_tail(const SharedAttnArgs& a, cudaStream_t stream) {
  static bool done[64] = {};
  if (!set_smem(shared_tail_kernel<D, kNarrow>, SharedRing<D>::kSmem, done)) return -6;
  const dim3 grid(a.B, a.Hk, a.tail_splits);
  if (a.tail_splits > 1) launch_kernel_clustered(shared_tail_kernel<D, kNarrow>, grid, dim3(128), dim3(1, 1, a.tail_splits), SharedRing<D>::kSmem, stream, a);
  else launch_kernel(shared_tail_kernel<D, kNarrow>, grid, dim3(128), SharedRing<D>::kSmem, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}

int launch_shared_prefix_tc(const SharedAttnArgs& a, int dim, bool two_tiles, cudaStream_t stream);  // attn_shared_tc.cu

template <int D>
static int launch_shared(const SharedAttnArgs& a, int tile, cudaStream_t stream) {
  int rc = 0;
  if constexpr (D <= 128) {
    if (a.prefix_splits)
      rc = tile == 8 ? launch_shared_prefix<D, true>(a, stream) : tile == 16 ? launch_shared_prefix<D, false>(a, stream) : launch_shared_prefix_tc(a, D, tile == 256, stream);
  }
  if (rc) return rc;
  return (a.Hq / a.Hk) * a.q_len <= 8 ? launch_shared_tail<D, true>(a, stream) : launch_shared_tail<D, false>(a, stream);
}

}  // namespace mfq

// q, out: [B * q_len, Hq, D] bf16; pages of the FP8 pool, `pages` of them; group_starts [groups + 1], prefix_lens [groups], members [B] or null; tile: query rows of a
// prefix CTA, 8, 16, 128 or 256; partials [B * q_len * Hq * slots] x D and x 2 floats, slots = prefix_splits (twice that for a tile of 128), 64 at most;
// prefix_splits: 0 has every sequence read whole through its own table (heads of 256: always); tail_splits: 8 at most.  (Hq / Hk) * q_len <= 16.
// q, out, pages and multipliers lie on 16 bytes.  Rows in no group are not written.
extern "C" int mfq_paged_attn_decode_shared(const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale, const int* table,
                                            const int* seq_lens, const int* group_starts, const int* prefix_lens, const int* members, void* out,
                                            float* part_o, float* part_ml, int B, int Hq, int Hk, int D, int max_pages, int pages, int groups, int q_len,
                                            int tile, int prefix_splits, int tail_splits, float sm_scale, int* status, cudaStream_t stream) {
  using namespace mfq;
  if (B <= 0 || B > 65535 || Hk <= 0 || Hk > 65535 || Hq % Hk || q_len < 1 || (Hq / Hk) * q_len > 16 || groups < 1 || groups > B || pages < 1 || max_pages < 1 || max_pages >= 1 << 27)
    return -1;
  if (prefix_splits < 0 || prefix_splits * (tile == 128 ? 2 : 1) > kMostSlots || tail_splits < 1 || tail_splits > kMostRanks) return -1;
  if (prefix_splits && (D > 128 || (tile != 8 && tile != 16 && tile != 128 && tile != 256))) return -1;
  for (const void* p : {q, k, v, static_cast<const void*>(k_scale), static_cast<const void*>(v_scale), static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return -1;
  const SharedAttnArgs a{static_cast<const __nv_bfloat16*>(q), static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), k_scale, v_scale, table, seq_lens,
                         group_starts, prefix_lens, members, part_o, part_ml, static_cast<__nv_bfloat16*>(out), status, B, Hq, Hk, max_pages, pages, groups,
                         q_len, prefix_splits * (tile == 128 ? 2 : 1), prefix_splits, tail_splits, sm_scale * 1.4426950408889634f};
  if (D == 128) return launch_shared<128>(a, tile, stream);
  if (D == 256) return launch_shared<256>(a, tile, stream);
  if (D == 64) return launch_shared<64>(a, tile, stream);
  return -1;
}
