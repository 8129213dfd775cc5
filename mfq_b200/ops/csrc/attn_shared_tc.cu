// The prefixes of attn_shared.cu on tcgen05, for groups with many query rows (heads of 64 and 128).
//
// One CTA = 128 or 256 query rows of a group, one KV head, one split of the prefix, in two streams that take turns on the tensor core: two
// tiles of 128 rows over the same keys (kTwoTiles), or one tile over the even and the odd blocks of 128 keys.  Per stream and block:
//   S = Q K^T       tcgen05.mma kind::f16, Q and K from shared memory (K-major, 128-byte swizzle), S in tensor memory
//   t = S ks + lv   ks: the key's multiplier times scale log2 e, lv = log2 of its V multiplier, so that P = 2^(t - m) has the V multiplier in it and
//                   stays in [0, 2^12] however the multipliers are spread; the sum of the softmax takes P / V multiplier, in fp32
//   O += P V        P as fp16 pairs over the first half of its S, V codes K-major ([dim][key], what a page holds), O in tensor memory
// m moves only where a row's maximum has grown by more than 2^8 since (O is then rescaled in place): as any m gives the same quotient, this costs no exactness.
// A warp takes tensor memory as matrix fragments: four lanes share a row and a lane has two columns of each eight, so that what belongs to
// columns is read from shared memory once for 16 rows; with a row per thread those reads alone took as long as the products.
// Four warps bring the codes of the next block to registers while the tensor core has the present ones, and put them down as fp16 (exact).
//
// Per block of 128 x 128 the tensor core and the exponentials both need 1024 cycles of an SM, shared memory (operands, codes) some 1250.
#include "attn_shared.cuh"

namespace mfq {

constexpr int kTcThreads = 512, kTcBlock = 128;
constexpr float kTcRoom = 4.f, kTcGrowth = 12.f;  // P begins at most at 2^4, where fp16 reaches 2^-28 of it, and may grow to 2^12
constexpr float kTcFloor = -5e29f, kTcMasked = -1e30f;  // below every score; what masked keys have (2^(kTcMasked - kTcFloor) = 0)

template <int D>
struct SharedTc {
  static constexpr int kTile = kTcBlock * D * 2;  // Q or K: D / 64 slices of [128 rows][128 bytes]; V: two slices of [D dims][64 keys]
  static constexpr int kConst = 6 * kTile;        // behind two Q, two stages of K, two of V
  static constexpr int kRowAt = kConst + 2 * (64 * 16 + 64 * 8);
  static constexpr int kBarsAt = kRowAt + 3 * 256 * 4;
  static constexpr int kSmem = kBarsAt + 256 + 1024;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D (+)= A B over 64 keys: A [128 x 64] fp16 in tensor memory (8 columns a k-step of 16), B K-major (32 bytes a k-step).  Whole warp, one elected lane issues.
__device__ __forceinline__ void umma_p_v(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred q, f, t;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
      "setp.ne.b32 f, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, f;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}"
      ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float u2f(uint32_t v) { return __uint_as_float(v); }

// 16 codes as fp16 in the order given: 32 bytes at two 16-byte places
__device__ __forceinline__ void put_halves(uint8_t* lo, uint8_t* hi, const uint32_t (&h)[8]) {
  *reinterpret_cast<uint4*>(lo) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4*>(hi) = make_uint4(h[4], h[5], h[6], h[7]);
}

template <int D, bool kTwoTiles>
__global__ void __launch_bounds__(kTcThreads, 1)
shared_attn_tc_kernel(const SharedAttnArgs a) {
  using L = SharedTc<D>;
  constexpr int kTile = L::kTile, kSlices = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = base, *sK = base + 2 * kTile, *sV = base + 4 * kTile;
  float4* s_col = reinterpret_cast<float4*>(base + L::kConst);          // [2 stages][64 column pairs]: ks, ks, lv, lv
  float2* s_inv = reinterpret_cast<float2*>(base + L::kConst + 2048);   // [2][64]: 1 / V multiplier
  float* s_rowc = reinterpret_cast<float*>(base + L::kRowAt);           // [256] power of two that the row's q was divided by
  int* s_len = reinterpret_cast<int*>(s_rowc + 256);                    // [256] keys that the row sees
  int* s_hq = s_len + 256;                                              // [256] row of the outputs, -1: none
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::kBarsAt);
  uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;  // [2 stages]
  uint64_t *s_full = bars + 8, *p_full = bars + 10, *o_full = bars + 12, *q_full = bars + 14;  // [2 streams], q_full: 8 warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_low = reinterpret_cast<int*>(tmem_slot + 2);  // fewest and most keys that a row of the CTA sees
  int* s_most = s_low + 1;
  int* s_scaled = s_low + 2;  // whether a row's q was scaled

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 4); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1);
    }
    mbar_init(q_full, 8);
    *abort_flag = 0;
    *s_low = 0x7fffffff;
    *s_most = 0;
    *s_scaled = 0;
    mbar_fence_init();
  }
  if (warp == 0) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);  // columns: S of the two streams, 128 each (P in the first 64), then their O
  pdl_trigger();  // TMEM is held by now
  pdl_wait();

  const int kvh = blockIdx.y, G = a.Hq / a.Hk, per_seq = G * a.q_len, split = blockIdx.z;
  int group = 0, tile = 0;
  const bool mine = find_tile(a, blockIdx.x, kTwoTiles ? 256 : 128, per_seq, group, tile);
  int first = 0, rows = 0, table_row = -1, page_lo = 0, page_hi = 0;
  if (mine) {
    first = min(max(a.group_starts[group], 0), a.B);
    rows = (min(max(a.group_starts[group + 1], first), a.B) - first) * per_seq;
    table_row = member_row(a, first);
    if (table_row >= 0) {
      const int n = min(max(a.prefix_lens[group], 0) >> 4, a.max_pages), per = (n + a.prefix_splits - 1) / a.prefix_splits;
      page_lo = min(split * per, n);
      page_hi = min(n, page_lo + per);
    }
  }
  // rows of the streams: what each sees
  if (warp >= 8) {
    const int i = threadIdx.x - 256, r = tile * (kTwoTiles ? 256 : 128) + (kTwoTiles ? i : i & 127);
    int hq = -1, len = 0x7fffffff;
    if (mine && r < rows) {
      const int row = member_row(a, first + r / per_seq), in = r % per_seq, qr = in / G;
      if (row >= 0) {
        hq = (row * a.q_len + qr) * a.Hq + kvh * G + in % G;
        len = a.seq_lens[row] - (a.q_len - 1 - qr);
        atomicMin(s_low, len);
        atomicMax(s_most, len);
      }
    }
    s_hq[i] = hq;
    s_len[i] = len;
  }
  __syncthreads();
  // keys of this CTA: whole pages of its split, none behind what its rows see; blocks of 128
  const int key_lo = page_lo * 16, key_hi = min(page_hi * 16, *s_most);
  const int steps = key_hi > key_lo ? (key_hi - key_lo + kTcBlock - 1) / kTcBlock : 0;
  const int turns = kTwoTiles ? 2 * steps : steps;  // turn u: stream u & 1

  if (warp < 4) {
    if (warp == 0 && steps > 0) {
      constexpr uint32_t idesc_qk = umma_idesc(128, 128, 0, 0), idesc_pv = umma_idesc(128, D, 0, 0);
      constexpr uint64_t kT = kTile >> 4, kQkSlice = (kTcBlock * 128) >> 4, kPvSlice = (D * 128) >> 4;
      const uint64_t q_desc = umma_desc_k_sw128(smem_u32(sQ)), k_desc = umma_desc_k_sw128(smem_u32(sK)), v_desc = umma_desc_k_sw128(smem_u32(sV));
      const auto step_of = [&](int u) { return kTwoTiles ? u >> 1 : u; };
      bool ok = mbar_wait_warp(q_full, 0, abort_flag, a.status, kStatusTimeoutMma);
      const auto issue_qk = [&](int u) {
        const int t = u & 1, s = step_of(u) & 1;
        ok = ok && mbar_wait_warp(&k_full[s], (step_of(u) >> 1) & 1, abort_flag, a.status, kStatusTimeoutMma);
        if (!ok) return;
        tc_fence_after();
        const uint64_t qd = q_desc + uint64_t(t) * kT, kd = k_desc + uint64_t(s) * kT;
        const uint32_t d = tmem_base + uint32_t(t) * 128u;
#pragma unroll
        for (int h = 0; h < kSlices; ++h) umma_f16_block(d, qd + h * kQkSlice, kd + h * kQkSlice, idesc_qk, h ? 1u : 0u);
        tc_commit_warp(&s_full[t]);
        if (!kTwoTiles || t == 1) tc_commit_warp(&k_empty[s]);
      };
      if (ok) issue_qk(0);
      if (ok && turns > 1) issue_qk(1);
      for (int u = 0; ok && u < turns; ++u) {
        const int t = u & 1, j = u >> 1, s = step_of(u) & 1;  // j: block of the stream
        ok = mbar_wait_warp(&v_full[s], (step_of(u) >> 1) & 1, abort_flag, a.status, kStatusTimeoutMma) &&
             mbar_wait_warp(&p_full[t], j & 1, abort_flag, a.status, kStatusTimeoutMma);
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = v_desc + uint64_t(s) * kT;
        const uint32_t p = tmem_base + uint32_t(t) * 128u, d = tmem_base + 256u + uint32_t(t) * D;
        umma_p_v(d, p, vd, idesc_pv, j > 0 ? 1u : 0u);
        umma_p_v(d, p + 32u, vd + kPvSlice, idesc_pv, 1u);
        if (!kTwoTiles || t == 1) tc_commit_warp(&v_empty[s]);
        if (u + 2 >= turns) tc_commit_warp(&o_full[t]);
        else issue_qk(u + 2);  // S takes the place of P, which the products before have read
      }
    }
  } else if (warp < 8) {
    // ----- codes to fp16: thread i has 16 bytes of each page's K and V -----
    const int i = threadIdx.x - 128;
    constexpr int kVecs = D / 16;          // 16-byte pieces of K (and of V) per thread and block
    constexpr int kPerPage = 128 * kVecs / 8;  // ... per page
    const int* bt = a.table + size_t(max(table_row, 0)) * a.max_pages;
    uint4 k_raw[kVecs], v_raw[kVecs];
    float ks = 0.f, vs = 0.f;
    const auto page_at = [&](int n) {
      const int at = page_lo + n;
      if (at * 16 >= key_hi) return -1;
      const int page = bt[at];
      if (page >= 0 && page < a.pages) return page;
      atomicCAS(a.status, 0, kStatusBadArgument);
      return 0;
    };
    const auto fetch = [&](int step) {
#pragma unroll
      for (int n = 0; n < kVecs; ++n) {
        const int v = i + 128 * n, page = page_at(step * 8 + v / kPerPage);
        const size_t at = (size_t(max(page, 0)) * a.Hk + kvh) * (16 * D) + (v % kPerPage) * 16;
        k_raw[n] = v_raw[n] = make_uint4(0, 0, 0, 0);
        if (page >= 0) {
          k_raw[n] = *reinterpret_cast<const uint4*>(a.k + at);
          v_raw[n] = *reinterpret_cast<const uint4*>(a.v + at);
        }
      }
      const int page = page_at(step * 8 + i / 16);
      ks = vs = 0.f;
      if (page >= 0 && key_lo + step * kTcBlock + i < key_hi) {
        const size_t at = (size_t(page) * a.Hk + kvh) * 16 + (i & 15);
        ks = a.k_scale[at];
        vs = a.v_scale[at];
      }
    };
    if (steps > 0) fetch(0);
    bool ok = true;
    for (int step = 0; step < steps; ++step) {
      const int s = step & 1;
      const uint32_t parity = ((step >> 1) & 1) ^ 1;
      const int key0 = key_lo + step * kTcBlock, left = key_hi - key0;  // keys of the block
      ok = mbar_wait_warp(&k_empty[s], parity, abort_flag, a.status, kStatusTimeoutProducer);
      if (!ok) break;
#pragma unroll
      for (int n = 0; n < kVecs; ++n) {
        const int v = i + 128 * n, in = v % kPerPage, key = v / kPerPage * 16 + in / 4 % 16, slice = in / 64, c = in & 3;
        uint32_t w[4] = {k_raw[n].x, k_raw[n].y, k_raw[n].z, k_raw[n].w};
        if (key >= left) w[0] = w[1] = w[2] = w[3] = 0;
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) { h[2 * e] = e4m3_pair(w[e]); h[2 * e + 1] = e4m3_pair(w[e] >> 16); }
        uint8_t* at = sK + s * kTile + slice * (kTcBlock * 128) + key * 128;
        put_halves(at + (((2 * c) ^ (key & 7)) << 4), at + (((2 * c + 1) ^ (key & 7)) << 4), h);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[s]);
      ok = mbar_wait_warp(&v_empty[s], parity, abort_flag, a.status, kStatusTimeoutProducer);
      if (!ok) break;
#pragma unroll
      for (int n = 0; n < kVecs; ++n) {
        const int v = i + 128 * n, page = v / kPerPage, dim = v % kPerPage;
        uint32_t w[4] = {v_raw[n].x, v_raw[n].y, v_raw[n].z, v_raw[n].w};
        const int keys = left - page * 16;
        if (keys < 16) {  // bytes of word e: keys 2e, 2e + 1, 2e + 8, 2e + 9
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t keep = 0;
            for (int x = 0; x < 4; ++x)
              if (2 * e + (x & 1) + 8 * (x >> 1) < keys) keep |= 0xffu << (8 * x);
            w[e] &= keep;
          }
        }
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) { h[e] = e4m3_pair(w[e]); h[4 + e] = e4m3_pair(w[e] >> 16); }
        uint8_t* at = sV + s * kTile + (page >> 2) * (D * 128) + dim * 128;
        const int c = 2 * (page & 3);
        put_halves(at + ((c ^ (dim & 7)) << 4), at + (((c + 1) ^ (dim & 7)) << 4), h);
      }
      {  // columns i: pair (i / 8, i % 8 / 2); a key that is not there has P = 0
        const bool there = i < left;
        const float up = fmaxf(vs, 7.888609e-31f);  // 2^-100: a multiplier of zero gives values of zero, and a finite quotient
        float* col = reinterpret_cast<float*>(s_col + s * 64 + (i >> 3) * 4 + ((i & 7) >> 1)) + (i & 1);
        col[0] = there ? ks * a.scale_log2 : 0.f;
        col[2] = there ? (isnan(vs) ? vs : log2f(up)) : kTcMasked;
        reinterpret_cast<float*>(s_inv + s * 64 + (i >> 3) * 4 + ((i & 7) >> 1))[i & 1] = there ? 1.f / up : 0.f;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[s]);
      if (step + 1 < steps) fetch(step + 1);
    }
  } else {
    // ----- softmax: warps 8 - 11 stream 0, 12 - 15 stream 1; a warp has 32 rows, a lane parts of four of them -----
    const int t = (warp - 8) >> 2, quarter = warp & 3, c = lane & 3;
    uint8_t* tile_q = sQ + t * kTile;
    {  // this thread's row of Q to fp16: as it is where its largest value is between 2^-4 and 2^15 (exact down to 2^-21 of that), else scaled to 2^13
      const int r = quarter * 32 + lane, hq = s_hq[t * 128 + r];
      float top = 0.f;
      uint4 raw[D / 8];
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        raw[n] = hq >= 0 ? *reinterpret_cast<const uint4*>(a.q + size_t(hq) * D + n * 8) : make_uint4(0, 0, 0, 0);
        const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(&raw[n]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(__bfloat162float(b[e])));
      }
      const float up = top == 0.f || (top >= 0.0625f && top < 32768.f) ? 1.f : power_to(top, 13);
      s_rowc[t * 128 + r] = 1.f / up;
      if (up != 1.f) atomicOr(s_scaled, 1);
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(&raw[n]);
        uint4 h;
        h.x = half_pair(__bfloat162float(b[0]) * up, __bfloat162float(b[1]) * up);
        h.y = half_pair(__bfloat162float(b[2]) * up, __bfloat162float(b[3]) * up);
        h.z = half_pair(__bfloat162float(b[4]) * up, __bfloat162float(b[5]) * up);
        h.w = half_pair(__bfloat162float(b[6]) * up, __bfloat162float(b[7]) * up);
        *reinterpret_cast<uint4*>(tile_q + (n >> 3) * (kTcBlock * 128) + r * 128 + (((n & 7) ^ (r & 7)) << 4)) = h;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const uint32_t tS = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(t) * 128u, tO = tmem_base + (uint32_t(quarter * 32) << 16) + 256u + uint32_t(t) * D;
    const int row0 = t * 128 + quarter * 32 + (lane >> 2);  // and 8, 16, 24 further
    float m[4], l[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) { m[x] = kTcFloor; l[x] = 0.f; }
    bool ok = mbar_wait_warp(q_full, 0, abort_flag, a.status, kStatusTimeoutEpilogue);  // s_scaled is final
    const bool special = *s_scaled != 0 || *s_low < key_hi;  // a row was scaled, or does not see all keys
    const int blocks = kTwoTiles ? steps : (steps + 1 - t) >> 1;
    for (int j = 0; ok && j < blocks; ++j) {
      const int step = kTwoTiles ? j : 2 * j + t, st = step & 1;
      ok = mbar_wait_warp(&v_full[st], (step >> 1) & 1, abort_flag, a.status, kStatusTimeoutEpilogue) &&
           mbar_wait_warp(&s_full[t], j & 1, abort_flag, a.status, kStatusTimeoutEpilogue);
      if (!ok) break;
      tc_fence_after();
      const float4* col = s_col + st * 64 + c;
      const float2* inv = s_inv + st * 64 + c;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // rows 0 - 15 and 16 - 31 of the warp: 64 scores a lane at a time
        const uint32_t tSh = tS + (uint32_t(16 * h) << 16), tOh = tO + (uint32_t(16 * h) << 16);
        uint32_t x[64];
        tmem_ld_frag128(tSh, x);
        tmem_wait_ld();
        if (special) {
          const float lo = s_rowc[row0 + 16 * h], hi = s_rowc[row0 + 16 * h + 8];
#pragma unroll
          for (int n = 0; n < 64; ++n) x[n] = __float_as_uint(u2f(x[n]) * (n & 2 ? hi : lo));
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const float4 k = col[u * 4];
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float2 v = fma_f2(make_float2(u2f(x[4 * u + e]), u2f(x[4 * u + e + 1])), make_float2(k.x, k.y), make_float2(k.z, k.w));
            x[4 * u + e] = __float_as_uint(v.x);
            x[4 * u + e + 1] = __float_as_uint(v.y);
          }
        }
        if (special) {
          const int key = key_lo + step * kTcBlock + 2 * c, lo = s_len[row0 + 16 * h] - key, hi = s_len[row0 + 16 * h + 8] - key;
#pragma unroll
          for (int n = 0; n < 64; ++n)
            if (8 * (n >> 2) + (n & 1) >= (n & 2 ? hi : lo)) x[n] = __float_as_uint(kTcMasked);
        }
        float mx[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = fmaxf(u2f(x[2 * e]), u2f(x[2 * e + 1]));
#pragma unroll
          for (int u = 1; u < 16; ++u) v = fmaxf(fmaxf(v, u2f(x[4 * u + 2 * e])), u2f(x[4 * u + 2 * e + 1]));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          mx[e] = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
        }
        if (j == 0) {
          m[2 * h] = fmaxf(mx[0] - kTcRoom, kTcFloor);
          m[2 * h + 1] = fmaxf(mx[1] - kTcRoom, kTcFloor);
        } else if (__any_sync(0xffffffffu, mx[0] > m[2 * h] + kTcGrowth || mx[1] > m[2 * h + 1] + kTcGrowth)) {
          // the product before is complete: it was issued ahead of the one that S came from
          float by[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float now = fmaxf(m[2 * h + e], mx[e] - kTcRoom);
            by[e] = exp2_fast(m[2 * h + e] - now);
            l[2 * h + e] *= by[e];
            m[2 * h + e] = now;
          }
#pragma unroll
          for (int d = 0; d < D; d += 32) {
            uint32_t o[16];
            tmem_ld_frag32(tOh + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(u2f(o[n]) * by[n >> 1 & 1]);
            tmem_st_frag32(tOh + d, o);
          }
        }
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t p[32];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const float2 iv = inv[u * 4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 pe = make_float2(exp2_fast(u2f(x[4 * u + 2 * e]) - m[2 * h + e]), exp2_fast(u2f(x[4 * u + 2 * e + 1]) - m[2 * h + e]));
            sum[e] = fma_f2(pe, iv, sum[e]);
            p[2 * u + e] = half_pair(pe.x, pe.y);
          }
        }
        l[2 * h] += sum[0].x + sum[0].y;
        l[2 * h + 1] += sum[1].x + sum[1].y;
        tmem_st_pairs(tSh, p);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok && blocks > 0) {
      ok = mbar_wait_warp(&o_full[t], 0, abort_flag, a.status, kStatusTimeoutEpilogue);
      tc_fence_after();
    }
    if (ok && mine) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      }
      const int slot = kTwoTiles ? split : 2 * split + t;
      size_t at[4];
      bool live[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int hq = s_hq[row0 + 8 * r];
        live[r] = hq >= 0;
        at[r] = size_t(max(hq, 0)) * a.slots + slot;
        if (live[r] && c == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at[r]) = make_float2(m[r], l[r]);
      }
      if (blocks > 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int d = 0; d < D; d += 32) {
            uint32_t o[16];
            tmem_ld_frag32(tO + (uint32_t(16 * h) << 16) + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int n = 0; n < 16; n += 2) {
              const int r = 2 * h + (n >> 1 & 1);
              if (live[r]) *reinterpret_cast<float2*>(a.part_o + at[r] * D + d + 8 * (n >> 2) + 2 * c) = make_float2(u2f(o[n]), u2f(o[n + 1]));
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem_base, 512);
}

template <int D, bool kTwoTiles>
static int launch_tc(const SharedAttnArgs& a, cudaStream_t stream) {
  auto kernel = &shared_attn_tc_kernel<D, kTwoTiles>;
  static bool attr[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -6;
  if (!attr[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SharedTc<D>::kSmem) != cudaSuccess) return -6;
    attr[dev] = true;
  }
  const int per_tile = kTwoTiles ? 256 : 128;
  launch_kernel(kernel, dim3(a.B * (a.Hq / a.Hk) * a.q_len / per_tile + a.groups, a.Hk, a.prefix_splits), dim3(kTcThreads), SharedTc<D>::kSmem, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}

int launch_shared_prefix_tc(const SharedAttnArgs& a, int dim, bool two_tiles, cudaStream_t stream) {
  if (dim == 128) return two_tiles ? launch_tc<128, true>(a, stream) : launch_tc<128, false>(a, stream);
  if (dim == 64) return two_tiles ? launch_tc<64, true>(a, stream) : launch_tc<64, false>(a, stream);
  return -1;
}

}  // namespace mfq
