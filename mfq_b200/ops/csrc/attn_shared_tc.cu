// The prefixes of attn_shared.cu on tcgen05, for groups with many query rows (heads of 64 and 128).
//
// One CTA = 128 or 256 query rows of a group, one KV head, one split of the prefix, in two streams that take turns on the tensor core: two
// tiles of 128 rows over the same keys (kTwoTiles), or one tile over the even and the odd blocks of 128 keys.  Per stream and block:
//   S = Q K^T       tcgen05.mma kind::f16, Q and K from shared memory (K-major, 128-byte swizzle), S in tensor memory
//   t = S ks + lv   ks: the key's multiplier times scale log2 e, lv = log2 of its V multiplier, so that P = 2^(t - m) has the V multiplier in it and
//                   stays in [0, 2^15] however the multipliers are spread; the sum of the softmax takes P / V multiplier, in fp32
//   O += P V        P as fp16 pairs, those of 64 keys over the first half of their S, V codes K-major ([dim][key], what a page holds), O in tensor memory
// m moves only where a row's maximum has grown by more than 2^11 since (O is then rescaled in place): as any m gives the same quotient, this costs no exactness.
// A warp takes tensor memory as matrix fragments: four lanes share a row and a lane has two columns of each eight, so that what belongs to
// columns is read from shared memory once for 32 rows.  It goes over S twice, 16 columns at a time, and two warps share the keys of a block and exchange
// their maxima (16 rows and all keys a warp: no exchange, twice the reads for columns, 2 % slower): registers for a whole block spilled, and the code of all
// roles together has to stay within the instruction cache (unrolled, a step took 9000 cycles, a third of them without an instruction).
// Seven warps put down codes as fp16 (exact) from rings of pages that bulk copies fill: loads to registers have to pass the few KB of L1 that such a CTA leaves,
// and took 4000 cycles a block.
//
// Per block of 128 x 128 the tensor core and the exponentials both need 1024 cycles of an SM, shared memory (operands, codes) some 1250.  A step of two
// tiles takes 5800 on a B200: a stream's softmax (3300 to 3900) and its products with their issue (1600) follow one another, and the two streams fill each
// other's gaps as far as that goes.  4.8 us pass from the launch to the first scores, some 5 from the last ones to the end.  64 sequences of 32 heads on 8 behind
// 32768 tokens: 65 us, of 21 for its operations at the measured rate; behind 8192 tokens 28.
#include "attn_shared.cuh"

namespace mfq {

constexpr int kTcBlock = 128;
constexpr int kTcThreads = 24 * 32;  // warps 0 - 3 bring K, 4 - 6 V, 7 issues products, 8 - 23 have the softmax
constexpr float kTcRoom = 4.f, kTcGrowth = 15.f;  // P begins at most at 2^4, where fp16 reaches 2^-28 of it, and may grow to 2^15
constexpr float kTcFloor = -5e29f, kTcMasked = -1e30f;  // below every score; what masked keys have (2^(kTcMasked - kTcFloor) = 0)

template <bool kYes>
struct Special {
  static constexpr bool value = kYes;
};

template <int D>
struct SharedTc {
  static constexpr int kTile = kTcBlock * D * 2;  // Q or K: D / 64 slices of [128 rows][128 bytes]; V: two slices of [D dims][64 keys]
  static constexpr int kVPage = 16 * D, kKPage = kVPage + 128;  // a page's V, its K and both multipliers, as they lie in the pool
  static constexpr int kKDepth = 3, kVDepth = 4;  // pages that a loading warp has under way
  static constexpr int kKRing = 5 * kTile;        // behind two Q, K and two stages of V: a ring for each of four warps, then of three
  static constexpr int kVRing = kKRing + 4 * kKDepth * kKPage;
  static constexpr int kConst = kVRing + 3 * kVDepth * kVPage, kConsts = 4;  // what belongs to columns: of four blocks
  static constexpr int kRowAt = kConst + kConsts * (64 * 16 + 64 * 8);
  static constexpr int kBarsAt = kRowAt + 7 * 256 * 4;
  static constexpr int kBars = 28 + 4 * kKDepth + 3 * kVDepth;
  static constexpr int kSmem = kBarsAt + kBars * 8 + 64 + 1024;
  static_assert(kSmem <= 227 * 1024 && kTile % 1024 == 0 && kConst % 16 == 0);
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
  uint8_t *sQ = base, *sK = base + 2 * kTile, *sV = base + 3 * kTile;
  float4* s_col = reinterpret_cast<float4*>(base + L::kConst);          // [block % 4][64 column pairs]: ks, ks, lv, lv
  float2* s_inv = reinterpret_cast<float2*>(s_col + L::kConsts * 64);   // [block % 4][64]: 1 / V multiplier
  float* s_rowc = reinterpret_cast<float*>(base + L::kRowAt);           // [256] power of two that the row's q was divided by
  int* s_len = reinterpret_cast<int*>(s_rowc + 256);                    // [256] keys that the row sees
  int* s_hq = s_len + 256;                                              // [256] row of the outputs, -1: none
  float* s_max = reinterpret_cast<float*>(s_hq + 256);                  // [2][2 halves][256] maxima of even and odd blocks, at last the sums
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::kBarsAt);
  uint64_t *k_full = bars, *k_empty = bars + 1, *v_full = bars + 2, *v_empty = bars + 4, *q_full = bars + 6;  // v: [2 stages]
  uint64_t *c_full = bars + 8;                                             // [block % 4] what belongs to the columns
  uint64_t *s_full = bars + 12, *p_full = bars + 14, *o_full = bars + 16;  // [2 streams]
  uint64_t* x_bar = bars + 18;                                             // [2 streams][4 quarters] two warps have put down their maxima
  uint64_t* ring_full = bars + 28;                                         // [4][kKDepth], [3][kVDepth]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_low = reinterpret_cast<int*>(tmem_slot + 2);  // fewest and most keys that a row of the CTA sees
  int* s_most = s_low + 1;
  int* s_scaled = s_low + 2;  // whether a row's q was scaled

  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(k_full, 4); mbar_init(k_empty, 1); mbar_init(q_full, 16);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v_full[i], 3); mbar_init(&v_empty[i], 1); mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 8); mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < L::kConsts; ++i) mbar_init(&c_full[i], 4);
    for (int i = 0; i < 8; ++i) mbar_init(&x_bar[i], 2);
    for (int i = 0; i < 4 * L::kKDepth + 3 * L::kVDepth; ++i) mbar_init(&ring_full[i], 1);
    *abort_flag = 0;
    *s_low = 0x7fffffff;
    *s_most = 0;
    *s_scaled = 0;
    mbar_fence_init();
  }
  pdl_wait();
  const int kvh = blockIdx.y, G = a.Hq / a.Hk, per_seq = G * a.q_len, split = blockIdx.z;
  int group = 0, tile = 0;
  if (!find_tile(a, blockIdx.x, kTwoTiles ? 256 : 128, per_seq, group, tile)) return;  // all threads alike
  if (warp == 7) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);  // columns: S of the two streams, 128 each, then their O
  pdl_trigger();  // TMEM is held by now
  const int first = min(max(a.group_starts[group], 0), a.B), rows = (min(max(a.group_starts[group + 1], first), a.B) - first) * per_seq;
  const int table_row = member_row(a, first);
  int page_lo = 0, page_hi = 0;
  if (table_row >= 0) {
    const int n = min(max(a.prefix_lens[group], 0) >> 4, a.max_pages), per = ((n + 7) / 8 + a.prefix_splits - 1) / a.prefix_splits * 8;  // whole blocks
    page_lo = min(split * per, n);
    page_hi = min(n, page_lo + per);
  }
  // ----- the loaders: four warps take K of every fourth page, three V of every third, through rings of their own -----
  const bool of_k = warp < 4;
  const int lanes = of_k ? 4 : 3, w = of_k ? warp : warp - 4, depth = of_k ? L::kKDepth : L::kVDepth, page_bytes = of_k ? L::kKPage : L::kVPage;
  uint8_t* ring = base + (of_k ? L::kKRing + w * L::kKDepth * L::kKPage : L::kVRing + w * L::kVDepth * L::kVPage);
  uint64_t* ring_bar = ring_full + (of_k ? w * L::kKDepth : 4 * L::kKDepth + w * L::kVDepth);
  const int own_pages = max(0, (page_hi - page_lo - w + lanes - 1) / lanes);
  const int* bt = a.table + size_t(max(table_row, 0)) * a.max_pages;
  int next_id = 0, asked = 0;  // one lane: the page that is requested next, and how many were
  const auto request = [&](int slot) {  // one lane: copies of the warp's next page; its id was fetched a page ahead
    int id = next_id;
    if (++asked < own_pages) next_id = bt[page_lo + w + lanes * asked];
    if (id < 0 || id >= a.pages) {
      atomicCAS(a.status, 0, kStatusBadArgument);
      id = 0;
    }
    const size_t ph = size_t(id) * a.Hk + kvh;
    uint8_t* to = ring + slot * page_bytes;
    uint64_t* bar = &ring_bar[slot];
    mbar_expect_tx(bar, page_bytes);
    shared_bulk_load(to, (of_k ? a.k : a.v) + ph * (16 * D), 16 * D, bar);
    if (of_k) {
      shared_bulk_load(to + 16 * D, a.k_scale + ph * 16, 64, bar);
      shared_bulk_load(to + 16 * D + 64, a.v_scale + ph * 16, 64, bar);
    }
  };
  if (warp < 7) {
    if (lane == 0 && own_pages > 0) {  // ahead of what the rows see
      next_id = bt[page_lo + w];
      for (int n = 0; n < min(own_pages, depth); ++n) request(n);
    }
    asked = __shfl_sync(0xffffffffu, asked, 0);
  } else if (warp >= 8 && !((warp - 8) & 4)) {
    const int x = ((warp - 8) >> 3) * 128 + (warp & 3) * 32 + lane, r = tile * (kTwoTiles ? 256 : 128) + (kTwoTiles ? x : x & 127);
    int hq = -1, len = 0x7fffffff;
    if (r < rows) {
      const int row = member_row(a, first + r / per_seq), of = r % per_seq, qr = of / G;
      if (row >= 0) {
        hq = (row * a.q_len + qr) * a.Hq + kvh * G + of % G;
        len = a.seq_lens[row] - (a.q_len - 1 - qr);
      }
    }
    s_hq[x] = hq;
    s_len[x] = len;
    const int low = __reduce_min_sync(0xffffffffu, len), most = __reduce_max_sync(0xffffffffu, hq >= 0 ? len : 0);
    if (lane == 0) {
      atomicMin(s_low, low);
      atomicMax(s_most, most);
    }
  }
  __syncthreads();
  // keys of this CTA: whole pages of its split, none behind what its rows see; blocks of 128
  const int key_lo = page_lo * 16, key_hi = min(page_hi * 16, *s_most);
  const int steps = key_hi > key_lo ? (key_hi - key_lo + kTcBlock - 1) / kTcBlock : 0;
  const int turns = kTwoTiles ? 2 * steps : steps;  // turn u: stream u & 1

  int slot = 0, taken = 0;  // the warp's next page: its place in the ring, its number
  uint32_t round = 0;
  const auto ring_wait = [&] { return mbar_wait_warp(&ring_bar[slot], round, abort_flag, a.status, kStatusTimeoutProducer); };
  const auto ring_next = [&] {  // (counted along: a division by the depth, which the roles do not share, took longer than the page)
    ++taken;
    if (++slot == depth) { slot = 0; round ^= 1; }
  };
  const auto drain = [&](bool ok) {  // copies end before the CTA does: of pages that no row sees, and of what a wait that ran out has left
    if (!ok) let_started_work_end();
    while (taken < asked) {
      if (!ring_wait()) let_started_work_end();
      ring_next();
    }
  };
  if (warp < 4) {
    const int tok = lane >> 2, c = lane & 3;  // of the first 8 tokens; the others are 8 on
    const uint32_t lo = ((2 * c) ^ tok) << 4, hi = ((2 * c + 1) ^ tok) << 4;
    bool ok = true;
    for (int step = 0; step < steps; ++step) {
      // what the next Q K^T waits for comes first: the codes of the block's two pages; then their multipliers, then the requests that follow them
      const int left = key_hi - key_lo - step * kTcBlock;  // keys of the block
      const int held = (left > w * 16) + (left > w * 16 + 64);
      const uint8_t* raw[2];
      int slots[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        raw[y] = ring + slot * L::kKPage;
        slots[y] = slot;
        if (y < held) {
          ok = ok && ring_wait();
          ring_next();
        }
      }
      ok = ok && mbar_wait_warp(k_empty, (step & 1) ^ 1, abort_flag, a.status, kStatusTimeoutProducer);
      if (!ok) break;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint4 v[D / 32];
#pragma unroll
        for (int x = 0; x < D / 32; ++x) v[x] = *reinterpret_cast<const uint4*>(raw[y] + lane * 16 + x * 512);
        uint8_t* at = sK + ((w + 4 * y) * 16 + tok) * 128;
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          if ((w + 4 * y) * 16 + tok + 8 * (x & 1) >= left) v[x] = make_uint4(0, 0, 0, 0);
          const uint32_t h[8] = {e4m3_pair(v[x].x), e4m3_pair(v[x].x >> 16), e4m3_pair(v[x].y), e4m3_pair(v[x].y >> 16),
                                 e4m3_pair(v[x].z), e4m3_pair(v[x].z >> 16), e4m3_pair(v[x].w), e4m3_pair(v[x].w >> 16)};
          uint8_t* to = at + (x >> 1) * (kTcBlock * 128) + (x & 1) * 1024;
          put_halves(to + lo, to + hi, h);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(k_full);
      {  // a lane to a column; the softmax of four blocks before is over: products behind its P V are
        const int y = lane >> 4, key = (w + 4 * y) * 16 + (lane & 15), pair = (step & 3) * 64 + (key >> 3) * 4 + ((key & 7) >> 1);
        const float* scales = reinterpret_cast<const float*>((y ? raw[1] : raw[0]) + 16 * D) + (lane & 15);
        const bool there = key < left;  // a key that is not there has P = 0
        const float vs = scales[16];
        // V multipliers under 2^-100 count as that: one of zero gives values of zero, and a finite quotient
        const float lv = !there ? kTcMasked : isnan(vs) ? vs : __log2f(fmaxf(vs, 7.888609e-31f));
        float* col = reinterpret_cast<float*>(s_col + pair) + (key & 1);
        col[0] = there ? scales[0] * a.scale_log2 : 0.f;
        col[2] = lv;
        reinterpret_cast<float*>(s_inv + pair)[key & 1] = there ? exp2_fast(-lv) : 0.f;
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&c_full[step & 3]);
#pragma unroll
        for (int y = 0; y < 2; ++y)
          if (y < held && asked < own_pages) request(slots[y]);
      }
      asked = __shfl_sync(0xffffffffu, asked, 0);
    }
    drain(ok);
  } else if (warp < 7) {
    int first_page = w;  // of the block's pages, the first of this warp
    bool ok = true;
    for (int step = 0; step < steps; ++step) {
      const int s = step & 1, left = key_hi - key_lo - step * kTcBlock, slot0 = slot;  // keys of the block
      ok = mbar_wait_warp(&v_empty[s], ((step >> 1) & 1) ^ 1, abort_flag, a.status, kStatusTimeoutProducer);
#pragma unroll 1
      for (int page = first_page; ok && page < 8; page += 3) {
        const int c = 2 * (page & 3), keys = left - page * 16;  // from the page on
        uint8_t* at = sV + s * kTile + (page >> 2) * (D * 128) + lane * 128;
        const uint32_t lo = (c ^ (lane & 7)) << 4, hi = ((c + 1) ^ (lane & 7)) << 4;
        const uint8_t* raw = ring + slot * L::kVPage + lane * 16;
        if (keys > 0) {
          ok = ring_wait();
          ring_next();
        }
        uint4 v[D / 32];
#pragma unroll
        for (int x = 0; x < D / 32; ++x) v[x] = *reinterpret_cast<const uint4*>(raw + x * 512);
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          if (keys <= 0) v[x] = make_uint4(0, 0, 0, 0);
          const uint32_t h[8] = {e4m3_pair(v[x].x), e4m3_pair(v[x].y), e4m3_pair(v[x].z), e4m3_pair(v[x].w),
                                 e4m3_pair(v[x].x >> 16), e4m3_pair(v[x].y >> 16), e4m3_pair(v[x].z >> 16), e4m3_pair(v[x].w >> 16)};
          put_halves(at + x * 4096 + lo, at + x * 4096 + hi, h);
        }
        if (keys > 0 && keys < 16) {  // no row sees all of this page: zeros behind what they see
#pragma unroll 1
          for (int key = keys; key < 16; ++key)
#pragma unroll 1
            for (int x = 0; x < D / 32; ++x) *reinterpret_cast<uint16_t*>(at + x * 4096 + (key < 8 ? lo : hi) + (key & 7) * 2) = 0;
        }
      }
      if (!ok) break;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_full[s]);
        int at = slot0;
#pragma unroll 1
        for (int page = first_page; page < 8 && page * 16 < left && asked < own_pages; page += 3) {
          request(at);
          at = at + 1 == L::kVDepth ? 0 : at + 1;
        }
      }
      asked = __shfl_sync(0xffffffffu, asked, 0);
      first_page = (first_page + 1) % 3;  // eight pages on: page p is warp p % 3's
    }
    drain(ok);
  } else if (warp == 7) {
    if (steps > 0) {
      constexpr uint32_t idesc_qk = umma_idesc(128, 128, 0, 0), idesc_pv = umma_idesc(128, D, 0, 0);
      constexpr uint64_t kT = kTile >> 4, kQkSlice = (kTcBlock * 128) >> 4, kPvSlice = (D * 128) >> 4;
      const uint64_t q_desc = umma_desc_k_sw128(smem_u32(sQ)), k_desc = umma_desc_k_sw128(smem_u32(sK)), v_desc = umma_desc_k_sw128(smem_u32(sV));
      const auto step_of = [&](int u) { return kTwoTiles ? u >> 1 : u; };
      bool ok = mbar_wait_warp(q_full, 0, abort_flag, a.status, kStatusTimeoutMma);
      // turn u < 0: nothing but the Q K^T of turn u + 2
#pragma unroll 1
      for (int u = -2; ok && u < turns; ++u) {
        const int t = u & 1;
        const uint32_t p = tmem_base + uint32_t(t) * 128u;
        if (u >= 0) {
          const int j = u >> 1, s = step_of(u) & 1;  // j: block of the stream
          ok = mbar_wait_warp(&v_full[s], (step_of(u) >> 1) & 1, abort_flag, a.status, kStatusTimeoutMma) &&
               mbar_wait_warp(&p_full[t], j & 1, abort_flag, a.status, kStatusTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = v_desc + uint64_t(s) * kT;
          const uint32_t d = tmem_base + 256u + uint32_t(t) * D;
          umma_p_v(d, p, vd, idesc_pv, j > 0 ? 1u : 0u);
          umma_p_v(d, p + 64u, vd + kPvSlice, idesc_pv, 1u);
          if (!kTwoTiles || t == 1) tc_commit_warp(&v_empty[s]);
          if (u + 2 >= turns) tc_commit_warp(&o_full[t]);
        }
        if (u + 2 < turns) {  // S takes the place of P, which the products before have read
          ok = mbar_wait_warp(k_full, step_of(u + 2) & 1, abort_flag, a.status, kStatusTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          const uint64_t qd = q_desc + uint64_t(t) * kT;
#pragma unroll
          for (int h = 0; h < kSlices; ++h) umma_f16_block(p, qd + h * kQkSlice, k_desc + h * kQkSlice, idesc_qk, h ? 1u : 0u);
          tc_commit_warp(&s_full[t]);
          if (!kTwoTiles || t == 1) tc_commit_warp(k_empty);
        }
      }
      if (!ok) let_started_work_end();
    }
  } else {
    // ----- softmax: warps 8 - 15 stream 0, 16 - 23 stream 1; a warp has 32 rows and 64 of a block's keys, a lane parts of four rows -----
    const int t = (warp - 8) >> 3, half = (warp - 8) >> 2 & 1, quarter = warp & 3, c = lane & 3;
    {  // 16 rows of Q to fp16, D / 8 lanes to a row: as they are where the largest value is between 2^-4 and 2^15 (bf16 values
       // are exact in fp16 down to 2^-17, which is 2^-13 of 2^-4; smaller ones are off by at most 2^-25, which is 2^-21 of it), else scaled to 2^13
      constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
      const int row16 = (warp - 8) * 16 + lane / kLanes, piece = lane % kLanes;
      uint4 v[16 / kAtOnce];
#pragma unroll
      for (int n = 0; n < 16 / kAtOnce; ++n) {
        const int hq = s_hq[row16 + n * kAtOnce];
        v[n] = *reinterpret_cast<const uint4*>(a.q + size_t(max(hq, 0)) * D + piece * 8);
        if (hq < 0) v[n] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int n = 0; n < 16 / kAtOnce; ++n) {
        const int r = row16 + n * kAtOnce;
        const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(&v[n]);
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(__bfloat162float(b[e])));
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float up = top == 0.f || (top >= 0.0625f && top < 32768.f) ? 1.f : power_to(top, 13);
        if (piece == 0) {
          s_rowc[r] = 1.f / up;
          if (up != 1.f) atomicOr(s_scaled, 1);
        }
        uint4 h;
        h.x = half_pair(__bfloat162float(b[0]) * up, __bfloat162float(b[1]) * up);
        h.y = half_pair(__bfloat162float(b[2]) * up, __bfloat162float(b[3]) * up);
        h.z = half_pair(__bfloat162float(b[4]) * up, __bfloat162float(b[5]) * up);
        h.w = half_pair(__bfloat162float(b[6]) * up, __bfloat162float(b[7]) * up);
        *reinterpret_cast<uint4*>(sQ + t * kTile + (piece >> 3) * (kTcBlock * 128) + (r & 127) * 128 + (((piece & 7) ^ (r & 7)) << 4)) = h;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const uint32_t tS = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(t) * 128u + uint32_t(half) * 64u;
    const uint32_t tO = tmem_base + (uint32_t(quarter * 32) << 16) + 256u + uint32_t(t) * D + uint32_t(half) * (D / 2);
    constexpr uint32_t kDown = 16u << 16;  // rows 16 - 31 of the warp
    const int row0 = t * 128 + quarter * 32 + (lane >> 2);  // and 8, 16, 24 further
    uint64_t* x_mine = &x_bar[t * 4 + quarter];
    float m[4], l[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) { m[r] = kTcFloor; l[r] = 0.f; }
    bool ok = mbar_wait_warp(q_full, 0, abort_flag, a.status, kStatusTimeoutEpilogue);  // s_scaled is final
    const bool special = *s_scaled != 0 || *s_low < key_hi;  // a row was scaled, or does not see all keys
    const int blocks = kTwoTiles ? steps : (steps + 1 - t) >> 1;
#pragma unroll 1
    for (int j = 0; j < blocks; ++j) {
      const int step = kTwoTiles ? j : 2 * j + t, st = step & 3;
      ok = ok && mbar_wait_warp(&c_full[st], (step >> 2) & 1, abort_flag, a.status, kStatusTimeoutEpilogue) &&
           mbar_wait_warp(&s_full[t], j & 1, abort_flag, a.status, kStatusTimeoutEpilogue);
      if (!ok) break;
      tc_fence_after();
      const float4* col = s_col + st * 64 + half * 32 + c;
      const float2* inv = s_inv + st * 64 + half * 32 + c;
      // t of 16 columns: row r = 2h + e, columns 8u + 2c and one more at x[h][4u + 2e].  kSpecial: rows of their own scale or length
      const auto scores = [&](auto special_rows, int part, uint32_t (&x)[2][8]) {
        constexpr bool kSpecial = decltype(special_rows)::value;
        if (kSpecial) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float by = s_rowc[row0 + 8 * r];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              x[r >> 1][4 * u + 2 * (r & 1)] = __float_as_uint(u2f(x[r >> 1][4 * u + 2 * (r & 1)]) * by);
              x[r >> 1][4 * u + 2 * (r & 1) + 1] = __float_as_uint(u2f(x[r >> 1][4 * u + 2 * (r & 1) + 1]) * by);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float4 k = col[(part * 2 + u) * 4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float2 v = fma_f2(make_float2(u2f(x[h][4 * u + e]), u2f(x[h][4 * u + e + 1])), make_float2(k.x, k.y), make_float2(k.z, k.w));
              x[h][4 * u + e] = __float_as_uint(v.x);
              x[h][4 * u + e + 1] = __float_as_uint(v.y);
            }
          }
        }
        if (kSpecial) {
          const int key = key_lo + step * kTcBlock + half * 64 + part * 16 + 2 * c;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int sees = s_len[row0 + 8 * r] - key;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (8 * u >= sees) x[r >> 1][4 * u + 2 * (r & 1)] = __float_as_uint(kTcMasked);
              if (8 * u + 1 >= sees) x[r >> 1][4 * u + 2 * (r & 1) + 1] = __float_as_uint(kTcMasked);
            }
          }
        }
      };
      float mx[4] = {kTcMasked, kTcMasked, kTcMasked, kTcMasked};
      const auto maxima = [&](auto special_rows, int part, uint32_t (&x)[2][8]) {
        scores(special_rows, part, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
            mx[r] = fmaxf(fmaxf(mx[r], u2f(x[r >> 1][4 * u + 2 * (r & 1)])), u2f(x[r >> 1][4 * u + 2 * (r & 1) + 1]));
        }
      };
      float2 sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      const auto exponentials = [&](auto special_rows, int part, uint32_t (&x)[2][8]) {
        uint32_t p[2][4];
        scores(special_rows, part, x);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float2 iv = inv[(part * 2 + u) * 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t* y = x[r >> 1] + 4 * u + 2 * (r & 1);
            const float2 e = make_float2(exp2_fast(u2f(y[0]) - m[r]), exp2_fast(u2f(y[1]) - m[r]));
            sum[r] = fma_f2(e, iv, sum[r]);
            p[r >> 1][2 * u + (r & 1)] = half_pair(e.x, e.y);
          }
        }
        tmem_st_pairs(tS + 8 * part, p[0]);  // over columns that have been read
        tmem_st_pairs(tS + kDown + 8 * part, p[1]);
      };
      const auto parts = [&](auto&& each) {  // the next 16 columns are requested ahead of the present ones' arithmetic
        uint32_t x[2][2][8];
        tmem_ld_frag16(tS, x[0][0]);
        tmem_ld_frag16(tS + kDown, x[0][1]);
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          tmem_wait_ld();
          if (part < 3) {
            tmem_ld_frag16(tS + 16 * part + 16, x[(part + 1) & 1][0]);
            tmem_ld_frag16(tS + kDown + 16 * part + 16, x[(part + 1) & 1][1]);
          }
          each(part, x[part & 1]);
        }
      };
      const auto one_by_one = [&](auto&& each) {
#pragma unroll 1
        for (int part = 0; part < 4; ++part) {
          uint32_t x[2][8];
          tmem_ld_frag16(tS + 16 * part, x[0]);
          tmem_ld_frag16(tS + kDown + 16 * part, x[1]);
          tmem_wait_ld();
          each(part, x);
        }
      };
      if (special) one_by_one([&](int part, uint32_t (&x)[2][8]) { maxima(Special<true>(), part, x); });
      else parts([&](int part, uint32_t (&x)[2][8]) { maxima(Special<false>(), part, x); });
      float* theirs = s_max + (j & 1) * 512;  // the other half's of two blocks before have been read: it was at the exchange since
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        if (c == r) theirs[half * 256 + row0 + 8 * r] = mx[r];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(x_mine);
      ok = mbar_wait_warp(x_mine, j & 1, abort_flag, a.status, kStatusTimeoutEpilogue);
      if (!ok) break;
      bool grown = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        mx[r] = fmaxf(mx[r], theirs[(half ^ 1) * 256 + row0 + 8 * r]);
        grown |= mx[r] > m[r] + kTcGrowth;
      }
      if (__any_sync(0xffffffffu, grown)) {  // always in the first block; both halves alike
        float by[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float now = fmaxf(m[r], mx[r] - kTcRoom);
          by[r] = exp2_fast(m[r] - now);
          l[r] *= by[r];
          m[r] = now;
        }
        if (j > 0) {  // the product before is complete: it was issued ahead of the one that S came from
#pragma unroll 1
          for (int d = 0; d < D / 2; d += 16) {
            uint32_t o[2][8];
            tmem_ld_frag16(tO + d, o[0]);
            tmem_ld_frag16(tO + kDown + d, o[1]);
            tmem_wait_ld();
#pragma unroll
            for (int n = 0; n < 16; ++n) o[n >> 3][n & 7] = __float_as_uint(u2f(o[n >> 3][n & 7]) * by[2 * (n >> 3) + (n >> 1 & 1)]);
            tmem_st_frag16(tO + d, o[0]);
            tmem_st_frag16(tO + kDown + d, o[1]);
          }
        }
      }
      if (special) one_by_one([&](int part, uint32_t (&x)[2][8]) { exponentials(Special<true>(), part, x); });
      else parts([&](int part, uint32_t (&x)[2][8]) { exponentials(Special<false>(), part, x); });
#pragma unroll
      for (int r = 0; r < 4; ++r) l[r] += sum[r].x + sum[r].y;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok) {  // the halves' sums
      float* sums = s_max + (blocks & 1) * 512;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (c == r) sums[half * 256 + row0 + 8 * r] = l[r];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(x_mine);
      ok = mbar_wait_warp(x_mine, blocks & 1, abort_flag, a.status, kStatusTimeoutEpilogue) &&
           (blocks == 0 || mbar_wait_warp(&o_full[t], 0, abort_flag, a.status, kStatusTimeoutEpilogue));
      tc_fence_after();
      if (ok) {
        const int slot = kTwoTiles ? split : 2 * split + t;
        size_t at[4];
        bool live[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int hq = s_hq[row0 + 8 * r];
          live[r] = hq >= 0;
          at[r] = size_t(max(hq, 0)) * a.slots + slot;
          if (live[r] && half == 0 && c == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at[r]) = make_float2(m[r], l[r] + sums[256 + row0 + 8 * r]);
        }
#pragma unroll 1
        for (int d = 0; d < (blocks > 0 ? D / 2 : 0); d += 16) {
          uint32_t o[2][8];
          tmem_ld_frag16(tO + d, o[0]);
          tmem_ld_frag16(tO + kDown + d, o[1]);
          tmem_wait_ld();
#pragma unroll
          for (int n = 0; n < 16; n += 2) {
            const int r = 2 * (n >> 3) + (n >> 1 & 1);
            if (live[r])
              *reinterpret_cast<float2*>(a.part_o + at[r] * D + half * (D / 2) + d + 8 * ((n & 7) >> 2) + 2 * c) = make_float2(u2f(o[n >> 3][n & 7]), u2f(o[n >> 3][(n & 7) + 1]));
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 7) tmem_dealloc(tmem_base, 512);
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
  launch_kernel(kernel, dim3(tiles_at_most(a, per_tile), a.Hk, a.prefix_splits), dim3(kTcThreads), SharedTc<D>::kSmem, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}

int launch_shared_prefix_tc(const SharedAttnArgs& a, int dim, bool two_tiles, cudaStream_t stream) {
  if (dim == 128) return two_tiles ? launch_tc<128, true>(a, stream) : launch_tc<128, false>(a, stream);
  if (dim == 64) return two_tiles ? launch_tc<64, true>(a, stream) : launch_tc<64, false>(a, stream);
  return -1;
}

}  // namespace mfq
