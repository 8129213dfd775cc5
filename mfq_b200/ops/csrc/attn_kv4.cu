// Decode / verify attention over pages held in 4 bits (kv4.cuh has the format and the layout of a page).
//
// With k = m + s c and v likewise, per group of 64 dims:
//   score(q, t) = sum_g (s_tg sum_d q_d c_td + m_tg sum_d q_d)          the sums over d are the products' work, on codes alone
//   o_d         = sum_t p_t (s_tg c_td + m_tg) / sum_t p_t                p_t s_tg is the products' operand, sum_t p_t m_tg is kept beside
// so that a code is never turned into a value.  A code becomes an operand by one AND: 0 .. 15 in the low bits of an fp16 is c 2^-24, which tensor cores
// multiply as any other number; in the next four bits it is 16 times that.  Two registers of a fragment have their codes 16 times as large: the dims
// d + 8 of K, whose queries are divided by 16, and the rows d + 8 of V's output, which are divided in the end.
//
// A unit is one sequence, one KV head and up to 4, 8 or 16 of its query rows (query token, head of the group), with all pairs of pages of the sequence.
// The pairs of all units in a row are cut into equal shares, one a CTA, as many as the GPU holds at once, whatever the lengths are: a CTA has the end of
// one unit, whole ones, and the beginning of another.  What it has of a unit that others have too it leaves in fp32 for the merge.  Where there are few
// units, or short ones, a cluster of 1 to 8 CTAs has a unit instead, cut into as many equal pieces, which meet in their shared memory: one kernel.
// The warps of a CTA take pairs in turn, each through a ring of its own that its lanes fill by 16-byte asynchronous copies; a lane reads the codes that it copied.
// A page's tokens are the rows of the products and the query rows their columns:
//   S^T [16 x 8] = K Q^T,   O^T [D x 8] += V^T (p s),   p s being S^T's accumulator transposed by movmatrix.
// Up to 4 query rows have the two pages side by side: the first page is multiplied by [Q 0], the second by [0 Q], into the same accumulator, so that no
// lane computes the softmax of columns that nobody has; O^T's halves are added in the end.
//
// Numbers: a row of q is scaled by a power of two to 2^10 <= max |q| < 2^11, so that fp16 holds its values exactly down to 2^-24 of the largest; in a product with
// codes, bits some 2^-15 below the largest of 16 dims are cut off.  Scores, maxima, sums and outputs are fp32.  p is exp2(score - ref): ref is at most 6 below
// the row's running maximum.  p s and p m are multiplied by a power of two that brings the largest scales of V to 2^7 .. 2^9, so that p s is rounded to fp16 as a
// normal number (2^-11) down to 2^-21 of the largest p times the largest scale that the warp has met; that is 1/8 of a bf16 output's rounding.  For fp16 outputs
// p s is a sum of two fp16 numbers (off by 2^-22, or 2^-27 of the largest where that is more), each multiplied by itself.  The sum of p has no such factor: warps,
// CTAs and pieces are joined by ref for p and by both for the rest, so that scales of V may lie apart as far as their type lets them and the softmax is the same
// wherever they are.  Scales of V between 2^-98 and 2^98, queries up to 2^100.
//
// Measured, 8 KV heads of 128, bf16: 64 rows of 16384 tokens (1.2 GB) 201 to 206 us, 0.90 to 0.92 of the measured copy rate, 213 to 230 where the power limit holds
// the clock at 1.64 GHz; 64 of 4096 60 us; 3 of up to 2000 8.4.  A pair of pages costs a warp 392 instructions, 223 of them on the half-rate integer
// pipe (160 to unpack codes, five for eight), where memory at its full rate leaves 780 issue slots: latency between dependent instructions with four warps a
// scheduler is what keeps it from hiding all of the arithmetic.  Queries in shared memory instead of registers: 214 -> 205 us; five CTAs an SM of 96
// registers took 217, a shift of the upper codes on the multiplier 251 instead of 214 (before V's sums met in between, which takes 1 %).
#include "attn_shared.cuh"
#include "kv4.cuh"

#include <cfloat>
#include <climits>

namespace mfq {

struct Kv4Join {  // the unit that ends in a CTA's first piece: how many CTAs have pieces of it (0: there is none), and whether the first of these has something in front
  int seq, unit, n, behind;
};
struct Kv4AttnArgs {
  const void* q;
  const uint8_t* pool;
  const int *table, *seq_lens;
  void* out;
  float *part_o, *part_ml;  // [2 * CTAs, kCols, D], [.., 4]: of a CTA's first piece, if others have the rest of the unit, and of its last one; null: a cluster has a unit
  Kv4Join* joins;           // [CTAs]
  int* status;
  int B, Hq, Hk, width, pages, q_len, least, tiles, cluster;  // least: pairs of a share at least; tiles: of query rows of a KV head; cluster: CTAs of a unit
  float scale_log2;
};

template <int D>
struct Kv4Ring {
  static constexpr int kRecord = 18 * D, kStage = 2 * kRecord, kStages = D == 64 ? 3 : 2, kWarps = 4;
  static constexpr int kWarp = kStages * kStage, kSmem = kWarps * kWarp;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)) : "memory");
}
__device__ __forceinline__ void copies_end_here() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copies_but_the_last() {  // all groups of this thread's copies but the last kLeft are there
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}
__device__ __forceinline__ float kv4_exp2(float x) {  // results under 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t kv4_transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void kv4_product(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  const uint32_t a[4] = {a0, a1, a2, a3};
  mma_half(d, a, b0, b1);
}
__device__ __forceinline__ void kv4_first_product(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {  // d was nothing
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float2 add_f2(float2 a, float2 b) {
  add2(a.x, a.y, __float_as_uint(b.x), __float_as_uint(b.y));
  return a;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
constexpr int kAtOnce = 8;  // pieces of the merge
constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;

template <typename T> __device__ __forceinline__ float2 kv4_pair(uint32_t v);
template <> __device__ __forceinline__ float2 kv4_pair<__nv_bfloat16>(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 kv4_pair<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// A unit's queries as a block has them in shared memory, for all of its warps: a lane's B operands of each step of 16 dims, kQ words of a column block, or of
// two; of 4 columns: [Q 0] and [0 Q].  Behind them, of each row, the power of two that it was multiplied by and the sums of its groups.
template <int D, int kCols, typename T>
struct Kv4Queries {
  static constexpr int G = D / 64, kSteps = D / 16, kQ = kCols == 8 ? 2 : 4, kWords = kSteps * 32 * kQ, kBytes = 4 * (kWords + kCols * (1 + G));
  // A warp takes rows in turn; a lane has D / 32 neighbouring dims of a row
  static __device__ __forceinline__ void load(const Kv4AttnArgs& a, int seq, int kvh, int first, int rows, uint32_t* q) {
    constexpr int kPairs = D / 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = a.Hq / a.Hk;
    float* scales = reinterpret_cast<float*>(q + kWords);
#pragma unroll
    for (int i = 0; i < kCols / 4; ++i) {
      const int n = warp + 4 * i, r = first + n;
      uint32_t raw[kPairs];
#pragma unroll
      for (int k = 0; k < kPairs; ++k) raw[k] = 0;
      if (r < rows) {
        const uint32_t* from = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + ((size_t(seq) * a.q_len + r / per) * a.Hq + kvh * per + r % per) * D) + kPairs * lane;
        if constexpr (kPairs == 1) {
          raw[0] = from[0];
        } else if constexpr (kPairs == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(from);
          raw[0] = v.x; raw[1] = v.y;
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(from);
          raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
        }
      }
      float big = 0.f;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const float2 v = kv4_pair<T>(raw[k]);
        big = fmaxf(big, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
      big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
      const float scale = a.scale_log2 < 0.f ? -power_to(big, 10) : power_to(big, 10);  // scores have the sign of their units
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const int d = 2 * (kPairs * lane + k), word = d >> 3 & 1, c = d >> 1 & 3;
        const float2 v = kv4_pair<T>(raw[k]);
        const float x = v.x * scale, y = v.y * scale, up = word ? 0.0625f : 1.f;
        sum += x + y;
        const uint32_t both = half_pair(x * up, y * up);
        uint32_t* to = q + (32 * (d >> 4) + 4 * (n & 7) + c) * kQ;
        if constexpr (kCols == 4) {
          to[word] = both;
          to[2 + word] = 0u;
          to[16 * kQ + word] = 0u;  // column n + 4
          to[16 * kQ + 2 + word] = both;
        } else {
          to[2 * (n >> 3) + word] = both;
        }
      }
#pragma unroll
      for (int o = 1; o < 32 / G; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) scales[n] = scale;
      if (lane % (32 / G) == 0) scales[kCols + n * G + lane / (32 / G)] = sum * 0x1p-24f;
    }
  }
};
template <typename T> __device__ __forceinline__ T kv4_out(float v);
template <> __device__ __forceinline__ __nv_bfloat16 kv4_out(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half kv4_out(float v) { return __float2half_rn(v); }

// Barrier of all threads of the cluster, in the form that asks nothing of the lanes of a warp; what was written before is seen behind it
__device__ __forceinline__ void cluster_meets() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_peer(const float* mine, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(mine)), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 of_peer4(const float* mine, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at_peer(mine, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void kv4_add4(float4& o, float4 v, float weight) {
  o = make_float4(fmaf(v.x, weight, o.x), fmaf(v.y, weight, o.y), fmaf(v.z, weight, o.z), fmaf(v.w, weight, o.w));
}
template <typename T>
__device__ __forceinline__ void kv4_store4(T* to, float4 o, float l, float power) {  // o 2^power / l; nothing seen: zeros
  const float by = l == 0.f ? 0.f : 1.f / l, times = l == 0.f ? 0.f : kv4_exp2(power);
  T y[4] = {kv4_out<T>(o.x * by * times), kv4_out<T>(o.y * by * times), kv4_out<T>(o.z * by * times), kv4_out<T>(o.w * by * times)};
  *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(y);
}
// What a warp has of its query rows: column blocks of 8, a lane has the columns 8 b + 2 c and the one behind it.  kCols 4: the columns n and n + 4 are row n,
// of the first and the second page of a pair.
template <int D, int kCols, typename T>
struct Kv4Rows {
  static constexpr bool kSide = kCols == 4, kSplit = __is_same(T, __half);  // kSplit: p s as two fp16 numbers
  // Products of an instruction are lined up by their operands' exponents, which of a code as a denormal number is 2^-14, ten bits above the code: of a p s, bits some 2^-15
  // of the 16 tokens' largest are cut off, always towards 0.  So the first of the two numbers has no bits below 2^-8, where the largest have 2^7 to 2^9 and more, and
  // the second, multiplied by itself, has them.  5000 keys, scores 2.3 powers of two apart: errors beside the output's rounding from 0.37 of it to 0.13; without bits below
  // 2^-4 0.04, but then p s of 2^-18 of the largest would be one number of 11 bits.
  static constexpr float kGrid = 6.f;  // 2^-8 is the step of fp16 between 4 and 8
  static constexpr int kApart = kSplit ? 4 : 32;  // pairs of pages after which o and om meet
  static constexpr int kQ = Kv4Queries<D, kCols, T>::kQ;
  static constexpr int G = D / 64, kSteps = D / 16, NB = kSide ? 1 : kCols / 8, P = kSide ? 1 : 2;  // P: pages of a pair whose scores a lane has
  float sums[NB][G][2];                            // of a group's q
  float2 to_log2[NB], less[NB], om[NB][G], l[NB];  // what a score in units of the products is times log2 e; -ref
  float o[NB][kSteps][4];
  float lift;  // the power of two by which o and om are multiplied, l is not
  int len[NB][2], low, most;

  __device__ __forceinline__ void load(const Kv4AttnArgs& a, int first, int rows, int length, const uint32_t* q) {
    const int c = threadIdx.x & 3, per = a.Hq / a.Hk;
    const float* scales = reinterpret_cast<const float*>(q + Kv4Queries<D, kCols, T>::kWords);
    int lo = INT_MAX, hi = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = 8 * b + (kSide ? 2 * (c & 1) : 2 * c) + e, mine = first + n;
        const float f = a.scale_log2 * 0x1p24f / scales[n];
        (e == 0 ? to_log2[b].x : to_log2[b].y) = f;
#pragma unroll
        for (int g = 0; g < G; ++g) sums[b][g][e] = scales[kCols + n * G + g];
        // a row that is not there has a zero query and is never stored: unmasked, it leaves `low` to the others
        len[b][e] = mine < rows ? max(0, length - (a.q_len - 1 - mine / per)) : INT_MAX;
        lo = min(lo, len[b][e]);
        if (mine < rows) hi = max(hi, len[b][e]);
      }
      less[b] = both(FLT_MAX);
      l[b] = both(0.f);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) o[b][s][0] = o[b][s][1] = o[b][s][2] = o[b][s][3] = 0.f;
#pragma unroll
      for (int g = 0; g < G; ++g) om[b][g] = both(0.f);
    }
    low = __reduce_min_sync(0xffffffffu, lo);
    most = __reduce_max_sync(0xffffffffu, hi);
    lift = 0x1p104f;
  }

  // Two pages whose first token is tok0; kWhole: all rows see all of both
  template <bool kWhole>
  __device__ __forceinline__ void pages(const uint8_t* rec0, const uint32_t* q, int tok0) {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
    const int side = kSide ? c >> 1 : 0;  // the page whose scores this lane has
    const auto sees = [&](int b, int e, int p, int h) { return tok0 + 16 * (p + side) + 8 * h + g8 < len[b][e]; };
    float2 sc[NB][P][2];  // [page][token g8, g8 + 8], of two columns
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float acc[NB][P][4];
      uint32_t w[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint4 raw = *reinterpret_cast<const uint4*>(rec0 + p * 18 * D + 512 * g + 16 * lane);
        w[p][0] = raw.x; w[p][1] = raw.y; w[p][2] = raw.z; w[p][3] = raw.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t qw[kQ];
        const uint32_t* from = q + (32 * (4 * g + j) + lane) * kQ;
        if constexpr (kQ == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(from);
          qw[0] = v.x; qw[1] = v.y; qw[2] = v.z; qw[3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(from);
          qw[0] = v.x; qw[1] = v.y;
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint32_t h = w[p][j] >> 8;
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const int of = 2 * (kSide ? p : b);
            float(&x)[4] = acc[b][kSide ? 0 : p];
            if (j == 0 && (p == 0 || !kSide)) kv4_first_product(x, w[p][j] & kLow, h & kLow, w[p][j] & kHigh, h & kHigh, qw[of], qw[of + 1]);
            else kv4_product(x, w[p][j] & kLow, h & kLow, w[p][j] & kHigh, h & kHigh, qw[of], qw[of + 1]);
          }
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        uint32_t par[2];  // of tokens g8 and g8 + 8
        const uint8_t* at = rec0 + (p + side) * 18 * D + 8 * D + g8 * (D / 8) + 4 * g;
        par[0] = *reinterpret_cast<const uint32_t*>(at);
        par[1] = *reinterpret_cast<const uint32_t*>(at + 4 * G);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float ps = __uint_as_float(par[h] << 16), pm = __uint_as_float(par[h] & 0xffff0000u);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float2& x = sc[b][p][h];
            x.x = fmaf(ps, acc[b][p][2 * h], g == 0 ? pm * sums[b][g][0] : fmaf(pm, sums[b][g][0], x.x));
            x.y = fmaf(ps, acc[b][p][2 * h + 1], g == 0 ? pm * sums[b][g][1] : fmaf(pm, sums[b][g][1], x.y));
          }
        }
      }
    }
    if constexpr (!kWhole) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!sees(b, 0, p, h)) sc[b][p][h].x = -INFINITY;
            if (!sees(b, 1, p, h)) sc[b][p][h].y = -INFINITY;
          }
        }
      }
    }
    // parameters of V, none where nobody sees the token: what is there may be anything
    uint32_t par[P][2][G];
    float widest = 0.f, largest = 0.f;  // scale, minimum
#pragma unroll
    for (int p = 0; p < P; ++p) {
      params(par[p], rec0 + (p + side) * 18 * D + 17 * D + g8 * (D / 8));
      if constexpr (!kWhole) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int g = 0; g < G; ++g)
            if (tok0 + 16 * (p + side) + g8 + 8 * h >= most) par[p][h][g] = 0;
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        widest = max3(widest, __uint_as_float(par[p][0][g] << 16), __uint_as_float(par[p][1][g] << 16));
        largest = max3(largest, fabsf(__uint_as_float(par[p][0][g] & 0xffff0000u)), fabsf(__uint_as_float(par[p][1][g] & 0xffff0000u)));
      }
    }
    float mx[NB][2];
    bool moves = fmaxf(widest, largest * 0x1p-77f) * lift > 0x1p9f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      mx[b][0] = fmaxf(sc[b][0][0].x, sc[b][0][1].x);
      mx[b][1] = fmaxf(sc[b][0][0].y, sc[b][0][1].y);
      if constexpr (P == 2) {
        mx[b][0] = max3(mx[b][0], sc[b][P - 1][0].x, sc[b][P - 1][1].x);
        mx[b][1] = max3(mx[b][1], sc[b][P - 1][0].y, sc[b][P - 1][1].y);
      }
      moves |= fmaf(mx[b][0], to_log2[b].x, less[b].x) > 6.f || fmaf(mx[b][1], to_log2[b].y, less[b].y) > 6.f;
    }
    if (__any_sync(0xffffffffu, moves)) move(mx, widest, largest);
    uint32_t pb[NB][P][G][2], rest[kSplit ? NB : 1][P][G][2];
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2 x = fma_f2(sc[b][p][h], to_log2[b], less[b]);
          if constexpr (!kWhole) {  // with a scale of 0 the products made it a NaN
            if (!sees(b, 0, p, h)) x.x = -INFINITY;
            if (!sees(b, 1, p, h)) x.y = -INFINITY;
          }
          sc[b][p][h] = make_float2(kv4_exp2(x.x), kv4_exp2(x.y));
          l[b] = add_f2(l[b], sc[b][p][h]);
          scale2(sc[b][p][h].x, sc[b][p][h].y, lift);
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float ps = __uint_as_float(par[p][h][g] << 16), pm = __uint_as_float(par[p][h][g] & 0xffff0000u);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float2 v = make_float2(sc[b][p][h].x * ps, sc[b][p][h].y * ps);
            if constexpr (!kWhole) {  // a NaN stays with the rows that see it
              const bool s0 = sees(b, 0, p, h), s1 = sees(b, 1, p, h);
              v = make_float2(s0 ? v.x : 0.f, s1 ? v.y : 0.f);
              om[b][g] = make_float2(s0 ? fmaf(sc[b][p][h].x, pm, om[b][g].x) : om[b][g].x, s1 ? fmaf(sc[b][p][h].y, pm, om[b][g].y) : om[b][g].y);
            } else {
              om[b][g] = make_float2(fmaf(sc[b][p][h].x, pm, om[b][g].x), fmaf(sc[b][p][h].y, pm, om[b][g].y));
            }
            if constexpr (kSplit) {
              const __half2 near = __hsub2(__floats2half2_rn(v.x + kGrid, v.y + kGrid), __float2half2_rn(kGrid));
              const float2 as = __half22float2(near);
              pb[b][p][g][h] = kv4_transposed(*reinterpret_cast<const uint32_t*>(&near));
              rest[b][p][g][h] = kv4_transposed(half_pair(v.x - as.x, v.y - as.y));
            } else {
              pb[b][p][g][h] = kv4_transposed(half_pair(v.x, v.y));
            }
          }
        }
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint8_t* rec = rec0 + p * 18 * D + 9 * D;
      const uint32_t keep = !kSide || (g8 < 4) == (p == 0) ? 0xffffffffu : 0u;  // this page's columns
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint4 raw = *reinterpret_cast<const uint4*>(rec + 512 * g + 16 * lane);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t b0[NB], b1[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) { b0[b] = pb[b][kSide ? 0 : p][g][0] & keep; b1[b] = pb[b][kSide ? 0 : p][g][1] & keep; }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t h = w[j] >> 8;
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            kv4_product(o[b][4 * g + j], w[j] & kLow, w[j] & kHigh, h & kLow, h & kHigh, b0[b], b1[b]);
            if constexpr (kSplit)
              kv4_product(o[b][4 * g + j], w[j] & kLow, w[j] & kHigh, h & kLow, h & kHigh, rest[b][kSide ? 0 : p][g][0] & keep, rest[b][kSide ? 0 : p][g][1] & keep);
          }
        }
      }
    }
  }

  // o, a sum of codes that are 0 or more, and om, a sum of minima that mostly are 0 or less, are many times their difference: an average over n tokens falls with sqrt(n).
  // What tensor cores cut off at an addition (2^-24 of the sum, always towards 0) then is an error of the average.  So they meet before either is large.
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float2 m = om[b][g];
#pragma unroll
        for (int x = 4; x < 32; x *= 2) m = add_f2(m, make_float2(__shfl_xor_sync(0xffffffffu, m.x, x), __shfl_xor_sync(0xffffffffu, m.y, x)));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float(&y)[4] = o[b][4 * g + j];
          y[0] = fmaf(m.x, 0x1p-24f, y[0]); y[1] = fmaf(m.y, 0x1p-24f, y[1]);
          y[2] = fmaf(m.x, 0x1p-20f, y[2]); y[3] = fmaf(m.y, 0x1p-20f, y[3]);
        }
        om[b][g] = both(0.f);
      }
    }
  }

  static __device__ __forceinline__ void params(uint32_t (&par)[2][G], const uint8_t* at) {  // [half][group] in a row
    if constexpr (G == 1) {
      const uint2 v = *reinterpret_cast<const uint2*>(at);
      par[0][0] = v.x; par[1][0] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < 2 * G; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(at + 4 * i);
        par[i / G][i % G] = v.x; par[(i + 1) / G][(i + 1) % G] = v.y; par[(i + 2) / G][(i + 2) % G] = v.z; par[(i + 3) / G][(i + 3) % G] = v.w;
      }
    }
  }

  // New references: the running maxima, and the power of two of V's sums.  It brings the scales to 2^7 .. 2^9 and leaves the minima below 2^87, which
  // matters where a group of one value (scale 0) stands beside values of 2^-77 of it.
  __device__ __forceinline__ void move(const float (&mx)[NB][2], float widest, float largest) {
    const auto exponent = [](float x) { return int(__reduce_max_sync(0xffffffffu, __float_as_uint(x)) >> 23) - 127; };  // of the warp's largest; a denormal one: -127
    const int before = int(__float_as_uint(lift) >> 23) - 127, up = min(before, min(7 - exponent(widest), 84 - exponent(largest)));
    lift = __uint_as_float(uint32_t(up + 127) << 23);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float corr[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f = e == 0 ? to_log2[b].x : to_log2[b].y;
        float& now = e == 0 ? less[b].x : less[b].y;
        float m = mx[b][e];
        if constexpr (kSide) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        const float next = m > -INFINITY ? fminf(now, -(m * f)) : now, by = next - now;
        corr[e] = kv4_exp2(by + float(up - before));
        (e == 0 ? l[b].x : l[b].y) *= kv4_exp2(by);
        now = next;
      }
#pragma unroll
      for (int g = 0; g < G; ++g) om[b][g] = make_float2(om[b][g].x * corr[0], om[b][g].y * corr[1]);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) { o[b][s][0] *= corr[0]; o[b][s][1] *= corr[1]; o[b][s][2] *= corr[0]; o[b][s][3] *= corr[1]; }
    }
  }
};

__device__ __forceinline__ long long kv4_quotient(long long a, long long b) {  // of numbers that are not negative; 64 bits take ten times as long
  return (a | b) >> 32 ? a / b : (long long)(uint32_t(a) / uint32_t(b));
}
// The units' pairs in a row, found by a whole warp
struct Kv4Shares {
  static constexpr int kHeld = 4;  // lengths that a lane keeps: of 128 sequences
  unsigned held[kHeld];
  long long total, share;
  int per_seq;  // units of a sequence
  __device__ __forceinline__ static int pairs(const Kv4AttnArgs& a, int seq) {
    return seq < a.B ? int((max(0ll, min((long long)a.seq_lens[seq], 16ll * a.width)) + 31) >> 5) : 0;
  }
  __device__ __forceinline__ Kv4Shares(const Kv4AttnArgs& a, int ctas) : total(0), per_seq(a.Hk * a.tiles) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) held[k] = unsigned(pairs(a, 32 * k + int(lane_id())));
#pragma unroll
    for (int k = 0; k < kHeld; ++k) total += __reduce_add_sync(0xffffffffu, held[k]);  // 32 * 2^26 at most
    for (int b = 32 * kHeld; b < a.B; b += 32) total += __reduce_add_sync(0xffffffffu, unsigned(pairs(a, b + int(lane_id()))));
    total *= per_seq;
    share = max((long long)a.least, kv4_quotient(total + ctas - 1, ctas));
  }
  // Among 32 sequences with n pairs each: the one that has the x-th pair, -1: it is behind them; `before`: the pairs in front of it (of them all)
  __device__ __forceinline__ int among(unsigned n, long long x, long long& before) const {
    unsigned upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
      if (int(lane_id()) >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, (before + upto) * per_seq > x);
    const int at = past ? __ffs(past) - 1 : 31;
    before += __shfl_sync(0xffffffffu, past ? upto - n : upto, at);
    return past ? at : -1;
  }
  __device__ __forceinline__ int find(const Kv4AttnArgs& a, long long x, long long& before) const {  // of all sequences, x < total
    before = 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int at = among(held[k], x, before);
      if (at >= 0) return 32 * k + at;
    }
    for (int b = 32 * kHeld; b < a.B; b += 32) {
      const int at = among(unsigned(pairs(a, b + int(lane_id()))), x, before);
      if (at >= 0) return b + at;
    }
    return a.B;
  }
};

template <int D, int kCols, typename T, int kMinBlocks>
__global__ void __launch_bounds__(128, kMinBlocks) kv4_attn_kernel(Kv4AttnArgs a) {
  pdl_trigger();
  using L = Kv4Ring<D>;
  using R = Kv4Rows<D, kCols, T>;
  constexpr int NB = R::NB, kStride = D + 4, kPart = 8 * NB * kStride + 16 * NB + 1;  // what a warp leaves, in floats: rows of columns on different banks, then (ref, l), log2 of what its sums are in units of
  static_assert(kPart * 4 <= L::kWarp && kCols * (D + 4) * 4 <= L::kSmem, "the rings are where the sums are left");
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * L::kWarp;
  uint32_t* block_q = reinterpret_cast<uint32_t*>(smem + L::kSmem);
  pdl_wait();

  const int rows = a.Hq / a.Hk * a.q_len, per_head = a.Hq / a.Hk;
  // sequences without a token: zeros
  for (int seq = blockIdx.x; seq < a.B; seq += gridDim.x) {
    if (a.seq_lens[seq] > 0) continue;
    uint4* y = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + size_t(seq) * a.q_len * a.Hq * D);
    for (long long i = threadIdx.x; i < (long long)a.q_len * a.Hq * D / 8; i += 128) y[i] = make_uint4(0, 0, 0, 0);
  }
  int seq, unit, off, pairs;  // where this CTA is: unit of the sequence, pair of the unit
  long long left, x = 0, share = 1;
  int rank = 0;  // in the cluster
  bool none = false;
  if (a.part_o == nullptr) {
    const int of = blockIdx.x / a.cluster;
    rank = blockIdx.x % a.cluster;
    seq = of / (a.Hk * a.tiles);
    unit = of % (a.Hk * a.tiles);
    pairs = Kv4Shares::pairs(a, seq);
    const int each = (pairs + a.cluster - 1) / a.cluster;
    off = min(rank * each, pairs);
    none = off == pairs;
    left = none ? (a.cluster > 1 ? 1 : 0) : min(each, pairs - off);  // an empty piece of a cluster takes part, whatever the lengths are
  } else {
    const Kv4Shares all(a, gridDim.x);
    share = all.share;
    x = blockIdx.x * share;
    left = min(share, all.total - x);
    if (left <= 0) {
      if (threadIdx.x == 0) a.joins[blockIdx.x].n = 0;
      return;
    }
    long long before;
    seq = all.find(a, x, before);
    pairs = Kv4Shares::pairs(a, seq);
    const long long in = x - before * all.per_seq;
    unit = int(kv4_quotient(in, pairs));
    off = int(in - (long long)unit * pairs);
    if (threadIdx.x == 0) {  // the last one of a unit's pieces says where the others are
      Kv4Join join{seq, unit, 0, 0};
      if (off > 0 && off + left >= pairs) {
        const long long first = kv4_quotient(x - off, share);
        join.n = int(blockIdx.x - first) + 1;
        join.behind = x - off != first * share;
      }
      a.joins[blockIdx.x] = join;
    }
  }
  constexpr int kParts = D / 8;  // pieces of 16 bytes of a page's parameters: K's, then V's
  const int piece = lane % (kParts < 32 ? kParts : 32);
  const uint32_t piece_at = piece < kParts / 2 ? 8 * D + 16 * piece : 17 * D + 16 * (piece - kParts / 2);
  bool begins = true;  // the share's first piece
  uint32_t strays = 0;  // not 0: a page out of range, the last one was read in its place

  while (left > 0) {
    const int here = none ? 0 : int(min(left, (long long)(pairs - off)));
    if (here <= 0 && !none) break;  // lengths that changed under the kernel
    const int kvh = unit / a.tiles, first = unit % a.tiles * kCols;
    const int length = int(min((long long)a.seq_lens[seq], 16ll * a.width)), total = (length + 15) >> 4;  // pages
    const int mine = here > warp ? (here - warp + L::kWarps - 1) / L::kWarps : 0;
    const int* bt = a.table + size_t(seq) * a.width;
    int asked = 2 * (off + warp), used = asked, id[2];  // pages
    const uint32_t page_bytes = uint32_t(a.Hk) * L::kRecord;
    const uint8_t *codes_at = a.pool + size_t(kvh) * L::kRecord + 16 * lane, *pieces_at = a.pool + size_t(kvh) * L::kRecord + piece_at;
    const auto look = [&] {  // the ids of the pair that is asked for next; a second page that is not there: the first again
      const int at = min(asked, total - 1);
      id[0] = bt[at];
      id[1] = bt[min(at + 1, total - 1)];
      asked += 2 * L::kWarps;
    };
    const auto request = [&](uint32_t stage) {
      uint32_t page[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        page[p] = min(uint32_t(id[p]), uint32_t(a.pages - 1));
        strays |= page[p] ^ uint32_t(id[p]);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint8_t* from = codes_at + (unsigned long long)page[p] * page_bytes;  // one multiplication and addition
        const uint32_t at = stage + 16 * lane + p * L::kRecord;
#pragma unroll
        for (int g = 0; g < D / 64; ++g) copy16(at + 512 * g, from + 512 * g);
#pragma unroll
        for (int g = 0; g < D / 64; ++g) copy16(at + 9 * D + 512 * g, from + 9 * D + 512 * g);
      }
      if constexpr (kParts == 32) {
        copy16(stage + piece_at, pieces_at + (unsigned long long)page[0] * page_bytes);
        copy16(stage + piece_at + L::kRecord, pieces_at + (unsigned long long)page[1] * page_bytes);
      } else {
        const uint8_t* from = pieces_at + (unsigned long long)(lane < kParts ? page[0] : page[1]) * page_bytes;
        if (kParts == 16 || lane < 2 * kParts) copy16(stage + piece_at + (lane < kParts ? 0 : L::kRecord), from);
      }
    };
    const uint32_t ring_at = smem_u32(ring);
    if (mine > 0) look();
#pragma unroll
    for (int i = 0; i < L::kStages; ++i) {
      if (i < mine) {
        request(ring_at + i * L::kStage);
        look();
      }
      copies_end_here();
    }
    Kv4Queries<D, kCols, T>::load(a, seq, kvh, first, rows, block_q);
    __syncthreads();
    R t;
    t.load(a, first, rows, length, block_q);
    // pairs that all rows see whole come first, the masked ones of a sequence's end behind them
    int stage = 0, more = mine - L::kStages;
    const auto next = [&] {
      used += 2 * L::kWarps;
      __syncwarp();
      if (more > 0) {
        request(ring_at + stage);
        look();
      }
      copies_end_here();
      --more;
      stage = stage == (L::kStages - 1) * L::kStage ? 0 : stage + L::kStage;
    };
    const int end = used + 2 * L::kWarps * mine, seen = min(end, (t.low >> 4) - 1);
    while (used < seen) {
      const int stop = min(seen, used + 2 * L::kWarps * R::kApart);
      do {
        copies_but_the_last<L::kStages - 1>();
        __syncwarp();
        t.template pages<true>(ring + stage, block_q, used << 4);
        next();
      } while (used < stop);
      if (used < seen) t.settle();
    }
    while (used < end) {
      copies_but_the_last<L::kStages - 1>();
      __syncwarp();
      t.template pages<false>(ring + stage, block_q, used << 4);
      next();
    }

    // ---- the lanes of a column, then the warps ----
    float* part = reinterpret_cast<float*>(ring);
    float* ml = part + 8 * NB * kStride;
    __syncwarp();
    if (lane == 0) ml[16 * NB] = float(127 - int(__float_as_uint(t.lift) >> 23));
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * b + 2 * c + e;
        float sum = e == 0 ? t.l[b].x : t.l[b].y;
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g8 == 0) { ml[2 * r] = -(e == 0 ? t.less[b].x : t.less[b].y); ml[2 * r + 1] = sum; }
#pragma unroll
        for (int g = 0; g < D / 64; ++g) {
          float om = e == 0 ? t.om[b][g].x : t.om[b][g].y;
          om += __shfl_xor_sync(0xffffffffu, om, 4);
          om += __shfl_xor_sync(0xffffffffu, om, 8);
          om += __shfl_xor_sync(0xffffffffu, om, 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            part[r * kStride + 64 * g + 16 * j + g8] = fmaf(t.o[b][4 * g + j][e], 0x1p24f, om);
            part[r * kStride + 64 * g + 16 * j + 8 + g8] = fmaf(t.o[b][4 * g + j][2 + e], 0x1p20f, om);
          }
        }
      }
    }
    __syncthreads();
    const bool whole = here == pairs || a.part_o == nullptr;
    const size_t slot = (2 * size_t(blockIdx.x) + (begins ? 0 : 1)) * kCols;
    const int live = min(rows - first, kCols);
    constexpr int kEach = (kCols * (D / 4) + 127) / 128;  // four values each of a thread
    float4 o[kEach];
    float ref[kEach], l[kEach], power[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = threadIdx.x + 128 * k, r = i / (D / 4), d = i % (D / 4) * 4;
      if (r >= live) break;
      const auto left_by = [&](int w) { return reinterpret_cast<const float*>(smem + w * L::kWarp); };
      const auto ref_of = [&](int w) { return left_by(w)[8 * NB * kStride + 2 * r]; };
      ref[k] = -FLT_MAX;
      power[k] = -FLT_MAX;
      l[k] = 0.f;
      o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < L::kWarps; ++w) ref[k] = fmaxf(ref[k], ref_of(w));
#pragma unroll
      for (int w = 0; w < L::kWarps; ++w) power[k] = fmaxf(power[k], ref_of(w) - ref[k] + left_by(w)[8 * NB * kStride + 16 * NB]);
#pragma unroll
      for (int w = 0; w < L::kWarps; ++w) {
        const float* from = left_by(w);
        const float weight = kv4_exp2(ref_of(w) - ref[k]), of_o = kv4_exp2(ref_of(w) - ref[k] + from[8 * NB * kStride + 16 * NB] - power[k]);
        l[k] += from[8 * NB * kStride + 2 * r + 1] * weight;
        kv4_add4(o[k], *reinterpret_cast<const float4*>(from + r * kStride + d), of_o);
        if constexpr (R::kSide) {
          l[k] += from[8 * NB * kStride + 2 * r + 9] * weight;
          kv4_add4(o[k], *reinterpret_cast<const float4*>(from + (r + 4) * kStride + d), of_o);
        }
      }
      if (a.cluster == 1) {
        if (whole) {
          const size_t row = (size_t(seq) * a.q_len + (first + r) / per_head) * a.Hq + kvh * per_head + (first + r) % per_head;
          kv4_store4(static_cast<T*>(a.out) + row * D + d, o[k], l[k], power[k]);
        } else {
          *reinterpret_cast<float4*>(a.part_o + (slot + r) * D + d) = o[k];
          if (d == 0) *reinterpret_cast<float4*>(a.part_ml + (slot + r) * 4) = make_float4(ref[k], l[k], power[k], 0.f);
        }
      }
    }
    if (a.cluster > 1) {  // every CTA of the cluster comes here once: its sums where the rings were, then a part of the rows of all
      float* mine = reinterpret_cast<float*>(smem);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const int i = threadIdx.x + 128 * k, r = i / (D / 4), d = i % (D / 4) * 4;
        if (r >= live) break;
        *reinterpret_cast<float4*>(mine + r * D + d) = o[k];
        if (d == 0) *reinterpret_cast<float4*>(mine + kCols * D + 4 * r) = make_float4(ref[k], l[k], power[k], 0.f);
      }
      cluster_meets();
      for (int i = threadIdx.x + 128 * rank; i < live * (D / 4); i += 128 * a.cluster) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float4 of[8], part[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // all requested before the first is used
          of[k] = make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
          part[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (k < a.cluster) {
            of[k] = of_peer4(mine + kCols * D + 4 * r, k);
            part[k] = of_peer4(mine + r * D + d, k);
          }
        }
        float most = -FLT_MAX, power = -FLT_MAX, sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) most = fmaxf(most, of[k].x);
#pragma unroll
        for (int k = 0; k < 8; ++k) power = fmaxf(power, of[k].x - most + of[k].z);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          sum += of[k].y * kv4_exp2(of[k].x - most);
          kv4_add4(y, part[k], kv4_exp2(of[k].x - most + of[k].z - power));
        }
        const size_t row = (size_t(seq) * a.q_len + (first + r) / per_head) * a.Hq + kvh * per_head + (first + r) % per_head;
        kv4_store4(static_cast<T*>(a.out) + row * D + d, y, sum, power);
      }
      cluster_meets();  // nobody leaves while its sums are read
      break;
    }
    left -= none ? left : here;
    begins = false;
    off = 0;
    if (left > 0) {
      __syncthreads();  // the rings are rings again
      if (++unit == a.Hk * a.tiles) {
        unit = 0;
        do pairs = Kv4Shares::pairs(a, ++seq);
        while (pairs == 0 && seq < a.B);
        if (seq >= a.B) break;  // lengths that changed under the kernel
      }
    }
  }
  if (strays && lane == 0) atomicCAS(a.status, 0, kStatusBadArgument);
}

// Joins the pieces of the unit that ends in a CTA's first one
template <int D, int kCols, typename T>
__global__ void __launch_bounds__(256) kv4_merge_kernel(Kv4AttnArgs a) {
  pdl_trigger();
  pdl_wait();
  const int cta = blockIdx.x, per_head = a.Hq / a.Hk;
  const Kv4Join join = a.joins[cta];
  const int n = join.n, kvh = join.unit / a.tiles, first = join.unit % a.tiles * kCols, live = n == 0 ? 0 : min(per_head * a.q_len - first, kCols);
  const float4* ml = reinterpret_cast<const float4*>(a.part_ml);
  for (int i = threadIdx.x; i < live * (D / 4); i += blockDim.x) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const auto slot = [&](int k) { return (2 * size_t(cta - n + 1 + k) + (k == 0 ? join.behind : 0)) * kCols + r; };
    float ref = -FLT_MAX, l = 0.f, power = -FLT_MAX;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < n; k += kAtOnce) {
      float4 of[kAtOnce], part[kAtOnce];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {  // all requested before the first is used
        of[e] = k + e < n ? ml[slot(k + e)] : make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
        part[e] = k + e < n ? *reinterpret_cast<const float4*>(a.part_o + slot(k + e) * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float most = ref;
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) most = fmaxf(most, of[e].x);
      const float had = ref - most + power;
      float next = had;
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) next = fmaxf(next, of[e].x - most + of[e].z);
      l *= kv4_exp2(ref - most);
      const float keep = kv4_exp2(had - next);
      o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
      ref = most;
      power = next;
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        l += of[e].y * kv4_exp2(of[e].x - ref);
        kv4_add4(o, part[e], kv4_exp2(of[e].x - ref + of[e].z - power));
      }
    }
    const size_t row = (size_t(join.seq) * a.q_len + (first + r) / per_head) * a.Hq + kvh * per_head + (first + r) % per_head;
    kv4_store4(static_cast<T*>(a.out) + row * D + d, o, l, power);
  }
}

template <int D, int kCols, typename T>
static int launch_kv4_attn_of(Kv4AttnArgs a, int ctas, cudaStream_t stream) {
  using L = Kv4Ring<D>;
  constexpr int kMinBlocks = D == 256 || kCols == 16 ? 2 : 4;
  constexpr int kSmem = L::kSmem + Kv4Queries<D, kCols, T>::kBytes;
  auto kernel = &kv4_attn_kernel<D, kCols, T, kMinBlocks>;
  static bool attr[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -6;
  if (!attr[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) return -6;
    attr[dev] = true;
  }
  const long long tiles = ((long long)a.Hq / a.Hk * a.q_len + kCols - 1) / kCols, units = (long long)a.B * a.Hk * tiles;
  if (units * 8 > 0x7fffffffll || ctas > 1 << 20) return -2;
  a.tiles = int(tiles);
  if (a.part_o) a.cluster = 1;
  if (a.cluster > 1) return launch_kernel_clustered(kernel, dim3(unsigned(units * a.cluster)), dim3(128), dim3(a.cluster), kSmem, stream, a) == cudaSuccess ? 0 : -7;
  if (launch_kernel(kernel, dim3(unsigned(a.part_o ? ctas : units)), dim3(128), kSmem, stream, a) != cudaSuccess) return -7;
  if (a.part_o && launch_kernel(&kv4_merge_kernel<D, kCols, T>, dim3(unsigned(ctas)), dim3(D * kCols / 4 < 256 ? D * kCols / 4 : 256), 0, stream, a) != cudaSuccess) return -7;
  return 0;
}
template <int D, typename T>
static int launch_kv4_attn_for(const Kv4AttnArgs& a, int ctas, cudaStream_t stream) {
  const long long rows = (long long)a.Hq / a.Hk * a.q_len;
  if (rows <= 4) return launch_kv4_attn_of<D, 4, T>(a, ctas, stream);
  if (D == 256 || rows <= 8) return launch_kv4_attn_of<D, 8, T>(a, ctas, stream);  // 16 columns of 256 dims leave the registers: 59 us instead of 44 for 16 windows of 32 rows
  if constexpr (D < 256) return launch_kv4_attn_of<D, 16, T>(a, ctas, stream);
  return -1;
}
template <int D>
static int launch_kv4_attn(const Kv4AttnArgs& a, int ctas, bool half, cudaStream_t stream) {
  return half ? launch_kv4_attn_for<D, __half>(a, ctas, stream) : launch_kv4_attn_for<D, __nv_bfloat16>(a, ctas, stream);
}

}  // namespace mfq

// q, out: [B * q_len, Hq, D] bf16 or fp16 (`half`); pool: [pages, Hk, 18 D]; table: [B, width]; seq_lens count every token visible to the last query row.
// scratch: null, and every unit has a cluster of `ctas` (1, 2, 4 or 8) CTAs, or for `ctas` equal shares of at least `least` pairs of pages, beginning on 16 bytes: 4 words a share, then
// fp32 [2 * ctas, cols, D] and [2 * ctas, cols, 4], cols being 4 for up to 4 query rows of a KV head, 8 for up to 8 or heads of 256, else 16.
extern "C" int mfq_paged_attn_decode_kv4(const void* q, const uint8_t* pool, const int* table, const int* seq_lens, void* out, void* scratch, int half,
                                         int B, int Hq, int Hk, int D, int width, int pages, int q_len, int ctas, int least, float sm_scale, int* status,
                                         cudaStream_t stream) {
  if (B <= 0 || Hk <= 0 || Hk > 65536 || Hq <= 0 || Hq % Hk || q_len < 1 || width <= 0 || pages <= 0 || ctas < 1 || least < 1 || ctas > 1 << 20) return -1;
  if (scratch == nullptr && ctas != 1 && ctas != 2 && ctas != 4 && ctas != 8) return -1;
  const long long cols = Hq / Hk * (long long)q_len <= 4 ? 4 : (D == 256 || Hq / Hk * (long long)q_len <= 8 ? 8 : 16);
  mfq::Kv4Join* joins = static_cast<mfq::Kv4Join*>(scratch);
  float* part_o = scratch ? reinterpret_cast<float*>(joins + ctas) : nullptr;
  const mfq::Kv4AttnArgs a{q, pool, table, seq_lens, out, part_o, scratch ? part_o + 2 * ctas * cols * D : nullptr, joins, status, B, Hq, Hk, width, pages, q_len, least, 0, scratch ? 1 : ctas, sm_scale * 1.4426950408889634f};
  if (D == 64) return mfq::launch_kv4_attn<64>(a, ctas, half != 0, stream);
  if (D == 128) return mfq::launch_kv4_attn<128>(a, ctas, half != 0, stream);
  if (D == 256) return mfq::launch_kv4_attn<256>(a, ctas, half != 0, stream);
  return -1;
}
