// Writing and reading back pages held in 4 bits (kv4.cuh has the format).
//
// A warp takes a run of tokens that follow one another in a page, up to all 16 of it, and one head's K or V.  Lane (g8, c) = (lane / 4, lane % 4) has the
// tokens at places g8 and g8 + 8 and, of every group of 64, the dims 16 c .. 16 c + 15, which are 32 neighbouring bytes in 16 bits: rows are read and written whole
// sectors at a time.  Its codes are the words j = c of the record's fragments (groups g, lanes (g8, 0 .. 3)); a transposition of 4 x 4 words among the four lanes
// of a row makes them the words j = 0 .. 3 of its own, which for K are what the record has and for V are transposed by movmatrix.  A whole page is stored
// by 16-byte accesses, of a part of one the bytes of its tokens alone.
#include "kv4.cuh"

namespace mfq {

struct Kv4WriteArgs {
  const void *k, *v;
  const int* slots;
  uint8_t* pool;
  int* status;
  long long k_token, k_head, v_token, v_head;  // strides in elements
  int T, Hk, pages, window;  // window: tokens in which the runs of a warp begin, 1 .. 16
  unsigned blocks;           // of a window
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t transposed8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Word j of lane c goes to word c of lane j, of the four lanes of a row
__device__ __forceinline__ void transpose4(uint32_t (&w)[4], int c) {
  const bool high = c & 2, odd = c & 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = __shfl_xor_sync(0xffffffffu, high ? w[i] : w[i + 2], 2);
    if (high) w[i] = v; else w[i + 2] = v;
  }
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint32_t v = __shfl_xor_sync(0xffffffffu, odd ? w[i] : w[i + 1], 1);
    if (odd) w[i] = v; else w[i + 1] = v;
  }
}

// 16 values of a token; their order is that of memory
template <typename T>
struct Kv4Sixteen {
  static constexpr int kWords = int(sizeof(T)) * 4;
  uint32_t raw[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
      raw[i] = v.x; raw[i + 1] = v.y; raw[i + 2] = v.z; raw[i + 3] = v.w;
    }
  }
  __device__ __forceinline__ void none() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw[i] = 0;
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(raw[i]);
    else if constexpr (__is_same(T, __half)) return __half2float(__ushort_as_half(uint16_t(raw[i / 2] >> (i & 1) * 16)));
    else return __uint_as_float(i & 1 ? raw[i / 2] & 0xffff0000u : raw[i / 2] << 16);
  }
  // The least magnitude that is not 0, as fp32
  __device__ __forceinline__ float least_magnitude() const {
    uint32_t m = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) m = min(m, (raw[i] & 0x7fffffffu) - 1u);
      else m = __viaddmin_u16x2(raw[i] & 0x7fff7fffu, 0xffffffffu, m);  // less 1: zeros are the largest
    }
    if constexpr (sizeof(T) == 4) return __uint_as_float(min(m, 0x7f7ffffeu) + 1u);
    m = min(min(m & 0xffffu, m >> 16), 0x7c00u) + 1u;  // beyond all finite fp16, and 2^121 in bf16: no matter
    return __is_same(T, __half) ? __half2float(__ushort_as_half(uint16_t(min(m, 0x7bffu)))) : __uint_as_float(m << 16);
  }
};

// Codes of 16 values, value i in the lowest 8 bits of code[i] (what is above them is anything).
// (x - m) / s by a reciprocal and one step that leaves it off by 2^-45 before it is rounded, so that a tie, c + 1/2 with its few bits, comes out as one and goes to the
// even code when 1.5 * 2^23 is added.  What is left of x - m then is exact; more than half a step would say that the quotient was rounded to a tie.
// x - m may be rounded itself, which matters where that makes a tie, s (c + 1/2) with its 13 bits.  In 32 bits ties are looked at again.  In 16 bits, where 0.3 % of
// normal values are ties, a rounded difference has as few bits only where all of the smaller number was lost in the larger one: a small x where -m by itself is a
// tie, or any x where m is as small.
template <typename T>
__device__ __forceinline__ void kv4_codes(uint32_t (&code)[16], const Kv4Sixteen<T>& x, Kv4Group g) {
  constexpr float kMagic = 12582912.f;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(g.s));
  if (g.s == 0.f) inv = 0.f;
  const float half = 0.5f * g.s, less_m = 0.f - g.m, less_s = -g.s;
  bool slow = !(g.s >= 0x1p-100f) && g.s != 0.f;
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    float2 h = make_float2(x.at(i), x.at(i + 1));
    add2(h.x, h.y, __float_as_uint(less_m), __float_as_uint(less_m));
    float2 q = h;
    scale2(q.x, q.y, inv);
    q = fma_f2(fma_f2(q, both(less_s), h), both(inv), q);
    add2(q.x, q.y, __float_as_uint(kMagic), __float_as_uint(kMagic));
    code[i] = __float_as_uint(q.x);
    code[i + 1] = __float_as_uint(q.y);
    add2(q.x, q.y, __float_as_uint(-kMagic), __float_as_uint(-kMagic));
    const float2 left = fma_f2(q, both(less_s), h);
    if constexpr (sizeof(T) == 4) slow |= fabsf(left.x) == half || fabsf(left.y) == half;
    asm("max.f32 %0, %0, %1, %2;" : "+f"(far) : "f"(fabsf(left.x)), "f"(fabsf(left.y)));
  }
  if constexpr (sizeof(T) == 4) slow &= g.s != 0.f;
  slow |= far > half;
  if constexpr (sizeof(T) < 4) {
    const float f = __fmaf_rd(less_m, inv * 0.9990234375f, kMagic), left = fmaf(f - kMagic, less_s, less_m);
    slow |= (left == half || left == half + g.s) && x.least_magnitude() < fabsf(g.m) * 0x1p-20f;
    slow |= g.m != 0.f && fabsf(g.m) < g.s * 0x1p-16f;
  }
  if (slow) {
#pragma unroll
    for (int i = 0; i < 16; ++i) code[i] = kv4_code(x.at(i), g);
  }
}

// A run of n tokens from `x` (`stride` elements apart) at places p0 .. p0 + n - 1 of the record `rec`: group g
template <int D, typename T>
__device__ __forceinline__ void kv4_write_run(const T* x, long long stride, int p0, int n, uint8_t* rec, int g, bool is_v) {
  constexpr int G = D / 64;
  const int lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
  const bool there[2] = {g8 >= p0 && g8 < p0 + n, g8 + 8 >= p0 && g8 + 8 < p0 + n};
  Kv4Sixteen<T> v[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (there[h]) v[h].load(x + (long long)(g8 + 8 * h - p0) * stride + 64 * g + 16 * c);
    else v[h].none();
  }
  uint32_t w[4], bytes[2][8], params[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float least = v[h].at(0), most = least;
#pragma unroll
    for (int i = 1; i < 15; i += 2) {
      least = min3_nan(least, v[h].at(i), v[h].at(i + 1));
      most = max3_nan(most, v[h].at(i), v[h].at(i + 1));
    }
    least = min_nan(least, v[h].at(15));
    most = max_nan(most, v[h].at(15));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, o));
      most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    const Kv4Group grp = kv4_group(least, most);
    params[h] = kv4_params(grp);
    uint32_t code[16];
    kv4_codes(code, v[h], grp);
#pragma unroll
    for (int i = 0; i < 8; ++i) bytes[h][i] = code[i] + code[i + 8] * 16u;  // in the lowest 8 bits
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t even = __byte_perm(bytes[0][2 * k], bytes[1][2 * k], 0x0040), odd = __byte_perm(bytes[0][2 * k + 1], bytes[1][2 * k + 1], 0x0040);
    w[k] = __byte_perm(even, odd, 0x5410);
  }
  transpose4(w, c);
  if (is_v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = transposed8(w[k]);
  }
  uint8_t* at = rec + 512 * g + 16 * lane;
  if (n == 16) {
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int b = 0; b < 4; ++b) {  // the token that has this byte of each word
      const int place = is_v ? 2 * c + (b >> 1) + 8 * (b & 1) : g8 + 8 * (b & 1);
      if (place >= p0 && place < p0 + n) {
#pragma unroll
        for (int k = 0; k < 4; ++k) at[4 * k + b] = uint8_t(w[k] >> (8 * b));
      }
    }
  }
  if (c < 2 && there[c]) reinterpret_cast<uint32_t*>(rec + 8 * D)[(g8 * 2 + c) * G + g] = params[c];
}

// One token, group g: a lane has the pair of dims of one byte
template <int D, typename T>
__device__ __forceinline__ void kv4_write_token(const T* x, int place, uint8_t* rec, int g, bool is_v) {
  const int lane = threadIdx.x & 31, j = lane >> 3, i = lane & 7;
  const T* at = x + 64 * g + 16 * j + i;
  float lo, hi;
  if constexpr (sizeof(T) == 4) { lo = at[0]; hi = at[8]; }
  else if constexpr (__is_same(T, __half)) { lo = __half2float(at[0]); hi = __half2float(at[8]); }
  else { lo = __bfloat162float(at[0]); hi = __bfloat162float(at[8]); }
  float least = min_nan(lo, hi), most = max_nan(lo, hi);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, o));
    most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  const Kv4Group grp = kv4_group(least, most);
  rec[is_v ? kv4_v_byte(place, g, j, i) : kv4_k_byte(place, g, j, i)] = uint8_t(kv4_code(lo, grp) | kv4_code(hi, grp) << 4);
  if (lane == 0) *reinterpret_cast<uint32_t*>(rec + 8 * D + kv4_param_byte<D>(place) + 4 * g) = kv4_params(grp);
}

// A warp has one group of 64 dims, which keeps small calls short: with two of them 4096 tokens of 8 heads of 128 took a fifth longer and 16384 a tenth less.  Eight
// blocks an SM in 16 bits, six in 32, and a path that fits the instruction cache (the exact choice of a code is a call): 49 -> 28 us for 16384 tokens.
// Now 26.9 us for these (half of the copy rate), 9.3 for 4096, 3.4 for 64 single ones.  19 instructions a value, issue and the latency of the loads
// together are what bounds it; several groups one after the other in a warp, to look its tokens up once, gave nothing.
template <int D, typename T>
__global__ void __launch_bounds__(128, sizeof(T) == 4 ? 6 : 8) kv4_write_kernel(Kv4WriteArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  constexpr int G = D / 64;
  const unsigned at_window = blockIdx.x / a.blocks, job = blockIdx.x % a.blocks * 4 + (threadIdx.x >> 5);  // of a window's (head, K or V, group)
  const long long first = (long long)at_window * a.window;
  if (job >= unsigned(2 * G * a.Hk)) return;
  const int head = job / (2 * G), g = job % G;
  const bool is_v = job / G & 1;
  // lane i: token first - 1 + i.  A run begins in the window and ends 15 tokens behind it at most
  const long long token = first - 1 + lane;
  int slot = token >= 0 && token < a.T ? a.slots[token] : -1;
  if (slot >= 0 && (slot >> 4) >= a.pages) {
    atomicCAS(a.status, 0, kStatusBadArgument);
    slot = -1;
  }
  const int before = __shfl_up_sync(0xffffffffu, slot, 1);
  const bool goes_on = slot >= 0 && (slot & 15) && before == slot - 1;
  const uint32_t on = __ballot_sync(0xffffffffu, goes_on);
  uint32_t begins = __ballot_sync(0xffffffffu, slot >= 0 && !goes_on) & (((1u << a.window) - 1u) << 1);
  while (begins) {
    const int i = __ffs(begins) - 1;
    begins &= begins - 1;
    const int n = __ffs(~(on >> (i + 1)));  // 1 and the ones behind bit i, which is 16 at most
    const int at = __shfl_sync(0xffffffffu, slot, i);
    uint8_t* rec = a.pool + (size_t(at >> 4) * a.Hk + head) * (18 * D) + (is_v ? 9 * D : 0);
    const long long t = first - 1 + i;
    const T* x = static_cast<const T*>(is_v ? a.v : a.k) + (is_v ? t * a.v_token + head * a.v_head : t * a.k_token + head * a.k_head);
    if (n == 1) kv4_write_token<D, T>(x, at & 15, rec, g, is_v);
    else kv4_write_run<D, T>(x, is_v ? a.v_token : a.k_token, at & 15, n, rec, g, is_v);
  }
}

struct Kv4GatherArgs {
  const uint8_t* pool;
  const int *table, *starts, *first;  // first: null: 0
  void *k, *v;
  int* status;
  long long k_token, k_head, v_token, v_head;
  int B, N, Hk, width, pages, window;
  unsigned blocks;
};

template <typename T>
__device__ __forceinline__ void kv4_store16(T* to, const float (&y)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 16 / int(sizeof(T))) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) {
        w[k] = __float_as_uint(y[i + k]);
      } else if constexpr (__is_same(T, __half)) {
        const __half2 v = __floats2half2_rn(y[i + 2 * k], y[i + 2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(y[i + 2 * k], y[i + 2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    reinterpret_cast<uint4*>(to + i)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// K or V of a record as a lane has them: requested first, used behind all that was requested
template <int D>
struct Kv4Raw {
  static constexpr int G = D / 64;
  uint4 raw[G];
  uint32_t params[2 * G];  // [place g8, g8 + 8][group]
  __device__ __forceinline__ void load(const uint8_t* rec) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < G; ++g) raw[g] = *reinterpret_cast<const uint4*>(rec + 512 * g + 16 * lane);
#pragma unroll
    for (int i = 0; i < 2 * G; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(rec + 8 * D + 8 * G * (lane >> 2) + 4 * i);
      params[i] = v.x; params[i + 1] = v.y;
    }
  }
};

// The tokens at places p0 .. p0 + n - 1 to `y` (`stride` elements apart)
template <int D, typename T, bool kV>
__device__ __forceinline__ void kv4_read_run(const Kv4Raw<D>& rec, int p0, int n, T* y, long long stride) {
  constexpr int G = D / 64;
  const int lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
  const auto& raw = rec.raw;
  const auto& params = rec.params;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
    if constexpr (kV) {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = transposed8(w[k]);
    }
    // 16 bits: a lane gets 16 neighbouring dims.  32 bits: the four lanes of a row have 8 neighbouring ones as they are, a sector
    if constexpr (sizeof(T) < 4) transpose4(w, c);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int place = g8 + 8 * h;
      const bool there = place >= p0 && place < p0 + n;
      T* to = y + (long long)(place - p0) * stride + 64 * g;
      const float s = __uint_as_float(params[h * G + g] << 16), m = __uint_as_float(params[h * G + g] & 0xffff0000u);
      const auto value = [&](uint32_t code) { return fmaf(s, __uint_as_float((code & 15u) | 0x4b000000u) - 8388608.f, m); };  // 2^23 + c, exactly
      if constexpr (sizeof(T) < 4) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t byte = w[i >> 1] >> (16 * (i & 1) + 8 * h);
          v[i] = value(byte);
          v[i + 8] = value(byte >> 4);
        }
        if (there) kv4_store16(to + 16 * c, v);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t code = w[k] >> (8 * h + 4 * e);
            if (there) *reinterpret_cast<float2*>(to + 16 * k + 8 * e + 2 * c) = make_float2(value(code), value(code >> 16));
          }
        }
      }
    }
  }
}

// The sequence whose rows have row r: the last one that starts at r or before, by a whole warp, in steps of a 32nd
__device__ __forceinline__ int kv4_sequence(const int* starts, int B, int r) {
  int lo = 0;
  for (int span = B; span > 1;) {
    const int part = (span + 31) >> 5, at = int(lane_id()) * part;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, at == 0 || (at < span && starts[lo + at] <= r)));
    lo += last * part;
    span = min(part, span - last * part);
  }
  return lo;
}

__host__ __device__ constexpr int kv4_gather_heads(int d) { return d == 64 ? 2 : 1; }

// 131072 tokens of 8 heads of 128 in bf16: 110 to 115 us, 0.92 to 0.96 of the copy rate, which bounds it; 4096 of them 7.9 us, by the lookups before the first load
// (sequence, position, page) and one round of warps.  K and V of a head in one warp, all requested first: 116 -> 110 us, heads of 64 (two of them) 35 -> 28.
template <int D, typename T>
__global__ void __launch_bounds__(128) kv4_gather_kernel(Kv4GatherArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  constexpr int kEach = D == 256 ? 1 : 2, kHeads = kv4_gather_heads(D);  // a warp has K or V of a head of 256, both of one of 128, of two of 64
  const unsigned at_window = blockIdx.x / a.blocks, job = blockIdx.x % a.blocks * 4 + (threadIdx.x >> 5);
  const long long first = (long long)at_window * a.window;
  const int head = job / (2 / kEach) * kHeads;
  if (head >= a.Hk) return;
  const bool is_v = kEach == 1 && (job & 1);
  // lane i: row first - 1 + i, as in the kernel above; a run is one of rows whose tokens follow one another in a page, whoever's they are
  const long long row = first - 1 + lane;
  int slot = -1, seq = kv4_sequence(a.starts, a.B, int(max(first - 1, 0ll)));
  if (row >= 0 && row < a.N && row >= a.starts[0] && row < a.starts[a.B]) {
    while (seq + 1 < a.B && a.starts[seq + 1] <= row) ++seq;
    const long long pos = (long long)(a.first ? a.first[seq] : 0) + row - a.starts[seq];
    const int page = pos >= 0 && (pos >> 4) < a.width ? a.table[size_t(seq) * a.width + (pos >> 4)] : -1;
    if (page < 0 || page >= a.pages) atomicCAS(a.status, 0, kStatusBadArgument);
    else slot = page * 16 + int(pos & 15);
  }
  const int before = __shfl_up_sync(0xffffffffu, slot, 1);
  const bool goes_on = slot >= 0 && (slot & 15) && before == slot - 1;
  const uint32_t on = __ballot_sync(0xffffffffu, goes_on);
  uint32_t begins = __ballot_sync(0xffffffffu, slot >= 0 && !goes_on) & (((1u << a.window) - 1u) << 1);
  while (begins) {
    const int i = __ffs(begins) - 1;
    begins &= begins - 1;
    const int n = __ffs(~(on >> (i + 1)));  // 1 and the ones behind bit i, which is 16 at most
    const int at = __shfl_sync(0xffffffffu, slot, i);
    const long long to = first - 1 + i;
    Kv4Raw<D> raw[kHeads][kEach];
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      const uint8_t* rec = a.pool + (size_t(at >> 4) * a.Hk + min(head + k, a.Hk - 1)) * (18 * D);
      raw[k][0].load(rec + (is_v ? 9 * D : 0));
      if constexpr (kEach == 2) raw[k][kEach - 1].load(rec + 9 * D);
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      if (head + k >= a.Hk) break;
      T *ky = static_cast<T*>(a.k) + to * a.k_token + (head + k) * a.k_head, *vy = static_cast<T*>(a.v) + to * a.v_token + (head + k) * a.v_head;
      if (!is_v) kv4_read_run<D, T, false>(raw[k][0], at & 15, n, ky, a.k_token);
      if (kEach == 2 || is_v) kv4_read_run<D, T, true>(raw[k][kEach - 1], at & 15, n, vy, a.v_token);
    }
  }
}

// Tokens in which the runs of a warp begin: one where the warps of all tokens have room at once, as in a decode step, since a run is one token there, and runs
// in a row take their time one after the other; 16 in a prompt, where these have one run or two
static int kv4_window(long long units) {
  int w = 1;
  while (w < 16 && units / w > 148 * 64) w *= 2;
  return w;
}

template <int D>
static int launch_write(Kv4WriteArgs a, int dtype, cudaStream_t stream) {
  a.window = kv4_window(2ll * a.T * a.Hk);
  a.blocks = (2 * a.Hk * (D / 64) + 3) / 4;
  const long long blocks = (a.T + a.window - 1ll) / a.window * a.blocks;
  if (blocks > 0x7fffffffll) return -2;
  auto kernel = dtype == 0 ? kv4_write_kernel<D, __nv_bfloat16> : (dtype == 1 ? kv4_write_kernel<D, __half> : kv4_write_kernel<D, float>);
  return launch_kernel(kernel, dim3(unsigned(blocks)), dim3(128), 0, stream, a) == cudaSuccess ? 0 : -7;
}
template <int D>
static int launch_gather(Kv4GatherArgs a, int dtype, cudaStream_t stream) {
  a.window = kv4_window(2ll * a.N * a.Hk);
  const int heads = kv4_gather_heads(D);
  a.blocks = ((a.Hk + heads - 1) / heads * (D == 256 ? 2 : 1) + 3) / 4;
  const long long blocks = (a.N + a.window - 1ll) / a.window * a.blocks;
  if (blocks > 0x7fffffffll) return -2;
  auto kernel = dtype == 0 ? kv4_gather_kernel<D, __nv_bfloat16> : (dtype == 1 ? kv4_gather_kernel<D, __half> : kv4_gather_kernel<D, float>);
  return launch_kernel(kernel, dim3(unsigned(blocks)), dim3(128), 0, stream, a) == cudaSuccess ? 0 : -7;
}

}  // namespace mfq

// k, v: [T, Hk, D] of dtype 0 bf16, 1 fp16, 2 fp32, strides in elements; pool: [pages, Hk, 18 D]; slots [T]: page * 16 + place, negative: none
extern "C" int mfq_kv4_write(const void* k, const void* v, const int* slots, uint8_t* pool, int dtype, int T, int Hk, int D, int pages, long long k_token,
                             long long k_head, long long v_token, long long v_head, int* status, cudaStream_t stream) {
  if (T <= 0 || Hk <= 0 || pages <= 0 || dtype < 0 || dtype > 2) return -1;
  const mfq::Kv4WriteArgs a{k, v, slots, pool, status, k_token, k_head, v_token, v_head, T, Hk, pages, 1, 1};
  if (D == 64) return mfq::launch_write<64>(a, dtype, stream);
  if (D == 128) return mfq::launch_write<128>(a, dtype, stream);
  if (D == 256) return mfq::launch_write<256>(a, dtype, stream);
  return -1;
}

// Rows starts[i] .. starts[i + 1] - 1 of k, v ([N, Hk, D], strides in elements) get sequence i's tokens from position first[i] on; table: [B, width]
extern "C" int mfq_kv4_gather(const uint8_t* pool, const int* table, const int* starts, const int* first, void* k, void* v, int dtype, int B, int N, int Hk, int D,
                              int width, int pages, long long k_token, long long k_head, long long v_token, long long v_head, int* status, cudaStream_t stream) {
  if (B <= 0 || N <= 0 || Hk <= 0 || width <= 0 || pages <= 0 || dtype < 0 || dtype > 2) return -1;
  const mfq::Kv4GatherArgs a{pool, table, starts, first, k, v, status, k_token, k_head, v_token, v_head, B, N, Hk, width, pages, 1, 1};
  if (D == 64) return mfq::launch_gather<64>(a, dtype, stream);
  if (D == 128) return mfq::launch_gather<128>(a, dtype, stream);
  if (D == 256) return mfq::launch_gather<256>(a, dtype, stream);
  return -1;
}
