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

// Codes of 16 values, value i in the lowest 4 bits of code[i] (what is above them is anything).
// floor((x - m) / s) is found by the rounded reciprocal, one too large or small at worst where the quotient is next to an integer, and what is left of x - m
// is exact: it says whether the value is nearer to the next code.  x - m may be rounded itself, which matters where that is a tie, s (c + 1/2) with its 13 bits.
// In 32 bits a tie is looked at again; in 16 bits, where 0.3 % of normal values are ties, a rounded difference has as few bits only where all of the smaller
// number was lost in the larger one, 2^-23 of it or less.
template <typename T>
__device__ __forceinline__ void kv4_codes(uint32_t (&code)[16], const Kv4Sixteen<T>& x, Kv4Group g) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: integers in the lowest bits
  const float inv = g.s != 0.f ? 1.f / g.s : 0.f, half = 0.5f * g.s;
  bool slow = !(g.s >= 0x1p-120f) && g.s != 0.f;
  if constexpr (sizeof(T) < 4) {
    const float big = fmaxf(fabsf(g.m), 15.f * g.s), small = fminf(x.least_magnitude(), g.m != 0.f ? fabsf(g.m) : big);
    slow |= small < big * 0x1p-20f;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float h = x.at(i) - g.m, v = __fmaf_rd(h, inv, kMagic), left = fmaf(-g.s, v - kMagic, h);
    const uint32_t bits = __float_as_uint(v);
    if constexpr (sizeof(T) == 4) slow |= left == half;
    code[i] = bits + (left > __uint_as_float(__float_as_uint(half) - (bits & 1u)) ? 1u : 0u);  // half a step from an odd code: to the even one
  }
  if (slow) {
#pragma unroll
    for (int i = 0; i < 16; ++i) code[i] = kv4_code(x.at(i), g);
  }
}

// A run of n tokens from `x` (`stride` elements apart) at places p0 .. p0 + n - 1 of the record `rec`
template <int D, typename T, bool kV>
__device__ __forceinline__ void kv4_write_run(const T* x, long long stride, int p0, int n, uint8_t* rec) {
  constexpr int G = D / 64, kAhead = G * int(sizeof(T)) <= 4 ? G : 4 / int(sizeof(T));  // groups whose values are requested at once
  const int lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
  const bool there[2] = {g8 >= p0 && g8 < p0 + n, g8 + 8 >= p0 && g8 + 8 < p0 + n};
  const T* from[2] = {x + (long long)(g8 - p0) * stride + 16 * c, x + (long long)(g8 + 8 - p0) * stride + 16 * c};
  uint32_t params[2][G];
#pragma unroll
  for (int g0 = 0; g0 < G; g0 += kAhead) {
    Kv4Sixteen<T> v[kAhead][2];
#pragma unroll
    for (int g = 0; g < kAhead; ++g) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (there[h]) v[g][h].load(from[h] + 64 * (g0 + g));
        else v[g][h].none();
      }
    }
#pragma unroll
    for (int g = 0; g < kAhead; ++g) {
      uint32_t w[4], bytes[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float least = v[g][h].at(0), most = least;
#pragma unroll
        for (int i = 1; i < 15; i += 2) {
          least = min3_nan(least, v[g][h].at(i), v[g][h].at(i + 1));
          most = max3_nan(most, v[g][h].at(i), v[g][h].at(i + 1));
        }
        least = min_nan(least, v[g][h].at(15));
        most = max_nan(most, v[g][h].at(15));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, o));
          most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        const Kv4Group grp = kv4_group(least, most);
        params[h][g0 + g] = kv4_params(grp);
        uint32_t code[16];
        kv4_codes(code, v[g][h], grp);
#pragma unroll
        for (int i = 0; i < 8; ++i) bytes[h][i] = (code[i] & 15u) + code[i + 8] * 16u;  // in the lowest 8 bits
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t even = __byte_perm(bytes[0][2 * k], bytes[1][2 * k], 0x0040), odd = __byte_perm(bytes[0][2 * k + 1], bytes[1][2 * k + 1], 0x0040);
        w[k] = __byte_perm(even, odd, 0x5410);
      }
      transpose4(w, c);
      if constexpr (kV) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = transposed8(w[k]);
      }
      uint8_t* at = rec + 512 * (g0 + g) + 16 * lane;
      if (n == 16) {
        *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int b = 0; b < 4; ++b) {  // the token that has this byte of each word
          const int place = kV ? 2 * c + (b >> 1) + 8 * (b & 1) : g8 + 8 * (b & 1);
          if (place >= p0 && place < p0 + n) {
#pragma unroll
            for (int k = 0; k < 4; ++k) at[4 * k + b] = uint8_t(w[k] >> (8 * b));
          }
        }
      }
    }
  }
  uint32_t* to = reinterpret_cast<uint32_t*>(rec + 8 * D) + g8 * 2 * G;  // [place g8, g8 + 8][group]
#pragma unroll
  for (int i = 0; i < 2 * G; ++i) {
    if (i % 4 == c && there[i / G]) to[i] = params[i / G][i % G];
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(128) kv4_write_kernel(Kv4WriteArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long of = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long first = of / (2 * a.Hk) * a.window;
  if (first >= a.T) return;
  const int head = int(of % (2 * a.Hk)) >> 1;
  const bool is_v = of & 1;
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
    if (is_v) kv4_write_run<D, T, true>(static_cast<const T*>(a.v) + t * a.v_token + head * a.v_head, a.v_token, at & 15, n, rec);
    else kv4_write_run<D, T, false>(static_cast<const T*>(a.k) + t * a.k_token + head * a.k_head, a.k_token, at & 15, n, rec);
  }
}

struct Kv4GatherArgs {
  const uint8_t* pool;
  const int *table, *starts, *first;  // first: null: 0
  void *k, *v;
  int* status;
  long long k_token, k_head, v_token, v_head;
  int B, N, Hk, width, pages, window;
};

// The sequence whose rows have row r: the last one that starts at r or before
__device__ __forceinline__ int kv4_sequence(const int* starts, int B, int r) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (starts[mid] <= r) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

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

// n tokens at places p0 .. p0 + n - 1 of the record `rec` to `y` (`stride` elements apart)
template <int D, typename T, bool kV>
__device__ __forceinline__ void kv4_read_run(const uint8_t* rec, int p0, int n, T* y, long long stride) {
  constexpr int G = D / 64;
  const int lane = threadIdx.x & 31, g8 = lane >> 2, c = lane & 3;
  uint4 raw[G];
  uint32_t params[2 * G];  // [place g8, g8 + 8][group]
#pragma unroll
  for (int g = 0; g < G; ++g) raw[g] = *reinterpret_cast<const uint4*>(rec + 512 * g + 16 * lane);
#pragma unroll
  for (int i = 0; i < 2 * G; i += 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(rec + 8 * D + 8 * G * g8 + 4 * i);
    params[i] = v.x; params[i + 1] = v.y;
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
    if constexpr (kV) {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = transposed8(w[k]);
    }
    transpose4(w, c);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float s = __uint_as_float(params[h * G + g] << 16), m = __uint_as_float(params[h * G + g] & 0xffff0000u);
      float v[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t byte = w[i >> 1] >> (16 * (i & 1) + 8 * h);
        v[i] = fmaf(s, __uint_as_float((byte & 15u) | 0x4b000000u) - 8388608.f, m);  // 2^23 + c, exactly
        v[i + 8] = fmaf(s, __uint_as_float((byte >> 4 & 15u) | 0x4b000000u) - 8388608.f, m);
      }
      const int place = g8 + 8 * h;
      if (place >= p0 && place < p0 + n) kv4_store16(y + (long long)(place - p0) * stride + 64 * g + 16 * c, v);
    }
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(128) kv4_gather_kernel(Kv4GatherArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long of = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long first = of / (2 * a.Hk) * a.window;
  if (first >= a.N) return;
  const int head = int(of % (2 * a.Hk)) >> 1;
  const bool is_v = of & 1;
  // lane i: row first - 1 + i, as in the kernel above; a run is one of rows whose tokens follow one another in a page, whoever's they are
  const long long row = first - 1 + lane;
  int slot = -1;
  if (row >= 0 && row < a.N && row >= a.starts[0] && row < a.starts[a.B]) {
    const int seq = kv4_sequence(a.starts, a.B, int(row));
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
    const uint8_t* rec = a.pool + (size_t(at >> 4) * a.Hk + head) * (18 * D) + (is_v ? 9 * D : 0);
    const long long to = first - 1 + i;
    if (is_v) kv4_read_run<D, T, true>(rec, at & 15, n, static_cast<T*>(a.v) + to * a.v_token + head * a.v_head, a.v_token);
    else kv4_read_run<D, T, false>(rec, at & 15, n, static_cast<T*>(a.k) + to * a.k_token + head * a.k_head, a.k_token);
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
  const long long blocks = ((a.T + a.window - 1ll) / a.window * 2 * a.Hk + 3) / 4;
  if (blocks > 0x7fffffffll) return -2;
  auto kernel = dtype == 0 ? kv4_write_kernel<D, __nv_bfloat16> : (dtype == 1 ? kv4_write_kernel<D, __half> : kv4_write_kernel<D, float>);
  return launch_kernel(kernel, dim3(unsigned(blocks)), dim3(128), 0, stream, a) == cudaSuccess ? 0 : -7;
}
template <int D>
static int launch_gather(Kv4GatherArgs a, int dtype, cudaStream_t stream) {
  a.window = kv4_window(2ll * a.N * a.Hk);
  const long long blocks = ((a.N + a.window - 1ll) / a.window * 2 * a.Hk + 3) / 4;
  if (blocks > 0x7fffffffll) return -2;
  auto kernel = dtype == 0 ? kv4_gather_kernel<D, __nv_bfloat16> : (dtype == 1 ? kv4_gather_kernel<D, __half> : kv4_gather_kernel<D, float>);
  return launch_kernel(kernel, dim3(unsigned(blocks)), dim3(128), 0, stream, a) == cudaSuccess ? 0 : -7;
}

}  // namespace mfq

// k, v: [T, Hk, D] of dtype 0 bf16, 1 fp16, 2 fp32, strides in elements; pool: [pages, Hk, 18 D]; slots [T]: page * 16 + place, negative: none
extern "C" int mfq_kv4_write(const void* k, const void* v, const int* slots, uint8_t* pool, int dtype, int T, int Hk, int D, int pages, long long k_token,
                             long long k_head, long long v_token, long long v_head, int* status, cudaStream_t stream) {
  if (T <= 0 || Hk <= 0 || pages <= 0 || dtype < 0 || dtype > 2) return -1;
  const mfq::Kv4WriteArgs a{k, v, slots, pool, status, k_token, k_head, v_token, v_head, T, Hk, pages, 1};
  if (D == 64) return mfq::launch_write<64>(a, dtype, stream);
  if (D == 128) return mfq::launch_write<128>(a, dtype, stream);
  if (D == 256) return mfq::launch_write<256>(a, dtype, stream);
  return -1;
}

// Rows starts[i] .. starts[i + 1] - 1 of k, v ([N, Hk, D], strides in elements) get sequence i's tokens from position first[i] on; table: [B, width]
extern "C" int mfq_kv4_gather(const uint8_t* pool, const int* table, const int* starts, const int* first, void* k, void* v, int dtype, int B, int N, int Hk, int D,
                              int width, int pages, long long k_token, long long k_head, long long v_token, long long v_head, int* status, cudaStream_t stream) {
  if (B <= 0 || N <= 0 || Hk <= 0 || width <= 0 || pages <= 0 || dtype < 0 || dtype > 2) return -1;
  const mfq::Kv4GatherArgs a{pool, table, starts, first, k, v, status, k_token, k_head, v_token, v_head, B, N, Hk, width, pages, 1};
  if (D == 64) return mfq::launch_gather<64>(a, dtype, stream);
  if (D == 128) return mfq::launch_gather<128>(a, dtype, stream);
  if (D == 256) return mfq::launch_gather<256>(a, dtype, stream);
  return -1;
}
