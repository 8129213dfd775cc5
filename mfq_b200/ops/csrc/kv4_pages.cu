// Writing and reading back pages held in 4 bits (kv4.cuh has the format).
// A warp takes one token of one head's K or V: a lane has the byte of one pair of dims in every group of 64.
#include "kv4.cuh"

namespace mfq {

struct Kv4WriteArgs {
  const void *k, *v;
  const int* slots;
  uint8_t* pool;
  int* status;
  long long k_token, k_head, v_token, v_head;  // strides in elements
  int T, Hk, pages;
};

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ float from_f32(float x) { return x; }

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

template <int D, typename T>
__global__ void __launch_bounds__(256) kv4_write_kernel(Kv4WriteArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, j = lane >> 3, i = lane & 7;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= 2ll * a.T * a.Hk) return;
  const int token = int(unit / (2 * a.Hk)), head = int(unit % (2 * a.Hk)) >> 1;
  const bool is_v = unit & 1;
  const int slot = a.slots[token];
  if (slot < 0) return;
  if ((slot >> 4) >= a.pages) {
    if (lane == 0) atomicCAS(a.status, 0, kStatusBadArgument);
    return;
  }
  const T* x = static_cast<const T*>(is_v ? a.v : a.k) + (is_v ? token * a.v_token + head * a.v_head : token * a.k_token + head * a.k_head);
  uint8_t* rec = a.pool + (size_t(slot >> 4) * a.Hk + head) * (18 * D) + (is_v ? 9 * D : 0);
  const int t = slot & 15;
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    const float lo = to_f32(x[64 * g + 16 * j + i]), hi = to_f32(x[64 * g + 16 * j + i + 8]);
    float least = min_nan(lo, hi), most = max_nan(lo, hi);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, o));
      most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    const Kv4Group grp = kv4_group(least, most);
    rec[is_v ? kv4_v_byte(t, g, j, i) : kv4_k_byte(t, g, j, i)] = uint8_t(kv4_code(lo, grp) | kv4_code(hi, grp) << 4);
    if (lane == 0) *reinterpret_cast<uint32_t*>(rec + 8 * D + kv4_param_byte<D>(t) + 4 * g) = kv4_params(grp);
  }
}

struct Kv4GatherArgs {
  const uint8_t* pool;
  const int *table, *starts, *first;  // first: null: 0
  void *k, *v;
  int* status;
  long long k_token, k_head, v_token, v_head;
  int B, N, Hk, width, pages;
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

template <int D, typename T>
__global__ void __launch_bounds__(256) kv4_gather_kernel(Kv4GatherArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, j = lane >> 3, i = lane & 7;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= 2ll * a.N * a.Hk) return;
  const int row = int(unit / (2 * a.Hk)), head = int(unit % (2 * a.Hk)) >> 1;
  const bool is_v = unit & 1;
  if (row < a.starts[0] || row >= a.starts[a.B]) return;
  const int seq = kv4_sequence(a.starts, a.B, row);
  const long long pos = (long long)(a.first ? a.first[seq] : 0) + row - a.starts[seq];
  const int page = pos >= 0 && (pos >> 4) < a.width ? a.table[size_t(seq) * a.width + (pos >> 4)] : -1;
  if (page < 0 || page >= a.pages) {
    if (lane == 0) atomicCAS(a.status, 0, kStatusBadArgument);
    return;
  }
  const int t = int(pos & 15);
  const uint8_t* rec = a.pool + (size_t(page) * a.Hk + head) * (18 * D) + (is_v ? 9 * D : 0);
  T* y = static_cast<T*>(is_v ? a.v : a.k) + (is_v ? row * a.v_token + head * a.v_head : row * a.k_token + head * a.k_head);
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    const uint32_t params = *reinterpret_cast<const uint32_t*>(rec + 8 * D + kv4_param_byte<D>(t) + 4 * g);
    const float s = __uint_as_float(params << 16), m = __uint_as_float(params & 0xffff0000u);
    const uint32_t both = rec[is_v ? kv4_v_byte(t, g, j, i) : kv4_k_byte(t, g, j, i)];
    y[64 * g + 16 * j + i] = from_f32<T>(fmaf(s, float(both & 15), m));
    y[64 * g + 16 * j + i + 8] = from_f32<T>(fmaf(s, float(both >> 4), m));
  }
}

template <int D>
static int launch_write(const Kv4WriteArgs& a, int dtype, cudaStream_t stream) {
  const long long blocks = (2ll * a.T * a.Hk + 7) / 8;
  if (blocks > 0x7fffffffll) return -2;
  auto kernel = dtype == 0 ? kv4_write_kernel<D, __nv_bfloat16> : (dtype == 1 ? kv4_write_kernel<D, __half> : kv4_write_kernel<D, float>);
  return launch_kernel(kernel, dim3(unsigned(blocks)), dim3(256), 0, stream, a) == cudaSuccess ? 0 : -7;
}
template <int D>
static int launch_gather(const Kv4GatherArgs& a, int dtype, cudaStream_t stream) {
  const long long blocks = (2ll * a.N * a.Hk + 7) / 8;
  if (blocks > 0x7fffffffll) return -2;
  auto kernel = dtype == 0 ? kv4_gather_kernel<D, __nv_bfloat16> : (dtype == 1 ? kv4_gather_kernel<D, __half> : kv4_gather_kernel<D, float>);
  return launch_kernel(kernel, dim3(unsigned(blocks)), dim3(256), 0, stream, a) == cudaSuccess ? 0 : -7;
}

}  // namespace mfq

// k, v: [T, Hk, D] of dtype 0 bf16, 1 fp16, 2 fp32, strides in elements; pool: [pages, Hk, 18 D]; slots [T]: page * 16 + place, negative: none
extern "C" int mfq_kv4_write(const void* k, const void* v, const int* slots, uint8_t* pool, int dtype, int T, int Hk, int D, int pages, long long k_token,
                             long long k_head, long long v_token, long long v_head, int* status, cudaStream_t stream) {
  if (T <= 0 || Hk <= 0 || pages <= 0 || dtype < 0 || dtype > 2) return -1;
  const mfq::Kv4WriteArgs a{k, v, slots, pool, status, k_token, k_head, v_token, v_head, T, Hk, pages};
  if (D == 64) return mfq::launch_write<64>(a, dtype, stream);
  if (D == 128) return mfq::launch_write<128>(a, dtype, stream);
  if (D == 256) return mfq::launch_write<256>(a, dtype, stream);
  return -1;
}

// Rows starts[i] .. starts[i + 1] - 1 of k, v ([N, Hk, D], strides in elements) get sequence i's tokens from position first[i] on; table: [B, width]
extern "C" int mfq_kv4_gather(const uint8_t* pool, const int* table, const int* starts, const int* first, void* k, void* v, int dtype, int B, int N, int Hk, int D,
                              int width, int pages, long long k_token, long long k_head, long long v_token, long long v_head, int* status, cudaStream_t stream) {
  if (B <= 0 || N <= 0 || Hk <= 0 || width <= 0 || pages <= 0 || dtype < 0 || dtype > 2) return -1;
  const mfq::Kv4GatherArgs a{pool, table, starts, first, k, v, status, k_token, k_head, v_token, v_head, B, N, Hk, width, pages};
  if (D == 64) return mfq::launch_gather<64>(a, dtype, stream);
  if (D == 128) return mfq::launch_gather<128>(a, dtype, stream);
  if (D == 256) return mfq::launch_gather<256>(a, dtype, stream);
  return -1;
}
