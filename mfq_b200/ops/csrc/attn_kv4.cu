// Decode / verify attention over pages held in 4 bits (kv4.cuh has the format).
// A warp takes one query row and head: token by token, with the running maximum and sum of the softmax; a lane has the dims of one byte of every group.
#include "kv4.cuh"

namespace mfq {

struct Kv4AttnArgs {
  const void* q;
  const uint8_t* pool;
  const int *table, *seq_lens;
  void* out;
  float *part_o, *part_ml;
  int* status;
  int B, Hq, Hk, width, pages, q_len, splits, chunk;
  float scale_log2;
};

template <int D, bool kHalf>
__global__ void __launch_bounds__(128) kv4_attn_kernel(Kv4AttnArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int G = D / 64;
  const int lane = threadIdx.x & 31, j = lane >> 3, i = lane & 7;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= (long long)a.B * a.q_len * a.Hq) return;
  const long long row = unit / a.Hq;
  const int head = int(unit % a.Hq), kvh = head / (a.Hq / a.Hk), seq = int(row / a.q_len);
  const int len = int(min((long long)a.seq_lens[seq], 16ll * a.width)) - (a.q_len - 1 - int(row % a.q_len));
  float q[G][2], o[G][2], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const size_t at = size_t(unit) * D + 64 * g + 16 * j + i + 8 * e;
      q[g][e] = (kHalf ? __half2float(static_cast<const __half*>(a.q)[at]) : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at])) * a.scale_log2;
      o[g][e] = 0.f;
    }
  }
  for (int t = 0; t < len; ++t) {
    int page = a.table[size_t(seq) * a.width + (t >> 4)];
    if (page < 0 || page >= a.pages) {
      if (lane == 0) atomicCAS(a.status, 0, kStatusBadArgument);
      page = 0;
    }
    const uint8_t* rec = a.pool + (size_t(page) * a.Hk + kvh) * (18 * D);
    float part = 0.f, v[G][2];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int at = 8 * D + kv4_param_byte<D>(t & 15) + 4 * g;
      const uint32_t kp = *reinterpret_cast<const uint32_t*>(rec + at), vp = *reinterpret_cast<const uint32_t*>(rec + 9 * D + at);
      const uint32_t kc = rec[kv4_k_byte(t & 15, g, j, i)], vc = rec[9 * D + kv4_v_byte(t & 15, g, j, i)];
      const float ks = __uint_as_float(kp << 16), km = __uint_as_float(kp & 0xffff0000u), vs = __uint_as_float(vp << 16), vm = __uint_as_float(vp & 0xffff0000u);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        part += q[g][e] * fmaf(ks, float(kc >> (4 * e) & 15), km);
        v[g][e] = fmaf(vs, float(vc >> (4 * e) & 15), vm);
      }
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) part += __shfl_xor_sync(0xffffffffu, part, x);
    const float next = fmaxf(top, part), keep = exp2f(top - next), p = exp2f(part - next);
    top = next;
    sum = sum * keep + p;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      o[g][0] = o[g][0] * keep + p * v[g][0];
      o[g][1] = o[g][1] * keep + p * v[g][1];
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const size_t at = size_t(unit) * D + 64 * g + 16 * j + i + 8 * e;
      const float y = len > 0 ? o[g][e] / sum : 0.f;
      if (kHalf) static_cast<__half*>(a.out)[at] = __float2half_rn(y);
      else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16(y);
    }
  }
}

template <int D>
static int launch_kv4_attn(const Kv4AttnArgs& a, bool half, cudaStream_t stream) {
  const long long blocks = ((long long)a.B * a.q_len * a.Hq + 3) / 4;
  if (blocks > 0x7fffffffll) return -2;
  return launch_kernel(half ? kv4_attn_kernel<D, true> : kv4_attn_kernel<D, false>, dim3(unsigned(blocks)), dim3(128), 0, stream, a) == cudaSuccess ? 0 : -7;
}

}  // namespace mfq

// q, out: [B * q_len, Hq, D] bf16 or fp16 (`half`); pool: [pages, Hk, 18 D]; table: [B, width]; seq_lens count every token visible to the last query row.
// The tokens of a sequence are taken in chunks of `chunk` pages by `splits` blocks in turn; part_o, part_ml: [B * q_len * Hq, splits, D], [.., 2] fp32.
extern "C" int mfq_paged_attn_decode_kv4(const void* q, const uint8_t* pool, const int* table, const int* seq_lens, void* out, float* part_o, float* part_ml, int half,
                                         int B, int Hq, int Hk, int D, int width, int pages, int q_len, int splits, int chunk, float sm_scale, int* status,
                                         cudaStream_t stream) {
  if (B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || q_len < 1 || width <= 0 || pages <= 0 || splits < 1 || chunk < 1) return -1;
  const mfq::Kv4AttnArgs a{q, pool, table, seq_lens, out, part_o, part_ml, status, B, Hq, Hk, width, pages, q_len, splits, chunk, sm_scale * 1.4426950408889634f};
  if (D == 64) return mfq::launch_kv4_attn<64>(a, half != 0, stream);
  if (D == 128) return mfq::launch_kv4_attn<128>(a, half != 0, stream);
  if (D == 256) return mfq::launch_kv4_attn<256>(a, half != 0, stream);
  return -1;
}
