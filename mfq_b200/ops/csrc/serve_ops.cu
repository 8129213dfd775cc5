// What a served batch needs beside its forward pass: the plan of a ragged batch before it, the processing of its logits after it.
//
//   process_logits   biases, penalties for repeated tokens and a grammar's mask on [B, V] logits, one pass, one rounding
//   count_tokens     the occurrences that the penalties go by
//   plan_batch       positions, KV slots and block tables of a ragged batch from the lengths of its requests
//
// The reference applies penalties from a count tensor in front of its sampler (mfq/kernels/cuda/sampling.cu) and plans batches on the
// host (cpp_runtime/engine/include/continuous_batch.h).
#include "common.cuh"

#include <cuda_fp16.h>

namespace mfq {

// ----- logits -----
// For row b with tables' row r and vocabulary id v:
//   l = logit + sum of the row's biases for v;   word = counts[r][v]: 15 bits of occurrences n, the top bit: the prompt has v
//   word != 0:  l = l > 0 ? l / repetition : l * repetition;   n > 0:  l -= presence + frequency * n
//   out = allowed[r] bit v ? round(l) : fill     (chosen, not added: a masked NaN or infinity is gone)
// All of it in fp32, rounded once to the logits' type.

struct LogitRecord {  // the 32 bytes a row's sampler reads; on 4 bytes, whatever the sampler wants
  float temperature;
  int top_k;
  float top_p, presence, frequency, repetition;
  unsigned seed[2];
};

struct LogitArgs {
  const void* logits;
  void* out;
  const LogitRecord* records;
  const unsigned short* counts;  // [R, >= V], null: no penalties
  const int* bias_ids;           // [R, K] vocabulary ids (null: no biases)
  const float* bias_values;
  const unsigned* allowed;       // [R, words], null: all allowed
  const int* rows;               // [B] row of the tables (null: b); outside 0 .. R - 1: the logits pass through
  int V, R, K, words, first;     // first: vocabulary id of column 0
  long long in_stride, out_stride, counts_stride;
  float fill;
};

constexpr int kLogitThreads = 256, kLogitVec = 8, kMaxBias = 1 << 16;

template <typename T> __device__ __forceinline__ float logit_to_f32(T v);
template <> __device__ __forceinline__ float logit_to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float logit_to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float logit_to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T logit_from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 logit_from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half logit_from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float logit_from_f32(float v) { return v; }

template <typename T>
struct alignas(16) LogitVec {
  T v[kLogitVec];
};
// A warp has kSets times 256 neighbouring columns, a thread eight of each 256: neighbours in 16-byte accesses (kVec: every row of every tensor starts on 16
// bytes), else eight that lie 32 apart, so that a warp's accesses are whole lines at any alignment.  Logits, counts, mask and the first ids of the biases
// are requested together, ahead of the record that says whether the row needs the counts.  A warp goes over the row's biases by itself, in their order
// (nothing waits for another warp): few are its own.  Where none of a thread's eight tokens has a count or a bias their bits stay as they are, and
// only the mask chooses; few of a warp's 256 are others, and a warp passes over the arithmetic of the places where it has none.  Logits of 16 bits are
// multiplied by the penalty's reciprocal, taken once: 2^-24 more of an error beside their own rounding of 2^-8 or 2^-11, for a division a value (1 x 32000: 2.4 us
// with, 2.0 without).
// 64 x 128256 bf16 with all three on a B200: 18.9 us with the arithmetic and a division for all values, 14.4 value by value behind block barriers that the
// gathering of the biases needed, 10.5 now (7.7 for its bytes at the rate of a copy; without any of the three 5.8, from L2).  Choosing registers by the number of a touched
// value, instead of passing over eight places, took 14.0.
template <typename T, bool kVec, int kSets>
__global__ void __launch_bounds__(kLogitThreads, kSets == 1 ? 5 : 4)
process_logits_kernel(const LogitArgs a) {
  constexpr int kMine = 256 * kSets, kAhead = 4;  // columns of a warp; ids of a lane that are requested together
  pdl_trigger();
  __shared__ float s_bias[kLogitThreads / 32][kMine];
  __shared__ unsigned s_biased[kLogitThreads / 32][kMine / 32];  // bit: whether the column has a bias
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lo = (blockIdx.x * (kLogitThreads / 32) + warp) * kMine;
  pdl_wait();
  if (lo >= a.V) return;
  const int r = a.rows ? a.rows[b] : b;
  const bool known = r >= 0 && r < a.R;
  const T* in = static_cast<const T*>(a.logits) + b * a.in_stride;
  T* out = static_cast<T*>(a.out) + b * a.out_stride;
  const auto column = [&](int s, int j) { return lo + s * 256 + (kVec ? lane * kLogitVec + j : lane + j * 32); };
  const bool inside = lo + kMine <= a.V;  // otherwise the row ends in this warp's columns
  const auto each = [&](int s, auto&& f) {
    if (inside) {
#pragma unroll
      for (int j = 0; j < kLogitVec; ++j) f(j);
    } else {
#pragma unroll
      for (int j = 0; j < kLogitVec; ++j)
        if (column(s, j) < a.V) f(j);
    }
  };
  const bool wide = kVec && inside;

  LogitVec<T> x[kSets];
  if (wide) {
#pragma unroll
    for (int s = 0; s < kSets; ++s) x[s] = *reinterpret_cast<const LogitVec<T>*>(in + column(s, 0));
  } else {
#pragma unroll
    for (int s = 0; s < kSets; ++s) each(s, [&](int j) { x[s].v[j] = in[column(s, j)]; });
  }
  const auto store = [&](int s) {
    if (wide) *reinterpret_cast<LogitVec<T>*>(out + column(s, 0)) = x[s];
    else each(s, [&](int j) { out[column(s, j)] = x[s].v[j]; });
  };
  if (!known) {
    if (in == out) return;
#pragma unroll
    for (int s = 0; s < kSets; ++s) store(s);
    return;
  }
  const int* ids = a.bias_ids + size_t(r) * a.K;  // (K is zero where there are none)
  const float* values = a.bias_values + size_t(r) * a.K;
  int id[kAhead];
#pragma unroll
  for (int q = 0; q < kAhead; ++q) id[q] = q * 32 + lane < a.K ? ids[q * 32 + lane] : -1;
  unsigned w[kSets][kLogitVec / 2] = {};  // eight words of counts
  const unsigned short* count_row = a.counts + r * a.counts_stride;
  if (!a.counts) {
  } else if (wide) {
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      const uint4 raw = *reinterpret_cast<const uint4*>(count_row + column(s, 0));
      w[s][0] = raw.x; w[s][1] = raw.y; w[s][2] = raw.z; w[s][3] = raw.w;
    }
  } else {
#pragma unroll
    for (int s = 0; s < kSets; ++s) each(s, [&](int j) { w[s][j >> 1] |= unsigned(count_row[column(s, j)]) << (16 * (j & 1)); });
  }
  unsigned allow[kSets];  // bit j: value j
  const unsigned* words = a.allowed + size_t(r) * a.words;
#pragma unroll
  for (int s = 0; s < kSets; ++s) allow[s] = 0xffu;
  if (!a.allowed) {
  } else if (wide && a.first % 8 == 0) {
#pragma unroll
    for (int s = 0; s < kSets; ++s) allow[s] = reinterpret_cast<const unsigned char*>(words)[(a.first + column(s, 0)) >> 3];
  } else {
#pragma unroll
    for (int s = 0; s < kSets; ++s)
      each(s, [&](int j) {
        const int of = a.first + column(s, j);
        if (!(words[of >> 5] >> (of & 31) & 1u)) allow[s] &= ~(1u << j);
      });
  }
  const float presence = a.records[r].presence, frequency = a.records[r].frequency, repetition = a.records[r].repetition;
  const bool penalties = presence != 0.f || frequency != 0.f || repetition != 1.f;
  const float inverse = 1.f / repetition;
  bool biases = false;  // whether a column of the warp has one
  for (int k = 0; k < a.K; k += kAhead * 32) {
    if (k > 0) {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) id[q] = k + q * 32 + lane < a.K ? ids[k + q * 32 + lane] : -1;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int n = id[q] - a.first - lo;
      const bool mine = id[q] >= 0 && n >= 0 && n < kMine;
      unsigned left = __ballot_sync(0xffffffffu, mine);
      if (!left) continue;
      const float value = mine ? values[k + q * 32 + lane] : 0.f;
      if (!biases) {
        for (int i = lane; i < kMine / 32; i += 32) s_biased[warp][i] = 0u;
        __syncwarp();
        biases = true;
      }
      for (; left; left &= left - 1) {  // in the order of the row
        const int from = __ffs(left) - 1;
        if (lane == from) {
          const unsigned had = s_biased[warp][n >> 5], bit = 1u << (n & 31);
          s_bias[warp][n] = (had & bit ? s_bias[warp][n] : 0.f) + value;
          s_biased[warp][n >> 5] = had | bit;
        }
        __syncwarp();
      }
    }
  }
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
    unsigned touched = 0, biased = 0;  // bit j: value j
    if (biases) {
      if (kVec) {
        biased = reinterpret_cast<const unsigned char*>(s_biased[warp])[s * 32 + lane];
      } else {
#pragma unroll
        for (int j = 0; j < kLogitVec; ++j) biased |= (s_biased[warp][s * 8 + j] >> lane & 1u) << j;
      }
    }
    if (penalties && (w[s][0] | w[s][1] | w[s][2] | w[s][3])) {
#pragma unroll
      for (int j = 0; j < kLogitVec / 2; ++j) touched |= (w[s][j] & 0xffffu ? 1u << 2 * j : 0u) | (w[s][j] >> 16 ? 2u << 2 * j : 0u);
    }
    if (touched | biased) {
#pragma unroll
      for (int j = 0; j < kLogitVec; ++j) {
        if (!((touched | biased) >> j & 1u)) continue;
        float l = logit_to_f32(x[s].v[j]);
        if (biased >> j & 1u) l += s_bias[warp][column(s, j) - lo];
        if (touched >> j & 1u) {
          const unsigned n = w[s][j >> 1] >> (16 * (j & 1)) & 0x7fffu;
          if constexpr (sizeof(T) == 4) l = l > 0.f ? l / repetition : l * repetition;
          else l *= l > 0.f ? inverse : repetition;
          if (n) l -= presence + frequency * float(n);
        }
        x[s].v[j] = logit_from_f32<T>(l);
      }
    }
    if (allow[s] != 0xffu) {
      const T fill = logit_from_f32<T>(a.fill);
#pragma unroll
      for (int j = 0; j < kLogitVec; ++j)
        if (!(allow[s] >> j & 1u)) x[s].v[j] = fill;
    }
    store(s);
  }
}

// counts[row][token] of every (row, token): its top bit is set (prompt) or its lower 15 go up by one and stay at their largest value.
// Pairs with a token or row outside the table are left out.
// A prompt's bit: read, and set by an atomic that nothing waits for unless it is there.
__global__ void __launch_bounds__(256)
mark_tokens_kernel(unsigned short* __restrict__ counts, long long stride, int R, int V, const int* __restrict__ tokens, const int* __restrict__ rows, int T) {
  pdl_trigger();
  pdl_wait();
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int token = i < T ? tokens[i] : -1, row = i < T ? rows[i] : -1;
  if (token < 0 || token >= V || row < 0 || row >= R) return;
  unsigned short* at = counts + row * stride + token;
  const uintptr_t p = reinterpret_cast<uintptr_t>(at);
  if (!(*reinterpret_cast<volatile unsigned short*>(at) & 0x8000u)) atomicOr(reinterpret_cast<unsigned*>(p & ~uintptr_t(3)), 0x8000u << (p & 2 ? 16 : 0));
}
// The pairs of a block are added up in shared memory first (open addressing; twice as many places as pairs, so that one is always free), and every
// different one goes to the table once.  The common tokens of a text then meet in a few blocks instead of in every warp, and where not even all of the
// call's tokens would bring a count past its largest value an addition that nothing waits for takes it there; a compare-and-swap does otherwise.
// 32000 tokens of 24 rows on a B200: 32 us with warps that swapped, 12 with blocks that swapped, 4.5 now; 30000 of one row 595, 37, 6.6; 900 of two 10 with either, 3.3.
// A call of more than 32767 tokens always swaps: 64000 of 24 rows 13 us, as by blocks that swapped before there were additions, 400000 of 200 rows 20 where those took 16.
// Blocks of 256 or 1024 pairs are within a tenth.
constexpr int kCountThreads = 512, kCountPlaces = 2 * kCountThreads;
__global__ void __launch_bounds__(kCountThreads)
count_tokens_kernel(unsigned short* __restrict__ counts, long long stride, int R, int V, const int* __restrict__ tokens, const int* __restrict__ rows, int T) {
  pdl_trigger();
  __shared__ unsigned long long s_key[kCountPlaces];  // row and token; all ones: free
  __shared__ unsigned s_times[kCountPlaces];
  for (int i = threadIdx.x; i < kCountPlaces; i += kCountThreads) { s_key[i] = ~0ull; s_times[i] = 0u; }
  __syncthreads();
  pdl_wait();
  const long long i = static_cast<long long>(blockIdx.x) * kCountThreads + threadIdx.x;
  const int token = i < T ? tokens[i] : -1, row = i < T ? rows[i] : -1;
  if (token >= 0 && token < V && row >= 0 && row < R) {
    const unsigned long long key = static_cast<unsigned long long>(row) << 32 | unsigned(token);
    unsigned place = (unsigned(token) * 2654435761u ^ unsigned(row) * 2246822519u) % kCountPlaces;  // odd multipliers spread neighbours
    for (;;) {
      const unsigned long long held = atomicCAS(&s_key[place], ~0ull, key);
      if (held == ~0ull || held == key) break;
      place = (place + 1) % kCountPlaces;
    }
    atomicAdd(&s_times[place], 1u);
  }
  __syncthreads();
  unsigned short* at[2];
  unsigned times[2], old[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int place = n * kCountThreads + threadIdx.x;
    times[n] = s_times[place];
    at[n] = counts + (s_key[place] >> 32) * stride + unsigned(s_key[place]);
    old[n] = times[n] ? *reinterpret_cast<volatile unsigned short*>(at[n]) : 0u;
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    if (!times[n]) continue;
    if ((old[n] & 0x7fffu) + unsigned(T) <= 0x7fffu) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(at[n]);
      atomicAdd(reinterpret_cast<unsigned*>(p & ~uintptr_t(3)), times[n] << (p & 2 ? 16 : 0));
      continue;
    }
    for (;;) {  // a failed exchange means that another one succeeded
      const unsigned now = (old[n] & 0x8000u) | min((old[n] & 0x7fffu) + times[n], 0x7fffu);
      if (now == old[n]) break;
      const unsigned seen = atomicCAS(at[n], static_cast<unsigned short>(old[n]), static_cast<unsigned short>(now));
      if (seen == old[n]) break;
      old[n] = seen;
    }
  }
}

// ----- plan of a ragged batch -----
// Request i has past_i tokens in the pages of table row rows_i and brings counts_i more.  With s_i the sum of the counts before it, token
// t of s_i <= t < s_{i+1} is at position past_i + t - s_i, in slot page * size + offset.  With a list of free pages, request i takes
// ceil((past_i + counts_i) / size) - ceil(past_i / size) of them, in the order of the requests, behind the pages of its past.
// Every block sums the lengths for itself (at most kPlanRequests, so that no block waits for another) and takes its share of tokens and table entries.
// Bound by latency: one request of 357 tokens takes 2.9 us of a replay on a B200, 256 requests of 4500 tokens with pages from a list 5.8.
constexpr int kPlanThreads = 256, kPlanRequests = 1024, kPlanPer = kPlanRequests / kPlanThreads, kPlanRows = 1 << 16;
enum : int { kPlanBadRequest = 1, kPlanNoRoom = 2, kPlanNoPages = 3 };

struct PlanArgs {
  int* table;  // [R, P]; written where pages are handed out
  const int *rows, *past, *counts, *pages;
  int *positions, *slots, *tok_seq, *q_starts, *seq_lens, *out_table, *info;
  int R, P, b, T, page_size, free_pages;  // free_pages < 0: none are handed out
};

__device__ __forceinline__ int pages_for(int tokens, int page_size) { return tokens / page_size + (tokens % page_size != 0); }  // a sum of the two may pass 31 bits

__global__ void __launch_bounds__(kPlanThreads)
plan_batch_kernel(const PlanArgs a) {
  pdl_trigger();
  __shared__ int s_start[kPlanRequests + 1], s_past[kPlanRequests], s_row[kPlanRequests], s_have[kPlanRequests], s_first[kPlanRequests];
  __shared__ long long s_sum[2][kPlanThreads / 32];
  __shared__ int s_bad;
  __shared__ unsigned s_seen[kPlanRows / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ps = a.page_size;
  if (tid == 0) s_bad = 0;
  const bool hand = a.free_pages >= 0;
  if (hand)
    for (int i = tid; i < (a.R + 31) / 32; i += kPlanThreads) s_seen[i] = 0u;
  __syncthreads();
  pdl_wait();
  // neighbouring requests per thread, so that one scan over the threads orders them
  long long tokens = 0, need = 0;
  int mine[kPlanPer], want[kPlanPer], bad = 0;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    const int i = tid * kPlanPer + k;
    mine[k] = want[k] = 0;
    if (i >= a.b) continue;
    const int row = a.rows[i], past = a.past[i], count = a.counts[i];
    const long long len = static_cast<long long>(past) + count;
    if (row < 0 || row >= a.R || past < 0 || count < 0) bad = max(bad, int(kPlanBadRequest));
    else if (len > static_cast<long long>(a.P) * ps) bad = max(bad, int(kPlanNoRoom));
    else {
      const int have = pages_for(past, ps);
      if (hand) {
        want[k] = int((len + ps - 1) / ps) - have;
        if (atomicOr(&s_seen[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u) bad = max(bad, int(kPlanBadRequest));  // two requests would take pages for one row
      }
      mine[k] = count;
      s_row[i] = row;
      s_past[i] = past;
      s_have[i] = have;
    }
    tokens += mine[k];
    need += want[k];
  }
  if (bad) atomicMax(&s_bad, bad);
  long long before_t = tokens, before_n = need;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, before_t, o), n = __shfl_up_sync(0xffffffffu, before_n, o);
    if (lane >= o) { before_t += t; before_n += n; }
  }
  if (lane == 31) { s_sum[0][warp] = before_t; s_sum[1][warp] = before_n; }
  __syncthreads();
  long long total = 0, taken = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) { before_t += s_sum[0][w]; before_n += s_sum[1][w]; }
    total += s_sum[0][w];
    taken += s_sum[1][w];
  }
  int refused = s_bad;
  if (!refused && total > a.T) refused = kPlanNoRoom;
  if (!refused && hand && taken > a.free_pages) refused = kPlanNoPages;
  if (blockIdx.x == 0 && tid == 0) {
    a.info[0] = refused ? -refused : int(total);
    a.info[1] = refused ? 0 : int(taken);
  }
  if (refused) total = 0;
  before_t -= tokens;
  before_n -= need;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    const int i = tid * kPlanPer + k;
    if (i < a.b) {
      s_start[i] = refused ? 0 : int(before_t);
      s_first[i] = refused ? 0 : int(before_n);
      if (blockIdx.x == 0) {
        a.q_starts[i] = s_start[i];
        a.seq_lens[i] = refused ? 0 : s_past[i] + mine[k];
      }
    }
    before_t += mine[k];
    before_n += want[k];
  }
  if (tid == 0) {
    s_start[a.b] = int(total);
    if (blockIdx.x == 0) a.q_starts[a.b] = int(total);
  }
  __syncthreads();
  const auto page_of = [&](int i, int j) {  // entry j of request i's row, its new pages included
    if (hand && j >= s_have[i]) return a.pages[s_first[i] + j - s_have[i]];
    return a.table[size_t(s_row[i]) * a.P + j];
  };
  const int step = gridDim.x * kPlanThreads;
  for (int t = blockIdx.x * kPlanThreads + tid; t < a.T; t += step) {
    int pos = 0, slot = -1, seq = -1;
    if (t < total) {
      int lo = 0, hi = a.b;  // the last request that starts at t or before
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= t) lo = mid; else hi = mid;
      }
      seq = lo;
      pos = s_past[lo] + t - s_start[lo];
      slot = page_of(lo, pos / ps) * ps + pos % ps;
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
    a.tok_seq[t] = seq;
  }
  const long long entries = static_cast<long long>(a.b) * a.P;
  for (long long e = static_cast<long long>(blockIdx.x) * kPlanThreads + tid; e < entries; e += step) {
    const int i = int(e / a.P), j = int(e - static_cast<long long>(i) * a.P);
    int page = 0;
    if (!refused && j < pages_for(s_past[i] + (s_start[i + 1] - s_start[i]), ps)) {
      page = page_of(i, j);
      if (hand && j >= s_have[i]) a.table[size_t(s_row[i]) * a.P + j] = page;
    }
    a.out_table[e] = page;
  }
}

template <typename T>
static int launch_logits(const LogitArgs& a, int B, bool vec, cudaStream_t stream) {
  constexpr int kColumns = kLogitThreads * kLogitVec, kMany = 2;
  // two sets for a thread, which then has twice as much under way, in exchange for fewer blocks (one set and two, us): 16 bits in wide accesses gain from six blocks an
  // SM on (16 x 128256 4.9 and 4.5, 64 x 128256 12.5 and 10.6, but 48 x 32000 4.5 and 4.9), others from some 24 on (64 x 128256 fp32 13.3 and 13.1, 40 x 128256 9.0
  // and 9.4); four spill
  const bool many = static_cast<long long>(B) * ((a.V + kColumns - 1) / kColumns) >= 148 * (vec && sizeof(T) == 2 ? 6 : 24);
  const int columns = many ? kColumns * kMany : kColumns;
  const dim3 grid((a.V + columns - 1) / columns, B);
  if (many) launch_kernel(vec ? process_logits_kernel<T, true, kMany> : process_logits_kernel<T, false, kMany>, grid, dim3(kLogitThreads), 0, stream, a);
  else launch_kernel(vec ? process_logits_kernel<T, true, 1> : process_logits_kernel<T, false, 1>, grid, dim3(kLogitThreads), 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}

}  // namespace mfq

// dtype: 0 bf16, 1 fp16, 2 fp32.  Strides count values.  What may be null, and what the tables hold: see LogitArgs.
extern "C" int mfq_process_logits(const void* logits, void* out, int dtype, int B, int V, long long in_stride, long long out_stride, const void* records, int R,
                                  const void* counts, long long counts_stride, const int* bias_ids, const float* bias_values, int K, const void* allowed,
                                  int words, const int* rows, int first, float fill, cudaStream_t stream) {
  using namespace mfq;
  if (B <= 0 || B > 65535 || V <= 0 || R <= 0 || first < 0 || K < 0 || K > kMaxBias || dtype < 0 || dtype > 2) return -1;
  if (V > 1 << 30 || first > INT32_MAX - V || (allowed && (static_cast<long long>(first) + V + 31) / 32 > words)) return -1;
  const LogitArgs a{logits, out, static_cast<const LogitRecord*>(records), static_cast<const unsigned short*>(counts), bias_ids, bias_values,
                    static_cast<const unsigned*>(allowed), rows, V, R, K, words, first, in_stride, out_stride, counts_stride, fill};
  const int size = dtype == 2 ? 4 : 2;
  const auto even = [](const void* p, long long stride, int bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * bytes % 16 == 0; };
  const bool vec = even(logits, in_stride, size) && even(out, out_stride, size) && (!counts || even(counts, counts_stride, 2));
  return dtype == 0 ? launch_logits<__nv_bfloat16>(a, B, vec, stream) : dtype == 1 ? launch_logits<__half>(a, B, vec, stream) : launch_logits<float>(a, B, vec, stream);
}

extern "C" int mfq_count_tokens(void* counts, long long stride, int R, int V, const int* tokens, const int* rows, int T, int prompt, cudaStream_t stream) {
  if (R <= 0 || V <= 0 || T < 0) return -1;
  if (T == 0) return 0;
  if (prompt)
    mfq::launch_kernel(mfq::mark_tokens_kernel, dim3((T - 1) / 256 + 1), dim3(256), 0, stream, static_cast<unsigned short*>(counts), stride, R, V, tokens, rows, T);
  else
    mfq::launch_kernel(mfq::count_tokens_kernel, dim3((T - 1) / mfq::kCountThreads + 1), dim3(mfq::kCountThreads), 0, stream, static_cast<unsigned short*>(counts),
                       stride, R, V, tokens, rows, T);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}

// table [R, P] int32; rows / past / counts [b]; pages [free_pages], or free_pages < 0; positions / slots / tok_seq [T], q_starts [b + 1], seq_lens [b], out_table [b, P],
// info [2]: tokens and pages taken, or minus the reason of a refusal and 0.
extern "C" int mfq_plan_batch(int* table, int R, int P, const int* rows, const int* past, const int* counts, int b, const int* pages, int free_pages, int* positions,
                              int* slots, int* tok_seq, int T, int* q_starts, int* seq_lens, int* out_table, int* info, int page_size, cudaStream_t stream) {
  using namespace mfq;
  if (R <= 0 || P <= 0 || b <= 0 || b > kPlanRequests || T < 0 || T > 1 << 30 || page_size <= 0 || (free_pages >= 0 && R > kPlanRows)) return -1;
  if (static_cast<long long>(P) * page_size > INT32_MAX) return -1;
  const PlanArgs a{table, rows, past, counts, pages, positions, slots, tok_seq, q_starts, seq_lens, out_table, info, R, P, b, T, page_size, free_pages};
  const long long work = T + static_cast<long long>(b) * P, per = 4 * kPlanThreads;
  const int blocks = int(work / per < 1 ? 1 : work / per > 148 ? 148 : (work + per - 1) / per);
  launch_kernel(plan_batch_kernel, dim3(blocks), dim3(kPlanThreads), 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -7;
}
