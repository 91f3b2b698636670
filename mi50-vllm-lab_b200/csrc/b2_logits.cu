// Logit processors between the lm_head and the sampler: penalties for repeated tokens, biases and
// grammar masks, in one pass over the logits.
//
// For row r and token v (global id vocab_start + column), with the row's history
// tokens[row_seq[r], 0 .. total_lens[r]) of which the first prompt_lens[r] are the prompt, and
// n = occurrences of v behind the prompt, seen = v occurs anywhere in the history:
//   x = float(logit)
//   seen:   x = x > 0 ? x / repetition : x * repetition
//   n > 0:  x = x - frequency * n - presence
//   x += sum of the row's biases for v
//   mask bit of v clear: x = -inf
//
// A thread-block cluster of 8 CTAs owns a row (or an equal part of its vocabulary): every CTA
// keeps one 32-bit word per token of its slice in shared memory. The CTAs read an eighth of the
// history each and post every token to the word of its owner through distributed shared memory
// (integer atomics: the order does not matter), so that the history crosses L2 once per cluster
// however long it is. Then each CTA takes its slice of logits through the words. The logits, the
// mask and the first tokens of the history are loaded into registers before all this, so that one
// latency covers them.
//   word = [31] in the prompt | [30:20] key of the token's first bias entry | [19:0] n
// The first of the bias entries for a token wins its word by an atomic maximum of keys that fall
// with the index; its thread adds the others, if there are any, in list order in fp64. The result
// does not depend on timing.
//
// Vectors: with columns counted from the last multiple of 8 elements at or before the row's start
// (`shift` columns before it), vectors of 8 are aligned in the logits and in the output alike, for
// any vocabulary size, as long as the rows of both start at the same place modulo 8.
//
// Bound: memory (logits once, fp32 out once); for few rows the latency of history -> words ->
// stream.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "b2_device.cuh"
#include "b2_internal.h"

namespace b2 {
namespace {

constexpr int kCluster = 8;
constexpr int kThreads = 512;
constexpr int kVec = 8;                                // tokens per thread and step
constexpr int kSteps = 5;                              // steps of a slice
constexpr int kMaxSlice = kThreads * kVec * kSteps;    // words of shared memory per CTA
constexpr int kAhead = 4;                              // tokens of the history loaded at a time
constexpr int kMaxBias = 2047;                         // 11 bits of the word
constexpr int kMaxHistory = (1 << 20) - 1;             // 20 bits
constexpr uint32_t kPromptBit = 0x80000000u;

struct LogitArgs {
  const void* logits;
  float* out;
  int64_t row_stride;
  const void* tokens;
  int64_t tokens_stride;
  const int32_t *row_seq, *prompt_lens, *total_lens;
  const float *repetition, *frequency, *presence;
  const int32_t* bias_ids;
  const float* bias_values;
  const uint32_t* mask;
  int64_t mask_stride;
  int mask_words;
  int vocab, vocab_start, seqs, max_tokens, n_bias;
  int tokens64;
  int slice;     // columns per CTA, a multiple of kVec
  int clusters;  // clusters per row
  FastDiv by_slice;
};

__device__ __forceinline__ void red_or_cluster(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void red_add_cluster(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ float lo_f(float v) { return v; }
__device__ __forceinline__ float lo_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float lo_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// kVec mask bits from bit position `bit` on (those before and behind the row read as zero).
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* row, int words, int bit) {
  const int w = bit >> 5, sh = bit & 31;  // bit may be negative: floor, remainder
  const uint32_t lo = w >= 0 && w < words ? row[w] : 0u;
  const uint32_t hi = (sh > 32 - kVec && w + 1 >= 0 && w + 1 < words) ? row[w + 1] : 0u;
  return __funnelshift_r(lo, hi, sh);
}

struct RowParams {
  float rep, freq, pres;
};

__device__ __forceinline__ float process(float x, uint32_t word, const RowParams& rp,
                                         const float* bias_sums) {
  if (word != 0) {
    const uint32_t n = word & (uint32_t)kMaxHistory;
    const uint32_t bias = (word >> 20) & 2047u;
    if (n != 0 || (word & kPromptBit)) {
      x = x > 0.f ? __fdiv_rn(x, rp.rep) : x * rp.rep;
      if (n != 0) x = __fsub_rn(__fsub_rn(x, __fmul_rn(rp.freq, (float)n)), rp.pres);
    }
    if (bias != 0) x += bias_sums[bias - 1];
  }
  return x;
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// kVector: vectors of 8 columns (see above); otherwise element by element, for any strides.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kThreads) logits_kernel(const LogitArgs p) {
  extern __shared__ __align__(16) uint32_t words[];
  const int rank = (int)cluster_ctarank();
  const int cluster = blockIdx.x / kCluster;
  const int row = cluster / p.clusters, part = cluster - row * p.clusters;
  // columns with the shift: the row's are shift .. shift + vocab - 1
  const int shift = kVector ? (int)((int64_t)row * p.vocab & 7) : 0;
  const int first = part * kCluster * p.slice, lo = first + rank * p.slice;  // of the cluster, the CTA
  const int from = max(0, shift - lo), to = min(p.slice, p.vocab + shift - lo);  // of the slice
  float* bias_sums = reinterpret_cast<float*>(words + p.slice);
  int32_t* bias_ids = reinterpret_cast<int32_t*>(bias_sums + p.n_bias);
  const bool history = p.tokens != nullptr;
  const bool use_words = history || p.n_bias > 0;

  if (use_words) {
    for (int i = threadIdx.x * 4; i < p.slice; i += kThreads * 4)
      *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
  }
  grid_dep_wait();
  grid_dep_launch();

  // ---- loads ahead: the slice's logits and mask, the first tokens
  const T* in = static_cast<const T*>(p.logits) + (int64_t)row * p.row_stride + lo - shift;
  float* out = p.out + (int64_t)row * p.vocab + lo - shift;
  const uint32_t* mask = p.mask ? p.mask + (int64_t)row * p.mask_stride : nullptr;
  const int bit0 = p.vocab_start + lo - shift;
  constexpr int kLoads = kVec * sizeof(T) / 16;
  uint4 raw[kVector ? kSteps : 1][kLoads];
  uint32_t bits[kVector ? kSteps : 1];
  if constexpr (kVector) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int i = (s * kThreads + threadIdx.x) * kVec;
      if (i >= from && i + kVec <= to) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) raw[s][j] = reinterpret_cast<const uint4*>(in + i)[j];
      } else {
        T e[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) e[j] = i + j >= from && i + j < to ? in[i + j] : T(0.f);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) raw[s][j] = reinterpret_cast<const uint4*>(e)[j];
      }
      bits[s] = mask && i < to ? mask_bits(mask, p.mask_words, bit0 + i) : ~0u;
    }
  }
  int total = 0, prompt = 0;
  int64_t at = 0;
  if (history) {
    const int seq = p.row_seq ? p.row_seq[row] : row;
    if (seq >= 0 && seq < p.seqs) {
      total = min(max(p.total_lens[row], 0), p.max_tokens);
      prompt = p.prompt_lens[row];
      at = (int64_t)seq * p.tokens_stride;
    }
  }
  int32_t ids[kAhead];  // columns of the cluster, or -1
  auto fetch = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kCluster * kThreads;
      int64_t id = -1;
      if (i < total)
        id = p.tokens64 ? static_cast<const int64_t*>(p.tokens)[at + i]
                        : (int64_t)static_cast<const int32_t*>(p.tokens)[at + i];
      const int64_t col = id - p.vocab_start;
      ids[k] = col >= 0 && col < p.vocab ? (int32_t)col + shift - first : -1;
    }
  };
  const int mine = rank * kThreads + threadIdx.x;
  if (history) fetch(mine);
  RowParams rp = {1.f, 0.f, 0.f};
  if (p.repetition) rp.rep = p.repetition[row];
  if (p.frequency) rp.freq = p.frequency[row];
  if (p.presence) rp.pres = p.presence[row];

  // ---- biases: keys into the words, sums by key
  if (p.n_bias > 0) {
    const int64_t list = (int64_t)row * p.n_bias;
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads) {
      const int id = p.bias_ids[list + e];
      const int64_t col = id < 0 ? -1 : (int64_t)id - p.vocab_start + shift - lo;
      bias_ids[e] = col >= from && col < to ? (int)col : -1;
      bias_sums[p.n_bias - 1 - e] = p.bias_values[list + e];  // by key - 1
    }
    __syncthreads();  // the words are zero, the list is here
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads)
      if (bias_ids[e] >= 0) atomicMax(&words[bias_ids[e]], (uint32_t)(p.n_bias - e) << 20);
    __syncthreads();
    // an entry that is not its token's first leaves a mark at the one that is
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads) {
      const uint32_t entry = (uint32_t)bias_ids[e];  // perhaps marked already
      if (entry == 0xffffffffu) continue;
      const int one = p.n_bias - (int)(words[entry & 0x3fffffffu] >> 20);
      if (one != e) atomicOr(reinterpret_cast<uint32_t*>(&bias_ids[one]), 0x40000000u);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads) {
      const uint32_t entry = (uint32_t)bias_ids[e];
      if (entry == 0xffffffffu || !(entry & 0x40000000u)) continue;
      const int col = (int)(entry & 0x3fffffffu);
      double sum = 0.0;
      for (int j = e; j < p.n_bias; ++j)
        if (((uint32_t)bias_ids[j] & 0xbfffffffu) == (uint32_t)col) sum += (double)p.bias_values[list + j];
      bias_sums[p.n_bias - 1 - e] = (float)sum;
    }
  }

  // ---- history
  if (history) {
    __syncwarp();
    cluster_arrive();  // this CTA's words are ready
    cluster_wait();
    const uint32_t base = smem_u32(words);
    for (int i = mine; i < total; i += kAhead * kCluster * kThreads) {
      if (i != mine) fetch(i);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (ids[k] < 0) continue;
        const int owner = p.by_slice.div(ids[k]);
        if (owner >= kCluster) continue;
        const uint32_t addr = mapa_shared(base + 4u * (uint32_t)(ids[k] - owner * p.slice), (uint32_t)owner);
        if (i + k * kCluster * kThreads < prompt)
          red_or_cluster(addr, kPromptBit);
        else
          red_add_cluster(addr, 1u);
      }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();  // every post has landed
  } else if (use_words) {
    __syncthreads();
  }

  // ---- the slice
  const float ninf = __int_as_float(0xff800000);
  if constexpr (kVector) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int i = (s * kThreads + threadIdx.x) * kVec;
      if (i >= to) break;
      const T* e = reinterpret_cast<const T*>(raw[s]);
      float x[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[j] = lo_f(e[j]);
      if (use_words) {
        const uint4 w0 = *reinterpret_cast<const uint4*>(words + i);
        const uint4 w1 = *reinterpret_cast<const uint4*>(words + i + 4);
        const uint32_t w[kVec] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
        if (((w0.x | w0.y) | (w0.z | w0.w)) | ((w1.x | w1.y) | (w1.z | w1.w))) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) x[j] = process(x[j], w[j], rp, bias_sums);
        }
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[j] = (bits[s] >> j) & 1u ? x[j] : ninf;
      if (i >= from && i + kVec <= to) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + i), "f"(x[0]),
                     "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                     : "memory");
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (i + j >= from && i + j < to) out[i + j] = x[j];
      }
    }
  } else {
    // a step covers kVec * kThreads consecutive tokens, kThreads apart in a thread
    for (int i0 = threadIdx.x; i0 < to; i0 += kThreads * kVec) {
      float x[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int i = i0 + j * kThreads;
        x[j] = i < to ? lo_f(in[i]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int i = i0 + j * kThreads;
        if (i >= to) continue;
        if (use_words) x[j] = process(x[j], words[i], rp, bias_sums);
        if (mask && !(mask_bits(mask, p.mask_words, bit0 + i) & 1u)) x[j] = ninf;
        out[i] = x[j];
      }
    }
  }
}

template <typename T, bool kVector>
int launch_typed(LogitArgs& p, int rows, cudaStream_t stream) {
  DeviceInfo di;
  int rc = device_info(&di);
  if (rc) return rc;
  // Enough clusters per row to give every SM work, as long as a CTA keeps a whole step.
  const int columns = p.vocab + kVec - 1;  // with the shift
  const int steps = (columns + kCluster * kThreads * kVec - 1) / (kCluster * kThreads * kVec);
  const int need = (columns + kCluster * kMaxSlice - 1) / (kCluster * kMaxSlice);
  const int64_t ctas = (int64_t)rows * kCluster;
  const int fill = (int)((di.sm_count + ctas - 1) / ctas);
  p.clusters = std::max(need, std::min(fill, steps));
  const int slice = (columns + p.clusters * kCluster - 1) / (p.clusters * kCluster);
  p.slice = (slice + kVec - 1) / kVec * kVec;
  p.by_slice = make_div(p.slice);
  const int64_t grid = (int64_t)rows * p.clusters * kCluster;
  if (grid > 0x7fffffff)
    return fail(B2_ERR_INVALID_ARG, "logits_process: %d rows of %d logits are too many", rows, p.vocab);
  const size_t smem = sizeof(uint32_t) * ((size_t)p.slice + 2 * (size_t)p.n_bias);
  static bool configured[64] = {};
  int dev = 0;
  B2_CUDA_TRY(cudaGetDevice(&dev));
  if (!configured[dev]) {
    B2_CUDA_TRY(cudaFuncSetAttribute(logits_kernel<T, kVector>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)(sizeof(uint32_t) * (kMaxSlice + 2 * kMaxBias))));
    configured[dev] = true;
  }
  return launch_kernel_clusters(logits_kernel<T, kVector>, (int)grid, kCluster, kThreads, smem,
                                stream, /*early=*/true, p);
}

}  // namespace
}  // namespace b2

extern "C" int b2_logits_process(const void* logits, int64_t row_stride, int dtype, float* out,
                                 int rows, int vocab, int vocab_start, const void* tokens,
                                 int tokens_64, int64_t tokens_stride, int n_seqs, int max_tokens,
                                 const int32_t* row_seq, const int32_t* prompt_lens,
                                 const int32_t* total_lens, const float* repetition,
                                 const float* frequency, const float* presence,
                                 const int32_t* bias_ids, const float* bias_values, int n_bias,
                                 const uint32_t* mask, int64_t mask_stride, int mask_words,
                                 void* stream) {
  using namespace b2;
  const char* op = "logits_process";
  if (rows < 0 || vocab < 1) return fail(B2_ERR_INVALID_ARG, "%s: %d rows of %d logits", op, rows, vocab);
  if (vocab_start < 0 || (int64_t)vocab_start + vocab > 0x7fffffff - 64)
    return fail(B2_ERR_INVALID_ARG, "%s: vocab_start=%d", op, vocab_start);
  if (dtype != B2_DTYPE_F16 && dtype != B2_DTYPE_BF16 && dtype != B2_DTYPE_F32)
    return fail(B2_ERR_INVALID_ARG, "%s: dtype %d", op, dtype);
  if (tokens) {
    if (!prompt_lens || !total_lens)
      return fail(B2_ERR_INVALID_ARG, "%s: a history needs prompt_lens and total_lens", op);
    if (n_seqs < 0 || max_tokens < 0 || max_tokens > kMaxHistory)
      return fail(B2_ERR_INVALID_ARG, "%s: histories of %d tokens (at most %d)", op, max_tokens,
                  kMaxHistory);
    if (!row_seq && n_seqs < rows)
      return fail(B2_ERR_INVALID_ARG, "%s: %d histories for %d rows and no row_seq", op, n_seqs, rows);
  } else if ((repetition || frequency || presence) && (max_tokens != 0 || !total_lens)) {
    return fail(B2_ERR_INVALID_ARG, "%s: penalties need a history", op);
  }
  if (n_bias < 0 || n_bias > kMaxBias)
    return fail(B2_ERR_INVALID_ARG, "%s: %d biases per row (at most %d)", op, n_bias, kMaxBias);
  if (n_bias > 0 && (!bias_ids || !bias_values))
    return fail(B2_ERR_INVALID_ARG, "%s: null bias pointer", op);
  if (mask && (int64_t)mask_words * 32 < (int64_t)vocab_start + vocab)
    return fail(B2_ERR_INVALID_ARG, "%s: mask of %d words for tokens up to %d", op, mask_words,
                vocab_start + vocab);
  if (rows == 0) return B2_OK;
  if (!logits || !out) return fail(B2_ERR_INVALID_ARG, "%s: null pointer", op);
  LogitArgs p = {};
  p.logits = logits, p.out = out, p.row_stride = row_stride;
  const bool penalties = repetition || frequency || presence;
  p.tokens = penalties && max_tokens > 0 ? tokens : nullptr;
  p.tokens64 = tokens_64, p.tokens_stride = tokens_stride, p.seqs = n_seqs, p.max_tokens = max_tokens;
  p.row_seq = row_seq, p.prompt_lens = prompt_lens, p.total_lens = total_lens;
  p.repetition = repetition, p.frequency = frequency, p.presence = presence;
  p.bias_ids = bias_ids, p.bias_values = bias_values, p.n_bias = n_bias;
  p.mask = mask, p.mask_stride = mask_stride, p.mask_words = mask_words;
  p.vocab = vocab, p.vocab_start = vocab_start;
  const bool vector = (reinterpret_cast<uintptr_t>(logits) & 15u) == 0 &&
                      (reinterpret_cast<uintptr_t>(out) & 31u) == 0 && (row_stride - vocab) % kVec == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B2_DTYPE_F16)
    return vector ? launch_typed<__half, true>(p, rows, s) : launch_typed<__half, false>(p, rows, s);
  if (dtype == B2_DTYPE_BF16)
    return vector ? launch_typed<__nv_bfloat16, true>(p, rows, s)
                  : launch_typed<__nv_bfloat16, false>(p, rows, s);
  return vector ? launch_typed<float, true>(p, rows, s) : launch_typed<float, false>(p, rows, s);
}
