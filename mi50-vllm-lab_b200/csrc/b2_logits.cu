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
// however long it is. Then each CTA streams its slice of logits through the words.
//   word = [31] in the prompt | [30:20] 1 + index of the token's first bias entry | [19:0] n
// Several bias entries for one token are added in list order in fp64 by the thread that holds the
// first of them; the result does not depend on timing.
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
constexpr int kVec = 8;                     // tokens per thread and step
constexpr int kMaxSlice = 40960;            // words of shared memory per CTA
constexpr int kMaxBias = 2047;              // 11 bits of the word
constexpr int kMaxHistory = (1 << 20) - 1;  // 20 bits
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
  int slice;     // tokens per CTA, a multiple of kVec
  int clusters;  // clusters per row
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

// 32 mask bits from bit position `bit` on (the words behind the row's end read as zero).
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* row, int words, int bit) {
  const int w = bit >> 5, sh = bit & 31;
  const uint32_t lo = w < words ? row[w] : 0u;
  const uint32_t hi = (sh && w + 1 < words) ? row[w + 1] : 0u;
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

// kVector: rows of logits and of the output are 16-byte aligned.
template <typename T, bool kVector>
__global__ void __launch_bounds__(kThreads) logits_kernel(const LogitArgs p) {
  extern __shared__ __align__(16) uint32_t words[];
  const int rank = (int)cluster_ctarank();
  const int cluster = blockIdx.x / kCluster;
  const int row = cluster / p.clusters, part = cluster - row * p.clusters;
  const int lo = (part * kCluster + rank) * p.slice;  // first column of this CTA
  const int n = max(0, min(p.slice, p.vocab - lo));
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

  RowParams rp = {1.f, 0.f, 0.f};
  if (p.repetition) rp.rep = p.repetition[row];
  if (p.frequency) rp.freq = p.frequency[row];
  if (p.presence) rp.pres = p.presence[row];

  if (history) {
    const int seq = p.row_seq ? p.row_seq[row] : row;
    int total = 0, prompt = 0;
    if (seq >= 0 && seq < p.seqs) {
      total = min(max(p.total_lens[row], 0), p.max_tokens);
      prompt = p.prompt_lens[row];
    }
    __syncwarp();
    cluster_sync_all();  // every CTA's words are zero
    const uint32_t base = smem_u32(words);
    const int first = part * kCluster * p.slice;  // first column of the cluster
    const int64_t at = (int64_t)seq * p.tokens_stride;
    for (int i = rank * kThreads + threadIdx.x; i < total; i += kCluster * kThreads) {
      const int64_t id = p.tokens64 ? static_cast<const int64_t*>(p.tokens)[at + i]
                                    : (int64_t)static_cast<const int32_t*>(p.tokens)[at + i];
      const int64_t col = id - p.vocab_start;
      if (col < first || col >= p.vocab) continue;
      const int off = (int)(col - first), owner = off / p.slice;
      if (owner >= kCluster) continue;
      const uint32_t addr = mapa_shared(base + 4u * (uint32_t)(off - owner * p.slice), (uint32_t)owner);
      if (i < prompt)
        red_or_cluster(addr, kPromptBit);
      else
        red_add_cluster(addr, 1u);
    }
    __syncwarp();
    cluster_sync_all();  // every post has landed
  } else if (use_words) {
    __syncthreads();
  }

  if (p.n_bias > 0) {
    const int64_t at = (int64_t)row * p.n_bias;
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads) bias_ids[e] = p.bias_ids[at + e];
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads) {
      const int id = bias_ids[e];
      const int64_t col = (int64_t)id - p.vocab_start - lo;
      if (id < 0 || col < 0 || col >= n) continue;
      bool is_first = true;
      for (int j = 0; j < e && is_first; ++j) is_first = bias_ids[j] != id;
      if (!is_first) continue;
      double sum = 0.0;
      for (int j = e; j < p.n_bias; ++j)
        if (bias_ids[j] == id) sum += (double)p.bias_values[at + j];
      bias_sums[e] = (float)sum;
      words[col] |= (uint32_t)(e + 1) << 20;  // one thread per token
    }
    __syncthreads();
  }

  const T* in = static_cast<const T*>(p.logits) + (int64_t)row * p.row_stride + lo;
  float* out = p.out + (int64_t)row * p.vocab + lo;
  const uint32_t* mask = p.mask ? p.mask + (int64_t)row * p.mask_stride : nullptr;
  const float ninf = __int_as_float(0xff800000);
  if constexpr (kVector) {
    for (int i = threadIdx.x * kVec; i < n; i += kThreads * kVec) {
      float x[kVec];
      if (i + kVec <= n) {
        constexpr int kLoads = kVec * sizeof(T) / 16;
        uint4 raw[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) raw[j] = reinterpret_cast<const uint4*>(in + i)[j];
        const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] = lo_f(e[j]);
      } else {
        for (int j = 0; j < kVec; ++j) x[j] = i + j < n ? lo_f(in[i + j]) : 0.f;
      }
      if (use_words) {
        const uint4 w0 = *reinterpret_cast<const uint4*>(words + i);
        const uint4 w1 = *reinterpret_cast<const uint4*>(words + i + 4);
        const uint32_t w[kVec] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] = process(x[j], w[j], rp, bias_sums);
      }
      if (mask) {
        const uint32_t bits = mask_bits(mask, p.mask_words, p.vocab_start + lo + i);
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] = (bits >> j) & 1u ? x[j] : ninf;
      }
      if (i + kVec <= n) {
        reinterpret_cast<float4*>(out + i)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(out + i)[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        for (int j = 0; j < kVec && i + j < n; ++j) out[i + j] = x[j];
      }
    }
  } else {
    // any stride: a step covers kVec * kThreads consecutive tokens, kThreads apart in a thread
    for (int i0 = threadIdx.x; i0 < n; i0 += kThreads * kVec) {
      float x[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int i = i0 + j * kThreads;
        x[j] = i < n ? lo_f(in[i]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int i = i0 + j * kThreads;
        if (i >= n) continue;
        if (use_words) x[j] = process(x[j], words[i], rp, bias_sums);
        if (mask && !(mask_bits(mask, p.mask_words, p.vocab_start + lo + i) & 1u)) x[j] = ninf;
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
  const int steps = (p.vocab + kCluster * kThreads * kVec - 1) / (kCluster * kThreads * kVec);
  int need = (p.vocab + kCluster * kMaxSlice - 1) / (kCluster * kMaxSlice);
  const int fill = (di.sm_count + rows * kCluster - 1) / (rows * kCluster);
  p.clusters = std::max(need, std::min(fill, steps));
  int slice = (p.vocab + p.clusters * kCluster - 1) / (p.clusters * kCluster);
  p.slice = (slice + kVec - 1) / kVec * kVec;
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
  const size_t es = dtype == B2_DTYPE_F32 ? 4 : 2;
  const bool vector = aligned16(logits) && aligned16(out) && row_stride * es % 16 == 0 && vocab % 4 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B2_DTYPE_F16)
    return vector ? launch_typed<__half, true>(p, rows, s) : launch_typed<__half, false>(p, rows, s);
  if (dtype == B2_DTYPE_BF16)
    return vector ? launch_typed<__nv_bfloat16, true>(p, rows, s)
                  : launch_typed<__nv_bfloat16, false>(p, rows, s);
  return vector ? launch_typed<float, true>(p, rows, s) : launch_typed<float, false>(p, rows, s);
}
