// Logit processors between the lm_head and the sampler: penalties for repeated tokens, biases and
// grammar masks, in one pass over the logits.
//
// For row r and token v (global id vocab_start + column), with the row's history
// tokens[row_seq[r], 0 .. total_lens[r]) of which the first prompt_lens[r] are the prompt, and
// n = occurrences of v behind the prompt, seen = v occurs anywhere in the history:
//   x = float(logit)
//   seen:   x = x > 0 ? x / repetition : x * repetition
//   n > 0:  x = x - frequency * n - presence
//   x += sum of the row's biases for v       (before the penalties where the caller asks for it)
//   mask bit of v clear: x = -inf
//
// A CTA owns a slice of a row's vocabulary and keeps one 32-bit word per token of it in shared
// memory. It reads the row's whole history (from L2, which the CTAs of the row share) and counts the
// tokens of its slice in its own memory; then the slice of logits, loaded into registers ahead of
// everything else, goes through the words and the mask to the output. The other splits measured, on
// 128 rows of 151936 logits with histories of up to 16384 tokens (this one then: 57 us, now 44): a cluster whose
// CTAs read a part of the history each and post the counts to one another's memory, 84 us (the posts
// of a token that a text repeats queue at one CTA); the words applied behind the stream, by a second
// look at the history 85 us, by a list of the touched columns 64 us; a launch of its own for the
// touched columns, 65 us and twice the latency for few rows.
//   word = [31] in the prompt | [30:20] key of the token's first bias entry | [19:0] n
// The first of the bias entries for a token wins its word by an atomic maximum of keys that fall
// with the index; a warp adds the other entries to it, if there are any, in a fixed order in fp64. The
// result does not depend on timing.
//
// Vectors: with columns counted from the last multiple of 8 elements at or before the row's start
// (`shift` columns before it), vectors of 8 are aligned in the logits and in the output alike, for
// any vocabulary size, as long as the rows of both start at the same place modulo 8.
//
// Bound: memory where histories are short (logits once, fp32 out once): 128 rows of 151936 fp16
// logits alone take 19.1 us, 6.1 TB/s; with biases and masks 25 us; with histories of 300 tokens as
// well 30 us. Long histories add their read out of L2 by each of a row's eight CTAs (10300 tokens per
// row on average: 13 us of instructions and latency; with a load per token 21 us), the atomics in
// shared memory and the touched tokens' arithmetic, in all 44 us (49 with all eight tokens of a vector
// going through it where one is touched). Few rows are bound by the latency of lengths -> history ->
// words -> stream: one row 2.6 us; 8 rows of 151936 logits with 300 biases each 6.2 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "b2_device.cuh"
#include "b2_internal.h"

namespace b2 {
namespace {

constexpr int kMostThreads = 512;
constexpr int kVec = 8;                                // tokens per thread and step
// Steps of a slice, chosen for 16-bit logits: five at two CTAs per SM (64 registers) keep 128 rows'
// stream at 19.1 us; four at three CTAs spill at 40 registers, 23.7 us. With fp32 logits, twice the
// registers for a step, five spill: 128 rows of 151936 with one token of history 35.8 us of 23.8 that
// their bytes take, with long histories, biases and mask 63. Smaller CTAs read the history more often: 256 threads
// took 73 us for the long histories where 512 took 56.
constexpr int kSteps = 5;
constexpr int kMaxSlice = kMostThreads * kVec * kSteps;    // words of shared memory per CTA
constexpr int kAhead = 8;                              // tokens of the history a thread loads at a time
constexpr int kMaxBias = 2047;                         // 11 bits of the word
constexpr int kMaxHistory = (1 << 20) - 1;             // 20 bits
constexpr int kMaxVocab = 1 << 30;                     // columns, with the rounding to slices, in 31 bits
constexpr uint32_t kPromptBit = 0x80000000u;
constexpr uint32_t kMark = 0x40000000u;

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
  int tokens64, tokens_by4;
  int slice;   // columns per CTA, a multiple of kVec
  int slices;  // CTAs per row
};

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

// A row's penalties. The division by `rep` is a product with its reciprocal and one correction by
// the residual (Markstein, IBM J. Res. Dev. 34, 1990), which gives the rounded quotient in a few
// instructions without a branch (for |x| of 2^-102 and more, where the residual is exact): a warp works
// on 32 tokens of which some are divided and others multiplied. Where the residual is no number (infinite x) the product stands. `plain`: the row's
// `rep` is too small or too large for that, or 0 or infinite, and the row divides.
struct RowParams {
  float rep, inv, freq, pres;
  bool plain;
};

__device__ __forceinline__ RowParams row_params(const LogitArgs& p, int row) {
  RowParams r = {1.f, 1.f, 0.f, 0.f, false};
  if (p.repetition) r.rep = p.repetition[row];
  if (p.frequency) r.freq = p.frequency[row];
  if (p.presence) r.pres = p.presence[row];
  return r;  // inv and plain are the caller's, once rep is here
}

template <bool kBiasFirst>
__device__ __forceinline__ float process(float x, uint32_t word, const RowParams& rp,
                                         const float* bias_sums) {
  const uint32_t n = word & (uint32_t)kMaxHistory, bias = (word >> 20) & 2047u;
  if (kBiasFirst && bias != 0) x += bias_sums[bias - 1];
  const float q = __fmul_rn(x, rp.inv), residual = __fmaf_rn(-q, rp.rep, x);
  float quotient = isfinite(residual) ? __fmaf_rn(residual, rp.inv, q) : q;
  if (rp.plain) quotient = __fdiv_rn(x, rp.rep);
  const float y = x > 0.f ? quotient : __fmul_rn(x, rp.rep);
  x = n != 0 || (word & kPromptBit) ? y : x;
  const float less = __fsub_rn(__fsub_rn(x, __fmul_rn(rp.freq, (float)n)), rp.pres);
  x = n != 0 ? less : x;
  if (!kBiasFirst && bias != 0) x += bias_sums[bias - 1];
  return x;
}

// Element j of a vector in registers.
template <typename T>
__device__ __forceinline__ float element(const uint4 (&v)[kVec * sizeof(T) / 16], int j) {
  auto pick = [](const uint4& w, int k) { return k & 2 ? (k & 1 ? w.w : w.z) : (k & 1 ? w.y : w.x); };
  if constexpr (sizeof(T) == 2) {
    const uint16_t half = (uint16_t)(pick(v[0], j >> 1) >> (j & 1) * 16);
    return lo_f(*reinterpret_cast<const T*>(&half));
  } else {
    return __uint_as_float(j & 4 ? pick(v[1], j & 3) : pick(v[0], j & 3));
  }
}

// kVector: vectors of 8 columns (see above); otherwise element by element, for any strides. kBiasFirst:
// an instance of its own, since a choice made per touched token took 128 rows with histories and
// biases from 44.1 us to 45.3.
template <typename T, bool kVector, bool kBiasFirst, int kThreads, int kCtas>
__global__ void __launch_bounds__(kThreads, kCtas) logits_kernel(const LogitArgs p) {
  extern __shared__ __align__(16) uint32_t words[];
  const int row = blockIdx.x / p.slices;
  // columns with the shift: the row's are shift .. shift + vocab - 1
  const int shift = kVector ? (int)((int64_t)row * p.vocab & 7) : 0;
  const int lo = (blockIdx.x - row * p.slices) * p.slice;  // the slice's first
  const int from = max(0, shift - lo), to = min(p.slice, p.vocab + shift - lo);  // of the slice
  float* bias_sums = reinterpret_cast<float*>(words + p.slice);
  uint32_t* bias_cols = reinterpret_cast<uint32_t*>(bias_sums + p.n_bias);  // or ~0
  const bool history = p.tokens != nullptr, touches = history || p.n_bias > 0;
  if (touches) {
    for (int i = threadIdx.x * 4; i < p.slice; i += kThreads * 4)
      *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
  }
  grid_dep_wait();
  grid_dep_launch();

  // ---- loads ahead: lengths, parameters, biases, the slice's logits and mask; then, with the
  // lengths, the first tokens
  int seq = row, total = 0, prompt = 0;
  if (history) {
    if (p.row_seq) seq = p.row_seq[row];
    total = p.total_lens[row];
    prompt = p.prompt_lens[row];
  }
  RowParams rp = row_params(p, row);
  const int64_t list = (int64_t)row * p.n_bias;
  int bias_id = -1;
  float bias_value = 0.f;
  if ((int)threadIdx.x < p.n_bias) {
    bias_id = p.bias_ids[list + threadIdx.x];
    bias_value = p.bias_values[list + threadIdx.x];
  }
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
      bits[s] = !mask || i >= to ? ~0u
                : (bit0 & 7) == 0 ? reinterpret_cast<const uint8_t*>(mask)[(bit0 + i) >> 3]
                                  : mask_bits(mask, p.mask_words, bit0 + i);
    }
  }
  // The first of the history's tokens in place k of a thread's batch from i0 on, and its column of
  // the slice, counted from `from` (or a value behind the slice): four neighbours per load where the
  // rows of int32 tokens are aligned for it.
  const uint32_t token0 = (uint32_t)(bit0 + from), width = (uint32_t)max(0, to - from);
  total = seq < 0 || seq >= p.seqs ? 0 : min(max(total, 0), p.max_tokens);
  const int64_t at = (int64_t)(total ? seq : 0) * p.tokens_stride;
  uint32_t cols[kAhead];
  auto place = [&](int i0, int k) {
    return p.tokens_by4 ? i0 + ((k >> 2) * kThreads + (int)threadIdx.x) * 4 + (k & 3)
                        : i0 + k * kThreads + (int)threadIdx.x;
  };
  auto fetch = [&](int i0) {
    if (p.tokens_by4) {
#pragma unroll
      for (int k = 0; k < kAhead; k += 4) {
        const int i = place(i0, k);
        uint4 four = make_uint4(~0u, ~0u, ~0u, ~0u);
        const int32_t* src = static_cast<const int32_t*>(p.tokens) + at + i;
        if (i + 4 <= total) {
          four = *reinterpret_cast<const uint4*>(src);
        } else {
          if (i < total) four.x = (uint32_t)src[0];
          if (i + 1 < total) four.y = (uint32_t)src[1];
          if (i + 2 < total) four.z = (uint32_t)src[2];
        }
        cols[k] = four.x, cols[k + 1] = four.y, cols[k + 2] = four.z, cols[k + 3] = four.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = place(i0, k);
        int64_t id = -1;
        if (i < total)
          id = p.tokens64 ? static_cast<const int64_t*>(p.tokens)[at + i]
                          : (int64_t)static_cast<const int32_t*>(p.tokens)[at + i];
        cols[k] = id >= 0 && id <= 0x7fffffff ? (uint32_t)id : ~0u;
      }
    }
  };
  if (history) fetch(0);
  rp.inv = __frcp_rn(rp.rep);
  rp.plain = !(fabsf(rp.rep) > 0x1p-100f && fabsf(rp.rep) < 0x1p100f);

  // ---- biases: keys into the words, sums by key
  if (p.n_bias > 0) {
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads) {
      if (e >= kThreads) bias_id = p.bias_ids[list + e], bias_value = p.bias_values[list + e];
      const uint32_t col = (uint32_t)bias_id - token0;
      bias_cols[e] = bias_id >= 0 && col < width ? (uint32_t)from + col : ~0u;
      bias_sums[p.n_bias - 1 - e] = bias_value;  // by key - 1
    }
    __syncthreads();  // the words are zero, the list is here
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads)
      if (bias_cols[e] != ~0u) atomicMax(&words[bias_cols[e]], (uint32_t)(p.n_bias - e) << 20);
    __syncthreads();
    // an entry that is not its token's first leaves a mark at the one that is
    for (int e = threadIdx.x; e < p.n_bias; e += kThreads) {
      const uint32_t col = bias_cols[e];  // perhaps marked already
      if (col == ~0u) continue;
      const int one = p.n_bias - (int)(words[col & ~kMark] >> 20);
      if (one != e) atomicOr(&bias_cols[one], kMark);
    }
    __syncthreads();
    // a warp per marked entry: the lanes' sums are joined in a fixed order
    const int lane = threadIdx.x & 31;
    for (int e0 = (int)threadIdx.x - lane; e0 < p.n_bias; e0 += kThreads) {
      const uint32_t mine = e0 + lane < p.n_bias ? bias_cols[e0 + lane] : ~0u;
      for (uint32_t left = __ballot_sync(~0u, mine != ~0u && (mine & kMark)); left; left &= left - 1) {
        const int e = e0 + __ffs(left) - 1;
        const uint32_t col = bias_cols[e];
        double sum = 0.0;
        for (int j = e + lane; j < p.n_bias; j += 32)
          if ((bias_cols[j] & ~kMark) == (col & ~kMark)) sum += (double)p.bias_values[list + j];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == 0) bias_sums[p.n_bias - 1 - e] = (float)sum;
      }
    }
  }

  // ---- history
  if (touches) __syncthreads();  // the words are zero, or hold the biases' keys
  for (int i0 = 0; i0 < total; i0 += kAhead * kThreads) {
    uint32_t now[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) now[k] = cols[k] - token0;  // ids below the slice: huge
    if (i0 + kAhead * kThreads < total) fetch(i0 + kAhead * kThreads);  // behind these counts
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (now[k] >= width) continue;
      if (place(i0, k) < prompt)
        atomicOr(&words[from + now[k]], kPromptBit);
      else
        atomicAdd(&words[from + now[k]], 1u);
    }
  }
  if (touches) __syncthreads();

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
      if (touches) {
        // A touched token's result takes the place of its word. A thread has few of them: one at a
        // time, all threads of a warp together.
        uint32_t touched = 0;
#pragma unroll
        for (int h = 0; h < kVec; h += 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(words + i + h);
          touched |= (w.x ? 1u << h : 0) | (w.y ? 2u << h : 0) | (w.z ? 4u << h : 0) | (w.w ? 8u << h : 0);
        }
        for (uint32_t left = touched; left; left &= left - 1) {
          const int j = __ffs(left) - 1;
          words[i + j] =
              __float_as_uint(process<kBiasFirst>(element<T>(raw[s], j), words[i + j], rp, bias_sums));
        }
        if (touched) {
#pragma unroll
          for (int h = 0; h < kVec; h += 4) {
            const float4 y = *reinterpret_cast<const float4*>(words + i + h);
            x[h] = touched & 1u << h ? y.x : x[h];
            x[h + 1] = touched & 2u << h ? y.y : x[h + 1];
            x[h + 2] = touched & 4u << h ? y.z : x[h + 2];
            x[h + 3] = touched & 8u << h ? y.w : x[h + 3];
          }
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
        if (touches && words[i]) x[j] = process<kBiasFirst>(x[j], words[i], rp, bias_sums);
        if (mask && !(mask_bits(mask, p.mask_words, bit0 + i) & 1u)) x[j] = ninf;
        out[i] = x[j];
      }
    }
  }
}

template <typename T, bool kVector, bool kBiasFirst, int kThreads, int kCtas>
int launch_sized(const LogitArgs& p, int grid, cudaStream_t stream) {
  const bool touches = p.tokens || p.n_bias > 0;
  const size_t smem = touches ? sizeof(uint32_t) * ((size_t)p.slice + 2 * (size_t)p.n_bias) : 0;
  auto kernel = logits_kernel<T, kVector, kBiasFirst, kThreads, kCtas>;
  static bool configured[64] = {};
  int dev = 0;
  B2_CUDA_TRY(cudaGetDevice(&dev));
  if (!configured[dev]) {
    B2_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)(sizeof(uint32_t) * (kMaxSlice + 2 * kMaxBias))));
    configured[dev] = true;
  }
  return launch_kernel(kernel, grid, kThreads, smem, stream, /*early=*/true, p);
}

template <typename T, bool kVector, bool kBiasFirst>
int launch_typed(LogitArgs& p, int rows, cudaStream_t stream) {
  DeviceInfo di;
  int rc = device_info(&di);
  if (rc) return rc;
  // Enough slices per row to give every SM a CTA and none two (8 rows of 151936 with 19 slices, 4 more
  // CTAs than SMs: 8.0 us, with 18: 6.6), as long as a CTA keeps a whole step.
  const int columns = p.vocab + kVec - 1;  // with the shift
  auto steps_of = [&](int threads) { return (columns + threads * kVec - 1) / (threads * kVec); };
  const int each = std::max(di.sm_count / rows, 1);
  // Half the threads where that puts more SMs to work and a history takes them one batch of loads: a
  // row of 18992, 10 CTAs instead of 5, 2.6 us instead of 3.1; with histories of 4000 a row of 151936
  // would take 4.5 us instead of 4.1, of 16384 8.4 instead of 6.4.
  const bool half = steps_of(kMostThreads) < each &&
                    (!p.tokens || p.max_tokens <= kAhead * kMostThreads / 2);
  const int steps = steps_of(half ? kMostThreads / 2 : kMostThreads);
  const int need = (columns + kMaxSlice - 1) / kMaxSlice;
  p.slices = std::max(need, std::min(each, steps));
  const int slice = (columns + p.slices - 1) / p.slices;
  p.slice = (slice + kVec - 1) / kVec * kVec;
  const int64_t grid = (int64_t)rows * p.slices;
  if (grid > 0x7fffffff)
    return fail(B2_ERR_INVALID_ARG, "logits_process: %d rows of %d logits are too many", rows, p.vocab);
  // Where an SM has one CTA it may have all the registers: 8 rows 6.2 us instead of 6.6.
  if (half && p.slice <= kMaxSlice / 2)
    return launch_sized<T, kVector, kBiasFirst, kMostThreads / 2, 1>(p, (int)grid, stream);
  if (grid <= di.sm_count)
    return launch_sized<T, kVector, kBiasFirst, kMostThreads, 1>(p, (int)grid, stream);
  return launch_sized<T, kVector, kBiasFirst, kMostThreads, 2>(p, (int)grid, stream);
}


template <typename T>
int launch_type(LogitArgs& p, int rows, bool vector, bool bias_first, cudaStream_t stream) {
  if (bias_first)
    return vector ? launch_typed<T, true, true>(p, rows, stream)
                  : launch_typed<T, false, true>(p, rows, stream);
  return vector ? launch_typed<T, true, false>(p, rows, stream)
                : launch_typed<T, false, false>(p, rows, stream);
}

int check_and_launch(const void* logits, int64_t row_stride, int dtype, float* out, int rows, int vocab,
                     int vocab_start, const void* tokens, int tokens_64, int64_t tokens_stride,
                     int n_seqs, int max_tokens, const int32_t* row_seq, const int32_t* prompt_lens,
                     const int32_t* total_lens, const float* repetition, const float* frequency,
                     const float* presence, const int32_t* bias_ids, const float* bias_values,
                     int n_bias, const uint32_t* mask, int64_t mask_stride, int mask_words,
                     bool bias_first, void* stream) {
  const char* op = "logits_process";
  if (rows < 0 || vocab < 1 || vocab > kMaxVocab)
    return fail(B2_ERR_INVALID_ARG, "%s: %d rows of %d logits (at most %d)", op, rows, vocab, kMaxVocab);
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
  p.tokens_by4 = !tokens_64 && tokens_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(tokens) & 15u) == 0;
  p.row_seq = row_seq, p.prompt_lens = prompt_lens, p.total_lens = total_lens;
  p.repetition = repetition, p.frequency = frequency, p.presence = presence;
  p.bias_ids = bias_ids, p.bias_values = bias_values, p.n_bias = n_bias;
  p.mask = mask, p.mask_stride = mask_stride, p.mask_words = mask_words;
  p.vocab = vocab, p.vocab_start = vocab_start;
  const bool vector = (reinterpret_cast<uintptr_t>(logits) & 15u) == 0 &&
                      (reinterpret_cast<uintptr_t>(out) & 31u) == 0 && (row_stride - vocab) % kVec == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // The order matters to a biased token that the penalties touch.
  const bool first = bias_first && p.tokens && n_bias > 0;
  if (dtype == B2_DTYPE_F16) return launch_type<__half>(p, rows, vector, first, s);
  if (dtype == B2_DTYPE_BF16) return launch_type<__nv_bfloat16>(p, rows, vector, first, s);
  return launch_type<float>(p, rows, vector, first, s);
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
  return b2::check_and_launch(logits, row_stride, dtype, out, rows, vocab, vocab_start, tokens, tokens_64,
                              tokens_stride, n_seqs, max_tokens, row_seq, prompt_lens, total_lens,
                              repetition, frequency, presence, bias_ids, bias_values, n_bias, mask,
                              mask_stride, mask_words, /*bias_first=*/false, stream);
}

extern "C" int b2_logits_process_bias_first(
    const void* logits, int64_t row_stride, int dtype, float* out, int rows, int vocab, int vocab_start,
    const void* tokens, int tokens_64, int64_t tokens_stride, int n_seqs, int max_tokens,
    const int32_t* row_seq, const int32_t* prompt_lens, const int32_t* total_lens,
    const float* repetition, const float* frequency, const float* presence, const int32_t* bias_ids,
    const float* bias_values, int n_bias, const uint32_t* mask, int64_t mask_stride, int mask_words,
    void* stream) {
  return b2::check_and_launch(logits, row_stride, dtype, out, rows, vocab, vocab_start, tokens, tokens_64,
                              tokens_stride, n_seqs, max_tokens, row_seq, prompt_lens, total_lens,
                              repetition, frequency, presence, bias_ids, bias_values, n_bias, mask,
                              mask_stride, mask_words, /*bias_first=*/true, stream);
}
