// Rotary positions for the rows of a step, and the same with the cache write that follows.
//
//   pair (a, b) of frequency i, row at position p:   t = p * inv_freq[i]
//     a' = scale * (a cos t - b sin t),   b' = scale * (b cos t + a sin t)
// The pairs are (x[i], x[i + rot/2]) (half layout) or (x[2i], x[2i+1]) (interleaved); dimensions
// from `rot` on are copied. b2_rope turns q and k into new tensors; b2_rope_cache turns q, and
// writes the turned k and the plain v to the rows' slots of a paged cache, which saves a launch
// and one write and one read of k.
//
// Angles: the product p * inv_freq is formed in fp64 and reduced there to a fraction of a turn in
// [-1/2, 1/2], whose sine and cosine are taken in fp32. A fp32 product would be off by p * 2^-24
// radians, 0.06 at position 10^6; the reduced fraction is off by 2^-26 turns, its rounding to fp32,
// and by 2.5 * 2^-53 of the turns themselves, which is a tenth of that at 2^25 radians. The fp64 work
// is three operations per frequency and row, shared by all heads of the row through a table in shared
// memory.
//
// Bound: memory. A row's heads are read and written once, 16 bytes per access; a thread owns both
// members of its pairs, so outputs may alias inputs. The table is built behind the loads of the
// first item (a block holds one row, or part of one when there are few rows). 4099 rows of
// 32 + 8 heads of 128 in bf16: b2_rope 15.8 us, 5.3 TB/s; 2048 such rows: b2_rope_cache 10.3 us, 4.9
// TB/s. 8 rows are bound by launch and the latency positions -> table -> stores: 1.7 and 2.1 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "b2_device.cuh"
#include "b2_internal.h"

namespace b2 {
namespace {

constexpr int kMaxDim = 1024;
constexpr int kRopeThreads = 128;
constexpr int kMaxGridY = 65535;
// Items of a thread whose loads are under way together, with many rows; with few, a thread has one.
// With one, 2048 rows with the cache write take 11.3 us instead of 10.3; with four 11.9, and 4099 rows
// 16.9 instead of 15.8. Blocks of 64 threads: 9.4 and 16.5; of 256: 13.8 and 19.9. Where a thread has
// one, room for three costs 8 rows 2.0 us instead of 1.7.
constexpr int kManyAhead = 3;

struct RopeArgs {
  const void *q, *k, *v;
  const void* positions;
  const float* inv_freq;
  const int64_t* slots;
  void *q_out, *k_out, *k_cache, *v_cache;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // input strides in elements
  int64_t kc[3], vc[3];                                 // cache strides: page, token, head
  int64_t n_slots;
  int q_heads, kv_heads, dim, rot, page;
  int units;        // work units per head
  int items;        // units of a whole row, 2^27 at most
  int chunk;        // items per block
  FastDiv by_units;
  int pos64;
  float scale;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// What one item of a row is: its input and where its output goes (null: nowhere).
template <typename T>
struct Item {
  const T* in;
  T* out;
  bool turn;  // a query or key head (a value head is copied)
};

template <typename T, bool kCache>
__device__ __forceinline__ Item<T> locate(const RopeArgs& p, int64_t row, int head, int64_t k_at,
                                          int64_t v_at) {
  Item<T> it;
  it.turn = true;
  if (head < p.q_heads) {
    it.in = static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head;
    it.out = static_cast<T*>(p.q_out) + (row * p.q_heads + head) * p.dim;
    return it;
  }
  head -= p.q_heads;
  if (head < p.kv_heads) {
    it.in = static_cast<const T*>(p.k) + row * p.k_row + head * p.k_head;
    if constexpr (kCache)
      it.out = k_at < 0 ? nullptr : static_cast<T*>(p.k_cache) + k_at + head * p.kc[2];
    else
      it.out = static_cast<T*>(p.k_out) + (row * p.kv_heads + head) * p.dim;
    return it;
  }
  head -= p.kv_heads;
  it.turn = false;
  it.in = static_cast<const T*>(p.v) + row * p.v_row + head * p.v_head;
  it.out = k_at < 0 ? nullptr : static_cast<T*>(p.v_cache) + v_at + head * p.vc[2];
  return it;
}

// kAhead > 0: units of two 8-element vectors (16-bit types, aligned); otherwise units of one pair, or of
// two copied elements behind the turned part (any type, stride and even rot).
template <typename T, bool kInterleaved, bool kCache, int kAhead>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs p) {
  __shared__ __align__(16) float s_cos[kMaxDim / 2], s_sin[kMaxDim / 2];
  const int64_t row = blockIdx.x;
  const int first = blockIdx.y * p.chunk;
  const int last = min(first + p.chunk, p.items);
  const int half = p.rot / 2;
  grid_dep_wait();
  grid_dep_launch();

  int64_t k_at = -1, v_at = -1;
  if constexpr (kCache) {
    const int64_t slot = p.slots[row];
    if (slot >= 0 && slot < p.n_slots) {
      const int64_t page = slot / p.page, at = slot % p.page;
      k_at = page * p.kc[0] + at * p.kc[1];
      v_at = page * p.vc[0] + at * p.vc[1];
    }
  }
  const double pos = p.pos64 ? (double)static_cast<const int64_t*>(p.positions)[row]
                             : (double)static_cast<const int32_t*>(p.positions)[row];
  auto table = [&] {
    for (int i = threadIdx.x; i < half; i += kRopeThreads) {
      double turns = pos * (double)p.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
      turns -= rint(turns);
      float s, c;
      sincospif(2.0f * (float)turns, &s, &c);
      s_cos[i] = c * p.scale;
      s_sin[i] = s * p.scale;
    }
    __syncthreads();
  };

  if constexpr (kAhead > 0) {
    const int turned = p.rot / 16, vectors = p.dim / 8;
    bool built = false;
    for (int base = first; base < last || !built; base += kAhead * kRopeThreads) {
      // all loads of kAhead items before the table and the arithmetic
      uint4 va[kAhead], vb[kAhead];
      Item<T> it[kAhead];
      int unit[kAhead], a[kAhead], b[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = base + k * kRopeThreads + threadIdx.x;
        const int head = i < last ? p.by_units.div(i) : 0;
        const int u = i < last ? i - head * p.units : 0;
        it[k] = locate<T, kCache>(p, row, head, k_at, v_at);
        if (i >= last) it[k].out = nullptr;
        it[k].turn = it[k].turn && u < turned;
        unit[k] = u;
        a[k] = (!kInterleaved && it[k].turn) ? u : 2 * u;
        b[k] = (!kInterleaved && it[k].turn) ? u + turned : 2 * u + 1;
        va[k] = vb[k] = make_uint4(0, 0, 0, 0);
        if (it[k].out) {
          va[k] = *reinterpret_cast<const uint4*>(it[k].in + 8 * a[k]);
          if (b[k] < vectors) vb[k] = *reinterpret_cast<const uint4*>(it[k].in + 8 * b[k]);
        }
      }
      if (!built) table();
      built = true;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (!it[k].out) continue;
        if (it[k].turn) {
          T* ea = reinterpret_cast<T*>(&va[k]);
          T* eb = reinterpret_cast<T*>(&vb[k]);
          float c[8], s[8];
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            *reinterpret_cast<float4*>(&c[j]) = *reinterpret_cast<const float4*>(&s_cos[8 * unit[k] + j]);
            *reinterpret_cast<float4*>(&s[j]) = *reinterpret_cast<const float4*>(&s_sin[8 * unit[k] + j]);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            T& ra = kInterleaved ? (j < 4 ? ea[2 * (j & 3)] : eb[2 * (j & 3)]) : ea[j];
            T& rb = kInterleaved ? (j < 4 ? ea[2 * (j & 3) + 1] : eb[2 * (j & 3) + 1]) : eb[j];
            const float x = to_f(ra), y = to_f(rb);
            ra = from_f<T>(x * c[j] - y * s[j]);
            rb = from_f<T>(y * c[j] + x * s[j]);
          }
        }
        *reinterpret_cast<uint4*>(it[k].out + 8 * a[k]) = va[k];
        if (b[k] < vectors) *reinterpret_cast<uint4*>(it[k].out + 8 * b[k]) = vb[k];
      }
    }
  } else {
    table();
    for (int i = first + threadIdx.x; i < last; i += kRopeThreads) {
      const int head = p.by_units.div(i), u = i - head * p.units;
      const Item<T> it = locate<T, kCache>(p, row, head, k_at, v_at);
      if (!it.out) continue;
      const bool turn = it.turn && u < half;
      const int a = (turn && !kInterleaved) ? u : 2 * u;
      const int b = (turn && !kInterleaved) ? u + half : 2 * u + 1;
      if (a >= p.dim) continue;
      const float x = to_f(it.in[a]), y = b < p.dim ? to_f(it.in[b]) : 0.f;
      if (turn) {
        const float c = s_cos[u], s = s_sin[u];
        it.out[a] = from_f<T>(x * c - y * s);
        it.out[b] = from_f<T>(y * c + x * s);
      } else {
        it.out[a] = from_f<T>(x);
        if (b < p.dim) it.out[b] = from_f<T>(y);
      }
    }
  }
}

template <typename T, bool kInterleaved, bool kCache>
int launch_typed(RopeArgs& p, int rows, bool vec, bool few, cudaStream_t stream) {
  const int heads = p.q_heads + p.kv_heads * (kCache ? 2 : 1);
  p.units = vec ? (p.dim + 15) / 16 : (p.dim + 1) / 2;
  p.items = heads * p.units;
  p.by_units = make_div(p.units);
  // A block per row, or with fewer rows than SMs an item per thread, so that more of them take part;
  // more items than that where a row of very many heads would have more blocks than a grid may along y.
  const int least = std::max(kRopeThreads, (p.items + kMaxGridY - 1) / kMaxGridY);
  p.chunk = few ? std::min(p.items, least) : p.items;
  const dim3 grid((unsigned)rows, (unsigned)((p.items + p.chunk - 1) / p.chunk));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kRopeThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = tuning(B2_TUNE_NO_PDL) == 0 ? 1 : 0;
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      if (p.chunk <= kRopeThreads)
        B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, rope_kernel<T, kInterleaved, kCache, 1>, p));
      else
        B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, rope_kernel<T, kInterleaved, kCache, kManyAhead>, p));
      return B2_OK;
    }
  }
  B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, rope_kernel<T, kInterleaved, kCache, 0>, p));
  return B2_OK;
}

template <bool kCache>
int launch_rope(RopeArgs& p, int rows, int interleaved, int dtype, cudaStream_t stream,
                const char* op) {
  if (rows < 0) return fail(B2_ERR_INVALID_ARG, "%s: rows=%d", op, rows);
  if (p.q_heads < 1 || p.kv_heads < 1 || p.q_heads > 65536 || p.kv_heads > 65536)
    return fail(B2_ERR_INVALID_ARG, "%s: %d query and %d key heads", op, p.q_heads, p.kv_heads);
  if (p.dim < 2 || p.dim > kMaxDim)
    return fail(B2_ERR_INVALID_ARG, "%s: head_dim=%d outside 2..%d", op, p.dim, kMaxDim);
  if (p.rot < 2 || p.rot > p.dim || p.rot % 2 != 0)
    return fail(B2_ERR_INVALID_ARG, "%s: rot_dim=%d must be even and within head_dim=%d", op, p.rot,
                p.dim);
  if (dtype != B2_DTYPE_F16 && dtype != B2_DTYPE_BF16 && dtype != B2_DTYPE_F32)
    return fail(B2_ERR_INVALID_ARG, "%s: dtype %d", op, dtype);
  if (rows == 0) return B2_OK;
  if (!p.q || !p.k || !p.positions || !p.inv_freq || !p.q_out)
    return fail(B2_ERR_INVALID_ARG, "%s: null pointer", op);
  if (kCache ? (!p.v || !p.slots || !p.k_cache || !p.v_cache) : !p.k_out)
    return fail(B2_ERR_INVALID_ARG, "%s: null pointer", op);
  DeviceInfo di;
  const int rc = device_info(&di);
  if (rc) return rc;
  const bool few = rows < di.sm_count;
  bool vec = dtype != B2_DTYPE_F32 && p.dim % 8 == 0 && p.rot % 16 == 0 && aligned16(p.q) &&
             aligned16(p.k) && aligned16(p.q_out);
  for (int64_t s : {p.q_row, p.q_head, p.k_row, p.k_head}) vec = vec && s % 8 == 0;
  if (kCache) {
    vec = vec && aligned16(p.v) && aligned16(p.k_cache) && aligned16(p.v_cache);
    vec = vec && p.v_row % 8 == 0 && p.v_head % 8 == 0;
    for (int i = 0; i < 3; ++i) vec = vec && p.kc[i] % 8 == 0 && p.vc[i] % 8 == 0;
  } else {
    vec = vec && aligned16(p.k_out);
  }
  switch (dtype * 2 + (interleaved ? 1 : 0)) {
    case B2_DTYPE_F16 * 2: return launch_typed<__half, false, kCache>(p, rows, vec, few, stream);
    case B2_DTYPE_F16 * 2 + 1: return launch_typed<__half, true, kCache>(p, rows, vec, few, stream);
    case B2_DTYPE_BF16 * 2: return launch_typed<__nv_bfloat16, false, kCache>(p, rows, vec, few, stream);
    case B2_DTYPE_BF16 * 2 + 1:
      return launch_typed<__nv_bfloat16, true, kCache>(p, rows, vec, few, stream);
    case B2_DTYPE_F32 * 2: return launch_typed<float, false, kCache>(p, rows, vec, few, stream);
    default: return launch_typed<float, true, kCache>(p, rows, vec, few, stream);
  }
}

}  // namespace
}  // namespace b2

extern "C" int b2_rope(const void* q, const int64_t* q_strides, const void* k,
                       const int64_t* k_strides, const void* positions, int positions_64,
                       const float* inv_freq, void* q_out, void* k_out, int rows, int q_heads,
                       int kv_heads, int head_dim, int rot_dim, float scale, int interleaved,
                       int dtype, void* stream) {
  using namespace b2;
  if (!q_strides || !k_strides) return fail(B2_ERR_INVALID_ARG, "rope: null strides");
  RopeArgs p = {};
  p.q = q, p.k = k;
  p.positions = positions, p.pos64 = positions_64;
  p.inv_freq = inv_freq;
  p.q_out = q_out, p.k_out = k_out;
  p.q_row = q_strides[0], p.q_head = q_strides[1];
  p.k_row = k_strides[0], p.k_head = k_strides[1];
  p.q_heads = q_heads, p.kv_heads = kv_heads, p.dim = head_dim, p.rot = rot_dim;
  p.scale = scale;
  return launch_rope<false>(p, rows, interleaved, dtype, static_cast<cudaStream_t>(stream), "rope");
}

extern "C" int b2_rope_cache(const void* q, const int64_t* q_strides, const void* k,
                             const int64_t* k_strides, const void* v, const int64_t* v_strides,
                             const void* positions, int positions_64, const float* inv_freq,
                             const int64_t* slots, void* q_out, void* k_cache,
                             const int64_t* k_cache_strides, void* v_cache,
                             const int64_t* v_cache_strides, int pages, int page_size, int rows,
                             int q_heads, int kv_heads, int head_dim, int rot_dim, float scale,
                             int interleaved, int dtype, void* stream) {
  using namespace b2;
  if (!q_strides || !k_strides || !v_strides || !k_cache_strides || !v_cache_strides)
    return fail(B2_ERR_INVALID_ARG, "rope_cache: null strides");
  if (pages < 1 || page_size < 1)
    return fail(B2_ERR_INVALID_ARG, "rope_cache: %d pages of %d tokens", pages, page_size);
  RopeArgs p = {};
  p.q = q, p.k = k, p.v = v;
  p.positions = positions, p.pos64 = positions_64;
  p.inv_freq = inv_freq;
  p.slots = slots;
  p.q_out = q_out, p.k_cache = k_cache, p.v_cache = v_cache;
  p.q_row = q_strides[0], p.q_head = q_strides[1];
  p.k_row = k_strides[0], p.k_head = k_strides[1];
  p.v_row = v_strides[0], p.v_head = v_strides[1];
  for (int i = 0; i < 3; ++i) p.kc[i] = k_cache_strides[i], p.vc[i] = v_cache_strides[i];
  p.n_slots = (int64_t)pages * page_size;
  p.page = page_size;
  p.q_heads = q_heads, p.kv_heads = kv_heads, p.dim = head_dim, p.rot = rot_dim;
  p.scale = scale;
  return launch_rope<true>(p, rows, interleaved, dtype, static_cast<cudaStream_t>(stream),
                           "rope_cache");
}
