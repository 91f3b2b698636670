// Attention of a step's rows over a paged cache in which all requests share a long prefix.
//
// Row t of request b (rows row_start[b] .. row_start[b+1]), query head h, KV head h / G:
//   s_j = scale * q[t,h] . k_j     over the prefix tokens, which every row sees, and the request's
//                                  own tokens, of which the row sees those up to itself (or, with
//                                  a tree mask, its ancestors among the request's new tokens)
//   out = sum_j exp(s_j - m) v_j / l,  m = max_j s_j,  l = sum_j exp(s_j - m),  lse = m + log l
// A row that sees nothing gives out = 0 and lse = -inf.
//
// The rows' queries of one KV head form the M side of the products: T*G rows for the prefix, which
// is read once for all of them, and n_b*G for a request's own tokens. Work is counted in units of
// one tile of kTok tokens for one block of rows and one KV head, over all segments (segment 0 =
// the prefix, segment b+1 = request b's own tokens). A persistent grid takes equal contiguous
// ranges of units, whatever the lengths on the device say, so a captured graph follows growing
// lengths. A range's piece of one (segment, head, row block) group ends in an unnormalised fp32
// partial (O, m, l) in the workspace, at slot cta + group (no two pieces share one); a second
// launch joins the partials of each row in a fixed order, so results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "b2_device.cuh"
#include "b2_internal.h"

namespace b2 {
namespace {

constexpr int kMaxRequests = 1024;
constexpr int kMaxRows = 4096;
constexpr int kSoftWarps = 4;      // one thread per row of a block
constexpr int kLoadThreads = 128;
constexpr int kAttnThreads = kSoftWarps * 32 + 32 + kLoadThreads;
constexpr int kBlockRows = 128;
constexpr int kJoinThreads = 128;
constexpr int kMaxCtas = 160;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head;
  int64_t ks[3], vs[3];  // page, token, head strides of the caches in elements
  const int32_t *prefix_pages, *prefix_len, *pages, *own_lens, *row_start;
  const int64_t* tree;
  void* out;
  float* lse;
  float* part_o;   // [slots][rows per block][dim]
  float2* part_ml; // [slots][rows per block]
  int64_t pages_stride;
  int total_pages, page_size, n_prefix_pages, max_pages;
  int requests, rows, q_heads, kv_heads, group, dim;
  int slots;
  int q_vec;  // queries allow 16-byte loads
  float scale_log2;
};

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  static constexpr uint32_t kExp = 0x7c00u;  // exponent bits: all set in infinities and NaN
  static constexpr uint32_t kFormat = 0;     // operand format of the instruction descriptor
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr uint32_t kFormat = 1;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Of two packed 16-bit numbers: is one of them an infinity or NaN; the two with those replaced by 0.
template <typename T>
__device__ __forceinline__ bool non_finite(uint32_t w) {
  constexpr uint32_t e = Pair<T>::kExp;
  return (w & e) == e || ((w >> 16) & e) == e;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
  constexpr uint32_t e = Pair<T>::kExp;
  return ((w & e) == e ? 0u : w & 0xffffu) | (((w >> 16) & e) == e ? 0u : w & 0xffff0000u);
}
// 16 bytes from global to shared memory; `bytes` = 16, or 0 to write zeros without reading.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
// One arrival on `bar` once this thread's copies so far have landed (counted in its init).
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ------------------------------------------------------------------------------------------------
// tcgen05: one CTA, accumulators and the A operand in tensor memory, B in 128-byte-swizzled shared
// memory. Addresses: lane << 16 | column.
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns)
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Arrive on `bar` when every tcgen05.mma this thread has issued has completed.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}
// D[128, N] (+)= A[128, 16] B[16, N]: A in tensor memory, B through a shared-memory descriptor.
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Shared-memory descriptor, 128-byte swizzle; byte offsets between repeats of the 8-row pattern.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(leading >> 4) << 16 |
         (uint64_t)(stride >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor: fp32 accumulator, M = 128, N columns, B with K or N contiguous.
template <typename T>
__host__ __device__ constexpr uint32_t instr_desc(int n, bool b_n_major) {
  return 1u << 4 | Pair<T>::kFormat << 7 | Pair<T>::kFormat << 10 | (b_n_major ? 1u << 16 : 0u) |
         (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}
// 32 columns of this warp's 32 lanes, one lane per thread.
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// ------------------------------------------------------------------------------------------------
// The plan: every block derives it from the lengths on the device.
// ------------------------------------------------------------------------------------------------
struct Plan {
  int units_end[kMaxRequests + 1];   // running sum of units up to and with segment s
  int groups_end[kMaxRequests + 1];  // running sum of groups
  int warp_sum[2][kAttnThreads / 32];
};

// Rows [first, first + count) of a request, and how many of its own tokens are stored.
__device__ __forceinline__ void request_rows(const AttnArgs& p, int b, int& first, int& count) {
  first = min(max(p.row_start[b], 0), p.rows);
  count = max(0, min(max(p.row_start[b + 1], 0), p.rows) - first);
}
__device__ __forceinline__ int own_length(const AttnArgs& p, int b) {
  return (int)min((int64_t)max(p.own_lens[b], 0), (int64_t)p.max_pages * p.page_size);
}
__device__ __forceinline__ int prefix_length(const AttnArgs& p) {
  return (int)min((int64_t)max(*p.prefix_len, 0), (int64_t)p.n_prefix_pages * p.page_size);
}
__device__ __forceinline__ void segment_shape(const AttnArgs& p, int s, int tok, int block_rows,
                                              int& first, int& count, int& len, int& tiles,
                                              int& blocks) {
  if (s == 0) {
    first = min(max(p.row_start[0], 0), p.rows);
    count = max(0, min(max(p.row_start[p.requests], 0), p.rows) - first);
    len = prefix_length(p);
  } else {
    request_rows(p, s - 1, first, count);
    len = own_length(p, s - 1);
  }
  tiles = (len + tok - 1) / tok;
  blocks = (count * p.group + block_rows - 1) / block_rows;
}

// Block-wide scan over the segments; kWarps warps take part. Row starts that decrease are outside
// the contract: the plan is then empty (every output 0, lse -inf), so that no index leaves its array.
template <int kWarps>
__device__ __forceinline__ void make_plan(const AttnArgs& p, int tok, int block_rows, Plan& plan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int u_base = 0, g_base = 0;
  int bad = 0;
  for (int b = threadIdx.x; b < p.requests; b += kWarps * 32) bad |= p.row_start[b + 1] < p.row_start[b];
  bad = __syncthreads_or(bad);
  for (int s0 = 0; s0 <= p.requests; s0 += kWarps * 32) {
    const int s = s0 + threadIdx.x;
    int u = 0, g = 0;
    if (s <= p.requests) {
      int first, count, len, tiles, blocks;
      segment_shape(p, s, tok, block_rows, first, count, len, tiles, blocks);
      if (tiles > 0 && !bad) {
        g = p.kv_heads * blocks;
        u = g * tiles;
      }
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int uu = __shfl_up_sync(~0u, u, d), gg = __shfl_up_sync(~0u, g, d);
      if (lane >= d) u += uu, g += gg;
    }
    if (lane == 31) plan.warp_sum[0][warp] = u, plan.warp_sum[1][warp] = g;
    __syncthreads();
    int ub = u_base, gb = g_base;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) ub += plan.warp_sum[0][w], gb += plan.warp_sum[1][w];
      u_base += plan.warp_sum[0][w];
      g_base += plan.warp_sum[1][w];
    }
    if (s <= p.requests) plan.units_end[s] = ub + u, plan.groups_end[s] = gb + g;
    __syncthreads();
  }
}

// CTAs that share `units` units: at most `ctas`, none of them empty.
__device__ __forceinline__ int plan_ctas(int units, int ctas) { return min(units, ctas); }
__device__ __forceinline__ int plan_begin(int units, int ctas, int c) {
  return (int)((int64_t)units * c / ctas);
}
__device__ __forceinline__ int plan_owner(int units, int ctas, int u) {
  return (int)((((int64_t)u + 1) * ctas - 1) / units);
}

// A position in the unit order: segment, group inside it (head-major), tile.
struct Cursor {
  int seg, group, tile;              // group = head * blocks + row block
  int first, count, len, tiles, blocks;
  __device__ __forceinline__ void load(const AttnArgs& p, int tok, int block_rows) {
    segment_shape(p, seg, tok, block_rows, first, count, len, tiles, blocks);
  }
  __device__ __forceinline__ void seek(const AttnArgs& p, const Plan& plan, int u, int tok,
                                       int block_rows) {
    int lo = 0, hi = p.requests;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (plan.units_end[mid] > u) hi = mid; else lo = mid + 1;
    }
    seg = lo;
    load(p, tok, block_rows);
    const int local = u - (seg ? plan.units_end[seg - 1] : 0);
    group = local / tiles;
    tile = local - group * tiles;
  }
  __device__ __forceinline__ void next(const AttnArgs& p, const Plan& plan, int tok, int block_rows) {
    if (++tile < tiles) return;
    tile = 0;
    if (++group < p.kv_heads * blocks) return;
    group = 0;
    const int done = plan.units_end[seg];
    while (seg < p.requests && plan.units_end[seg + 1] == done) ++seg;
    if (seg < p.requests) {
      ++seg;
      load(p, tok, block_rows);
    }
  }
};

// ------------------------------------------------------------------------------------------------
// Main kernel. kDim: head dimension rounded up (64, 128, 256), the rest of it zero.
//
// Per tile: S[128 rows, kTok] = Q K^T and O[128 rows, kDim] += P V on the tensor cores, with Q, S,
// P and O in tensor memory (P takes the place of its S), K and V in a ring of shared-memory stages.
// K is the product's B operand with the dimension contiguous, V its B operand with N contiguous:
// both lie as loaded, [token][64 dimensions] rows of 128 bytes, swizzled.
//   warps 0-3  softmax: a thread owns a row (its lane of tensor memory), so the running maximum and
//              sum need no exchange between threads; they also bring Q in and take O out
//   warp 4     one thread issues the products: those of tile i + 1 before tile i's second one, so
//              that the tensor cores work while the softmax of tile i runs
//   warps 5-8  copy K and V, 16 bytes per cp.async, page by page, for any page size and strides
// O is rescaled only when a row's maximum has grown by more than 2^8 over the one its weights refer
// to (the weights stay below 2^8, in range of fp16, with the same relative rounding); the sum l and
// the partial refer to the same maximum, so nothing is approximated.
// ------------------------------------------------------------------------------------------------
template <int kDim>
struct Shape {
  static constexpr int kTok = kDim == 64 ? 128 : 64;  // tokens per tile
  static constexpr int kStages = kDim == 256 ? 3 : 6;
  static constexpr int kSub = kTok * 128;              // [token][64 dimensions] of K or V
  static constexpr int kHalf = kSub * (kDim / 64);     // K or V of a stage
  static constexpr int kRing = kStages * 2 * kHalf;
  static constexpr int kS = kDim, kQ = kDim + 2 * kTok;  // columns of tensor memory; O at 0
  static constexpr int kColumns = 512;
  static_assert(kQ + kDim / 2 <= kColumns, "tensor memory of an SM");
};

struct Control {
  uint64_t full[6], empty[6];
  uint64_t s_full[2], p_full[2], o_done[2], q_full, o_free, sync, drain;
  uint32_t tmem;
  int abort;
  int bad_unit[6];  // per stage: 1 + the unit, if any, for which a page id outside the cache was met
  int bad_value;    // 1 + the unit for which a value that is no number was met in a masked tile
  unsigned char bad_token[128];
};

template <int kDim>
constexpr size_t attn_smem() {
  return 1024 + Shape<kDim>::kRing + sizeof(Plan) + sizeof(Control) + 16;
}

__device__ int g_attn_status;

template <typename T, int kDim>
__global__ void __launch_bounds__(kAttnThreads, 1) attn_kernel(const AttnArgs p) {
  using S = Shape<kDim>;
  constexpr int kTok = S::kTok, kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Control& c = *reinterpret_cast<Control*>(smem + S::kRing);
  Plan& plan = *reinterpret_cast<Plan*>((reinterpret_cast<uintptr_t>(&c + 1) + 15) & ~(uintptr_t)15);
  volatile int* s_abort = &c.abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&c.full[s], kLoadThreads + kLoadThreads / 32);
      mbar_init(&c.empty[s], 1);
      c.bad_unit[s] = 0;
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&c.s_full[b], 1);
      mbar_init(&c.p_full[b], kSoftWarps);
      mbar_init(&c.o_done[b], 1);
    }
    mbar_init(&c.q_full, kSoftWarps);
    mbar_init(&c.o_free, kSoftWarps);
    mbar_init(&c.sync, kSoftWarps);
    mbar_init(&c.drain, 1);
    c.abort = 0;
    c.bad_value = 0;
    mbar_fence_init();
  }
  if (warp == kSoftWarps) tmem_alloc(&c.tmem, S::kColumns);
  grid_dep_wait();
  grid_dep_launch();
  make_plan<kAttnThreads / 32>(p, kTok, kBlockRows, plan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c.tmem;
  const int units = plan.units_end[p.requests];
  const int ctas = plan_ctas(units, gridDim.x);
  const bool idle = (int)blockIdx.x >= ctas;
  const int u_lo = idle ? 0 : plan_begin(units, ctas, blockIdx.x);
  const int u_hi = idle ? 0 : plan_begin(units, ctas, blockIdx.x + 1);
  const uint32_t ring = smem_u32(smem);
  const int stage_bytes = 2 * S::kHalf;

  Cursor cur;
  if (!idle) cur.seek(p, plan, u_lo, kTok, kBlockRows);

  if (warp > kSoftWarps) {
    // ------------------------------------------------------------------------------ loaders
    constexpr int kChunks = kDim / 8;               // 16-byte chunks per token
    constexpr int kWarpRows = 32 / kChunks;         // tokens per warp and copy
    constexpr int kLoadWarps = kLoadThreads / 32;
    constexpr int kIters = kTok / (kWarpRows * kLoadWarps);
    const int lw = warp - kSoftWarps - 1;
    const int chunk = lane % kChunks;
    const bool chunk_in = chunk * 8 < p.dim;
    // this lane looks up the page of one of the warp's tokens; shuffles hand it out
    const int my_row = (lane / kWarpRows) * (kWarpRows * kLoadWarps) + lw * kWarpRows + lane % kWarpRows;
    auto look_up = [&](int& id, int& at) {
      id = -1;
      at = 0;
      const int tok = cur.tile * kTok + my_row;
      if (my_row < kTok && tok < cur.len) {
        const int32_t* table = cur.seg ? p.pages + (int64_t)(cur.seg - 1) * p.pages_stride : p.prefix_pages;
        const int pg = tok / p.page_size;
        id = table[pg];
        at = tok - pg * p.page_size;
        if (id < 0 || id >= p.total_pages) id = -2;
      }
    };
    int id = -1, at = 0;
    if (!idle) look_up(id, at);
    for (int u = u_lo, i = 0; u < u_hi; ++u, ++i) {
      const int stage = i % kStages;
      const int head = cur.group / cur.blocks;
      const int tile_id = id, tile_at = at;
      const T* kc = static_cast<const T*>(p.k) + head * p.ks[2] + chunk * 8;
      const T* vc = static_cast<const T*>(p.v) + head * p.vs[2] + chunk * 8;
      cur.next(p, plan, kTok, kBlockRows);
      if (u + 1 < u_hi) look_up(id, at);  // its latency passes behind this tile's wait and copies
      bool ok = true;
      if (lane == 0) ok = mbar_wait(&c.empty[stage], ((i / kStages) & 1) ^ 1, s_abort);
      ok = __shfl_sync(~0u, ok, 0);
      if (!ok) break;
      if (tile_id == -2) c.bad_unit[stage] = u + 1;
      const uint32_t kb = ring + stage * stage_bytes + (chunk >> 3) * S::kSub;
#pragma unroll
      for (int j = 0; j < kIters; ++j) {
        const int src = j * kWarpRows + lane / kChunks;
        const int pid = __shfl_sync(~0u, tile_id, src), pat = __shfl_sync(~0u, tile_at, src);
        const int r = j * (kWarpRows * kLoadWarps) + lw * kWarpRows + lane / kChunks;
        const bool have = pid >= 0 && chunk_in;
        const T* ks = have ? kc + pid * p.ks[0] + pat * p.ks[1] : static_cast<const T*>(p.k);
        const T* vs = have ? vc + pid * p.vs[0] + pat * p.vs[1] : static_cast<const T*>(p.v);
        const uint32_t dst = kb + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
        cp_async16(dst, ks, have ? 16 : 0);
        cp_async16(dst + S::kHalf, vs, have ? 16 : 0);
      }
      cp_async_arrive(&c.full[stage]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.full[stage]);  // orders bad_unit before the stage is full
    }
    cp_async_wait_all();
  } else if (warp == kSoftWarps) {
    // ------------------------------------------------------------------------------ products
    if (lane == 0 && !idle) {
      constexpr uint32_t kIdescS = instr_desc<T>(kTok, false), kIdescO = instr_desc<T>(kDim, true);
      int pieces = 0;         // pieces whose second product has begun
      bool first[2] = {};     // tile i (by parity) opens its piece
      bool ok = true;
      auto second = [&](int i) {  // O += P V of tile i
        ok = ok && mbar_wait(&c.p_full[i & 1], (i >> 1) & 1, s_abort);
        if (first[i & 1]) {
          if (pieces > 0) ok = ok && mbar_wait(&c.o_free, (pieces - 1) & 1, s_abort);
          ++pieces;
        }
        if (!ok) return;
        tc_fence_after();
        const uint32_t vb = ring + (i % kStages) * stage_bytes + S::kHalf;
        const uint32_t pa = tmem + S::kS + (i & 1) * kTok;
#pragma unroll
        for (int ks = 0; ks < kTok / 16; ++ks)
          tc_mma(tmem, pa + ks * 8, smem_desc(vb + ks * 2048, S::kSub, 1024), kIdescO,
                 !(first[i & 1] && ks == 0));
        tc_commit(&c.empty[i % kStages]);
        tc_commit(&c.o_done[i & 1]);
      };
      int starts = 0;
      int n = 0;
      for (int u = u_lo; u < u_hi && ok; ++u, ++n) {
        const bool start = n == 0 || cur.tile == 0;
        // A new piece's queries arrive after the last weights of the old one: take those first.
        if (start && n > 0) second(n - 1);
        if (start) {
          ok = ok && mbar_wait(&c.q_full, starts & 1, s_abort);
          ++starts;
        }
        ok = ok && mbar_wait(&c.full[n % kStages], (n / kStages) & 1, s_abort);
        if (!ok) break;
        fence_proxy_async_smem();  // the copies wrote through the generic proxy
        tc_fence_after();
        const uint32_t kb = ring + (n % kStages) * stage_bytes;
        const uint32_t sd = tmem + S::kS + (n & 1) * kTok;
#pragma unroll
        for (int ks = 0; ks < kDim / 16; ++ks)
          tc_mma(sd, tmem + S::kQ + ks * 8, smem_desc(kb + (ks / 4) * S::kSub + (ks % 4) * 32, 16, 1024),
                 kIdescS, ks > 0);
        tc_commit(&c.s_full[n & 1]);
        if (!start) second(n - 1);
        first[n & 1] = start;
        cur.next(p, plan, kTok, kBlockRows);
      }
      if (ok && n > 0) second(n - 1);
      if (!ok) {  // let what is in flight land before the tensor memory is freed
        tc_commit(&c.drain);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_test(&c.drain, 0) && globaltimer_ns() - t0 < kPipeWaitNs) {
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------------------ softmax
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const uint32_t t_o = tmem + lanes, t_q = tmem + lanes + S::kQ;
    bool ok = !idle;
    // The rows of a piece and what they see.
    int rows_here = 0, base = 0, seen = 0;
    unsigned long long branch = 0;
    // Queries of the piece at the cursor into tensor memory.
    auto open_piece = [&] {
      const int head = cur.group / cur.blocks, block = cur.group - head * cur.blocks;
      rows_here = min(kBlockRows, cur.count * p.group - block * kBlockRows);
      base = cur.len - cur.count;
      const int f = block * kBlockRows + threadIdx.x;
      const bool act = (int)threadIdx.x < rows_here;
      const int local = act ? f / p.group : 0;
      const int t = cur.first + local;
      seen = !act ? 0x7fffffff : cur.seg == 0 ? cur.len : min(cur.len, base + local + 1);
      branch = 0;
      if (p.tree && cur.seg && act) {
        branch = (unsigned long long)p.tree[t];
        seen = min(cur.len, base);
      }
      if (warp * 32 < rows_here) {
        const T* src = static_cast<const T*>(p.q) + (int64_t)t * p.q_row +
                       (int64_t)(head * p.group + (act ? f - local * p.group : 0)) * p.q_head;
#pragma unroll
        for (int c0 = 0; c0 < kDim / 2; c0 += 32) {
          uint32_t w[32];
          if (p.q_vec) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int d = (c0 + 4 * j) * 2;
              uint4 v = make_uint4(0, 0, 0, 0);
              if (act && d < p.dim) v = *reinterpret_cast<const uint4*>(src + d);
              w[4 * j] = v.x, w[4 * j + 1] = v.y, w[4 * j + 2] = v.z, w[4 * j + 3] = v.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const int d = (c0 + j) * 2;
              w[j] = act && d < p.dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
            }
          }
          tmem_st32(t_q + c0, w);
        }
        tc_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.q_full);
    };
    if (ok) open_piece();
    // A barrier of the softmax warps whose wait is bounded like the others.
    int syncs = 0;
    auto sync_rows = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.sync);
      ok = mbar_wait(&c.sync, syncs++ & 1, s_abort) && ok;
      __syncwarp();
    };

    float m_ref = neg_inf(), l = 0.f;  // the maximum the weights refer to, and their sum
    bool piece_start = true;
    for (int u = u_lo, i = 0; u < u_hi && ok; ++u, ++i) {
      const int b = i & 1, stage = i % kStages;
      const bool act_warp = warp * 32 < rows_here;
      const uint32_t t_s = tmem + lanes + S::kS + b * kTok;
      const int tile0 = cur.tile * kTok;
      if (piece_start) {
        m_ref = neg_inf();
        l = 0.f;
      }
      ok = mbar_wait(&c.s_full[b], (i >> 1) & 1, s_abort);
      // already complete: S was computed from this stage. Makes its flags and values visible here.
      ok = ok && mbar_wait(&c.full[stage], (i / kStages) & 1, s_abort);
      if (!__all_sync(~0u, ok)) break;
      tc_fence_after();
      const bool bad_page = *const_cast<volatile int*>(&c.bad_unit[stage]) == u + 1;
      const int32_t* table = cur.seg ? p.pages + (int64_t)(cur.seg - 1) * p.pages_stride : p.prefix_pages;
      auto sees = [&](int tok) {
        bool see = tok < seen;
        if (!see && branch) {
          const int n = tok - base;
          see = n >= 0 && n < 64 && tok < cur.len && ((branch >> n) & 1);
        }
        if (see && bad_page) {
          const int id = table[tok / p.page_size];
          see = id >= 0 && id < p.total_pages;
        }
        return see;
      };
      // Some row of the block may not see a token of this tile (uniform over the block).
      const int sure = cur.seg == 0 ? cur.len : min(cur.len, p.tree ? base : base + 1);
      const bool masked = tile0 + kTok > sure || bad_page;
      if (act_warp) {
        // 64 scores at a time. Of a tile of 128 the second half is read twice: holding both would
        // cost the registers that the rest needs.
        uint32_t s[64];
        const bool plain = !masked && p.scale_log2 > 0.f;
        const float mul = plain ? p.scale_log2 : 1.f;
        auto scores = [&](int h) {
#pragma unroll
          for (int j = 0; j < 64; j += 32)
            tmem_ld32(*reinterpret_cast<uint32_t(*)[32]>(&s[j]), t_s + h * 64 + j);
          tc_wait_ld();
          if (!plain) {
#pragma unroll
            for (int j = 0; j < 64; ++j) {
              const float x = __uint_as_float(s[j]) * p.scale_log2;
              s[j] = __float_as_uint(!masked || sees(tile0 + h * 64 + j) ? x : neg_inf());
            }
            __syncwarp();
          }
        };
        float mx4[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
#pragma unroll
        for (int h = kTok / 64 - 1; h >= 0; --h) {
          scores(h);
#pragma unroll
          for (int j = 0; j < 64; ++j) mx4[j & 3] = fmaxf(mx4[j & 3], __uint_as_float(s[j]));
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * mul;
        const bool grow = mx > m_ref + 8.f || (m_ref == neg_inf() && mx > neg_inf());
        if (__any_sync(~0u, grow)) {
          const float f = grow ? ex2(m_ref - mx) : 1.f;
          if (grow) m_ref = mx;
          l *= f;
          if (!piece_start) {
            ok = mbar_wait(&c.o_done[b ^ 1], ((i - 1) >> 1) & 1, s_abort);
            tc_fence_after();
            __syncwarp();
#pragma unroll 1
            for (int c0 = 0; c0 < kDim; c0 += 32) {
              uint32_t w[32];
              tmem_ld32(w, t_o + c0);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(__uint_as_float(w[j]) * f);
              tmem_st32(t_o + c0, w);
            }
          }
        }
        const float ref = m_ref == neg_inf() ? 0.f : m_ref;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < kTok / 64; ++h) {
          if (h > 0) scores(h);
#pragma unroll
          for (int j = 0; j < 64; j += 2) {
            const float x = ex2(fmaf(__uint_as_float(s[j]), mul, -ref));
            const float y = ex2(fmaf(__uint_as_float(s[j + 1]), mul, -ref));
            sum[j & 2] += x;
            sum[(j & 2) + 1] += y;
            s[j / 2] = Pair<T>::pack(x, y);
          }
          // over scores that have been read: weights take half the columns
          tmem_st32(t_s + h * 32, *reinterpret_cast<const uint32_t(*)[32]>(&s[0]));
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tc_wait_st();
      }
      // A masked tile of a request's own tokens may hold infinities or NaN that some rows do not
      // see; 0 * NaN would carry them into those rows. They are replaced by zeros before the second
      // product, and added afterwards to the rows that see them.
      bool poisoned = false;
      if (masked && cur.seg) {
        uint8_t* vt = smem + stage * stage_bytes + S::kHalf;
        bool found = false;
        for (int x = threadIdx.x; x < S::kHalf / 16; x += kSoftWarps * 32) {
          const uint4 w = *reinterpret_cast<const uint4*>(vt + x * 16);
          found |= non_finite<T>(w.x) | non_finite<T>(w.y) | non_finite<T>(w.z) | non_finite<T>(w.w);
        }
        if (found) *const_cast<volatile int*>(&c.bad_value) = u + 1;
        sync_rows();
        poisoned = *const_cast<volatile int*>(&c.bad_value) == u + 1;
        if (poisoned) {
          for (int x = threadIdx.x; x < kTok; x += kSoftWarps * 32) c.bad_token[x] = 0;
          sync_rows();
          for (int x = threadIdx.x; x < S::kHalf / 16; x += kSoftWarps * 32) {
            uint4 w = *reinterpret_cast<const uint4*>(vt + x * 16);
            if (!(non_finite<T>(w.x) | non_finite<T>(w.y) | non_finite<T>(w.z) | non_finite<T>(w.w))) continue;
            *const_cast<volatile unsigned char*>(&c.bad_token[(x / 8) % kTok]) = 1;
            w = make_uint4(finite_or_zero<T>(w.x), finite_or_zero<T>(w.y), finite_or_zero<T>(w.z),
                           finite_or_zero<T>(w.w));
            *reinterpret_cast<uint4*>(vt + x * 16) = w;
          }
          fence_proxy_async_smem();
          sync_rows();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.p_full[b]);
      if (poisoned) {
        ok = ok && mbar_wait(&c.o_done[b], (i >> 1) & 1, s_abort);
        tc_fence_after();
        __syncwarp();
        const int head = cur.group / cur.blocks;
        for (int x = 0; x < kTok && act_warp; ++x) {
          if (!*const_cast<volatile unsigned char*>(&c.bad_token[x])) continue;
          const int tok = tile0 + x, pg = tok / p.page_size;
          const bool see = (int)threadIdx.x < rows_here && sees(tok);
          const T* v = static_cast<const T*>(p.v) + table[pg] * p.vs[0] +
                       (tok - pg * p.page_size) * p.vs[1] + head * p.vs[2];
#pragma unroll 1
          for (int c0 = 0; c0 < kDim; c0 += 32) {
            uint32_t w[32];
            tmem_ld32(w, t_o + c0);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (c0 + j >= p.dim || !see) continue;
              const float y = (float)v[c0 + j];
              if (!isfinite(y)) w[j] = __float_as_uint(__uint_as_float(w[j]) + y);
            }
            tmem_st32(t_o + c0, w);
          }
          tc_wait_st();
        }
        tc_fence_before();
        sync_rows();  // bad_token is free again
      }

      const bool piece_end = cur.tile + 1 == cur.tiles || u + 1 == u_hi;
      piece_start = piece_end;
      if (!piece_end) {
        ++cur.tile;
        continue;
      }
      // ---- end of a piece: the next one's queries first, then O out
      const int slot = (int)blockIdx.x + (cur.seg ? plan.groups_end[cur.seg - 1] : 0) + cur.group;
      const int done_rows = rows_here;
      cur.next(p, plan, kTok, kBlockRows);
      if (u + 1 < u_hi) open_piece();
      ok = ok && mbar_wait(&c.o_done[b], (i >> 1) & 1, s_abort);
      tc_fence_after();
      __syncwarp();
      if (warp * 32 < done_rows) {
        const bool act = (int)threadIdx.x < done_rows && slot >= 0 && slot < p.slots;
        const int64_t at = (int64_t)slot * kBlockRows + threadIdx.x;
        float* dst = p.part_o + at * p.dim;
#pragma unroll 1
        for (int c0 = 0; c0 < p.dim; c0 += 32) {
          uint32_t w[32];
          tmem_ld32(w, t_o + c0);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            if (act && c0 + j < p.dim)
              *reinterpret_cast<uint4*>(dst + c0 + j) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
        }
        if (act) p.part_ml[at] = make_float2(m_ref, l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.o_free);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftWarps) {
    __syncwarp();
    tc_fence_after();
    tmem_free(tmem, S::kColumns);
  }
  if (threadIdx.x == 0 && *s_abort) atomicCAS(&g_attn_status, 0, B2_ERR_TIMEOUT);
}

// ------------------------------------------------------------------------------------------------
// Join: one block per (row, query head). The row's partials are those of its prefix group and of
// its request's own group, each from a run of CTAs; they are added in that order.
// ------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttnArgs p, int tok, int grid) {
  constexpr int block_rows = kBlockRows;
  __shared__ Plan plan;
  __shared__ int s_seg;
  const int t = blockIdx.x / p.q_heads, h = blockIdx.x - t * p.q_heads;
  grid_dep_wait();
  grid_dep_launch();
  make_plan<kJoinThreads / 32>(p, tok, block_rows, plan);
  if (threadIdx.x == 0) {
    int seg = -1;
    for (int b = 0; b < p.requests; ++b) {
      int first, count;
      request_rows(p, b, first, count);
      if (t >= first && t < first + count) {
        seg = b + 1;
        break;
      }
    }
    s_seg = seg;
  }
  __syncthreads();
  const int seg = s_seg, units = plan.units_end[p.requests];
  const int ctas = units > 0 ? plan_ctas(units, grid) : 1;
  const int head = h / p.group, g = h - head * p.group;
  // the two runs of pieces: slots from[i] + 0 .. n[i] - 1, row[i] in each
  int from[2], n[2], row[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    n[i] = from[i] = row[i] = 0;
    if (seg < 0) continue;
    const int s = i == 0 ? 0 : seg;
    int first, count, len, tiles, blocks;
    segment_shape(p, s, tok, block_rows, first, count, len, tiles, blocks);
    if (tiles == 0 || units == 0) continue;
    const int f = (t - first) * p.group + g;
    const int group = head * blocks + f / block_rows;
    row[i] = f % block_rows;
    const int u0 = (s ? plan.units_end[s - 1] : 0) + group * tiles;
    const int c0 = plan_owner(units, ctas, u0), c1 = plan_owner(units, ctas, u0 + tiles - 1);
    from[i] = c0 + (s ? plan.groups_end[s - 1] : 0) + group;
    n[i] = min(c1 - c0 + 1, max(0, p.slots - from[i]));
  }
  float top = neg_inf();
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < n[i]; ++j)
      top = fmaxf(top, p.part_ml[(int64_t)(from[i] + j) * block_rows + row[i]].x);
  const float safe = top == neg_inf() ? 0.f : top;
  float sum = 0.f, acc[2] = {0.f, 0.f};
  const int d0 = threadIdx.x, d1 = threadIdx.x + kJoinThreads;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < n[i]; ++j) {
      const int64_t at = (int64_t)(from[i] + j) * block_rows + row[i];
      const float2 ml = p.part_ml[at];
      const float w = ex2(ml.x - safe);
      sum += ml.y * w;
      if (d0 < p.dim) acc[0] += p.part_o[at * p.dim + d0] * w;
      if (d1 < p.dim) acc[1] += p.part_o[at * p.dim + d1] * w;
    }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  T* out = static_cast<T*>(p.out) + ((int64_t)t * p.q_heads + h) * p.dim;
  if (d0 < p.dim) out[d0] = T(acc[0] * inv);
  if (d1 < p.dim) out[d1] = T(acc[1] * inv);
  if (threadIdx.x == 0)
    p.lse[(int64_t)t * p.q_heads + h] = sum == 0.f ? neg_inf() : (top + log2f(sum)) * kLn2;
}

int round_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
int64_t slots_for(int requests, int rows, int group, int kv_heads) {
  const int64_t blocks = ((int64_t)rows * group + kBlockRows - 1) / kBlockRows;
  return kMaxCtas + kv_heads * (2 * blocks + requests);
}

template <typename T, int kDim>
int launch_typed(const AttnArgs& p, int ctas, cudaStream_t stream) {
  constexpr size_t smem = attn_smem<kDim>();
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  auto kernel = attn_kernel<T, kDim>;
  static bool configured[64] = {};
  int dev = 0;
  B2_CUDA_TRY(cudaGetDevice(&dev));
  if (!configured[dev]) {
    B2_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured[dev] = true;
  }
  int rc = launch_kernel(kernel, ctas, kAttnThreads, smem, stream, /*early=*/true, p);
  if (rc) return rc;
  return launch_kernel(join_kernel<T>, p.rows * p.q_heads, kJoinThreads, 0, stream, /*early=*/true,
                       p, Shape<kDim>::kTok, ctas);
}

template <typename T>
int launch_dim(const AttnArgs& p, int ctas, cudaStream_t stream) {
  switch (round_dim(p.dim)) {
    case 64: return launch_typed<T, 64>(p, ctas, stream);
    case 128: return launch_typed<T, 128>(p, ctas, stream);
    default: return launch_typed<T, 256>(p, ctas, stream);
  }
}

int check_shape(int requests, int rows, int q_heads, int kv_heads, int head_dim) {
  const char* op = "prefix_attn";
  if (requests < 0 || requests > kMaxRequests)
    return fail(B2_ERR_INVALID_ARG, "%s: %d requests (at most %d)", op, requests, kMaxRequests);
  if (rows < 0 || rows > kMaxRows)
    return fail(B2_ERR_INVALID_ARG, "%s: %d rows (at most %d)", op, rows, kMaxRows);
  if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0 || q_heads > 1024)
    return fail(B2_ERR_INVALID_ARG, "%s: %d query heads on %d KV heads", op, q_heads, kv_heads);
  if (head_dim < 8 || head_dim > 256 || head_dim % 8 != 0)
    return fail(B2_ERR_INVALID_ARG, "%s: head_dim=%d must be a multiple of 8 up to 256", op, head_dim);
  return B2_OK;
}

}  // namespace
}  // namespace b2

extern "C" size_t b2_prefix_attn_workspace(int requests, int rows, int q_heads, int kv_heads,
                                           int head_dim) {
  using namespace b2;
  if (check_shape(requests, rows, q_heads, kv_heads, head_dim)) return 0;
  const int64_t slots = slots_for(requests, rows, q_heads / kv_heads, kv_heads);
  return (size_t)slots * kBlockRows * (head_dim * sizeof(float) + sizeof(float2)) + 256;
}

extern "C" int b2_prefix_attn(const void* q, const int64_t* q_strides, const void* k_cache,
                              const int64_t* k_strides, const void* v_cache,
                              const int64_t* v_strides, int total_pages, int page_size,
                              const int32_t* prefix_pages, int n_prefix_pages,
                              const int32_t* prefix_len, const int32_t* pages, int64_t pages_stride,
                              int max_pages, const int32_t* own_lens, const int32_t* row_start,
                              const int64_t* tree, int requests, int rows, int q_heads,
                              int kv_heads, int head_dim, float scale, int dtype, void* out,
                              float* lse, void* ws, size_t ws_bytes, void* stream) {
  using namespace b2;
  const char* op = "prefix_attn";
  int rc = check_shape(requests, rows, q_heads, kv_heads, head_dim);
  if (rc) return rc;
  if (dtype != B2_DTYPE_F16 && dtype != B2_DTYPE_BF16)
    return fail(B2_ERR_INVALID_ARG, "%s: dtype %d", op, dtype);
  if (total_pages < 0 || page_size < 1 || n_prefix_pages < 0 || max_pages < 0)
    return fail(B2_ERR_INVALID_ARG, "%s: %d pages of %d tokens, tables of %d and %d", op, total_pages,
                page_size, n_prefix_pages, max_pages);
  if (!(scale == scale) || scale - scale != 0.f)
    return fail(B2_ERR_INVALID_ARG, "%s: scale is not finite", op);
  if (rows == 0) return B2_OK;
  if (!q_strides || !k_strides || !v_strides || !q || !k_cache || !v_cache || !prefix_len ||
      (requests > 0 && !own_lens) || !row_start || !out || !lse || (n_prefix_pages > 0 && !prefix_pages) ||
      (max_pages > 0 && !pages))
    return fail(B2_ERR_INVALID_ARG, "%s: null pointer", op);
  if ((int64_t)n_prefix_pages * page_size > 0x7ffffff0 || (int64_t)max_pages * page_size > 0x7ffffff0)
    return fail(B2_ERR_INVALID_ARG, "%s: tables of more than 2^31 tokens", op);
  if (!aligned16(k_cache) || !aligned16(v_cache) || (reinterpret_cast<uintptr_t>(q) & 3u) != 0)
    return fail(B2_ERR_INVALID_ARG, "%s: caches must be 16-byte and q 4-byte aligned", op);
  if (q_strides[0] % 2 != 0 || q_strides[1] % 2 != 0)
    return fail(B2_ERR_INVALID_ARG, "%s: strides of q must be even", op);
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
      return fail(B2_ERR_INVALID_ARG, "%s: cache strides must be multiples of 8 elements", op);
  const size_t need = b2_prefix_attn_workspace(requests, rows, q_heads, kv_heads, head_dim);
  if (!ws || ws_bytes < need || !aligned16(ws))
    return fail(B2_ERR_WORKSPACE, "%s: workspace of %zu B, need %zu B", op, ws_bytes, need);
  const int group = q_heads / kv_heads;
  const int tok = round_dim(head_dim) == 64 ? 128 : 64;
  // units are counted in 32 bits
  const int64_t blocks = ((int64_t)rows * group + kBlockRows - 1) / kBlockRows;
  const int64_t tiles = ((int64_t)std::max(n_prefix_pages, max_pages) * page_size + tok - 1) / tok;
  if ((2 * blocks + requests) * kv_heads * tiles > 0x7fffffff)
    return fail(B2_ERR_INVALID_ARG, "%s: tables too long for %d rows", op, rows);
  DeviceInfo di;
  rc = device_info(&di);
  if (rc) return rc;
  const int ctas = std::min(di.sm_count, kMaxCtas);
  AttnArgs p = {};
  p.q = q, p.k = k_cache, p.v = v_cache;
  p.q_row = q_strides[0], p.q_head = q_strides[1];
  for (int i = 0; i < 3; ++i) p.ks[i] = k_strides[i], p.vs[i] = v_strides[i];
  p.prefix_pages = prefix_pages, p.prefix_len = prefix_len, p.pages = pages, p.own_lens = own_lens;
  p.row_start = row_start, p.tree = tree;
  p.out = out, p.lse = lse;
  p.q_vec = aligned16(q) && q_strides[0] % 8 == 0 && q_strides[1] % 8 == 0;
  p.pages_stride = pages_stride;
  p.total_pages = total_pages, p.page_size = page_size;
  p.n_prefix_pages = n_prefix_pages, p.max_pages = max_pages;
  p.requests = requests, p.rows = rows, p.q_heads = q_heads, p.kv_heads = kv_heads, p.group = group;
  p.dim = head_dim;
  p.slots = (int)slots_for(requests, rows, group, kv_heads);
  p.scale_log2 = scale * kLog2e;
  p.part_ml = static_cast<float2*>(ws);
  const size_t ml_bytes = ((size_t)p.slots * kBlockRows * sizeof(float2) + 255) & ~(size_t)255;
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + ml_bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == B2_DTYPE_F16 ? launch_dim<__half>(p, ctas, s)
                               : launch_dim<__nv_bfloat16>(p, ctas, s);
}
