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
constexpr int kAttnWarps = 8;
constexpr int kAttnThreads = kAttnWarps * 32;
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
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    mma_16816(c, a[0], a[1], a[2], a[3], b0, b1);
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static constexpr uint32_t kExp = 0x7f80u;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes from global to shared memory; `bytes` = 16, or 0 to write zeros without reading.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------------------------------------
// The plan: every block derives it from the lengths on the device.
// ------------------------------------------------------------------------------------------------
struct Plan {
  int units_end[kMaxRequests + 1];   // running sum of units up to and with segment s
  int groups_end[kMaxRequests + 1];  // running sum of groups
  int warp_sum[2][kAttnWarps];
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
// Main kernel. kDim: head dimension rounded up (64, 128, 256). kRowWarps groups of 16 rows; the
// other kAttnWarps / kRowWarps warps split a tile's tokens, each with its own running maximum and
// sum, and are joined at the end of a piece.
// ------------------------------------------------------------------------------------------------
template <int kDim>
struct Shape {
  static constexpr int kTok = kDim == 64 ? 128 : 64;  // tokens per tile
  static constexpr int kStages = kDim == 256 ? 3 : 6;
  static constexpr int kHalfBytes = kTok * kDim * 2;  // K or V of a stage
  static constexpr int kRing = kStages * 2 * kHalfBytes;
  static constexpr int kJoinCols = 32;  // columns of O joined per round
};

template <int kDim, int kRowWarps>
constexpr size_t attn_smem() {
  return Shape<kDim>::kRing +
         sizeof(float) * ((kAttnWarps / kRowWarps) * kRowWarps * 16 * (Shape<kDim>::kJoinCols + 4)) +
         sizeof(float2) * kAttnWarps * 16 + sizeof(Plan) + 64;
}

template <typename T, int kDim, int kRowWarps>
__global__ void __launch_bounds__(kAttnThreads, 1) attn_kernel(const AttnArgs p) {
  using S = Shape<kDim>;
  constexpr int kTok = S::kTok, kStages = S::kStages;
  constexpr int kTokWarps = kAttnWarps / kRowWarps;
  constexpr int kWarpTok = kTok / kTokWarps;  // tokens of a tile per warp
  constexpr int kBlockRows = kRowWarps * 16;
  constexpr int kChunks = kDim / 8;           // 16-byte chunks per token
  constexpr int kCols = S::kJoinCols;
  static_assert(kWarpTok % 16 == 0, "a warp takes whole k-steps of the second product");

  extern __shared__ __align__(128) uint8_t smem[];
  float* s_join = reinterpret_cast<float*>(smem + S::kRing);  // [tokwarp][row][kCols + 4]
  float2* s_ml = reinterpret_cast<float2*>(s_join + kTokWarps * kBlockRows * (kCols + 4));
  Plan& plan = *reinterpret_cast<Plan*>(s_ml + kAttnWarps * 16);
  // per stage: 1 + the unit, if any, for which a page id outside the cache was met there
  volatile int* s_bad = reinterpret_cast<volatile int*>(&plan + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rw = warp % kRowWarps, tw = warp / kRowWarps;
  grid_dep_wait();
  grid_dep_launch();
  make_plan<kAttnWarps>(p, kTok, kBlockRows, plan);
  const int units = plan.units_end[p.requests];
  if (units == 0) return;
  const int ctas = plan_ctas(units, gridDim.x);
  if ((int)blockIdx.x >= ctas) return;
  const int u_lo = plan_begin(units, ctas, blockIdx.x), u_hi = plan_begin(units, ctas, blockIdx.x + 1);

  const uint32_t ring = smem_u32(smem);
  const T* kc = static_cast<const T*>(p.k);
  const T* vc = static_cast<const T*>(p.v);

  // ---- loads: this thread's chunk column and rows of every tile
  Cursor lc;
  lc.seek(p, plan, u_lo, kTok, kBlockRows);
  int lu = u_lo;
  const int chunk = threadIdx.x % kChunks;
  const bool chunk_in = chunk * 8 < p.dim;
  auto fill = [&](int stage) {
    if (lu < u_hi) {
      const int head = lc.group / lc.blocks;
      const int32_t* table = lc.seg ? p.pages + (int64_t)(lc.seg - 1) * p.pages_stride : p.prefix_pages;
      const uint32_t kb = ring + stage * 2 * S::kHalfBytes, vb = kb + S::kHalfBytes;
#pragma unroll
      for (int i = 0; i < kTok / (kAttnThreads / kChunks); ++i) {
        const int r = threadIdx.x / kChunks + i * (kAttnThreads / kChunks);
        const int tok = lc.tile * kTok + r;
        const T *ks = kc, *vs = vc;
        int bytes = 0;
        if (tok < lc.len) {
          const int pg = tok / p.page_size;
          const int id = table[pg];
          if (id >= 0 && id < p.total_pages) {
            const int at = tok - pg * p.page_size;
            ks = kc + id * p.ks[0] + at * p.ks[1] + head * p.ks[2] + chunk * 8;
            vs = vc + id * p.vs[0] + at * p.vs[1] + head * p.vs[2] + chunk * 8;
            bytes = chunk_in ? 16 : 0;
          } else {
            s_bad[stage] = lu + 1;
          }
        }
        if (!bytes) ks = kc, vs = vc;
        const uint32_t off = r * (kDim * 2) + ((chunk ^ (r & 7)) << 4);
        cp_async16(kb + off, ks, bytes);
        cp_async16(vb + off, vs, bytes);
      }
      lc.next(p, plan, kTok, kBlockRows);
      ++lu;
    }
    cp_async_commit();
  };
  if (threadIdx.x < kStages) s_bad[threadIdx.x] = 0;
  __syncthreads();  // the flags are cleared before a fill sets one
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) fill(s);

  // ---- compute
  Cursor cc;
  cc.seek(p, plan, u_lo, kTok, kBlockRows);
  const int g4 = lane >> 2, t4 = lane & 3;
  uint32_t qf[kDim / 16][4];
  float o[kDim / 8][4];
  float m[2] = {}, l[2] = {};
  int seen[2] = {};             // tokens of the segment the lane's two rows see
  unsigned long long branch[2] = {};
  int base = 0;                 // first new token of the request
  bool piece_start = true;
  int stage = 0;

  for (int u = u_lo; u < u_hi; ++u) {
    const int head = cc.group / cc.blocks, block = cc.group - head * cc.blocks;
    const int row_lim = cc.count * p.group;  // rows of the segment
    const int my_rows = row_lim - block * kBlockRows - rw * 16;  // of this warp's 16
    if (piece_start) {
#pragma unroll
      for (int j = 0; j < kDim / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
      base = cc.len - cc.count;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[e] = neg_inf();
        l[e] = 0.f;
        const int r = g4 + 8 * e;
        const int f = block * kBlockRows + rw * 16 + r;
        const bool act = r < my_rows;
        const int local = act ? f / p.group : 0;
        const int t = cc.first + local;
        const T* src = static_cast<const T*>(p.q) + t * p.q_row +
                       (int64_t)(head * p.group + (act ? f - local * p.group : 0)) * p.q_head;
        seen[e] = !act ? 0x7fffffff : cc.seg == 0 ? cc.len : min(cc.len, base + local + 1);
        branch[e] = 0;
        if (p.tree && cc.seg && act) {
          branch[e] = (unsigned long long)p.tree[t];
          seen[e] = min(cc.len, base);
        }
#pragma unroll
        for (int ks = 0; ks < kDim / 16; ++ks) {
          const int d = ks * 16 + t4 * 2;
          qf[ks][e] = act && d < p.dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
          qf[ks][2 + e] = act && d + 8 < p.dim ? *reinterpret_cast<const uint32_t*>(src + d + 8) : 0u;
        }
      }
      piece_start = false;
    }

    cp_async_wait<kStages - 2>();
    __syncthreads();
    fill(stage == 0 ? kStages - 1 : stage - 1);  // the stage that every warp has left behind

    if (my_rows > 0) {
      const uint32_t kb = ring + stage * 2 * S::kHalfBytes, vb = kb + S::kHalfBytes;
      const int tok0 = tw * kWarpTok;
      float s[kWarpTok / 8][4];
#pragma unroll
      for (int j = 0; j < kWarpTok / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
      // S = Q K^T. One ldmatrix.x4 = two 8-token groups x two 8-element chunks.
      const int lr = (lane & 7) + ((lane >> 4) << 3), lch = (lane >> 3) & 1;
#pragma unroll
      for (int ks = 0; ks < kDim / 16; ++ks) {
#pragma unroll
        for (int j = 0; j < kWarpTok / 16; ++j) {
          const int r = tok0 + j * 16 + lr;
          uint32_t b[4];
          ldsm4(b, kb + r * (kDim * 2) + (((ks * 2 + lch) ^ (r & 7)) << 4));
          Pair<T>::mma(s[2 * j], qf[ks], b[0], b[1]);
          Pair<T>::mma(s[2 * j + 1], qf[ks], b[2], b[3]);
        }
      }
      const int tile0 = cc.tile * kTok;
      const bool masked = tile0 + kTok > min(seen[0], seen[1]) || s_bad[stage] == u + 1;
#pragma unroll
      for (int j = 0; j < kWarpTok / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] *= p.scale_log2;
      const int32_t* table = cc.seg ? p.pages + (int64_t)(cc.seg - 1) * p.pages_stride : p.prefix_pages;
      auto sees = [&](int e, int tok) {
        bool see = tok < seen[e];
        if (!see && branch[e]) {
          const int n = tok - base;
          see = n >= 0 && n < 64 && tok < cc.len && ((branch[e] >> n) & 1);
        }
        if (see && s_bad[stage] == u + 1) {
          const int id = table[tok / p.page_size];
          see = id >= 0 && id < p.total_pages;
        }
        return see;
      };
      bool bad_v = false;  // a masked tile holds values that are no numbers
      if (__any_sync(~0u, masked)) {
#pragma unroll
        for (int j = 0; j < kWarpTok / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!sees(e >> 1, tile0 + tok0 + j * 8 + t4 * 2 + (e & 1))) s[j][e] = neg_inf();
        for (int i = lane; i < kWarpTok * kChunks; i += 32) {
          const uint4 w = lds128(vb + tok0 * (kDim * 2) + i * 16);
          bad_v |= non_finite<T>(w.x) | non_finite<T>(w.y) | non_finite<T>(w.z) | non_finite<T>(w.w);
        }
        bad_v = __any_sync(~0u, bad_v);
      }
      float mx[2] = {neg_inf(), neg_inf()};
#pragma unroll
      for (int j = 0; j < kWarpTok / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
      float corr[2], ms[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(~0u, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(~0u, mx[e], 2));
        const float nm = fmaxf(m[e], mx[e]);
        ms[e] = nm == neg_inf() ? 0.f : nm;
        corr[e] = ex2(m[e] - ms[e]);
        m[e] = nm;
        l[e] *= corr[e];
      }
#pragma unroll
      for (int j = 0; j < kWarpTok / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[j][e] = ex2(s[j][e] - ms[e >> 1]);
          l[e >> 1] += s[j][e];
        }
#pragma unroll
      for (int j = 0; j < kDim / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= corr[e >> 1];
      // O += P V. P is rounded to the cache's type for the tensor cores; its sum l is not.
      auto weigh = [&](auto clean) {
#pragma unroll
        for (int kt = 0; kt < kWarpTok / 16; ++kt) {
          const uint32_t a[4] = {Pair<T>::pack(s[2 * kt][0], s[2 * kt][1]),
                                 Pair<T>::pack(s[2 * kt][2], s[2 * kt][3]),
                                 Pair<T>::pack(s[2 * kt + 1][0], s[2 * kt + 1][1]),
                                 Pair<T>::pack(s[2 * kt + 1][2], s[2 * kt + 1][3])};
          const int r = tok0 + kt * 16 + (lane & 15);
          const uint32_t rb = vb + r * (kDim * 2);
#pragma unroll
          for (int j = 0; j < kDim / 16; ++j) {
            uint32_t b[4];
            ldsm4_t(b, rb + (((2 * j + (lane >> 4)) ^ (r & 7)) << 4));
            if constexpr (decltype(clean)::value) {
#pragma unroll
              for (int i = 0; i < 4; ++i) b[i] = finite_or_zero<T>(b[i]);
            }
            Pair<T>::mma(o[2 * j], a, b[0], b[1]);
            Pair<T>::mma(o[2 * j + 1], a, b[2], b[3]);
          }
        }
      };
      if (!bad_v) {
        weigh(std::false_type{});
      } else {
        // 0 * NaN would reach rows that do not see the token: the product runs on the numbers, and
        // what is none is added to the rows that see it (whose result it makes inf or NaN).
        weigh(std::true_type{});
        for (int r = tok0; r < tok0 + kWarpTok; ++r) {
          const bool s0 = sees(0, tile0 + r), s1 = sees(1, tile0 + r);
#pragma unroll
          for (int j = 0; j < kDim / 8; ++j) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(
                smem + stage * 2 * S::kHalfBytes + S::kHalfBytes + r * (kDim * 2) +
                ((j ^ (r & 7)) << 4) + t4 * 4);
            if (!non_finite<T>(w)) continue;
            const float2 v = unpack2<T>(w);
            if (!isfinite(v.x)) {
              if (s0) o[j][0] += v.x;
              if (s1) o[j][2] += v.x;
            }
            if (!isfinite(v.y)) {
              if (s0) o[j][1] += v.y;
              if (s1) o[j][3] += v.y;
            }
          }
        }
      }
    }

    // ---- end of a piece: join the token warps and write the partial
    const bool piece_end = cc.tile + 1 == cc.tiles || u + 1 == u_hi;
    if (piece_end) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(~0u, l[e], 1);
        l[e] += __shfl_xor_sync(~0u, l[e], 2);
      }
      if (t4 == 0) {
        s_ml[tw * kBlockRows + rw * 16 + g4] = make_float2(m[0], l[0]);
        s_ml[tw * kBlockRows + rw * 16 + g4 + 8] = make_float2(m[1], l[1]);
      }
      __syncthreads();
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = neg_inf();
#pragma unroll
        for (int w = 0; w < kTokWarps; ++w)
          top = fmaxf(top, s_ml[w * kBlockRows + rw * 16 + g4 + 8 * e].x);
        f[e] = ex2(m[e] - (top == neg_inf() ? 0.f : top));
      }
      const int slot = (int)blockIdx.x + (cc.seg ? plan.groups_end[cc.seg - 1] : 0) + cc.group;
      const int rows_here = min(kBlockRows, row_lim - block * kBlockRows);
      const bool room = slot >= 0 && slot < p.slots;
      if (room && (int)threadIdx.x < rows_here) {
        float top = neg_inf(), sum = 0.f;
        for (int w = 0; w < kTokWarps; ++w) top = fmaxf(top, s_ml[w * kBlockRows + threadIdx.x].x);
        const float safe = top == neg_inf() ? 0.f : top;
        for (int w = 0; w < kTokWarps; ++w) {
          const float2 ml = s_ml[w * kBlockRows + threadIdx.x];
          sum += ml.y * ex2(ml.x - safe);
        }
        p.part_ml[(int64_t)slot * kBlockRows + threadIdx.x] = make_float2(top, sum);
      }
      float* dst = p.part_o + (int64_t)slot * kBlockRows * p.dim;
#pragma unroll
      for (int c0 = 0; c0 < kDim; c0 += kCols) {
        if (c0 < p.dim) {
#pragma unroll
          for (int j = 0; j < kCols / 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float* to = s_join + (tw * kBlockRows + rw * 16 + g4 + 8 * e) * (kCols + 4) + j * 8 + t4 * 2;
              to[0] = o[c0 / 8 + j][2 * e] * f[e];
              to[1] = o[c0 / 8 + j][2 * e + 1] * f[e];
            }
        }
        __syncthreads();
        if (c0 < p.dim && room) {
          for (int i = threadIdx.x; i < rows_here * (kCols / 4); i += kAttnThreads) {
            const int r = i / (kCols / 4), c = (i % (kCols / 4)) * 4;
            if (c0 + c >= p.dim) continue;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kTokWarps; ++w) {
              const float4 x = *reinterpret_cast<const float4*>(
                  s_join + (w * kBlockRows + r) * (kCols + 4) + c);
              v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
            *reinterpret_cast<float4*>(dst + (int64_t)r * p.dim + c0 + c) = v;
          }
        }
        __syncthreads();
      }
      piece_start = true;
    }
    cc.next(p, plan, kTok, kBlockRows);
    if (++stage == kStages) stage = 0;
  }
  cp_async_wait<0>();
}

// ------------------------------------------------------------------------------------------------
// Join: one block per (row, query head). The row's partials are those of its prefix group and of
// its request's own group, each from a run of CTAs; they are added in that order.
// ------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttnArgs p, int tok, int block_rows,
                                                            int grid) {
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
// Rows of a block: 32 where no group has more, else 64.
int block_rows_for(int rows, int group) { return (int64_t)rows * group <= 32 ? 32 : 64; }
int64_t slots_for(int requests, int rows, int group, int kv_heads, int block_rows, int ctas) {
  const int64_t blocks = ((int64_t)rows * group + block_rows - 1) / block_rows;
  return ctas + kv_heads * (2 * blocks + requests);
}

template <typename T, int kDim, int kRowWarps>
int launch_typed(const AttnArgs& p, int ctas, cudaStream_t stream) {
  constexpr size_t smem = attn_smem<kDim, kRowWarps>();
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  auto kernel = attn_kernel<T, kDim, kRowWarps>;
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
                       p, Shape<kDim>::kTok, kRowWarps * 16, ctas);
}

template <typename T>
int launch_dim(const AttnArgs& p, int block_rows, int ctas, cudaStream_t stream) {
  switch (round_dim(p.dim) + block_rows) {
    case 64 + 32: return launch_typed<T, 64, 2>(p, ctas, stream);
    case 64 + 64: return launch_typed<T, 64, 4>(p, ctas, stream);
    case 128 + 32: return launch_typed<T, 128, 2>(p, ctas, stream);
    case 128 + 64: return launch_typed<T, 128, 4>(p, ctas, stream);
    case 256 + 32: return launch_typed<T, 256, 2>(p, ctas, stream);
    default: return launch_typed<T, 256, 4>(p, ctas, stream);
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
  const int group = q_heads / kv_heads, br = block_rows_for(rows, group);
  const int64_t slots = slots_for(requests, rows, group, kv_heads, br, kMaxCtas);
  return (size_t)slots * br * (head_dim * sizeof(float) + sizeof(float2)) + 256;
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
  const int group = q_heads / kv_heads, br = block_rows_for(rows, group);
  const int tok = round_dim(head_dim) == 64 ? 128 : 64;
  // units are counted in 32 bits
  const int64_t blocks = ((int64_t)rows * group + br - 1) / br;
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
  p.pages_stride = pages_stride;
  p.total_pages = total_pages, p.page_size = page_size;
  p.n_prefix_pages = n_prefix_pages, p.max_pages = max_pages;
  p.requests = requests, p.rows = rows, p.q_heads = q_heads, p.kv_heads = kv_heads, p.group = group;
  p.dim = head_dim;
  p.slots = (int)slots_for(requests, rows, group, kv_heads, br, kMaxCtas);
  p.scale_log2 = scale * kLog2e;
  p.part_ml = static_cast<float2*>(ws);
  const size_t ml_bytes = ((size_t)p.slots * br * sizeof(float2) + 255) & ~(size_t)255;
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + ml_bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == B2_DTYPE_F16 ? launch_dim<__half>(p, br, ctas, s)
                               : launch_dim<__nv_bfloat16>(p, br, ctas, s);
}
