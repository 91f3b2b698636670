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
// is read once for all of them (up to 256; beyond, once per 256), and n_b*G for a request's own
// tokens. A persistent grid takes equal contiguous ranges of work, counted in tiles of kTok tokens
// for one group of rows and one KV head over all segments (segment 0 = the prefix, segment b+1 =
// request b's own tokens), whatever the lengths on the device say, so a captured graph follows
// growing lengths. A range's piece of one (segment, head, rows) group ends in unnormalised fp32
// partials (O, m, l) in the workspace; a second launch joins the partials of each row in a fixed order,
// so results do not depend on timing. The partials of CTA c's piece of group g begin at row
// (rows of all groups before g) + c * (rows of the largest group): from one piece to the next the
// group, the CTA or both go up by one, so no two pieces share a row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "b2_device.cuh"
#include "b2_internal.h"

namespace b2 {
namespace {

constexpr int kMaxRequests = 1024;
constexpr int kMaxRows = 4096;
constexpr int kMaxTokens = 0x7fffff00;  // a tile that begins below it ends below 2^31
constexpr int kLoadThreads = 128;
constexpr int kBlockRows = 128;  // rows of one product: the lanes of tensor memory
constexpr unsigned int kMaxPolls = 1u << 20;  // of two barriers in turn, before the wait with a clock
constexpr int kMaxCtas = 160;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Where the partials of a row are: written by the main launch, read by the one that joins them.
struct RowPlan {
  int cost;                                       // of the whole call
  int prefix_tiles, prefix_first, prefix_count, prefix_span;  // of the prefix
  int tiles, first, count, span;                  // of the row's request; tiles = 0: none
  int cost0, rows0;                               // cost and rows of partials before the request's
  int owned;                                      // the row belongs to a request
  int even;                                       // every tile costs the same (Cost)
};

struct AttnArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head;
  int64_t ks[3], vs[3];  // page, token, head strides of the caches in elements
  const int32_t *prefix_pages, *prefix_len, *pages, *own_lens, *row_start;
  const int64_t* tree;
  void* out;
  float* lse;
  float* part_o;    // [part_rows][dim]
  float2* part_ml;  // [part_rows]
  RowPlan* row_plan;  // [rows]
  int64_t pages_stride;
  int total_pages, page_size, n_prefix_pages, max_pages;
  int requests, rows, q_heads, kv_heads, group, dim;
  int part_rows, piece_rows;  // rows of partials, of the largest piece
  int q_vec;     // queries allow 16-byte loads
  int box_rows;  // tokens per TMA box: a power of two that divides the page size
  FastDiv by_page, by_group;
  float scale_log2;
  uint64_t minus_zero;  // two of them: a * b + -0 is a rounded product that no sum is fused with
};

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 numbers in 64 bits, and operations on both at once.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  static constexpr uint32_t kExp = 0x7c00u;  // exponent bits: all set in infinities and NaN
  static constexpr uint32_t kFormat = 0;     // operand format of the instruction descriptor
  static constexpr float kTop = 11.f, kGrow = 4.f;  // of the weights, see the main kernel
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr uint32_t kFormat = 1;
  static constexpr float kTop = 0.f, kGrow = 8.f;
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
__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}
// 32 bytes, a whole sector, in one store.
__device__ __forceinline__ void st_256(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
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
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(p));
  return p != 0;
}
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
// The same with A in shared memory.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
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
// The plan: every block derives it from the lengths on the device. A group is kChains blocks of rows
// of one head and segment. Costs, in halves of the time a tile takes from memory (1400 clocks at 64
// tokens of 128 dimensions, 23 bytes a clock for each SM): 2 for a tile, 4 where it is used for two
// blocks of rows (2350 clocks), and 4 more to open a group: queries in, a chain's first and last tile
// alone, the mask of the tail, O out, 3000 clocks of which the other chain's work hides some. With 2
// for that, one request of 8 rows on a prefix of 32768 tokens (48 query and 8 KV heads of 128) took
// 43.7 us instead of 38.0, the last CTAs having all its own short pieces, and 64 requests on a prefix
// 103 instead of 100; with 6, requests of 300 own tokens lose 3 %. With few tiles for each CTA, every
// tile costs 1: one each is best then.
// ------------------------------------------------------------------------------------------------
struct Cost {
  int tile, both, open;
  __device__ __forceinline__ explicit Cost(bool even)
      : tile(even ? 1 : 2), both(even ? 1 : 4), open(even ? 0 : 4) {}
  // CTAs that share a cost: each range is as long as the longest way from one tile's start to the
  // next one's, so that a tile starts in it. A tile belongs to the CTA in whose range it starts.
  __device__ __forceinline__ int ctas(int cost, int most) const {
    return max(1, min(cost / (both + open), most));
  }
};
struct Plan {
  int cost_end[kMaxRequests + 1];    // running sum of costs up to and with segment s
  int rows_end[kMaxRequests + 1];    // running sum of rows of partials, one CTA's for each group
  int first[kMaxRequests + 1];       // first row of the segment
  int count[kMaxRequests + 1];       // and how many
  int len[kMaxRequests + 1];         // tokens
  int even;
};

template <int kChains>
__device__ __forceinline__ int groups_of(int count, int group) {
  return (count * group + kChains * kBlockRows - 1) / (kChains * kBlockRows);
}
template <int kChains>
__device__ __forceinline__ int tile_cost(const Cost& cost, int count, int group) {
  return kChains > 1 && count * group > kBlockRows ? cost.both : cost.tile;
}
// Rows of group g of a segment.
template <int kChains>
__device__ __forceinline__ int group_rows(int count, int group, int g) {
  return min(kChains * kBlockRows, count * group - g * kChains * kBlockRows);
}
// Rows of partials of a CTA's piece of a group with so many rows: one for each, or one for each and
// chain where the chains take its tiles in turn; and of one CTA's pieces of all groups of a head.
template <int kChains>
__device__ __forceinline__ int piece_rows(int rows) {
  return kChains > 1 && rows <= kBlockRows ? kChains * rows : rows;
}
template <int kChains>
__device__ __forceinline__ int head_rows(int count, int group) {
  constexpr int kWhole = kChains * kBlockRows;
  const int whole = count * group / kWhole * kWhole;
  return whole + piece_rows<kChains>(count * group - whole);
}

// Lengths and rows of every segment, cut at the tables and at the rows there are, and the running
// sums. Row starts that decrease are outside the contract: the plan is then empty (every output 0,
// lse -inf), so that no index leaves its array. Ends with a block-wide barrier.
template <int kChains>
__device__ __forceinline__ void make_plan(const AttnArgs& p, int tok, Plan& plan) {
  int bad = 0;
  for (int s = threadIdx.x; s <= p.requests; s += blockDim.x) {
    const int r0 = p.row_start[s ? s - 1 : 0], r1 = p.row_start[s ? s : p.requests];
    const int len = s ? p.own_lens[s - 1] : *p.prefix_len;
    const int64_t room = (int64_t)(s ? p.max_pages : p.n_prefix_pages) * p.page_size;
    bad |= r1 < r0;
    const int first = min(max(r0, 0), p.rows);
    plan.first[s] = first;
    plan.count[s] = max(0, min(max(r1, 0), p.rows) - first);
    plan.len[s] = (int)min((int64_t)max(len, 0), room);
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x < 32) {
    auto groups = [&](int s) { return bad ? 0 : p.kv_heads * groups_of<kChains>(plan.count[s], p.group); };
    auto tiles = [&](int s) { return (plan.len[s] + tok - 1) / tok; };
    int all = 0;
    for (int s = threadIdx.x; s <= p.requests; s += 32) all += groups(s) * tiles(s);
    all = __reduce_add_sync(~0u, all);
    const bool even = all <= 2 * (int)gridDim.x;
    const Cost cost(even);
    int c_base = 0, r_base = 0;
    for (int s0 = 0; s0 <= p.requests; s0 += 32) {
      const int s = s0 + threadIdx.x;
      int c = 0, r = 0;
      if (s <= p.requests && plan.len[s] > 0 && !bad) {
        c = groups(s) * (cost.open + tiles(s) * tile_cost<kChains>(cost, plan.count[s], p.group));
        r = p.kv_heads * head_rows<kChains>(plan.count[s], p.group);
      }
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int cc = __shfl_up_sync(~0u, c, d), rr = __shfl_up_sync(~0u, r, d);
        if ((int)threadIdx.x >= d) c += cc, r += rr;
      }
      c += c_base, r += r_base;
      if (s <= p.requests) plan.cost_end[s] = c, plan.rows_end[s] = r;
      c_base = __shfl_sync(~0u, c, 31);
      r_base = __shfl_sync(~0u, r, 31);
    }
    if (threadIdx.x == 0) plan.even = even;
  }
  __syncthreads();
}

// The plan of row t for the launch that joins its partials.
template <int kChains>
__device__ __forceinline__ void write_row_plan(const AttnArgs& p, int tok, const Plan& plan, int t) {
  RowPlan r = {};
  r.cost = plan.cost_end[p.requests];
  r.even = plan.even;
  r.prefix_tiles = (plan.len[0] + tok - 1) / tok;
  r.prefix_first = plan.first[0];
  r.prefix_count = plan.count[0];
  r.prefix_span = head_rows<kChains>(plan.count[0], p.group);
  // the last request that starts at or before t: requests without rows share a start with the next
  int lo = 0, hi = p.requests;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (plan.first[mid] <= t) lo = mid; else hi = mid - 1;
  }
  if (r.cost > 0 && lo > 0 && t < plan.first[lo] + plan.count[lo]) {
    r.owned = 1;
    r.tiles = (plan.len[lo] + tok - 1) / tok;
    r.first = plan.first[lo];
    r.count = plan.count[lo];
    r.span = head_rows<kChains>(plan.count[lo], p.group);
    r.cost0 = plan.cost_end[lo - 1];
    r.rows0 = plan.rows_end[lo - 1];
  }
  p.row_plan[t] = r;
}

// Below this, costs times kMaxCtas fit 31 bits: divisions of 64 bits take four times as long, which
// shows in calls of a few microseconds.
constexpr int kShortCost = 0x7fffffff / kMaxCtas;
__device__ __forceinline__ int plan_begin(int cost, int ctas, int c) {
  if (cost < kShortCost) return (int)((uint32_t)(cost * c) / (uint32_t)ctas);
  return (int)((int64_t)cost * c / ctas);
}
__device__ __forceinline__ int plan_owner(int cost, int ctas, int at) {
  if (cost < kShortCost) return (int)((uint32_t)((at + 1) * ctas - 1) / (uint32_t)cost);
  return (int)((((int64_t)at + 1) * ctas - 1) / cost);
}

// A position in the order of tiles: segment, head, group, tile.
template <int kChains>
struct Cursor {
  int seg, head, group, tile, at;  // at: the cost before it
  int first, count, len, tiles, groups, weight, span;  // span: rows of partials of a head
  int open;
  __device__ __forceinline__ void load(const AttnArgs& p, const Plan& plan, int tok) {
    const Cost cost(plan.even);
    first = plan.first[seg], count = plan.count[seg], len = plan.len[seg];
    tiles = (len + tok - 1) / tok;
    groups = groups_of<kChains>(count, p.group);
    weight = tile_cost<kChains>(cost, count, p.group);
    span = head_rows<kChains>(count, p.group);
    open = cost.open;
  }
  // The first row of partials of this CTA's piece.
  __device__ __forceinline__ int part_row(const AttnArgs& p, const Plan& plan) const {
    return (seg ? plan.rows_end[seg - 1] : 0) + head * span + group * (kChains * kBlockRows) +
           (int)blockIdx.x * p.piece_rows;
  }
  __device__ __forceinline__ int rows(const AttnArgs& p) const {
    return group_rows<kChains>(count, p.group, group);
  }
  // The first tile at or behind cost c.
  __device__ __forceinline__ void seek(const AttnArgs& p, const Plan& plan, int c, int tok) {
    int lo = 0, hi = p.requests;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (plan.cost_end[mid] > c) hi = mid; else lo = mid + 1;
    }
    seg = lo;
    load(p, plan, tok);
    const int start = seg ? plan.cost_end[seg - 1] : 0, whole = open + tiles * weight;
    int g = (c - start) / whole;
    const int rest = c - start - g * whole;
    tile = rest == 0 ? 0 : max(1, (rest - open + weight - 1) / weight);
    if (tile >= tiles) tile = 0, ++g;
    at = start + g * whole + cost_to(tile);
    head = groups == 1 ? g : g / groups;
    group = g - head * groups;
    if (head == p.kv_heads) next_segment(p, plan, tok);
  }
  // From the group's start to tile t of it.
  __device__ __forceinline__ int cost_to(int t) const { return t == 0 ? 0 : open + t * weight; }
  // The start of the tile n on, in the same group.
  __device__ __forceinline__ int ahead(int n) const { return at + cost_to(tile + n) - cost_to(tile); }
  // Tiles from here on that start before `end`, in the same group.
  __device__ __forceinline__ int tiles_before(int end) const {
    const int left = end - at - (tile == 0 ? open : 0);
    return min(tiles - tile, max(1, (left + weight - 1) / weight));
  }
  __device__ __forceinline__ void next_segment(const AttnArgs& p, const Plan& plan, int tok) {
    head = group = tile = 0;
    const int done = plan.cost_end[seg];
    while (seg < p.requests && plan.cost_end[seg + 1] == done) ++seg;
    if (seg < p.requests) {
      ++seg;
      load(p, plan, tok);
    }
  }
  // n >= 1 tiles on, not beyond the group's end
  __device__ __forceinline__ void skip(const AttnArgs& p, const Plan& plan, int n, int tok) {
    at = ahead(n);
    tile += n;
    if (tile < tiles) return;
    tile = 0;
    if (++group < groups) return;
    group = 0;
    if (++head < p.kv_heads) return;
    next_segment(p, plan, tok);
  }
};

// ------------------------------------------------------------------------------------------------
// Main kernel. kDim: head dimension rounded up (64, 128, 256), the rest of it zero.
//
// Per tile: S[128 rows, kTok] = Q K^T and O[128 rows, kDim] += P V on the tensor cores, with Q, S and
// O in tensor memory, K and V in a ring of shared-memory stages. K is the product's B operand with
// the dimension contiguous, V its B operand with N contiguous: both lie as loaded, [token][64
// dimensions] rows of 128 bytes, swizzled.
//
// Chains: tensor memory holds two sets of O, S and Q up to kDim = 128, one at 256. With two, groups
// of more than 128 rows give each chain a block of rows and both take every tile, so K and V are
// brought in once for 256 rows; smaller groups give both chains the same rows, and the tiles in
// turn, so two tiles are under way at a time. P goes through shared memory, which frees S as soon as
// it has been read: the next tile's first product runs while the softmax works. With one chain, S
// is held twice, and P takes the place of its S.
//   warps 0-3 (4-7)  softmax of a chain: a thread owns a row (its lane of tensor memory), so the
//                    running maximum and sum need no exchange between threads; they also bring Q
//                    in and take O out
//   next warp        issues the products, in the order in which their operands become ready
//   next 2 warps     (kTma) K and V: one TMA box per group of tokens of one page and 64 dimensions
//   next 4 warps     (otherwise) 16 bytes per cp.async, for any page size and strides
// The weights of the second product are rounded to the operands' type, as the tensor cores take them;
// the sum l is of the weights before that. The error is as large as the output's own rounding: against
// 64 bits outputs are off by 2.8e-4 (fp16) and 2.3e-3 (bf16) of their norm, where weights of 32 bits
// give 2.1e-4 and 1.7e-3. Remainders as a second operand gave those, for twice the product and the
// stores of P: 64 requests on a prefix 129.9 us instead of 101.0, 8 rows on 32775 tokens 35.3 instead
// of 33.6.
// A weight is 2^(s - m_ref), where m_ref is kTop below the row's maximum when it is set. O is rescaled,
// and m_ref set again, only when the maximum has grown by more than kGrow since: weights stay below
// 2^(kTop + kGrow), and O, l and the partial refer to the same m_ref, so nothing is approximated.
// bf16 has the exponents of fp32: 0 and 8. fp16 ends at 2^16 and loses bits from 2^-14 down: with 11
// and 4 that begins 2^-25 below the largest weight, with 0 and 8 at 2^-14, where thousands of keys
// behind one that stands 10 to 18 nats above them count for much and were lost. 7 and 8 would lose
// some of them and save 0.4 us of the 33.6 that 8 rows on 32775 tokens take (24 query and 4 KV heads of
// 256), which rescale more often; 13 and 2 take 34.7.
// ------------------------------------------------------------------------------------------------
template <int kDim, bool kTma>
struct Shape {
  static constexpr int kChains = kTma && kDim <= 128 ? 2 : 1;
  static constexpr int kSoftWarps = 4 * kChains;
  static constexpr int kLoadWarps = kTma ? 2 : kLoadThreads / 32;
  static constexpr int kThreads = 32 * (kSoftWarps + 1 + kLoadWarps);
  static constexpr int kTok = kDim == 64 ? 128 : 64;  // tokens per tile
  static constexpr int kStages = kDim == 256 ? 3 : kDim == 128 ? 5 : 4;
  static constexpr int kP = kChains > 1 ? kTok * kBlockRows * 2 : 0;  // P of a chain, in shared memory
  static constexpr int kSub = kTok * 128;           // [token][64 dimensions] of K or V
  static constexpr int kHalf = kSub * (kDim / 64);  // K or V of a stage
  static constexpr int kRing = kStages * 2 * kHalf;
  // columns of tensor memory: O of each chain, two S, Q of each chain
  static constexpr int kS = kChains * kDim, kQ = kS + 2 * kTok;
  static constexpr int kColumns = 512;
  static_assert(kQ + kChains * kDim / 2 <= kColumns, "tensor memory of an SM");
};

struct Control {
  uint64_t full[6], empty[6];
  uint64_t s_full[2], p_full[2], o_done[2];  // per S: of a chain, or of every other tile
  uint64_t s_free[2];                        // per chain: S has been read
  uint64_t q_full[2], o_free[2], sync[3];    // per chain; sync[2]: both
  uint64_t drain;
  uint32_t tmem;
  int abort;
  int bad_page[6];   // per stage: 1 + the tile, if any, for which a page outside the cache was met
  int bad_value[2];  // per chain: 1 + the tile for which a value that is no number was met
  unsigned char bad_token[2][128];
};

template <int kDim, bool kTma>
constexpr size_t attn_smem() {
  return 1024 + Shape<kDim, kTma>::kRing + Shape<kDim, kTma>::kChains * Shape<kDim, kTma>::kP + sizeof(Plan) + sizeof(Control) + 16;
}

__device__ int g_attn_status;

// mbar_wait without its suspend-time hint: the waits of this kernel are short. One test in line,
// which suspends the thread for a while, and the rest out of line: the code of the roles shares the
// instruction caches of an SM.
__device__ __noinline__ bool bar_wait_on(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const unsigned long long t0 = globaltimer_ns();
  for (unsigned int it = 1; it < kMaxSpin; ++it) {
    if (mbar_test(bar, parity)) return true;
    if ((it & 63u) == 0) {
      if (*abort) return false;
      if (globaltimer_ns() - t0 > kPipeWaitNs) break;
    }
  }
  *abort = 1;
  return false;
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return mbar_test(bar, parity) || bar_wait_on(bar, parity, abort);
}
// Has the phase completed? Never suspends the thread.
__device__ __forceinline__ bool mbar_test_now(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

template <typename T, int kDim, bool kTma>
__global__ void __launch_bounds__(Shape<kDim, kTma>::kThreads, 1)
    attn_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const AttnArgs p) {
  using S = Shape<kDim, kTma>;
  constexpr int kTok = S::kTok, kStages = S::kStages, kChains = S::kChains;
  constexpr int kSoftWarps = S::kSoftWarps;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Control& c = *reinterpret_cast<Control*>(smem + S::kRing + kChains * S::kP);
  Plan& plan = *reinterpret_cast<Plan*>((reinterpret_cast<uintptr_t>(&c + 1) + 15) & ~(uintptr_t)15);
  volatile int* s_abort = &c.abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (kTma && warp > kSoftWarps && lane == 0)
    tma_prefetch_desc(warp == kSoftWarps + 2 ? &map_v : &map_k);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&c.full[s], kTma ? 2 : kLoadThreads + kLoadThreads / 32);
      mbar_init(&c.empty[s], 1);
      c.bad_page[s] = 0;
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&c.s_full[b], 2);  // the products' completion, and the thread that issued them
      mbar_init(&c.p_full[b], 4);
      mbar_init(&c.o_done[b], 1);
      mbar_init(&c.s_free[b], 4);
      mbar_init(&c.q_full[b], 4);
      mbar_init(&c.o_free[b], 4);
      mbar_init(&c.sync[b], 4);
      c.bad_value[b] = 0;
    }
    mbar_init(&c.sync[2], 8);
    mbar_init(&c.drain, 1);
    c.abort = 0;
    mbar_fence_init();
  }
  if (warp == kSoftWarps) tmem_alloc(&c.tmem, S::kColumns);
  {  // page tables and queries into L2 behind the plan
    const int line = 32, step = gridDim.x * blockDim.x * line;
    const int at = (blockIdx.x * blockDim.x + threadIdx.x) * line;
    for (int64_t i = at; i < p.n_prefix_pages; i += step) prefetch_l2(p.prefix_pages + i);
    const int64_t all = p.requests > 0 && p.max_pages > 0 ? (p.requests - 1) * p.pages_stride + p.max_pages : 0;
    for (int64_t i = at; i < all; i += step) prefetch_l2(p.pages + i);
    const int n = p.rows * p.q_heads, first = blockIdx.x * blockDim.x + threadIdx.x;
    for (int i = first; i < n; i += gridDim.x * blockDim.x) {
      const int row = i / p.q_heads;
      const T* q = static_cast<const T*>(p.q) + row * p.q_row + (i - row * p.q_heads) * p.q_head;
      for (int d = 0; d < p.dim; d += 64) prefetch_l2(q + d);
    }
  }
  grid_dep_wait();
  grid_dep_launch();
  make_plan<kChains>(p, kTok, plan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, c.tmem, 0);
  const int cost = plan.cost_end[p.requests];
  const int ctas = Cost(plan.even).ctas(cost, gridDim.x);
  const bool idle = cost == 0 || (int)blockIdx.x >= ctas;
  const int c_lo = idle ? 0 : plan_begin(cost, ctas, blockIdx.x);
  const int c_hi = idle ? 0 : plan_begin(cost, ctas, blockIdx.x + 1);
  const uint32_t ring = smem_u32(smem);
  const int stage_bytes = 2 * S::kHalf;

  Cursor<kChains> cur;
  cur.at = c_hi;
  if (!idle) cur.seek(p, plan, c_lo, kTok);

  if (kTma && warp > kSoftWarps) {
    // ------------------------------------------------------------------------------ loaders (TMA)
    // Boxes of box_rows tokens x 64 dimensions, their pages looked up by a lane each. A box behind
    // the length, or of a page that does not exist, is loaded from behind the last page: zeros,
    // without a read.
    const int groups = kTok / p.box_rows;  // a power of two, at most 16
    const int box_bytes = p.box_rows * 128;
    const bool leader = elect_one();
    const bool is_v = warp == kSoftWarps + 2;
    const CUtensorMap* map = is_v ? &map_v : &map_k;
    const int row0 = (lane & (groups - 1)) * p.box_rows;
    int id = -1, at = 0;
    auto look_up = [&] {
      const int tok = cur.tile * kTok + row0;
      id = -1, at = 0;
      if (tok < cur.len) {
        const int32_t* table = cur.seg ? p.pages + (int64_t)(cur.seg - 1) * p.pages_stride : p.prefix_pages;
        const int pg = p.by_page.div(tok);
        id = table[pg];
        at = tok - pg * p.page_size;
      }
    };
    const uint64_t once = l2_evict_first_policy(), again = l2_evict_normal_policy();
    if (!idle) look_up();
    int issued = 0;
    for (int i = 0; cur.at < c_hi; ++i) {
      const int stage = i % kStages, at_cost = cur.at;
      const int head = cur.head, tok = cur.tile * kTok + row0, len = cur.len;
      const uint64_t pol = cur.groups > 1 ? again : once;
      const int raw = id, tile_at = at;
      cur.skip(p, plan, 1, kTok);
      if (cur.at < c_hi) look_up();  // its latency passes behind this tile's wait
      if (!__all_sync(~0u, bar_wait(&c.empty[stage], ((i / kStages) & 1) ^ 1, s_abort))) break;
      const bool exists = raw >= 0 && raw < p.total_pages;
      const int page = tok < len && exists ? raw : p.total_pages;
      if (tok < len && !exists) *const_cast<volatile int*>(&c.bad_page[stage]) = at_cost + 1;
      __syncwarp();
      // One lane issues every box, with operands that are the same in the whole warp.
      const uint32_t dst = ring + stage * stage_bytes + (is_v ? S::kHalf : 0);
      if (leader) mbar_arrive_expect_tx(&c.full[stage], S::kHalf);
#pragma unroll 1
      for (int g = 0; g < groups; ++g) {
        const int pid = __shfl_sync(~0u, page, g), pat = __shfl_sync(~0u, tile_at, g);
        if (leader) {
#pragma unroll
          for (int sub = 0; sub < kDim / 64; ++sub)
            tma_load_4d(dst + g * box_bytes + sub * S::kSub, map, &c.full[stage], sub * 64, pat, head,
                        pid, pol);
        }
      }
      __syncwarp();
      issued = i + 1;
    }
    // After an abort: do not retire while copies may still be landing in shared memory.
    if (*s_abort) {
      for (int k = max(0, issued - kStages); k < issued; ++k) {
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_test(&c.full[k % kStages], (k / kStages) & 1) && globaltimer_ns() - t0 < kPipeWaitNs) {
        }
      }
    }
  } else if (warp > kSoftWarps) {
    // ------------------------------------------------------------------------------ loaders
    constexpr int kChunks = kDim / 8;               // 16-byte chunks per token
    constexpr int kWarpRows = 32 / kChunks;         // tokens per warp and copy
    constexpr int kLoadWarps = S::kLoadWarps;
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
        const int pg = p.by_page.div(tok);
        id = table[pg];
        at = tok - pg * p.page_size;
        if (id < 0 || id >= p.total_pages) id = -2;
      }
    };
    int id = -1, at = 0;
    if (!idle) look_up(id, at);
    for (int i = 0; cur.at < c_hi; ++i) {
      const int stage = i % kStages, at_cost = cur.at;
      const int head = cur.head;
      const int tile_id = id, tile_at = at;
      const T* kc = static_cast<const T*>(p.k) + head * p.ks[2] + chunk * 8;
      const T* vc = static_cast<const T*>(p.v) + head * p.vs[2] + chunk * 8;
      cur.skip(p, plan, 1, kTok);
      if (cur.at < c_hi) look_up(id, at);  // its latency passes behind this tile's wait and copies
      bool ok = true;
      if (lane == 0) ok = bar_wait(&c.empty[stage], ((i / kStages) & 1) ^ 1, s_abort);
      ok = __shfl_sync(~0u, ok, 0);
      if (!ok) break;
      if (tile_id == -2) c.bad_page[stage] = at_cost + 1;
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
      if (lane == 0) mbar_arrive(&c.full[stage]);  // orders bad_page before the stage is full
    }
    cp_async_wait_all();
  } else if (warp == kSoftWarps) {
    // ------------------------------------------------------------------------------ products
    // The whole warp runs this loop, so that addresses and descriptors stay in uniform registers;
    // one elected lane issues.
    for (int r = blockIdx.x + gridDim.x * lane; r < p.rows; r += gridDim.x * 32)
      write_row_plan<kChains>(p, kTok, plan, r);
    __syncwarp();
    if (!idle) {
      constexpr uint32_t kIdescS = instr_desc<T>(kTok, false), kIdescO = instr_desc<T>(kDim, true);
      const bool leader = elect_one();
      bool ok = true;
      [[maybe_unused]] auto wait = [&](uint64_t* bar, int phase) {
        ok = ok && __all_sync(~0u, bar_wait(bar, phase & 1, s_abort));
      };
      auto ready = [&](uint64_t* bar, int phase) {
        return __any_sync(~0u, mbar_test_now(bar, phase & 1));
      };
      // S = Q K^T of a stage, for chain w into S number b
      auto scores = [&](int w, int b, int stage) {
        if constexpr (!kTma) fence_proxy_async_smem();  // cp.async writes through the generic proxy
        tc_fence_after();
        const uint64_t kd = smem_desc(ring + stage * stage_bytes, 16, 1024);
        const uint32_t sd = tmem + S::kS + b * kTok, qd = tmem + S::kQ + w * (kDim / 2);
        if (leader) {
#pragma unroll
          for (int ks = 0; ks < kDim / 16; ++ks)
            tc_mma(sd, qd + ks * 8, kd + (((ks / 4) * S::kSub + (ks % 4) * 32) >> 4), kIdescS, ks > 0);
          tc_commit(&c.s_full[b]);
          mbar_arrive(&c.s_full[b]);
        }
        if constexpr (kChains == 1) __syncwarp();
      };
      // O (+)= P V of a stage, for chain w from S number b; `last`: nothing else reads the stage
      auto weigh = [&](int w, int b, int stage, bool first, bool last) {
        tc_fence_after();
        const uint64_t vd = smem_desc(ring + stage * stage_bytes + S::kHalf, S::kSub, 1024);
        const uint32_t pa = tmem + S::kS + b * kTok, od = tmem + w * kDim;
        const uint64_t pd = smem_desc(ring + S::kRing + w * S::kP, 16, 1024);
        if (leader) {
#pragma unroll
          for (int ks = 0; ks < kTok / 16; ++ks) {
            const uint64_t v = vd + ks * (2048 >> 4);
            if constexpr (kChains > 1)
              tc_mma_ss(od, pd + (((ks / 4) * kBlockRows * 128 + (ks % 4) * 32) >> 4), v, kIdescO,
                        ks > 0 || !first);
            else
              tc_mma(od, pa + ks * 8, v, kIdescO, ks > 0 || !first);
          }
          if (last) tc_commit(&c.empty[stage]);
          tc_commit(&c.o_done[b]);
        }
        if constexpr (kChains == 1) __syncwarp();
      };
      if constexpr (kChains == 1) {
        int opened = 0, starts = 0, n = 0;
        bool before = false;  // the tile before opened its piece
        auto second = [&](int i, bool first) {
          wait(&c.p_full[i & 1], i >> 1);
          if (first && opened++ > 0) wait(&c.o_free[0], opened - 2);
          if (ok) weigh(0, i & 1, i % kStages, first, true);
        };
        for (; cur.at < c_hi && ok; ++n) {
          const bool start = n == 0 || cur.tile == 0;
          // A new piece's queries arrive after the last weights of the old one: take those first.
          if (start && n > 0) second(n - 1, before);
          if (start) wait(&c.q_full[0], starts++);
          const int stage = n % kStages;
          // While this tile's keys are on their way, the weights of the one before may be ready.
          bool pending = !start;
          for (unsigned int it = 0; pending && it < kMaxPolls; ++it) {
            if (ready(&c.full[stage], n / kStages)) break;
            if (!ready(&c.p_full[(n - 1) & 1], (n - 1) >> 1)) continue;
            second(n - 1, before);
            pending = false;
          }
          wait(&c.full[stage], n / kStages);
          if (!ok) break;
          scores(0, n & 1, stage);
          if (pending) second(n - 1, before);
          before = start;
          cur.skip(p, plan, 1, kTok);
        }
        if (n > 0) second(n - 1, before);
      } else {
        // One thread: straight code that waits for what it needs, in the order in which it is needed.
        // Per chain, a bit each: parity of the first and second products issued, of the pieces opened
        // by a first and by a second product, and whether there was one at all.
        int issued = 0, weighed = 0, starts = 0, opened = 0, any_issued = 0, any_opened = 0;
        auto wait1 = [&](uint64_t* bar, int phase) { ok = ok && bar_wait(bar, phase & 1, s_abort); };
        auto first = [&](int w, int stage) {
          if ((any_issued >> w) & 1) wait1(&c.s_free[w], (issued >> w) ^ 1);
          if (ok) scores(w, w, stage);
          issued ^= 1 << w, any_issued |= 1 << w;
        };
        auto second = [&](int w, int stage, bool opens, bool last) {
          wait1(&c.p_full[w], weighed >> w);
          if (opens && ((any_opened >> w) & 1)) wait1(&c.o_free[w], (opened >> w) ^ 1);
          if (ok) weigh(w, w, stage, opens, last);
          weighed ^= 1 << w;
          if (opens) opened ^= 1 << w, any_opened |= 1 << w;
        };
        auto queries = [&](int w) {
          wait1(&c.q_full[w], starts >> w);
          starts ^= 1 << w;
        };
        int due = 0, due_opens = 0, due_stage0 = 0, due_stage1 = 0;  // second products, per chain
        auto settle = [&](int w) {
          if (!((due >> w) & 1)) return;
          second(w, w ? due_stage1 : due_stage0, (due_opens >> w) & 1, true);
          due &= ~(1 << w);
        };
        for (int n = 0, stage = 0, turn = 0; leader && cur.at < c_hi && ok;) {
          const int tiles = cur.tiles_before(c_hi);
          auto step = [&] {
            if (++stage == kStages) stage = 0, turn ^= 1;
            ++n;
          };
          if (cur.rows(p) > kBlockRows) {
            // Both chains take every tile: its first products before the second ones of the tile
            // before, for which the softmax has yet to finish.
            settle(n & 1);
            settle((n & 1) ^ 1);
            queries(0);
            queries(1);
            int before = 0;
            for (int t = 0; t <= tiles && ok; ++t) {
              if (t < tiles) {
                wait1(&c.full[stage], turn);
                first(0, stage);
                first(1, stage);
              }
              if (t > 0) {
                second(0, before, t == 1, false);
                second(1, before, t == 1, true);
              }
              before = stage;
              if (t < tiles) step();
            }
          } else {
            // The chains take turns. The second product of a chain's tile comes before the first one
            // of its next, which may wait for its keys; the other chain works meanwhile.
            for (int t = 0; t < tiles && ok; ++t) {
              const int w = n & 1;
              settle(w);
              if (t < 2) queries(w);
              wait1(&c.full[stage], turn);
              first(w, stage);
              due |= 1 << w;
              due_opens = t < 2 ? due_opens | 1 << w : due_opens & ~(1 << w);
              if (w) due_stage1 = stage; else due_stage0 = stage;
              step();
            }
          }
          cur.skip(p, plan, tiles, kTok);
          if (cur.at >= c_hi) {
            settle(n & 1);
            settle((n & 1) ^ 1);
          }
        }
        ok = __all_sync(~0u, ok);
      }
      if (!ok) {  // let what is in flight land before the tensor memory is freed
        if (leader) tc_commit(&c.drain);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_test(&c.drain, 0) && globaltimer_ns() - t0 < kPipeWaitNs) {
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------------------ softmax
    const int w = kChains > 1 ? warp >> 2 : 0;            // the chain
    const int row = threadIdx.x & (kBlockRows - 1);       // of its block
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + lanes + w * kDim, t_q = tmem + lanes + S::kQ + w * (kDim / 2);
    bool ok = true;
    // A barrier of the warps that work on a tile; bounded like the other waits.
    int syncs[2] = {0, 0};
    auto sync_rows = [&](bool both) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.sync[both ? 2 : w]);
      ok = bar_wait(&c.sync[both ? 2 : w], syncs[both]++ & 1, s_abort) && ok;
      __syncwarp();
    };
    // The piece at a cursor: its tiles, and those among them that this chain takes (from its first
    // on, every `step`-th).
    struct Piece {
      int tiles, mine, from, step;
      bool both;
    };
    auto piece_at = [&](const Cursor<kChains>& at, int index) {
      Piece x;
      x.tiles = at.tiles_before(c_hi);
      x.both = kChains > 1 && at.rows(p) > kBlockRows;
      const bool split = kChains > 1 && !x.both;
      x.step = split ? 2 : 1;
      x.from = split ? (w + index) & 1 : 0;
      x.mine = split ? (x.tiles - x.from + 1) / 2 : x.tiles;
      return x;
    };
    // What this thread's row of the open piece sees, and its queries into tensor memory.
    int my_rows = 0, base = 0, seen = 0;
    unsigned long long branch = 0;
    auto open_piece = [&](const Cursor<kChains>& at, bool both) {
      const int off = at.group * kChains * kBlockRows + (both ? w * kBlockRows : 0);
      my_rows = min(kBlockRows, at.count * p.group - off);
      base = at.len - at.count;
      const bool act = row < my_rows;
      const int f = off + row, local = act ? p.by_group.div(f) : 0;
      const int t = at.first + local;
      seen = !act ? 0x7fffffff : at.seg == 0 ? at.len : min(at.len, base + local + 1);
      branch = 0;
      if (p.tree && at.seg && act) {
        branch = (unsigned long long)p.tree[t];
        seen = min(at.len, base);
      }
      if ((warp & 3) * 32 < my_rows) {
        const T* src = static_cast<const T*>(p.q) + (int64_t)t * p.q_row +
                       (int64_t)(at.head * p.group + (act ? f - local * p.group : 0)) * p.q_head;
        uint32_t x[kDim / 2];  // all loads before the first store
        if (p.q_vec) {
#pragma unroll
          for (int j = 0; j < kDim / 8; ++j) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (act && 8 * j < p.dim) v = *reinterpret_cast<const uint4*>(src + 8 * j);
            x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < kDim / 2; ++j)
            x[j] = act && 2 * j < p.dim ? *reinterpret_cast<const uint32_t*>(src + 2 * j) : 0u;
        }
        __syncwarp();
#pragma unroll
        for (int c0 = 0; c0 < kDim / 2; c0 += 32)
          tmem_st32(t_q + c0, *reinterpret_cast<const uint32_t(*)[32]>(&x[c0]));
        tc_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.q_full[w]);
    };

    int task = 0;        // tiles this chain has taken
    int tile_index = 0;  // tiles of the CTA before the piece
    Piece piece;
    int part = 0;  // where this row's partial goes
    bool room = false;
    // To the next piece that this chain takes tiles of, and open it. A single tile that is the other
    // chain's leaves an empty partial.
    auto advance = [&] {
      while (cur.at < c_hi) {
        piece = piece_at(cur, tile_index);
        part = cur.part_row(p, plan) + w * (piece.both ? kBlockRows : cur.rows(p)) + row;
        room = part < p.part_rows;
        if (kChains == 1 || piece.mine > 0) {
          open_piece(cur, piece.both);
          return true;
        }
        if (room && row < cur.rows(p)) p.part_ml[part] = make_float2(neg_inf(), 0.f);
        tile_index += piece.tiles;
        cur.skip(p, plan, piece.tiles, kTok);
      }
      return false;
    };
    for (bool more = advance(); more && ok;) {
      const bool both = piece.both;
      const bool act_warp = (warp & 3) * 32 < my_rows;
      const int32_t* table = cur.seg ? p.pages + (int64_t)(cur.seg - 1) * p.pages_stride : p.prefix_pages;
      // The first token that some row of the group may not see.
      const int sure = cur.seg == 0 ? cur.len : max(0, min(cur.len, p.tree ? base : base + 1));
      float m_ref = neg_inf(), l = 0.f;  // the maximum the weights refer to, and their sum

      for (int k = 0; k < piece.mine; ++k, ++task) {
        const int step = piece.from + k * piece.step, i = tile_index + step, stage = i % kStages;
        const int b = kChains > 1 ? w : task & 1, phase = kChains > 1 ? task : task >> 1;
        const uint32_t t_s = tmem + lanes + S::kS + b * kTok;
        const int tile0 = (cur.tile + step) * kTok, mark = cur.ahead(step) + 1;
        bool bad_page = false;
        // Which of the 64 tokens from t0 on this row sees, one bit each.
        auto visible = [&](int t0) {
          auto below = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
          unsigned long long bits = below(seen - t0);
          if (branch) {
            const int off = t0 - base;
            const unsigned long long m =
                off >= 64 || off <= -64 ? 0ull : off >= 0 ? branch >> off : branch << -off;
            bits |= m & below(cur.len - t0);
          }
          if (bad_page) {
#pragma unroll 1
            for (int j = 0; j < 64 && t0 + j < cur.len; ++j) {
              const int id = table[p.by_page.div(t0 + j)];
              if (id < 0 || id >= p.total_pages) bits &= ~(1ull << j);
            }
          }
          return bits;
        };
        const bool tail = tile0 + kTok > sure;  // the same in the whole group
        // 0 * NaN would carry values that are no numbers into rows that do not see them. Behind the
        // length, a box may have brought what the rest of its page holds: zeros in its place. Tokens
        // that only some rows see are searched for infinities and NaN: those are replaced by zeros
        // before the second product, and added afterwards to the rows that see them. All this while
        // the first product runs.
        bool poisoned = false;
        const int set = both ? 0 : w;  // whose flags
        if (tail) {
          ok = bar_wait(&c.full[stage], (i / kStages) & 1, s_abort);
          if (!__all_sync(~0u, ok)) break;
          uint8_t* vt = smem + stage * stage_bytes + S::kHalf;
          const int stored = min(cur.len - tile0, kTok);  // tokens of the tile
          // a thread's chunk column, and every kPass-th token from its first
          constexpr int kCols = kDim / 8, kPass = kBlockRows / kCols;
          const int col = row % kCols, tok0 = row / kCols;
          uint8_t* column = vt + (col / 8) * S::kSub + (col & 7) * 16;
          if (kTma && stored < kTok) {
            const int end = (stored + p.box_rows - 1) & -p.box_rows;
            for (int r = stored + tok0; r < end; r += kPass)
              *reinterpret_cast<uint4*>(column + r * 128) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
          }
          const int from = max(sure - tile0, 0);
          if (from < stored) {
            auto no_number = [](const uint4& x) {
              return non_finite<T>(x.x) | non_finite<T>(x.y) | non_finite<T>(x.z) | non_finite<T>(x.w);
            };
            bool found = false;
            for (int r = from + tok0; r < stored; r += kPass)
              found |= no_number(*reinterpret_cast<const uint4*>(column + r * 128));
            if (found) *const_cast<volatile int*>(&c.bad_value[set]) = mark;
            sync_rows(both);
            poisoned = *const_cast<volatile int*>(&c.bad_value[set]) == mark;
            if (poisoned) {
              for (int x = row; x < kTok; x += kBlockRows) c.bad_token[set][x] = 0;
              sync_rows(both);
              for (int r = from + tok0; r < stored; r += kPass) {
                uint4& x = *reinterpret_cast<uint4*>(column + r * 128);
                if (!no_number(x)) continue;
                *const_cast<volatile unsigned char*>(&c.bad_token[set][r]) = 1;
                x = make_uint4(finite_or_zero<T>(x.x), finite_or_zero<T>(x.y), finite_or_zero<T>(x.z),
                               finite_or_zero<T>(x.w));
              }
              fence_proxy_async_smem();
              sync_rows(both);
            }
          }
        }
        ok = bar_wait(&c.s_full[b], phase & 1, s_abort) && ok;
        if (!__all_sync(~0u, ok)) break;
        tc_fence_after();
        if (act_warp) {
          // 64 scores at a time. Of a tile of 128 the second half is read twice: holding both would
          // cost the registers that the rest needs.
          uint32_t s[64];
          bool masked = tail, plain = false;
          float mul = 1.f;
          auto scores = [&](int h, bool again) {
#pragma unroll
            for (int j = 0; j < 64; j += 32)
              tmem_ld32(*reinterpret_cast<uint32_t(*)[32]>(&s[j]), t_s + h * 64 + j);
            if (!again && h == kTok / 64 - 1) {
              // The stage's flag, while the scores arrive: visible through the issuing thread, which
              // waited for the stage and then arrived on s_full.
              bad_page = *const_cast<volatile int*>(&c.bad_page[stage]) == mark;
              masked = tail || bad_page;
              plain = !masked && p.scale_log2 > 0.f;
              mul = plain ? p.scale_log2 : 1.f;
            }
            tc_wait_ld();
            if (!plain) {
              const unsigned long long bits = masked ? visible(tile0 + h * 64) : ~0ull;
              const uint32_t lo = (uint32_t)bits, hi = (uint32_t)(bits >> 32);
#pragma unroll
              for (int j = 0; j < 64; ++j) {
                const float x = __uint_as_float(s[j]) * p.scale_log2;
                s[j] = __float_as_uint((j < 32 ? lo >> j : hi >> (j - 32)) & 1u ? x : neg_inf());
              }
              __syncwarp();
            }
          };
          // S has been read: the next tile's may take its place
          auto give_back = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.s_free[w]);
          };
          float mx4[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
#pragma unroll
          for (int h = kTok / 64 - 1; h >= 0; --h) {
            scores(h, false);
#pragma unroll
            for (int j = 0; j < 64; ++j) mx4[j & 3] = fmaxf(mx4[j & 3], __uint_as_float(s[j]));
          }
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * mul;
          if constexpr (kChains > 1 && kTok == 64) give_back();
          const bool grow = mx > m_ref + (Pair<T>::kTop + Pair<T>::kGrow) ||
                            (m_ref == neg_inf() && mx > neg_inf());
          if (__any_sync(~0u, grow)) {
            // (rounded up: the largest weight is 2^kTop at most, however large the scores are)
            const float to = __fadd_ru(mx, -Pair<T>::kTop), f = grow ? ex2(m_ref - to) : 1.f;
            if (grow) m_ref = to;
            l *= f;
            if (k > 0) {  // O holds the chain's tiles so far
              const int last = task - 1;
              ok = kChains > 1 ? bar_wait(&c.o_done[w], last & 1, s_abort)
                               : bar_wait(&c.o_done[last & 1], (last >> 1) & 1, s_abort);
              tc_fence_after();
              __syncwarp();
#pragma unroll 1
              for (int c0 = 0; c0 < kDim; c0 += 32) {
                uint32_t x[32];
                tmem_ld32(x, t_o + c0);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * f);
                tmem_st32(t_o + c0, x);
              }
              tc_wait_st();
            }
          }
          const float ref = m_ref == neg_inf() ? 0.f : m_ref;
          const uint64_t mul2 = pair_of(mul, mul), ref2 = pair_of(-ref, -ref);
          uint64_t sum2[2] = {0, 0};
#pragma unroll
          for (int h = 0; h < kTok / 64; ++h) {
            if (h > 0) {
              scores(h, true);
              if constexpr (kChains > 1) give_back();
            }
#pragma unroll
            for (int j = 0; j < 64; j += 2) {
              // The product is rounded, as the maximum was, before the difference: left exact, as by one
              // fma, it may lie above the rounded maximum by half a step, which is more than 1 from 2^25
              // on, and weights of large scores have no bound then. 64 requests on a prefix take 99.7 us
              // instead of 98.4 for it.
              const uint64_t e = add_pair(fma_pair((uint64_t)s[j + 1] << 32 | s[j], mul2, p.minus_zero), ref2);
              const float x = ex2(__uint_as_float((uint32_t)e)), y = ex2(__uint_as_float((uint32_t)(e >> 32)));
              sum2[(j >> 1) & 1] = add_pair(sum2[(j >> 1) & 1], pair_of(x, y));
              s[j / 2] = Pair<T>::pack(x, y);
            }
            if constexpr (kChains > 1) {
              // once P of the chain's last tile has been used
              if (h == 0 && task > 0) ok = bar_wait(&c.o_done[w], (task - 1) & 1, s_abort) && ok;
              uint8_t* to = smem + S::kRing + w * S::kP + h * kBlockRows * 128 + row * 128;
#pragma unroll
              for (int j = 0; j < 8; ++j)
                *reinterpret_cast<uint4*>(to + ((j ^ (row & 7)) << 4)) =
                    make_uint4(s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]);
            } else {
              // over scores that have been read: weights take half the columns
              tmem_st32(t_s + h * 32, *reinterpret_cast<const uint32_t(*)[32]>(&s[0]));
            }
          }
          const uint64_t sum = add_pair(sum2[0], sum2[1]);
          l += __uint_as_float((uint32_t)sum) + __uint_as_float((uint32_t)(sum >> 32));
          if constexpr (kChains > 1)
            fence_proxy_async_smem();
          else
            tc_wait_st();
        } else if constexpr (kChains > 1) {
          if (lane == 0) mbar_arrive(&c.s_free[w]);
          // A warp without rows waits as the others do: its arrival for this tile must not be counted
          // for the one before.
          if (task > 0) ok = bar_wait(&c.o_done[w], (task - 1) & 1, s_abort) && ok;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c.p_full[b]);
        if (poisoned) {
          ok = ok && bar_wait(&c.o_done[b], phase & 1, s_abort);
          tc_fence_after();
          __syncwarp();
          for (int x = 0; x < kTok && act_warp; ++x) {
            if (!*const_cast<volatile unsigned char*>(&c.bad_token[set][x])) continue;
            const int tok = tile0 + x, pg = p.by_page.div(tok);
            const bool see = row < my_rows && (visible(tok) & 1ull);
            const T* v = static_cast<const T*>(p.v) + table[pg] * p.vs[0] +
                         (tok - pg * p.page_size) * p.vs[1] + cur.head * p.vs[2];
#pragma unroll 1
            for (int c0 = 0; c0 < kDim; c0 += 32) {
              uint32_t y[32];
              tmem_ld32(y, t_o + c0);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (c0 + j >= p.dim || !see) continue;
                const float z = (float)v[c0 + j];
                if (!isfinite(z)) y[j] = __float_as_uint(__uint_as_float(y[j]) + z);
              }
              __syncwarp();
              tmem_st32(t_o + c0, y);
            }
            tc_wait_st();
          }
          tc_fence_before();
          sync_rows(both);  // the flags are free again
        }
      }
      if (!__all_sync(~0u, ok)) {
        ok = false;
        break;
      }

      // ---- end of a piece: the next one's queries first, then O out
      const int done_rows = my_rows, last = task - 1;
      const int done_part = part;
      const bool done_room = room;
      tile_index += piece.tiles;
      cur.skip(p, plan, piece.tiles, kTok);
      more = advance();
      ok = kChains > 1 ? bar_wait(&c.o_done[w], last & 1, s_abort)
                       : bar_wait(&c.o_done[last & 1], (last >> 1) & 1, s_abort);
      tc_fence_after();
      __syncwarp();
      if ((warp & 3) * 32 < done_rows) {
        const bool act = row < done_rows && done_room;
        float* dst = p.part_o + (int64_t)done_part * p.dim;
#pragma unroll 1
        for (int c0 = 0; c0 < p.dim; c0 += 32) {
          uint32_t x[32];
          tmem_ld32(x, t_o + c0);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 8)
            if (act && c0 + j < p.dim) st_256(dst + c0 + j, &x[j]);
          __syncwarp();
        }
        if (act) p.part_ml[done_part] = make_float2(m_ref, l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.o_free[w]);
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
// Join of the partials of a row: those of its prefix group and of its request's own group, each
// from a run of CTAs.
// ------------------------------------------------------------------------------------------------
constexpr int kMaxPartials = 4 * kMaxCtas;

// Where the partials of (row t, query head h) are: n[0] of the prefix, then n[1] of the request; two
// of each CTA, `chain` rows apart, where the chains took turns.
template <int kChains>
struct Partials {
  int n[2], from[2], chain[2], step;
  __device__ __forceinline__ Partials(const AttnArgs& p, const RowPlan& r, int grid, int t, int h) {
    const int head = p.by_group.div(h), g = h - head * p.group;
    const Cost cost(r.even);
    const int ctas = cost.ctas(r.cost, grid);
    step = p.piece_rows;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      n[i] = from[i] = chain[i] = 0;
      const int tiles = i ? r.tiles : r.prefix_tiles, count = i ? r.count : r.prefix_count;
      const int span = i ? r.span : r.prefix_span;  // rows of partials of a head
      if (!r.owned || tiles == 0) continue;
      const int f = (t - (i ? r.first : r.prefix_first)) * p.group + g;
      const int index = f / (kChains * kBlockRows);
      const int group = head * groups_of<kChains>(count, p.group) + index;
      const int rows = group_rows<kChains>(count, p.group, index);
      if (kChains > 1 && rows <= kBlockRows) chain[i] = rows;
      const int weight = tile_cost<kChains>(cost, count, p.group);
      const int at = (i ? r.cost0 : 0) + group * (cost.open + tiles * weight);
      const int last = at + (tiles > 1 ? cost.open + (tiles - 1) * weight : 0);
      const int c0 = plan_owner(r.cost, ctas, at), c1 = plan_owner(r.cost, ctas, last);
      const int n_ctas = min(c1 - c0 + 1, kMaxCtas);
      from[i] = (i ? r.rows0 : 0) + head * span + f + c0 * step;
      if (from[i] + (n_ctas - 1) * step + chain[i] < p.part_rows) n[i] = n_ctas * (chain[i] ? 2 : 1);
    }
  }
  __device__ __forceinline__ int64_t place(int j) const {
    const bool own = j >= n[0];
    const int k = own ? j - n[0] : j, f = own ? from[1] : from[0], c = own ? chain[1] : chain[0];
    return c ? f + (k >> 1) * step + (k & 1) * c : f + k * step;
  }
};

template <typename T>
__device__ __forceinline__ void write_row(const AttnArgs& p, int t, int h, int col, const float4& acc,
                                          float sum) {
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  T* out = static_cast<T*>(p.out) + ((int64_t)t * p.q_heads + h) * p.dim + col * 4;
  out[0] = T(acc.x * inv), out[1] = T(acc.y * inv), out[2] = T(acc.z * inv), out[3] = T(acc.w * inv);
}
template <typename T>
__device__ __forceinline__ void write_lse(const AttnArgs& p, int t, int h, float top, float sum) {
  // log2(sum) near its smallest, where the maxima were: the scaling is exact
  constexpr float kScale = Pair<T>::kTop == 0.f ? 1.f : 1.f / (float)(1 << (int)Pair<T>::kTop);
  p.lse[(int64_t)t * p.q_heads + h] =
      sum == 0.f ? neg_inf() : ((top + Pair<T>::kTop) + log2f(sum * kScale)) * kLn2;
}

// Few rows, many partials: one block per (row, query head). kThreads / kCols threads (8, or 16 at
// dimension 64) take the partials in turn, a thread four dimensions of each; the first loads of O are on their way before
// the weights are known. Sums run over fixed sets in a fixed order.
template <typename T, int kCols, int kThreads, int kChains>
__global__ void __launch_bounds__(kThreads) join_kernel(const AttnArgs p, int grid) {
  constexpr int kWarps = kThreads / 32, kTeams = kThreads / kCols, kAhead = 4;
  __shared__ float s_w[kMaxPartials];
  __shared__ float s_red[2][kWarps];
  __shared__ float4 s_acc[kThreads];
  const int t = blockIdx.x / p.q_heads, h = blockIdx.x - t * p.q_heads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = threadIdx.x % kCols, team = threadIdx.x / kCols;
  const bool col_in = col * 4 < p.dim;
  grid_dep_wait();
  grid_dep_launch();
  const Partials<kChains> at(p, p.row_plan[t], grid, t, h);
  const int total = at.n[0] + at.n[1];
  float4 x[kAhead];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = j0 + k * kTeams;
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j < total && col_in) x[k] = *reinterpret_cast<const float4*>(p.part_o + at.place(j) * p.dim + col * 4);
    }
  };
  constexpr int kMine = (kMaxPartials + kThreads - 1) / kThreads;
  float2 ml[kMine];
  float top = neg_inf();
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int j = threadIdx.x + k * kThreads;
    ml[k] = make_float2(neg_inf(), 0.f);
    if (j < total) ml[k] = p.part_ml[at.place(j)];
  }
  fetch(team);
#pragma unroll
  for (int k = 0; k < kMine; ++k) top = fmaxf(top, ml[k].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  if (lane == 0) s_red[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_red[0][w]);
  const float safe = top == neg_inf() ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int j = threadIdx.x + k * kThreads;
    const float w = ex2(ml[k].x - safe);
    if (j < total) s_w[j] = w;
    sum += ml[k].y * w;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
  if (lane == 0) s_red[1][warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += s_red[1][w];
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j0 = team; j0 < total; j0 += kAhead * kTeams) {
    if (j0 != team) fetch(j0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = j0 + k * kTeams;
      if (j >= total) continue;
      const float w = s_w[j];
      if (w == 0.f) continue;  // an empty partial has no O
      acc.x += x[k].x * w, acc.y += x[k].y * w, acc.z += x[k].z * w, acc.w += x[k].w * w;
    }
  }
  s_acc[threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.x < kCols && col_in) {
    for (int k = 1; k < kTeams; ++k) {
      const float4 y = s_acc[k * kCols + threadIdx.x];
      acc.x += y.x, acc.y += y.y, acc.z += y.z, acc.w += y.w;
    }
    write_row<T>(p, t, h, col, acc, sum);
  }
  if (threadIdx.x == 0) write_lse<T>(p, t, h, top, sum);
}

// Many rows, few partials each: one warp per (row, query head), 32 partials at a time.
constexpr int kJoinWarps = 8;

template <typename T, int kCols, int kChains>
__global__ void __launch_bounds__(kJoinWarps * 32) join_rows_kernel(const AttnArgs p, int grid) {
  constexpr int kMine = (kCols + 31) / 32, kAhead = 4;
  const int lane = threadIdx.x & 31, i = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  grid_dep_wait();
  grid_dep_launch();
  if (i >= p.rows * p.q_heads) return;
  const int t = i / p.q_heads, h = i - t * p.q_heads;
  const Partials<kChains> at(p, p.row_plan[t], grid, t, h);
  const int total = at.n[0] + at.n[1];
  float top = neg_inf(), sum = 0.f;
  float4 acc[kMine];
#pragma unroll
  for (int c = 0; c < kMine; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j0 = 0; j0 < total; j0 += 32) {
    const int n = min(32, total - j0);
    float2 ml = make_float2(neg_inf(), 0.f);
    if (lane < n) ml = p.part_ml[at.place(j0 + lane)];
    float m = ml.x;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    m = fmaxf(m, top);
    const float safe = m == neg_inf() ? 0.f : m, f = ex2(top - safe), w = ex2(ml.x - safe);
    top = m;
    float part = ml.y * w;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(~0u, part, d);
    sum = sum * f + part;
#pragma unroll
    for (int c = 0; c < kMine; ++c) acc[c].x *= f, acc[c].y *= f, acc[c].z *= f, acc[c].w *= f;
    for (int j = 0; j < n; j += kAhead) {
      float4 x[kAhead][kMine];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int c = 0; c < kMine; ++c) {
          const int col = lane + 32 * c;
          x[k][c] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (j + k < n && col * 4 < p.dim)
            x[k][c] = *reinterpret_cast<const float4*>(p.part_o + at.place(j0 + j + k) * p.dim + col * 4);
        }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float v = __shfl_sync(~0u, w, (j + k) & 31);
        if (j + k >= n || v == 0.f) continue;  // an empty partial has no O
#pragma unroll
        for (int c = 0; c < kMine; ++c) {
          acc[c].x += x[k][c].x * v, acc[c].y += x[k][c].y * v;
          acc[c].z += x[k][c].z * v, acc[c].w += x[k][c].w * v;
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kMine; ++c)
    if ((lane + 32 * c) * 4 < p.dim) write_row<T>(p, t, h, lane + 32 * c, acc[c], sum);
  if (lane == 0) write_lse<T>(p, t, h, top, sum);
}

int round_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// Rows of the largest piece, and of partials in all, with so many chains: every row is in a group of the
// prefix and in one of its request, and has a partial for each chain at most.
int piece_rows_for(int rows, int group, int chains) {
  return std::min(chains * kBlockRows, chains * rows * group);
}
int part_rows_for(int rows, int group, int kv_heads, int chains) {
  return 2 * chains * rows * group * kv_heads + kMaxCtas * piece_rows_for(rows, group, chains);
}
// The workspace: row plans, statistics and outputs of the partials. Two chains, where the head
// dimension allows them, take the more of it.
struct Layout {
  size_t ml, o, bytes;
  Layout(int rows, int q_heads, int kv_heads, int dim) {
    const size_t n = part_rows_for(rows, q_heads / kv_heads, kv_heads, round_dim(dim) <= 128 ? 2 : 1);
    auto aligned = [](size_t b) { return (b + 255) & ~(size_t)255; };
    ml = aligned(rows * sizeof(RowPlan));
    o = ml + aligned(n * sizeof(float2));
    bytes = o + n * dim * sizeof(float);
  }
};

template <typename T, int kDim, bool kTma>
int launch_typed(const CUtensorMap& mk, const CUtensorMap& mv, AttnArgs& p, int ctas,
                 cudaStream_t stream) {
  using S = Shape<kDim, kTma>;
  constexpr int kChains = S::kChains;
  constexpr size_t smem = attn_smem<kDim, kTma>();
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  p.part_rows = part_rows_for(p.rows, p.group, p.kv_heads, kChains);
  p.piece_rows = piece_rows_for(p.rows, p.group, kChains);
  auto kernel = attn_kernel<T, kDim, kTma>;
  static bool configured[64] = {};
  int dev = 0;
  B2_CUDA_TRY(cudaGetDevice(&dev));
  if (!configured[dev]) {
    B2_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured[dev] = true;
  }
  int rc = launch_kernel(kernel, ctas, S::kThreads, smem, stream, /*early=*/true, mk, mv, p);
  if (rc) return rc;
  // A warp each where there are many rows with few partials, else a block each: 8192 rows of dimension
  // 128 with 5 partials take 10 us against 35; 384 rows with 37 partials 16 us against 6. Of a prefix a row has
  // about as many partials as CTAs work on its group.
  const int64_t groups = p.kv_heads * (((int64_t)p.rows * p.group + kChains * kBlockRows - 1) /
                                       (kChains * kBlockRows));
  const int grid = p.rows * p.q_heads;
  if (grid > 3 * ctas && ctas <= 24 * groups)
    return launch_kernel(join_rows_kernel<T, kDim / 4, kChains>, (grid + kJoinWarps - 1) / kJoinWarps,
                         kJoinWarps * 32, 0, stream, /*early=*/true, p, ctas);
  // 8 partials at a time: 384 rows of dimension 128 with 512 threads 1.1 us more, with 128 threads
  // 1.7 us; 192 rows of dimension 256 with 256 threads 2 us more.
  constexpr int kJoin = kDim == 256 ? 512 : 256;
  return launch_kernel(join_kernel<T, kDim / 4, kJoin, kChains>, grid, kJoin, 0, stream, /*early=*/true, p,
                       ctas);
}

// A cache as a tensor map (dimension, place in the page, head, page), boxes of box_rows tokens and
// 64 dimensions. False where TMA cannot take it; the kernel then copies with cp.async.
template <typename T>
bool cache_map(CUtensorMap* map, const void* base, const int64_t* s, const AttnArgs& p) {
  const uint64_t dims[4] = {(uint64_t)p.dim, (uint64_t)p.page_size, (uint64_t)p.kv_heads,
                            (uint64_t)p.total_pages};
  uint64_t strides[3] = {(uint64_t)s[1] * 2, (uint64_t)s[2] * 2, (uint64_t)s[0] * 2};
  for (int i = 0; i < 3; ++i) {
    const int64_t e = i == 0 ? s[1] : i == 1 ? s[2] : s[0];
    if (dims[i + 1] == 1) strides[i] = (uint64_t)p.dim * 2;  // never stepped
    else if (e <= 0 || e >= (int64_t)1 << 38) return false;
  }
  const uint32_t box[4] = {64, (uint32_t)p.box_rows, 1, 1};
  return encode_4d(map, Pair<T>::kFormat == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                   base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B) == B2_OK;
}

// TMA where a page holds whole groups of 8 tokens (the rows of one swizzle pattern); a box then
// never crosses a page.
template <typename T, int kDim>
int launch_dim(AttnArgs& p, int ctas, cudaStream_t stream) {
  CUtensorMap mk = {}, mv = {};
  p.box_rows = std::min(Shape<kDim, true>::kTok, p.page_size & -p.page_size);
  if (p.box_rows >= 8 && p.dim >= 64 && cache_map<T>(&mk, p.k, p.ks, p) &&
      cache_map<T>(&mv, p.v, p.vs, p))
    return launch_typed<T, kDim, true>(mk, mv, p, ctas, stream);
  return launch_typed<T, kDim, false>(mk, mv, p, ctas, stream);
}

template <typename T>
int launch_type(AttnArgs& p, int ctas, cudaStream_t stream) {
  switch (round_dim(p.dim)) {
    case 64: return launch_dim<T, 64>(p, ctas, stream);
    case 128: return launch_dim<T, 128>(p, ctas, stream);
    default: return launch_dim<T, 256>(p, ctas, stream);
  }
}

// Costs are counted in 32 bits, for whatever lengths the tables can hold. With b blocks of 128 rows per
// KV head: of the prefix, b groups of 2 a tile, or with two chains half as many, rounded up, of 4; of
// a request with x rows 2 a tile up to 128 rows, else 4 for every 256 begun, both at most 2 + 4 x / 128
// (x = 257: 8 of 10). The opening of a group costs two such tiles at most.
bool costs_fit(int requests, int rows, int q_heads, int kv_heads, int dim, int64_t prefix, int64_t own) {
  const int tok = round_dim(dim) == 64 ? 128 : 64;
  const int64_t b = ((int64_t)rows * (q_heads / kv_heads) + kBlockRows - 1) / kBlockRows;
  const int64_t per_prefix = 2 * b + 2, per_own = 4 * b + 2 * std::min(requests, rows);
  return kv_heads * (per_prefix * (prefix / tok + 3) + per_own * (own / tok + 3)) <= 0x7fff0000;
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

extern "C" int b2_prefix_attn_status(int clear, int* device_status) {
  using namespace b2;
  if (!device_status) return fail(B2_ERR_INVALID_ARG, "prefix_attn_status: null output");
  int v = 0;
  B2_CUDA_TRY(cudaDeviceSynchronize());
  B2_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_attn_status, sizeof(v)));
  if (clear && v) {
    const int zero = 0;
    B2_CUDA_TRY(cudaMemcpyToSymbol(g_attn_status, &zero, sizeof(zero)));
  }
  *device_status = v;
  return B2_OK;
}

extern "C" size_t b2_prefix_attn_workspace(int requests, int rows, int q_heads, int kv_heads,
                                           int head_dim) {
  using namespace b2;
  if (check_shape(requests, rows, q_heads, kv_heads, head_dim)) return 0;
  return Layout(rows, q_heads, kv_heads, head_dim).bytes;
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
  if (!(std::fabs(scale * kLog2e) <= 3.4e38f))
    return fail(B2_ERR_INVALID_ARG, "%s: scale=%g is not finite", op, (double)scale);
  if (rows == 0) return B2_OK;
  if (!q_strides || !k_strides || !v_strides || !q || !k_cache || !v_cache || !prefix_len ||
      (requests > 0 && !own_lens) || !row_start || !out || !lse || (n_prefix_pages > 0 && !prefix_pages) ||
      (max_pages > 0 && !pages))
    return fail(B2_ERR_INVALID_ARG, "%s: null pointer", op);
  if ((int64_t)n_prefix_pages * page_size > kMaxTokens || (int64_t)max_pages * page_size > kMaxTokens)
    return fail(B2_ERR_INVALID_ARG, "%s: tables of more than %d tokens", op, kMaxTokens);
  if (!aligned16(k_cache) || !aligned16(v_cache) || (reinterpret_cast<uintptr_t>(q) & 3u) != 0)
    return fail(B2_ERR_INVALID_ARG, "%s: caches must be 16-byte and q 4-byte aligned", op);
  if (q_strides[0] % 2 != 0 || q_strides[1] % 2 != 0)
    return fail(B2_ERR_INVALID_ARG, "%s: strides of q must be even", op);
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
      return fail(B2_ERR_INVALID_ARG, "%s: cache strides must be multiples of 8 elements", op);
  if (!costs_fit(requests, rows, q_heads, kv_heads, head_dim, (int64_t)n_prefix_pages * page_size,
                 (int64_t)max_pages * page_size))
    return fail(B2_ERR_INVALID_ARG, "%s: tables too long for %d rows of %d requests", op, rows, requests);
  const size_t need = b2_prefix_attn_workspace(requests, rows, q_heads, kv_heads, head_dim);
  if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u) != 0)
    return fail(B2_ERR_WORKSPACE, "%s: workspace of %zu B, need %zu B, 256-byte aligned", op, ws_bytes,
                need);
  const int group = q_heads / kv_heads;
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
  p.by_page = make_div(page_size), p.by_group = make_div(group);
  p.n_prefix_pages = n_prefix_pages, p.max_pages = max_pages;
  p.requests = requests, p.rows = rows, p.q_heads = q_heads, p.kv_heads = kv_heads, p.group = group;
  p.dim = head_dim;
  p.scale_log2 = scale * kLog2e;
  p.minus_zero = 0x8000000080000000ull;
  p.row_plan = static_cast<RowPlan*>(ws);
  const Layout layout(rows, q_heads, kv_heads, head_dim);
  p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + layout.ml);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + layout.o);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == B2_DTYPE_F16 ? launch_type<__half>(p, ctas, s)
                               : launch_type<__nv_bfloat16>(p, ctas, s);
}
