// Attention over the 8-bit paged K/V pool for few query rows at a time (decode, and short prefill chunks): the pages of
// all rows divided evenly among a fixed set of CTAs, online softmax on the warp-level tensor cores.
//
// Mathematics. With codes c and the block scales s_k, s_v of a (16-token page, KV head), score_j = s_k (q . ck_j) /
// sqrt(D) and out = sum_j p_j s_v cv_j / sum_j p_j, p_j = exp(score_j - m). The codes are exact fp16 operands, so the
// scales never touch the products: s_k multiplies a block's scores and s_v its weights.
//
// Work. A unit is one (item, KV head, tile of query rows); row r of an (item, KV head) is token r / G, head r % G, and a
// tile is 8 or 16 rows. The units' pages, end to end, are cut into gridDim.x equal stretches, one per CTA, whatever the
// rows' lengths (each CTA finds its stretch from the lengths). A CTA walks the segments of its stretch (pages of one
// unit). Its last warp fills a ring of chunks with bulk copies, running ahead across segments; the others take the
// chunks round-robin, each with a softmax state of its own, and merge through shared memory at a segment's end. A unit
// that spans CTAs leaves partials in scratch, and the last of its CTAs to arrive merges them.
//
// m16n8k16: S[16 rows x 8 tokens] = Q (A) K^T (B), O[16 rows x 8 dims] = P (A) V (B). The C fragment of S is the A
// fragment of P, so P never leaves its lane. HILO (fp32 queries): a tile is 8 rows; rows 0-7 of the instruction carry
// the leading fp16 term of q (and of p), rows 8-15 the remainder (x = hi + lo to 2^-22 relative), and the two halves of
// the accumulator are added: fp32 accuracy at no extra instruction. 16-bit queries: a tile is 16 rows; q is exact in
// fp16 once each row is scaled by a power of two, p is rounded to fp16 (2^-12 relative, below the output's rounding).
//
// What each choice is for: issue slots (a page of one head, 2 KB at D = 64, is 89 clocks of HBM time per SM and takes
// ~130 warp instructions, most of them the widening of the codes).
// - I8 keys are widened to the codes themselves, a byte permute and a subtraction for two of them. (As code + 128, by the
//   permute alone, with 128 * sum(q) taken off the scores afterwards, 256 rows of 4097 tokens took 215 us in place of 222 and
//   4 rows of 131073 194 in place of 209; but for queries of one sign that difference cancels: with q ~ N(4, 1) at
//   D = 128 outputs were 6.5e-6 and lse up to 7e-5 off, where fp32 products are 1.6e-6 and 9e-6, and these 3.5e-7 and 3e-6.)
// - p * s_v is formed relative to the largest s_v that the warp has met (vref) and scaled by 2^14, so fp16 holds it
//   whatever the cache's magnitudes: the accumulators are O * 2^14 / vref.
// - A chunk's P V is accumulated from zero by the tensor cores and added to O in fp32: the tensor cores truncate, and
//   over thousands of pages that shows (4e-6 relative at 131k tokens, 8e-7 this way). The addition is the
//   multiply-add that rescales O anyway.
//
// Measured: 256 rows of 4097 tokens, 32/8 heads of 64: 222 us, 4.9 TB/s of codes and scales (75 % of the measured copy rate)
// with other pools of that size read in between; 4 rows of 131073, 32/8 heads of 128: 209 us, 5.1 TB/s (79 %). Counters of smaller
// calls of both: issue slots 47 % and 39 % busy, 3.6 and 2.8 warps resident a scheduler and 0.8 and 0.6 of them ready: the
// latency of few warps. 48 rows of 511..16384, 28/4 heads of 128: 55 us, 4.1 TB/s: the launch, the CTAs' search for their
// stretch, the first loads and the joining of partials take about 12 us of a call that short. One row of 257 tokens: 8 us, the
// launch and one chain of loads. Walking the KV heads of the same pages side by side in neighbouring CTAs, for the sake of
// whole pages: 217 us where it took 217, 199 where it took 195, and 18.4 against 16.8 for 8 items of 5 drafted tokens.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "kv8.cuh"
#include "softmax_tile.cuh"

namespace nbl {
namespace {

using namespace kv8;

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kPScale = 16384.f;  // 2^14

template <int D, bool HILO>
struct Cfg {
  static constexpr int kCtas = D == 64 ? 3 : 2;             // per SM
  static constexpr int kConsumers = D == 64 ? 4 : 5;        // attending warps; one more issues the loads
  static constexpr int kThreads = (kConsumers + 1) * 32;
  static constexpr int kRows = HILO ? 8 : 16;        // query rows of a tile
  static constexpr int kPages = 2;                   // pages of a chunk (the loads below are written for 2)
  static constexpr int kBlock = block_bytes(D);
  static constexpr int kStageBytes = kPages * kBlock;
  static constexpr int kMergeFloats = kRows * (D + 2);  // per warp: outputs, maxima, sums
  static constexpr int kQBytes = (D / 16) * 32 * 16;    // a tile's queries in operand order
  static constexpr int kRowFloats = kRows;              // per row: the factor of its scores
  static constexpr int kFixed = kConsumers * kMergeFloats * 4 + kQBytes + kRowFloats * 4;
  // A whole number of stages for each attending warp: chunk k is warp k % kConsumers's, and so are all the chunks
  // of its stage, so a warp never waits on a barrier that is two phases behind.
  static constexpr int kStages = ((227 * 1024 / kCtas - 1152) - kFixed) / (kStageBytes + 32) / kConsumers * kConsumers;
  static constexpr int kOffMerge = (kStages * kStageBytes + 15) / 16 * 16;
  static constexpr int kOffQ = kOffMerge + kConsumers * kMergeFloats * 4;
  static constexpr int kOffRow = kOffQ + kQBytes;
  static constexpr int kOffBar = kOffRow + kRowFloats * 4;   // full[kStages], empty[kStages]
  static constexpr int kOffMask = kOffBar + kStages * 16;    // pages of the stage that were loaded
  static constexpr int kSmemBytes = kOffMask + kStages * 4;
  static constexpr int kBatch = D == 64 ? 8 : 4;  // pages that the loading warp issues at once
  // What a segment costs besides its pages, in pages (a CTA attends 4-7 pages a microsecond; a segment's start, merge and
  // store take 2-4 us). Units up to kSnapPages long are not cut.
  static constexpr int kSegCost = 16, kSnapPages = 48;
  static_assert(kOffQ % 16 == 0 && kOffBar % 8 == 0 && kStages >= kConsumers, "layout");
};

struct AttnArgs {
  Kv8Items it;
  const void* q;
  void* out;
  float* lse;
  const uint8_t* pool;
  float* part;       // [CTA][2][rows * (D + 2)]: a CTA's first and last segment, where they are part of a unit
  unsigned* counts;  // [CTA] arrivals at the unit that starts in the CTA and goes on in others; 0 between launches
  int* err;
  int64_t n_pages;
  int q_dtype, out_dtype;
  int n_heads, n_kv_heads, group;
  int tile0, n_tiles;  // the items' query tiles of this launch
  Divisor by_group, by_kv_heads;
  int q_vec;         // q allows 4-element loads
  float scale_log2;  // log2(e) / sqrt(D)
};

// D = A B (+ C): m16n8k16, fp16 operands, fp32 accumulation. Not volatile: the compiler may interleave independent ones.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Four consecutive elements of q as fp32.
__device__ __forceinline__ void load4q(const AttnArgs& a, int64_t i, float (&v)[4]) {
  if (!a.q_vec) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = load_as(a.q, i + k, a.q_dtype);
  } else if (a.q_dtype == NBL_F32) {
    const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + i);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + i);
    float2 p, r;
    if (a.q_dtype == NBL_F16) {
      p = __half22float2(*reinterpret_cast<const __half2*>(&x.x));
      r = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
    } else {
      p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x.x));
      r = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x.y));
    }
    v[0] = p.x, v[1] = p.y, v[2] = r.x, v[3] = r.y;
  }
}

__device__ __forceinline__ void split_half2(float2 x, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  const float2 r = __ffma2_rn(__half22float2(h), make_float2(-1.f, -1.f), x);  // exact
  lo = pack2<false>(r.x, r.y);
}

// An item's rows and keys as the kernel takes them; pages 0 when there is nothing to do.
struct Item {
  int q_start, q_len, pos0, pages, subs;
};

template <int ROWS>
__device__ __forceinline__ Item load_item(const AttnArgs& a, int i) {
  Item x;
  const int64_t max_kv = int64_t(a.it.pt_stride) * kPage;
  if (a.it.len) {
    x.q_start = a.it.start[i], x.q_len = a.it.len[i], x.pos0 = a.it.pos0[i];
    const int64_t kv = int64_t(x.pos0) + x.q_len;
    const bool ok = item_fits(a.it, x.q_start, x.q_len, x.pos0);
    if (x.q_len > 0 && !ok) flag_error(a.err, kErrLength);
    x.pages = x.q_len > 0 && ok ? static_cast<int>((kv + kPage - 1) / kPage) : 0;
    if (x.pages == 0) x.q_len = 0;
  } else {  // a decode row of pos0[i] keys
    int len = a.it.pos0[i];
    if (len < 0 || len > max_kv) {
      flag_error(a.err, kErrLength);
      len = len < 0 ? 0 : static_cast<int>(max_kv);
    }
    x.q_start = i, x.q_len = 1, x.pos0 = len - 1;
    x.pages = (len + kPage - 1) / kPage;
  }
  x.subs = a.n_kv_heads * min(max((x.q_len * a.group + ROWS - 1) / ROWS - a.tile0, 0), a.n_tiles);  // ROWS: 8 or 16
  if (x.subs == 0) x.pages = 0;
  return x;
}

// Where a stretch stands: unit (item, sub), the unit'th of all, and the segment [page, page + seg) of it; rem pages after
// the segment.
struct Cursor {
  int item, sub, unit, page, seg, rem;
  Item x;
};
template <int ROWS>
__device__ __forceinline__ void next_segment(const AttnArgs& a, Cursor& c) {
  ++c.sub;
  ++c.unit;
  c.page = 0;
  if (c.sub >= c.x.subs) {
    c.sub = 0;
    do {
      c.x = load_item<ROWS>(a, ++c.item);
    } while (c.x.pages == 0);  // rem > 0: some later item has pages
  }
  c.seg = min(c.x.pages, c.rem);
  c.rem -= c.seg;
}

template <int D, int KIND, bool HILO>
__global__ void __launch_bounds__(Cfg<D, HILO>::kThreads, Cfg<D, HILO>::kCtas) kv8_attn_kernel(const AttnArgs a) {
  using C = Cfg<D, HILO>;
  constexpr int kConsumers = C::kConsumers, kThreads = C::kThreads;
  constexpr int ROWS = C::kRows, NP = C::kPages;
  constexpr int NR = HILO ? 1 : 2;        // query rows whose scores a lane holds: g (and g + 8)
  constexpr int kSb = D / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_item, s_sub, s_unit, s_page, s_begin, s_end, s_pages[kThreads / 32], s_units[kThreads / 32];
  __shared__ int s_last, s_due[2][6];  // a unit whose parts this CTA may have to merge
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n_items = a.it.n_items;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + C::kStages;
  uint32_t* mask = reinterpret_cast<uint32_t*>(smem + C::kOffMask);
  if (threadIdx.x < C::kStages) {
    mbar_init(&full[threadIdx.x], 1);
    mbar_init(&empty[threadIdx.x], 1);
    fence_barrier_init();
  }

  // ---- this CTA's stretch: pages [s_begin, s_end) of the units' pages end to end. The cuts are at multiples of `per`
  // on a line where a unit takes kSegCost + its pages; a cut in the kSegCost, or inside a unit of at most kSnapPages, is
  // at the unit's start.
  int per;
  {
    const int each = (n_items + kThreads - 1) / kThreads;
    const int i0 = min(int(threadIdx.x) * each, n_items), i1 = min(i0 + each, n_items);
    int my_pages = 0, my_units = 0;
    for (int i = i0; i < i1; ++i) {
      const Item x = load_item<ROWS>(a, i);
      my_pages += x.pages * x.subs;
      my_units += x.pages ? x.subs : 0;
    }
    int pages = my_pages, units = my_units;  // up to and with this thread's items
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, pages, o), z = __shfl_up_sync(0xffffffffu, units, o);
      if (lane >= o) pages += y, units += z;
    }
    if (lane == 31) s_pages[warp] = pages, s_units[warp] = units;
    __syncthreads();
    int all_pages = 0, all_units = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) pages += s_pages[w], units += s_units[w];
      all_pages += s_pages[w], all_units += s_units[w];
    }
    const int total = all_pages + all_units * C::kSegCost;
    per = max((total + int(gridDim.x) - 1) / int(gridDim.x), C::kSegCost + 1);
    const int hi = pages + units * C::kSegCost, lo = hi - my_pages - my_units * C::kSegCost;
    // the cuts before and after this CTA, found by the threads in whose items they fall
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      const int64_t cut64 = (int64_t(blockIdx.x) + k) * per;
      const int cut = cut64 < total ? static_cast<int>(cut64) : total;
      if (cut == total) {
        if (threadIdx.x == 0) (k ? s_end : s_begin) = all_pages;
      } else if (cut >= lo && cut < hi) {
        int at = lo, pg = pages - my_pages, un = units - my_units, i = i0;
        Item x = load_item<ROWS>(a, i);
        for (;;) {
          const int cost = x.pages ? (x.pages + C::kSegCost) * x.subs : 0;
          if (cut - at < cost) break;
          at += cost, pg += x.pages * x.subs, un += x.pages ? x.subs : 0;
          x = load_item<ROWS>(a, ++i);
        }
        const int sub = (cut - at) / (x.pages + C::kSegCost), in = (cut - at) - sub * (x.pages + C::kSegCost);
        const int page = x.pages <= C::kSnapPages ? 0 : max(0, in - C::kSegCost);
        if (k) {
          s_end = pg + sub * x.pages + page;
        } else {
          s_begin = pg + sub * x.pages + page;
          s_item = i, s_sub = sub, s_unit = un + sub, s_page = page;
        }
      }
    }
    __syncthreads();
  }
  const int begin = s_begin, end = s_end;
  // Rows without keys: out 0, lse -inf (decode; an item of a prefill has at least its own keys).
  if (!a.it.len) {
    for (int i = blockIdx.x; i < n_items; i += gridDim.x) {
      if (a.it.pos0[i] > 0) continue;
      for (int u = threadIdx.x; u < a.n_heads * D; u += kThreads) store_as(a.out, int64_t(i) * a.n_heads * D + u, 0.f, a.out_dtype);
      if (a.lse)
        for (int h = threadIdx.x; h < a.n_heads; h += kThreads) a.lse[int64_t(i) * a.n_heads + h] = -INFINITY;
    }
  }
  if (begin >= end) return;

  Cursor cc;  // the segment at hand
  cc.item = s_item, cc.sub = s_sub, cc.unit = s_unit, cc.page = s_page;
  cc.x = load_item<ROWS>(a, cc.item);
  cc.seg = min(cc.x.pages - cc.page, end - begin);
  cc.rem = end - begin - cc.seg;

  if (warp == kConsumers) {
    // ================= loads: every chunk of every segment in order, as the stages become free
    const int64_t pg_bytes = page_bytes(D, a.n_kv_heads);
    int k = 0;  // chunks so far
    bool ok = true;
    for (;;) {
      const int kvh = cc.sub - a.by_kv_heads.div(cc.sub) * a.n_kv_heads;
      const int32_t* pt = a.it.page_table + int64_t(cc.item) * a.it.pt_stride + cc.page;
      const uint8_t* head = a.pool + int64_t(kvh) * C::kBlock;
      int32_t pid = lane < cc.seg ? pt[lane] : -1;  // 32 pages at a time, the next ones read ahead
      for (int p0 = 0; p0 < cc.seg && ok; p0 += 32) {
        const int32_t ahead = p0 + 32 + lane < cc.seg ? pt[p0 + 32 + lane] : -1;
        const int n = min(32, cc.seg - p0);
        for (int c0 = 0; c0 < n && ok; c0 += C::kBatch) {  // some chunks at a time, a lane for each page
          const int32_t mine = __shfl_sync(0xffffffffu, pid, c0 + (lane & (C::kBatch - 1)));
          const bool in = lane < C::kBatch && c0 + lane < n, there = in && mine >= 0 && mine < a.n_pages;
          if (in && !there) flag_error(a.err, kErrPageId);
          const int kk = k + (lane >> 1), s = kk % C::kStages;
          ok = __all_sync(0xffffffffu, !in || kk < C::kStages ||
                                           mbar_wait(&empty[s], ((kk / C::kStages) & 1) ^ 1, a.err));
          if (!ok) break;
          const uint32_t m = (__ballot_sync(0xffffffffu, there) >> (lane & ~1)) & 3u;
          if (in && (lane & 1) == 0) {
            mask[s] = m;
            mbar_arrive_expect_tx(&full[s], __popc(m) * uint32_t(C::kBlock));
          }
          __syncwarp();
          if (there)
            bulk_load(smem + s * C::kStageBytes + (lane & 1) * C::kBlock, head + int64_t(mine) * pg_bytes, C::kBlock,
                      &full[s]);
          k += (min(C::kBatch, n - c0) + 1) / 2;
        }
        pid = ahead;
      }
      if (!ok || cc.rem == 0) break;
      next_segment<ROWS>(a, cc);
    }
    // No load outlives the CTA: the last ones are waited for (bounded) whether or not a consumer attends them.
    for (int i = max(0, k - C::kStages); i < k; ++i) mbar_wait(&full[i % C::kStages], (i / C::kStages) & 1, a.err);
    return;
  }

  // ================= the attending warps
  // The queries of a segment's tile into shared memory in operand order -- 16 bytes for each k-step (4 dims of
  // every lane t) and lane -- each row over its largest power of two, so fp16 holds it whatever its magnitude; and
  // per row the factor that makes a raw product a score: raw * factor * s_k (log2 units).
  uint4* s_q = reinterpret_cast<uint4*>(smem + C::kOffQ);
  float* s_row = reinterpret_cast<float*>(smem + C::kOffRow);
  constexpr int kLanes = D / 4;                                               // threads of a row, 4 dims each
  constexpr int kQSteps = (ROWS * kLanes + kConsumers * 32 - 1) / (kConsumers * 32);
  auto read_queries = [&](const Cursor& c, float (&x)[kQSteps][4]) {
    const int t_sub = a.by_kv_heads.div(c.sub), kvh = c.sub - t_sub * a.n_kv_heads, tile = a.tile0 + t_sub;
    const int n_rows_item = c.x.q_len * a.group;
#pragma unroll
    for (int i = 0; i < kQSteps; ++i) {
      const int u = i * kConsumers * 32 + threadIdx.x;
      const int row = u / kLanes, d = (u % kLanes) * 4, r = tile * ROWS + row;
      x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
      if (row < ROWS && r < n_rows_item) {
        const int tok = a.by_group.div(r), hd = kvh * a.group + r - tok * a.group;
        load4q(a, ((int64_t(c.x.q_start) + tok) * a.n_heads + hd) * D + d, x[i]);
      }
    }
  };
  auto write_queries = [&](const float (&xs)[kQSteps][4]) {
#pragma unroll
    for (int i = 0; i < kQSteps; ++i) {
      const int u = i * kConsumers * 32 + threadIdx.x;
      if (u >= ROWS * kLanes) break;  // whole warps
      const int row = u / kLanes, d = (u % kLanes) * 4;
      const float(&x)[4] = xs[i];
      float mx = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const uint32_t e = min(max(__float_as_uint(mx) >> 23, 1u), 253u);
      // an infinity makes the row's scores NaN, as a NaN does (its own products could be -inf, like those of masked keys)
      const float inv = mx <= FLT_MAX ? __uint_as_float((254u - e) << 23) : NAN;
      // dim d = 64 sb + 16 t + 4 ks: k-step 4 sb + ks, lane (row % 8, t)
      const int at = ((d >> 6) * 4 + ((d >> 2) & 3)) * 32 + (row & 7) * 4 + ((d >> 4) & 3);
      uint32_t hi0, hi1, lo0 = 0, lo1 = 0;
      if constexpr (HILO) {
        split_half2(make_float2(x[0] * inv, x[1] * inv), hi0, lo0);
        split_half2(make_float2(x[2] * inv, x[3] * inv), hi1, lo1);
        s_q[at] = make_uint4(hi0, lo0, hi1, lo1);
      } else {
        hi0 = pack2<false>(x[0] * inv, x[1] * inv);
        hi1 = pack2<false>(x[2] * inv, x[3] * inv);
        uint32_t* w = reinterpret_cast<uint32_t*>(&s_q[at]) + (row >> 3);
        w[0] = hi0;
        w[2] = hi1;
      }
      if (d == 0) s_row[row] = __uint_as_float(e << 23) * (a.scale_log2 * unit<KIND>());
    }
  };
  // A barrier of the attending warps.
  auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); };
  float xq[kQSteps][4];
  read_queries(cc, xq);
  write_queries(xq);
  sync();
  // Four outputs of row rr of (item, KV head): dims d.. of its head.
  auto store4 = [&](int q_start, int kvh, int rr, int d, float4 v, float L, float m) {
    const int tok = a.by_group.div(rr);
    const int64_t row = (int64_t(q_start) + tok) * a.n_heads + kvh * a.group + rr - tok * a.group;
    const float inv = L == 0.f ? 0.f : 1.f / L;  // 0: no keys; NaN: a query that is not finite, and so is the row
    if (a.out_dtype == NBL_F32 && a.q_vec) {
      *reinterpret_cast<float4*>(static_cast<float*>(a.out) + row * D + d) =
          make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    } else {
      store_as(a.out, row * D + d, v.x * inv, a.out_dtype);
      store_as(a.out, row * D + d + 1, v.y * inv, a.out_dtype);
      store_as(a.out, row * D + d + 2, v.z * inv, a.out_dtype);
      store_as(a.out, row * D + d + 3, v.w * inv, a.out_dtype);
    }
    if (d == 0 && a.lse) a.lse[row] = L == 0.f ? -INFINITY : (m + log2f(L)) * kLn2;
  };
  // The unit in s_due, whose parts are all in scratch, if this CTA was the last to arrive.
  int seg_parity = 0;
  auto merge_parts = [&] {
    if (!s_last) return;
    __threadfence();
    const int* w = s_due[seg_parity];
    const int q_start = w[0], kvh = w[1], row0 = w[2], n_here = w[3], first = w[4], last = w[5];
    // CTA k's part of the unit
    auto part = [&](int k) -> const float* {
      return a.part + (int64_t(k) * 2 + (k == first ? 1 : 0)) * C::kMergeFloats;
    };
    for (int u = threadIdx.x; u < n_here * (D / 4); u += kConsumers * 32) {
      const int r = u / (D / 4), d = (u % (D / 4)) * 4;
      float mx = -INFINITY;
#pragma unroll 8
      for (int k = first; k <= last; ++k) mx = fmaxf(mx, __ldcg(part(k) + ROWS * D + r));
      const float mu = mx == -INFINITY ? 0.f : mx;  // (a sum that is NaN has a maximum of -inf, and stays NaN)
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int k = first; k <= last; ++k) {
        const float* pb = part(k);
        const float e = fast_exp2(__ldcg(pb + ROWS * D + r) - mu);
        const float4 x = __ldcg(reinterpret_cast<const float4*>(pb + r * D + d));
        L = fmaf(e, __ldcg(pb + ROWS * D + ROWS + r), L);
        O.x = fmaf(e, x.x, O.x), O.y = fmaf(e, x.y, O.y), O.z = fmaf(e, x.z, O.z), O.w = fmaf(e, x.w, O.w);
      }
      store4(q_start, kvh, row0 + r, d, O, L, mx);
    }
  };
  bool due = false;  // whether the segment before was part of a unit
  int k0 = 0;  // chunks before this segment
  bool alive = true;  // false after a wait that gave up
  float* mrg = reinterpret_cast<float*>(smem + C::kOffMerge);

  for (;;) {  // segments
    const int t_sub = a.by_kv_heads.div(cc.sub), kvh = cc.sub - t_sub * a.n_kv_heads, tile = a.tile0 + t_sub;
    const int row0 = tile * ROWS, n_rows_item = cc.x.q_len * a.group;
    const int n_here = min(ROWS, n_rows_item - row0);
    const int kv_min = cc.x.pos0 + a.by_group.div(row0) + 1;  // keys that every row of the tile sees
    float row_scale[NR];
    int lim[NR];  // keys the row sees
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      row_scale[n] = s_row[g + 8 * n];
      lim[n] = row0 + g + 8 * n < n_rows_item ? cc.x.pos0 + a.by_group.div(row0 + g + 8 * n) + 1 : 0;
    }
    float2 o[D / 8][2];  // dims (8j + 2t, 8j + 2t + 1) of row g; of row g + 8, or of row g's remainder terms
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = make_float2(0.f, 0.f);
    float m_run[NR], l_run[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) m_run[n] = -INFINITY, l_run[n] = 0.f;
    float vref = 0.f, vinv = 0.f;  // largest value scale so far, and 2^14 / it

    // Two pages at st; FULL when both are loaded and every row sees all their tokens (else `there` has a bit for each
    // loaded one, and the rows see the tokens below lim).
    auto attend = [&](auto whole, const uint8_t* st, uint32_t there, int tok0) {
      constexpr bool FULL = decltype(whole)::value;
      float2 s[NR][NP][2];  // lane's tokens (2t, 2t+1) and (8+2t, 9+2t) of each page
      float2 sc[NP];
      float c0[NP][4], c1[NP][4];
#pragma unroll
      for (int sb = 0; sb < kSb; ++sb) {
        uint4 ka[NP], kb[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const uint8_t* kp = st + j * C::kBlock + sb * 1024 + lane * 16;
          ka[j] = *reinterpret_cast<const uint4*>(kp);
          kb[j] = *reinterpret_cast<const uint4*>(kp + 512);
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint4 q = s_q[(sb * 4 + ks) * 32 + lane];
          const uint32_t q4[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const uint32_t wa = ks == 0 ? ka[j].x : ks == 1 ? ka[j].y : ks == 2 ? ka[j].z : ka[j].w;
            const uint32_t wb = ks == 0 ? kb[j].x : ks == 1 ? kb[j].y : ks == 2 ? kb[j].z : kb[j].w;
            uint32_t b0, b1;
            widen4<KIND>(wa, b0, b1);
            if (sb == 0 && ks == 0) mma_first(c0[j], q4, b0, b1);
            else mma(c0[j], q4, b0, b1);
            widen4<KIND>(wb, b0, b1);
            if (sb == 0 && ks == 0) mma_first(c1[j], q4, b0, b1);
            else mma(c1[j], q4, b0, b1);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        sc[j] = *reinterpret_cast<const float2*>(st + j * C::kBlock + scale_off(D));
        const bool got = FULL || ((there >> j) & 1u);
        if (!got) sc[j] = make_float2(0.f, 0.f);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          if constexpr (HILO) {
            s[n][j][0] = __fadd2_rn(make_float2(c0[j][0], c0[j][1]), make_float2(c0[j][2], c0[j][3]));
            s[n][j][1] = __fadd2_rn(make_float2(c1[j][0], c1[j][1]), make_float2(c1[j][2], c1[j][3]));
          } else {
            s[n][j][0] = make_float2(c0[j][2 * n], c0[j][2 * n + 1]);
            s[n][j][1] = make_float2(c1[j][2 * n], c1[j][2 * n + 1]);
          }
          if constexpr (!FULL) {
            const int tok = tok0 + j * kPage + 2 * t, see = got ? lim[n] : 0;
            if (tok >= see) s[n][j][0].x = -INFINITY;
            if (tok + 1 >= see) s[n][j][0].y = -INFINITY;
            if (tok + 8 >= see) s[n][j][1].x = -INFINITY;
            if (tok + 9 >= see) s[n][j][1].y = -INFINITY;
          }
        }
      }
      // ---- running maximum (log2 units), weights and sums
      float al[NR];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float pm = fmaxf(fmaxf(s[n][j][0].x, s[n][j][0].y), fmaxf(s[n][j][1].x, s[n][j][1].y));
          // a page with nothing to see keeps -inf (its scale may be 0, and 0 * -inf is not a number)
          const float x = pm * (row_scale[n] * sc[j].x);
          mx = fmaxf(mx, !FULL && pm == -INFINITY ? -INFINITY : x);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m_run[n], mx);
        const float mu = mn == -INFINITY ? 0.f : mn;
        al[n] = fast_exp2(m_run[n] - mu);
        m_run[n] = mn;
        float2 ps = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float f = row_scale[n] * sc[j].x;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float2 x = __ffma2_rn(s[n][j][c], make_float2(f, f), make_float2(-mu, -mu));
            float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            if constexpr (!FULL) {
              if (s[n][j][c].x == -INFINITY) p.x = 0.f;
              if (s[n][j][c].y == -INFINITY) p.y = 0.f;
            }
            s[n][j][c] = p;
            ps = __fadd2_rn(ps, p);
          }
        }
        l_run[n] = fmaf(l_run[n], al[n], ps.x + ps.y);
      }
      float vmax = sc[0].y;
#pragma unroll
      for (int j = 1; j < NP; ++j) vmax = fmaxf(vmax, sc[j].y);
      if (vmax > vref) {  // a larger value scale: the accumulators move to it
        const float f = vref / vmax;
#pragma unroll
        for (int n = 0; n < NR; ++n) al[n] *= f;
        vref = vmax;
        vinv = kPScale / vmax;
      }
      uint32_t pa[NP][4];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const float2 r = make_float2(sc[j].y * vinv, sc[j].y * vinv);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 x = __fmul2_rn(s[0][j][c], r);
          if constexpr (HILO) {
            split_half2(x, pa[j][2 * c], pa[j][2 * c + 1]);
          } else {
            const float2 y = __fmul2_rn(s[NR - 1][j][c], r);
            pa[j][2 * c] = pack2<false>(x.x, x.y);
            pa[j][2 * c + 1] = pack2<false>(y.x, y.y);
          }
        }
      }
      // ---- O = O * al + P V, 32 dims at a time
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          uint4 v4 = *reinterpret_cast<const uint4*>(st + j * C::kBlock + kPage * D + c * 512 + lane * 16);
          if constexpr (!FULL) {
            if (!((there >> j) & 1u)) v4 = uint4{};  // nothing was loaded: any finite codes will do
          }
          const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t b0, b1;
            widen4<KIND>(w[k], b0, b1);
            if (j == 0) mma_first(acc[k], pa[j], b0, b1);
            else mma(acc[k], pa[j], b0, b1);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[4 * c + k][0] = __ffma2_rn(o[4 * c + k][0], make_float2(al[0], al[0]), make_float2(acc[k][0], acc[k][1]));
          o[4 * c + k][1] =
              __ffma2_rn(o[4 * c + k][1], make_float2(al[NR - 1], al[NR - 1]), make_float2(acc[k][2], acc[k][3]));
        }
      }
    };

    const int n_chunks = (cc.seg + C::kPages - 1) / C::kPages;
    for (int i = (warp + kConsumers - k0 % kConsumers) % kConsumers; i < n_chunks && alive; i += kConsumers) {
      const int stage = (k0 + i) % C::kStages;
      alive = warp_wait_all(&full[stage], ((k0 + i) / C::kStages) & 1, a.err);
      if (!alive) break;
      const uint32_t there = mask[stage];
      const uint8_t* st = smem + stage * C::kStageBytes;
      const int tok0 = (cc.page + i * NP) * kPage;
      if (there == (1u << NP) - 1u && tok0 + NP * kPage <= kv_min) attend(std::true_type{}, st, there, tok0);
      else if (there) attend(std::false_type{}, st, there, tok0);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }
    k0 += n_chunks;

    // ---- merge the warps through shared memory; the next segment's queries are on their way meanwhile
    const Cursor done = cc;
    const bool more = cc.rem > 0;
    if (more) {
      next_segment<ROWS>(a, cc);
      read_queries(cc, xq);
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      l_run[n] += __shfl_xor_sync(0xffffffffu, l_run[n], 1);
      l_run[n] += __shfl_xor_sync(0xffffffffu, l_run[n], 2);
    }
    sync();  // every warp is done with the segment's queries, and with the merge of the segment before
    {
      float* w_o = mrg + warp * C::kMergeFloats;
      float* w_m = w_o + ROWS * D;
      const float vsc = vref * (unit<KIND>() / kPScale);
#pragma unroll
      for (int n = 0; n < NR; ++n)
        if (t == 0) {
          w_m[g + 8 * n] = m_run[n];
          w_m[ROWS + g + 8 * n] = l_run[n];
        }
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        if constexpr (HILO) {
          *reinterpret_cast<float2*>(w_o + g * D + 8 * j + 2 * t) =
              make_float2((o[j][0].x + o[j][1].x) * vsc, (o[j][0].y + o[j][1].y) * vsc);
        } else {
          *reinterpret_cast<float2*>(w_o + g * D + 8 * j + 2 * t) = make_float2(o[j][0].x * vsc, o[j][0].y * vsc);
          *reinterpret_cast<float2*>(w_o + (g + 8) * D + 8 * j + 2 * t) = make_float2(o[j][1].x * vsc, o[j][1].y * vsc);
        }
      }
    }
    if (more) write_queries(xq);
    sync();
    if (due) merge_parts();
    const bool whole = done.page == 0 && done.seg == done.x.pages;
    // a part of a unit: slot 1 where the unit starts in this CTA's stretch, else slot 0
    float* mine = a.part + (int64_t(blockIdx.x) * 2 + (done.page == 0 ? 1 : 0)) * C::kMergeFloats;
    for (int u = threadIdx.x; u < n_here * (D / 4); u += kConsumers * 32) {
      const int r = u / (D / 4), d = (u % (D / 4)) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) mx = fmaxf(mx, mrg[w * C::kMergeFloats + ROWS * D + r]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) {
        const float* wb = mrg + w * C::kMergeFloats;
        const float k = fast_exp2(wb[ROWS * D + r] - mu);  // 0 for warps that saw no key
        const float4 x = *reinterpret_cast<const float4*>(wb + r * D + d);
        L = fmaf(k, wb[ROWS * D + ROWS + r], L);
        O.x = fmaf(k, x.x, O.x), O.y = fmaf(k, x.y, O.y), O.z = fmaf(k, x.z, O.z), O.w = fmaf(k, x.w, O.w);
      }
      if (whole) {
        store4(done.x.q_start, kvh, row0 + r, d, O, L, mx);
      } else {
        *reinterpret_cast<float4*>(mine + r * D + d) = O;
        if (d == 0) {
          mine[ROWS * D + r] = mx;
          mine[ROWS * D + ROWS + r] = L;
        }
      }
    }
    due = !whole;
    if (due) {
      // The CTAs whose stretches hold the unit: first .. last (page p of a unit that starts at `at` on the cuts' line is
      // behind the cuts up to at + kSegCost + p). The last of them to arrive merges; the counter (of the first) wraps
      // back to 0 for the next launch. Only warp 0 waits for the arrival; the merge is done at the next barrier.
      const int at = end - done.rem - done.seg - done.page + done.unit * C::kSegCost + C::kSegCost;
      const int first = at / per, last = (at + done.x.pages - 1) / per;
      seg_parity ^= 1;
      __threadfence();
      if (warp == 0) {
        asm volatile("bar.sync 2, %0;" ::"n"(kConsumers * 32) : "memory");
        if (lane == 0) {
          s_last = atomicInc(&a.counts[first], static_cast<unsigned>(last - first)) == static_cast<unsigned>(last - first);
          int* d = s_due[seg_parity];
          d[0] = done.x.q_start, d[1] = kvh, d[2] = row0, d[3] = n_here, d[4] = first, d[5] = last;
        }
      } else {
        asm volatile("bar.arrive 2, %0;" ::"n"(kConsumers * 32) : "memory");
      }
    }
    if (!more) break;
  }
  if (due) {
    sync();
    merge_parts();
  }
}

template <int D, int KIND, bool HILO>
void launch_t(cudaStream_t st, const AttnArgs& a, int grid) {
  using C = Cfg<D, HILO>;
  static std::atomic<uint64_t> configured{0};  // one bit per device
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(configured.load() & bit)) {
    check_cuda(cudaFuncSetAttribute(kv8_attn_kernel<D, KIND, HILO>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    C::kSmemBytes),
               "kv8 attention smem attribute");
    configured.fetch_or(bit);
  }
  kv8_attn_kernel<D, KIND, HILO><<<grid, C::kThreads, C::kSmemBytes, st>>>(a);
}

template <int D, int KIND>
void launch_q(cudaStream_t st, const AttnArgs& a, int grid) {
  if (a.q_dtype == NBL_F32) launch_t<D, KIND, true>(st, a, grid);
  else launch_t<D, KIND, false>(st, a, grid);
}

// Pages of a CTA's stretch at least, CTAs that fit an SM, and floats of a part, for (head_dim, fp32 queries).
template <class F>
auto with_cfg(int d, bool hilo, F&& f) {
  if (d == 64) return hilo ? f(Cfg<64, true>{}) : f(Cfg<64, false>{});
  return hilo ? f(Cfg<128, true>{}) : f(Cfg<128, false>{});
}

}  // namespace

namespace {
constexpr size_t kCountBytes = 4096;  // of the counters
}

size_t kv8_attn_scratch(int num_sms) {
  size_t most = 0;
  for (int d : {64, 128})
    for (bool hilo : {false, true})
      with_cfg(d, hilo, [&](auto cfg) {
        using C = decltype(cfg);
        const size_t ctas = size_t(num_sms) * C::kCtas;
        if (ctas * sizeof(unsigned) > kCountBytes) fail(NBL_E_UNSUPPORTED, "8-bit attention: more SMs than its counters are for");
        most = std::max(most, ctas * 2 * C::kMergeFloats * sizeof(float));
      });
  return kCountBytes + most;
}

Kv8AttnPlan plan_kv8_attn(const nbl_kv* kv, int n_items, int max_len, int n_heads, int max_kv, int q_dtype,
                          int num_sms) {
  return with_cfg(kv->cfg.head_dim, q_dtype == NBL_F32, [&](auto cfg) {
    using C = decltype(cfg);
    Kv8AttnPlan p;
    p.seg_cost = C::kSegCost;
    const int64_t tiles = p.tiles = (int64_t(max_len) * (n_heads / kv->cfg.n_kv_heads) + C::kRows - 1) / C::kRows;
    const int64_t max_pages = std::max(1, (max_kv + kPage - 1) / kPage);
    // one wave of CTAs, or one for each kSegCost + 1 of the most that the call can cost
    const double bound = double(n_items) * kv->cfg.n_kv_heads * double(tiles) * (double(max_pages) + C::kSegCost) / (C::kSegCost + 1);
    const int slots = num_sms * C::kCtas;
    p.grid = bound >= slots ? slots : std::max(1, static_cast<int>(std::ceil(bound)));
    return p;
  });
}

void launch_kv8_attn(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, const void* q, int q_dtype, int n_heads,
                     void* out, int out_dtype, float* lse, const Kv8AttnPlan& plan, void* scratch, int* err) {
  const auto& c = kv->cfg;
  AttnArgs a{};
  a.it = items;
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.pool = static_cast<const uint8_t*>(kv->pool);
  a.counts = static_cast<unsigned*>(scratch);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + kCountBytes);
  a.err = err;
  a.n_pages = c.n_pages;
  a.q_dtype = q_dtype;
  a.out_dtype = out_dtype;
  a.n_heads = n_heads;
  a.n_kv_heads = c.n_kv_heads;
  a.group = n_heads / c.n_kv_heads;
  a.by_group = Divisor(static_cast<uint32_t>(a.group));
  a.by_kv_heads = Divisor(static_cast<uint32_t>(c.n_kv_heads));
  const uintptr_t bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out);
  a.q_vec = (bits & 15u) == 0;
  a.scale_log2 = 1.4426950408889634f / std::sqrt(static_cast<float>(c.head_dim));
  // The kernel counts the pages of all units in 32 bits: a launch takes as many items and query tiles as that allows, were
  // every item as long as its page-table row (one launch but for many fp32 queries or very wide tables).
  const int64_t cost = int64_t(c.n_kv_heads) * (items.pt_stride + plan.seg_cost), most = 2000000000;
  if (cost > most) fail(NBL_E_INVALID, "attention: over 2^31 pages of all heads in a page-table row");
  const int64_t tiles = std::min(plan.tiles, most / cost), n = std::min<int64_t>(items.n_items, most / (cost * tiles));
  for (int64_t i = 0; i < items.n_items; i += n) {
    a.it.n_items = static_cast<int>(std::min(n, items.n_items - i));
    a.it.page_table = items.page_table + i * items.pt_stride;
    a.it.pos0 = items.pos0 + i;
    if (items.len) {
      a.it.start = items.start + i, a.it.len = items.len + i;
    } else {
      const int64_t row = int64_t(n_heads) * c.head_dim;
      a.q = static_cast<const float*>(q) + i * row, a.out = static_cast<float*>(out) + i * row;
      if (lse) a.lse = lse + i * n_heads;
    }
    for (int64_t t = 0; t < plan.tiles; t += tiles) {
      a.tile0 = static_cast<int>(t), a.n_tiles = static_cast<int>(tiles);
      if (c.head_dim == 64) {
        if (c.dtype == NBL_I8) launch_q<64, NBL_I8>(st, a, plan.grid);
        else launch_q<64, NBL_E4M3>(st, a, plan.grid);
      } else {
        if (c.dtype == NBL_I8) launch_q<128, NBL_I8>(st, a, plan.grid);
        else launch_q<128, NBL_E4M3>(st, a, plan.grid);
      }
    }
  }
  check_cuda(cudaGetLastError(), "kv8 attention launch");
}

}  // namespace nbl
