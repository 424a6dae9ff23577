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
// unit); its 4 warps take a segment's chunks round-robin, each with a private ring in shared memory that bulk copies
// keep filled across segments, and a softmax state of its own. At a segment's end the warps merge through shared
// memory; a unit that spans CTAs leaves partials in scratch, and the last of its CTAs to arrive merges them.
//
// m16n8k16: S[16 rows x 8 tokens] = Q (A) K^T (B), O[16 rows x 8 dims] = P (A) V (B). The C fragment of S is the A
// fragment of P, so P never leaves its lane. HILO (fp32 queries): a tile is 8 rows; rows 0-7 of the instruction carry
// the leading fp16 term of q (and of p), rows 8-15 the remainder (x = hi + lo to 2^-22 relative), and the two halves of
// the accumulator are added: fp32 accuracy at no extra instruction. 16-bit queries: a tile is 16 rows; q is exact in
// fp16 once each row is scaled by a power of two, p is rounded to fp16 (2^-12 relative, below the output's rounding).
//
// What each choice is for: issue slots (a page of one head, 2 KB at D = 64, is 89 clocks of HBM time per SM and takes
// ~130 warp instructions, most of them the widening of the codes).
// - I8 keys are widened by the byte permute alone: code + 128 in the low bits of an fp16 is (code + 128) * 2^-24, a
//   subnormal, and the 128 * sum(q) it adds to a score is a constant of the row, taken off in the exponent's
//   fused multiply-add. (Values would lose accuracy that way: sum(p v) is far smaller than 128 sum(p).)
// - p * s_v is formed relative to the largest s_v that the warp has met (vref) and scaled by 2^14, so fp16 holds it
//   whatever the cache's magnitudes: the accumulators are O * 2^14 / vref.
// - A chunk's P V is accumulated from zero by the tensor cores and added to O in fp32: the tensor cores truncate, and
//   over thousands of pages that shows (4e-6 relative at 131k tokens, 8e-7 this way). The addition is the
//   multiply-add that rescales O anyway.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kv8.cuh"

namespace nbl {
namespace {

using namespace kv8;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kPScale = 16384.f;  // 2^14

template <int D, bool HILO>
struct Cfg {
  static constexpr int kRows = HILO ? 8 : 16;           // query rows of a tile
  static constexpr int kPages = D == 64 ? 4 : 2;        // pages of a chunk
  static constexpr int kStages = D == 64 || !HILO ? 2 : 3;
  static constexpr int kCtasPerSm = D == 64 && HILO ? 3 : 2;
  static constexpr int kBlock = block_bytes(D);
  static constexpr int kStageBytes = kPages * (kBlock + 16);
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kMergeFloats = kRows * (D + 2);  // per warp: outputs, maxima, sums
  static constexpr int kOffMerge = kRingBytes;
  static constexpr int kOffBar = kOffMerge + kWarps * kMergeFloats * 4;
  static constexpr int kSmemBytes = kOffBar + kWarps * kStages * 8;
  static constexpr int kMinPages = kWarps * kPages;     // fewest pages of a CTA's stretch
  static constexpr int kSnapPages = 3 * kMinPages;      // units up to this long are not cut
};

// n / d for 0 <= n < 2^31 by a multiplication (the divisors are a call's constants): with 2^l >= d, the quotient is
// (n + floor(n m / 2^32)) >> l for m = floor(2^32 (2^l - d) / d) + 1.
struct FastDiv {
  uint32_t d = 1, m = 1, l = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((uint64_t(1) << l) < d) ++l;
    m = static_cast<uint32_t>((uint64_t(1) << 32) * ((uint64_t(1) << l) - d) / d + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), m) + static_cast<uint32_t>(n)) >> l);
  }
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
  FastDiv by_group, by_kv_heads;
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

__device__ __forceinline__ uint32_t pack(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void split_half2(float2 x, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  const float2 r = __ffma2_rn(__half22float2(h), make_float2(-1.f, -1.f), x);  // exact
  lo = pack(r.x, r.y);
}

// Four key codes as two fp16 pairs times key_unit<KIND>, plus the row's constant (see the file comment).
template <int KIND>
__device__ __forceinline__ void widen4_key(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == NBL_I8) {
    lo = __byte_perm(w, 0u, 0x4140);
    hi = __byte_perm(w, 0u, 0x4342);
  } else {
    widen4<KIND>(w, lo, hi);
  }
}
template <int KIND>
constexpr float key_unit() {  // what a score in those units is multiplied by
  return KIND == NBL_I8 ? 16777216.f : unit<KIND>();
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
    const bool ok = x.pos0 >= 0 && x.q_start >= 0 && int64_t(x.q_start) + x.q_len <= a.it.n_rows && kv <= max_kv;
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
  x.subs = a.n_kv_heads * ((x.q_len * a.group + ROWS - 1) / ROWS);  // ROWS: 8 or 16
  return x;
}

// Where a stretch stands: unit (item, sub) and the segment [page, page + seg) of it; rem pages after the segment.
struct Cursor {
  int item, sub, page, seg, rem;
  Item x;
};
template <int ROWS>
__device__ __forceinline__ void next_segment(const AttnArgs& a, Cursor& c) {
  ++c.sub;
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
__global__ void __launch_bounds__(kThreads, Cfg<D, HILO>::kCtasPerSm) kv8_attn_kernel(const AttnArgs a) {
  using C = Cfg<D, HILO>;
  constexpr int ROWS = C::kRows, NP = C::kPages;
  constexpr int NR = HILO ? 1 : 2;  // query rows whose scores a lane holds: g (and g + 8)
  constexpr int kSb = D / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_item, s_sub, s_page, s_begin, s_end, s_flag, s_sum[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n_items = a.it.n_items;

  // ---- this CTA's stretch [s_begin, s_end) of the units' pages end to end: `per` pages from blockIdx.x * per on, but a
  // cut inside a unit of at most kSnapPages moves to the unit's start
  int total, per;
  {
    const int each = (n_items + kThreads - 1) / kThreads;
    const int i0 = min(int(threadIdx.x) * each, n_items), i1 = min(i0 + each, n_items);
    int mine = 0;
    for (int i = i0; i < i1; ++i) {
      const Item x = load_item<ROWS>(a, i);
      mine += x.pages * x.subs;
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s_sum[warp] = inc;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) inc += s_sum[w];
      total += s_sum[w];
    }
    per = max((total + int(gridDim.x) - 1) / int(gridDim.x), C::kMinPages);
    // the cuts before and after this CTA, found by the threads in whose items they fall
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t cut64 = (int64_t(blockIdx.x) + k) * per;
      const int cut = cut64 < total ? static_cast<int>(cut64) : total;
      if (cut == total) {
        if (threadIdx.x == 0) (k ? s_end : s_begin) = total;
      } else if (cut >= inc - mine && cut < inc) {
        int at = inc - mine, i = i0;
        Item x = load_item<ROWS>(a, i);
        while (cut - at >= x.pages * x.subs) {
          at += x.pages * x.subs;
          x = load_item<ROWS>(a, ++i);
        }
        const int sub = (cut - at) / x.pages, page = x.pages <= C::kSnapPages ? 0 : (cut - at) - sub * x.pages;
        if (k) {
          s_end = at + sub * x.pages + page;
        } else {
          s_begin = at + sub * x.pages + page;
          s_item = i, s_sub = sub, s_page = page;
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

  Cursor cc;  // the segment being attended
  cc.item = s_item, cc.sub = s_sub, cc.page = s_page;
  cc.x = load_item<ROWS>(a, cc.item);
  cc.seg = min(cc.x.pages - cc.page, end - begin);
  cc.rem = end - begin - cc.seg;
  Cursor ic = cc;                // the segment of the next load
  int ipos = warp * NP;          // and this warp's next chunk in it
  const int64_t pg_bytes = page_bytes(D, a.n_kv_heads);

  uint8_t* ring = smem + warp * C::kStages * C::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar) + warp * C::kStages;
  if (lane == 0) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(&bars[s], 1);
    fence_barrier_init();
  }
  __syncwarp();

  // The next chunk to load: lane j < NP gets its page j's id (-1: past the segment, -2: no such page); ikvh its head.
  // False when the stretch holds no further chunk for this warp.
  int ikvh = 0;
  auto next_chunk = [&](int32_t& pid) -> bool {
    while (ipos >= ic.seg) {
      if (ic.rem == 0) return false;
      next_segment<ROWS>(a, ic);
      ipos = warp * NP;
    }
    pid = -1;
    if (lane < NP && ipos + lane < ic.seg) {
      pid = a.it.page_table[int64_t(ic.item) * a.it.pt_stride + ic.page + ipos + lane];
      if (pid < 0 || pid >= a.n_pages) pid = -2;
    }
    ikvh = ic.sub - a.by_kv_heads.div(ic.sub) * a.n_kv_heads;
    ipos += kWarps * NP;
    return true;
  };
  // loaded: NP bits per ring stage, the pages that were loaded (the same in every lane).
  uint32_t loaded = 0;
  auto issue = [&](int stage, int32_t pid, int kvh) {
    const uint32_t there = __ballot_sync(0xffffffffu, pid >= 0);
    loaded = (loaded & ~(((1u << NP) - 1u) << (NP * stage))) | (there << (NP * stage));
    uint8_t* st = ring + stage * C::kStageBytes;
    if (lane == 0) {
      fence_proxy_async_smem();  // this warp's reads of the stage come before its next write
      mbar_arrive_expect_tx(&bars[stage], __popc(there) * (C::kBlock + 16u));
    }
    __syncwarp();
    if (pid >= 0) {
      const uint8_t* pg = a.pool + int64_t(pid) * pg_bytes;
      bulk_load(st + lane * C::kBlock, pg + int64_t(kvh) * C::kBlock, C::kBlock, &bars[stage]);
      bulk_load(st + NP * C::kBlock + lane * 16, pg + scale_off(D, a.n_kv_heads, kvh), 16, &bars[stage]);
    } else if (pid == -2) {
      flag_error(a.err, kErrPageId);
    }
  };
  int n_issued = 0;  // chunks whose loads were issued, and attended (ring stage = count % kStages)
  {
    int32_t pid[C::kStages];
    int kvh[C::kStages];
    bool go = true;
#pragma unroll
    for (int s = 0; s < C::kStages; ++s) {  // the page-table reads of all stages before the first copy
      pid[s] = -1;
      go = go && next_chunk(pid[s]);
      kvh[s] = ikvh;
      if (go) n_issued = s + 1;
    }
#pragma unroll
    for (int s = 0; s < C::kStages; ++s)
      if (s < n_issued) issue(s, pid[s], kvh[s]);
  }
  int n_done = 0;
  bool alive = true;  // false after a wait that gave up

  for (;;) {  // segments
    const int tile = a.by_kv_heads.div(cc.sub), kvh = cc.sub - tile * a.n_kv_heads;
    const int row0 = tile * ROWS, n_rows_item = cc.x.q_len * a.group;
    const int n_here = min(ROWS, n_rows_item - row0);
    const int kv_min = cc.x.pos0 + a.by_group.div(row0) + 1;  // keys that every row of the tile sees

    // ---- Q as the A operand: row g's (and row g + 8's) dims 64 sb + 16 t + 4 ks ..+3 for k-step (sb, ks)
    uint32_t qa[kSb * 4][4];
    float row_scale[NR], row_off[NR];  // score = raw * row_scale * s_k - row_off * s_k (log2 units)
    int lim[NR];                       // keys the row sees
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = row0 + g + 8 * n;
      const bool valid = r < n_rows_item;
      const int tok = valid ? a.by_group.div(r) : 0, head = kvh * a.group + (valid ? r - tok * a.group : 0);
      const int64_t base = ((int64_t(cc.x.q_start) + tok) * a.n_heads + head) * D;
      lim[n] = valid ? cc.x.pos0 + tok + 1 : 0;
      float x[kSb * 4][4];
      float mx = 0.f;
#pragma unroll
      for (int k = 0; k < kSb * 4; ++k) {
        if (valid) load4q(a, base + 64 * (k >> 2) + 16 * t + 4 * (k & 3), x[k]);
        else x[k][0] = x[k][1] = x[k][2] = x[k][3] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, fabsf(x[k][j]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // the row over its largest power of two: fp16 then holds it whatever its magnitude
      const uint32_t e = min(max(__float_as_uint(mx) >> 23, 1u), 253u);
      const float inv = __uint_as_float((254u - e) << 23);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kSb * 4; ++k) {
        uint32_t hi0, hi1, lo0 = 0, lo1 = 0;
        if constexpr (HILO) {
          split_half2(make_float2(x[k][0] * inv, x[k][1] * inv), hi0, lo0);
          split_half2(make_float2(x[k][2] * inv, x[k][3] * inv), hi1, lo1);
          qa[k][0] = hi0, qa[k][1] = lo0, qa[k][2] = hi1, qa[k][3] = lo1;
        } else {
          qa[k][n] = hi0 = pack(x[k][0] * inv, x[k][1] * inv);
          qa[k][2 + n] = hi1 = pack(x[k][2] * inv, x[k][3] * inv);
        }
        if constexpr (KIND == NBL_I8) {
          const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&hi0));
          const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&hi1));
          const float2 l0 = __half22float2(*reinterpret_cast<const __half2*>(&lo0));
          const float2 l1 = __half22float2(*reinterpret_cast<const __half2*>(&lo1));
          sum += ((f0.x + f0.y) + (f1.x + f1.y)) + ((l0.x + l0.y) + (l1.x + l1.y));
        }
      }
      const float scale = __uint_as_float(e << 23) * a.scale_log2;
      row_scale[n] = scale * key_unit<KIND>();
      row_off[n] = 0.f;
      if constexpr (KIND == NBL_I8) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        row_off[n] = 128.f * sum * scale;
      }
    }

    float2 o[D / 8][2];  // dims (8j + 2t, 8j + 2t + 1) of row g; of row g + 8, or of row g's remainder terms
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = make_float2(0.f, 0.f);
    float m_run[NR], l_run[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) m_run[n] = -INFINITY, l_run[n] = 0.f;
    float vref = 0.f, vinv = 0.f;  // largest value scale so far, and 2^14 / it

    // One chunk: FULL when all its pages are loaded and every row sees all their tokens.
    auto attend = [&](auto full, const uint8_t* st, uint32_t there, int tok0) {
      constexpr bool FULL = decltype(full)::value;
      float2 s[NR][NP][2];  // lane's tokens (2t, 2t+1) and (8+2t, 9+2t) of each page
      float2 sc[NP];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        sc[j] = *reinterpret_cast<const float2*>(st + NP * C::kBlock + j * 16);
        if constexpr (!FULL) {
          if (!((there >> j) & 1u)) {
            sc[j] = make_float2(0.f, 0.f);
#pragma unroll
            for (int n = 0; n < NR; ++n) s[n][j][0] = s[n][j][1] = make_float2(-INFINITY, -INFINITY);
            continue;
          }
        }
        float c0[4], c1[4];
#pragma unroll
        for (int sb = 0; sb < kSb; ++sb) {
          const uint8_t* kp = st + j * C::kBlock + sb * 1024 + lane * 16;
          const uint4 ka = *reinterpret_cast<const uint4*>(kp);
          const uint4 kb = *reinterpret_cast<const uint4*>(kp + 512);
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint32_t(&q4)[4] = qa[sb * 4 + ks];
            uint32_t b0, b1;
            widen4_key<KIND>(wa[ks], b0, b1);
            if (sb == 0 && ks == 0) mma_first(c0, q4, b0, b1);
            else mma(c0, q4, b0, b1);
            widen4_key<KIND>(wb[ks], b0, b1);
            if (sb == 0 && ks == 0) mma_first(c1, q4, b0, b1);
            else mma(c1, q4, b0, b1);
          }
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          if constexpr (HILO) {
            s[n][j][0] = __fadd2_rn(make_float2(c0[0], c0[1]), make_float2(c0[2], c0[3]));
            s[n][j][1] = __fadd2_rn(make_float2(c1[0], c1[1]), make_float2(c1[2], c1[3]));
          } else {
            s[n][j][0] = make_float2(c0[2 * n], c0[2 * n + 1]);
            s[n][j][1] = make_float2(c1[2 * n], c1[2 * n + 1]);
          }
          if constexpr (!FULL) {
            const int tok = tok0 + j * kPage + 2 * t;
            if (tok >= lim[n]) s[n][j][0].x = -INFINITY;
            if (tok + 1 >= lim[n]) s[n][j][0].y = -INFINITY;
            if (tok + 8 >= lim[n]) s[n][j][1].x = -INFINITY;
            if (tok + 9 >= lim[n]) s[n][j][1].y = -INFINITY;
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
          const float x = fmaf(pm, row_scale[n] * sc[j].x, -row_off[n] * sc[j].x);
          mx = fmaxf(mx, !FULL && pm == -INFINITY ? -INFINITY : x);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m_run[n], mx);
        const float mu = mn == -INFINITY ? 0.f : mn;
        al[n] = ex2(m_run[n] - mu);
        m_run[n] = mn;
        float2 ps = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float f = row_scale[n] * sc[j].x, off = fmaf(-row_off[n], sc[j].x, -mu);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float2 x = __ffma2_rn(s[n][j][c], make_float2(f, f), make_float2(off, off));
            float2 p = make_float2(ex2(x.x), ex2(x.y));
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
            pa[j][2 * c] = pack(x.x, x.y);
            pa[j][2 * c + 1] = pack(y.x, y.y);
          }
        }
      }
      // ---- O = O * al + P V, 32 dims at a time
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float acc[4][4];
        if constexpr (!FULL) {
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[k][0] = acc[k][1] = acc[k][2] = acc[k][3] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          if constexpr (!FULL) {
            if (!((there >> j) & 1u)) continue;
          }
          const uint4 v4 = *reinterpret_cast<const uint4*>(st + j * C::kBlock + kPage * D + c * 512 + lane * 16);
          const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t b0, b1;
            widen4<KIND>(w[k], b0, b1);
            if (FULL && j == 0) mma_first(acc[k], pa[j], b0, b1);
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

    for (int pos = warp * NP; pos < cc.seg && alive; pos += kWarps * NP) {
      const int stage = n_done % C::kStages;
      alive = warp_wait_all(&bars[stage], (n_done / C::kStages) & 1, a.err);
      if (!alive) break;
      ++n_done;
      // the ids of the chunk this stage takes next, read now and used below
      int32_t pid = -1;
      const bool more = next_chunk(pid);
      const int kvh_next = ikvh;
      const uint8_t* st = ring + stage * C::kStageBytes;
      const uint32_t there = (loaded >> (NP * stage)) & ((1u << NP) - 1u);
      const int tok0 = (cc.page + pos) * kPage;
      if (there == (1u << NP) - 1u && tok0 + NP * kPage <= kv_min) attend(std::true_type{}, st, there, tok0);
      else attend(std::false_type{}, st, there, tok0);
      __syncwarp();
      if (more) {
        issue(stage, pid, kvh_next);
        ++n_issued;
      }
    }

    // ---- merge the 4 warps through shared memory
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      l_run[n] += __shfl_xor_sync(0xffffffffu, l_run[n], 1);
      l_run[n] += __shfl_xor_sync(0xffffffffu, l_run[n], 2);
    }
    __syncthreads();  // the merge area is free: every warp is past the segment before
    float* mrg = reinterpret_cast<float*>(smem + C::kOffMerge);
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
    __syncthreads();
    // Row r of the tile as a row of the packed (token, head) outputs.
    auto out_row = [&](int r) -> int64_t {
      const int rr = row0 + r, tok = a.by_group.div(rr);
      return (int64_t(cc.x.q_start) + tok) * a.n_heads + kvh * a.group + rr - tok * a.group;
    };
    auto store4 = [&](int r, int d, float4 v, float L, float m) {
      const float inv = L > 0.f ? 1.f / L : 0.f;
      const int64_t row = out_row(r);
      if (a.out_dtype == NBL_F32 && a.q_vec) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + row * D + d) =
            make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      } else {
        store_as(a.out, row * D + d, v.x * inv, a.out_dtype);
        store_as(a.out, row * D + d + 1, v.y * inv, a.out_dtype);
        store_as(a.out, row * D + d + 2, v.z * inv, a.out_dtype);
        store_as(a.out, row * D + d + 3, v.w * inv, a.out_dtype);
      }
      if (d == 0 && a.lse) a.lse[row] = L > 0.f ? (m + log2f(L)) * kLn2 : -INFINITY;
    };
    const bool whole = cc.page == 0 && cc.seg == cc.x.pages;
    // a part of a unit: slot 1 where the unit starts in this CTA's stretch, else slot 0
    float* mine = a.part + (int64_t(blockIdx.x) * 2 + (cc.page == 0 ? 1 : 0)) * C::kMergeFloats;
    for (int u = threadIdx.x; u < ROWS * (D / 4); u += kThreads) {
      const int r = u / (D / 4), d = (u % (D / 4)) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, mrg[w * C::kMergeFloats + ROWS * D + r]);
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
      if (mx != -INFINITY) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float* wb = mrg + w * C::kMergeFloats;
          const float k = ex2(wb[ROWS * D + r] - mx);  // 0 for warps that saw no key
          const float4 x = *reinterpret_cast<const float4*>(wb + r * D + d);
          L = fmaf(k, wb[ROWS * D + ROWS + r], L);
          O.x = fmaf(k, x.x, O.x), O.y = fmaf(k, x.y, O.y), O.z = fmaf(k, x.z, O.z), O.w = fmaf(k, x.w, O.w);
        }
      }
      if (whole) {
        if (r < n_here) store4(r, d, O, L, mx);
      } else {
        *reinterpret_cast<float4*>(mine + r * D + d) = O;
        if (d == 0) {
          mine[ROWS * D + r] = mx;
          mine[ROWS * D + ROWS + r] = L;
        }
      }
    }
    if (!whole) {
      // The CTAs whose stretches hold the unit: first .. last. The last of them to arrive merges; the counter (of the
      // first) wraps back to 0 for the next launch.
      // (Cuts inside a unit long enough to be cut are exact multiples of `per`.)
      const int u0 = end - cc.rem - cc.seg - cc.page, u1 = u0 + cc.x.pages;  // the unit's place, pages end to end
      const int first = u0 / per, last = (u1 - 1) / per;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0)
        s_flag = atomicInc(&a.counts[first], static_cast<unsigned>(last - first)) == static_cast<unsigned>(last - first);
      __syncthreads();
      if (s_flag) {
        __threadfence();
        for (int u = threadIdx.x; u < n_here * (D / 4); u += kThreads) {
          const int r = u / (D / 4), d = (u % (D / 4)) * 4;
          // CTA k's part of the unit
          auto part = [&](int k) -> const float* {
            return a.part + (int64_t(k) * 2 + (k == first ? 1 : 0)) * C::kMergeFloats;
          };
          float mx = -INFINITY;
#pragma unroll 8
          for (int k = first; k <= last; ++k) mx = fmaxf(mx, __ldcg(part(k) + ROWS * D + r));
          float L = 0.f;
          float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
          if (mx != -INFINITY) {
#pragma unroll 4
            for (int k = first; k <= last; ++k) {
              const float* pb = part(k);
              const float w = ex2(__ldcg(pb + ROWS * D + r) - mx);
              const float4 x = __ldcg(reinterpret_cast<const float4*>(pb + r * D + d));
              L = fmaf(w, __ldcg(pb + ROWS * D + ROWS + r), L);
              O.x = fmaf(w, x.x, O.x), O.y = fmaf(w, x.y, O.y), O.z = fmaf(w, x.z, O.z), O.w = fmaf(w, x.w, O.w);
            }
          }
          store4(r, d, O, L, mx);
        }
      }
    }
    if (cc.rem == 0) break;
    next_segment<ROWS>(a, cc);
  }
  // After a wait that gave up, the loads still in flight are drained (bounded) before the CTA ends.
  for (int i = n_done; i < n_issued; ++i) mbar_wait(&bars[i % C::kStages], (i / C::kStages) & 1, a.err);
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
  kv8_attn_kernel<D, KIND, HILO><<<grid, kThreads, C::kSmemBytes, st>>>(a);
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

Kv8AttnPlan plan_kv8_attn(const nbl_kv* kv, int n_items, int max_len, int n_heads, int max_kv, int q_dtype,
                          int num_sms) {
  return with_cfg(kv->cfg.head_dim, q_dtype == NBL_F32, [&](auto cfg) {
    using C = decltype(cfg);
    Kv8AttnPlan p;
    const int64_t tiles = (int64_t(max_len) * (n_heads / kv->cfg.n_kv_heads) + C::kRows - 1) / C::kRows;
    const int64_t max_pages = std::max(1, (max_kv + kPage - 1) / kPage);
    // the most pages that the call can have, in stretches of at least kMinPages: at most one wave of CTAs
    if (double(n_items) * kv->cfg.n_kv_heads * double(tiles) * (double(kv->cfg.page_size) * double(max_pages)) > 3.0e10)
      fail(NBL_E_INVALID, "attention: over 2^31 pages of all rows, heads and query tiles in one call");
    const double bound = double(n_items) * kv->cfg.n_kv_heads * double(tiles) * double(max_pages) / C::kMinPages;
    const int slots = num_sms * C::kCtasPerSm;
    p.grid = bound >= slots ? slots : std::max(1, static_cast<int>(std::ceil(bound)));
    p.scratch_bytes = size_t(p.grid) * 2 * C::kMergeFloats * sizeof(float);
    return p;
  });
}

void launch_kv8_attn(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, const void* q, int q_dtype, int n_heads,
                     void* out, int out_dtype, float* lse, const Kv8AttnPlan& plan, void* scratch, unsigned* counts,
                     int* err) {
  const auto& c = kv->cfg;
  AttnArgs a{};
  a.it = items;
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.pool = static_cast<const uint8_t*>(kv->pool);
  a.part = static_cast<float*>(scratch);
  a.counts = counts;
  a.err = err;
  a.n_pages = c.n_pages;
  a.q_dtype = q_dtype;
  a.out_dtype = out_dtype;
  a.n_heads = n_heads;
  a.n_kv_heads = c.n_kv_heads;
  a.group = n_heads / c.n_kv_heads;
  a.by_group = FastDiv(static_cast<uint32_t>(a.group));
  a.by_kv_heads = FastDiv(static_cast<uint32_t>(c.n_kv_heads));
  const uintptr_t bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out);
  a.q_vec = (bits & 15u) == 0;
  a.scale_log2 = 1.4426950408889634f / std::sqrt(static_cast<float>(c.head_dim));
  if (c.head_dim == 64) {
    if (c.dtype == NBL_I8) launch_q<64, NBL_I8>(st, a, plan.grid);
    else launch_q<64, NBL_E4M3>(st, a, plan.grid);
  } else {
    if (c.dtype == NBL_I8) launch_q<128, NBL_I8>(st, a, plan.grid);
    else launch_q<128, NBL_E4M3>(st, a, plan.grid);
  }
  check_cuda(cudaGetLastError(), "kv8 attention launch");
}

}  // namespace nbl
