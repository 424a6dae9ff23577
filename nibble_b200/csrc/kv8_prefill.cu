// Causal attention of many query tokens over the 8-bit paged K/V pool on the 5th-generation tensor cores.
//
// Mathematics. With codes c and block scales s_k, s_v: score_j = s_k (q . ck_j) / sqrt(D), out = sum_j p_j s_v cv_j /
// sum_j p_j. The codes are exact fp16 (bf16) operands, so the tensor cores multiply codes and the scales meet scores and
// weights in fp32: a score is raw * f_b (f_b one number per 16-key block), and the weight that multiplies the value codes
// is p'_j = 2^(score + log2 s_v - M + 6), the same fused multiply-add with another addend. M is the row's largest score +
// log2 s_v (to 2^8: it moves rarely, with the accumulators), so p' <= 2^14 fits fp16, which holds it to 2^-12 relative: below
// the output's rounding, and whatever the scales of pages that the row hardly attends (with the largest s_v met in place
// of M, the values of a row that attends quiet pages after a loud one were lost). The row sum needs p without s_v: per block,
// sum(p') / s_v * 2^(M - m - 6), m being the row's largest score.
//
// Work. Persistent CTAs walk works, a work being a 128-row query tile of two or four heads of a KV group over all of its
// keys (or a part of them, see Walk). Warps:
//   softmax, one warpgroup per head: thread = query row = TMEM lane. A tile is 64 keys (4 pages).
//   converters: find the works, and bring each page's block straight from global memory (L2: the works that run at one time
//           share their keys) through registers, widened, into the MMA operands: K [64 keys][D] and V transposed,
//           [D][64 keys], both K-major with 128-byte swizzle. A block's value words hold the tokens 2t, 2t+1, 2t+8, 2t+9 of
//           a dim, so key 2t + (i & 1) + 8 (i >> 1) of a block is at place 4t + i of its V columns, and P is packed in that
//           order. They share the pages in turn and run up to three tiles ahead, across works. The first also hands the
//           works on and loads their Q tiles by TMA into one of two buffers.
//   last    MMA issuer: S_g = Q_g K^T, O_g += P_g V with P read from TMEM.
// D = 64, groups of three heads or more: four heads a CTA (TMEM is then full: S and P share 64 columns a head), so a
// converted tile serves four heads; three converting warps (with two, which also kept the pace of 4200 cycles a tile, 4
// prompts of 2048 tokens at 32/4 heads took 138 us, with three 126; a fourth would leave the others too few registers).
// Smaller groups: two heads, two CTAs per SM. D = 128: two heads fill TMEM with S double-buffered, the next tile's S is
// computed during a tile's softmax; four converting warps.
// What bounds it: at D = 64 the chain S -> max -> exponentials -> P -> P V of a head (the SFU, 16 exponentials a clock, is
// busy 50 % of the time, the tensor cores 25 %); at D = 128 the tensor cores' reading of Q and K from shared memory for
// 64-key tiles (48 cycles an instruction where the product takes 32) beside the same chain. Measured: 4 prompts of 2048
// tokens, 32/4 heads of 64: 126 us; one of 8192: 409 us, 670 TFLOP/s; at 32/8 heads of 128 572 us, 960 TFLOP/s.
// Taking the weights against the last tiles' maximum while this tile's is found (to shorten the chain) spilled registers:
// 208 us. Polynomials for one exponential in 8, 4, 3: 145, 147, 151 us where none took 138. With the works found, and Q
// fetched, by the issuing warp and the softmax warps each for itself, starting on a work took 4000 cycles, as long as a tile.
//
// Every mbarrier wait is bounded (nbl_device.cuh): a lost completion ends the CTA with kErrTimeout set.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kv8.cuh"
#include "softmax_tile.cuh"

namespace nbl {
namespace {

using namespace kv8;

constexpr int kBM = 128;                   // query rows of a tile
constexpr int kBN = 64;                    // keys of a tile
constexpr int kTilePages = kBN / kPage;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: p may reach 2^8 before the reference max moves
constexpr float kPShift = 6.0f;            // p' carries 2^6
// Smallest log2 s_v - (M - m) kept in a block's exponents, for the sum's sake: below it p' is at most 2^(8 - 40 + 6), which
// fp16 weights round to 0 as they would the smaller one.
constexpr float kMinLv = -40.0f;

constexpr int kRing = 4;                   // works handed from the first converting warp to the other roles

// A work as the issuing and the softmax warps need it.
struct alignas(16) Slot {
  int t0, n, n_g, head0;  // first tile, tiles (0: no more works), heads, the first
  int pos, row, live;     // position of the tile's first query token, its row of the output (or of the parts), rows of the tile
  int part;               // which part of the work; + kLastPart: the last one
};
constexpr int kLastPart = 1 << 16;

template <int D, int HEADS>
struct PCfg {
  static constexpr int NH = HEADS;                      // heads of a CTA
  static constexpr int kCtas = D == 64 && NH == 2 ? 2 : 1;  // per SM
  static constexpr int SB = D == 64 ? 1 : 2;            // S buffers of a head
  static constexpr int ST = 3;                          // tiles of K and V operands
  static constexpr int kConv = D == 128 ? 4 : NH == 4 ? 3 : 1;  // converting warps
  static constexpr int kAhead = kConv == 1 ? 2 : 1;     // pages whose codes are on their way
  static constexpr int kWarpConv = 4 * NH, kWarpMma = kWarpConv + kConv;
  static constexpr int kThreads = (kWarpMma + 1) * 32;
  static constexpr int kQBytes = kBM * D * 2;           // one head's Q tile: D / 64 parts of [128][64]
  static constexpr int kTileBytes = kBN * D * 2;        // K (or V) operand tile
  static constexpr int kBlock = block_bytes(D);
  static constexpr int kOffQ = 0;                       // 2 buffers x NH heads
  static constexpr int kOffKV = 2 * NH * kQBytes;
  static constexpr int kOffScale = kOffKV + ST * 2 * kTileBytes;  // [ST][4] float4
  static constexpr int kOffBar = kOffScale + ST * kTilePages * 16;
  static constexpr int kBarQFull = 0, kBarQFree = 2, kBarKVFull = 4, kBarKVEmpty = kBarKVFull + ST, kBarS = kBarKVEmpty + ST,
                       kBarP = kBarS + NH * SB, kBarODone = kBarP + NH * SB, kBarODrained = kBarODone + NH,
                       kBarPV = kBarODrained + NH, kBarWFull = kBarPV + NH, kBarWFree = kBarWFull + kRing, kNumBars = kBarWFree + kRing;
  static constexpr int kOffTmemSlot = kOffBar + ((kNumBars * 8 + 15) & ~15);
  static constexpr int kOffRing = kOffTmemSlot + 16;
  static constexpr int kSmemBytes = kOffRing + kRing * 32;
  static constexpr uint32_t kTmemCols = kCtas == 2 ? 256 : 512;
  __host__ __device__ static constexpr uint32_t col_s(int g, int buf) { return (g * SB + buf) * kBN; }
  __host__ __device__ static constexpr uint32_t col_o(int g) { return NH * SB * kBN + g * D; }
};

struct PrefillArgs {
  Kv8Items it;
  const uint8_t* pool;
  void* out;
  float *part_o, *part_lse;  // [n_splits][part_rows][heads][D] and [n_splits][part_rows][heads] when n_splits > 1
  int64_t part_rows;         // rows of q, or (fewer) n_items * max_len: a token's row is then item * max_len + its place
  int* err;
  int64_t n_pages;
  int out_dtype;
  int n_heads, n_kv_heads, group, n_hgroups, m_tiles;
  int n_splits;  // > 1: tiles are dealt evenly (Walk), a work's parts to at most so many CTAs
  Divisor by_hgroups, by_kv_heads, by_items;
  int n_works;  // query tiles x items x KV heads x head groups
  float scale_log2;
};

struct Work {
  int kvh, n_g, head0, qlen, pos0, qs, m0, t0, t1, n_item_pages;
  int out_row;  // the item's first row of the output, or of the parts
  int split;  // which part of the work this is
  const int32_t* pt_row;
  bool valid, last;  // last: the work's last part
};

// An item's first row of the parts.
__device__ __forceinline__ int part_row(const Kv8Items& it, int64_t part_rows, int item, int start) {
  return part_rows < it.n_rows ? item * it.max_len : start;
}

// Work w (-1: none); the same in every warp. Works are numbered with the query tile (latest, so heaviest, first) slowest,
// then the item, the KV head and the heads of the group: the works of a round are about equally long, whatever the
// number of items (with the item slowest, 4 prompts of 2048 tokens left the busiest CTA with 1.6 times the mean).
template <int NH>
__device__ __forceinline__ Work decode_work(const PrefillArgs& a, int w) {
  Work k{};
  k.valid = false;
  if (w < 0) return k;
  const int hg = a.by_hgroups.split(w);
  k.kvh = a.by_kv_heads.split(w);
  const int item = a.by_items.split(w);
  const int mt = a.m_tiles - 1 - w;
  k.n_g = min(NH, a.group - NH * hg);  // the last heads of a group may be fewer
  k.head0 = k.kvh * a.group + NH * hg;
  k.qlen = a.it.len[item];
  k.pos0 = a.it.pos0[item];
  k.qs = a.it.start[item];
  k.out_row = a.n_splits > 1 ? part_row(a.it, a.part_rows, item, k.qs) : k.qs;
  k.m0 = mt * kBM;
  k.valid = k.qlen > 0 && k.m0 < k.qlen;
  if (!k.valid) return k;
  const int64_t kv_len = int64_t(k.pos0) + k.qlen;
  if (!item_fits(a.it, k.qs, k.qlen, k.pos0)) {
    flag_error(a.err, kErrLength);
    k.valid = false;
    return k;
  }
  const int kv_end = static_cast<int>(min(kv_len, int64_t(k.pos0) + k.m0 + kBM));
  k.t1 = (kv_end + kBN - 1) / kBN;
  k.last = true;
  k.n_item_pages = static_cast<int>((kv_len + kPage - 1) / kPage);
  k.pt_row = a.it.page_table + int64_t(item) * a.it.pt_stride;
  return k;
}

// Which works a CTA takes; every role walks the same. Many works: rounds of gridDim.x consecutive ones; CTA c takes work c
// of even rounds and gridDim.x - 1 - c of odd ones (heavy and light query tiles of a round even out over two). Few: all
// their tiles in a row are dealt in equal shares, so a CTA has the end of one work, perhaps whole ones, and the start of
// another; the parts' results are joined afterwards (511 tokens over 16.4k, 32/8 heads of 128: 157 us; with each work's
// tiles cut in two equal parts 165).
struct Walk {
  int w = 0;                         // next work (rounds: the round's first)
  int round = 0;
  int base = 0, x = 0, end = 0;      // dealt: tiles before work w, the CTA's next tile and its end
  int share = 1;                     // tiles of a share; 0: one whole work instead
};

template <int NH>
__device__ __forceinline__ Work next_work(const PrefillArgs& a, Walk& k) {
  if (a.n_splits > 1 && k.share == 0) {
    const Work wk = decode_work<NH>(a, k.w < a.n_works ? k.w : -1);
    k.w = a.n_works;
    return wk;
  }
  if (a.n_splits > 1) {
    while (k.x < k.end && k.w < a.n_works) {
      Work wk = decode_work<NH>(a, k.w++);
      if (!wk.valid) continue;
      const int n = wk.t1;
      wk.t0 = k.x - k.base;
      wk.t1 = min(n, k.end - k.base);
      wk.split = k.x / k.share - k.base / k.share;
      wk.last = wk.t1 == n;
      k.x = k.base + wk.t1;
      k.base += n;
      return wk;
    }
  } else {
    while (k.w < a.n_works) {
      const int grid = static_cast<int>(gridDim.x), c = static_cast<int>(blockIdx.x);
      const int w = k.w + ((k.round++ & 1) ? grid - 1 - c : c);
      k.w += grid;
      const Work wk = decode_work<NH>(a, w < a.n_works ? w : -1);
      if (wk.valid) return wk;
    }
  }
  Work none{};
  none.valid = false;
  return none;
}

// The CTA's share, by a whole warp: equal shares of all tiles, of at least kMinShare tiles (or a work) each, and so that no
// work has more than n_splits parts. Starting on another work costs a CTA about kSwitch tiles; where short works make that
// dearer than leaving CTAs idle, each work goes to a CTA of its own (one prompt of 1300 tokens would otherwise end with
// works of two tiles).
constexpr int kMinShare = 8, kSwitch = 3;
template <int NH>
__device__ __forceinline__ Walk deal(const PrefillArgs& a) {
  const int lane = threadIdx.x & 31, n = a.m_tiles * a.it.n_items, per = a.n_kv_heads * a.n_hgroups;
  auto tiles_of = [&](int p) -> int {  // of each of the `per` works of query tile and item p
    if (p >= n) return 0;
    const Work wk = decode_work<NH>(a, p * per);
    return wk.valid ? wk.t1 : 0;
  };
  int total = 0, longest = 0, shortest = INT32_MAX;
  for (int p0 = 0; p0 < n; p0 += 32) {
    const int t = tiles_of(p0 + lane);
    total += __reduce_add_sync(0xffffffffu, t) * per;
    longest = max(longest, __reduce_max_sync(0xffffffffu, t));
    shortest = min(shortest, __reduce_min_sync(0xffffffffu, t > 0 ? t : INT32_MAX));
  }
  Walk k;
  const int grid = static_cast<int>(gridDim.x);
  k.share = max(max((total + grid - 1) / grid, (longest + a.n_splits - 2) / (a.n_splits - 1)), max(1, min(kMinShare, longest)));
  if (a.n_works <= grid && longest < k.share + kSwitch * ((k.share - 1) / shortest + 1)) {
    k.share = 0;
    k.w = static_cast<int>(blockIdx.x);
    return k;
  }
  k.x = min(total, k.share * static_cast<int>(blockIdx.x));
  k.end = min(total, k.x + k.share);
  for (int p0 = 0, before = 0; p0 < n && k.x < k.end; p0 += 32) {
    const int t = tiles_of(p0 + lane), mine = t * per;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > k.x);
    if (hit) {
      const int l = __ffs(hit) - 1, first = before + __shfl_sync(0xffffffffu, upto - mine, l), tl = __shfl_sync(0xffffffffu, t, l);
      const int h = (k.x - first) / tl;
      k.w = (p0 + l) * per + h;
      k.base = first + h * tl;
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return k;
}

// Four key codes as two pairs of the operand type, divided by unit<KIND>() (fp16, or bf16 for E4M3) -- exact.
template <int KIND, bool BF16>
__device__ __forceinline__ void widen4_key(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (!BF16) {
    widen4<KIND>(w, lo, hi);
  } else if constexpr (KIND == NBL_I8) {
    // byte in the low bits of 2^23, minus 2^23 + 128: the code as fp32, whose upper half is the bf16
    const float2 off = make_float2(-8388736.f, -8388736.f);
    const float2 x = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)),
                                            __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441))), off);
    const float2 y = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)),
                                            __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443))), off);
    lo = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
    hi = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x7632);
  } else {
    uint32_t a, b;
    widen4<KIND>(w, a, b);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    lo = pack2<true>(x.x, x.y);
    hi = pack2<true>(y.x, y.y);
  }
}

// One lane of the converged warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

template <int D, int HEADS, int KIND, bool BF16>
__global__ void __launch_bounds__(PCfg<D, HEADS>::kThreads, PCfg<D, HEADS>::kCtas)
    kv8_prefill_kernel(const __grid_constant__ CUtensorMap qmap, const PrefillArgs a) {
  using C = PCfg<D, HEADS>;
  constexpr int NH = C::NH, SB = C::SB, ST = C::ST;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023u) {  // 128-byte-swizzled tiles need 1024-byte alignment; never expected to trip
    if (threadIdx.x == 0) flag_error(a.err, kErrSmemAlign);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffTmemSlot);
  float4* scales = reinterpret_cast<float4*>(smem + C::kOffScale);  // (s_k, log2 s_v, 1 / s_v) of a tile's pages
  auto sQ = [&](int buf, int g) { return smem + C::kOffQ + (buf * NH + g) * C::kQBytes; };
  auto sK = [&](int s) { return smem + C::kOffKV + s * 2 * C::kTileBytes; };
  auto sV = [&](int s) { return smem + C::kOffKV + s * 2 * C::kTileBytes + C::kTileBytes; };
  auto bar_s = [&](int g, int buf) { return &bars[C::kBarS + g * SB + buf]; };
  auto bar_p = [&](int g, int buf) { return &bars[C::kBarP + g * SB + buf]; };

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars[C::kBarQFull + b], 1);
      mbar_init(&bars[C::kBarQFree + b], 4 * NH);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&bars[C::kBarWFull + i], 1);
      mbar_init(&bars[C::kBarWFree + i], 4 * NH + 1);
    }
    for (int s = 0; s < ST; ++s) {
      mbar_init(&bars[C::kBarKVFull + s], kTilePages);
      mbar_init(&bars[C::kBarKVEmpty + s], 1);
    }
    for (int g = 0; g < NH; ++g) {
      for (int b = 0; b < SB; ++b) {
        mbar_init(bar_s(g, b), 1);
        mbar_init(bar_p(g, b), 128);
      }
      mbar_init(&bars[C::kBarODone + g], 1);
      mbar_init(&bars[C::kBarODrained + g], 128);
      mbar_init(&bars[C::kBarPV + g], 1);
    }
    fence_barrier_init();
  }
  if (warp == C::kWarpMma) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // The converting warps find the CTA's works; the first of them hands each to the other roles in a ring of kRing slots.
  // Phases: lw = the CTA's works so far (Q buffer lw & 1, slot lw % kRing), kt = its tiles so far (stage kt % ST), and per
  // head the tiles and works that the head took part in.
  Slot* ring = reinterpret_cast<Slot*>(smem + C::kOffRing);
  auto take = [&](int lw, Slot& w) -> bool {  // by a whole warp
    const int i = lw % kRing;
    if (!warp_wait(&bars[C::kBarWFull + i], (lw / kRing) & 1, a.err)) return false;
    w = ring[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[C::kBarWFree + i]);
    return true;
  };
  if (warp >= C::kWarpConv && warp < C::kWarpMma) {
    // ================= converters: a page at a time, in order across works; the codes of the next kAhead pages are on
    // their way while one is widened and stored
    constexpr int kRaw = D / 16;  // 16-byte pieces of a page's block per lane: its keys, then its values
    constexpr int kA = C::kAhead, NB = kA + 1;
    const int cw = warp - C::kWarpConv;
    const int64_t pg_bytes = page_bytes(D, a.n_kv_heads);
    Walk walk;
    if (a.n_splits > 1) walk = deal<NH>(a);
    int works = 0;  // handed on (first warp)
    if (cw == 0 && elect_one()) prefetch_tensormap(&qmap);
    // Hands a work on (one that is not valid: the end), its Q tiles on their way to their buffer.
    auto publish = [&](const Work& wk) -> bool {
      const int i = works % kRing, qb = works & 1;
      if (works >= kRing && !warp_wait(&bars[C::kBarWFree + i], ((works / kRing) & 1) ^ 1, a.err)) return false;
      if (wk.valid && works >= 2 && !warp_wait(&bars[C::kBarQFree + qb], ((works >> 1) & 1) ^ 1, a.err)) return false;
      if (elect_one()) {
        Slot w{};
        if (wk.valid)
          w = Slot{wk.t0, wk.t1 - wk.t0, wk.n_g, wk.head0, wk.pos0 + wk.m0, wk.out_row + wk.m0, wk.qlen - wk.m0,
                   wk.split + (wk.last ? kLastPart : 0)};
        ring[i] = w;
        mbar_arrive(&bars[C::kBarWFull + i]);
        if (wk.valid) {
          mbar_arrive_expect_tx(&bars[C::kBarQFull + qb], wk.n_g * C::kQBytes);
          for (int g = 0; g < wk.n_g; ++g)
            for (int x = 0; x < D; x += 64)
              tma_load_3d(sQ(qb, g) + x * kBM * 2, &qmap, x, wk.head0 + g, wk.qs + wk.m0, &bars[C::kBarQFull + qb]);
        }
      }
      __syncwarp();
      works += wk.valid;
      return true;
    };
    bool run = true;
    uint4 raw[NB][kRaw];
    float2 scale[NB];
    int meta[NB];  // tile of the CTA * 4 + page of the tile; -1: no more
    // The page that is read next: its place among the work's pages and their number (0: no more works), the tile of the CTA
    // before the work's first; the work's first page and its end, the page table row, the KV head's place in a page, and
    // the ids of the 32 pages around it and the next 32 (lane = place % 32).
    int at = cw - C::kConv, n = -1, kt = 0, page0 = 0, last = 0;
    int32_t ids = -1, ids2 = -1;
    const int32_t* pt_row = nullptr;
    const uint8_t* head = nullptr;
    auto read_ids = [&](int place) -> int32_t {
      const int pg = page0 + place;
      if (place >= n || pg >= last) return -1;
      const int32_t id = pt_row[pg];
      if (id >= 0 && id < a.n_pages) return id;
      flag_error(a.err, kErrPageId);
      return -1;
    };
    auto read_next = [&](uint4 (&x)[kRaw], float2& sc, int& m) {
      m = -1;
      if (n == 0) return;
      const int was = at >> 5;
      at += C::kConv;
      if (at >= n) {  // (a work has four pages or more, so every warp has some of each)
        if (n > 0) at -= n, kt += n / kTilePages;
        n = 0;
        const Work wk = next_work<NH>(a, walk);
        if (cw == 0 && !publish(wk)) run = false;
        if (!wk.valid || !run) return;
        n = (wk.t1 - wk.t0) * kTilePages, pt_row = wk.pt_row;
        head = a.pool + int64_t(wk.kvh) * C::kBlock;
        page0 = wk.t0 * kTilePages, last = min(wk.n_item_pages, wk.t1 * kTilePages);
        ids = read_ids(lane);
        ids2 = read_ids(32 + lane);
      } else if ((at >> 5) != was) {
        ids = ids2;
        ids2 = read_ids((at & ~31) + 32 + lane);
      }
      m = kt * kTilePages + at;
      const int32_t id = __shfl_sync(0xffffffffu, ids, at & 31);
      sc = make_float2(0.f, 0.f);
      if (id < 0) {  // no such page: codes of 0
        constexpr uint32_t zero = to_word<KIND>(0u);
#pragma unroll
        for (int k = 0; k < kRaw; ++k) x[k] = make_uint4(zero, zero, zero, zero);
        return;
      }
      const uint8_t* blk = head + int64_t(id) * pg_bytes;
      const uint4* src = reinterpret_cast<const uint4*>(blk) + lane;
#pragma unroll
      for (int k = 0; k < kRaw; ++k) x[k] = __ldg(src + 32 * k);
      sc = __ldg(reinterpret_cast<const float2*>(blk + scale_off(D)));
    };
    // A page's codes as operands; false after a wait that gave up.
    auto write = [&](const uint4 (&x)[kRaw], float2 sc, int m) -> bool {
      const int tile = m / kTilePages, b = m % kTilePages, s = tile % ST;
      if (tile >= ST && !warp_wait(&bars[C::kBarKVEmpty + s], ((tile / ST) & 1) ^ 1, a.err)) return false;
      // keys: 16 dims of a token a piece, to its row's chunks 2c and 2c + 1
#pragma unroll
      for (int k = 0; k < kRaw / 2; ++k) {
        const int u = k * 32 + lane, sb = u >> 6, tok = (u >> 2) & 15, ch = u & 3, row = b * kPage + tok;
        uint4 y0, y1;
        widen4_key<KIND, BF16>(x[k].x, y0.x, y0.y);
        widen4_key<KIND, BF16>(x[k].y, y0.z, y0.w);
        widen4_key<KIND, BF16>(x[k].z, y1.x, y1.y);
        widen4_key<KIND, BF16>(x[k].w, y1.z, y1.w);
        uint8_t* dst = sK(s) + sb * (kBN * 128);
        *reinterpret_cast<uint4*>(dst + swz128(row, 2 * ch)) = y0;
        *reinterpret_cast<uint4*>(dst + swz128(row, 2 * ch + 1)) = y1;
      }
      // values: dims 8j + g (j = 0..3) of tokens 2t, 2t+1, 2t+8, 2t+9 a piece, 8 bytes to each dim's row
#pragma unroll
      for (int k = 0; k < kRaw / 2; ++k) {
        const int g = lane >> 2, t = lane & 3;
        const uint32_t w[4] = {x[kRaw / 2 + k].x, x[kRaw / 2 + k].y, x[kRaw / 2 + k].z, x[kRaw / 2 + k].w};
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          uint2 y;
          widen4<KIND>(w[jj], y.x, y.y);
          *reinterpret_cast<uint2*>(sV(s) + swz128(32 * k + 8 * jj + g, 2 * b + (t >> 1)) + 8 * (t & 1)) = y;
        }
      }
      // a scale of 0 comes with codes of 0: any other scale gives the same (here the smallest there is)
      const float ks = fmaxf(sc.x, kTiny / 448.f), vs = fmaxf(sc.y, kTiny / 448.f);
      const float4 out = make_float4(ks * (unit<KIND>() * a.scale_log2), __log2f(vs), __fdividef(1.f, vs), 0.f);
      if (lane == 0) scales[s * kTilePages + b] = out;
      fence_proxy_async_smem();  // the operands, for the tensor core
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[C::kBarKVFull + s]);
      return true;
    };
#pragma unroll
    for (int i = 0; i < kA; ++i) read_next(raw[i], scale[i], meta[i]);
    while (run) {
#pragma unroll
      for (int h = 0; h < NB; ++h) {
        if (meta[h] < 0) run = false;
        if (!run) break;
        read_next(raw[(h + kA) % NB], scale[(h + kA) % NB], meta[(h + kA) % NB]);
        if (run) run = write(raw[h], scale[h], meta[h]);
      }
    }
    // Q tiles in flight end before the CTA does (bounded)
    for (int i = max(0, works - 2); i < works; ++i) warp_wait(&bars[C::kBarQFull + (i & 1)], (i >> 1) & 1, a.err);
  } else if (warp >= C::kWarpMma) {
    // ================= MMA issuer. The whole warp walks the loop and waits; one lane, always the
    // same, issues. The descriptors are then values of the warp, kept in uniform registers: with the loop inside one
    // lane's branch every instruction's operands were moved there one by one, which cost 80 cycles an instruction (511
    // tokens over 16.4k at head_dim 128: 241 us against 176).
    constexpr uint32_t idesc_qk = make_idesc_f16(kBM, kBN, BF16, false, false);
    constexpr uint32_t idesc_pv = make_idesc_f16(kBM, D, false, false, false);
    int lw = 0, kt = 0;
    int h_tiles[NH] = {}, h_works[NH] = {};  // per head: S tiles consumed, works finished
    // descriptors differ in the address alone: 16-byte units, whose sums stay inside its 14 bits
    const uint64_t desc0 = make_sdesc(smem_u32(smem), 16, 1024, 2);
    auto desc_of = [&](const uint8_t* p) { return desc0 + (static_cast<uint32_t>(p - smem) >> 4); };
    // S_g (buffer buf) = Q_g K^T from Q buffer qb and stage s.
    auto qk = [&](int g, int buf, int qb, int s) {
      const uint64_t q_desc = desc_of(sQ(qb, g)), k_desc = desc_of(sK(s));
      const uint32_t to = tmem + C::col_s(g, buf);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc_mma_ss(to, q_desc + ((kk >> 2) * (kBM * 128) + (kk & 3) * 32) / 16,
                    k_desc + ((kk >> 2) * (kBN * 128) + (kk & 3) * 32) / 16, idesc_qk, kk > 0 ? 1u : 0u);
        tc_commit(bar_s(g, buf));
      }
    };
    auto kv_ready = [&](int t) -> bool {
      if (!warp_wait(&bars[C::kBarKVFull + t % ST], (t / ST) & 1, a.err)) return false;
      tc_fence_after();
      return true;
    };
    bool ok = true;
    for (;; ++lw) {
      Slot wk;
      ok = take(lw, wk);
      if (!ok || wk.n == 0) break;
      const int qb = lw & 1, n = wk.n, n_g = wk.n_g;
      ok = warp_wait(&bars[C::kBarQFull + qb], (lw >> 1) & 1, a.err) && kv_ready(kt);
      if (!ok) break;
      // S_g(0) may overwrite columns that an earlier PV_g reads P from: MMAs run in issue order.
#pragma unroll
      for (int g = 0; g < NH; ++g)
        if (g < n_g) qk(g, h_tiles[g] % SB, qb, kt % ST);
      for (int j = 0; j < n && ok; ++j, ++kt) {
        const bool more = j + 1 < n;
        if (more) ok = kv_ready(kt + 1);
        if (SB == 2 && more && ok)  // the next S during this tile's softmax
#pragma unroll
          for (int g = 0; g < NH; ++g)
            if (g < n_g) qk(g, (h_tiles[g] + 1) % SB, qb, (kt + 1) % ST);
#pragma unroll
        for (int g = 0; g < NH; ++g) {
          if (g >= n_g || !ok) break;
          // O_g += P_g V once head g's softmax has written P_g; the work's first PV overwrites O_g, so it also
          // waits for the epilogue of the work before to have read it.
          const int buf = h_tiles[g] % SB;
          if (j == 0 && h_works[g] > 0) ok = warp_wait(&bars[C::kBarODrained + g], (h_works[g] - 1) & 1, a.err);
          if (ok) ok = warp_wait(bar_p(g, buf), (h_tiles[g] / SB) & 1, a.err);
          if (!ok) break;
          ++h_tiles[g];
          tc_fence_after();
          const uint64_t v_desc = desc_of(sV(kt % ST));
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kBN / 16; ++kk)
              tc_mma_ts(tmem + C::col_o(g), tmem + C::col_s(g, buf) + kk * 8, v_desc + kk * 2, idesc_pv,
                        (j > 0 || kk > 0) ? 1u : 0u);
            if (SB == 2) tc_commit(&bars[C::kBarPV + g]);
          }
          if (SB == 1 && more) qk(g, 0, qb, (kt + 1) % ST);
        }
        if (elect_one()) tc_commit(&bars[C::kBarKVEmpty + kt % ST]);  // K and V of this stage are consumed
      }
      if (!ok) break;
#pragma unroll
      for (int g = 0; g < NH; ++g) {
        if (g >= n_g) break;
        if (elect_one()) tc_commit(&bars[C::kBarODone + g]);
        ++h_works[g];
      }
    }
  } else {
    // ================= softmax / correction / epilogue of head g: thread = query row = TMEM lane
    const int g = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tO = tmem + C::col_o(g) + lane_off;
    int h_tiles = 0, h_works = 0, kt = 0;
    bool ok = true;
    for (int lw = 0; ok; ++lw) {
      Slot wk;
      ok = take(lw, wk);
      if (!ok || wk.n == 0) break;
      const int n = wk.n, kt0 = kt;
      kt += n;
      if (g >= wk.n_g) {
        if (lane == 0) mbar_arrive(&bars[C::kBarQFree + (lw & 1)]);
        continue;
      }
      const int qpos = wk.pos + r;
      const int64_t orow = (int64_t(wk.row) + r) * a.n_heads + wk.head0 + g;
      const bool live = r < wk.live;
      float m_ref = -INFINITY, l_run = 0.f;
      float o_ref = -INFINITY;       // M
      float lref = 0.f, vrefc = 0.f;  // M - m, and 2^(M - m - 6)
      for (int j = 0; j < n; ++j, ++h_tiles) {
        const int buf = h_tiles % SB, s = (kt0 + j) % ST;
        const uint32_t tS = tmem + C::col_s(g, buf) + lane_off;
        ok = warp_wait(bar_s(g, buf), (h_tiles / SB) & 1, a.err) &&
             warp_wait(&bars[C::kBarKVFull + s], ((kt0 + j) / ST) & 1, a.err);  // (complete already: the scales are visible)
        if (!ok) break;
        tc_fence_after();
        uint32_t t[kBN];
        tmem_ld64_wait(tS, t);
        const int kbase = (wk.t0 + j) * kBN;
        if (kbase + kBN - 1 > qpos) {  // the tile holds keys past this row's position
#pragma unroll
          for (int c = 0; c < kBN; ++c)
            if (kbase + c > qpos) t[c] = __float_as_uint(-INFINITY);
        }
        float4 sc[kTilePages];
        float m_tile = -INFINITY, o_tile = -INFINITY;
#pragma unroll
        for (int b = 0; b < kTilePages; ++b) {
          sc[b] = scales[s * kTilePages + b];
          const uint32_t* x = &t[16 * b];
          float mx[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mx[i] = fmax3(__uint_as_float(x[i]), __uint_as_float(x[i + 2]), __uint_as_float(x[i + 4]));
            mx[i] = fmax3(mx[i], __uint_as_float(x[i + 6]), __uint_as_float(x[i + 8]));
            mx[i] = fmax3(mx[i], __uint_as_float(x[i + 10]), __uint_as_float(x[i + 12]));
          }
          const float top = fmax3(fmax3(mx[0], mx[1], __uint_as_float(x[14])), __uint_as_float(x[15]), -INFINITY) * sc[b].x;
          m_tile = fmaxf(m_tile, top);
          o_tile = fmaxf(o_tile, top + sc[b].y);
        }
        const bool need = m_tile > m_ref + kRescaleThreshold || o_tile > o_ref + kRescaleThreshold;  // false for -inf
        float alpha = 1.f;
        if (need) {
          const float m_new = fmaxf(m_ref, m_tile), o_new = fmaxf(o_ref, o_tile);
          l_run *= fast_exp2(m_ref - m_new);  // m_ref = -inf gives 0
          alpha = fast_exp2(o_ref - o_new);
          m_ref = m_new, o_ref = o_new;
          lref = o_new - m_new;
          vrefc = fast_exp2(lref - kPShift);
        }
        const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
        uint32_t p[kBN / 2];
#pragma unroll
        for (int b = 0; b < kTilePages; ++b) {
          const float2 f = make_float2(sc[b].x, sc[b].x);
          const float lv = sc[b].y - lref, add = fmaxf(lv, kMinLv) + kPShift - m_use;
          const float2 add2 = make_float2(add, add);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int u = 0; u < 8; ++u) {  // pair of keys 2u, 2u + 1: to pair 2 (u & 3) + (u >> 2) of the block's columns
            const int c = 16 * b + 2 * u;
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(t[c]), __uint_as_float(t[c + 1])), f, add2);
            const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            sum[u & 1] = __fadd2_rn(sum[u & 1], e);
            p[8 * b + 2 * (u & 3) + (u >> 2)] = pack2<false>(e.x, e.y);
          }
          const float2 s2 = __fadd2_rn(sum[0], sum[1]);
          const float w = lv < kMinLv ? 17179869184.f : sc[b].z * vrefc;  // 2^(40 - 6), or 2^(M - m - 6) / s_v
          l_run = fmaf(s2.x + s2.y, w, l_run);
        }
        // P into the first columns of the S buffer (the PV MMA's A operand)
        tmem_st32(tS, p);
        if (j > 0 && __any_sync(0xffffffffu, need)) {
          // PV_g(j - 1) has to be done: with one S buffer S_g(j) being there says so (MMAs run in order)
          if (SB == 2) {
            ok = warp_wait(&bars[C::kBarPV + g], (h_tiles - 1) & 1, a.err);
            if (!ok) break;
            tc_fence_after();
          }
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32_wait(tO + c * 32, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + c * 32, o);
          }
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(bar_p(g, buf));
      }
      if (!ok) break;
      // ---- epilogue: O_g out of TMEM, normalised and stored; then the next work's first PV may overwrite it
      // no key seen (a part past the row's position): 0; keys, but no score above -inf: a query that is not finite
      if (m_ref == -INFINITY) l_run = wk.t0 * kBN <= qpos ? NAN : 0.f;
      const float inv = l_run == 0.f ? 0.f : vrefc * unit<KIND>() / l_run;
      ok = warp_wait(&bars[C::kBarODone + g], h_works & 1, a.err);
      if (!ok) break;
      ++h_works;
      tc_fence_after();
      // through shared memory (the head's own Q tile, no longer read), so that 8 lanes store 128 bytes of a row: a lane
      // storing its own row takes a cycle for each 16 bytes, 13000 a work for fp32 parts of four heads
      const bool wide = a.n_splits > 1 || a.out_dtype == NBL_F32;
      uint8_t* stage = sQ(lw & 1, g) + quarter * (32 * 128);
      const int64_t row_bytes = int64_t(a.n_heads) * D * (wide ? 4 : 2);
      uint8_t* dst = a.n_splits > 1
                         ? reinterpret_cast<uint8_t*>(a.part_o + int64_t(wk.part & (kLastPart - 1)) * a.part_rows * a.n_heads * D)
                         : static_cast<uint8_t*>(a.out);
      dst += (int64_t(wk.row) + quarter * 32 + (lane >> 3)) * row_bytes + int64_t(wk.head0 + g) * D * (wide ? 4 : 2) + (lane & 7) * 16;
      const int rows = wk.live - quarter * 32 - (lane >> 3);  // of this warp, from this lane's first on
      auto put = [&](int chunk, uint4 v) { *reinterpret_cast<uint4*>(stage + swz128(lane, chunk)) = v; };
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld32_wait(tO + c, o);
        if (c + 32 == D) {
          tc_fence_before();
          mbar_arrive(&bars[C::kBarODrained + g]);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
        if (wide) {
#pragma unroll
          for (int i = 0; i < 8; ++i) put(i, make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
        } else {
          auto two = [&](int i) { return pack2<BF16>(__uint_as_float(o[i]), __uint_as_float(o[i + 1])); };
#pragma unroll
          for (int i = 0; i < 4; ++i) put((c & 32) / 8 + i, make_uint4(two(8 * i), two(8 * i + 2), two(8 * i + 4), two(8 * i + 6)));
          if (!(c & 32)) continue;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(stage + swz128(4 * i + (lane >> 3), lane & 7));
          if (4 * i < rows) *reinterpret_cast<uint4*>(dst + 4 * i * row_bytes) = v;
        }
        dst += 128;
        __syncwarp();
      }
      fence_proxy_async_smem();  // the next Q tile in this place comes by TMA
      if (lane == 0) mbar_arrive(&bars[C::kBarQFree + (lw & 1)]);
      if (live && a.n_splits > 1) {
        float* lse = a.part_lse + orow;
        const int64_t step = a.part_rows * a.n_heads;
        const int part = wk.part & (kLastPart - 1);
        lse[part * step] = l_run == 0.f ? -INFINITY : m_ref + log2f(l_run);
        if (wk.part & kLastPart)
          for (int p = part + 1; p < a.n_splits; ++p) lse[p * step] = -INFINITY;  // parts that the work does not have
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Joins the parts of each (token, head) row: part_lse in log2 units. A thread takes 4 dims.
template <int D>
__global__ void __launch_bounds__(256) kv8_prefill_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse,
                                                                int n_splits, int64_t part_rows, const Kv8Items it,
                                                                int n_heads, void* out, int out_dtype) {
  const int item = blockIdx.y;
  const int start = it.start[item], len = it.len[item], pos0 = it.pos0[item];
  if (len <= 0 || !item_fits(it, start, len, pos0)) return;
  const int64_t rows = part_rows * n_heads, first = int64_t(part_row(it, part_rows, item, start)) * n_heads;
  for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u < int64_t(len) * n_heads * (D / 4); u += gridDim.x * 256ll) {
    const int64_t row = first + u / (D / 4), to = int64_t(start) * n_heads + u / (D / 4);
    const int d = static_cast<int>(u % (D / 4)) * 4;
    float mx = -INFINITY;
    for (int p = 0; p < n_splits; ++p) mx = fmaxf(mx, part_lse[p * rows + row]);
    float W = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    const float mu = mx == -INFINITY ? 0.f : mx;
    for (int p = 0; p < n_splits; ++p) {
      const float w = fast_exp2(part_lse[p * rows + row] - mu);  // NaN: a query that is not finite, and so is the row
      const float4 x = *reinterpret_cast<const float4*>(part_o + (p * rows + row) * D + d);
      W += w;
      if (w > 0.f) O.x += w * x.x, O.y += w * x.y, O.z += w * x.z, O.w += w * x.w;
    }
    const float inv = W == 0.f ? 0.f : 1.f / W;
    store_as(out, to * D + d, O.x * inv, out_dtype);
    store_as(out, to * D + d + 1, O.y * inv, out_dtype);
    store_as(out, to * D + d + 2, O.z * inv, out_dtype);
    store_as(out, to * D + d + 3, O.w * inv, out_dtype);
  }
}

template <int D, int HEADS, int KIND, bool BF16>
void launch_t(cudaStream_t st, const CUtensorMap& qmap, const PrefillArgs& a, int grid) {
  using C = PCfg<D, HEADS>;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(configured.load() & bit)) {
    check_cuda(cudaFuncSetAttribute(kv8_prefill_kernel<D, HEADS, KIND, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    C::kSmemBytes),
               "kv8 prefill smem attribute");
    configured.fetch_or(bit);
  }
  kv8_prefill_kernel<D, HEADS, KIND, BF16><<<grid, C::kThreads, C::kSmemBytes, st>>>(qmap, a);
}

template <int D, int HEADS>
void launch_d(cudaStream_t st, int kind, bool bf16, const CUtensorMap& qmap, const PrefillArgs& a, int grid) {
  if (kind == NBL_I8) {
    if (bf16) launch_t<D, HEADS, NBL_I8, true>(st, qmap, a, grid);
    else launch_t<D, HEADS, NBL_I8, false>(st, qmap, a, grid);
  } else {
    if (bf16) launch_t<D, HEADS, NBL_E4M3, true>(st, qmap, a, grid);
    else launch_t<D, HEADS, NBL_E4M3, false>(st, qmap, a, grid);
  }
}

}  // namespace

namespace {
// Heads of a CTA: four at D = 64 where a group has three or more (one CTA per SM: each converted tile serves four heads),
// two otherwise (D = 64: two CTAs per SM, so that with small groups four softmax chains still run on an SM; D = 128: two
// fill TMEM).
int heads_of(int d, int group) { return d == 64 && group > 2 ? 4 : 2; }
}  // namespace

Kv8PrefillPlan plan_kv8_prefill(const nbl_kv* kv, int n_items, int max_len, int64_t n_rows, int n_heads, int max_kv,
                                int num_sms) {
  Kv8PrefillPlan p;
  const int group = n_heads / kv->cfg.n_kv_heads;
  const int64_t m_tiles = (max_len + kBM - 1) / kBM;
  const int heads = heads_of(kv->cfg.head_dim, group);
  const int64_t works = int64_t(n_items) * kv->cfg.n_kv_heads * ((group + heads - 1) / heads) * m_tiles;
  const int64_t slots = int64_t(num_sms) * (kv->cfg.head_dim == 64 && heads == 2 ? 2 : 1);
  if (works > INT32_MAX) fail(NBL_E_INVALID, "prefill: items * heads * query tiles exceeds 2^31 works");
  p.n_works = static_cast<int>(works);
  p.grid = static_cast<int>(std::min<int64_t>(works, slots));
  // A quarter of the CTAs or more without a work, and keys enough to share them: dealt, with room for the parts that equal
  // works have. (With 144 works on 148 SMs dealing took 96 us where a work each takes 72; one prompt of 1300 tokens, whose
  // works end up whole anyway, 57 us with the joining kernel and 46 without.)
  const int64_t max_tiles = (max_kv + kBN - 1) / kBN;
  if (4 * works <= 3 * slots && max_tiles >= 4 * kMinShare && max_tiles * 4 * slots < INT32_MAX) {
    p.n_splits = static_cast<int>(std::min({(slots + works - 1) / works + 1, max_tiles / kMinShare + 2, int64_t(64)}));
    p.grid = static_cast<int>(slots);
  }
  p.part_rows = std::min(n_rows, int64_t(n_items) * max_len);
  if (p.n_splits > 1)
    p.scratch_bytes = size_t(p.n_splits) * size_t(p.part_rows) * size_t(n_heads) * (kv->cfg.head_dim + 1) * sizeof(float);
  return p;
}

void launch_kv8_prefill(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, const void* q, int q_dtype, int n_heads,
                        void* out, int out_dtype, const Kv8PrefillPlan& plan, void* scratch, int* err) {
  const auto& c = kv->cfg;
  const int d = c.head_dim;
  CUtensorMap qmap;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(n_heads), static_cast<cuuint64_t>(items.n_rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(d) * 2, static_cast<cuuint64_t>(n_heads) * d * 2};
  const cuuint32_t box[3] = {64, 1, kBM};
  encode_tmap(&qmap, q_dtype == NBL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
              const_cast<void*>(q), dims, strides, box);
  PrefillArgs a{};
  a.it = items;
  a.pool = static_cast<const uint8_t*>(kv->pool);
  a.out = out;
  a.part_o = static_cast<float*>(scratch);
  a.part_rows = plan.part_rows;
  a.part_lse = a.part_o + int64_t(plan.n_splits) * plan.part_rows * n_heads * d;
  a.err = err;
  a.n_pages = c.n_pages;
  a.out_dtype = out_dtype;
  a.n_heads = n_heads;
  a.n_kv_heads = c.n_kv_heads;
  a.group = n_heads / c.n_kv_heads;
  const int heads = heads_of(d, a.group);
  a.n_hgroups = (a.group + heads - 1) / heads;
  a.m_tiles = (items.max_len + kBM - 1) / kBM;
  a.n_splits = plan.n_splits;
  a.n_works = plan.n_works;
  a.by_hgroups = Divisor(a.n_hgroups);
  a.by_kv_heads = Divisor(a.n_kv_heads);
  a.by_items = Divisor(items.n_items);
  a.scale_log2 = 1.4426950408889634f / std::sqrt(static_cast<float>(d));
  if (d == 128) launch_d<128, 2>(st, c.dtype, q_dtype == NBL_BF16, qmap, a, plan.grid);
  else if (heads == 4) launch_d<64, 4>(st, c.dtype, q_dtype == NBL_BF16, qmap, a, plan.grid);
  else launch_d<64, 2>(st, c.dtype, q_dtype == NBL_BF16, qmap, a, plan.grid);
  check_cuda(cudaGetLastError(), "kv8 prefill launch");
  if (plan.n_splits > 1) {
    const int64_t units = int64_t(items.max_len) * n_heads * (d / 4);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((units + 255) / 256, 1184)), static_cast<unsigned>(items.n_items));
    if (d == 64)
      kv8_prefill_merge_kernel<64><<<grid, 256, 0, st>>>(a.part_o, a.part_lse, plan.n_splits, plan.part_rows, items, n_heads, out,
                                                         out_dtype);
    else
      kv8_prefill_merge_kernel<128><<<grid, 256, 0, st>>>(a.part_o, a.part_lse, plan.n_splits, plan.part_rows, items, n_heads, out,
                                                         out_dtype);
    check_cuda(cudaGetLastError(), "kv8 prefill merge launch");
  }
}

}  // namespace nbl
