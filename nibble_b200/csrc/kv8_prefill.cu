// Causal attention of many query tokens over the 8-bit paged K/V pool on the 5th-generation tensor cores.
//
// Mathematics. With codes c and block scales s_k, s_v: score_j = s_k (q . ck_j) / sqrt(D), out = sum_j p_j s_v cv_j /
// sum_j p_j. The codes are exact fp16 (bf16) operands, so the tensor cores multiply codes and the scales meet scores and
// weights in fp32: a score is raw * f_b (f_b one number per 16-key block), and the weight that multiplies the value codes
// is p'_j = 2^(score - m + log2(s_v / vref) + 6), the same fused multiply-add with another addend. The row sum needs p
// without s_v: per block, sum(p') * (vref / s_v) / 2^6. vref is at least twice every s_v met so far (it moves rarely,
// with the accumulators), so p' <= 2^13 fits fp16, which holds it to 2^-12 relative: below the output's rounding.
//
// Work. As the 16-bit prefill: persistent CTAs walk works, a work being a 128-row query tile of two heads of a KV group
// (all of its keys, or one of n_splits stretches of them when there are fewer works than SMs). Warps:
//   0..7    softmax, one warpgroup per head: thread = query row = TMEM lane. A tile is 64 keys (4 pages).
//   converters (D = 64: the softmax warps themselves, while they would wait for S, each the keys or the values of one of
//           the tile's pages; D = 128: four more warps, each a page): the block's codes straight from global memory (L2: the
//           works that run at one time share their keys) through registers, widened, into the MMA operands: K [64 keys][D]
//           and V transposed, [D][64 keys], both K-major with 128-byte swizzle. A block's value words hold the tokens
//           2t, 2t+1, 2t+8, 2t+9 of a dim, so key 2t + (i & 1) + 8 (i >> 1) of a block is at place 4t + i of its V
//           columns, and P is packed in that order. They run two tiles ahead, across works.
//   last    MMA issuer (one thread): Q tiles by TMA into one of two buffers, S_g = Q_g K^T, O_g += P_g V with P read from
//           TMEM.
// D = 64: S and P share 64 columns, two CTAs per SM (four softmax chains hide each other's hand-offs; the exponentials
// set the pace). D = 128: O takes 128 columns a head, so one CTA fills TMEM; S is double-buffered instead, and the next
// tile's S is computed during a tile's softmax. Converting in one warp of its own (D = 64) took 232 us for 4 prompts of
// 2048 tokens, 32/4 heads, where the same kernel without any conversion takes 138.
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
constexpr float kMinLv = -24.0f;           // smallest log2(s_v / vref) kept: below it a block adds nothing to fp16 weights

template <int D, int HEADS>
struct PCfg {
  static constexpr int NH = HEADS;                      // heads of a CTA
  static constexpr int kCtas = D == 64 && NH == 2 ? 2 : 1;  // per SM
  static constexpr int SB = D == 64 ? 1 : 2;            // S buffers of a head
  static constexpr int ST = 3;                          // tiles of K and V operands
  static constexpr int kConv = D == 128 ? 4 : NH / 2;   // converting warps
  static constexpr int kConvPages = kTilePages / kConv; // pages of a tile that one of them converts
  static constexpr int kAhead = D == 64 ? 2 : 1;        // pages whose codes are on their way
  static constexpr int kMma = NH / 2;                   // issuing warps, two heads each
  static constexpr int kWarpConv = 4 * NH, kWarpMma = kWarpConv + kConv;
  static constexpr int kThreads = (kWarpMma + kMma) * 32;
  static constexpr int kQBytes = kBM * D * 2;           // one head's Q tile: D / 64 parts of [128][64]
  static constexpr int kTileBytes = kBN * D * 2;        // K (or V) operand tile
  static constexpr int kBlock = block_bytes(D);
  static constexpr int kOffQ = 0;                       // 2 buffers x NH heads
  static constexpr int kOffKV = 2 * NH * kQBytes;
  static constexpr int kOffScale = kOffKV + ST * 2 * kTileBytes;  // [ST][4] float4
  static constexpr int kOffBar = kOffScale + ST * kTilePages * 16;
  static constexpr int kBarQFull = 0, kBarQFree = 2, kBarKVFull = 4, kBarKVEmpty = kBarKVFull + ST, kBarS = kBarKVEmpty + ST,
                       kBarP = kBarS + NH * SB, kBarODone = kBarP + NH * SB, kBarODrained = kBarODone + NH,
                       kBarPV = kBarODrained + NH, kNumBars = kBarPV + NH;
  static constexpr int kOffTmemSlot = kOffBar + ((kNumBars * 8 + 15) & ~15);
  static constexpr int kSmemBytes = kOffTmemSlot + 16;
  static constexpr uint32_t kTmemCols = kCtas == 2 ? 256 : 512;
  __host__ __device__ static constexpr uint32_t col_s(int g, int buf) { return (g * SB + buf) * kBN; }
  __host__ __device__ static constexpr uint32_t col_o(int g) { return NH * SB * kBN + g * D; }
};

struct PrefillArgs {
  Kv8Items it;
  const uint8_t* pool;
  void* out;
  float *part_o, *part_lse;  // [n_splits][rows][heads][D] and [n_splits][rows][heads] when n_splits > 1
  int* err;
  int64_t n_pages;
  int out_dtype;
  int n_heads, n_kv_heads, group, n_hgroups, m_tiles, n_splits;
  int n_works;  // query tiles x splits x items x KV heads x head pairs
  float scale_log2;
};

struct Work {
  int kvh, n_g, head0, qlen, pos0, qs, m0, t0, t1, n_item_pages, split;
  const int32_t* pt_row;
  bool valid;
};

// Work w (-1: none); the same in every warp. Works are numbered with the query tile (latest, so heaviest, first) slowest,
// then the split, the item, the KV head and the head pair: the works of a round are about equally long, whatever the
// number of items (with the item slowest, 4 prompts of 2048 tokens left the busiest CTA with 1.6 times the mean).
template <int NH>
__device__ __forceinline__ Work decode_work(const PrefillArgs& a, int w) {
  Work k{};
  k.valid = false;
  if (w < 0) return k;
  const int hg = w % a.n_hgroups;
  w /= a.n_hgroups;
  k.kvh = w % a.n_kv_heads;
  w /= a.n_kv_heads;
  const int item = w % a.it.n_items;
  w /= a.it.n_items;
  k.split = w % a.n_splits;
  const int mt = a.m_tiles - 1 - w / a.n_splits;
  k.n_g = min(NH, a.group - NH * hg);  // the last heads of a group may be fewer
  k.head0 = k.kvh * a.group + NH * hg;
  k.qlen = a.it.len[item];
  k.pos0 = a.it.pos0[item];
  k.qs = a.it.start[item];
  k.m0 = mt * kBM;
  k.valid = k.qlen > 0 && k.m0 < k.qlen;
  if (!k.valid) return k;
  const int64_t kv_len = int64_t(k.pos0) + k.qlen;
  if (k.pos0 < 0 || k.qs < 0 || int64_t(k.qs) + k.qlen > a.it.n_rows || kv_len > int64_t(a.it.pt_stride) * kPage) {
    flag_error(a.err, kErrLength);
    k.valid = false;
    return k;
  }
  const int kv_end = static_cast<int>(min(kv_len, int64_t(k.pos0) + k.m0 + kBM));
  const int n_tiles = (kv_end + kBN - 1) / kBN;
  k.t0 = static_cast<int>(int64_t(n_tiles) * k.split / a.n_splits);
  k.t1 = static_cast<int>(int64_t(n_tiles) * (k.split + 1) / a.n_splits);
  k.n_item_pages = static_cast<int>((kv_len + kPage - 1) / kPage);
  k.pt_row = a.it.page_table + int64_t(item) * a.it.pt_stride;
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
      mbar_init(&bars[C::kBarQFree + b], C::kMma);
    }
    for (int s = 0; s < ST; ++s) {
      mbar_init(&bars[C::kBarKVFull + s], C::kConv);
      mbar_init(&bars[C::kBarKVEmpty + s], C::kMma);
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

  // Rounds of gridDim.x consecutive works; CTA c takes work c of even rounds and gridDim.x - 1 - c of odd ones (heavy and
  // light query tiles of a round even out over two), -1 past the end. Every role walks the same works, so the phase counts
  // below agree: lw = this CTA's valid works so far (Q buffer lw & 1), kt = its tiles so far (stage kt % ST), and per
  // head the tiles and works that the head took part in.
  auto work_of = [](int w0, int n_works) {
    const int w = w0 + (((w0 / static_cast<int>(gridDim.x)) & 1)
                            ? static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x)
                            : static_cast<int>(blockIdx.x));
    return w < n_works ? w : -1;
  };
  if (warp >= C::kWarpConv && warp < C::kWarpMma) {
    // ================= converters: a page at a time, in order across works; the codes of the next kAhead pages are on
    // their way while one is widened and stored
    constexpr int kRaw = D / 16;  // 16-byte pieces of a page's block per lane: its keys, then its values
    constexpr int kA = C::kAhead, NB = kA + 1;
    const int cw = warp - C::kWarpConv;
    const int64_t pg_bytes = page_bytes(D, a.n_kv_heads);
    uint4 raw[NB][kRaw];
    float2 scale[NB];
    int meta[NB];  // tile of the CTA * 4 + page of this warp in it; -1: no more
    // The page that is read next: round, place among the work's pages of this warp and their number, tile of the CTA; the
    // work's first page and its end, the page table row, the KV head's place in a page, and the ids of 32 of the
    // work's pages of this warp (lane = place % 32) and the next 32.
    int w0 = -static_cast<int>(gridDim.x), at = 0, n = 1, kt = -1, page0 = 0, last = 0;
    int32_t ids = -1, ids2 = -1;
    const int32_t* pt_row = nullptr;
    const uint8_t* head = nullptr;
    auto read_ids = [&](int place) -> int32_t {
      const int pg = page0 + place / C::kConvPages * kTilePages + place % C::kConvPages;
      if (place >= n || pg >= last) return -1;
      const int32_t id = pt_row[pg];
      if (id >= 0 && id < a.n_pages) return id;
      flag_error(a.err, kErrPageId);
      return -1;
    };
    auto read_next = [&](uint4 (&x)[kRaw], float2& sc, int& m) {
      m = -1;
      if (n == 0) return;
      if (++at >= n) {
        at = n = 0;
        while (n == 0) {
          w0 += gridDim.x;
          if (w0 >= a.n_works) return;
          const Work wk = decode_work<NH>(a, work_of(w0, a.n_works));
          if (!wk.valid) continue;
          n = (wk.t1 - wk.t0) * C::kConvPages, pt_row = wk.pt_row;
          head = a.pool + int64_t(wk.kvh) * C::kBlock;
          page0 = wk.t0 * kTilePages + cw * C::kConvPages, last = min(wk.n_item_pages, wk.t1 * kTilePages);
        }
        ids = read_ids(lane);
        ids2 = read_ids(32 + lane);
      } else if ((at & 31) == 0) {
        ids = ids2;
        ids2 = read_ids(at + 32 + lane);
      }
      const int step = at % C::kConvPages;
      if (step == 0) ++kt;
      m = kt * 4 + step;
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
      const int tile = m >> 2, st = m & 3, s = tile % ST, b = cw * C::kConvPages + st;  // b: page of the tile
      if (st == 0 && tile >= ST && !warp_wait(&bars[C::kBarKVEmpty + s], ((tile / ST) & 1) ^ 1, a.err)) return false;
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
      // a scale of 0 comes with codes of 0: any other scale gives the same
      const float ks = fmaxf(sc.x, 1e-34f), vs = fmaxf(sc.y, 1e-34f);
      const float4 out = make_float4(ks * (unit<KIND>() * a.scale_log2), __log2f(vs), __fdividef(1.f, vs), 0.f);
      if (lane == 0) scales[s * kTilePages + b] = out;
      if (st == C::kConvPages - 1) {
        fence_proxy_async_smem();  // the operands, for the tensor core
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[C::kBarKVFull + s]);
      }
      return true;
    };
#pragma unroll
    for (int i = 0; i < kA; ++i) read_next(raw[i], scale[i], meta[i]);
    for (bool run = true; run;) {
#pragma unroll
      for (int h = 0; h < NB; ++h) {
        if (meta[h] < 0) run = false;
        if (!run) break;
        read_next(raw[(h + kA) % NB], scale[(h + kA) % NB], meta[(h + kA) % NB]);
        run = write(raw[h], scale[h], meta[h]);
      }
    }
  } else if (warp >= C::kWarpMma) {
    // ================= MMA issuers: heads 2 mw and 2 mw + 1. The whole warp walks the loop and waits; one lane, always the
    // same, issues. The descriptors are then values of the warp, kept in uniform registers: with the loop inside one
    // lane's branch every instruction's operands were moved there one by one, which cost 80 cycles an instruction (511
    // tokens over 16.4k at head_dim 128: 241 us against 176).
    const int mw = __shfl_sync(0xffffffffu, warp - C::kWarpMma, 0);
    constexpr uint32_t idesc_qk = make_idesc_f16(kBM, kBN, BF16, false, false);
    constexpr uint32_t idesc_pv = make_idesc_f16(kBM, D, false, false, false);
    int lw = 0, kt = 0;
    int h_tiles[2] = {0, 0}, h_works[2] = {0, 0};  // per head: S tiles consumed, works finished
    // descriptors differ in the address alone: 16-byte units, whose sums stay inside its 14 bits
    const uint64_t desc0 = make_sdesc(smem_u32(smem), 16, 1024, 2);
    auto desc_of = [&](const uint8_t* p) { return desc0 + (static_cast<uint32_t>(p - smem) >> 4); };
    // S_g (buffer buf) = Q_g K^T from Q buffer qb and stage s, for head g = 2 mw + i.
    auto qk = [&](int i, int buf, int qb, int s) {
      const int g = 2 * mw + i;
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
    if (mw == 0 && elect_one()) prefetch_tensormap(&qmap);
    // The Q tiles of work wk (the CTA's lw'th) into its buffer.
    auto load_q = [&](const Work& wk, int lw) -> bool {
      const int qb = lw & 1, use = lw >> 1;
      if (use > 0 && !warp_wait(&bars[C::kBarQFree + qb], (use - 1) & 1, a.err)) return false;
      if (elect_one()) {
        mbar_arrive_expect_tx(&bars[C::kBarQFull + qb], wk.n_g * C::kQBytes);
        for (int g = 0; g < wk.n_g; ++g)
          for (int x = 0; x < D; x += 64)
            tma_load_3d(sQ(qb, g) + x * kBM * 2, &qmap, x, wk.head0 + g, wk.qs + wk.m0, &bars[C::kBarQFull + qb]);
      }
      return true;
    };
    auto next_work = [&](int& w0) -> Work {  // the next work of this CTA that has tiles
      Work wk{};
      for (wk.valid = false; w0 < a.n_works; w0 += gridDim.x) {
        wk = decode_work<NH>(a, work_of(w0, a.n_works));
        if (wk.valid && wk.t0 < wk.t1) break;
        wk.valid = false;
      }
      return wk;
    };
    bool ok = true;
    int w0 = 0, loaded = 0;  // works whose Q is on its way
    Work wk = next_work(w0);
    if (wk.valid && mw == 0) ok = load_q(wk, 0), loaded = 1;
    while (wk.valid && ok) {
      w0 += gridDim.x;
      const Work nextw = next_work(w0);
      const int qb = lw & 1, n = wk.t1 - wk.t0, n_g = min(2, wk.n_g - 2 * mw);  // (none or fewer: this warp only counts along)
      ok = warp_wait(&bars[C::kBarQFull + qb], (lw >> 1) & 1, a.err) && kv_ready(kt);
      if (!ok) break;
      // S_g(0) may overwrite columns that an earlier PV_g reads P from: MMAs run in issue order.
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (i < n_g) qk(i, h_tiles[i] % SB, qb, kt % ST);
      for (int j = 0; j < n && ok; ++j, ++kt) {
        const bool more = j + 1 < n;
        if (more) ok = kv_ready(kt + 1);
        if (SB == 2 && more && ok)  // the next S during this tile's softmax
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (i < n_g) qk(i, (h_tiles[i] + 1) % SB, qb, (kt + 1) % ST);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i >= n_g || !ok) break;
          // O_g += P_g V once head g's softmax has written P_g; the work's first PV overwrites O_g, so it also
          // waits for the epilogue of the work before to have read it.
          const int g = 2 * mw + i, buf = h_tiles[i] % SB;
          if (j == 0 && h_works[i] > 0) ok = warp_wait(&bars[C::kBarODrained + g], (h_works[i] - 1) & 1, a.err);
          if (ok) ok = warp_wait(bar_p(g, buf), (h_tiles[i] / SB) & 1, a.err);
          if (!ok) break;
          ++h_tiles[i];
          tc_fence_after();
          const uint64_t v_desc = desc_of(sV(kt % ST));
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kBN / 16; ++kk)
              tc_mma_ts(tmem + C::col_o(g), tmem + C::col_s(g, buf) + kk * 8, v_desc + kk * 2, idesc_pv,
                        (j > 0 || kk > 0) ? 1u : 0u);
            if (SB == 2) tc_commit(&bars[C::kBarPV + g]);
          }
          if (SB == 1 && more) qk(i, 0, qb, (kt + 1) % ST);
        }
        if (elect_one()) tc_commit(&bars[C::kBarKVEmpty + kt % ST]);  // K and V of this stage are consumed
        // the next work's Q, once the work before this one is done with the buffer (its last MMAs are issued)
        if (j == 0 && ok && mw == 0 && nextw.valid) {
          ok = load_q(nextw, lw + 1);
          loaded = lw + 2;
        }
      }
      if (!ok) break;
      if (elect_one()) tc_commit(&bars[C::kBarQFree + qb]);  // every QK of this work has read its Q tiles
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= n_g) break;
        if (elect_one()) tc_commit(&bars[C::kBarODone + 2 * mw + i]);
        ++h_works[i];
      }
      ++lw;
      wk = nextw;
    }
    // Q tiles in flight end before the CTA does (bounded)
    if (!ok)
      for (int i = max(0, loaded - 2); i < loaded; ++i) warp_wait(&bars[C::kBarQFull + (i & 1)], (i >> 1) & 1, a.err);
  } else {
    // ================= softmax / correction / epilogue of head g: thread = query row = TMEM lane
    const int g = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tO = tmem + C::col_o(g) + lane_off;
    int h_tiles = 0, h_works = 0, kt = 0;
    bool ok = true;
    for (int w0 = 0; w0 < a.n_works && ok; w0 += gridDim.x) {
      const Work wk = decode_work<NH>(a, work_of(w0, a.n_works));
      if (!wk.valid) continue;
      const int n = wk.t1 - wk.t0, kt0 = kt;
      kt += n;
      if (g >= wk.n_g) continue;
      const int qpos = wk.pos0 + wk.m0 + r;
      const int64_t orow = (int64_t(wk.qs) + wk.m0 + r) * a.n_heads + wk.head0 + g;
      const bool live = wk.m0 + r < wk.qlen;
      float m_ref = -INFINITY, l_run = 0.f;
      float lref = -INFINITY, vrefc = 0.f;  // log2 of vref, and vref / 2^6
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
        float m_tile = -INFINITY, lmax = -INFINITY;
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
          m_tile = fmaxf(m_tile, fmax3(fmax3(mx[0], mx[1], __uint_as_float(x[14])), __uint_as_float(x[15]), -INFINITY) * sc[b].x);
          lmax = fmaxf(lmax, sc[b].y);
        }
        const bool need_m = m_tile > m_ref + kRescaleThreshold;  // false for m_tile = -inf
        const float m_new = need_m ? m_tile : m_ref;
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        float l_scale = need_m ? fast_exp2(m_ref - m_use) : 1.f, alpha = l_scale;  // m_ref = -inf gives 0
        bool need = need_m;
        if (lmax > lref) {  // the same in every row
          const float lnew = lmax + 1.f;
          alpha *= fast_exp2(lref - lnew);
          need = true;
          lref = lnew;
          vrefc = fast_exp2(lref - kPShift);
        }
        m_ref = m_new;
        l_run *= l_scale;
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
          const float w = lv < kMinLv ? 262144.f : sc[b].z * vrefc;  // 2^(24 - 6), or vref / s_v / 2^6
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
      if (m_ref == -INFINITY) l_run = 0.f;  // no key seen (a split past the row's position)
      const float inv = l_run > 0.f ? vrefc * unit<KIND>() / l_run : 0.f;
      if (n > 0) {
        ok = warp_wait(&bars[C::kBarODone + g], h_works & 1, a.err);
        if (!ok) break;
        ++h_works;
        tc_fence_after();
      }
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32_wait(tO + c, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (c + 32 == D && n > 0) {
          tc_fence_before();
          mbar_arrive(&bars[C::kBarODrained + g]);
        }
        if (!live) continue;
        if (a.n_splits > 1 || a.out_dtype == NBL_F32) {
          float* base = a.n_splits > 1 ? a.part_o + int64_t(wk.split) * a.it.n_rows * a.n_heads * D : static_cast<float*>(a.out);
          float4* dst = reinterpret_cast<float4*>(base + orow * D + c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[i] = make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv,
                                 __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + orow * D + c);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            dst[i] = make_uint4(pack2<BF16>(__uint_as_float(o[8 * i]) * inv, __uint_as_float(o[8 * i + 1]) * inv),
                                pack2<BF16>(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv),
                                pack2<BF16>(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv),
                                pack2<BF16>(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv));
        }
      }
      if (live && a.n_splits > 1)
        a.part_lse[int64_t(wk.split) * a.it.n_rows * a.n_heads + orow] = l_run > 0.f ? m_ref + log2f(l_run) : -INFINITY;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Joins the splits of each (token, head) row: part_lse in log2 units. A thread takes 4 dims.
template <int D>
__global__ void __launch_bounds__(256) kv8_prefill_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse,
                                                                int n_splits, const Kv8Items it, int n_heads, void* out,
                                                                int out_dtype) {
  const int item = blockIdx.y;
  const int start = it.start[item], len = it.len[item], pos0 = it.pos0[item];
  if (len <= 0 || pos0 < 0 || start < 0 || int64_t(start) + len > it.n_rows ||
      int64_t(pos0) + len > int64_t(it.pt_stride) * kPage)
    return;
  const int64_t rows = it.n_rows * n_heads;
  for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u < int64_t(len) * n_heads * (D / 4); u += gridDim.x * 256ll) {
    const int64_t row = int64_t(start) * n_heads + u / (D / 4);
    const int d = static_cast<int>(u % (D / 4)) * 4;
    float mx = -INFINITY;
    for (int p = 0; p < n_splits; ++p) mx = fmaxf(mx, part_lse[p * rows + row]);
    float W = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mx != -INFINITY)
      for (int p = 0; p < n_splits; ++p) {
        const float w = fast_exp2(part_lse[p * rows + row] - mx);
        const float4 x = *reinterpret_cast<const float4*>(part_o + (p * rows + row) * D + d);
        W += w;
        if (w > 0.f) O.x += w * x.x, O.y += w * x.y, O.z += w * x.z, O.w += w * x.w;
      }
    const float inv = W > 0.f ? 1.f / W : 0.f;
    store_as(out, row * D + d, O.x * inv, out_dtype);
    store_as(out, row * D + d + 1, O.y * inv, out_dtype);
    store_as(out, row * D + d + 2, O.z * inv, out_dtype);
    store_as(out, row * D + d + 3, O.w * inv, out_dtype);
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
  const int64_t pairs = int64_t(n_items) * kv->cfg.n_kv_heads * ((group + heads - 1) / heads) * m_tiles;
  const int64_t slots = int64_t(num_sms) * (kv->cfg.head_dim == 64 && heads == 2 ? 2 : 1);
  // Fewer works than CTAs: split the keys, each stretch at least 8 tiles.
  int64_t splits = 1;
  if (pairs < slots) splits = std::max<int64_t>(1, std::min<int64_t>(slots / std::max<int64_t>(pairs, 1), max_kv / (8 * kBN)));
  p.n_splits = static_cast<int>(std::min<int64_t>(splits, 64));
  const int64_t works = pairs * p.n_splits;
  if (works > INT32_MAX) fail(NBL_E_INVALID, "prefill: items * heads * query tiles exceeds 2^31 works");
  p.n_works = static_cast<int>(works);
  p.grid = static_cast<int>(std::min<int64_t>(works, slots));
  if (p.n_splits > 1)
    p.scratch_bytes = size_t(p.n_splits) * size_t(n_rows) * size_t(n_heads) * (kv->cfg.head_dim + 1) * sizeof(float);
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
  a.part_lse = a.part_o + int64_t(plan.n_splits) * items.n_rows * n_heads * d;
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
  a.scale_log2 = 1.4426950408889634f / std::sqrt(static_cast<float>(d));
  if (d == 128) launch_d<128, 2>(st, c.dtype, q_dtype == NBL_BF16, qmap, a, plan.grid);
  else if (heads == 4) launch_d<64, 4>(st, c.dtype, q_dtype == NBL_BF16, qmap, a, plan.grid);
  else launch_d<64, 2>(st, c.dtype, q_dtype == NBL_BF16, qmap, a, plan.grid);
  check_cuda(cudaGetLastError(), "kv8 prefill launch");
  if (plan.n_splits > 1) {
    const int64_t units = int64_t(items.max_len) * n_heads * (d / 4);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((units + 255) / 256, 1184)), static_cast<unsigned>(items.n_items));
    if (d == 64)
      kv8_prefill_merge_kernel<64><<<grid, 256, 0, st>>>(a.part_o, a.part_lse, plan.n_splits, items, n_heads, out, out_dtype);
    else
      kv8_prefill_merge_kernel<128><<<grid, 256, 0, st>>>(a.part_o, a.part_lse, plan.n_splits, items, n_heads, out, out_dtype);
    check_cuda(cudaGetLastError(), "kv8 prefill merge launch");
  }
}

}  // namespace nbl
