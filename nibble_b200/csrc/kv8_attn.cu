// Attention over the 8-bit paged K/V pool for few query rows at a time (decode, and prefill chunks): split-KV with
// online softmax on the warp-level tensor cores.
//
// Mathematics. With codes c and the block scales s_k, s_v of a (16-token page, KV head), score_j = s_k (q . ck_j) /
// sqrt(D) and out = sum_j p_j s_v cv_j / sum_j p_j, p_j = exp(score_j - m). The codes are exact fp16 operands, so the
// scales never touch the products: s_k multiplies a block's scores and s_v its weights.
//
// Work. One CTA per (item, KV head, tile of query rows, split of the pages). A tile packs the query heads of the KV
// head and consecutive tokens: row r of (item, KV head) is token r / G, head r % G. The CTA's 4 warps take the split's
// 2-page chunks round-robin; each has a private ring in shared memory filled by bulk copies (a block is one piece of
// memory, in operand order; see kv8.cuh) and its own softmax state, so the main loop has no CTA barrier. The warps
// merge through shared memory, and splits through scratch by the last CTA of the tile to finish.
//
// m16n8k16: S[16 rows x 8 tokens] = Q (A) K^T (B), O[16 rows x 8 dims] = P (A) V (B). The C fragment of S is the A
// fragment of P, so P never leaves its lane. HILO (fp32 queries): a tile is 8 rows; rows 0-7 of the instruction carry
// the leading fp16 term of q (and of p), rows 8-15 the remainder (x = hi + lo to 2^-22 relative), and the two halves of
// the accumulator are added: fp32 accuracy at no extra instruction. 16-bit queries: a tile is 16 rows; q is exact in
// fp16 once each row is scaled by a power of two, p is rounded to fp16 (2^-12 relative, below the output's rounding).
//
// p * s_v is formed relative to the largest s_v that the warp has met (vref) and scaled by 2^14, so fp16 holds it
// whatever the cache's magnitudes: the accumulators are O * 2^14 / vref.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kv8.cuh"

namespace nbl {
namespace {

using namespace kv8;

constexpr int kWarps = 4;
constexpr int kChunkPages = 2;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kPScale = 16384.f;  // 2^14

template <int D>
struct Cfg {
  static constexpr int kStages = D == 64 ? 4 : 3;
  static constexpr int kCtasPerSm = D == 64 ? 3 : 2;
  static constexpr int kBlock = block_bytes(D);
  static constexpr int kStageBytes = kChunkPages * (kBlock + 16);
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kMergeBytes = kWarps * 16 * (D + 2) * 4;
  static constexpr int kBody = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;
  static constexpr int kSmemBytes = kBody + kWarps * kStages * 8;
};

struct AttnArgs {
  Kv8Items it;
  const void* q;
  void* out;
  float* lse;
  const uint8_t* pool;
  float* part_o;    // [n_splits][n_rows][n_heads][D] when n_splits > 1
  float* part_lse;  // [n_splits][n_rows][n_heads]
  unsigned* counts; // one arrival counter per unit, 0 between launches
  int* err;
  int64_t n_pages;
  int q_dtype, out_dtype;
  int n_heads, n_kv_heads, group, tiles;
  int n_splits, min_pages;  // splits of each unit's own pages, of at least min_pages (even)
  int q_vec;         // q allows 4-element loads
  float scale_log2;  // log2(e) / sqrt(D)
};

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

__device__ __forceinline__ void split_half2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half a = __float2half_rn(x), b = __float2half_rn(y);
  hi = pack_half2(a, b);
  lo = pack_half2(__float2half_rn(x - __half2float(a)), __float2half_rn(y - __half2float(b)));
}

template <int D, int KIND, bool HILO>
__global__ void __launch_bounds__(kWarps * 32, Cfg<D>::kCtasPerSm) kv8_attn_kernel(const AttnArgs a) {
  using C = Cfg<D>;
  constexpr int kTileRows = HILO ? 8 : 16;
  constexpr int NR = HILO ? 1 : 2;  // query rows whose scores a lane holds: g (and g + 8)
  constexpr int kSb = D / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % a.n_splits;
  const int unit = blockIdx.x / a.n_splits;
  const int tile = a.tiles - 1 - unit % a.tiles;  // a later tile sees more keys: it starts first
  const int kvh = unit / a.tiles % a.n_kv_heads;
  const int item = unit / a.tiles / a.n_kv_heads;

  // ---- the item's rows and keys
  int q_start, q_len, pos0;
  if (a.it.len) {
    q_start = a.it.start[item], q_len = a.it.len[item], pos0 = a.it.pos0[item];
  } else {
    q_start = item, q_len = 1, pos0 = a.it.pos0[item] - 1;  // a decode row: pos0 is its length
  }
  const int max_kv = a.it.pt_stride * kPage;
  const int row0 = tile * kTileRows, n_rows_item = q_len * a.group;
  if (q_len <= 0 || row0 >= n_rows_item) return;  // every split of the unit leaves here
  if (a.it.len ? (pos0 < 0 || q_start < 0 || int64_t(q_start) + q_len > a.it.n_rows || int64_t(pos0) + q_len > max_kv)
               : (pos0 < -1 || pos0 >= max_kv)) {
    if (threadIdx.x == 0) flag_error(a.err, kErrLength);
    if (a.it.len) return;
    pos0 = pos0 < -1 ? -1 : max_kv - 1;
  }
  const int last_row = min(row0 + kTileRows, n_rows_item) - 1;
  const int kv_len = pos0 + last_row / a.group + 1;   // keys the tile's last row sees
  const int kv_min = pos0 + row0 / a.group + 1;       // keys every row sees
  const int kv_pages = (kv_len + kPage - 1) / kPage;
  const int share = (kv_pages + a.n_splits - 1) / a.n_splits;
  const int pages_per_split = max(a.min_pages, (share + kChunkPages - 1) / kChunkPages * kChunkPages);
  const int p_begin = min(split * pages_per_split, kv_pages);
  const int p_end = min(kv_pages, p_begin + pages_per_split);
  const int n_chunks = p_end > p_begin ? (p_end - p_begin + kChunkPages - 1) / kChunkPages : 0;
  const int my_n = n_chunks > warp ? (n_chunks - warp + kWarps - 1) / kWarps : 0;
  const int32_t* pt_row = a.it.page_table + int64_t(item) * a.it.pt_stride;
  const int64_t pg_bytes = page_bytes(D, a.n_kv_heads);

  uint8_t* ring = smem + warp * C::kStages * C::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBody) + warp * C::kStages;
  if (lane == 0) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(&bars[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  // Page id of page j of this warp's chunk i, read by one lane; -1 past the split.
  auto chunk_pid = [&](int i, int j) -> int32_t {
    const int pg = p_begin + (warp + kWarps * i) * kChunkPages + j;
    return i < my_n && pg < p_end ? pt_row[pg] : -1;
  };
  // loaded: bit 2 * stage + j set when page j of the chunk in ring stage `stage` was loaded (the same in every lane).
  uint32_t loaded = 0;
  auto issue = [&](int i, int stage, int32_t pid0, int32_t pid1) {
    const int pg0 = p_begin + (warp + kWarps * i) * kChunkPages;
    const bool two = pg0 + 1 < p_end;
    const bool ok0 = pid0 >= 0 && pid0 < a.n_pages, ok1 = two && pid1 >= 0 && pid1 < a.n_pages;
    loaded = (loaded & ~(3u << (2 * stage))) | ((ok0 ? 1u : 0u) << (2 * stage)) | ((ok1 ? 2u : 0u) << (2 * stage));
    if (lane != 0) return;
    if (!ok0 || (two && !ok1)) flag_error(a.err, kErrPageId);
    uint8_t* st = ring + stage * C::kStageBytes;
    mbar_arrive_expect_tx(&bars[stage], (int(ok0) + int(ok1)) * (C::kBlock + 16u));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (!(j ? ok1 : ok0)) continue;
      const uint8_t* pg = a.pool + int64_t(j ? pid1 : pid0) * pg_bytes;
      bulk_load(st + j * C::kBlock, pg + int64_t(kvh) * C::kBlock, C::kBlock, &bars[stage]);
      bulk_load(st + 2 * C::kBlock + j * 16, pg + scale_off(D, a.n_kv_heads, kvh), 16, &bars[stage]);
    }
  };
  // The first chunks: lane 2c + j reads page j of chunk c, so their loads issue after one page-table latency.
  {
    const int32_t pf = lane < 2 * C::kStages ? chunk_pid(lane >> 1, lane & 1) : -1;
    for (int i = 0; i < min(C::kStages, my_n); ++i)
      issue(i, i, __shfl_sync(0xffffffffu, pf, 2 * i), __shfl_sync(0xffffffffu, pf, 2 * i + 1));
  }

  // ---- Q as the A operand: row g's (and row g + 8's) dims 64 sb + 16 t + 4 ks ..+3 for k-step (sb, ks)
  uint32_t qa[kSb * 4][4];
  float row_scale[NR];
  int lim[NR];       // keys the row sees
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = row0 + g + 8 * n;
    const bool valid = r < n_rows_item;
    const int tok = valid ? r / a.group : 0, head = kvh * a.group + (valid ? r % a.group : 0);
    const int64_t base = ((int64_t(q_start) + tok) * a.n_heads + head) * D;
    lim[n] = valid ? pos0 + tok + 1 : 0;
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
    row_scale[n] = __uint_as_float(e << 23) * a.scale_log2;
#pragma unroll
    for (int k = 0; k < kSb * 4; ++k) {
      if constexpr (HILO) {
        split_half2(x[k][0] * inv, x[k][1] * inv, qa[k][0], qa[k][1]);
        split_half2(x[k][2] * inv, x[k][3] * inv, qa[k][2], qa[k][3]);
      } else {
        qa[k][n] = pack_half2(__float2half_rn(x[k][0] * inv), __float2half_rn(x[k][1] * inv));
        qa[k][2 + n] = pack_half2(__float2half_rn(x[k][2] * inv), __float2half_rn(x[k][3] * inv));
      }
    }
  }

  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[j][c] = 0.f;
  float m_run[NR], l_run[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) m_run[n] = -INFINITY, l_run[n] = 0.f;
  float vref = 0.f, vinv = 0.f;  // largest value scale so far, and 2^14 / it
  int done = 0;

  for (int i = 0; i < my_n; ++i) {
    const int stage = i % C::kStages;
    if (!warp_wait_all(&bars[stage], (i / C::kStages) & 1, a.err)) break;
    done = i + 1;
    const int tok0 = (p_begin + (warp + kWarps * i) * kChunkPages) * kPage;
    // page ids of the chunk this stage takes next, read now and used at the end of the iteration
    const int32_t nxt = lane < kChunkPages ? chunk_pid(i + C::kStages, lane) : -1;
    const uint8_t* st = ring + stage * C::kStageBytes;

    // ---- scores of 2 pages x 16 tokens: lane's tokens 2t, 2t+1, 8+2t, 9+2t of each page
    float s[NR][kChunkPages][4];
    float vs[kChunkPages];
#pragma unroll
    for (int j = 0; j < kChunkPages; ++j) {
      if (!((loaded >> (2 * stage + j)) & 1u)) {
        vs[j] = 0.f;
#pragma unroll
        for (int n = 0; n < NR; ++n) s[n][j][0] = s[n][j][1] = s[n][j][2] = s[n][j][3] = -INFINITY;
        continue;
      }
      const float2 sc = *reinterpret_cast<const float2*>(st + 2 * C::kBlock + j * 16);
      vs[j] = sc.y;
      float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
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
          widen4<KIND>(wa[ks], b0, b1);
          mma_f16_16816(c0, q4[0], q4[1], q4[2], q4[3], b0, b1);
          widen4<KIND>(wb[ks], b0, b1);
          mma_f16_16816(c1, q4[0], q4[1], q4[2], q4[3], b0, b1);
        }
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float f = row_scale[n] * sc.x;
        if constexpr (HILO) {
          s[n][j][0] = (c0[0] + c0[2]) * f, s[n][j][1] = (c0[1] + c0[3]) * f;
          s[n][j][2] = (c1[0] + c1[2]) * f, s[n][j][3] = (c1[1] + c1[3]) * f;
        } else {
          s[n][j][0] = c0[2 * n] * f, s[n][j][1] = c0[2 * n + 1] * f;
          s[n][j][2] = c1[2 * n] * f, s[n][j][3] = c1[2 * n + 1] * f;
        }
      }
      const int base = tok0 + j * kPage;
      if (base + kPage > kv_min) {  // some row does not see the whole page
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (base + 2 * t + (c & 1) + 8 * (c >> 1) >= lim[n]) s[n][j][c] = -INFINITY;
      }
    }
    // ---- running maximum, weights and sums
    float al[NR];
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float mx = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                       fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m_run[n], mx);
      const float mu = mn == -INFINITY ? 0.f : mn;
      al[n] = exp2f(m_run[n] - mu);
      moved = moved || mn != m_run[n];
      m_run[n] = mn;
      float ps = 0.f;
#pragma unroll
      for (int j = 0; j < kChunkPages; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[n][j][c] = exp2f(s[n][j][c] - mu);
          ps += s[n][j][c];
        }
      l_run[n] = l_run[n] * al[n] + ps;
    }
    const float vmax = fmaxf(vs[0], vs[1]);
    if (vmax > vref) {  // a larger value scale: the accumulators move to it
      const float f = vref > 0.f ? vref / vmax : 0.f;
#pragma unroll
      for (int n = 0; n < NR; ++n) al[n] *= f;
      moved = true;
      vref = vmax;
      vinv = kPScale / vmax;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] *= al[0];
        o[j][1] *= al[0];
        o[j][2] *= al[NR - 1];
        o[j][3] *= al[NR - 1];
      }
    }
    // ---- O += P V
#pragma unroll
    for (int j = 0; j < kChunkPages; ++j) {
      if (!((loaded >> (2 * stage + j)) & 1u)) continue;
      const float r = vs[j] * vinv;
      uint32_t a0, a1, a2, a3;
      if constexpr (HILO) {
        split_half2(s[0][j][0] * r, s[0][j][1] * r, a0, a1);
        split_half2(s[0][j][2] * r, s[0][j][3] * r, a2, a3);
      } else {
        a0 = pack_half2(__float2half_rn(s[0][j][0] * r), __float2half_rn(s[0][j][1] * r));
        a1 = pack_half2(__float2half_rn(s[1][j][0] * r), __float2half_rn(s[1][j][1] * r));
        a2 = pack_half2(__float2half_rn(s[0][j][2] * r), __float2half_rn(s[0][j][3] * r));
        a3 = pack_half2(__float2half_rn(s[1][j][2] * r), __float2half_rn(s[1][j][3] * r));
      }
      const uint8_t* vp = st + j * C::kBlock + kPage * D + lane * 16;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint4 v4 = *reinterpret_cast<const uint4*>(vp + c * 512);
        const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t b0, b1;
          widen4<KIND>(w[k], b0, b1);
          mma_f16_16816(o[4 * c + k], a0, a1, a2, a3, b0, b1);
        }
      }
    }
    __syncwarp();
    if (i + C::kStages < my_n) {
      const int32_t p0 = __shfl_sync(0xffffffffu, nxt, 0), p1 = __shfl_sync(0xffffffffu, nxt, 1);
      if (lane == 0) fence_proxy_async_smem();  // this warp's reads of the stage come before its next write
      issue(i + C::kStages, stage, p0, p1);
    }
  }
  // After a wait that gave up, the loads still in flight are drained (bounded) before the ring is reused.
  if (done < my_n)
    for (int i = done; i < min(my_n, done + C::kStages); ++i)
      mbar_wait(&bars[i % C::kStages], (i / C::kStages) & 1, a.err);

  // ---- merge the 4 warps through shared memory: per warp [16 rows][D] outputs, [16] maxima, [16] sums
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    l_run[n] += __shfl_xor_sync(0xffffffffu, l_run[n], 1);
    l_run[n] += __shfl_xor_sync(0xffffffffu, l_run[n], 2);
  }
  __syncthreads();  // every warp is past its ring
  float* mrg = reinterpret_cast<float*>(smem);
  float* w_o = mrg + warp * 16 * (D + 2);
  float* w_m = w_o + 16 * D;
  const float vsc = vref * (1.f / kPScale);
#pragma unroll
  for (int n = 0; n < NR; ++n)
    if (t == 0) {
      w_m[g + 8 * n] = m_run[n];
      w_m[16 + g + 8 * n] = l_run[n];
    }
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if constexpr (HILO) {
        w_o[g * D + 8 * j + 2 * t + c] = (o[j][c] + o[j][2 + c]) * vsc;
      } else {
        w_o[g * D + 8 * j + 2 * t + c] = o[j][c] * vsc;
        w_o[(g + 8) * D + 8 * j + 2 * t + c] = o[j][2 + c] * vsc;
      }
    }
  __syncthreads();
  const int n_here = last_row - row0 + 1;
  const int64_t lse_stride = a.it.n_rows * a.n_heads;
  // Row r of the tile as a row of the packed (token, head) outputs.
  auto out_row = [&](int r) -> int64_t {
    const int rr = row0 + r;
    return (int64_t(q_start) + rr / a.group) * a.n_heads + kvh * a.group + rr % a.group;
  };
  for (int idx = threadIdx.x; idx < n_here * D; idx += kWarps * 32) {
    const int r = idx / D, d = idx % D;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, mrg[w * 16 * (D + 2) + 16 * D + r]);
    float L = 0.f, O = 0.f;
    if (mx != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* wb = mrg + w * 16 * (D + 2);
        const float sc = exp2f(wb[16 * D + r] - mx);  // 0 for warps that saw no key
        L += sc * wb[16 * D + 16 + r];
        O += sc * wb[r * D + d];
      }
    }
    const float val = L > 0.f ? O / L : 0.f;
    const float lse = L > 0.f ? (mx + log2f(L)) * kLn2 : -INFINITY;
    const int64_t row = out_row(r);
    if (a.n_splits == 1) {
      store_as(a.out, row * D + d, val, a.out_dtype);
      if (d == 0 && a.lse) a.lse[row] = lse;
    } else {
      a.part_o[(split * lse_stride + row) * D + d] = val;
      if (d == 0) a.part_lse[split * lse_stride + row] = lse;
    }
  }
  if (a.n_splits == 1) return;
  // The last split of this unit to finish merges all of them; its counter wraps back to 0 for the next launch.
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0)
    last = atomicInc(&a.counts[unit], static_cast<unsigned>(a.n_splits - 1)) == static_cast<unsigned>(a.n_splits - 1);
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int idx = threadIdx.x; idx < n_here * D; idx += kWarps * 32) {
    const int64_t row = out_row(idx / D);
    const int d = idx % D;
    float mx = -INFINITY;
    for (int p = 0; p < a.n_splits; ++p) mx = fmaxf(mx, __ldcg(a.part_lse + p * lse_stride + row));
    float W = 0.f, O = 0.f;
    if (mx != -INFINITY) {
      for (int p = 0; p < a.n_splits; ++p) {
        const float w = expf(__ldcg(a.part_lse + p * lse_stride + row) - mx);
        W += w;
        if (w > 0.f) O += w * __ldcg(a.part_o + (p * lse_stride + row) * D + d);
      }
    }
    store_as(a.out, row * D + d, W > 0.f ? O / W : 0.f, a.out_dtype);
    if (d == 0 && a.lse) a.lse[row] = W > 0.f ? mx + logf(W) : -INFINITY;
  }
}

template <int D, int KIND, bool HILO>
void launch_t(cudaStream_t st, const AttnArgs& a, int64_t grid) {
  static std::atomic<uint64_t> configured{0};  // one bit per device
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(configured.load() & bit)) {
    check_cuda(cudaFuncSetAttribute(kv8_attn_kernel<D, KIND, HILO>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Cfg<D>::kSmemBytes),
               "kv8 attention smem attribute");
    configured.fetch_or(bit);
  }
  kv8_attn_kernel<D, KIND, HILO><<<static_cast<unsigned>(grid), kWarps * 32, Cfg<D>::kSmemBytes, st>>>(a);
}

template <int D, int KIND>
void launch_q(cudaStream_t st, const AttnArgs& a, int64_t grid) {
  if (a.q_dtype == NBL_F32) launch_t<D, KIND, true>(st, a, grid);
  else launch_t<D, KIND, false>(st, a, grid);
}

}  // namespace

Kv8AttnPlan plan_kv8_attn(const nbl_kv* kv, int n_items, int max_len, int64_t n_rows, int n_heads, int max_kv,
                          int q_dtype, int num_sms, int requested_splits) {
  Kv8AttnPlan p;
  const int group = n_heads / kv->cfg.n_kv_heads, tile_rows = q_dtype == NBL_F32 ? 8 : 16;
  const int64_t tiles = (int64_t(max_len) * group + tile_rows - 1) / tile_rows;
  p.units = int64_t(n_items) * kv->cfg.n_kv_heads * tiles;
  if (tiles > INT32_MAX || p.units > INT32_MAX)
    fail(NBL_E_INVALID, "attention: items * heads * query rows exceeds 2^31 row tiles");
  p.tiles = static_cast<int>(std::max<int64_t>(tiles, 1));
  const int max_pages = std::max(1, (max_kv + kPage - 1) / kPage);
  const int64_t slots = int64_t(num_sms) * (kv->cfg.head_dim == 64 ? Cfg<64>::kCtasPerSm : Cfg<128>::kCtasPerSm);
  p.min_pages = requested_splits > 0 ? kChunkPages : 8;
  int64_t ns = requested_splits;
  if (ns <= 0) ns = p.units > 0 ? std::max<int64_t>(1, std::min<int64_t>(max_pages / p.min_pages, slots / p.units)) : 1;
  p.n_splits = static_cast<int>(std::min<int64_t>(ns, (max_pages + kChunkPages - 1) / kChunkPages));
  if (p.n_splits > 1)
    p.scratch_bytes = size_t(p.n_splits) * size_t(n_rows) * size_t(n_heads) * (kv->cfg.head_dim + 1) * sizeof(float);
  if (p.units * p.n_splits > INT32_MAX) fail(NBL_E_INVALID, "attention: row tiles * splits exceeds 2^31 CTAs");
  return p;
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
  a.part_o = static_cast<float*>(scratch);
  a.part_lse = a.part_o + int64_t(plan.n_splits) * items.n_rows * n_heads * c.head_dim;
  a.counts = counts;
  a.err = err;
  a.n_pages = c.n_pages;
  a.q_dtype = q_dtype;
  a.out_dtype = out_dtype;
  a.n_heads = n_heads;
  a.n_kv_heads = c.n_kv_heads;
  a.group = n_heads / c.n_kv_heads;
  a.tiles = plan.tiles;
  a.n_splits = plan.n_splits;
  a.min_pages = plan.min_pages;
  a.q_vec = (reinterpret_cast<uintptr_t>(q) & (q_dtype == NBL_F32 ? 15u : 7u)) == 0;
  a.scale_log2 = 1.4426950408889634f / std::sqrt(static_cast<float>(c.head_dim));
  const int64_t grid = plan.units * plan.n_splits;
  if (grid == 0) return;
  if (c.head_dim == 64) {
    if (c.dtype == NBL_I8) launch_q<64, NBL_I8>(st, a, grid);
    else launch_q<64, NBL_E4M3>(st, a, grid);
  } else {
    if (c.dtype == NBL_I8) launch_q<128, NBL_I8>(st, a, grid);
    else launch_q<128, NBL_E4M3>(st, a, grid);
  }
  check_cuda(cudaGetLastError(), "kv8 attention launch");
}

}  // namespace nbl
