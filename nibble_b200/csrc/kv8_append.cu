// Writing and reading the 8-bit K/V pool: the fused bias -> rotary -> quantize -> page write of new tokens, the read
// of cache rows as floats, and the import / export of whole pages.
//
// Quantization. A block is the 16 places of one (page, KV head), keys and values apart. With amax the largest
// magnitude among the tokens that a call adds to the block and s_old the scale of the tokens that were there,
//   s = max(s_old, amax * (1 / code_max)),   new code = round(x / s),   old code = round(code * s_old / s),
// so a block's scale only grows while it fills, and each growth adds at most half a step to an old token's error. The
// places after the last token are set to 0. Products use the fp32 reciprocal of s; all of it is IEEE fp32, each step
// rounded once, so the codes do not depend on how the work is spread over threads.
//
// Measured, append and read back of the same tokens: 24 prompts of 97..2047 tokens, 32/4 heads of 64, bf16: 51 us, 3.6 TB/s;
// 8191 tokens, 28/4 heads of 128, fp16, scaled positions: 56 us, 3.0 TB/s; 64 single tokens of 32/8 heads, fp32: 17 us, the
// two calls' time on the host. What the longer ones lose to the copy rate goes to issue slots (68 % busy: rotation, rounding,
// byte exchange) and to the latency of short CTAs (one page of one head: 2-4 KB in, the block's maximum, 1-2 KB out).
#include <algorithm>

#include "kv8.cuh"

namespace nbl {
namespace {

using namespace kv8;

constexpr int kThreads = 128;  // import / export

// Threads of an append or read CTA, which has one (page, KV head): 8 dims (chunk c) of one token each. Warp w has the tokens
// 2t, 2t + 1, 2t + 8, 2t + 9 with t = w % 4 (lane / 8 = place i among them), the four that share a value word, and
// chunks 8 (w / 4) + lane % 8.
template <int D>
constexpr int kCtaThreads = kPage * D / 8;
struct Place {
  int t, i, tok, c;
};
__device__ __forceinline__ Place place_of(int thread) {
  const int warp = thread >> 5, lane = thread & 31;
  Place p;
  p.t = warp & 3, p.i = lane >> 3;
  p.tok = 2 * p.t + (p.i & 1) + 8 * (p.i >> 1);
  p.c = (warp >> 2) * 8 + (lane & 7);
  return p;
}
// The four lanes of a value word (lane bits 3 and 4) exchange bytes: lane i's byte k becomes lane k's byte i.
__device__ __forceinline__ uint32_t transpose4(uint32_t w, int i) {
  uint32_t x = __shfl_xor_sync(0xffffffffu, w, 8);
  w = __byte_perm(w, x, i & 1 ? 0x3715 : 0x6240);
  x = __shfl_xor_sync(0xffffffffu, w, 16);
  return __byte_perm(w, x, i & 2 ? 0x3276 : 0x5410);
}

// Loads are typed by the template parameter IN, so that a thread's loads are all issued before the first is used (a branch
// on the type at each load would wait for it there). IN < 0: any type and alignment, element by element.
template <int IN>
__device__ __forceinline__ void load8(const void* p, int64_t i, int dtype, float (&v)[8]) {
  if constexpr (IN < 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = load_as(p, i + k, dtype);
  } else if constexpr (IN == NBL_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = IN == NBL_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[k]))
                                     : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
      v[2 * k] = f.x, v[2 * k + 1] = f.y;
    }
  }
}
// Eight elements as they are (elements lo .. lo + 3 and hi .. hi + 3; whole: hi = lo + 4), and widened: a thread reads several
// before it widens the first.
template <int IN>
struct Raw8 {
  uint4 r[IN == NBL_F32 ? 2 : 1];
};
template <int IN>
__device__ __forceinline__ Raw8<IN> read8(const void* p, int64_t lo, int64_t hi, bool whole) {
  Raw8<IN> x;
  if constexpr (IN == NBL_F32) {
    x.r[0] = *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + lo);
    x.r[1] = *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + hi);
  } else if (whole) {
    x.r[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + lo);
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + lo);
    const uint2 b = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + hi);
    x.r[0] = make_uint4(a.x, a.y, b.x, b.y);
  }
  return x;
}
template <int IN>
__device__ __forceinline__ void widen8(const Raw8<IN>& x, float (&v)[8]) {
  const uint32_t w[4] = {x.r[0].x, x.r[0].y, x.r[0].z, x.r[0].w};
  if constexpr (IN == NBL_F32) {
    const uint32_t z[4] = {x.r[1].x, x.r[1].y, x.r[1].z, x.r[1].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]), v[4 + k] = __uint_as_float(z[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = IN == NBL_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[k]))
                                     : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
      v[2 * k] = f.x, v[2 * k + 1] = f.y;
    }
  }
}
// Eight (four) consecutive fp32 values as `dtype`; 16-byte (8-byte for four 16-bit ones) aligned.
__device__ __forceinline__ void store8v(void* p, int64_t i, int dtype, const float (&v)[8]) {
  if (dtype == NBL_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (dtype == NBL_F16) {
        const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void store4v(void* p, int64_t i, int dtype, const float* v) {
  if (dtype == NBL_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (dtype == NBL_F16) {
        const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = make_uint2(w[0], w[1]);
  }
}
__device__ __forceinline__ void store8(void* p, int64_t i, int dtype, const float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) store_as(p, i + k, v[k], dtype);
}
__device__ __forceinline__ void add8(float (&v)[8], const float* b) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = __fadd_rn(v[k], b[k]);
}

// A chunk of a head with bias, rotated: element e and its partner (e ^ 1, or half the rotated part away) turn by the angle
// of their pair. cs[k]: (cos, sin) for element 8c + k. IN >= 0: the chunk, and its partner chunk where the partners are
// elsewhere, are whole and 16-byte aligned.
template <int IN>
__device__ __forceinline__ void rotated8(const void* src, int64_t row, int c, int dtype, const float* bias, bool neox, int rd,
                                         const float2 (&cs)[8], float (&v)[8]) {
  constexpr bool VEC = IN >= 0;
  const int e0 = 8 * c, half = rd / 2;
  load8<IN>(src, row + e0, dtype, v);
  if (bias) add8(v, bias + e0);
  if (e0 >= rd) return;
  float other[8];
  if (!neox) {
#pragma unroll
    for (int k = 0; k < 8; ++k) other[k] = v[k ^ 1];
  } else if (VEC) {
    const int o0 = e0 < half ? e0 + half : e0 - half;
    load8<IN>(src, row + o0, dtype, other);
    if (bias) add8(other, bias + o0);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int e = e0 + k, o = e < half ? e + half : e - half;
      other[k] = 0.f;
      if (e >= rd) continue;
      other[k] = load_as(src, row + o, dtype);
      if (bias) other[k] = __fadd_rn(other[k], bias[o]);
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int e = e0 + k;
    if (!VEC && e >= rd) continue;
    const bool first = neox ? e < half : (k & 1) == 0;
    float ra, rb;
    rope_rotate(first ? v[k] : other[k], first ? other[k] : v[k], cs[k], ra, rb);
    other[k] = first ? ra : rb;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (VEC || e0 + k < rd) v[k] = other[k];
}

// Pairs 4c .. 4c + 3 of a query head: both elements of a pair are one thread's, so the rotation may be in place. The first
// rd / 2 pairs are the rotated ones, the others the untouched elements two by two. cs[k]: (cos, sin) of pair 4c + k.
// The pairs of a whole chunk: elements lo .. lo + 3 and hi .. hi + 3 (rd is a multiple of 8: a chunk is rotated whole or not
// at all).
struct Chunk {
  bool turn, split;
  int lo, hi;
};
__device__ __forceinline__ Chunk chunk_of(int c, bool neox, int rd) {
  Chunk k;
  k.turn = 8 * c < rd, k.split = neox && k.turn;
  k.lo = k.split ? 4 * c : 8 * c, k.hi = k.split ? rd / 2 + 4 * c : 8 * c + 4;
  return k;
}
__device__ __forceinline__ void turn8(const Chunk& k, const float2 (&cs)[4], const float* bias, float (&v)[8]) {
  if (bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __fadd_rn(v[i], bias[k.lo + i]), v[4 + i] = __fadd_rn(v[4 + i], bias[k.hi + i]);
  }
  if (k.split) {
#pragma unroll
    for (int i = 0; i < 4; ++i) rope_rotate(v[i], v[4 + i], cs[i], v[i], v[4 + i]);
  } else if (k.turn) {
#pragma unroll
    for (int i = 0; i < 4; ++i) rope_rotate(v[2 * i], v[2 * i + 1], cs[i], v[2 * i], v[2 * i + 1]);
  }
}
__device__ __forceinline__ void query8_any(const void* src, void* dst, int64_t row, int c, int in_dtype, int out_dtype,
                                           const float* bias, bool neox, int rd, const float2 (&cs)[4]) {
  const int half = rd / 2;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int p = 4 * c + k;
    const bool turn = p < half;
    const int e0 = turn ? (neox ? p : 2 * p) : rd + 2 * (p - half), e1 = turn && neox ? p + half : e0 + 1;
    float x = load_as(src, row + e0, in_dtype), y = load_as(src, row + e1, in_dtype);
    if (bias) x = __fadd_rn(x, bias[e0]), y = __fadd_rn(y, bias[e1]);
    if (turn) rope_rotate(x, y, cs[k], x, y);
    store_as(dst, row + e0, x, out_dtype);
    store_as(dst, row + e1, y, out_dtype);
  }
}

// The touched pages of the items, one after another: page u's item, its fields, and the page's number in the sequence.
// With one page an item at most (decode steps), or more than kScanItems items, page u is page u % max_blocks of item
// u / max_blocks, and may be empty; otherwise every warp adds up the items' pages, 32 items at a time, and the grid is
// bounded by the rows of the packed activations (24 prompts of 97..2047 tokens: 1085 pages in place of 3096, of which two
// thirds were empty; an empty CTA still reads its item). Items whose rows overlap can have more pages
// than that: the last CTA flags it.
constexpr int kScanItems = 256;
struct Page {
  int item, start, len, pos0, block;
  bool valid;
};
__host__ __device__ inline bool scanned(int n_items, int max_blocks) { return max_blocks > 1 && n_items <= kScanItems; }
__device__ __forceinline__ bool item_ok(const Kv8Items& it, int start, int len, int pos0, int64_t tab_pos) {
  return item_fits(it, start, len, pos0) && int64_t(pos0) + len <= tab_pos;
}
__device__ __forceinline__ Page page_at(const Kv8Items& it, int max_blocks, int64_t tab_pos, int u, int* err) {
  Page p;
  p.valid = false;
  if (!scanned(it.n_items, max_blocks)) {
    p.item = u / max_blocks;
    p.start = it.start[p.item], p.len = it.len[p.item], p.pos0 = it.pos0[p.item];
    if (p.len <= 0) return p;
    if (!item_ok(it, p.start, p.len, p.pos0, tab_pos)) {
      if (threadIdx.x == 0) flag_error(err, kErrLength);
      return p;
    }
    p.block = p.pos0 / kPage + u % max_blocks;
    p.valid = int64_t(p.block) * kPage < int64_t(p.pos0) + p.len;
    return p;
  }
  const int lane = threadIdx.x & 31;
  const bool last = u == static_cast<int>(gridDim.x) - 1;
  int before = 0;
  for (int i0 = 0; i0 < it.n_items; i0 += 32) {
    const int i = i0 + lane;
    int start = 0, len = 0, pos0 = 0, n = 0;
    if (i < it.n_items) {
      start = it.start[i], len = it.len[i], pos0 = it.pos0[i];
      if (len > 0) {
        if (item_ok(it, start, len, pos0, tab_pos)) n = (pos0 + len - 1) / kPage - pos0 / kPage + 1;
        else if (u == 0) flag_error(err, kErrLength);
      }
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const uint32_t at = __ballot_sync(0xffffffffu, u < before + inc);
    if (at && !p.valid) {
      const int l = __ffs(at) - 1;  // the first item that ends behind u
      p.item = i0 + l;
      p.start = __shfl_sync(0xffffffffu, start, l), p.len = __shfl_sync(0xffffffffu, len, l);
      p.pos0 = __shfl_sync(0xffffffffu, pos0, l);
      p.block = p.pos0 / kPage + u - before - __shfl_sync(0xffffffffu, inc - n, l);
      p.valid = true;
      if (!last) return p;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (before > static_cast<int>(gridDim.x) && threadIdx.x == 0) flag_error(err, kErrLength);
  return p;
}

// CTAs (touched page, part): a part for every KV head (the page's new tokens' keys and values), then one for every 8 query
// heads of those tokens, 8 (fp32: 4) of them in flight. Bound: memory (each input once, each output once). One part per CTA:
// 888 CTAs that took the parts in turn were slower (83 against 48 us for 24 ragged prompts).
template <int D, int KIND, int IN>
__global__ void __launch_bounds__(kCtaThreads<D>, D == 64 ? 7 : 4)
    kv8_append_kernel(const Kv8Items it, const Kv8Append a, uint8_t* pool, int64_t n_pages, int n_kv_heads, int max_blocks,
                      int* err) {
  constexpr bool VEC = IN >= 0;
  __shared__ float red[2][kCtaThreads<D> / 32];
  const int rd = a.rotary_dim, part = blockIdx.y;
  const Page pg = page_at(it, max_blocks, a.tab_pos, blockIdx.x, err);
  if (!pg.valid) return;
  const Place pl = place_of(threadIdx.x);
  const int c = pl.c, tok = pl.tok;
  const int64_t end = int64_t(pg.pos0) + pg.len;
  const int base = pg.block * kPage;
  const int slot0 = max(pg.pos0 - base, 0), slot1 = static_cast<int>(min(end - base, int64_t(kPage)));  // the new tokens' places
  const bool is_new = tok >= slot0 && tok < slot1, is_old = tok < slot0;
  const int64_t row = int64_t(pg.start) + (base + tok - pg.pos0);  // of the packed activations
  const float2* tab = a.tab + int64_t(base + tok) * (rd / 2);

  if (part >= n_kv_heads) {
    if (!is_new) return;
    const int head0 = (part - n_kv_heads) * 8, heads = min(8, a.n_heads - head0);
    const int64_t q0 = (row * a.n_heads + head0) * D;
    const float* bq = a.bq ? a.bq + head0 * D : nullptr;
    float2 cs[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) cs[k] = 4 * c + k < rd / 2 ? tab[4 * c + k] : make_float2(1.f, 0.f);
    if constexpr (VEC) {
      const Chunk ch = chunk_of(c, a.neox, rd);
      constexpr int kQHeads = IN == NBL_F32 ? 4 : 8;
      for (int h0 = 0; h0 < heads; h0 += kQHeads) {
        Raw8<IN> x[kQHeads];
#pragma unroll
        for (int h = 0; h < kQHeads; ++h)
          if (h0 + h < heads) x[h] = read8<IN>(a.q_in, q0 + (h0 + h) * D + ch.lo, q0 + (h0 + h) * D + ch.hi, !ch.split);
#pragma unroll
        for (int h = 0; h < kQHeads; ++h) {
          if (h0 + h >= heads) break;
          float v[8];
          widen8<IN>(x[h], v);
          turn8(ch, cs, bq ? bq + (h0 + h) * D : nullptr, v);
          if (ch.split) {
            store4v(a.q_out, q0 + (h0 + h) * D + ch.lo, a.q_out_dtype, v);
            store4v(a.q_out, q0 + (h0 + h) * D + ch.hi, a.q_out_dtype, v + 4);
          } else {
            store8v(a.q_out, q0 + (h0 + h) * D + ch.lo, a.q_out_dtype, v);
          }
        }
      }
    } else {
      for (int h = 0; h < heads; ++h)
        query8_any(a.q_in, a.q_out, q0 + h * D, c, a.in_dtype, a.q_out_dtype, bq ? bq + h * D : nullptr, a.neox, rd, cs);
    }
    return;
  }

  const int kvh = part;
  const int32_t page = it.page_table[int64_t(pg.item) * it.pt_stride + pg.block];
  float k8[8], v8[8];
  if (is_new) {
    float2 cs[8];
    if (8 * c < rd) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = 8 * c + k;
        if (VEC && !a.neox && (k & 1)) cs[k] = cs[k - 1];
        else if (VEC || e < rd) cs[k] = tab[a.neox ? (e < rd / 2 ? e : e - rd / 2) : e >> 1];
      }
    }
    load8<IN>(a.v_in, (row * n_kv_heads + kvh) * D + 8 * c, a.in_dtype, v8);
    rotated8<IN>(a.k_in, (row * n_kv_heads + kvh) * D, c, a.in_dtype, a.bk ? a.bk + kvh * D : nullptr, a.neox, rd, cs, k8);
    if (a.bv) add8(v8, a.bv + kvh * D + 8 * c);
  }
  if (page < 0 || page >= n_pages) {
    if (threadIdx.x == 0) flag_error(err, kErrPageId);
    return;
  }
  uint8_t* blk = pool + int64_t(page) * page_bytes(D, n_kv_heads) + int64_t(kvh) * block_bytes(D);
  float* sc = reinterpret_cast<float*>(blk + scale_off(D));
  // largest magnitudes of the new tokens
  float amax[2] = {0.f, 0.f};
  bool odd = false;
  if (is_new) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      odd = odd || !(fabsf(k8[k]) <= kHuge) || !(fabsf(v8[k]) <= kHuge);
      k8[k] = k8[k] != k8[k] ? 0.f : fminf(fmaxf(k8[k], -kHuge), kHuge);
      v8[k] = v8[k] != v8[k] ? 0.f : fminf(fmaxf(v8[k], -kHuge), kHuge);
      amax[0] = fmaxf(amax[0], fabsf(k8[k]));
      amax[1] = fmaxf(amax[1], fabsf(v8[k]));
    }
  }
  if (odd) flag_error(err, kErrNonFinite);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax[w] = fmaxf(amax[w], __shfl_xor_sync(0xffffffffu, amax[w], o));
    if ((threadIdx.x & 31) == 0) red[w][threadIdx.x >> 5] = amax[w];
  }
  float s[2], inv[2], ratio[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) s[w] = slot0 > 0 ? sc[w] : 0.f;  // the scale of the tokens already there
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kCtaThreads<D> / 32; ++i) m = fmaxf(m, red[w][i]);
    const float old = s[w];
    s[w] = fmaxf(old, m >= kTiny ? __fmul_rn(m, 1.f / code_max<KIND>()) : 0.f);
    inv[w] = s[w] > 0.f ? __fdiv_rn(1.f, s[w]) : 0.f;
    ratio[w] = __fmul_rn(old, inv[w]);
  }
  // keys: two words of 4 dims; old ones are rounded again to the new scale
  uint2* kdst = reinterpret_cast<uint2*>(blk + key_off(tok, 8 * c));
  uint32_t kw[2];
  if (is_old) {
    const uint2 was = *kdst;
    kw[0] = from_word<KIND>(was.x), kw[1] = from_word<KIND>(was.y);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t w = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float x = is_old ? __fmul_rn(decode<KIND>(kw[j] >> (8 * b)), ratio[0])
                             : (is_new ? __fmul_rn(k8[4 * j + b], inv[0]) : 0.f);
      w |= encode<KIND>(x) << (8 * b);
    }
    kw[j] = to_word<KIND>(w);
  }
  *kdst = make_uint2(kw[0], kw[1]);
  // values: this token's codes, exchanged among the four lanes of a word, so that lane i has the words of dims 8c + i and
  // 8c + 4 + i
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t w = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) w |= encode<KIND>(is_new ? __fmul_rn(v8[4 * j + b], inv[1]) : 0.f) << (8 * b);
    w = transpose4(w, pl.i);
    uint32_t* dst = reinterpret_cast<uint32_t*>(blk + value_off(D, pl.t, 8 * c + 4 * j + pl.i));
    if (slot0 > 0) {
      const uint32_t old = from_word<KIND>(*dst);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (2 * pl.t + (b & 1) + 8 * (b >> 1) >= slot0) continue;
        const uint32_t x = encode<KIND>(__fmul_rn(decode<KIND>(old >> (8 * b)), ratio[1]));
        w = (w & ~(0xffu << (8 * b))) | x << (8 * b);
      }
    }
    *dst = to_word<KIND>(w);
  }
  if (threadIdx.x < 2) sc[threadIdx.x] = s[threadIdx.x];
}

// CTAs (touched page, stretch of kReadHeads KV heads, all in flight): a row is code * scale.
constexpr int kReadHeads = 4;
template <int D, int KIND>
__global__ void __launch_bounds__(kCtaThreads<D>) kv8_read_kernel(const Kv8Items it, const uint8_t* pool, int64_t n_pages,
                                                                  int n_kv_heads, int max_blocks, void* k_out, void* v_out,
                                                                  int out_dtype, bool vec, int* err) {
  const Page at_page = page_at(it, max_blocks, INT64_MAX, blockIdx.x, err);
  if (!at_page.valid) return;
  const Place pl = place_of(threadIdx.x);
  const int start = at_page.start, pos0 = at_page.pos0;
  const int64_t end = int64_t(pos0) + at_page.len;
  const int base = at_page.block * kPage;
  const int32_t page = it.page_table[int64_t(at_page.item) * it.pt_stride + at_page.block];
  if (page < 0 || page >= n_pages) {
    if (threadIdx.x == 0) flag_error(err, kErrPageId);
    return;
  }
  const int pos = base + pl.tok;
  const bool mine = pos >= pos0 && pos < end;
  const int64_t row = int64_t(start) + (pos - pos0);
  const uint8_t* pg = pool + int64_t(page) * page_bytes(D, n_kv_heads);
  const int h0 = blockIdx.y * kReadHeads, n = min(kReadHeads, n_kv_heads - h0);
  uint2 kw[kReadHeads];
  uint32_t vw[kReadHeads][2];
  float2 sc[kReadHeads];
#pragma unroll
  for (int h = 0; h < kReadHeads; ++h) {
    if (h >= n) break;
    const uint8_t* blk = pg + int64_t(h0 + h) * block_bytes(D);
    kw[h] = *reinterpret_cast<const uint2*>(blk + key_off(pl.tok, 8 * pl.c));
#pragma unroll
    for (int j = 0; j < 2; ++j)
      vw[h][j] = *reinterpret_cast<const uint32_t*>(blk + value_off(D, pl.t, 8 * pl.c + 4 * j + pl.i));
    sc[h] = *reinterpret_cast<const float2*>(blk + scale_off(D));
  }
#pragma unroll
  for (int h = 0; h < kReadHeads; ++h) {
    if (h >= n) break;
    const uint32_t v2[2] = {transpose4(from_word<KIND>(vw[h][0]), pl.i), transpose4(from_word<KIND>(vw[h][1]), pl.i)};
    const uint32_t k2[2] = {from_word<KIND>(kw[h].x), from_word<KIND>(kw[h].y)};
    float k8[8], v8[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      k8[k] = __fmul_rn(decode<KIND>(k2[k >> 2] >> (8 * (k & 3))), sc[h].x);
      v8[k] = __fmul_rn(decode<KIND>(v2[k >> 2] >> (8 * (k & 3))), sc[h].y);
    }
    if (!mine) continue;
    const int64_t at = (row * n_kv_heads + h0 + h) * D + 8 * pl.c;
    if (vec) {
      if (k_out) store8v(k_out, at, out_dtype, k8);
      if (v_out) store8v(v_out, at, out_dtype, v8);
    } else {
      if (k_out) store8(k_out, at, out_dtype, k8);
      if (v_out) store8(v_out, at, out_dtype, v8);
    }
  }
}

// codes [n, 2, n_kv_heads, 16, D] (int8, or e4m3 bytes) and scales [n, 2, n_kv_heads] to / from pages page_ids[i].
template <int D, int KIND, bool IMPORT>
__global__ void __launch_bounds__(kThreads) kv8_pages_kernel(uint8_t* pool, int64_t n_pages, int n_kv_heads,
                                                             const int32_t* __restrict__ page_ids, uint8_t* codes,
                                                             float* scales, int* err) {
  const int64_t i = blockIdx.x;
  const int kvh = blockIdx.y;
  const int32_t page = page_ids[i];
  if (page < 0 || page >= n_pages) {
    if (threadIdx.x == 0) flag_error(err, kErrPageId);
    return;
  }
  uint8_t* pg = pool + int64_t(page) * page_bytes(D, n_kv_heads);
  uint8_t* blk = pg + int64_t(kvh) * block_bytes(D);
  float* sc = reinterpret_cast<float*>(blk + scale_off(D));
  for (int w = 0; w < 2; ++w) {
    float v = 0.f;
    if constexpr (IMPORT) {
      v = scales[(i * 2 + w) * n_kv_heads + kvh];
      if (!(v >= 0.f && v <= kHuge)) {
        if (threadIdx.x == 0) flag_error(err, kErrNonFinite);
        v = 0.f;
      }
      if (v < kTiny / 448.f) v = 0.f;  // as the append: no scale whose reciprocal is not finite
    }
    uint8_t* src = codes + ((i * 2 + w) * n_kv_heads + kvh) * (kPage * D);
    for (int u = threadIdx.x; u < kPage * D / 4; u += kThreads) {  // words
      int at, tok[4], dim[4];
      if (w == 0) {
        const int d0 = (u % (D / 4)) * 4;
        at = key_off(u / (D / 4), d0);
#pragma unroll
        for (int b = 0; b < 4; ++b) tok[b] = u / (D / 4), dim[b] = d0 + b;
      } else {
        const int t = u / D;
        at = value_off(D, t, u % D);
#pragma unroll
        for (int b = 0; b < 4; ++b) tok[b] = 2 * t + (b & 1) + 8 * (b >> 1), dim[b] = u % D;
      }
      uint32_t* word = reinterpret_cast<uint32_t*>(blk + at);
      if constexpr (IMPORT) {
        uint32_t c = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t x = src[tok[b] * D + dim[b]];
          if (KIND == NBL_E4M3 && (x & 0x7f) == 0x7f) {  // e4m3's NaN
            flag_error(err, kErrNonFinite);
            x = 0;
          }
          c |= x << (8 * b);
        }
        *word = to_word<KIND>(v > 0.f ? c : 0u);  // a scale of 0 has codes of 0
      } else {
        const uint32_t c = from_word<KIND>(*word);
#pragma unroll
        for (int b = 0; b < 4; ++b) src[tok[b] * D + dim[b]] = static_cast<uint8_t>(c >> (8 * b));
      }
    }
    if (threadIdx.x == 0) {
      float* s = scales + (i * 2 + w) * n_kv_heads + kvh;
      if constexpr (IMPORT) {
        sc[w] = v;
      } else {
        *s = sc[w];
      }
    }
  }
}

__global__ void kv8_clear_kernel(uint8_t* pool, int64_t n_pages, int n_kv_heads, int d) {
  for (int64_t u = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; u < n_pages * n_kv_heads;
       u += int64_t(gridDim.x) * blockDim.x) {
    uint8_t* blk = pool + u / n_kv_heads * page_bytes(d, n_kv_heads) + u % n_kv_heads * block_bytes(d);
    *reinterpret_cast<uint4*>(blk + scale_off(d)) = uint4{};
  }
}

__global__ void rotary_table_kernel(float2* __restrict__ tab, int64_t n, const double* __restrict__ freq, int n_pairs,
                                    double mul) {
  for (int64_t u = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; u < n; u += int64_t(gridDim.x) * blockDim.x) {
    double s, c;
    sincos(static_cast<double>(u / n_pairs) * freq[u % n_pairs], &s, &c);
    tab[u] = make_float2(static_cast<float>(c * mul), static_cast<float>(s * mul));
  }
}

// Runs f.operator()<D, KIND>() for the pool's head_dim and dtype.
template <class F>
void with_kind(const nbl_kv* kv, F&& f) {
  const bool i8 = kv->cfg.dtype == NBL_I8;
  if (kv->cfg.head_dim == 64) {
    if (i8) f(std::integral_constant<int, 64>{}, std::integral_constant<int, NBL_I8>{});
    else f(std::integral_constant<int, 64>{}, std::integral_constant<int, NBL_E4M3>{});
  } else {
    if (i8) f(std::integral_constant<int, 128>{}, std::integral_constant<int, NBL_I8>{});
    else f(std::integral_constant<int, 128>{}, std::integral_constant<int, NBL_E4M3>{});
  }
}

// Pages that max_len tokens can touch, from any first position.
int touched_pages(int max_len) { return (max_len + kPage - 2) / kPage + 1; }

// Pages that the items can touch (see page_at).
unsigned pages_bound(const Kv8Items& it, const char* what) {
  const int blocks = touched_pages(it.max_len);
  int64_t n = int64_t(it.n_items) * blocks;
  if (scanned(it.n_items, blocks)) n = std::min<int64_t>(n, it.n_rows / kPage + 2 * int64_t(it.n_items));
  if (n > 0x7fffffff) fail(NBL_E_INVALID, std::string(what) + ": n_items * pages per item exceeds 2^31");
  return static_cast<unsigned>(n);
}

}  // namespace

void launch_kv8_clear(cudaStream_t st, const nbl_kv* kv) {
  // code 0 is the byte 128 for I8, 0 for E4M3
  check_cuda(cudaMemsetAsync(kv->pool, kv->cfg.dtype == NBL_I8 ? 0x80 : 0, kv->bytes, st), "kv pool zero-fill");
  kv8_clear_kernel<<<1184, 256, 0, st>>>(static_cast<uint8_t*>(kv->pool), kv->cfg.n_pages, kv->cfg.n_kv_heads,
                                         kv->cfg.head_dim);
  check_cuda(cudaGetLastError(), "kv pool zero-fill");
}

void launch_kv8_append(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, const Kv8Append& a, int* err) {
  const int blocks = touched_pages(items.max_len);
  const int64_t parts = kv->cfg.n_kv_heads + (a.n_heads + 7) / 8;
  if (parts > 65535) fail(NBL_E_INVALID, "rotary_kv_append: too many heads");
  const dim3 grid(pages_bound(items, "rotary_kv_append"), static_cast<unsigned>(parts));
  const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const bool vec = ((bits(a.q_in) | bits(a.k_in) | bits(a.v_in) | bits(a.q_out)) & 15u) == 0 &&
                   a.rotary_dim % (a.neox ? 16 : 8) == 0;
  with_kind(kv, [&](auto d, auto kind) {
    auto* k = !vec                      ? kv8_append_kernel<d(), kind(), -1>
              : a.in_dtype == NBL_F32 ? kv8_append_kernel<d(), kind(), NBL_F32>
              : a.in_dtype == NBL_F16 ? kv8_append_kernel<d(), kind(), NBL_F16>
                                      : kv8_append_kernel<d(), kind(), NBL_BF16>;
    k<<<grid, kCtaThreads<d()>, 0, st>>>(items, a, static_cast<uint8_t*>(kv->pool), kv->cfg.n_pages, kv->cfg.n_kv_heads,
                                         blocks, err);
  });
  check_cuda(cudaGetLastError(), "rotary_kv_append launch");
}

void launch_kv8_read(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, void* k_out, void* v_out, int out_dtype,
                     int* err) {
  const int blocks = touched_pages(items.max_len);
  const dim3 grid(pages_bound(items, "kv_read"), static_cast<unsigned>((kv->cfg.n_kv_heads + kReadHeads - 1) / kReadHeads));
  const bool vec = ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u) == 0;
  with_kind(kv, [&](auto d, auto kind) {
    kv8_read_kernel<d(), kind()><<<grid, kCtaThreads<d()>, 0, st>>>(items, static_cast<const uint8_t*>(kv->pool),
                                                                    kv->cfg.n_pages, kv->cfg.n_kv_heads, blocks, k_out, v_out,
                                                                    out_dtype, vec, err);
  });
  check_cuda(cudaGetLastError(), "kv_read launch");
}

void launch_kv8_import(cudaStream_t st, const nbl_kv* kv, const int32_t* page_ids, int64_t n, const void* codes,
                       const float* scales, int* err) {
  const dim3 grid(static_cast<unsigned>(n), static_cast<unsigned>(kv->cfg.n_kv_heads));
  with_kind(kv, [&](auto d, auto kind) {
    kv8_pages_kernel<d(), kind(), true><<<grid, kThreads, 0, st>>>(
        static_cast<uint8_t*>(kv->pool), kv->cfg.n_pages, kv->cfg.n_kv_heads, page_ids,
        static_cast<uint8_t*>(const_cast<void*>(codes)), const_cast<float*>(scales), err);
  });
  check_cuda(cudaGetLastError(), "kv_import launch");
}

void launch_kv8_export(cudaStream_t st, const nbl_kv* kv, const int32_t* page_ids, int64_t n, void* codes,
                       float* scales, int* err) {
  const dim3 grid(static_cast<unsigned>(n), static_cast<unsigned>(kv->cfg.n_kv_heads));
  with_kind(kv, [&](auto d, auto kind) {
    kv8_pages_kernel<d(), kind(), false><<<grid, kThreads, 0, st>>>(static_cast<uint8_t*>(kv->pool), kv->cfg.n_pages,
                                                                    kv->cfg.n_kv_heads, page_ids,
                                                                    static_cast<uint8_t*>(codes), scales, err);
  });
  check_cuda(cudaGetLastError(), "kv_export launch");
}

void launch_rotary_table(cudaStream_t st, float2* tab, int64_t n_pos, const double* freq, int n_pairs, double mul) {
  const int64_t n = n_pos * n_pairs;
  const int grid = static_cast<int>(std::min<int64_t>((n + 255) / 256, 148 * 16));
  rotary_table_kernel<<<grid, 256, 0, st>>>(tab, n, freq, n_pairs, mul);
  check_cuda(cudaGetLastError(), "rotary table launch");
}

}  // namespace nbl
