// Writing and reading the 8-bit K/V pool: the fused bias -> rotary -> quantize -> page write of new tokens, the read
// of cache rows as floats, and the import / export of whole pages.
//
// Quantization. A block is the 16 places of one (page, KV head), keys and values apart. With amax the largest
// magnitude among the tokens that a call adds to the block and s_old the scale of the tokens that were there,
//   s = max(s_old, amax * (1 / code_max)),   new code = round(x / s),   old code = round(code * s_old / s),
// so a block's scale only grows while it fills, and each growth adds at most half a step to an old token's error. The
// places after the last token are set to 0. Products use the fp32 reciprocal of s; all of it is IEEE fp32, each step
// rounded once, so the codes do not depend on how the work is spread over threads.
#include <algorithm>

#include "kv8.cuh"

namespace nbl {
namespace {

using namespace kv8;

constexpr int kThreads = 128;

// Element indices of rotation pair p of a head (p < rotary_dim / 2), or of the p-th pair of untouched elements.
__device__ __forceinline__ void pair_of(int p, int rd, bool neox, int& e0, int& e1) {
  const int half = rd / 2;
  if (p < half) {
    e0 = neox ? p : 2 * p;
    e1 = neox ? p + half : 2 * p + 1;
  } else {
    e0 = rd + 2 * (p - half);
    e1 = e0 + 1;
  }
}

// One CTA per (touched page of an item, KV head): the page's new tokens' keys and values, and the query heads of that
// KV head for those tokens.
template <int D, int KIND>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const Kv8Items it, const Kv8Append a, uint8_t* pool,
                                                              int64_t n_pages, int n_kv_heads, int max_blocks, int* err) {
  __shared__ float xs[2][kPage][D + 1];
  __shared__ float red[2][kThreads / 32];
  const int item = blockIdx.x / max_blocks, kvh = blockIdx.y;
  const int start = it.start[item], len = it.len[item], pos0 = it.pos0[item];
  if (len <= 0) return;
  const int64_t end = int64_t(pos0) + len;
  const int64_t block = int64_t(pos0) / kPage + blockIdx.x % max_blocks;
  if (pos0 < 0 || start < 0 || int64_t(start) + len > it.n_rows || end > int64_t(it.pt_stride) * kPage || end > a.tab_pos) {
    if (threadIdx.x == 0) flag_error(err, kErrLength);
    return;
  }
  if (block * kPage >= end) return;
  const int first = static_cast<int>(max(int64_t(pos0), block * kPage));       // positions first .. last
  const int last = static_cast<int>(min(end, block * kPage + kPage)) - 1;
  const int n_new = last - first + 1, slot0 = first - static_cast<int>(block) * kPage;
  const int group = a.n_heads / n_kv_heads, rd = a.rotary_dim, half = rd / 2;

  // queries: rotated straight to q_out
  for (int u = threadIdx.x; u < n_new * group * (D / 2); u += kThreads) {
    const int p = u % (D / 2), h = kvh * group + (u / (D / 2)) % group, i = u / (D / 2 * group);
    const int64_t base = (int64_t(start) + (first - pos0) + i) * a.n_heads * D + int64_t(h) * D;
    int e0, e1;
    pair_of(p, rd, a.neox, e0, e1);
    float x0 = load_as(a.q_in, base + e0, a.in_dtype), x1 = load_as(a.q_in, base + e1, a.in_dtype);
    if (a.bq) x0 = __fadd_rn(x0, a.bq[h * D + e0]), x1 = __fadd_rn(x1, a.bq[h * D + e1]);
    if (p < half) rope_rotate(x0, x1, a.tab[int64_t(first + i) * half + p], x0, x1);
    store_as(a.q_out, base + e0, x0, a.q_out_dtype);
    store_as(a.q_out, base + e1, x1, a.q_out_dtype);
  }
  const int32_t page = it.page_table[int64_t(item) * it.pt_stride + block];
  if (page < 0 || page >= n_pages) {
    if (threadIdx.x == 0) flag_error(err, kErrPageId);
    return;
  }
  // keys and values of the new tokens into shared memory, with their largest magnitudes
  float amax[2] = {0.f, 0.f};
  bool odd = false;
  for (int u = threadIdx.x; u < 2 * n_new * (D / 2); u += kThreads) {
    const int p = u % (D / 2), i = u / (D / 2) % n_new, w = u / (D / 2 * n_new);
    const int64_t base = (int64_t(start) + (first - pos0) + i) * n_kv_heads * D + int64_t(kvh) * D;
    int e0, e1;
    pair_of(p, rd, a.neox, e0, e1);
    const void* src = w ? a.v_in : a.k_in;
    const float* bias = w ? a.bv : a.bk;
    float x0 = load_as(src, base + e0, a.in_dtype), x1 = load_as(src, base + e1, a.in_dtype);
    if (bias) x0 = __fadd_rn(x0, bias[kvh * D + e0]), x1 = __fadd_rn(x1, bias[kvh * D + e1]);
    if (w == 0 && p < half) rope_rotate(x0, x1, a.tab[int64_t(first + i) * half + p], x0, x1);
    odd = odd || !(fabsf(x0) <= kHuge) || !(fabsf(x1) <= kHuge);
    x0 = x0 != x0 ? 0.f : fminf(fmaxf(x0, -kHuge), kHuge);
    x1 = x1 != x1 ? 0.f : fminf(fmaxf(x1, -kHuge), kHuge);
    xs[w][slot0 + i][e0] = x0;
    xs[w][slot0 + i][e1] = x1;
    amax[w] = fmaxf(amax[w], fmaxf(fabsf(x0), fabsf(x1)));
  }
  if (odd) flag_error(err, kErrNonFinite);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax[w] = fmaxf(amax[w], __shfl_xor_sync(0xffffffffu, amax[w], o));
    if ((threadIdx.x & 31) == 0) red[w][threadIdx.x >> 5] = amax[w];
  }
  uint8_t* pg = pool + int64_t(page) * page_bytes(D, n_kv_heads);
  uint8_t* blk = pg + int64_t(kvh) * block_bytes(D);
  float* sc = reinterpret_cast<float*>(blk + scale_off(D));
  float s[2], inv[2], ratio[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) s[w] = slot0 > 0 ? sc[w] : 0.f;  // the scale of the tokens already there
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) m = fmaxf(m, red[w][i]);
    const float old = s[w];
    s[w] = fmaxf(old, m >= kTiny ? __fmul_rn(m, 1.f / code_max<KIND>()) : 0.f);
    inv[w] = s[w] > 0.f ? __fdiv_rn(1.f, s[w]) : 0.f;
    ratio[w] = __fmul_rn(old, inv[w]);
  }
  const int slot1 = slot0 + n_new;
  // keys: 16 consecutive dims of one token per step
  for (int u = threadIdx.x; u < kPage * D / 16; u += kThreads) {
    const int tok = u / (D / 16), d0 = (u % (D / 16)) * 16;
    uint4* dst = reinterpret_cast<uint4*>(blk + key_off(tok, d0));
    const uint4 was = tok < slot0 ? *dst : uint4{};
    const uint32_t o[4] = {was.x, was.y, was.z, was.w};
    uint32_t w4[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t old = from_word<KIND>(o[k]);
      w4[k] = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float x = tok < slot0 ? __fmul_rn(decode<KIND>(old >> (8 * b)), ratio[0])
                                    : (tok < slot1 ? __fmul_rn(xs[0][tok][d0 + 4 * k + b], inv[0]) : 0.f);
        w4[k] |= encode<KIND>(x) << (8 * b);
      }
      w4[k] = to_word<KIND>(w4[k]);
    }
    *dst = make_uint4(w4[0], w4[1], w4[2], w4[3]);
  }
  // values: dims 8j + g (j = 0..3) of tokens 2t, 2t+1, 2t+8, 2t+9 per step
  for (int u = threadIdx.x; u < kPage * D / 16; u += kThreads) {
    const int c = u >> 5, g = (u & 31) >> 2, t = u & 3;
    uint4* dst = reinterpret_cast<uint4*>(blk + kPage * D + u * 16);
    const uint4 was = slot0 > 0 ? *dst : uint4{};
    const uint32_t o[4] = {was.x, was.y, was.z, was.w};
    uint32_t w4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t old = from_word<KIND>(o[j]);
      w4[j] = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int tok = 2 * t + (b & 1) + 8 * (b >> 1), dim = 32 * c + 8 * j + g;
        const float x = tok < slot0 ? __fmul_rn(decode<KIND>(old >> (8 * b)), ratio[1])
                                    : (tok < slot1 ? __fmul_rn(xs[1][tok][dim], inv[1]) : 0.f);
        w4[j] |= encode<KIND>(x) << (8 * b);
      }
      w4[j] = to_word<KIND>(w4[j]);
    }
    *dst = make_uint4(w4[0], w4[1], w4[2], w4[3]);
  }
  if (threadIdx.x < 2) sc[threadIdx.x] = s[threadIdx.x];
}

// One CTA per (touched page of an item, KV head): its rows as code * scale.
template <int D, int KIND>
__global__ void __launch_bounds__(kThreads) kv8_read_kernel(const Kv8Items it, const uint8_t* pool, int64_t n_pages,
                                                            int n_kv_heads, int max_blocks, void* k_out, void* v_out,
                                                            int out_dtype, int* err) {
  const int item = blockIdx.x / max_blocks, kvh = blockIdx.y;
  const int start = it.start[item], len = it.len[item], pos0 = it.pos0[item];
  if (len <= 0) return;
  const int64_t end = int64_t(pos0) + len;
  const int64_t block = int64_t(pos0) / kPage + blockIdx.x % max_blocks;
  if (pos0 < 0 || start < 0 || int64_t(start) + len > it.n_rows || end > int64_t(it.pt_stride) * kPage) {
    if (threadIdx.x == 0) flag_error(err, kErrLength);
    return;
  }
  if (block * kPage >= end) return;
  const int32_t page = it.page_table[int64_t(item) * it.pt_stride + block];
  if (page < 0 || page >= n_pages) {
    if (threadIdx.x == 0) flag_error(err, kErrPageId);
    return;
  }
  const int first = static_cast<int>(max(int64_t(pos0), block * kPage));
  const int n = static_cast<int>(min(end, block * kPage + kPage)) - first;
  const int slot0 = first - static_cast<int>(block) * kPage;
  const uint8_t* pg = pool + int64_t(page) * page_bytes(D, n_kv_heads);
  const uint8_t* blk = pg + int64_t(kvh) * block_bytes(D);
  const float* sc = reinterpret_cast<const float*>(blk + scale_off(D));
  const float ks = sc[0], vs = sc[1];
  for (int u = threadIdx.x; u < n * D; u += kThreads) {
    const int i = u / D, dim = u % D, tok = slot0 + i;
    const int64_t at = (int64_t(start) + (first - pos0) + i) * n_kv_heads * D + int64_t(kvh) * D + dim;
    if (k_out) {
      const uint32_t w = from_word<KIND>(*reinterpret_cast<const uint32_t*>(blk + key_off(tok, dim & ~3)));
      store_as(k_out, at, __fmul_rn(decode<KIND>(w >> (8 * (dim & 3))), ks), out_dtype);
    }
    if (v_out) {
      const uint32_t w = from_word<KIND>(*reinterpret_cast<const uint32_t*>(blk + value_off(D, value_t(tok), dim)));
      store_as(v_out, at, __fmul_rn(decode<KIND>(w >> (8 * value_i(tok))), vs), out_dtype);
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

void grid_check(int64_t ctas, const char* what) {
  if (ctas > 0x7fffffff) fail(NBL_E_INVALID, std::string(what) + ": n_items * pages per item exceeds 2^31");
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
  grid_check(int64_t(items.n_items) * blocks, "rotary_kv_append");
  const dim3 grid(static_cast<unsigned>(items.n_items) * blocks, static_cast<unsigned>(kv->cfg.n_kv_heads));
  with_kind(kv, [&](auto d, auto kind) {
    kv8_append_kernel<d(), kind()><<<grid, kThreads, 0, st>>>(items, a, static_cast<uint8_t*>(kv->pool),
                                                              kv->cfg.n_pages, kv->cfg.n_kv_heads, blocks, err);
  });
  check_cuda(cudaGetLastError(), "rotary_kv_append launch");
}

void launch_kv8_read(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, void* k_out, void* v_out, int out_dtype,
                     int* err) {
  const int blocks = touched_pages(items.max_len);
  grid_check(int64_t(items.n_items) * blocks, "kv_read");
  const dim3 grid(static_cast<unsigned>(items.n_items) * blocks, static_cast<unsigned>(kv->cfg.n_kv_heads));
  with_kind(kv, [&](auto d, auto kind) {
    kv8_read_kernel<d(), kind()><<<grid, kThreads, 0, st>>>(items, static_cast<const uint8_t*>(kv->pool),
                                                            kv->cfg.n_pages, kv->cfg.n_kv_heads, blocks, k_out, v_out,
                                                            out_dtype, err);
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
