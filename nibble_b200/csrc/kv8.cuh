// The 8-bit paged K/V pool (dtype NBL_I8 or NBL_E4M3): where a code lies, and the conversions of codes.
//
// A page holds 16 token positions of every KV head. Each (page, KV head) is one block of 32 * D + 16 bytes -- its keys,
// its values, then their two scales -- so attention fetches it with one bulk copy:
//   page = [n_kv_heads][ keys 16 * D | values 16 * D | key scale, value scale, 0, 0 (fp32) ]  (rounded to 128)
// A key element is code * key scale, a value element code * value scale.
//
// The codes lie in the order in which the m16n8k16 tensor-core instruction wants them, so a lane (g = lane / 4,
// t = lane % 4) of a warp fetches its operands with 16-byte loads that meet no bank twice:
//   keys    [D / 64][16 tokens][64 dims]: lane (g, t) reads the 16 dims 16t.. of token g (and of g + 8). The order of
//           the dims inside the contraction is free as long as the query has the same one.
//   values  [D / 32][32 lanes][4 tiles j][4 tokens i]: lane (g, t) holds dim 8j + g of tokens 2t, 2t+1, 2t+8, 2t+9.
// A word is four codes (four dims of a token, or four tokens of a dim), stored so that they widen to two fp16 pairs with
// few instructions:
//   NBL_I8    byte i = code i + 128: the widening is a byte permute and a subtraction.
//   NBL_E4M3  an fp16 whose sign is a code's and whose next bits are 0, eeee, mmm, 0... is the code times 2^-8 (also for
//             the subnormal codes), so codes 0 and 1 stand at those bits of the word's two halves, and codes 2 and 3 at the
//             bits between (sign at bit 14, the rest at 6..0): one mask gives the first pair, two shifts and two
//             masks the second. (The conversion instruction runs at a quarter of that rate: decode of 256 rows of 4097
//             tokens took 262 us with it, when NBL_I8 took 207.)
// Every code and scale in a pool is finite: the append saturates and the import refuses, so a masked token's weight
// of 0 always gives 0.
#pragma once
#include <cuda_fp8.h>

#include "nbl_device.cuh"
#include "nbl_internal.h"

namespace nbl {
namespace kv8 {

constexpr int kPage = 16;

__host__ __device__ constexpr int block_bytes(int d) { return 2 * kPage * d + 16; }
__host__ __device__ inline int64_t page_bytes(int d, int n_kv_heads) {
  return (int64_t(n_kv_heads) * block_bytes(d) + 127) / 128 * 128;
}
// Offset of the two scales inside their block.
__host__ __device__ constexpr int scale_off(int d) { return 2 * kPage * d; }
// Offset of the word with a token's dims dim .. dim + 3 (dim a multiple of 4).
__device__ __forceinline__ int key_off(int tok, int dim) { return (dim >> 6) * 1024 + tok * 64 + (dim & 63); }
// Offset of the word with a dim's tokens 2t, 2t + 1, 2t + 8, 2t + 9.
__device__ __forceinline__ int value_off(int d, int t, int dim) {
  return kPage * d + (dim >> 5) * 512 + ((dim & 7) * 4 + t) * 16 + ((dim >> 3) & 3) * 4;
}
// KIND: NBL_I8 or NBL_E4M3.
template <int KIND>
__host__ __device__ constexpr float code_max() {
  return KIND == NBL_I8 ? 127.0f : 448.0f;
}
// Magnitudes below this are stored as 0 with scale 0: the reciprocal of a smaller scale would not be finite.
constexpr float kTiny = 1e-30f;
// Non-finite inputs are stored as 0 (NaN) or saturated at this (and flagged): its scale and products stay finite.
constexpr float kHuge = 3e38f;

// The code (as a byte: int8 or e4m3) of a value already divided by its scale. The scale makes |x| <= code_max up to
// rounding; the clamp covers that rounding.
template <int KIND>
__device__ __forceinline__ uint32_t encode(float x) {
  if constexpr (KIND == NBL_I8) {
    return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x, -127.f), 127.f))) & 0xffu;
  } else {
    return static_cast<uint32_t>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
  }
}
template <int KIND>
__device__ __forceinline__ float decode(uint32_t code) {
  if constexpr (KIND == NBL_I8) {
    return static_cast<float>(static_cast<int8_t>(code & 0xffu));
  } else {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code & 0xffu), __NV_E4M3);
    return __half2float(__half(h));
  }
}
// Four codes (byte i of `codes`) as the word that is stored, and back.
template <int KIND>
__host__ __device__ constexpr uint32_t to_word(uint32_t codes) {
  if constexpr (KIND == NBL_I8) return codes ^ 0x80808080u;
  const uint32_t a = (codes & 0xffu) | ((codes & 0xff00u) << 8), b = ((codes >> 16) & 0xffu) | ((codes >> 8) & 0xff0000u);
  return ((a & 0x00800080u) << 8) | ((a & 0x007f007fu) << 7) | ((b & 0x00800080u) << 7) | (b & 0x007f007fu);
}
template <int KIND>
__host__ __device__ __forceinline__ uint32_t from_word(uint32_t w) {
  if constexpr (KIND == NBL_I8) return w ^ 0x80808080u;
  const uint32_t a = ((w >> 8) & 0x00800080u) | ((w >> 7) & 0x007f007fu);
  const uint32_t b = ((w >> 7) & 0x00800080u) | (w & 0x007f007fu);
  return (a & 0xffu) | ((a >> 8) & 0xff00u) | ((b & 0xffu) << 16) | ((b & 0xff0000u) << 8);
}
// A word as two fp16 pairs (codes 0, 1 and 2, 3), each the code divided by unit<KIND>(). Exact for both kinds. For I8 the
// byte becomes the low mantissa bits of 1024 (0x6400 | byte = 1024 + byte), from which 1024 + 128 is subtracted.
template <int KIND>
__host__ __device__ constexpr float unit() {
  return KIND == NBL_I8 ? 1.f : 256.f;
}
template <int KIND>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == NBL_I8) {
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    lo = w & 0xbf80bf80u;
    hi = ((w << 7) & 0x3f803f80u) | ((w << 1) & 0x80008000u);
  }
}

// Bulk copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) into shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(smem_dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// Quotient and remainder of 0 <= n < 2^31 by a call's constant, without a division (Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994): with 2^l >= d, the quotient is (n + floor(n m / 2^32)) >> l for
// m = floor(2^32 (2^l - d) / d) + 1.
struct Divisor {
  uint32_t d = 1, m = 1, l = 0;
  Divisor() = default;
  explicit Divisor(uint32_t by) : d(by) {
    while ((uint64_t(1) << l) < d) ++l;
    m = static_cast<uint32_t>((uint64_t(1) << 32) * ((uint64_t(1) << l) - d) / d + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), m) + static_cast<uint32_t>(n)) >> l);
  }
  __device__ __forceinline__ int split(int& n) const {  // n becomes the quotient; returns the remainder
    const int q = div(n), r = n - q * static_cast<int>(d);
    n = q;
    return r;
  }
};

// An element of a float type as fp32, and back (one rounding).
__device__ __forceinline__ float load_as(const void* p, int64_t i, int dtype) {
  if (dtype == NBL_F32) return static_cast<const float*>(p)[i];
  if (dtype == NBL_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_as(void* p, int64_t i, float v, int dtype) {
  if (dtype == NBL_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == NBL_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

}  // namespace kv8

inline bool is_kv8(int dtype) { return dtype == NBL_I8 || dtype == NBL_E4M3; }

// Launches (kv8_append.cu, kv8_attn.cu); all asynchronous on `st`.
// A sequence's stretch of tokens: item i has rows start[i] .. start[i] + len[i] of the packed activations, at
// positions pos0[i].. of page-table row i.
struct Kv8Items {
  const int32_t* start = nullptr;
  const int32_t* len = nullptr;
  const int32_t* pos0 = nullptr;
  const int32_t* page_table = nullptr;
  int32_t pt_stride = 0;
  int n_items = 0, max_len = 0;
  int64_t n_rows = 0;  // rows of the packed activations
};
// Whether an item of len > 0 tokens is inside the launch (max_len), the activations and its page-table row; one that is
// not is flagged and left out by every kernel.
__device__ __forceinline__ bool item_fits(const Kv8Items& it, int start, int len, int pos0) {
  return len <= it.max_len && pos0 >= 0 && start >= 0 && int64_t(start) + len <= it.n_rows &&
         int64_t(pos0) + len <= int64_t(it.pt_stride) * kv8::kPage;
}
struct Kv8Append {
  const void *q_in = nullptr, *k_in = nullptr, *v_in = nullptr;
  const float *bq = nullptr, *bk = nullptr, *bv = nullptr;
  void* q_out = nullptr;
  int in_dtype = 0, q_out_dtype = 0, n_heads = 0;
  bool neox = false;
  int rotary_dim = 0;
  const float2* tab = nullptr;  // (cos, sin) [tab_pos][rotary_dim / 2]
  int64_t tab_pos = 0;
};
// A new pool's codes and scales: all 0.
void launch_kv8_clear(cudaStream_t st, const nbl_kv* kv);
void launch_kv8_append(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, const Kv8Append& a, int* err);
void launch_kv8_read(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, void* k_out, void* v_out, int out_dtype,
                     int* err);
void launch_kv8_import(cudaStream_t st, const nbl_kv* kv, const int32_t* page_ids, int64_t n, const void* codes,
                       const float* scales, int* err);
void launch_kv8_export(cudaStream_t st, const nbl_kv* kv, const int32_t* page_ids, int64_t n, void* codes,
                       float* scales, int* err);
// tab[pos][i] = (cos, sin)(pos * freq[i]) * mul in double, rounded to float; freq: n_pairs doubles on the device.
void launch_rotary_table(cudaStream_t st, float2* tab, int64_t n_pos, const double* freq, int n_pairs, double mul);

struct Kv8AttnPlan {
  int grid = 1;              // CTAs
  int64_t tiles = 1;         // query tiles of the longest item
  int seg_cost = 0;          // what a unit costs besides its pages, in pages
};
// max_kv: longest key range. q_dtype decides the row tile (8 rows of fp32 queries, whose two fp16 terms fill the 16 rows
// of the instruction, or 16 rows of 16-bit queries).
Kv8AttnPlan plan_kv8_attn(const nbl_kv* kv, int n_items, int max_len, int n_heads, int max_kv, int q_dtype,
                          int num_sms);
// What any launch needs of scratch: arrival counters (0 between launches), then parts of units that span CTAs.
size_t kv8_attn_scratch(int num_sms);
// items.len == NULL: one fp32 query row per item at position pos0[i] - 1 (pos0 = sequence lengths, 0 = no keys).
void launch_kv8_attn(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, const void* q, int q_dtype, int n_heads,
                     void* out, int out_dtype, float* lse, const Kv8AttnPlan& plan, void* scratch, int* err);

// Whether the warp-level kernel takes query stretches of max_len tokens (else the tcgen05 one): its time grows with the rows
// (tokens x heads of a group) that share each key, the other's stays until they pass 128 tokens. Measured, warp-level against
// tcgen05, 8 items at 4000 keys, heads of 64: 32/4 heads 27 / 38 / 61 us for 8 / 16 / 32 tokens against 68 / 68 / 72, 8/8
// heads 41 for 64 tokens against 76. Heads of 128: one item at 16k, 32/8 heads, 45 / 52 / 75 for 8 / 16 / 32 against 54 / 54 /
// 59; 8 items at 4000, 8/8 heads, 77 for 64 against 49.
inline bool kv8_few_tokens(int head_dim, int group, int max_len) {
  return head_dim == 64 ? max_len <= 64 && int64_t(max_len) * group <= 288
                        : max_len <= 24 && int64_t(max_len) * group <= 72;
}
// kv8_prefill.cu: the same for many query tokens of 16-bit type (q and out 16-byte aligned) on the tensor cores. n_rows:
// rows of q; split keys leave partial results in scratch, as large as the items' rows can be.
struct Kv8PrefillPlan {
  int n_splits = 1, n_works = 0, grid = 1;
  int64_t part_rows = 0;  // rows that a part of the split keys has room for
  size_t scratch_bytes = 0;
};
Kv8PrefillPlan plan_kv8_prefill(const nbl_kv* kv, int n_items, int max_len, int64_t n_rows, int n_heads, int max_kv,
                                int num_sms);
void launch_kv8_prefill(cudaStream_t st, const nbl_kv* kv, const Kv8Items& items, const void* q, int q_dtype, int n_heads,
                        void* out, int out_dtype, const Kv8PrefillPlan& plan, void* scratch, int* err);

}  // namespace nbl
