// C ABI entry points of the 8-bit K/V pool (append, read, import, export) and of the page bookkeeping (copy, fork,
// release, extend, compact). Attention over an 8-bit pool goes through nbl_attn_decode / nbl_attn_prefill (api.cu).
#include <algorithm>
#include <cmath>
#include <new>
#include <string>

#include "kv8.cuh"
#include "kv_pages.h"

namespace {

template <class F>
int guarded(F&& f) {
  try {
    f();
    return NBL_OK;
  } catch (const nbl::Failure& e) {
    return nbl::record_error(e.status, e.what());
  } catch (const std::bad_alloc&) {
    return nbl::record_error(NBL_E_NOMEM, "host allocation failed");
  } catch (const std::exception& e) {
    return nbl::record_error(NBL_E_INVALID, e.what());
  }
}

void require(bool ok, const char* what, const char* msg) {
  if (!ok) nbl::fail(NBL_E_INVALID, std::string(what) + ": " + msg);
}

// The arrays of a call that has work: an empty one's pointer may be NULL.
template <class... P>
void require_arrays(const char* what, const P*... p) {
  require((... && (p != nullptr)), what, "NULL argument");
}

void use(nbl_ctx* ctx) {
  nbl::check_cuda(cudaSetDevice(ctx->device), "cudaSetDevice");
  nbl::route_flush_queries(ctx);
}

bool is_float(int32_t d) { return d == NBL_F32 || d == NBL_F16 || d == NBL_BF16; }

void require_pool(const nbl_ctx* ctx, const nbl_kv* kv, const char* what) {
  require(kv->ctx == ctx, what, "pool belongs to another context");
}
void require_kv8(const nbl_ctx* ctx, const nbl_kv* kv, const char* what) {
  require_pool(ctx, kv, what);
  require(nbl::is_kv8(kv->cfg.dtype), what, "takes an NBL_I8 or NBL_E4M3 pool");
}

nbl::Kv8Items items_of(const nbl_kv* kv, int64_t n_rows, const int32_t* start, const int32_t* len, const int32_t* pos0,
                       const int32_t* page_table, int32_t pt_stride, int32_t n_items, int32_t max_len,
                       const char* what) {
  require(n_rows >= 0 && n_items >= 0 && max_len >= 0 && pt_stride > 0, what, "negative size");
  require(int64_t(pt_stride) * kv->cfg.page_size <= INT32_MAX && max_len <= pt_stride * kv->cfg.page_size,
          what, "max_len exceeds pt_stride * page_size");
  nbl::Kv8Items it;
  it.start = start;
  it.len = len;
  it.pos0 = pos0;
  it.page_table = page_table;
  it.pt_stride = pt_stride;
  it.n_items = n_items;
  it.max_len = max_len;
  it.n_rows = n_rows;
  return it;
}

// The angle per position of each rotated pair, and the factor on cos and sin. base^(-2i/n) with n rotated elements,
// then, for a context `factor` times as long as the `original` one:
//   linear      every frequency / factor
//   ntk         the base * factor^(n / (n - 2)): the slowest pair is interpolated, the fastest kept
//   yarn        pairs that turn less than beta_slow times over the original context are interpolated, those that turn
//               more than beta_fast times kept, a linear ramp (over the pair index) between; cos and sin * attn_factor
//   wavelength  the same by the wavelength: longer than original / low_freq_factor interpolated, shorter than
//               original / high_freq_factor kept, blended between
void rotary_frequencies(const nbl_rotary_params& rp, int n, std::vector<double>& freq, double& mul) {
  const double pi = 3.14159265358979323846;
  double base = rp.freq_base;
  const double factor = rp.factor, original = rp.original_ctx;
  if (rp.scaling == NBL_ROTARY_NTK && n > 2) base *= std::pow(factor, double(n) / (n - 2));
  freq.resize(static_cast<size_t>(n / 2));
  for (int i = 0; i < n / 2; ++i) freq[i] = std::pow(base, -2.0 * i / n);
  mul = 1.0;
  if (rp.scaling == NBL_ROTARY_LINEAR) {
    for (double& f : freq) f /= factor;
  } else if (rp.scaling == NBL_ROTARY_YARN) {
    // the pair index at which a pair turns `beta` times over the original context
    auto turns = [&](double beta) { return n * std::log(original / (beta * 2 * pi)) / (2 * std::log(base)); };
    const double low = std::max(std::floor(turns(rp.beta_fast)), 0.0);
    const double high = std::min(std::ceil(turns(rp.beta_slow)), n - 1.0);
    for (int i = 0; i < n / 2; ++i) {
      const double ramp = std::min(std::max((i - low) / std::max(high - low, 0.001), 0.0), 1.0);
      freq[i] = freq[i] / factor * ramp + freq[i] * (1 - ramp);
    }
    mul = 0.1 * std::log(factor) + 1.0;
  } else if (rp.scaling == NBL_ROTARY_WAVELENGTH) {
    for (double& f : freq) {
      const double lo = rp.low_freq_factor, hi = rp.high_freq_factor;
      const double smooth = std::min(std::max((original / (2 * pi / f) - lo) / (hi - lo), 0.0), 1.0);
      f = (1 - smooth) * f / factor + smooth * f;
    }
  }
  if (rp.attn_factor != 0.f) mul = rp.attn_factor;
  if (rp.freq_factors)
    for (int i = 0; i < n / 2; ++i) freq[i] /= rp.freq_factors[i];
}

void check_rotary(const nbl_rotary_params& rp, int head_dim, const char* what) {
  require(std::isfinite(rp.freq_base) && rp.freq_base > 1.f, what, "freq_base must be greater than 1");
  require(rp.rotary_dim >= 0 && rp.rotary_dim <= head_dim && rp.rotary_dim % 2 == 0,
          what, "rotary_dim must be even and at most head_dim (0: all of it)");
  require(rp.scaling >= NBL_ROTARY_NONE && rp.scaling <= NBL_ROTARY_WAVELENGTH, what, "unknown scaling");
  require(std::isfinite(rp.attn_factor) && rp.attn_factor >= 0.f, what, "attn_factor must not be negative");
  if (rp.scaling != NBL_ROTARY_NONE)
    require(std::isfinite(rp.factor) && rp.factor >= 1.f, what, "the scaling factor must be at least 1");
  if (rp.scaling == NBL_ROTARY_YARN)
    require(rp.original_ctx > 0 && rp.beta_slow > 0.f && rp.beta_fast >= rp.beta_slow && std::isfinite(rp.beta_fast),
            what, "yarn needs original_ctx > 0 and beta_fast >= beta_slow > 0");
  if (rp.scaling == NBL_ROTARY_WAVELENGTH)
    require(rp.original_ctx > 0 && rp.low_freq_factor > 0.f && rp.high_freq_factor > rp.low_freq_factor &&
                std::isfinite(rp.high_freq_factor),
            what, "wavelength needs original_ctx > 0 and high_freq_factor > low_freq_factor > 0");
}

bool same_rotary(const nbl::RotaryTable& t, const nbl_rotary_params& rp, int n) {
  const nbl_rotary_params& o = t.params;
  if (t.n != n || o.freq_base != rp.freq_base || o.scaling != rp.scaling || o.attn_factor != rp.attn_factor) return false;
  if (rp.scaling != NBL_ROTARY_NONE && o.factor != rp.factor) return false;
  if (rp.scaling == NBL_ROTARY_YARN &&
      (o.original_ctx != rp.original_ctx || o.beta_fast != rp.beta_fast || o.beta_slow != rp.beta_slow))
    return false;
  if (rp.scaling == NBL_ROTARY_WAVELENGTH && (o.original_ctx != rp.original_ctx || o.low_freq_factor != rp.low_freq_factor ||
                                              o.high_freq_factor != rp.high_freq_factor))
    return false;
  if (!rp.freq_factors) return t.factors.empty();
  return t.factors.size() == static_cast<size_t>(n / 2) &&
         std::equal(t.factors.begin(), t.factors.end(), rp.freq_factors);
}

// The device cos/sin table of these parameters for positions [0, n_pos), made on first use. The context keeps the
// kRotaryTables used last (a caller may change the scaling factor with every call).
const nbl::RotaryTable& rotary_table(nbl_ctx* ctx, const nbl_rotary_params& rp, int n, int64_t n_pos) {
  ++ctx->rotary_uses;
  for (auto& t : ctx->rotary_tables)
    if (same_rotary(t, rp, n) && t.n_pos >= n_pos) {
      t.used = ctx->rotary_uses;
      return t;
    }
  nbl::RotaryTable t;
  t.used = ctx->rotary_uses;
  t.params = rp;
  t.params.freq_factors = nullptr;
  if (rp.freq_factors) t.factors.assign(rp.freq_factors, rp.freq_factors + n / 2);
  t.n = n;
  t.n_pos = std::max<int64_t>(n_pos, ctx->reserved_ctx);
  std::vector<double> freq;
  double mul = 1.0;
  rotary_frequencies(rp, n, freq, mul);
  auto* dev_freq = static_cast<double*>(nbl::device_alloc(freq.size() * sizeof(double), "rotary frequencies"));
  try {
    t.dev = static_cast<float2*>(nbl::device_alloc(static_cast<size_t>(t.n_pos) * freq.size() * sizeof(float2), "rotary table"));
    nbl::check_cuda(cudaMemcpyAsync(dev_freq, freq.data(), freq.size() * sizeof(double), cudaMemcpyHostToDevice, ctx->stream),
                    "rotary table");
    nbl::launch_rotary_table(ctx->stream, t.dev, t.n_pos, dev_freq, n / 2, mul);
    nbl::check_cuda(cudaStreamSynchronize(ctx->stream), "rotary table");
    ctx->rotary_tables.reserve(ctx->rotary_tables.size() + 1);
  } catch (...) {
    cudaFree(dev_freq);
    if (t.dev) cudaFree(t.dev);
    throw;
  }
  cudaFree(dev_freq);
  // A shorter table of the same parameters goes, or the one not used for longest (its readers are done: the stream is idle).
  auto& all = ctx->rotary_tables;
  auto gone = std::find_if(all.begin(), all.end(), [&](const auto& o) { return same_rotary(o, rp, n); });
  if (gone == all.end() && all.size() >= nbl::kRotaryTables)
    gone = std::min_element(all.begin(), all.end(), [](const auto& x, const auto& y) { return x.used < y.used; });
  if (gone != all.end()) {
    cudaFree(gone->dev);
    all.erase(gone);
  }
  ctx->rotary_tables.push_back(std::move(t));
  return ctx->rotary_tables.back();
}

nbl::PageBook book_of(const nbl_kv* kv, int32_t* table, int32_t pt_stride, int32_t n_rows, int32_t* lens, int32_t* refs,
                      const char* what) {
  require(pt_stride > 0 && n_rows >= 0, what, "negative size");
  require(int64_t(pt_stride) * kv->cfg.page_size <= INT32_MAX, what, "pt_stride too large");
  nbl::PageBook b;
  b.table = table;
  b.lens = lens;
  b.refs = refs;
  b.pt_stride = pt_stride;
  b.n_rows = n_rows;
  b.n_pages = kv->cfg.n_pages;
  return b;
}

}  // namespace

extern "C" {

int nbl_rotary_kv_append(nbl_ctx* ctx, nbl_kv* kv, const void* q_in, const void* k_in, const void* v_in,
                         int32_t in_dtype, const float* bq, const float* bk, const float* bv, void* q_out,
                         int32_t q_out_dtype, int64_t n_rows, const int32_t* q_start, const int32_t* q_len,
                         const int32_t* kv_pos0, const int32_t* page_table, int32_t pt_stride, int32_t n_items,
                         int32_t n_heads, int32_t max_q_len, const nbl_rotary_params* rotary) {
  return guarded([&] {
    const char* what = "rotary_kv_append";
    require(ctx && kv && rotary, what, "NULL argument");
    require_kv8(ctx, kv, what);
    require(is_float(in_dtype) && is_float(q_out_dtype), what, "bad dtype");
    require(n_heads > 0 && n_heads % kv->cfg.n_kv_heads == 0, what, "n_heads must be a multiple of n_kv_heads");
    const auto it = items_of(kv, n_rows, q_start, q_len, kv_pos0, page_table, pt_stride, n_items, max_q_len, what);
    check_rotary(*rotary, kv->cfg.head_dim, what);
    if (n_items == 0 || max_q_len == 0 || n_rows == 0) return;
    require_arrays(what, q_in, k_in, v_in, q_out, q_start, q_len, kv_pos0, page_table);
    use(ctx);
    nbl::Kv8Append a;
    a.q_in = q_in;
    a.k_in = k_in;
    a.v_in = v_in;
    a.bq = bq;
    a.bk = bk;
    a.bv = bv;
    a.q_out = q_out;
    a.in_dtype = in_dtype;
    a.q_out_dtype = q_out_dtype;
    a.n_heads = n_heads;
    a.neox = rotary->neox != 0;
    a.rotary_dim = rotary->rotary_dim ? rotary->rotary_dim : kv->cfg.head_dim;
    const auto& tab = rotary_table(ctx, *rotary, a.rotary_dim, int64_t(pt_stride) * kv->cfg.page_size);
    a.tab = tab.dev;
    a.tab_pos = tab.n_pos;
    nbl::launch_kv8_append(ctx->stream, kv, it, a, ctx->d_err);
  });
}

int nbl_kv_read(nbl_ctx* ctx, const nbl_kv* kv, int64_t n_rows, const int32_t* start, const int32_t* len,
                const int32_t* kv_pos0, const int32_t* page_table, int32_t pt_stride, int32_t n_items, int32_t max_len,
                void* k_out, void* v_out, int32_t out_dtype) {
  return guarded([&] {
    const char* what = "kv_read";
    require(ctx && kv, what, "NULL argument");
    require_kv8(ctx, kv, what);
    require(is_float(out_dtype), what, "bad dtype");
    const auto it = items_of(kv, n_rows, start, len, kv_pos0, page_table, pt_stride, n_items, max_len, what);
    if (n_items == 0 || max_len == 0 || n_rows == 0) return;
    require_arrays(what, start, len, kv_pos0, page_table, k_out ? k_out : v_out);
    use(ctx);
    nbl::launch_kv8_read(ctx->stream, kv, it, k_out, v_out, out_dtype, ctx->d_err);
  });
}

int nbl_kv_import(nbl_ctx* ctx, nbl_kv* kv, const int32_t* page_ids, int64_t n, const void* codes, const float* scales) {
  return guarded([&] {
    require(ctx && kv, "kv_import", "NULL argument");
    require_kv8(ctx, kv, "kv_import");
    require(n >= 0 && n <= INT32_MAX, "kv_import", "bad page count");
    if (n == 0) return;
    require_arrays("kv_import", page_ids, codes, scales);
    use(ctx);
    nbl::launch_kv8_import(ctx->stream, kv, page_ids, n, codes, scales, ctx->d_err);
  });
}

int nbl_kv_export(nbl_ctx* ctx, const nbl_kv* kv, const int32_t* page_ids, int64_t n, void* codes, float* scales) {
  return guarded([&] {
    require(ctx && kv, "kv_export", "NULL argument");
    require_kv8(ctx, kv, "kv_export");
    require(n >= 0 && n <= INT32_MAX, "kv_export", "bad page count");
    if (n == 0) return;
    require_arrays("kv_export", page_ids, codes, scales);
    use(ctx);
    nbl::launch_kv8_export(ctx->stream, kv, page_ids, n, codes, scales, ctx->d_err);
  });
}

int nbl_kv_copy_pages(nbl_ctx* ctx, nbl_kv* kv, const int32_t* src_pages, const int32_t* dst_pages, int32_t n) {
  return guarded([&] {
    require(ctx && kv, "kv_copy_pages", "NULL argument");
    require_pool(ctx, kv, "kv_copy_pages");
    require(n >= 0, "kv_copy_pages", "negative size");
    if (n == 0) return;
    require_arrays("kv_copy_pages", src_pages, dst_pages);
    use(ctx);
    nbl::launch_copy_pages(ctx->stream, kv, src_pages, dst_pages, n, ctx->d_err);
  });
}

int nbl_kv_fork(nbl_ctx* ctx, nbl_kv* kv, int32_t* page_table, int32_t pt_stride, int32_t n_rows, int32_t* seq_lens,
                int32_t* ref_counts, const int32_t* src_rows, const int32_t* dst_rows, int32_t n) {
  return guarded([&] {
    require(ctx && kv, "kv_fork", "NULL argument");
    require_pool(ctx, kv, "kv_fork");
    const auto b = book_of(kv, page_table, pt_stride, n_rows, seq_lens, ref_counts, "kv_fork");
    require(n >= 0 && n <= n_rows, "kv_fork", "n must be 0..n_rows");
    if (n == 0) return;
    require_arrays("kv_fork", page_table, seq_lens, ref_counts, src_rows, dst_rows);
    use(ctx);
    nbl::ensure_scratch(ctx, nbl::kv_book_scratch(n, kv->cfg.n_pages));
    nbl::launch_kv_fork(ctx->stream, kv, b, src_rows, dst_rows, n, ctx->scratch, nbl::split_counts(ctx, 1), ctx->d_err);
  });
}

int nbl_kv_release(nbl_ctx* ctx, nbl_kv* kv, int32_t* page_table, int32_t pt_stride, int32_t n_rows, int32_t* seq_lens,
                   int32_t* ref_counts, const int32_t* rows, int32_t n) {
  return guarded([&] {
    require(ctx && kv, "kv_release", "NULL argument");
    require_pool(ctx, kv, "kv_release");
    const auto b = book_of(kv, page_table, pt_stride, n_rows, seq_lens, ref_counts, "kv_release");
    require(n >= 0, "kv_release", "negative size");
    if (n == 0) return;
    require_arrays("kv_release", page_table, seq_lens, ref_counts, rows);
    use(ctx);
    nbl::launch_kv_release(ctx->stream, b, rows, n, ctx->d_err);
  });
}

int nbl_kv_extend(nbl_ctx* ctx, nbl_kv* kv, int32_t* page_table, int32_t pt_stride, int32_t n_rows, int32_t* seq_lens,
                  int32_t* ref_counts, const int32_t* rows, const int32_t* new_lens, int32_t n) {
  return guarded([&] {
    require(ctx && kv, "kv_extend", "NULL argument");
    require_pool(ctx, kv, "kv_extend");
    const auto b = book_of(kv, page_table, pt_stride, n_rows, seq_lens, ref_counts, "kv_extend");
    require(n >= 0 && n <= n_rows, "kv_extend", "n must be 0..n_rows");
    if (n == 0) return;
    require_arrays("kv_extend", page_table, seq_lens, ref_counts, rows, new_lens);
    use(ctx);
    nbl::ensure_scratch(ctx, nbl::kv_book_scratch(n, kv->cfg.n_pages));
    nbl::launch_kv_extend(ctx->stream, b, rows, new_lens, n, ctx->scratch, ctx->d_err);
  });
}

int nbl_kv_compact(nbl_ctx* ctx, const nbl_kv* src, nbl_kv* dst, const int32_t* page_table, int32_t pt_stride,
                   int32_t n_rows, const int32_t* seq_lens, int32_t* table_out, int32_t* ref_counts_out,
                   int32_t* n_used) {
  return guarded([&] {
    require(ctx && src && dst && ref_counts_out && n_used, "kv_compact", "NULL argument");
    require_pool(ctx, src, "kv_compact");
    require_pool(ctx, dst, "kv_compact");
    const auto &s = src->cfg, &d = dst->cfg;
    require(src != dst && s.dtype == d.dtype && s.head_dim == d.head_dim && s.n_kv_heads == d.n_kv_heads &&
                s.page_size == d.page_size,
            "kv_compact", "the pools must be two of the same dtype, head_dim, n_kv_heads and page_size");
    require(n_rows == 0 || page_table != table_out, "kv_compact", "table_out must not be page_table");
    const auto b = book_of(src, const_cast<int32_t*>(page_table), pt_stride, n_rows, const_cast<int32_t*>(seq_lens),
                           nullptr, "kv_compact");
    require(int64_t(n_rows) * pt_stride <= INT32_MAX, "kv_compact", "n_rows * pt_stride exceeds 2^31");
    use(ctx);
    if (n_rows == 0) {
      nbl::check_cuda(cudaMemsetAsync(n_used, 0, sizeof(int32_t), ctx->stream), "kv_compact");
      nbl::check_cuda(cudaMemsetAsync(ref_counts_out, 0, size_t(d.n_pages) * sizeof(int32_t), ctx->stream), "kv_compact");
      return;
    }
    require_arrays("kv_compact", page_table, seq_lens, table_out);
    nbl::ensure_scratch(ctx, nbl::kv_compact_scratch(n_rows, s.n_pages));
    nbl::launch_kv_compact(ctx->stream, src, dst, b, table_out, ref_counts_out, n_used, ctx->scratch, ctx->d_err,
                           ctx->num_sms);
  });
}

}  // extern "C"
