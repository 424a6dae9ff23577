// Page bookkeeping of the paged K/V pools on the device: copy, fork, release, extend and compact, for pools of every
// dtype (a page is opaque bytes here).
//
// A page belongs to as many table entries as name it; refs[page] is that number and a page with 0 is free. A forked
// row shares its source's full pages (they are never written again) and gets its own copy of the part-filled last one,
// so a shared page is never appended to. Free pages are handed out lowest id first, in the order of the request list,
// whatever order the CTAs run in: counts are integer atomics, and one CTA hands out the pages in order.
//
// Bound: latency for fork, release and extend (24 forks of rows of 130..2100 tokens: 13 us, 12 of them the call's time on the
// host); memory for compact (14k shared pages of 8 heads of 64, 458 MB read and written: 88 us, of which the move takes 67,
// 6.8 TB/s, and numbering the pages 21 in a clear and three short launches).
#include <algorithm>

#include "kv8.cuh"
#include "kv_pages.h"

namespace nbl {
namespace {

constexpr int kPage = 16;
constexpr int kThreads = 256;

__device__ __forceinline__ bool page_ok(const PageBook& b, int32_t e) { return e >= 0 && e < b.n_pages; }

// Drops every page that row's table names and empties the row (each entry is taken exactly once, so a row that two
// CTAs release at the same time is released once).
__device__ __forceinline__ void release_row(const PageBook& b, int32_t row, int* err) {
  int32_t* tr = b.table + int64_t(row) * b.pt_stride;
  for (int j = threadIdx.x; j < b.pt_stride; j += blockDim.x) {
    if (tr[j] == -1) continue;
    const int32_t e = atomicExch(&tr[j], -1);
    if (e == -1) continue;
    if (!page_ok(b, e)) {
      flag_error(err, kErrPageId);
    } else if (atomicSub(&b.refs[e], 1) <= 0) {  // nobody held it: leave the count at 0
      atomicAdd(&b.refs[e], 1);
      flag_error(err, kErrPageId);
    }
  }
}

// Sum over the block's threads of the values before this one (exclusive), and the total; every thread calls it.
template <class T>
__device__ __forceinline__ T block_scan(T v, T& total) {
  __shared__ T part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  T inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();  // part may still be read by an earlier call
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  T before = 0;
  total = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += part[w];
    total += part[w];
  }
  return before + inc - v;
}

// Collects the lowest `want` free page ids in order into list; returns how many there are (at most want). One CTA.
// Pages are read four per thread and step, each thread's four adjacent, so ids come out in order.
__device__ int collect_free(const PageBook& b, int want, int32_t* list) {
  int found = 0;
  for (int64_t p0 = 0; p0 < b.n_pages && found < want; p0 += int64_t(blockDim.x) * 4) {
    const int64_t p = p0 + threadIdx.x * 4;
    bool free4[4];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      free4[k] = p + k < b.n_pages && __ldcg(b.refs + p + k) == 0;
      mine += free4[k];
    }
    int total;
    int at = found + block_scan(mine, total);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (free4[k]) {
        if (at < want) list[at] = static_cast<int32_t>(p + k);
        ++at;
      }
    found = min(found + total, want);
  }
  __syncthreads();
  return found;
}

// What a fork of list position i wants: where its part-filled page goes (page < 0: nothing to copy).
struct ForkCopy {
  int32_t row, slot, src_page;
};

// CTA i: fork i. The last CTA to finish hands out the pages for the part-filled ones.
__global__ void __launch_bounds__(kThreads) kv_fork_kernel(const PageBook b, const int32_t* __restrict__ src_rows,
                                                           const int32_t* __restrict__ dst_rows, int n, ForkCopy* want,
                                                           int32_t* list, unsigned* count, int* err) {
  const int i = blockIdx.x;
  const int32_t src = src_rows[i], dst = dst_rows[i];
  bool bad = src < 0 || src >= b.n_rows || dst < 0 || dst >= b.n_rows || src == dst;
  for (int j = threadIdx.x; j < n; j += kThreads) bad = bad || src_rows[j] == dst || (j < i && dst_rows[j] == dst);
  bad = __syncthreads_or(bad);
  if (bad) {
    if (threadIdx.x == 0) {
      flag_error(err, kErrRow);
      want[i].src_page = -1;
    }
  } else {
    release_row(b, dst, err);
    __syncthreads();
    int len = b.lens[src];
    if (len < 0 || int64_t(len) > int64_t(b.pt_stride) * kPage) {
      if (threadIdx.x == 0) flag_error(err, kErrLength);
      len = 0;
    }
    const int full = len / kPage;
    const int32_t* ts = b.table + int64_t(src) * b.pt_stride;
    int32_t* td = b.table + int64_t(dst) * b.pt_stride;
    for (int j = threadIdx.x; j < full; j += kThreads) {
      const int32_t e = ts[j];
      if (page_ok(b, e)) {
        atomicAdd(&b.refs[e], 1);
        td[j] = e;
      } else {
        flag_error(err, kErrPageId);
      }
    }
    if (threadIdx.x == 0) {
      b.lens[dst] = len;
      ForkCopy w{dst, full, -1};
      if (len % kPage) {
        if (page_ok(b, ts[full])) w.src_page = ts[full];
        else flag_error(err, kErrPageId);
      }
      want[i] = w;
    }
  }
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicInc(count, static_cast<unsigned>(n - 1)) == static_cast<unsigned>(n - 1);
  __syncthreads();
  if (!last) return;
  __threadfence();
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int k = i0 + threadIdx.x;
    int add;
    block_scan<int>(k < n && __ldcg(&want[k].src_page) >= 0, add);
    total += add;
  }
  const int found = collect_free(b, total, list);
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int k = i0 + threadIdx.x;
    const bool wants = k < n && __ldcg(&want[k].src_page) >= 0;
    int add;
    const int at = before + block_scan<int>(wants, add);
    if (wants) {
      const int32_t row = __ldcg(&want[k].row), slot = __ldcg(&want[k].slot);
      if (at < found) {
        const int32_t page = list[at];
        b.table[int64_t(row) * b.pt_stride + slot] = page;
        b.refs[page] = 1;
      } else {  // no page left: the row keeps its full pages
        flag_error(err, kErrNoPage);
        b.lens[row] = slot * kPage;
        want[k].src_page = -1;
      }
    }
    before += add;
  }
}

// CTAs (i, piece): a piece of fork i's part-filled page.
__global__ void __launch_bounds__(kThreads) kv_fork_copy_kernel(const PageBook b, const ForkCopy* __restrict__ want,
                                                                uint8_t* pool, int64_t page_bytes) {
  const ForkCopy w = want[blockIdx.x];
  if (w.src_page < 0) return;
  const int32_t page = b.table[int64_t(w.row) * b.pt_stride + w.slot];
  const uint4* s = reinterpret_cast<const uint4*>(pool + w.src_page * page_bytes);
  uint4* d = reinterpret_cast<uint4*>(pool + page * page_bytes);
  for (int64_t u = blockIdx.y * int64_t(kThreads) + threadIdx.x; u < page_bytes / 16; u += int64_t(gridDim.y) * kThreads)
    d[u] = s[u];
}

__global__ void __launch_bounds__(kThreads) kv_copy_pages_kernel(uint8_t* pool, int64_t page_bytes, int64_t n_pages,
                                                                 const int32_t* __restrict__ src,
                                                                 const int32_t* __restrict__ dst, int* err) {
  const int32_t a = src[blockIdx.x], c = dst[blockIdx.x];
  if (a < 0 || a >= n_pages || c < 0 || c >= n_pages) {
    if (threadIdx.x == 0) flag_error(err, kErrPageId);
    return;
  }
  const uint4* s = reinterpret_cast<const uint4*>(pool + a * page_bytes);
  uint4* d = reinterpret_cast<uint4*>(pool + c * page_bytes);
  for (int64_t u = blockIdx.y * int64_t(kThreads) + threadIdx.x; u < page_bytes / 16; u += int64_t(gridDim.y) * kThreads)
    d[u] = s[u];
}

__global__ void __launch_bounds__(kThreads) kv_release_kernel(const PageBook b, const int32_t* __restrict__ rows,
                                                              int* err) {
  const int32_t row = rows[blockIdx.x];
  if (row < 0 || row >= b.n_rows) {
    if (threadIdx.x == 0) flag_error(err, kErrRow);
    return;
  }
  release_row(b, row, err);
  if (threadIdx.x == 0) b.lens[row] = 0;
}

// One CTA: row rows[i] grows to new_lens[i] tokens. All rows get their pages, or (too few free ones) none do.
constexpr int kExtendThreads = 1024;
__global__ void __launch_bounds__(kExtendThreads) kv_extend_kernel(const PageBook b, const int32_t* __restrict__ rows,
                                                                   const int32_t* __restrict__ new_lens, int n,
                                                                   int64_t* before, int32_t* list, int* err) {
  // before[i]: pages wanted by the list's rows before i
  __shared__ int64_t total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += kExtendThreads) {
    const int i = i0 + threadIdx.x;
    int64_t need = 0;  // (the rows of one step may want more than 2^31 together)
    if (i < n) {
      const int32_t row = rows[i], to = new_lens[i];
      bool ok = row >= 0 && row < b.n_rows;
      for (int j = 0; ok && j < i; ++j) ok = rows[j] != row;
      if (!ok) flag_error(err, kErrRow);
      if (ok) {
        const int32_t len = b.lens[row];
        if (len < 0 || to < len || int64_t(to) > int64_t(b.pt_stride) * kPage) flag_error(err, kErrLength);
        else need = (to + kPage - 1) / kPage - (len + kPage - 1) / kPage;
      }
    }
    int64_t add;
    const int64_t at = block_scan(need, add);
    if (i < n) before[i] = total + at;
    __syncthreads();
    if (threadIdx.x == 0) total += add;
    __syncthreads();
  }
  if (total > b.n_pages) {
    if (threadIdx.x == 0) flag_error(err, kErrNoPage);
    return;
  }
  const int want = static_cast<int>(total);
  const int found = collect_free(b, want, list);
  if (found < want) {
    if (threadIdx.x == 0) flag_error(err, kErrNoPage);
    return;
  }
  for (int k = threadIdx.x; k < want; k += kExtendThreads) {
    int lo = 0, hi = n - 1;  // the last i with before[i] <= k holds page k
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (before[mid] <= k) lo = mid;
      else hi = mid - 1;
    }
    const int32_t row = rows[lo];
    const int slot = (b.lens[row] + kPage - 1) / kPage + static_cast<int>(k - before[lo]);
    b.table[int64_t(row) * b.pt_stride + slot] = list[k];
    b.refs[list[k]] = 1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kExtendThreads) {
    const int32_t row = rows[i], to = new_lens[i];
    if (row < 0 || row >= b.n_rows) continue;
    bool ok = b.lens[row] >= 0 && to >= b.lens[row] && int64_t(to) <= int64_t(b.pt_stride) * kPage;
    for (int j = 0; ok && j < i; ++j) ok = rows[j] != row;
    if (ok) b.lens[row] = to;
  }
}

// ---- compact: a page's new id is its rank by first appearance in the tables (row by row): the first entry that names each
// page (an integer minimum), the firsts of each row, their ranks, then the move. Latency bound up to the move, so each kernel
// is launched while the one before still runs (all of whose CTAs have started then) and waits for its end before it reads
// anything (128 rows, 458 MB moved: 96 -> 88 us). What an earlier kernel of the chain writes comes through plain pointers and
// is read with __ldcg: a const __restrict__ one would promise that it does not change while the kernel lives, and let the
// compiler read it before the wait.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ int held_pages(const PageBook& b, int row, int* err) {
  const int len = b.lens[row];
  if (len < 0 || int64_t(len) > int64_t(b.pt_stride) * kPage) {
    if (threadIdx.x == 0) flag_error(err, kErrLength);
    return 0;
  }
  return (len + kPage - 1) / kPage;
}

__global__ void __launch_bounds__(kThreads) compact_first_kernel(const PageBook b, unsigned* first, int* err) {
  next_may_start();
  const int row = blockIdx.x, held = held_pages(b, row, err);
  for (int j = threadIdx.x; j < held; j += kThreads) {
    const int64_t at = int64_t(row) * b.pt_stride + j;
    const int32_t e = b.table[at];
    if (page_ok(b, e)) atomicMin(&first[e], static_cast<unsigned>(at));
    else flag_error(err, kErrPageId);
  }
}

__global__ void __launch_bounds__(kThreads) compact_count_kernel(const PageBook b, const unsigned* first,
                                                                 int32_t* counts, int32_t* refs_out, int64_t n_dst) {
  next_may_start();
  wait_for_previous();
  const int row = blockIdx.x, held = held_pages(b, row, nullptr);
  for (int64_t i = int64_t(row) * kThreads + threadIdx.x; i < n_dst; i += int64_t(gridDim.x) * kThreads) refs_out[i] = 0;
  int mine = 0;
  for (int j = threadIdx.x; j < held; j += kThreads) {
    const int64_t at = int64_t(row) * b.pt_stride + j;
    const int32_t e = b.table[at];
    mine += page_ok(b, e) && __ldcg(&first[e]) == static_cast<unsigned>(at);
  }
  int total;
  block_scan(mine, total);
  if (threadIdx.x == 0) counts[row] = total;
}

__global__ void __launch_bounds__(kThreads) compact_rank_kernel(const PageBook b, const unsigned* first,
                                                                const int32_t* counts, int32_t* new_id,
                                                                int32_t* source, int32_t* n_used, int64_t n_dst,
                                                                int* err) {
  next_may_start();
  wait_for_previous();
  const int row = blockIdx.x, held = held_pages(b, row, nullptr);
  int sum = 0, all = 0;
  for (int r = threadIdx.x; r < b.n_rows; r += kThreads) {
    const int c = __ldcg(&counts[r]);
    all += c;
    if (r < row) sum += c;
  }
  int before, total;
  block_scan(sum, before);
  block_scan(all, total);
  if (row == 0 && threadIdx.x == 0) {
    *n_used = total;
    if (total > n_dst) flag_error(err, kErrNoPage);
  }
  for (int j0 = 0; j0 < held; j0 += kThreads) {
    const int j = j0 + threadIdx.x;
    const int64_t at = int64_t(row) * b.pt_stride + j;
    const int32_t e = j < held ? b.table[at] : -1;
    const bool lead = page_ok(b, e) && __ldcg(&first[e]) == static_cast<unsigned>(at);
    int add;
    const int id = before + block_scan<int>(lead, add);
    if (lead) {
      new_id[e] = id;
      source[id] = e;
    }
    before += add;
  }
}

// CTAs 0 .. n_rows - 1 also rewrite one table row each; all of them copy pages.
__global__ void __launch_bounds__(kThreads) compact_move_kernel(const PageBook b, const int32_t* new_id,
                                                                const int32_t* source, const int32_t* n_used, int64_t n_dst,
                                                                int32_t* table_out, int32_t* refs_out,
                                                                const uint8_t* __restrict__ from, uint8_t* __restrict__ to,
                                                                int64_t page_bytes) {
  wait_for_previous();
  for (int row = blockIdx.x; row < b.n_rows; row += gridDim.x) {
    const int held = held_pages(b, row, nullptr);
    for (int j = threadIdx.x; j < b.pt_stride; j += kThreads) {
      const int64_t at = int64_t(row) * b.pt_stride + j;
      const int32_t e = j < held ? b.table[at] : -1;
      int32_t id = page_ok(b, e) ? __ldcg(&new_id[e]) : -1;
      if (id >= n_dst) id = -1;
      if (id >= 0) atomicAdd(&refs_out[id], 1);
      table_out[at] = id;
    }
  }
  const int used = static_cast<int>(min(int64_t(__ldcg(n_used)), n_dst));
  for (int p = blockIdx.x; p < used; p += gridDim.x) {
    const uint4* s = reinterpret_cast<const uint4*>(from + __ldcg(&source[p]) * page_bytes);
    uint4* d = reinterpret_cast<uint4*>(to + p * page_bytes);
    for (int64_t u = threadIdx.x; u < page_bytes / 16; u += kThreads) d[u] = s[u];
  }
}

template <class... Params, class... Args>
void launch_after(cudaStream_t st, void (*kernel)(Params...), unsigned grid, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...), "kv_compact launch");
}

unsigned copy_pieces(int64_t page_bytes) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(page_bytes / (kThreads * 16), 64)));
}

}  // namespace

int64_t kv_page_bytes(const nbl_kv* kv) { return static_cast<int64_t>(kv->bytes / static_cast<size_t>(kv->cfg.n_pages)); }

void launch_copy_pages(cudaStream_t st, const nbl_kv* kv, const int32_t* src, const int32_t* dst, int n, int* err) {
  const int64_t pb = kv_page_bytes(kv);
  kv_copy_pages_kernel<<<dim3(static_cast<unsigned>(n), copy_pieces(pb)), kThreads, 0, st>>>(
      static_cast<uint8_t*>(kv->pool), pb, kv->cfg.n_pages, src, dst, err);
  check_cuda(cudaGetLastError(), "kv_copy_pages launch");
}

size_t kv_book_scratch(int n, int64_t n_pages) {
  return size_t(n) * sizeof(ForkCopy) + 16 + size_t(n) * sizeof(int64_t) + size_t(n_pages) * sizeof(int32_t);
}

void launch_kv_fork(cudaStream_t st, const nbl_kv* kv, const PageBook& b, const int32_t* src_rows,
                    const int32_t* dst_rows, int n, void* scratch, unsigned* count, int* err) {
  auto* list = static_cast<int32_t*>(scratch);
  auto* want = reinterpret_cast<ForkCopy*>(list + b.n_pages);
  kv_fork_kernel<<<n, kThreads, 0, st>>>(b, src_rows, dst_rows, n, want, list, count, err);
  check_cuda(cudaGetLastError(), "kv_fork launch");
  const int64_t pb = kv_page_bytes(kv);
  kv_fork_copy_kernel<<<dim3(static_cast<unsigned>(n), copy_pieces(pb)), kThreads, 0, st>>>(
      b, want, static_cast<uint8_t*>(kv->pool), pb);
  check_cuda(cudaGetLastError(), "kv_fork copy launch");
}

void launch_kv_release(cudaStream_t st, const PageBook& b, const int32_t* rows, int n, int* err) {
  kv_release_kernel<<<n, kThreads, 0, st>>>(b, rows, err);
  check_cuda(cudaGetLastError(), "kv_release launch");
}

void launch_kv_extend(cudaStream_t st, const PageBook& b, const int32_t* rows, const int32_t* new_lens, int n,
                      void* scratch, int* err) {
  auto* before = static_cast<int64_t*>(scratch);
  auto* list = reinterpret_cast<int32_t*>(before + n);
  kv_extend_kernel<<<1, kExtendThreads, 0, st>>>(b, rows, new_lens, n, before, list, err);
  check_cuda(cudaGetLastError(), "kv_extend launch");
}

size_t kv_compact_scratch(int n_rows, int64_t n_pages) {
  return (size_t(n_rows) + 3 * size_t(n_pages)) * sizeof(int32_t);
}

void launch_kv_compact(cudaStream_t st, const nbl_kv* src, const nbl_kv* dst, const PageBook& b, int32_t* table_out,
                       int32_t* refs_out, int32_t* n_used, void* scratch, int* err, int num_sms) {
  auto* first = static_cast<unsigned*>(scratch);
  auto* new_id = reinterpret_cast<int32_t*>(first + b.n_pages);
  int32_t* source = new_id + b.n_pages;
  int32_t* counts = source + b.n_pages;
  const int64_t n_dst = dst->cfg.n_pages;
  check_cuda(cudaMemsetAsync(first, 0xff, size_t(b.n_pages) * sizeof(unsigned), st), "kv_compact");
  const unsigned rows = static_cast<unsigned>(b.n_rows);
  compact_first_kernel<<<rows, kThreads, 0, st>>>(b, first, err);
  check_cuda(cudaGetLastError(), "kv_compact launch");
  launch_after(st, compact_count_kernel, rows, b, first, counts, refs_out, n_dst);
  launch_after(st, compact_rank_kernel, rows, b, first, counts, new_id, source, n_used, n_dst, err);
  launch_after(st, compact_move_kernel, static_cast<unsigned>(num_sms) * 8, b, new_id, source, n_used, n_dst, table_out, refs_out,
               static_cast<const uint8_t*>(src->pool), static_cast<uint8_t*>(dst->pool), kv_page_bytes(src));
}

}  // namespace nbl
