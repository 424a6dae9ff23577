// Page bookkeeping of the paged K/V pools on the device (kv_pages.cu), shared with the entry points.
#pragma once

#include "nbl_internal.h"

namespace nbl {

// Page tables [n_rows][pt_stride] of page ids (-1: none), lengths in tokens, and the number of table entries that
// name each page (0: free). All device memory, owned by the caller.
struct PageBook {
  int32_t* table = nullptr;
  int32_t* lens = nullptr;
  int32_t* refs = nullptr;
  int32_t pt_stride = 0;
  int32_t n_rows = 0;
  int64_t n_pages = 0;
};

int64_t kv_page_bytes(const nbl_kv* kv);
void launch_copy_pages(cudaStream_t st, const nbl_kv* kv, const int32_t* src, const int32_t* dst, int n, int* err);
// scratch: at least kv_book_scratch(n, n_pages) bytes; count: one arrival counter, 0 between launches.
size_t kv_book_scratch(int n, int64_t n_pages);
void launch_kv_fork(cudaStream_t st, const nbl_kv* kv, const PageBook& b, const int32_t* src_rows,
                    const int32_t* dst_rows, int n, void* scratch, unsigned* count, int* err);
void launch_kv_release(cudaStream_t st, const PageBook& b, const int32_t* rows, int n, int* err);
void launch_kv_extend(cudaStream_t st, const PageBook& b, const int32_t* rows, const int32_t* new_lens, int n,
                      void* scratch, int* err);
size_t kv_compact_scratch(int n_rows, int64_t n_pages);
void launch_kv_compact(cudaStream_t st, const nbl_kv* src, const nbl_kv* dst, const PageBook& b, int32_t* table_out,
                       int32_t* refs_out, int32_t* n_used, void* scratch, int* err, int num_sms);

}  // namespace nbl
