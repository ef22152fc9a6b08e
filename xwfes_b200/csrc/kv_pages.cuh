// kv_pages.cuh -- what the paged-cache kernels share: the device view of a
// cache and of a batch, and the host checks of both.
#pragma once

#include "common.cuh"

namespace ftc {

// Device view of ftc_kv_pages and ftc_page_batch (passed by value).
struct PageView {
    const int32_t* start;
    const int32_t* kv_len;
    const int32_t* table;
    int64_t table_stride;
    int table_cols;
    int n_seqs;
    int n_tokens;
    int n_pages;
    int page_size;   // a power of two
    int page_shift;
    int n_kv;
    int64_t page_stride;
    int64_t scale_stride;
};

// Row range of sequence s, kept inside the buffers whatever the device
// arrays hold.
__device__ __forceinline__ void seq_rows(const PageView& b, int s, int& r0, int& n) {
    r0 = min(max(b.start[s], 0), b.n_tokens);
    n = max(min(b.start[s + 1], b.n_tokens) - r0, 0);
}

// Positions in the cache after the call's rows.
__device__ __forceinline__ int seq_len(const PageView& b, int s) { return max(b.kv_len[s], 0); }

// Page of position pos of sequence s, or -1 when it is not mapped.
__device__ __forceinline__ int page_of(const PageView& b, int s, int pos) {
    if (pos < 0) return -1;
    const int c = pos >> b.page_shift;
    if (c >= b.table_cols) return -1;
    const int p = b.table[(int64_t)s * b.table_stride + c];
    return p >= 0 && p < b.n_pages ? p : -1;
}

// Checks of both structs (host); fills the view.
int page_view(const ftc_kv_pages* c, const ftc_page_batch* b, const char* who, PageView* out);

}  // namespace ftc
