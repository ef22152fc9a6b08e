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

// Two floats in a 64-bit register, for the packed instructions.
__device__ __forceinline__ uint64_t f2(float a, float b) {
    return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
__device__ __forceinline__ float f2lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float f2hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t f2add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t f2mul(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t f2fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// Checks of both structs (host); fills the view.
int page_view(const ftc_kv_pages* c, const ftc_page_batch* b, const char* who, PageView* out);

}  // namespace ftc
