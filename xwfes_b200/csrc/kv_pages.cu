// kv_pages.cu -- the paged KV cache: storing new K and V rows (rounded to 16
// bits, or quantised to 8 with one scale per position and KV head) and
// reading rows back.
//
// Both move every byte once and are bound by HBM, or for a decode step by
// the launch: a thread takes 8 consecutive values of a row of K and the same
// 8 of V (two 16-byte loads of fp32 each, both tensors' loads in flight
// together), so a row of head_dim values is head_dim / 8 neighbouring lanes
// and its maximum is a shuffle reduction inside a warp.
#include <cuda_bf16.h>

#include <climits>

#include "kv_pages.cuh"

namespace ftc {

int page_view(const ftc_kv_pages* c, const ftc_page_batch* b, const char* who, PageView* out) {
    const std::string w(who);
    FTC_REQUIRE(c && b, FTC_E_INVALID, w + ": null pointer");
    FTC_REQUIRE(c->dtype == FTC_F16 || c->dtype == FTC_BF16 || c->dtype == FTC_KV_Q8,
                FTC_E_UNSUPPORTED, w + ": cache dtype must be F16, BF16 or KV_Q8");
    FTC_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, FTC_E_UNSUPPORTED,
                w + ": head_dim must be 64, 128 or 256");
    FTC_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 ||
                    c->page_size == 128 || c->page_size == 256,
                FTC_E_UNSUPPORTED, w + ": page_size must be 16, 32, 64, 128 or 256");
    FTC_REQUIRE(c->n_head_kv >= 1 && c->n_head_kv <= 1024, FTC_E_INVALID,
                w + ": n_head_kv must be 1..1024");
    FTC_REQUIRE(c->n_pages >= 1 && c->n_pages <= INT_MAX, FTC_E_INVALID,
                w + ": n_pages must be positive and fit 32 bits");
    const bool q8 = c->dtype == FTC_KV_Q8;
    const int64_t page_elems = c->n_head_kv * c->page_size * c->head_dim;
    FTC_REQUIRE(c->page_stride >= page_elems && c->page_stride * (q8 ? 1 : 2) % 16 == 0 &&
                    c->page_stride <= ((int64_t)1 << 36),
                FTC_E_INVALID,
                w + ": page_stride must cover a page and be a multiple of 16 bytes");
    FTC_REQUIRE(c->k && c->v, FTC_E_INVALID, w + ": null pointer");
    auto a16 = [](const void* p) { return (uintptr_t)p % 16 == 0; };
    FTC_REQUIRE(a16(c->k) && a16(c->v), FTC_E_INVALID, w + ": buffers must be 16-byte aligned");
    if (q8) {
        FTC_REQUIRE(c->k_scale && c->v_scale, FTC_E_INVALID, w + ": null pointer");
        FTC_REQUIRE(a16(c->k_scale) && a16(c->v_scale), FTC_E_INVALID,
                    w + ": buffers must be 16-byte aligned");
        FTC_REQUIRE(c->scale_stride >= c->n_head_kv * c->page_size && c->scale_stride % 4 == 0 &&
                        c->scale_stride <= ((int64_t)1 << 36),
                    FTC_E_INVALID, w + ": scale_stride must cover a page and be a multiple of 4");
    }
    FTC_REQUIRE(b->n_seqs >= 0 && b->n_tokens >= 0 && b->max_new >= 0, FTC_E_INVALID,
                w + ": negative batch size");
    FTC_REQUIRE(b->n_seqs <= 2048, FTC_E_UNSUPPORTED, w + ": at most 2048 sequences a call");
    FTC_REQUIRE(b->n_tokens <= (1 << 24), FTC_E_UNSUPPORTED, w + ": at most 2^24 rows a call");
    if (b->n_seqs > 0 && b->n_tokens > 0) {
        FTC_REQUIRE(b->start && b->kv_len && b->page_table, FTC_E_INVALID, w + ": null pointer");
        FTC_REQUIRE(b->table_cols >= 1 && b->table_stride >= b->table_cols &&
                        b->table_cols * c->page_size <= INT_MAX - 1024,
                    FTC_E_INVALID, w + ": table_cols must be positive, within table_stride, and "
                                       "the positions fit 31 bits");
    }
    out->start = b->start;
    out->kv_len = b->kv_len;
    out->table = b->page_table;
    out->table_stride = b->table_stride;
    out->table_cols = (int)b->table_cols;
    out->n_seqs = (int)b->n_seqs;
    out->n_tokens = (int)b->n_tokens;
    out->n_pages = (int)c->n_pages;
    out->page_size = (int)c->page_size;
    out->page_shift = __builtin_ctz((unsigned)c->page_size);
    out->n_kv = (int)c->n_head_kv;
    out->page_stride = c->page_stride;
    out->scale_stride = c->scale_stride;
    return FTC_OK;
}

namespace {

constexpr int kRowThreads = 256;

// 8 values in fp32 from / to a row of T
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0];
        const float4 b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                x[2 * i] = h2f(w[i]);
                x[2 * i + 1] = h2f(w[i] >> 16);
            } else {
                x[2 * i] = bf2f(w[i]);
                x[2 * i + 1] = bf2f(w[i] >> 16);
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]),
                                                  pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
}

// The cache slot of this thread's row: CTA rows start at token t0.  The
// CTA's first sequence is the number of sequences that end at or before t0
// (one round of loads over all threads); a later row walks on from there.
struct Slot {
    int page;  // -1: not mapped
    int slot;
    bool live;  // false: padding
};

__device__ __forceinline__ Slot find_slot(const PageView& b, int t0, int t) {
    int before = 0;
    for (int i0 = 0; i0 < b.n_seqs; i0 += kRowThreads) {
        const int i = i0 + (int)threadIdx.x;
        before += __syncthreads_count(i < b.n_seqs && b.start[i + 1] <= t0);
    }
    Slot r = {-1, 0, false};
    if (t >= b.n_tokens) return r;
    int s = before;
    while (s < b.n_seqs && b.start[s + 1] <= t) ++s;
    if (s >= b.n_seqs) return r;
    int r0, n;
    seq_rows(b, s, r0, n);
    if (t < r0 || t >= r0 + n) return r;
    const int pos = seq_len(b, s) - n + (t - r0);
    r.live = true;
    r.page = page_of(b, s, pos);
    r.slot = pos & (b.page_size - 1);
    return r;
}

// Row of 8-bit codes: d = max|x| / 127 and the codes of this thread's 8
// values.  |x| is compared as integer bits, so a NaN wins over an infinity
// and both over every finite value.  The code is the exactly rounded
// quotient: c = rint(x * (1 / d)) is within one of it, and the residual
// r = x - c d (one fused multiply-add, exact here: c d has at most 32 bits
// and cancels to within d) says which side of the half it is on, so no
// division per value.  Tiny d are scaled by 2^64 first to keep 1 / d finite.
template <int LANES>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float& d) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top >= 0x7F800000u) {
        d = __uint_as_float(0x7FC00000u);
        return make_uint2(0, 0);
    }
    d = __fdiv_rn(__uint_as_float(top), 127.f);
    if (d == 0.f) return make_uint2(0, 0);
    const float up = d < 1e-30f ? 18446744073709551616.f : 1.f;
    const float ds = d * up, inv = __frcp_rn(ds);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float xs = x[i] * up;
        float c = rintf(xs * inv);
        const float r2 = 2.f * fmaf(-c, ds, xs);
        const bool odd = ((int)c & 1) != 0;
        if (r2 > ds || (r2 == ds && odd)) c += 1.f;
        else if (r2 < -ds || (r2 == -ds && odd)) c -= 1.f;
        c = fminf(fmaxf(c, -127.f), 127.f);  // a subnormal d may be far below max|x| / 127
        w[i >> 2] |= ((uint32_t)(int)c & 0xFFu) << (8 * (i & 3));
    }
    return make_uint2(w[0], w[1]);
}

// C: cache element (__half, __nv_bfloat16 or int8_t), X: row element
template <typename X, typename C, int HD>
__global__ void __launch_bounds__(kRowThreads)
kv_pages_write_kernel(const PageView b, const X* __restrict__ kx, const X* __restrict__ vx,
                      int64_t x_stride, C* kc, C* vc, float* ks, float* vs) {
    constexpr int LANES = HD / 8;
    const int per_token = b.n_kv * LANES;  // threads
    const int64_t g0 = (int64_t)blockIdx.x * kRowThreads;
    const int64_t g = g0 + threadIdx.x;
    const int t = (int)(g / per_token), rest = (int)(g - (int64_t)t * per_token);
    const int h = rest / LANES, lane = rest % LANES;
    const Slot at = find_slot(b, (int)(g0 / per_token), t);
    float k[8] = {}, v[8] = {};
    if (at.live) {
        const int64_t off = (int64_t)t * x_stride + (int64_t)h * HD + 8 * lane;
        load8(kx + off, k);
        load8(vx + off, v);
    }
    const int64_t row = (int64_t)h * b.page_size + at.slot;
    const int64_t dst = at.page * b.page_stride + row * HD + 8 * lane;
    if constexpr (sizeof(C) == 1) {
        float dk, dv;
        const uint2 ck = quantise8<LANES>(k, dk), cv = quantise8<LANES>(v, dv);
        if (at.page < 0) return;
        *reinterpret_cast<uint2*>(kc + dst) = ck;
        *reinterpret_cast<uint2*>(vc + dst) = cv;
        if (lane == 0) {
            ks[at.page * b.scale_stride + row] = dk;
            vs[at.page * b.scale_stride + row] = dv;
        }
    } else {
        if (at.page < 0) return;
        store8(kc + dst, k);
        store8(vc + dst, v);
    }
}

template <typename X, typename C, int HD>
__global__ void __launch_bounds__(kRowThreads)
kv_pages_read_kernel(const PageView b, X* __restrict__ kx, X* __restrict__ vx, int64_t x_stride,
                     const C* kc, const C* vc, const float* ks, const float* vs) {
    constexpr int LANES = HD / 8;
    const int per_token = b.n_kv * LANES;
    const int64_t g0 = (int64_t)blockIdx.x * kRowThreads;
    const int64_t g = g0 + threadIdx.x;
    const int t = (int)(g / per_token), rest = (int)(g - (int64_t)t * per_token);
    const int h = rest / LANES, lane = rest % LANES;
    const Slot at = find_slot(b, (int)(g0 / per_token), t);
    if (!at.live) return;
    float k[8] = {}, v[8] = {};
    if (at.page >= 0) {
        const int64_t row = (int64_t)h * b.page_size + at.slot;
        const int64_t src = at.page * b.page_stride + row * HD + 8 * lane;
        if constexpr (sizeof(C) == 1) {
            const float dk = ks[at.page * b.scale_stride + row];
            const float dv = vs[at.page * b.scale_stride + row];
            const uint2 ck = *reinterpret_cast<const uint2*>(kc + src);
            const uint2 cv = *reinterpret_cast<const uint2*>(vc + src);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                k[i] = dk * (float)(int8_t)((i < 4 ? ck.x : ck.y) >> (8 * (i & 3)));
                v[i] = dv * (float)(int8_t)((i < 4 ? cv.x : cv.y) >> (8 * (i & 3)));
            }
        } else {
            load8(kc + src, k);
            load8(vc + src, v);
        }
    }
    const int64_t off = (int64_t)t * x_stride + (int64_t)h * HD + 8 * lane;
    store8(kx + off, k);
    store8(vx + off, v);
}

struct RowCall {
    PageView b;
    const ftc_kv_pages* c;
    void *k, *v;
    int64_t stride;
    bool write;
    cudaStream_t st;
};

template <typename X, typename C, int HD>
int launch_rows(const RowCall& r) {
    const int64_t threads = (int64_t)r.b.n_tokens * r.b.n_kv * (HD / 8);
    const int64_t grid64 = (threads + kRowThreads - 1) / kRowThreads;
    FTC_REQUIRE(grid64 <= INT_MAX, FTC_E_UNSUPPORTED, "ftc_kv_pages: too many rows for one launch");
    const unsigned grid = (unsigned)grid64;
    C* kc = static_cast<C*>(r.c->k);
    C* vc = static_cast<C*>(r.c->v);
    X* k = static_cast<X*>(r.k);
    X* v = static_cast<X*>(r.v);
    if (r.write)
        kv_pages_write_kernel<X, C, HD><<<grid, kRowThreads, 0, r.st>>>(
            r.b, k, v, r.stride, kc, vc, r.c->k_scale, r.c->v_scale);
    else
        kv_pages_read_kernel<X, C, HD><<<grid, kRowThreads, 0, r.st>>>(
            r.b, k, v, r.stride, kc, vc, r.c->k_scale, r.c->v_scale);
    FTC_CUDA(cudaGetLastError());
    return FTC_OK;
}

template <typename X, typename C>
int rows_hd(const RowCall& r) {
    return r.c->head_dim == 64    ? launch_rows<X, C, 64>(r)
           : r.c->head_dim == 128 ? launch_rows<X, C, 128>(r)
                                  : launch_rows<X, C, 256>(r);
}

template <typename X>
int rows_cache(const RowCall& r) {
    return r.c->dtype == FTC_F16    ? rows_hd<X, __half>(r)
           : r.c->dtype == FTC_BF16 ? rows_hd<X, __nv_bfloat16>(r)
                                    : rows_hd<X, int8_t>(r);
}

}  // namespace

int kv_pages_rows(const ftc_kv_pages* c, const ftc_page_batch* b, const void* k, const void* v,
                  int dtype, int64_t stride, bool write, cudaStream_t st) {
    const char* who = write ? "ftc_kv_pages_write" : "ftc_kv_pages_read";
    const std::string w(who);
    RowCall r;
    const int rc = page_view(c, b, who, &r.b);
    if (rc) return rc;
    FTC_REQUIRE(dtype == FTC_F32 || dtype == FTC_F16 || dtype == FTC_BF16, FTC_E_UNSUPPORTED,
                w + ": rows must be F32, F16 or BF16");
    if (b->n_seqs == 0 || b->n_tokens == 0) return FTC_OK;
    FTC_REQUIRE(k && v, FTC_E_INVALID, w + ": null pointer");
    FTC_REQUIRE((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, FTC_E_INVALID,
                w + ": buffers must be 16-byte aligned");
    FTC_REQUIRE(stride >= c->n_head_kv * c->head_dim && stride % (dtype == FTC_F32 ? 4 : 8) == 0 &&
                    stride <= ((int64_t)1 << 36),
                FTC_E_INVALID,
                w + ": row stride must cover n_head_kv * head_dim and be a multiple of 16 bytes");
    r.c = c;
    r.k = const_cast<void*>(k);
    r.v = const_cast<void*>(v);
    r.stride = stride;
    r.write = write;
    r.st = st;
    return dtype == FTC_F32   ? rows_cache<float>(r)
           : dtype == FTC_F16 ? rows_cache<__half>(r)
                              : rows_cache<__nv_bfloat16>(r);
}

}  // namespace ftc
