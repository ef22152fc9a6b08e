// attention_pages.cu -- causal grouped-query attention of a ragged batch of
// new rows over a paged KV cache, with an optional sliding window and sink
// positions (Engine::Impl::attn, ft/src/engine.cpp:137-177, for many
// sequences).
//
// One warp per (row, query head): the visible positions one after another,
// an online softmax (running maximum m and sum l, the accumulator rescaled
// when m grows), head_dim / 32 values per lane.
#include <cuda_bf16.h>

#include <climits>
#include <cmath>

#include "kv_pages.cuh"

namespace ftc {
namespace {

template <typename T>
__device__ __forceinline__ float to_f(T x) {
    if constexpr (std::is_same<T, __half>::value) return __half2float(x);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(x);
    else return (float)x;
}

template <typename T>
__device__ __forceinline__ T from_f(float x) {
    if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
    else return x;
}

struct PagedArgs {
    PageView b;
    const void *q, *k, *v;
    const float *ks, *vs;
    void* out;
    int64_t q_stride, out_stride;
    int n_head, gqa;
    int window, n_sink;
    float scale;
};

template <typename X, typename C, int HD>
__global__ void __launch_bounds__(128) paged_simple(const PagedArgs a) {
    constexpr int E = HD / 32;
    const int h = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int t = blockIdx.y + 65535 * blockIdx.z;
    if (h >= a.n_head || t >= a.b.n_tokens) return;
    int s = 0;
    while (s < a.b.n_seqs && a.b.start[s + 1] <= t) ++s;
    if (s >= a.b.n_seqs) return;
    int r0, n;
    seq_rows(a.b, s, r0, n);
    if (t < r0 || t >= r0 + n) return;
    const int p = seq_len(a.b, s) - n + (t - r0);
    const int kvh = h / a.gqa;
    float q[E], acc[E] = {};
    const X* qr = static_cast<const X*>(a.q) + (int64_t)t * a.q_stride + (int64_t)h * HD;
#pragma unroll
    for (int i = 0; i < E; ++i) q[i] = to_f(qr[lane + 32 * i]) * a.scale;
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j <= p; ++j) {
        if (a.window > 0 && p - j >= a.window && j >= a.n_sink) {
            j = p - a.window;
            continue;
        }
        const int page = page_of(a.b, s, j);
        if (page < 0) continue;
        const int64_t row = (int64_t)kvh * a.b.page_size + (j & (a.b.page_size - 1));
        const int64_t off = page * a.b.page_stride + row * HD;
        const C* kr = static_cast<const C*>(a.k) + off;
        const C* vr = static_cast<const C*>(a.v) + off;
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) d = fmaf(q[i], to_f(kr[lane + 32 * i]), d);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        float vsc = 1.f;
        if constexpr (sizeof(C) == 1) {
            d *= a.ks[page * a.b.scale_stride + row];
            vsc = a.vs[page * a.b.scale_stride + row];
        }
        const float mn = fmaxf(m, d), al = expf(m - mn), e = expf(d - mn);
        l = l * al + e;
        m = mn;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = fmaf(e * vsc, to_f(vr[lane + 32 * i]), acc[i] * al);
    }
    X* o = static_cast<X*>(a.out) + (int64_t)t * a.out_stride + (int64_t)h * HD;
#pragma unroll
    for (int i = 0; i < E; ++i) o[lane + 32 * i] = from_f<X>(l == 0.f ? 0.f : acc[i] / l);
}

template <typename X, typename C>
int launch(const PagedArgs& a, int64_t head_dim, cudaStream_t st) {
    const dim3 grid((unsigned)((a.n_head + 3) / 4),
                    (unsigned)(a.b.n_tokens < 65535 ? a.b.n_tokens : 65535),
                    (unsigned)((a.b.n_tokens + 65534) / 65535));
    if (head_dim == 64) paged_simple<X, C, 64><<<grid, 128, 0, st>>>(a);
    else if (head_dim == 128) paged_simple<X, C, 128><<<grid, 128, 0, st>>>(a);
    else paged_simple<X, C, 256><<<grid, 128, 0, st>>>(a);
    FTC_CUDA(cudaGetLastError());
    return FTC_OK;
}

int check(const ftc_kv_pages* c, const ftc_page_batch* b, int64_t n_head, int q_dtype,
          const char* who, PageView* view) {
    const std::string w(who);
    const int rc = page_view(c, b, who, view);
    if (rc) return rc;
    FTC_REQUIRE(n_head >= 1 && n_head <= 8192 && n_head % c->n_head_kv == 0, FTC_E_INVALID,
                w + ": n_head must be a multiple of n_head_kv, at most 8192");
    FTC_REQUIRE(q_dtype == FTC_F32 || q_dtype == FTC_F16 || q_dtype == FTC_BF16, FTC_E_UNSUPPORTED,
                w + ": q must be F32, F16 or BF16");
    FTC_REQUIRE(q_dtype == FTC_F32 || c->dtype == FTC_KV_Q8 || c->dtype == q_dtype,
                FTC_E_UNSUPPORTED, w + ": 16-bit q over a 16-bit cache of the other type");
    return FTC_OK;
}

}  // namespace

size_t attention_pages_workspace_bytes(const ftc_kv_pages* c, const ftc_page_batch* b,
                                       int64_t n_head, int q_dtype) {
    PageView v;
    if (check(c, b, n_head, q_dtype, "ftc_attention_pages_workspace_bytes", &v)) return 0;
    return 0;
}

int attention_pages(const ftc_kv_pages* c, const ftc_page_batch* b, const void* q, int q_dtype,
                    int64_t q_stride, int64_t n_head, float scale, int64_t window, int64_t n_sink,
                    void* out, int64_t out_stride, void* ws, size_t ws_bytes, cudaStream_t st) {
    PagedArgs a;
    const int rc = check(c, b, n_head, q_dtype, "ftc_attention_pages", &a.b);
    if (rc) return rc;
    FTC_REQUIRE(scale > 0.f && std::isfinite(scale), FTC_E_INVALID,
                "ftc_attention_pages: scale must be positive and finite");
    FTC_REQUIRE(window >= 0 && n_sink >= 0, FTC_E_INVALID,
                "ftc_attention_pages: negative window or n_sink");
    if (b->n_seqs == 0 || b->n_tokens == 0) return FTC_OK;
    FTC_REQUIRE(q && out, FTC_E_INVALID, "ftc_attention_pages: null pointer");
    FTC_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0, FTC_E_INVALID,
                "ftc_attention_pages: buffers must be 16-byte aligned");
    const int64_t unit = q_dtype == FTC_F32 ? 4 : 8;
    FTC_REQUIRE(q_stride >= n_head * c->head_dim && q_stride % unit == 0 &&
                    out_stride >= n_head * c->head_dim && out_stride % unit == 0 &&
                    q_stride <= ((int64_t)1 << 36) && out_stride <= ((int64_t)1 << 36),
                FTC_E_INVALID,
                "ftc_attention_pages: strides must cover n_head * head_dim and be multiples of 16 "
                "bytes");
    const size_t need = attention_pages_workspace_bytes(c, b, n_head, q_dtype);
    FTC_REQUIRE(ws_bytes >= need && (need == 0 || (ws && (uintptr_t)ws % 256 == 0)), FTC_E_INVALID,
                "ftc_attention_pages: workspace smaller than ftc_attention_pages_workspace_bytes "
                "or not 256-byte aligned");
    a.q = q;
    a.k = c->k;
    a.v = c->v;
    a.ks = c->k_scale;
    a.vs = c->v_scale;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.n_head = (int)n_head;
    a.gqa = (int)(n_head / c->n_head_kv);
    a.window = window > INT_MAX ? 0 : (int)window;
    a.n_sink = n_sink > INT_MAX ? INT_MAX : (int)n_sink;
    a.scale = scale;
    if (q_dtype == FTC_F32)
        return c->dtype == FTC_F16    ? launch<float, __half>(a, c->head_dim, st)
               : c->dtype == FTC_BF16 ? launch<float, __nv_bfloat16>(a, c->head_dim, st)
                                      : launch<float, int8_t>(a, c->head_dim, st);
    if (q_dtype == FTC_F16)
        return c->dtype == FTC_F16 ? launch<__half, __half>(a, c->head_dim, st)
                                   : launch<__half, int8_t>(a, c->head_dim, st);
    return c->dtype == FTC_BF16 ? launch<__nv_bfloat16, __nv_bfloat16>(a, c->head_dim, st)
                                : launch<__nv_bfloat16, int8_t>(a, c->head_dim, st);
}

}  // namespace ftc
