// attention_pages.cu -- causal grouped-query attention of a ragged batch of
// new rows over a paged KV cache, with an optional sliding window and sink
// positions (Engine::Impl::attn, ft/src/engine.cpp:137-177, for many
// sequences): argument checks, the choice of kernels, the workspace and the
// joining of cut tiles.
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>

#include "attention_pages.cuh"

namespace ftc {
namespace paged {

int launch_f16(const PagedJob& j, int q_dtype);
int launch_bf16(const PagedJob& j, int q_dtype);
int launch_q8(const PagedJob& j, int q_dtype);
PagedSet geom_f16(int64_t hd, int q_dtype, int cls);
PagedSet geom_bf16(int64_t hd, int q_dtype, int cls);
PagedSet geom_q8(int64_t hd, int q_dtype, int cls);

namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

}  // namespace

// The pool as [page][KV head and slot][head_dim], boxes of up to 128 bytes by
// one page's share of a key chunk.
// plain8: rows of 8-bit codes stay as they lie (they are converted, not fed to
// matrix loads).
int page_map(CUtensorMap* m, const void* base, const ftc_kv_pages* c, int key_step, bool plain8) {
    auto enc = encode_fn();
    FTC_REQUIRE(enc, FTC_E_CUDA, "ftc_attention_pages: cuTensorMapEncodeTiled unavailable");
    const bool q8 = c->dtype == FTC_KV_Q8;
    const int es = q8 ? 1 : 2;
    const int64_t row = c->head_dim * es;
    const cuuint64_t dims[3] = {(cuuint64_t)c->head_dim, (cuuint64_t)(c->n_head_kv * c->page_size),
                                (cuuint64_t)c->n_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)row, (cuuint64_t)(c->page_stride * es)};
    const int64_t boxb = row < 128 ? row : 128;
    const cuuint32_t box[3] = {(cuuint32_t)(boxb / es),
                               (cuuint32_t)std::min<int64_t>(c->page_size, key_step), 1};
    const cuuint32_t ones[3] = {1, 1, 1};
    const CUresult r =
        enc(m,
            q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
               : c->dtype == FTC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            q8 && plain8 ? CU_TENSOR_MAP_SWIZZLE_NONE
            : boxb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FTC_REQUIRE(r == CUDA_SUCCESS, FTC_E_CUDA, "ftc_attention_pages: page tensor map rejected");
    return FTC_OK;
}

}  // namespace paged

namespace {

using namespace paged;

constexpr int kJoinWarps = 8;

// Where a set of tiles keeps its pieces.
struct JoinSet {
    const CutTile* cut;
    const float2* stat;
    const float* part;
    int G, TR;
    // a row per warp, or four in flight where tiles have many rows and so few
    // pieces (256-row tiles, a prompt of 8191 under a window, 14 us instead of
    // 30; but a call of 64-row tiles in 5 pieces 115 us instead of 102)
    __host__ __device__ int rows_per_cta() const { return kJoinWarps * (TR >= 128 ? 4 : 1); }
    __host__ __device__ int blocks() const { return (TR + rows_per_cta() - 1) / rows_per_cta(); }
};

struct JoinArgs {
    JoinSet set[2];
    int blocks0;  // blocks of set 0
    void* out;
    int64_t out_stride;
    int gqa;
};

// The lane's dimensions of a joined row, divided by its sum of weights (no
// maximum: the row sees nothing).
template <typename X, int HD>
__device__ __forceinline__ void store_row(const JoinArgs& a, const CutTile& ct, int r,
                                          const float* acc, float M, float l) {
    constexpr int E = HD / 32;
    const int pr = ct.r0 + r, t = pr / a.gqa, h = ct.kvh * a.gqa + pr - t * a.gqa;
    X* o = static_cast<X*>(a.out) + (int64_t)(ct.row + t) * a.out_stride + (int64_t)h * HD +
           E * (threadIdx.x & 31);
    const float inv = M == -INFINITY && l == l ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
        if constexpr (sizeof(X) == 4)
            *reinterpret_cast<float2*>(o + i) = make_float2(acc[i] * inv, acc[i + 1] * inv);
        else *reinterpret_cast<uint32_t*>(o + i) = pack<X>(acc[i] * inv, acc[i + 1] * inv);
    }
}

// E neighbouring floats.
template <int E>
__device__ __forceinline__ void load_part(const float* p, float* x) {
    if constexpr (E == 2) {
        const float2 v = *reinterpret_cast<const float2*>(p);
        x[0] = v.x, x[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
        }
    }
}

// Row r of a cut tile by a warp: the pieces in order (the CTA that holds the
// tile's start has the first in its slot 1, the CTAs after it theirs in slot
// 0), out = sum_k O_k 2^(M_k - M) / sum_k l_k 2^(M_k - M).
template <typename X, int HD>
__device__ __forceinline__ void join_row(const JoinArgs& a, const JoinSet& s, const CutTile& ct,
                                         int b, int r) {
    const int lane = threadIdx.x & 31;
    auto slot = [&](int k) { return 2 * (int64_t)(b + k) + (k == 0 ? 1 : 0); };
    float M = -INFINITY;
    for (int k = lane; k < ct.pieces; k += 32) M = fmaxf(M, s.stat[slot(k) * s.TR + r].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float R = M == -INFINITY ? 0.f : M;
    constexpr int E = HD / 32;
    float acc[E] = {}, l = 0.f;
    for (int k0 = 0; k0 < ct.pieces; k0 += 32) {
        float w = 0.f, wl = 0.f;
        if (k0 + lane < ct.pieces) {
            const float2 st = s.stat[slot(k0 + lane) * s.TR + r];
            w = ex2(st.x - R);
            wl = st.y * w;
        }
        const int n = min(32, ct.pieces - k0);
        for (int k1 = 0; k1 < n; k1 += 4) {
            float x[4][E];  // four pieces in flight
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int i = 0; i < E; ++i) x[k][i] = 0.f;
                if (k1 + k >= n) continue;
                load_part<E>(s.part + (slot(k0 + k1 + k) * s.TR + r) * HD + E * lane, x[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float wk = __shfl_sync(0xffffffffu, w, k1 + k);
                if (k1 + k >= n) break;
                l += __shfl_sync(0xffffffffu, wl, k1 + k);
#pragma unroll
                for (int i = 0; i < E; ++i) acc[i] = fmaf(x[k][i], wk, acc[i]);
            }
        }
    }
    store_row<X, HD>(a, ct, r, acc, M, l);
}

// Rows r to r + 3 at once, for few pieces: their loads in flight together, the
// maximum as it comes.
template <typename X, int HD>
__device__ __forceinline__ void join_rows4(const JoinArgs& a, const JoinSet& s, const CutTile& ct,
                                           int b, int r) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31;
    float M[4], l[4] = {}, acc[4][E] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) M[i] = -INFINITY;
#pragma unroll 2
    for (int k = 0; k < ct.pieces; ++k) {
        const int64_t row = (2 * (int64_t)(b + k) + (k == 0 ? 1 : 0)) * s.TR + r;
        float2 st[4];
        float x[4][E];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool live = r + i < ct.rows;
            st[i] = live ? s.stat[row + i] : make_float2(-INFINITY, 0.f);
            if (live) load_part<E>(s.part + (row + i) * HD + E * lane, x[i]);
            else
#pragma unroll
                for (int e = 0; e < E; ++e) x[i][e] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float N = fmaxf(M[i], st[i].x), R = N == -INFINITY ? 0.f : N;
            const float f = ex2(M[i] - R), w = ex2(st[i].x - R);
            M[i] = N;
            l[i] = fmaf(st[i].y, w, l[i] * f);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[i][e] = fmaf(x[i][e], w, acc[i][e] * f);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r + i < ct.rows) store_row<X, HD>(a, ct, r + i, acc[i], M[i], l[i]);
}

// kMany: a set has four rows a warp (the others keep the registers that it takes).
template <typename X, int HD, bool kMany>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join(const JoinArgs a) {
    const int which = (int)blockIdx.x >= a.blocks0;
    const JoinSet& s = a.set[which];
    const int blk = blockIdx.x - (which ? a.blocks0 : 0);
    const int rows = kMany ? s.rows_per_cta() / kJoinWarps : 1;
    const int per = kMany ? s.blocks() : (s.TR + kJoinWarps - 1) / kJoinWarps;
    const int b = blk / per, r = ((blk - b * per) * kJoinWarps + (threadIdx.x >> 5)) * rows;
    grid_dependency_wait();
    grid_launch_dependents();
    const CutTile ct = s.cut[b];
    if (ct.pieces == 0 || r >= ct.rows) return;
    if constexpr (kMany) {
        if (rows == 4 && ct.pieces <= 8) return join_rows4<X, HD>(a, s, ct, b, r);
    }
    // many pieces: lanes over their statistics
    for (int i = 0; i < rows && r + i < ct.rows; ++i) join_row<X, HD>(a, s, ct, b, r + i);
}

template <typename X, int HD>
int launch_join(const JoinArgs& a, int blocks, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool many = a.set[0].rows_per_cta() > kJoinWarps || a.set[1].rows_per_cta() > kJoinWarps;
    const cudaError_t e = many ? cudaLaunchKernelEx(&cfg, paged_join<X, HD, true>, a)
                               : cudaLaunchKernelEx(&cfg, paged_join<X, HD, false>, a);
    if (e != cudaSuccess) return cuda_error(e, "launch paged_join");
    return FTC_OK;
}

template <typename X>
int join_hd(const JoinArgs& a, int blocks, int64_t hd, cudaStream_t st) {
    return hd == 64    ? launch_join<X, 64>(a, blocks, st)
           : hd == 128 ? launch_join<X, 128>(a, blocks, st)
                       : launch_join<X, 256>(a, blocks, st);
}

// The launches of a call: which sequences (by packed rows) go to which class.
// Decode sequences and chunks differ too much for one shape; a batch that may
// hold both gets two launches.
struct CallPlan {
    int n = 0;
    int cls[2], min_rows[2], max_rows[2];
    PagedSet set[2];
    size_t off[2], bytes = 0;
};

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

CallPlan call_plan(const ftc_kv_pages* c, const ftc_page_batch* b, int64_t n_head, int q_dtype) {
    CallPlan p;
    const int64_t gqa = n_head / c->n_head_kv;
    const int64_t most = b->max_new > 0 ? std::min(b->max_new, b->n_tokens) : b->n_tokens;
    const int64_t rows = most * gqa;
    auto add = [&](int cls, int lo, int hi) {
        p.cls[p.n] = cls;
        p.min_rows[p.n] = lo;
        p.max_rows[p.n] = hi;
        p.set[p.n] = c->dtype == FTC_F16    ? geom_f16(c->head_dim, q_dtype, cls)
                     : c->dtype == FTC_BF16 ? geom_bf16(c->head_dim, q_dtype, cls)
                                            : geom_q8(c->head_dim, q_dtype, cls);
        const PagedSet& s = p.set[p.n];
        p.off[p.n] = p.bytes;
        const size_t slots = 2 * (size_t)s.G * s.TR;
        p.bytes += up256(s.G * sizeof(CutTile)) + up256(slots * sizeof(float2)) +
                   up256(slots * (size_t)c->head_dim * sizeof(float));
        ++p.n;
    };
    auto cls_of = [](int64_t r) { return r <= 8 ? 0 : r <= 16 ? 1 : r <= 64 ? 2 : 3; };
    const int big = cls_of(rows), one = cls_of(gqa);
    if (big <= 1 || one >= 2 || b->n_seqs == 1 ||
        (b->max_new > 0 && b->n_tokens == b->n_seqs * b->max_new)) {
        add(big, 1, INT_MAX);  // few rows, or sequences of one size
    } else {
        add(one, 1, one == 0 ? 8 : 16);
        add(big, one == 0 ? 9 : 17, INT_MAX);
    }
    return p;
}

int check(const ftc_kv_pages* c, const ftc_page_batch* b, int64_t n_head, int q_dtype,
          const char* who, PageView* view) {
    const std::string w(who);
    const int rc = page_view(c, b, who, view);
    if (rc) return rc;
    FTC_REQUIRE(n_head >= 1 && n_head <= 8192 && n_head % c->n_head_kv == 0, FTC_E_INVALID,
                w + ": n_head must be a multiple of n_head_kv, at most 8192");
    FTC_REQUIRE(b->n_tokens * (n_head / c->n_head_kv) <= (1 << 30), FTC_E_UNSUPPORTED,
                w + ": too many rows for one launch");
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
    if (b->n_seqs == 0 || b->n_tokens == 0) return 0;
    return call_plan(c, b, n_head, q_dtype).bytes;
}

int attention_pages(const ftc_kv_pages* c, const ftc_page_batch* b, const void* q, int q_dtype,
                    int64_t q_stride, int64_t n_head, float scale, int64_t window, int64_t n_sink,
                    void* out, int64_t out_stride, void* ws, size_t ws_bytes, cudaStream_t st) {
    PagedJob j;
    PagedArgs& a = j.a;
    int rc = check(c, b, n_head, q_dtype, "ftc_attention_pages", &a.b);
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
    const CallPlan plan = call_plan(c, b, n_head, q_dtype);
    FTC_REQUIRE(ws && ws_bytes >= plan.bytes && (uintptr_t)ws % 256 == 0, FTC_E_INVALID,
                "ftc_attention_pages: workspace smaller than ftc_attention_pages_workspace_bytes "
                "or not 256-byte aligned");
    a.q = q;
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
    a.c = (float)((double)scale * 1.4426950408889634);
    FTC_REQUIRE(a.c > 0.f && std::isfinite(a.c), FTC_E_INVALID,
                "ftc_attention_pages: scale out of range");
    j.c = c;
    j.st = st;
    JoinArgs jn = {};
    jn.out = out;
    jn.out_stride = out_stride;
    jn.gqa = a.gqa;
    int blocks = 0;
    for (int i = 0; i < plan.n; ++i) {
        const PagedSet& s = plan.set[i];
        uint8_t* base = static_cast<uint8_t*>(ws) + plan.off[i];
        const size_t slots = 2 * (size_t)s.G * s.TR;
        a.cut = reinterpret_cast<CutTile*>(base);
        a.stat = reinterpret_cast<float2*>(base + up256(s.G * sizeof(CutTile)));
        a.part = reinterpret_cast<float*>(base + up256(s.G * sizeof(CutTile)) +
                                          up256(slots * sizeof(float2)));
        a.min_rows = plan.min_rows[i];
        a.max_rows = plan.max_rows[i];
        a.second = i > 0;
        j.set = s;
        j.cls = plan.cls[i];
        rc = c->dtype == FTC_F16    ? launch_f16(j, q_dtype)
             : c->dtype == FTC_BF16 ? launch_bf16(j, q_dtype)
                                    : launch_q8(j, q_dtype);
        if (rc) return rc;
        jn.set[i] = {a.cut, a.stat, a.part, s.G, s.TR};
        blocks += s.G * jn.set[i].blocks();
        if (i == 0) jn.blocks0 = blocks;
    }
    return q_dtype == FTC_F32   ? join_hd<float>(jn, blocks, c->head_dim, st)
           : q_dtype == FTC_F16 ? join_hd<__half>(jn, blocks, c->head_dim, st)
                                : join_hd<__nv_bfloat16>(jn, blocks, c->head_dim, st);
}

}  // namespace ftc
