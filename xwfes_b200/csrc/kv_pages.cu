// kv_pages.cu -- the paged KV cache: storing new K and V rows (rounded to 16
// bits, or quantised to 8 with one scale per position and KV head) and
// reading rows back.
//
// Both move every byte once and are bound by HBM, for a decode step by the
// launch, and 8-bit stores of 16-bit rows by the instructions of a piece (70 % of
// the issue slots at 20 % of HBM; fp32 rows take the same time for 1.7 times the
// bytes).  A piece of work is 8 values of a row of K and the same 8 of V, both
// tensors' loads in flight together, so a row of head_dim values is head_dim / 8
// neighbouring lanes and its maximum is a shuffle reduction inside a warp.
// Measured: 28004 rows of 8 KV heads of 128 read from 8 bits to fp32 49 us (5.9
// TB/s); 8192 bf16 rows stored in 8 bits and read back, two launches, 28 us (3.0
// TB/s); one row each of 48 sequences 5.6 us the pair.
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

// Where lane l's 8 values of a row lie: next to each other, or with fp32 rows
// 4 in each half of the row, so that a warp's 16-byte accesses of the fp32 side
// are whole sectors (8 neighbours made every store write half sectors).
template <typename X, int HD>
struct Spread {
    static constexpr bool kSplit = sizeof(X) == 4;
    static __device__ __forceinline__ int lo(int lane) { return (kSplit ? 4 : 8) * lane; }
    static __device__ __forceinline__ int hi(int lane) {
        return kSplit ? HD / 2 + 4 * lane : 8 * lane + 4;
    }
};

// 8 values of a row of T as loaded, and in fp32
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
};

// p: the row; S: the spread of the side whose type is X (T the type read)
template <class S, typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int lane) {
    Raw8<T> r;
    if constexpr (sizeof(T) == 4) {
        r.w[0] = *reinterpret_cast<const uint4*>(p + S::lo(lane));
        r.w[1] = *reinterpret_cast<const uint4*>(p + S::hi(lane));
    } else if constexpr (S::kSplit) {
        const uint2 a = *reinterpret_cast<const uint2*>(p + S::lo(lane));
        const uint2 b = *reinterpret_cast<const uint2*>(p + S::hi(lane));
        r.w[0] = make_uint4(a.x, a.y, b.x, b.y);
    } else {
        r.w[0] = *reinterpret_cast<const uint4*>(p + S::lo(lane));
    }
    return r;
}

// 8 codes of a row
template <class S>
__device__ __forceinline__ uint2 load_codes(const int8_t* p, int lane) {
    if constexpr (S::kSplit)
        return make_uint2(*reinterpret_cast<const uint32_t*>(p + S::lo(lane)),
                          *reinterpret_cast<const uint32_t*>(p + S::hi(lane)));
    else return *reinterpret_cast<const uint2*>(p + S::lo(lane));
}

template <class S>
__device__ __forceinline__ void store_codes(int8_t* p, int lane, uint2 c) {
    if constexpr (S::kSplit) {
        *reinterpret_cast<uint32_t*>(p + S::lo(lane)) = c.x;
        *reinterpret_cast<uint32_t*>(p + S::hi(lane)) = c.y;
    } else {
        *reinterpret_cast<uint2*>(p + S::lo(lane)) = c;
    }
}

template <typename T>
__device__ __forceinline__ void floats(const Raw8<T>& r, float (&x)[8]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
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

// Bits of the largest |x| of the 8 (16-bit types: both halves of a word at once).
template <typename T>
__device__ __forceinline__ uint32_t top8(const Raw8<T>& r) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
    uint32_t t = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t = max(t, w[i] & 0x7FFFFFFFu);
        return t;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) t = __vmaxu2(t, w[i] & 0x7FFF7FFFu);
        t = max(t & 0xFFFFu, t >> 16);
        return std::is_same<T, __half>::value ? __float_as_uint(h2f(t)) : t << 16;
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

template <class S, typename T>
__device__ __forceinline__ void store8(T* p, int lane, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p + S::lo(lane)) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + S::hi(lane)) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        const uint2 a = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
        const uint2 b = make_uint2(pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
        if constexpr (S::kSplit) {
            *reinterpret_cast<uint2*>(p + S::lo(lane)) = a;
            *reinterpret_cast<uint2*>(p + S::hi(lane)) = b;
        } else {
            *reinterpret_cast<uint4*>(p + S::lo(lane)) = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
}

// The cache slot of a row.
struct Slot {
    int page;  // -1: not mapped
    int slot;
    bool live;  // false: padding
};

// Sequences that end at or before token t0: where a CTA's rows begin to look
// (one round of loads over all threads; a later row walks on from there).
__device__ __forceinline__ int first_seq(const PageView& b, int t0) {
    int before = 0;
    for (int i0 = 0; i0 < b.n_seqs; i0 += kRowThreads) {
        const int i = i0 + (int)threadIdx.x;
        before += __syncthreads_count(i < b.n_seqs && b.start[i + 1] <= t0);
    }
    return before;
}

__device__ __forceinline__ Slot find_slot(const PageView& b, int s, int t) {
    Slot r = {-1, 0, false};
    if (t >= b.n_tokens) return r;
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

// Row and head of piece g of the batch's rows (32-bit arithmetic: a 64-bit
// division a piece cost more than the piece).
template <int HD>
struct Piece {
    int t, h, lane;
    __device__ __forceinline__ Piece(const PageView& b, uint32_t g) {
        constexpr uint32_t LANES = HD / 8;
        const uint32_t row = g / LANES;
        t = (int)(row / (uint32_t)b.n_kv);
        h = (int)(row - (uint32_t)t * (uint32_t)b.n_kv);
        lane = (int)(g % LANES);
    }
};

// Row of 8-bit codes: d = max|x| / 127 and the codes of this thread's 8
// values.  |x| is compared as integer bits, so a NaN wins over an infinity
// and both over every finite value.  The code is the exactly rounded
// quotient: c = x * (1 / d) rounded (by adding 1.5 * 2^23, whose low byte then
// is the code) is within one of it, and the residual r = x - c d (one fused
// multiply-add, exact here: c d has at most 32 bits and cancels to within d)
// tells: |r| < d / 2 and c stands, else the half that it is on decides.  So no
// division and no conversion per value.  Tiny d are scaled by 2^64 first, which
// keeps 1 / d finite.
// top: the bits of this thread's largest |x|.
template <int LANES>
__device__ __forceinline__ uint2 quantise8(float (&x)[8], uint32_t top, float& d) {
    constexpr float kRound = 12582912.f;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top >= 0x7F800000u) {
        d = __uint_as_float(0x7FC00000u);
        return make_uint2(0, 0);
    }
    d = __fdiv_rn(__uint_as_float(top), 127.f);
    if (d == 0.f) return make_uint2(0, 0);
    float ds = d;
    if (d < 1e-30f) {
        ds = d * 18446744073709551616.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= 18446744073709551616.f;
    }
    const float inv = __frcp_rn(ds), half = 0.5f * ds;
    uint32_t q[8];
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t v = f2(x[i], x[i + 1]);
        const uint64_t t = f2add(f2mul(v, f2(inv, inv)), f2(kRound, kRound));
        const uint64_t r = f2fma(f2add(f2(kRound, kRound), f2mul(t, f2(-1.f, -1.f))), f2(ds, ds), v);
        q[i] = (uint32_t)t;
        q[i + 1] = (uint32_t)(t >> 32);
        far = fmaxf(far, fmaxf(fabsf(f2lo(r)), fabsf(f2hi(r))));
    }
    if (far >= half || d < 1e-30f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float c = __uint_as_float(q[i]) - kRound;
            const float r = fmaf(-c, ds, x[i]);
            const bool odd = q[i] & 1;
            if (r > half || (r == half && odd)) c += 1.f;
            else if (r < -half || (r == -half && odd)) c -= 1.f;
            // (a subnormal d may be far below max|x| / 127)
            c = fminf(fmaxf(c, -127.f), 127.f);
            q[i] = __float_as_uint(c + kRound);
        }
    }
    auto bytes = [](uint32_t a, uint32_t b, uint32_t c, uint32_t e) {
        return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, e, 0x0040), 0x5410);
    };
    return make_uint2(bytes(q[0], q[1], q[2], q[3]), bytes(q[4], q[5], q[6], q[7]));
}

// C: cache element (__half, __nv_bfloat16 or int8_t), X: row element.  A
// piece a thread; the rows' loads are issued before the slots are looked up
// (start, kv_len and the table hang on one another).
template <typename X, typename C, int HD>
__global__ void __launch_bounds__(kRowThreads)
kv_pages_write_kernel(const PageView b, const X* __restrict__ kx, const X* __restrict__ vx,
                      int64_t x_stride, C* kc, C* vc, float* ks, float* vs) {
    using S = Spread<X, HD>;
    constexpr int LANES = HD / 8;
    const uint32_t g0 = blockIdx.x * (uint32_t)kRowThreads;
    const Piece<HD> p(b, g0 + threadIdx.x);
    Raw8<X> kr = {}, vr = {};
    if (p.t < b.n_tokens) {
        const int64_t off = (int64_t)p.t * x_stride + (int64_t)p.h * HD;
        kr = load8<S>(kx + off, p.lane);
        vr = load8<S>(vx + off, p.lane);
    }
    const Slot at = find_slot(b, first_seq(b, Piece<HD>(b, g0).t), p.t);
    const int64_t row = (int64_t)p.h * b.page_size + at.slot;
    const int64_t dst = at.page * b.page_stride + row * HD;
    if constexpr (sizeof(C) == 1) {
        float k[8], v[8], dk, dv;
        floats(kr, k);
        floats(vr, v);
        const uint2 ck = quantise8<LANES>(k, top8(kr), dk);
        const uint2 cv = quantise8<LANES>(v, top8(vr), dv);
        if (at.page < 0) return;
        store_codes<S>(kc + dst, p.lane, ck);
        store_codes<S>(vc + dst, p.lane, cv);
        if (p.lane == 0) {
            ks[at.page * b.scale_stride + row] = dk;
            vs[at.page * b.scale_stride + row] = dv;
        }
    } else {
        if (at.page < 0) return;
        if constexpr (std::is_same<X, C>::value) {
            *reinterpret_cast<uint4*>(kc + dst + 8 * p.lane) = kr.w[0];
            *reinterpret_cast<uint4*>(vc + dst + 8 * p.lane) = vr.w[0];
        } else {
            float k[8], v[8];
            floats(kr, k);
            floats(vr, v);
            store8<S>(kc + dst, p.lane, k);
            store8<S>(vc + dst, p.lane, v);
        }
    }
}

// R: pieces per thread, kRowThreads apart.
template <typename X, typename C, int HD, int R>
__global__ void __launch_bounds__(kRowThreads)
kv_pages_read_kernel(const PageView b, X* __restrict__ kx, X* __restrict__ vx, int64_t x_stride,
                     const C* __restrict__ kc, const C* __restrict__ vc,
                     const float* __restrict__ ks, const float* __restrict__ vs) {
    using S = Spread<X, HD>;
    const uint32_t g0 = blockIdx.x * (uint32_t)(kRowThreads * R);
    const int s0 = first_seq(b, Piece<HD>(b, g0).t);
    // all pieces' loads in flight together
    uint2 kq[R], vq[R];
    Raw8<typename std::conditional<sizeof(C) == 1, __half, C>::type> kr[R], vr[R];
    float dk[R], dv[R];
    Slot at[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const Piece<HD> p(b, g0 + i * kRowThreads + threadIdx.x);
        at[i] = find_slot(b, s0, p.t);
        const int64_t row = (int64_t)p.h * b.page_size + at[i].slot;
        const int64_t src = at[i].page * b.page_stride + row * HD;
        if constexpr (sizeof(C) == 1) {
            kq[i] = vq[i] = make_uint2(0, 0);
            dk[i] = dv[i] = 0.f;
            if (at[i].page >= 0) {
                kq[i] = load_codes<S>(kc + src, p.lane);
                vq[i] = load_codes<S>(vc + src, p.lane);
                dk[i] = ks[at[i].page * b.scale_stride + row];
                dv[i] = vs[at[i].page * b.scale_stride + row];
            }
        } else {
            kr[i] = {}, vr[i] = {};
            if (at[i].page >= 0) {
                kr[i] = load8<S>(kc + src, p.lane);
                vr[i] = load8<S>(vc + src, p.lane);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (!at[i].live) continue;
        const Piece<HD> p(b, g0 + i * kRowThreads + threadIdx.x);
        const int64_t off = (int64_t)p.t * x_stride + (int64_t)p.h * HD;
        if constexpr (std::is_same<X, C>::value) {
            *reinterpret_cast<uint4*>(kx + off + 8 * p.lane) = kr[i].w[0];
            *reinterpret_cast<uint4*>(vx + off + 8 * p.lane) = vr[i].w[0];
        } else {
            float k[8], v[8];
            if constexpr (sizeof(C) == 1) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    k[e] = dk[i] * (float)(int8_t)((e < 4 ? kq[i].x : kq[i].y) >> (8 * (e & 3)));
                    v[e] = dv[i] * (float)(int8_t)((e < 4 ? vq[i].x : vq[i].y) >> (8 * (e & 3)));
                }
            } else {
                floats(kr[i], k);
                floats(vr[i], v);
            }
            store8<S>(kx + off, p.lane, k);
            store8<S>(vx + off, p.lane, v);
        }
    }
}

struct RowCall {
    PageView b;
    const ftc_kv_pages* c;
    void *k, *v;
    int64_t stride;
    bool write;
    cudaStream_t st;
};

// Reads of 16-bit rows that fill the device have four pieces a thread in flight
// (28004 rows from 8 bits 35 us, with one 39); fp32 rows (50 and 49 us), writes
// (94 and 90) and small calls (4.7 and 3.5) take one.
template <typename X, typename C, int HD>
int launch_rows(const RowCall& r) {
    const int64_t threads = (int64_t)r.b.n_tokens * r.b.n_kv * (HD / 8);
    FTC_REQUIRE(threads <= INT_MAX - 65536, FTC_E_UNSUPPORTED,
                "ftc_kv_pages: too many rows for one launch");
    auto grid = [&](int pieces) {
        return (unsigned)((threads + kRowThreads * pieces - 1) / (kRowThreads * pieces));
    };
    C* kc = static_cast<C*>(r.c->k);
    C* vc = static_cast<C*>(r.c->v);
    X* k = static_cast<X*>(r.k);
    X* v = static_cast<X*>(r.v);
    constexpr int R = sizeof(X) == 2 ? 4 : 1;
    if (r.write)
        kv_pages_write_kernel<X, C, HD><<<grid(1), kRowThreads, 0, r.st>>>(
            r.b, k, v, r.stride, kc, vc, r.c->k_scale, r.c->v_scale);
    else if (R == 1 || threads < (int64_t)device_sms() * 2048)
        kv_pages_read_kernel<X, C, HD, 1><<<grid(1), kRowThreads, 0, r.st>>>(
            r.b, k, v, r.stride, kc, vc, r.c->k_scale, r.c->v_scale);
    else
        kv_pages_read_kernel<X, C, HD, R><<<grid(R), kRowThreads, 0, r.st>>>(
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
