// attention_pages.cuh -- the paged attention on warp-level tensor cores
// (mma.sync m16n8k16, fp32 accumulators): decode, a few new tokens, and every
// fp32 query.
//
//   out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q.k_j - M),  c = scale log2(e)
// in one pass over the keys (running maximum M, running sum, the accumulator
// rescaled when M grows).  Both products are taken transposed, keys and then
// dimensions as the 16 rows of an instruction (K and V are the A operands,
// read with ldmatrix; q and the weights the B operands of 8 packed rows each),
// so that a decode tile of one KV head's 4 or 8 query heads wastes little and
// the weights go from one product to the next by movmatrix, in registers.
//
// A CTA is NW consumer warps and one producer warp.  The producer brings key
// chunks (KS positions of K and V, one box per page and 128 bytes of head_dim,
// swizzled by TMA so that the matrix loads are free of bank conflicts) into a
// ring of slots; a chunk of a page that is not mapped is fetched out of bounds,
// which fills zeros.  A slot belongs to one group of MW warps, warp i of the
// group taking packed rows 8 NT i onwards; the groups take slots in turn, each
// with a softmax state of its own, and meet only at a tile's end.  Decode (MW =
// 1, 8 or 16 packed rows) has 4 independent warps on one tile's keys and its
// next q prepared by the producer; chunks (MW = 4, 8: one group) read each key
// once for 64 or 128 rows.
//
// Decode is bound by HBM: 2 (head_dim bytes) a position and KV head; 64
// sequences of 100 to 16000 positions, 32 heads on 8, 8-bit: 202 us, 5.5 TB/s.
// Why matrix instructions for it: with 4 query heads on a KV head the CUDA
// cores would need 8 multiply-adds a byte of cache, 1.5 times what they have at
// HBM speed, and the 8-bit decode on top.  A few sequences are bound by latency
// (one of 517 positions: 17 us, the plan, a chunk and the join in turn), and
// groups of 4 warps by it too: 40 fp32 rows over an f16 cache (8 sequences of
// 900 to 6000) take 106 us, 1.1 TB/s, 2.4 warps a scheduler, a third of the
// issue slots used.  fp32 queries in chunks stay on this path: 1024 tokens on
// 8192, 32 heads, 1.11 ms over 8 bits, 1.42 over f16, 1.70 over bf16 (2 or 3
// pieces of q and of the weights: 2 or 3 times the products); so does head_dim
// 256, 2.14 ms with bf16.  fp32 instances spill: at head_dim 128 over 8 bits
// 34 to 142 bytes, over 16 bits 4 to 50.
//
// Types.  Operands are f16 for f16 and 8-bit caches, bf16 for bf16 caches; the
// 8-bit codes are exact in f16 (byte -> 1024 + code + 128 in the mantissa, one
// subtraction), their scales stay outside: K's multiplies the score, V's the
// weight.  q: a 16-bit q is one operand; a bf16 q over an 8-bit cache becomes
// f16 with a power-of-two scale per row; an fp32 q is 2 f16 pieces (scaled the
// same way, 2^-22 kept: one bit or two short of fp32's own) or 3 bf16 pieces.
// Weights: fp32 q also splits them (2 or 3 pieces), else they are rounded once
// to the operand type, which a 16-bit result tolerates (an f16 result of a chunk
// is 0.00029 from exact where fp32 weights give 0.00021, a bf16 one 0.0023 and
// 0.0017, relative to the results) and saves half of PV's products; 2^14 up in
// f16 (and V's scale relative to the running maximum of those that the row
// sees, 2^E) so that weights 2^-38 of the largest still count.  With fp32 q the
// matrix unit's own accumulation, which truncates, is kept to short chains that
// fp32 adds join.
#pragma once

#include <cuda_bf16.h>

#include <cfloat>
#include <type_traits>

#include "paged_plan.cuh"

namespace ftc {
namespace paged {

template <typename X_, typename C_, int HD_, int NT_, int MW_, int NW_>
struct Cfg {
    using X = X_;
    using C = C_;
    static constexpr int HD = HD_, NT = NT_, MW = MW_, NW = NW_;
    static constexpr int NG = NW / MW;      // warp groups
    static_assert(MW == 1 || NG == 1, "one group of several warps, or groups of one");
    static constexpr int WR = 8 * NT;       // packed rows per warp
    static constexpr int TR = WR * MW;      // packed rows per tile
    using OT = typename std::conditional<std::is_same<C, __nv_bfloat16>::value, __nv_bfloat16,
                                         __half>::type;
    static constexpr bool kF32 = sizeof(X) == 4, kQ8 = sizeof(C) == 1;
    static constexpr bool kHalf = std::is_same<OT, __half>::value;
    // pieces of q and of the weights
    static constexpr int NP = kF32 ? (kHalf ? 2 : 3) : 1;
    static constexpr bool kRowScale = kHalf && !std::is_same<X, __half>::value;
    static constexpr int ROWB = HD * (int)sizeof(C);  // bytes of a cached row
    static constexpr int BOXB = ROWB < 128 ? ROWB : 128;
    static constexpr int NBOX = ROWB / BOXB;
    // slots of about 8 KB: each of the NW warps holds one while it computes
    static constexpr int KS = 64 * ROWB <= 8192 ? 32 : 16;
    static constexpr int SLOT = 2 * KS * ROWB;
    static constexpr int NQB = MW == 1 ? 2 : 1;        // q buffers
    static constexpr int QB1 = MW * NT * NP * (HD / 16) * 256;
    static constexpr int QB = NQB * QB1;
    static constexpr int PER = HD / 4 * NT + 4 * NT;   // floats a lane hands over in a join
    static constexpr int XB = NG > 1 ? (NG / 2) * 32 * PER * 4 : 0;
    static constexpr int CTL = 1536;                   // barriers, flags, row factors
    static constexpr int kFixed = 1024 /* alignment */ + QB + XB + CTL;
    static constexpr int SLOT_ALL = SLOT + (kQ8 ? 2 * KS * 4 : 0);
    // CTAs per SM: as many as leave a thread its registers (the accumulator is
    // HD / 4 * NT of them) and the ring slots in flight beside the held ones
    static constexpr int fit(int occ) { return (224 * 1024 / occ - kFixed) / SLOT_ALL; }
    static constexpr int OCC = NW <= 4 && NT == 1 && HD < 256 && fit(3) >= NG + 2 ? 3
                               : NW <= 4 && NT * HD <= 256 && fit(2) >= NG + 2    ? 2
                                                                                  : 1;
    static constexpr int NSLOT = fit(OCC) < 24 ? fit(OCC) : 24;
    static_assert(NSLOT >= NG + 1, "ring holds every group's slot and one in flight");
    static constexpr int OFF_RING = 0;
    static constexpr int OFF_SCALE = OFF_RING + NSLOT * SLOT;
    static constexpr int OFF_Q = OFF_SCALE + (kQ8 ? NSLOT * 2 * KS * 4 : 0);
    static constexpr int OFF_X = OFF_Q + QB;
    static constexpr int OFF_BAR = OFF_X + XB;
    static constexpr int SMEM = OFF_BAR + CTL + 1024;
    static_assert(NSLOT * SLOT >= Plan<TR, KS>::kSmem, "the plan's prefix sums fit in the ring");
    static constexpr int THREADS = (NW + 1) * 32;
};

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tma_box(void* dst, const CUtensorMap* map, int x, int y, int z,
                                        uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z),
        "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// 8 x 8 matrix of 16-bit elements, one row per four lanes, transposed.
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src)
                 : "memory");
}

// Arrives on `bar` (counted in its phase) when this thread's cp.async so far
// have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    if constexpr (kHalf)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Bytes i and j of w (codes + 128) as two f16 codes: 0x64uu is 1024 + u, and
// subtracting 1152 is exact.
template <int SEL>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
    const uint32_t u = __byte_perm(w, 0x64646464u, SEL);
    const uint32_t b = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u),
                              *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename OT>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    if constexpr (std::is_same<OT, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// The rounded pair back in fp32.
template <typename OT>
__device__ __forceinline__ float2 unpack(uint32_t w) {
    if constexpr (std::is_same<OT, __half>::value) return make_float2(h2f(w), h2f(w >> 16));
    else return make_float2(bf2f(w), bf2f(w >> 16));
}

// a, b as NP operands whose sum is a, b.
template <typename OT, int NP>
__device__ __forceinline__ void split(float a, float b, uint32_t (&out)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        out[i] = pack<OT>(a, b);
        if (i + 1 < NP) {
            const float2 r = unpack<OT>(out[i]);
            a -= r.x;
            b -= r.y;
        }
    }
}

template <typename X>
__device__ __forceinline__ float load1(const X* p) {
    if constexpr (std::is_same<X, __half>::value) return __half2float(*p);
    else return __bfloat162float(*p);
}

template <typename X>
__device__ __forceinline__ float2 load2(const X* p) {
    if constexpr (sizeof(X) == 4) return *reinterpret_cast<const float2*>(p);
    else return unpack<X>(*reinterpret_cast<const uint32_t*>(p));
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }

// 16-byte chunk `c` of row `r` in a box tile of K or V.
template <class F>
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
    constexpr int CPB = F::BOXB / 16;
    const int sw = F::BOXB == 128 ? (r & 7) : ((r >> 1) & 3);
    return (uint32_t)((c / CPB) * (F::KS * F::BOXB) + r * F::BOXB + (((c % CPB) ^ sw) << 4));
}

__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *dead != 0)) return false;
    if (mbar_wait_warp(bar, parity)) return true;
    *dead = 1;
    return false;
}

// Waits until the producer has begun chunk k in its slot.  A slot's uses go to
// the groups in turn, so a group that is ahead may come to its use while the
// one before it, another group's, has not landed: the barrier's parity would
// then answer for the use before that.  Once the tag says k, the barrier is in
// this use's phase.
__device__ __forceinline__ bool tag_wait(volatile int* tag, int k, volatile int* dead) {
    const int lane = threadIdx.x & 31;
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
        if (__all_sync(0xffffffffu, *tag == k)) return true;
        if (__any_sync(0xffffffffu, *dead != 0)) return false;
        if ((i & 255u) == 255u) {
            int late = 0;
            if (lane == 0) {
                const uint64_t now = global_ns();
                if (t0 == 0) t0 = now;
                else late = now - t0 > kWaitLimitNs;
            }
            if (__shfl_sync(0xffffffffu, late, 0)) {
                if (lane == 0) record_timeout();
                *dead = 1;
                return false;
            }
        }
    }
}

struct Vis {
    int window, n_sink;
    __device__ __forceinline__ bool operator()(int key, int p) const {
        return key <= p && (window == 0 || p - key < window || key < n_sink);
    }
};

// Whether a row at `pos` sees a position of chunks p.i to p.i + m - 1 of its
// tile (for rows that end without a maximum: the loop over keys has no part
// in it).
template <int KS, class Tile>
__device__ __noinline__ bool sees_any(const PagedArgs& a, const PlanPos& p, const Tile& tw, int m,
                                      int pos) {
    for (int j = 0; j < m; ++j) {
        const int key0 = tw.key0(p.i + j);
        for (int k = key0; k < key0 + KS && k <= pos; k += 16)
            if ((a.window == 0 || pos - min(k + 15, pos) < a.window || k < a.n_sink) &&
                page_of(a.b, p.s, k) >= 0)
                return true;
    }
    return false;
}

// Where the packed row pr of a tile's sequence comes from and goes to.
struct RowRef {
    int tok, head;
    __device__ __forceinline__ RowRef(const PagedArgs& a, const PlanPos& p, int pr) {
        tok = pr / a.gqa;
        head = p.kvh * a.gqa + pr - tok * a.gqa;
    }
};

// One warp's rows of q as B operands: pieces to sQ, score factors to sC.
template <class F>
__device__ __forceinline__ void prepare_q(const PagedArgs& a, const PlanPos& p, int pr0, uint2* sQ,
                                          float* sC) {
    using X = typename F::X;
    using OT = typename F::OT;
    constexpr int HD = F::HD, NP = F::NP;
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int rows = p.n * a.gqa;
    // the order of the 16 k of an instruction is free: with 8-bit codes a
    // lane's four are neighbours (one word of the cache row)
    const int kl = F::kQ8 ? 4 * t4 : 2 * t4, kh = F::kQ8 ? 4 * t4 + 2 : 2 * t4 + 8;
#pragma unroll
    for (int n = 0; n < F::NT; ++n) {
        const int pr = pr0 + 8 * n + g;
        const bool live = pr < rows;
        const RowRef r(a, p, live ? pr : 0);
        const X* q = static_cast<const X*>(a.q) + (int64_t)(p.row + r.tok) * a.q_stride +
                     (int64_t)r.head * HD;
        float2 x[HD / 16], y[HD / 16];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            x[i] = y[i] = make_float2(0.f, 0.f);
            if (live) x[i] = load2(q + 16 * i + kl), y[i] = load2(q + 16 * i + kh);
        }
        float fa = 1.f, fb = 1.f, c = a.c;
        if constexpr (F::kRowScale) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
                top = max(max(max(top, __float_as_uint(fabsf(x[i].x))),
                              __float_as_uint(fabsf(x[i].y))),
                          max(__float_as_uint(fabsf(y[i].x)), __float_as_uint(fabsf(y[i].y))));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the row's largest value lands in [2^14, 2^15); 2^-e as two
            // factors that are in range
            const int e = top > 0 && top < 0x7F800000u ? (int)(top >> 23) - 141 : 0;
            fa = pow2(-e / 2), fb = pow2(-e - -e / 2);
            c = fmaxf(a.c * pow2(e / 2) * pow2(e - e / 2), 1e-38f);
        }
        if (t4 == 0) sC[8 * n + g] = c;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            if constexpr (F::kRowScale) {
                x[i].x = x[i].x * fa * fb, x[i].y = x[i].y * fa * fb;
                y[i].x = y[i].x * fa * fb, y[i].y = y[i].y * fa * fb;
            }
            uint32_t b0[NP], b1[NP];
            split<OT, NP>(x[i].x, x[i].y, b0);
            split<OT, NP>(y[i].x, y[i].y, b1);
#pragma unroll
            for (int q2 = 0; q2 < NP; ++q2)
                sQ[((n * NP + q2) * (HD / 16) + i) * 32 + lane] = make_uint2(b0[q2], b1[q2]);
        }
    }
}

template <typename X>
__device__ __forceinline__ void store1(X* o, float v) {
    if constexpr (sizeof(X) == 4) *o = v;
    else if constexpr (std::is_same<X, __half>::value) *o = __float2half_rn(v);
    else *o = __float2bfloat16_rn(v);
}

template <class F>
__global__ void __launch_bounds__(F::THREADS, F::OCC)
paged_mma(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
          const __grid_constant__ PagedArgs a, int least) {
    using X = typename F::X;
    using C = typename F::C;
    using OT = typename F::OT;
    constexpr int HD = F::HD, NT = F::NT, MW = F::MW, NG = F::NG, NP = F::NP, KS = F::KS;
    constexpr int TR = F::TR, DT = HD / 16, KT = KS / 16;  // 16-dimension and 16-key tiles
    using P = Plan<TR, KS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* sScale = reinterpret_cast<float*>(smem + F::OFF_SCALE);
    float* sX = reinterpret_cast<float*>(smem + F::OFF_X);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + F::OFF_BAR);
    uint64_t* empty = full + F::NSLOT;
    uint64_t* q_full = empty + F::NSLOT;  // [2]
    uint64_t* q_empty = q_full + 2;
    volatile int* dead = reinterpret_cast<volatile int*>(q_empty + 2);
    int* sFlag = const_cast<int*>(dead) + 4;  // [NSLOT] mapped halves
    volatile int* sTag = sFlag + 24;          // [NSLOT] chunk in the slot
    PlanPos* sPos = reinterpret_cast<PlanPos*>(sFlag + 48);
    float* sC = reinterpret_cast<float*>(sPos + 1);  // [NQB][TR]
    static_assert(F::NSLOT * 16 + 32 + 16 + 192 + (int)sizeof(PlanPos) + F::NQB * TR * 4 <= F::CTL,
                  "control block");
    int64_t* sPre = reinterpret_cast<int64_t*>(smem + F::OFF_RING);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < F::NSLOT; ++i) {
            mbar_init(&full[i], F::kQ8 ? 33 : 1);
            mbar_init(&empty[i], MW);
            sTag[i] = -1;
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], F::NW);
        }
        *dead = 0;
        mbar_fence_init();
    }
    // The second launch of a call needs nothing of the first, whose CTAs all
    // passed this wait before they let it start: it waits at its end instead,
    // so that its own end still means that both are done.
    if (!a.second) grid_dependency_wait();
    grid_launch_dependents();
    __syncthreads();

    // this CTA's share of the units
    int64_t tiles;
    int largest;
    const int64_t W = P::template scan<false>(a, sPre, tiles, largest);
    const int64_t L = plan_share(W, tiles, (int)gridDim.x, NG, least);
    const int64_t u0 = (int64_t)blockIdx.x * L;
    if (u0 >= W) {
        if (threadIdx.x == 0) a.cut[blockIdx.x].pieces = 0;
        if (a.second) grid_dependency_wait();
        return;
    }
    const int total = (int)min(L, W - u0);
    if (warp == 0) {
        const PlanPos p = P::locate(a, sPre, u0);
        if (lane == 0) *sPos = p;
    }
    fence_proxy_async_smem();  // the prefix sums are done with: the ring may be filled
    __syncthreads();
    PlanPos p = *sPos;
    auto q_buf = [&](int buf, int mt) {
        return reinterpret_cast<uint2*>(smem + F::OFF_Q + buf * F::QB1) +
               mt * NT * NP * (HD / 16) * 32;
    };

    if (warp == F::NW) {
        // -------------------------------------------------------- producer
        const int box = min(a.b.page_size, KS);  // rows of a box
        const int halves = KS / box;             // boxes over the keys (1 or 2)
        uint32_t it = 0, seg = 0;
        for (int left = total; left > 0; ++seg) {
            const TileWork<TR, KS> tw(a, p.n, p.len, p.t);
            const int m = min(tw.count - p.i, left);
            for (int j0 = 0; j0 < m; j0 += 32) {
                int key = 0, id0 = -1, id1 = -1;
                if (j0 + lane < m) {
                    key = tw.key0(p.i + j0 + lane);
                    id0 = page_of(a.b, p.s, key);
                    if (halves == 2) id1 = page_of(a.b, p.s, key + box);
                }
                if (MW == 1 && j0 == 0) {
                    // the tile's q, while the consumers are on the last one
                    const int buf = seg & 1;
                    if (!ring_wait(&q_empty[buf], ((seg >> 1) & 1) ^ 1, dead)) break;
                    prepare_q<F>(a, p, p.t * TR, q_buf(buf, 0), sC + buf * TR);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_full[buf]);
                }
                const int jn = min(32, m - j0);
                for (int j = 0; j < jn; ++j, ++it) {
                    const int k0 = __shfl_sync(0xffffffffu, key, j);
                    const int ia = __shfl_sync(0xffffffffu, id0, j);
                    const int ib = __shfl_sync(0xffffffffu, id1, j);
                    const int s = it % F::NSLOT;
                    if (!ring_wait(&empty[s], ((it / F::NSLOT) & 1) ^ 1, dead)) break;
                    if (lane == 0) {
                        sFlag[s] = halves == 2 ? (ia >= 0 ? 1 : 0) | (ib >= 0 ? 2 : 0)
                                               : (ia >= 0 ? 3 : 0);
                        sTag[s] = (int)it;
                        mbar_arrive_expect_tx(&full[s], F::SLOT);
                    }
                    __syncwarp();
                    const int y = p.kvh * a.b.page_size + (k0 & (a.b.page_size - 1));
                    {
                        // lane l: tensor (K, V), 128-byte column, page half
                        const int kv = lane & 1, col = (lane >> 1) % F::NBOX;
                        const int half = (lane >> 1) / F::NBOX;
                        const int id = half ? ib : ia;
                        if (half < halves)  // past the last page: zeros
                            tma_box(smem + F::OFF_RING + s * F::SLOT + kv * (KS * F::ROWB) +
                                        col * (KS * F::BOXB) + half * box * F::BOXB,
                                    kv ? &tv : &tk, col * (F::BOXB / (int)sizeof(C)), y,
                                    id < 0 ? a.b.n_pages : id, &full[s]);
                    }
                    if constexpr (F::kQ8) {
                        // four scales a lane (a copy of its own per page would
                        // cost the TMA unit as much as a box)
                        const int kv = lane / (KS / 4), q4 = lane % (KS / 4) * 4;
                        const int id = q4 >= box ? ib : ia;
                        if (kv < 2 && id >= 0)
                            cp_async16(sScale + (s * 2 + kv) * KS + q4,
                                       (kv ? a.vs : a.ks) + (int64_t)id * a.b.scale_stride + y +
                                           (q4 >= box ? q4 - box : q4));
                        cp_async_arrive(&full[s]);
                    }
                    __syncwarp();
                }
                if (*dead) break;
            }
            if (*dead) break;
            left -= m;
            if (left > 0) P::next_tile(a, p);
        }
        if (*dead && lane == 0)  // let issued copies land before the CTA leaves
            for (uint32_t j = it > (uint32_t)F::NSLOT ? it - F::NSLOT : 0; j < it; ++j)
                mbar_wait(&full[j % F::NSLOT], (j / F::NSLOT) & 1);
        if (a.second) grid_dependency_wait();
        return;
    }

    // ------------------------------------------------------------ consumers
    const int grp = warp / MW, mt = warp % MW;
    const int g = lane >> 2, t4 = lane & 3;
    const Vis vis = {a.window, a.n_sink};
    uint32_t it = 0, seg = 0;
    bool owner = false;
    for (int left = total; left > 0; ++seg) {
        const TileWork<TR, KS> tw(a, p.n, p.len, p.t);
        const int m = min(tw.count - p.i, left);
        const bool cut_l = p.i > 0, cut_r = p.i + m < tw.count;
        const int rows = p.n * a.gqa;
        const int pr = p.t * TR + mt * F::WR;         // the warp's first packed row
        const int wrows = min(rows - pr, F::WR);      // <= 0: none
        const int buf = F::NQB == 2 ? seg & 1 : 0;
        const uint2* sQ = q_buf(buf, mt);
        const float* cq = sC + buf * TR + mt * F::WR;
        if constexpr (MW == 1) {
            ring_wait(&q_full[buf], (seg >> 1) & 1, dead);
        } else {
            __syncwarp();
            prepare_q<F>(a, p, pr, q_buf(0, mt), sC + mt * F::WR);
            __syncwarp();
        }
        // this lane's rows: 2 t4 and 2 t4 + 1 of each 8
        float c[NT][2];
        int pos[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * n + 2 * t4 + e;
                c[n][e] = cq[r];
                pos[n][e] = r < wrows ? p.len - p.n + (pr + r) / a.gqa : -1;
            }
        // rows of this warp for the mask tests
        const int p_lo = p.len - p.n + pr / a.gqa;
        const int p_hi = wrows > 0 ? p.len - p.n + (pr + wrows - 1) / a.gqa : -1;

        constexpr float kLeastE = -100.f;  // weights 2^(14 - E) fit fp32
        float O[DT][NT][4];  // dimensions g, g + 8 of a tile by rows 2 t4, 2 t4 + 1
        float M[NT][2], l[NT][2];
        // 8-bit V: weights times scales, and with them both sums, are held
        // relative to 2^E, the largest scale that this row sees
        float E[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            M[n][0] = M[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
            E[n][0] = E[n][1] = kLeastE;
#pragma unroll
            for (int d = 0; d < DT; ++d) O[d][n][0] = O[d][n][1] = O[d][n][2] = O[d][n][3] = 0.f;
        }

        for (int j = grp; j < m; j += NG) {
            const uint32_t k = it + j;
            const int s = k % F::NSLOT;
            if (!tag_wait(&sTag[s], (int)k, dead)) continue;
            if (!ring_wait(&full[s], (k / F::NSLOT) & 1, dead)) continue;
            const int key0 = tw.key0(p.i + j);
            const int flag = sFlag[s];
            if (key0 > p_hi || flag == 0) {  // nothing here for this warp's rows
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
                continue;
            }
            const bool whole = flag == 3 && key0 + KS - 1 <= p_lo &&
                               (a.window == 0 || p_hi - key0 < a.window ||
                                key0 + KS - 1 < a.n_sink);
            const uint32_t ks_addr = smem_u32(smem + F::OFF_RING + s * F::SLOT);
            const uint32_t vs_addr = ks_addr + KS * F::ROWB;

            // ---- scores, keys by rows: K is the A operand, q the B operand
            float S[KT][NT][4], lo[F::kF32 ? KT : 1][F::kF32 ? NT : 1][4];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    S[kt][n][0] = S[kt][n][1] = S[kt][n][2] = S[kt][n][3] = 0.f;
                    if constexpr (F::kF32)
                        lo[kt][n][0] = lo[kt][n][1] = lo[kt][n][2] = lo[kt][n][3] = 0.f;
                }
            constexpr int CPI = F::kQ8 ? 1 : 2;  // 16-byte chunks per 16 k
#pragma unroll
            for (int i2 = 0; i2 < HD / 16; i2 += 2 / CPI) {
                // two chunks of 16 keys: 8-bit, two steps of 16 k; 16-bit, one
                uint32_t r[KT][4];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
                    ldsm4(r[kt], ks_addr + chunk_off<F>(16 * kt + (lane & 15),
                                                        i2 * CPI + (lane >> 4)));
#pragma unroll
                for (int st = 0; st < 2 / CPI; ++st) {
                    const int i = i2 + st;
                    uint2 qv[NT][NP];
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int q = 0; q < NP; ++q)
                            qv[n][q] = sQ[((n * NP + q) * (HD / 16) + i) * 32 + lane];
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        uint32_t ka[4];  // keys g, g + 8 of the low k, then of the high
                        if constexpr (F::kQ8) {
                            const uint32_t u0_ = r[kt][2 * st] ^ 0x80808080u;
                            const uint32_t u1_ = r[kt][2 * st + 1] ^ 0x80808080u;
                            ka[0] = codes2<0x4140>(u0_);
                            ka[1] = codes2<0x4140>(u1_);
                            ka[2] = codes2<0x4342>(u0_);
                            ka[3] = codes2<0x4342>(u1_);
                        } else {
                            ka[0] = r[kt][0], ka[1] = r[kt][1], ka[2] = r[kt][2], ka[3] = r[kt][3];
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma16816<F::kHalf>(S[kt][n], ka, qv[n][0].x, qv[n][0].y);
#pragma unroll
                            for (int q = 1; q < NP; ++q)
                                mma16816<F::kHalf>(lo[kt][n], ka, qv[n][q].x, qv[n][q].y);
                        }
                    }
                }
            }
            if constexpr (F::kF32) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            // (an infinite key times a lower piece that is 0 or of the
                            // other sign: the first piece says what the score is)
                            const float x = S[kt][n][i] + lo[kt][n][i];
                            S[kt][n][i] = x == x ? x : S[kt][n][i];
                        }
            }

            // ---- the 8-bit scales of this lane's keys, 16 kt + g and + 8
            float vsc[KT][2];
            float Ec[NT][2];  // of this chunk
            if constexpr (F::kQ8) {
                const float* ksc = sScale + (s * 2) * KS;
                auto exponent = [](uint32_t bits) { return (float)((int)(bits >> 23) - 126); };
                uint32_t sb[KT][2];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int kk = 16 * kt + 8 * h + g;
                        const float kf = ksc[kk];
                        vsc[kt][h] = ksc[KS + kk];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            S[kt][n][2 * h] *= kf;
                            S[kt][n][2 * h + 1] *= kf;
                        }
                        sb[kt][h] = __float_as_uint(fabsf(vsc[kt][h]));
                        if (sb[kt][h] >= 0x7F800000u) sb[kt][h] = 0;
                    }
                if (whole) {
                    uint32_t t = 0;
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) t = max(t, max(sb[kt][0], sb[kt][1]));
                    const float x = exponent(__reduce_max_sync(0xffffffffu, t));
#pragma unroll
                    for (int n = 0; n < NT; ++n) Ec[n][0] = Ec[n][1] = x;
                } else {
                    // (a slot hidden from a row may hold any scale)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint32_t t = 0;
#pragma unroll
                            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const int kk = 16 * kt + 8 * h + g;
                                    if (((flag >> (kk / (KS / 2))) & 1) &&
                                        vis(key0 + kk, pos[n][e]))
                                        t = max(t, sb[kt][h]);
                                }
                            t = max(t, __shfl_xor_sync(0xffffffffu, t, 4));
                            t = max(t, __shfl_xor_sync(0xffffffffu, t, 8));
                            t = max(t, __shfl_xor_sync(0xffffffffu, t, 16));
                            Ec[n][e] = exponent(t);
                        }
                }
            }

            // ---- softmax: new maxima, weights (2^14 up in f16), sums
            if (!whole) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int kk = 16 * kt + 8 * h + g;
                        const bool on = (flag >> (kk / (KS / 2))) & 1;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                // a hidden score is marked by a NaN with this payload
                                if (!(on && vis(key0 + kk, pos[n][e])))
                                    S[kt][n][2 * h + e] = __uint_as_float(0xFFFFDEADu);
                    }
            }
            float al[NT][2], D[NT][2];
            constexpr float kUp = F::kHalf ? 14.f : 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mx = fmaxf(S[0][n][e], S[0][n][2 + e]);  // fmaxf skips NaN
#pragma unroll
                    for (int kt = 1; kt < KT; ++kt)
                        mx = fmaxf(mx, fmaxf(S[kt][n][e], S[kt][n][2 + e]));
                    mx = fmaxf(mx, -INFINITY);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float N = fmaxf(M[n][e], mx * c[n][e]);
                    const float R = N == -INFINITY ? 0.f : N;
                    al[n][e] = M[n][e] - R;
                    M[n][e] = N;
                    D[n][e] = kUp - R;
                    if constexpr (F::kQ8) {
                        const float En = fmaxf(E[n][e], Ec[n][e]);
                        al[n][e] += E[n][e] - En;
                        D[n][e] -= En;
                        E[n][e] = En;
                    }
                    al[n][e] = ex2(al[n][e]);  // 0 while M is -inf
                }
            uint32_t pb[KT][NT][NP][2];  // weights as B operand: keys by rows
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float sum[2] = {0.f, 0.f};
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float sv = S[kt][n][2 * h + e];
                            const bool hid = !whole && __float_as_uint(sv) == 0xFFFFDEADu;
                            w[e] = hid ? 0.f : ex2(fmaf(sv, c[n][e], D[n][e]));
                            sum[e] += w[e];
                            // (a scale that is not finite reaches who sees it at any weight)
                            if constexpr (F::kQ8) w[e] = hid ? 0.f : w[e] * vsc[kt][h];
                        }
                        uint32_t x[NP];
                        split<OT, NP>(w[0], w[1], x);
#pragma unroll
                        for (int q = 0; q < NP; ++q) pb[kt][n][q][h] = movm_t(x[q]);
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e) l[n][e] = fmaf(l[n][e], al[n][e], sum[e]);
            }

            // ---- weighted V, dimensions by rows: V is the A operand.  16-bit
            // results tolerate the matrix unit's own accumulation over all
            // keys, fp32 ones get fresh sums per chunk
            bool odd = false;
            if constexpr (!F::kF32) {
                bool grow = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) grow |= al[n][0] != 1.f || al[n][1] != 1.f;
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            O[d][n][0] *= al[n][0], O[d][n][1] *= al[n][1];
                            O[d][n][2] *= al[n][0], O[d][n][3] *= al[n][1];
                        }
                }
            }
            constexpr int DPI = F::kQ8 ? 2 : 1;  // 16-dimension tiles in two chunks
#pragma unroll
            for (int d2 = 0; d2 < DT; d2 += DPI) {
                float acc[F::kF32 ? DPI : 1][F::kF32 ? NT : 1][4];
                if constexpr (F::kF32) {
#pragma unroll
                    for (int i = 0; i < DPI; ++i)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f;
                }
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    uint32_t r[4];  // keys 0-7 and 8-15 of one chunk, then of the next
                    ldsm4_t(r, vs_addr + chunk_off<F>(16 * kt + (lane & 15),
                                                      d2 * (F::kQ8 ? 1 : 2) + (lane >> 4)));
                    if constexpr (!F::kQ8) {
                        // V that is not finite may be hidden from some rows,
                        // and pieces of a weight may be 0 or of either sign:
                        // out of the product, added below where it is seen.
                        // (A full exponent field carries into the sign bit.)
                        if (F::kF32 || !whole) {
                            constexpr uint32_t kInf = F::kHalf ? 0x7C007C00u : 0x7F807F80u;
                            constexpr uint32_t kOne = F::kHalf ? 0x04000400u : 0x00800080u;
                            uint32_t z = 0;
#pragma unroll
                            for (int i = 0; i < 4; ++i) z |= (r[i] & kInf) + kOne;
                            if (__any_sync(0xffffffffu, (z & 0x80008000u) != 0)) {
                                odd = true;
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const uint32_t b = ((r[i] & kInf) + kOne) & 0x80008000u;
                                    r[i] &= ~((b & 0x8000u ? 0xFFFFu : 0u) |
                                              (b & 0x80000000u ? 0xFFFF0000u : 0u));
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < DPI; ++i) {
                        uint32_t va[4];
                        if constexpr (F::kQ8) {
                            // rows of the tile: even dimensions, then odd ones
                            const uint32_t ua = r[2 * i] ^ 0x80808080u;
                            const uint32_t ub = r[2 * i + 1] ^ 0x80808080u;
                            va[0] = codes2<0x4240>(ua);
                            va[1] = codes2<0x4341>(ua);
                            va[2] = codes2<0x4240>(ub);
                            va[3] = codes2<0x4341>(ub);
                        } else {
                            va[0] = r[0], va[1] = r[2], va[2] = r[1], va[3] = r[3];
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if constexpr (F::kF32) {
#pragma unroll
                                for (int q = 0; q < NP; ++q)
                                    mma16816<F::kHalf>(acc[i][n], va, pb[kt][n][q][0],
                                                       pb[kt][n][q][1]);
                            } else {
                                mma16816<F::kHalf>(O[d2 + i][n], va, pb[kt][n][0][0],
                                                   pb[kt][n][0][1]);
                            }
                        }
                    }
                }
                if constexpr (F::kF32) {
#pragma unroll
                    for (int i = 0; i < DPI; ++i)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float(&o)[4] = O[d2 + i][n];
                            o[0] = fmaf(o[0], al[n][0], acc[i][n][0]);
                            o[1] = fmaf(o[1], al[n][1], acc[i][n][1]);
                            o[2] = fmaf(o[2], al[n][0], acc[i][n][2]);
                            o[3] = fmaf(o[3], al[n][1], acc[i][n][3]);
                        }
                }
            }
            if constexpr (!F::kQ8) {
                if (odd) {
                    const uint8_t* vt = smem + F::OFF_RING + s * F::SLOT + KS * F::ROWB;
                    for (int kk = 0; kk < KS; ++kk) {
                        const bool on = (flag >> (kk / (KS / 2))) & 1;
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float x = load1(reinterpret_cast<const OT*>(
                                                          vt + chunk_off<F>(kk, 2 * d + h)) + g);
                                if (fabsf(x) < INFINITY) continue;
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        if (on && vis(key0 + kk, pos[n][e]))
                                            O[d][n][2 * h + e] += x;
                            }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        it += m;
        __syncwarp();
        if (MW == 1 && lane == 0) mbar_arrive(&q_empty[buf]);

        // ---- join the groups, halving their number per round
        if constexpr (F::kQ8) {
            // (sums stand relative to 2^(M + E) from here on)
#pragma unroll
            for (int n = 0; n < NT; ++n) M[n][0] += E[n][0], M[n][1] += E[n][1];
        }
        if constexpr (NG > 1) {
            constexpr int PER = F::PER;
            named_barrier(1, F::NW * 32);  // the last tile's join has been read
            for (int h = NG / 2; h >= 1; h >>= 1) {
                // rounds after the first write where this warp has read
                if (grp >= h && grp < 2 * h) {
                    float* x = sX + ((h == NG / 2 ? grp - h : grp) * PER) * 32 + lane;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                x[((n * DT + d) * 4 + i) * 32] = O[d][n][i];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            x[(4 * NT * DT + 4 * n + e) * 32] = M[n][e];
                            x[(4 * NT * DT + 4 * n + 2 + e) * 32] = l[n][e];
                        }
                    }
                }
                named_barrier(1, F::NW * 32);
                if (grp < h) {
                    const float* x = sX + ((h == NG / 2 ? grp : grp + h) * PER) * 32 + lane;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float fa[2], fb[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float B = x[(4 * NT * DT + 4 * n + e) * 32];
                            const float N = fmaxf(M[n][e], B), R = N == -INFINITY ? 0.f : N;
                            fa[e] = ex2(M[n][e] - R);
                            fb[e] = ex2(B - R);
                            M[n][e] = N;
                            l[n][e] = l[n][e] * fa[e] +
                                      x[(4 * NT * DT + 4 * n + 2 + e) * 32] * fb[e];
                        }
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                O[d][n][i] = O[d][n][i] * fa[i & 1] +
                                             x[((n * DT + d) * 4 + i) * 32] * fb[i & 1];
                    }
                }
            }
        }

        // ---- store: the finished rows, or this piece of them
        if (grp == 0 && wrows > 0) {
            const bool piece = cut_l || cut_r;
            const int64_t pslot = 2 * (int64_t)blockIdx.x + (cut_l ? 0 : 1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float sum = l[n][e];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    const int r = 8 * n + 2 * t4 + e;
                    if (r >= wrows) continue;
                    // a row that sees nothing has no maximum and gives zeros; one
                    // whose scores are all -inf has no weights either: NaN
                    if (M[n][e] == -INFINITY && sum == 0.f &&
                        sees_any<F::KS>(a, p, tw, m, pos[n][e]))
                        M[n][e] = -FLT_MAX;
                    if (piece) {
                        const int64_t row = pslot * TR + mt * F::WR + r;
                        if (g == 0) a.stat[row] = make_float2(M[n][e], sum);
                        float* o = a.part + row * HD;
#pragma unroll
                        for (int d = 0; d < DT; ++d) {
                            if constexpr (F::kQ8) {
                                *reinterpret_cast<float2*>(o + 16 * d + 2 * g) =
                                    make_float2(O[d][n][e], O[d][n][2 + e]);
                            } else {
                                o[16 * d + g] = O[d][n][e];
                                o[16 * d + 8 + g] = O[d][n][2 + e];
                            }
                        }
                    } else {
                        const float inv = M[n][e] == -INFINITY && sum == 0.f ? 0.f : 1.f / sum;
                        const RowRef rr(a, p, pr + r);
                        X* o = static_cast<X*>(a.out) + (int64_t)(p.row + rr.tok) * a.out_stride +
                               (int64_t)rr.head * HD;
#pragma unroll
                        for (int d = 0; d < DT; ++d) {
                            if constexpr (F::kQ8) {
                                store1<X>(o + 16 * d + 2 * g, O[d][n][e] * inv);
                                store1<X>(o + 16 * d + 2 * g + 1, O[d][n][2 + e] * inv);
                            } else {
                                store1<X>(o + 16 * d + g, O[d][n][e] * inv);
                                store1<X>(o + 16 * d + 8 + g, O[d][n][2 + e] * inv);
                            }
                        }
                    }
                }
        }
        if (cut_r && !cut_l) {
            owner = true;
            if (threadIdx.x == 0) {
                // the tile's last unit says which CTA holds its last piece
                const int64_t end = u0 + (total - left) + tw.count;
                CutTile ct;
                ct.pieces = (int)((end - 1) / L - blockIdx.x) + 1;
                ct.row = p.row;
                ct.kvh = p.kvh;
                ct.r0 = p.t * TR;
                ct.rows = min(rows - p.t * TR, TR);
                a.cut[blockIdx.x] = ct;
            }
        }
        left -= m;
        if (left > 0) P::next_tile(a, p);
    }
    if (!owner && threadIdx.x == 0) a.cut[blockIdx.x].pieces = 0;
    if (a.second) grid_dependency_wait();
}

// ------------------------------------------------------------- host side

// One set of tiles: the launch that takes the sequences of min_rows to
// max_rows packed rows, with its part of the workspace.
struct PagedSet {
    int G, TR;  // CTAs, packed rows per tile
};

struct PagedJob {
    PagedArgs a;
    const ftc_kv_pages* c;
    PagedSet set;
    int cls;  // 0: 8 rows a tile, 1: 16, 2: 64, 3: as many as fit
    cudaStream_t st;
};

int page_map(CUtensorMap* m, const void* base, const ftc_kv_pages* c, int key_step, bool plain8);

// Shortest range of chunks worth a CTA of its own, in rounds of its groups.
// (One sequence, 8-bit cache, us with 1, 2, 4 and 8 rounds: 2100 positions 18.1,
// 17.2, 17.9, 21.9; 517 positions 14.8, 15.2, 16.3, 21.2; 16000 all 28.)
constexpr int kLeastRounds = 2;

template <class F>
int launch_cfg(const PagedJob& j) {
    auto fn = paged_mma<F>;
    int rc = opt_in_smem(reinterpret_cast<const void*>(fn), F::SMEM,
                         "cudaFuncSetAttribute(paged_mma)");
    if (rc) return rc;
    CUtensorMap tk, tv;
    if ((rc = page_map(&tk, j.c->k, j.c, F::KS, false)) ||
        (rc = page_map(&tv, j.c->v, j.c, F::KS, false)))
        return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)j.set.G);
    cfg.blockDim = dim3(F::THREADS);
    cfg.dynamicSmemBytes = F::SMEM;
    cfg.stream = j.st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, tk, tv, j.a, kLeastRounds * F::NG);
    if (e != cudaSuccess) return cuda_error(e, "launch paged_mma");
    return FTC_OK;
}

template <class F>
PagedSet geom_cfg() {
    return {F::OCC * device_sms(), F::TR};
}

}  // namespace paged
}  // namespace ftc
