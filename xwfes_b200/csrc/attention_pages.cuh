// attention_pages.cuh -- the paged attention on warp-level tensor cores
// (mma.sync m16n8k16, fp32 accumulators): decode, a few new tokens, and every
// fp32 query.
//
//   out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q.k_j - M),  c = scale log2(e)
// in one pass over the keys (running maximum M, running sum, the accumulator
// rescaled when M grows).  A CTA is NW consumer warps and one producer warp.
// The producer brings key chunks (KS positions of K and V, one box per page
// and 128 bytes of head_dim, swizzled by TMA so that the matrix loads are free
// of bank conflicts) into a ring of slots; a chunk of a page that is not
// mapped is fetched out of bounds, which fills zeros.  A slot belongs to one
// group of MW warps, warp i of the group taking packed rows 16 i .. 16 i + 15;
// the groups take slots in turn, each with a softmax state of its own, and
// meet only at a tile's end.  So decode (MW = 1, 16 packed rows) has 4
// independent warps on one tile's keys, and chunks (MW = 4, 8) read each key
// once for 64 or 128 rows.
//
// Decode is bound by HBM: 2 (head_dim bytes) a position and KV head.  Why
// matrix instructions for it: with 4 query heads on a KV head the CUDA cores
// would need 8 multiply-adds a byte of cache, 1.5 times what they have at HBM
// speed, and the 8-bit decode on top; as 16-row tiles the same work is a
// fifth of the tensor rate.
//
// Types.  Operands are f16 for f16 and 8-bit caches, bf16 for bf16 caches; the
// 8-bit codes are exact in f16 (byte -> 1024 + code + 128 in the mantissa, one
// subtraction), their scales stay outside: K's multiplies the score, V's the
// weight.  q: a 16-bit q is one operand; a bf16 q over an 8-bit cache becomes
// f16 with a power-of-two scale per row; an fp32 q is 2 f16 pieces (scaled the
// same way, 2^-22 kept) or 3 bf16 pieces.  Weights: fp32 q also splits them
// (2 or 3 pieces), else they are rounded once to the operand type, 2^14 up in
// f16 (and V's scale relative to its running maximum) so that weights 2^-38 of
// the largest still count.  With fp32 q the matrix unit's own accumulation,
// which truncates, is kept to short chains that fp32 adds join.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "paged_plan.cuh"

namespace ftc {
namespace paged {

template <typename X, typename C, int HD_, int MW_, int NW_>
struct Cfg {
    static constexpr int HD = HD_, MW = MW_, NW = NW_;
    static constexpr int NG = NW / MW;  // warp groups
    static constexpr int TR = 16 * MW;  // packed rows per tile
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
    static constexpr int QB = MW * NP * (HD / 16) * 512;
    static constexpr int XB = NG > 1 ? (NG / 2) * MW * 32 * (HD / 2 + 4) * 4 : 0;
    static constexpr int kFixed = 1024 /* alignment */ + QB + XB + 1024 /* barriers, flags */;
    static constexpr int SLOT_ALL = SLOT + (kQ8 ? 2 * KS * 4 : 0);
    // two CTAs per SM where each still has slots in flight beside the held
    // ones, and where 168 registers hold the accumulator (head_dim < 256)
    static constexpr int OCC = NW <= 4 && HD < 256 && (112 * 1024 - kFixed) / SLOT_ALL >= NG + 4 ? 2 : 1;
    static constexpr int kFit = ((OCC == 2 ? 112 : 224) * 1024 - kFixed) / SLOT_ALL;
    static constexpr int NSLOT = kFit < 24 ? kFit : 24;
    static_assert(NSLOT >= NG + 1, "ring holds every group's slot and one in flight");
    static constexpr int OFF_RING = 0;
    static constexpr int OFF_SCALE = OFF_RING + NSLOT * SLOT;
    static constexpr int OFF_Q = OFF_SCALE + (kQ8 ? NSLOT * 2 * KS * 4 : 0);
    static constexpr int OFF_X = OFF_Q + QB;
    static constexpr int OFF_BAR = OFF_X + XB;
    static constexpr int SMEM = OFF_BAR + 1024 + 1024;
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

template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    if constexpr (kHalf)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
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
    if (*dead) return false;
    if (mbar_wait_warp(bar, parity)) return true;
    *dead = 1;
    return false;
}

struct Vis {
    int window, n_sink;
    __device__ __forceinline__ bool operator()(int key, int p) const {
        return key <= p && (window == 0 || p - key < window || key < n_sink);
    }
};

template <typename X, class F>
__device__ __forceinline__ void store4(const PagedArgs& a, float4 v, int64_t off) {
    X* o = static_cast<X*>(a.out) + off;
    if constexpr (sizeof(X) == 4) *reinterpret_cast<float4*>(o) = v;
    else *reinterpret_cast<uint2*>(o) = make_uint2(pack<X>(v.x, v.y), pack<X>(v.z, v.w));
}

template <typename X, typename C, class F>
__global__ void __launch_bounds__(F::THREADS, F::OCC)
paged_mma(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
          const __grid_constant__ PagedArgs a, int least) {
    constexpr int HD = F::HD, MW = F::MW, NG = F::NG, NP = F::NP, KS = F::KS, TR = F::TR;
    constexpr int NT = HD / 8;  // output tiles of 8 dimensions
    using OT = typename F::OT;
    using P = Plan<TR, KS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* sScale = reinterpret_cast<float*>(smem + F::OFF_SCALE);
    uint4* sQ = reinterpret_cast<uint4*>(smem + F::OFF_Q);
    float* sX = reinterpret_cast<float*>(smem + F::OFF_X);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + F::OFF_BAR);
    uint64_t* empty = full + F::NSLOT;
    volatile int* dead = reinterpret_cast<volatile int*>(empty + F::NSLOT);
    int* sFlag = const_cast<int*>(dead) + 4;                       // [NSLOT] mapped halves
    PlanPos* sPos = reinterpret_cast<PlanPos*>(sFlag + 32);
    int64_t* sPre = reinterpret_cast<int64_t*>(smem + F::OFF_RING);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < F::NSLOT; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], MW);
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
    const int64_t W = P::scan(a, sPre);
    const int64_t L = plan_share(W, (int)gridDim.x, NG, least);
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

    if (warp == F::NW) {
        // -------------------------------------------------------- producer
        if (lane == 0) {
            prefetch_tensormap(&tk);
            prefetch_tensormap(&tv);
        }
        const int box = min(a.b.page_size, KS);  // rows of a box
        const int halves = KS / box;             // boxes over the keys (1 or 2)
        uint32_t it = 0;
        for (int left = total; left > 0;) {
            const TileWork<TR, KS> tw(a, p.n, p.len, p.t);
            const int m = min(tw.count - p.i, left);
            for (int j0 = 0; j0 < m; j0 += 32) {
                int key = 0, id0 = -1, id1 = -1;
                if (j0 + lane < m) {
                    key = tw.key0(p.i + j0 + lane);
                    id0 = page_of(a.b, p.s, key);
                    if (halves == 2) id1 = page_of(a.b, p.s, key + box);
                }
                const int jn = min(32, m - j0);
                for (int j = 0; j < jn; ++j, ++it) {
                    const int k0 = __shfl_sync(0xffffffffu, key, j);
                    const int ia = __shfl_sync(0xffffffffu, id0, j);
                    const int ib = __shfl_sync(0xffffffffu, id1, j);
                    const int s = it % F::NSLOT;
                    if (!ring_wait(&empty[s], ((it / F::NSLOT) & 1) ^ 1, dead)) break;
                    const int mapped = (ia >= 0 ? 1 : 0) + (ib >= 0 ? 1 : 0);
                    if (lane == 0) {
                        sFlag[s] = halves == 2 ? (ia >= 0 ? 1 : 0) | (ib >= 0 ? 2 : 0)
                                               : (ia >= 0 ? 3 : 0);
                        mbar_arrive_expect_tx(&full[s],
                                              F::SLOT + (F::kQ8 ? mapped * 2 * box * 4 : 0));
                    }
                    __syncwarp();
                    // lane l: tensor (K, V), 128-byte column, page half
                    const int kv = lane & 1, col = (lane >> 1) % F::NBOX;
                    const int half = (lane >> 1) / F::NBOX;
                    const int id = half ? ib : ia;
                    const int y = p.kvh * a.b.page_size + (k0 & (a.b.page_size - 1));
                    if (half < halves) {
                        uint8_t* dst = smem + F::OFF_RING + s * F::SLOT + kv * (KS * F::ROWB) +
                                       col * (KS * F::BOXB) + half * box * F::BOXB;
                        // past the last page: zeros
                        tma_box(dst, kv ? &tv : &tk, col * (F::BOXB / (int)sizeof(C)), y,
                                id < 0 ? a.b.n_pages : id, &full[s]);
                        if (F::kQ8 && col == 0 && id >= 0)
                            bulk_copy(sScale + (s * 2 + kv) * KS + half * box,
                                      (kv ? a.vs : a.ks) + (int64_t)id * a.b.scale_stride + y,
                                      box * 4, &full[s]);
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
    uint32_t it = 0;
    bool owner = false;
    for (int left = total; left > 0;) {
        const TileWork<TR, KS> tw(a, p.n, p.len, p.t);
        const int m = min(tw.count - p.i, left);
        const bool cut_l = p.i > 0, cut_r = p.i + m < tw.count;
        const int rows = p.n * a.gqa;
        const int pr = p.t * TR + mt * 16;  // the warp's first packed row
        const int wrows = min(rows - pr, 16);  // <= 0: none
        const bool two = wrows > 8;

        // q: operand pieces to shared memory, row scales kept
        float c0 = a.c, c1 = a.c;
        int pos0 = -1, pos1 = -1;
        int64_t off0 = 0, off1 = 0;  // of the rows in out
        {
            const int ra = pr + g, rb = ra + 8;
            const bool va = ra < rows, vb = rb < rows;
            const int ta = ra / a.gqa, tb = rb / a.gqa;
            const int ha = p.kvh * a.gqa + ra - ta * a.gqa, hb = p.kvh * a.gqa + rb - tb * a.gqa;
            if (va) pos0 = p.len - p.n + ta;
            if (vb) pos1 = p.len - p.n + tb;
            off0 = (int64_t)(p.row + ta) * a.out_stride + (int64_t)ha * HD;
            off1 = (int64_t)(p.row + tb) * a.out_stride + (int64_t)hb * HD;
            const X* qa = static_cast<const X*>(a.q) + (int64_t)(p.row + ta) * a.q_stride +
                          (int64_t)ha * HD;
            const X* qb = static_cast<const X*>(a.q) + (int64_t)(p.row + tb) * a.q_stride +
                          (int64_t)hb * HD;
            // the order of the 16 k of an instruction is free: with 8-bit
            // codes a lane's four are neighbours (one word of the cache row)
            const int kl = F::kQ8 ? 4 * t4 : 2 * t4, kh = F::kQ8 ? 4 * t4 + 2 : 2 * t4 + 8;
            int e0 = 0, e1 = 0;
            float fa0 = 1.f, fb0 = 1.f, fa1 = 1.f, fb1 = 1.f;
            if constexpr (F::kRowScale) {
                uint32_t m0 = 0, m1 = 0;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) {
                    if (va) {
                        const float2 x = load2(qa + 16 * i + kl), y = load2(qa + 16 * i + kh);
                        m0 = max(max(m0, __float_as_uint(fabsf(x.x))),
                                 max(__float_as_uint(fabsf(x.y)),
                                     max(__float_as_uint(fabsf(y.x)), __float_as_uint(fabsf(y.y)))));
                    }
                    if (vb) {
                        const float2 x = load2(qb + 16 * i + kl), y = load2(qb + 16 * i + kh);
                        m1 = max(max(m1, __float_as_uint(fabsf(x.x))),
                                 max(__float_as_uint(fabsf(x.y)),
                                     max(__float_as_uint(fabsf(y.x)), __float_as_uint(fabsf(y.y)))));
                    }
                }
#pragma unroll
                for (int o = 1; o <= 2; o <<= 1) {
                    m0 = max(m0, __shfl_xor_sync(0xffffffffu, m0, o));
                    m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, o));
                }
                // the row's largest value lands in [2^14, 2^15)
                if (m0 > 0 && m0 < 0x7F800000u) e0 = (int)(m0 >> 23) - 141;
                if (m1 > 0 && m1 < 0x7F800000u) e1 = (int)(m1 >> 23) - 141;
                fa0 = pow2(-e0 / 2), fb0 = pow2(-e0 - -e0 / 2);
                fa1 = pow2(-e1 / 2), fb1 = pow2(-e1 - -e1 / 2);
                c0 = fmaxf(a.c * pow2(e0 / 2) * pow2(e0 - e0 / 2), 1e-38f);
                c1 = fmaxf(a.c * pow2(e1 / 2) * pow2(e1 - e1 / 2), 1e-38f);
            }
            if (grp == 0) {
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) {
                    float2 x0 = make_float2(0.f, 0.f), y0 = x0, x1 = x0, y1 = x0;
                    if (va) x0 = load2(qa + 16 * i + kl), y0 = load2(qa + 16 * i + kh);
                    if (vb) x1 = load2(qb + 16 * i + kl), y1 = load2(qb + 16 * i + kh);
                    if constexpr (F::kRowScale) {  // 2^-e as two factors in range
                        x0.x = x0.x * fa0 * fb0, x0.y = x0.y * fa0 * fb0;
                        y0.x = y0.x * fa0 * fb0, y0.y = y0.y * fa0 * fb0;
                        x1.x = x1.x * fa1 * fb1, x1.y = x1.y * fa1 * fb1;
                        y1.x = y1.x * fa1 * fb1, y1.y = y1.y * fa1 * fb1;
                    }
                    uint32_t r0[NP], r1[NP], r2[NP], r3[NP];
                    split<OT, NP>(x0.x, x0.y, r0);
                    split<OT, NP>(x1.x, x1.y, r1);
                    split<OT, NP>(y0.x, y0.y, r2);
                    split<OT, NP>(y1.x, y1.y, r3);
#pragma unroll
                    for (int n = 0; n < NP; ++n)
                        sQ[((mt * NP + n) * (HD / 16) + i) * 32 + lane] =
                            make_uint4(r0[n], r1[n], r2[n], r3[n]);
                }
            }
        }
        if constexpr (NG > 1) named_barrier(1, F::NW * 32);
        else __syncwarp();
        // rows of this warp for the mask tests
        const int p_lo = p.len - p.n + pr / a.gqa;
        const int p_hi = wrows > 0 ? p.len - p.n + (pr + wrows - 1) / a.gqa : -1;

        float O[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.f;
        float M0 = -INFINITY, M1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        int E = -126;  // 8-bit V: the accumulator's unit is 2^E

        for (int j = grp; j < m; j += NG) {
            const uint32_t k = it + j;
            const int s = k % F::NSLOT;
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

            // ---- scores: KS / 8 tiles of 8 keys
            // (k outside, so that a piece of q is read once for all of them)
            float S[KS / 8][4], lo[F::kF32 ? KS / 8 : 1][4];
#pragma unroll
            for (int n = 0; n < KS / 8; ++n) {
                S[n][0] = S[n][1] = S[n][2] = S[n][3] = 0.f;
                if constexpr (F::kF32) lo[n][0] = lo[n][1] = lo[n][2] = lo[n][3] = 0.f;
            }
#pragma unroll
            for (int c4 = 0; c4 < F::ROWB / 64; ++c4) {
                constexpr int STEPS = F::kQ8 ? 4 : 2;  // k-steps in four chunks
                uint32_t r[KS / 8][4];
#pragma unroll
                for (int n = 0; n < KS / 8; ++n)
                    ldsm4(r[n], ks_addr + chunk_off<F>(8 * n + (lane & 7), 4 * c4 + (lane >> 3)));
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    const uint4* qf = sQ + (mt * NP * (HD / 16) + c4 * STEPS + st) * 32 + lane;
                    uint4 qv[NP];
#pragma unroll
                    for (int q = 0; q < NP; ++q) qv[q] = qf[q * (HD / 16) * 32];
#pragma unroll
                    for (int n = 0; n < KS / 8; ++n) {
                        uint32_t b0, b1;
                        if constexpr (F::kQ8) {
                            const uint32_t u = r[n][st] ^ 0x80808080u;
                            b0 = codes2<0x4140>(u);
                            b1 = codes2<0x4342>(u);
                        } else {
                            b0 = r[n][2 * st];
                            b1 = r[n][2 * st + 1];
                        }
                        mma16816<F::kHalf>(S[n], qv[0], b0, b1);
#pragma unroll
                        for (int q = 1; q < NP; ++q) mma16816<F::kHalf>(lo[n], qv[q], b0, b1);
                    }
                }
            }
            if constexpr (F::kF32) {
#pragma unroll
                for (int n = 0; n < KS / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[n][i] += lo[n][i];
            }

            // ---- the 8-bit scales of this lane's keys
            float vsc[KS / 8][2];
            float mul = 1.f;  // what E's growth does to the accumulator
            if constexpr (F::kQ8) {
                const float* ksc = sScale + (s * 2) * KS;
                float top = 0.f;
#pragma unroll
                for (int n = 0; n < KS / 8; ++n) {
                    const float2 kk = *reinterpret_cast<const float2*>(ksc + 8 * n + 2 * t4);
                    const float2 vv = *reinterpret_cast<const float2*>(ksc + KS + 8 * n + 2 * t4);
                    S[n][0] *= kk.x, S[n][2] *= kk.x;
                    S[n][1] *= kk.y, S[n][3] *= kk.y;
                    vsc[n][0] = vv.x, vsc[n][1] = vv.y;
                    const int key = key0 + 8 * n + 2 * t4;
                    const bool on = whole || ((flag >> (8 * n / (KS / 2))) & 1);
                    if (on && key <= p_hi) top = fmaxf(top, fabsf(vv.x));
                    if (on && key + 1 <= p_hi) top = fmaxf(top, fabsf(vv.y));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int Ek = min(max((int)(__float_as_uint(top) >> 23) - 126, -126), 126);
                if (Ek > E) {
                    mul = E - Ek < -126 ? 0.f : pow2(E - Ek);
                    E = Ek;
                }
                const float f = pow2(-E);
#pragma unroll
                for (int n = 0; n < KS / 8; ++n) vsc[n][0] *= f, vsc[n][1] *= f;
            }

            // ---- softmax: new maxima, weights (2^14 up in f16), sums
            if (!whole) {
#pragma unroll
                for (int n = 0; n < KS / 8; ++n) {
                    const bool on = (flag >> (8 * n / (KS / 2))) & 1;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = key0 + 8 * n + 2 * t4 + i;
                        // a hidden score is marked by a NaN with this sign and payload
                        if (!(on && vis(key, pos0))) S[n][i] = __uint_as_float(0xFFFFDEADu);
                        if (!(on && vis(key, pos1))) S[n][2 + i] = __uint_as_float(0xFFFFDEADu);
                    }
                }
            }
            float m0 = -INFINITY, m1 = -INFINITY;  // fmaxf skips NaN
#pragma unroll
            for (int n = 0; n < KS / 8; ++n) {
                m0 = fmaxf(m0, fmaxf(S[n][0], S[n][1]));
                m1 = fmaxf(m1, fmaxf(S[n][2], S[n][3]));
            }
            m0 *= c0, m1 *= c1;
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) {
                m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
                m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
            }
            const float N0 = fmaxf(M0, m0), N1 = fmaxf(M1, m1);
            const float R0 = N0 == -INFINITY ? 0.f : N0, R1 = N1 == -INFINITY ? 0.f : N1;
            float al0 = ex2(M0 - R0), al1 = ex2(M1 - R1);  // 0 while M is -inf
            M0 = N0, M1 = N1;
            constexpr float kUp = F::kHalf ? 14.f : 0.f;
            const float D0 = kUp - R0, D1 = kUp - R1;
            float s0 = 0.f, s1 = 0.f;
            uint4 pf[KS / 16][NP];
#pragma unroll
            for (int n = 0; n < KS / 8; ++n) {
                float w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    w[i] = ex2(fmaf(S[n][i], c0, D0));
                    if (two) w[2 + i] = ex2(fmaf(S[n][2 + i], c1, D1));
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (__float_as_uint(S[n][i]) == 0xFFFFDEADu) w[i] = 0.f;
                }
                s0 += w[0] + w[1];
                s1 += w[2] + w[3];
                if constexpr (F::kQ8) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = w[i] == 0.f ? 0.f : w[i] * vsc[n][i & 1];
                }
                uint32_t x[NP], y[NP];
                split<OT, NP>(w[0], w[1], x);
                split<OT, NP>(w[2], w[3], y);
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    if (n & 1) pf[n / 2][q].z = x[q], pf[n / 2][q].w = y[q];
                    else pf[n / 2][q].x = x[q], pf[n / 2][q].y = y[q];
                }
            }
            l0 = fmaf(l0, al0, s0);
            l1 = fmaf(l1, al1, s1);
            if constexpr (F::kQ8) al0 *= mul, al1 *= mul;

            // ---- weighted V: 16-bit results tolerate the matrix unit's own
            // accumulation over all keys, fp32 ones get fresh sums per chunk
            bool odd = false;
            if constexpr (!F::kF32) {
                if (__any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        O[i][0] *= al0, O[i][1] *= al0;
                        O[i][2] *= al1, O[i][3] *= al1;
                    }
                }
            }
#pragma unroll
            for (int c2 = 0; c2 < F::ROWB / 32; ++c2) {
                constexpr int TPC = F::kQ8 ? 2 : 1;  // output tiles in a 16-byte chunk
                float acc[2 * TPC][4];
                if constexpr (F::kF32) {
#pragma unroll
                    for (int i = 0; i < 2 * TPC; ++i)
                        acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
                }
#pragma unroll
                for (int st = 0; st < KS / 16; ++st) {
                    uint32_t r[4];
                    ldsm4_t(r, vs_addr + chunk_off<F>(16 * st + (lane & 15), 2 * c2 + (lane >> 4)));
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
                    for (int i = 0; i < 2 * TPC; ++i) {
                        uint32_t b0, b1;
                        if constexpr (F::kQ8) {
                            const uint32_t ua = r[i & 2] ^ 0x80808080u;
                            const uint32_t ub = r[(i & 2) + 1] ^ 0x80808080u;
                            b0 = (i & 1) ? codes2<0x4341>(ua) : codes2<0x4240>(ua);
                            b1 = (i & 1) ? codes2<0x4341>(ub) : codes2<0x4240>(ub);
                        } else {
                            b0 = r[2 * i];
                            b1 = r[2 * i + 1];
                        }
                        if constexpr (F::kF32) {
#pragma unroll
                            for (int q = 0; q < NP; ++q)
                                mma16816<F::kHalf>(acc[i], pf[st][q], b0, b1);
                        } else {
                            mma16816<F::kHalf>(O[2 * TPC * c2 + i], pf[st][0], b0, b1);
                        }
                    }
                }
                if constexpr (F::kF32) {
#pragma unroll
                    for (int i = 0; i < 2 * TPC; ++i) {
                        float(&o)[4] = O[2 * TPC * c2 + i];
                        o[0] = fmaf(o[0], al0, acc[i][0]);
                        o[1] = fmaf(o[1], al0, acc[i][1]);
                        o[2] = fmaf(o[2], al1, acc[i][2]);
                        o[3] = fmaf(o[3], al1, acc[i][3]);
                    }
                }
            }
            if constexpr (!F::kQ8) {
                if (odd) {
                    const uint8_t* vt = smem + F::OFF_RING + s * F::SLOT + KS * F::ROWB;
                    for (int kk = 0; kk < KS; ++kk) {
                        const bool on = (flag >> (kk / (KS / 2))) & 1;
                        const bool see0 = on && vis(key0 + kk, pos0);
                        const bool see1 = on && vis(key0 + kk, pos1);
                        if (!__any_sync(0xffffffffu, see0 || see1)) continue;
#pragma unroll
                        for (int i = 0; i < NT; ++i) {
                            const float2 x = unpack<OT>(*reinterpret_cast<const uint32_t*>(
                                vt + chunk_off<F>(kk, i) + 4 * t4));
                            const bool bx = !(fabsf(x.x) < INFINITY), by = !(fabsf(x.y) < INFINITY);
                            if (bx && see0) O[i][0] += x.x;
                            if (by && see0) O[i][1] += x.y;
                            if (bx && see1) O[i][2] += x.x;
                            if (by && see1) O[i][3] += x.y;
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        it += m;

        // ---- join the groups, halving their number per round
        if constexpr (F::kQ8) {
            const float f = pow2(E);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) O[i][e] *= f;
        }
        if constexpr (NG > 1) {
            constexpr int PER = HD / 2 + 4;  // floats per lane
            for (int h = NG / 2; h >= 1; h >>= 1) {
                if (grp >= h && grp < 2 * h) {
                    // rounds after the first write where this warp has read
                    float* x = sX + (((h == NG / 2 ? grp - h : grp) * MW + mt) * PER) * 32 + lane;
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[(4 * i + e) * 32] = O[i][e];
                    x[(PER - 4) * 32] = M0;
                    x[(PER - 3) * 32] = M1;
                    x[(PER - 2) * 32] = l0;
                    x[(PER - 1) * 32] = l1;
                }
                named_barrier(1, F::NW * 32);
                if (grp < h) {
                    const float* x =
                        sX + (((h == NG / 2 ? grp : grp + h) * MW + mt) * PER) * 32 + lane;
                    const float B0 = x[(PER - 4) * 32], B1 = x[(PER - 3) * 32];
                    const float N0 = fmaxf(M0, B0), N1 = fmaxf(M1, B1);
                    const float R0 = N0 == -INFINITY ? 0.f : N0, R1 = N1 == -INFINITY ? 0.f : N1;
                    const float a0 = ex2(M0 - R0), a1 = ex2(M1 - R1);
                    const float b0 = ex2(B0 - R0), b1 = ex2(B1 - R1);
                    M0 = N0, M1 = N1;
                    l0 = l0 * a0 + x[(PER - 2) * 32] * b0;
                    l1 = l1 * a1 + x[(PER - 1) * 32] * b1;
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        O[i][0] = O[i][0] * a0 + x[(4 * i + 0) * 32] * b0;
                        O[i][1] = O[i][1] * a0 + x[(4 * i + 1) * 32] * b0;
                        O[i][2] = O[i][2] * a1 + x[(4 * i + 2) * 32] * b1;
                        O[i][3] = O[i][3] * a1 + x[(4 * i + 3) * 32] * b1;
                    }
                }
            }
        }

        // ---- store: the finished rows, or this piece of them
        if (grp == 0 && wrows > 0) {
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, o);
                l1 += __shfl_xor_sync(0xffffffffu, l1, o);
            }
            const bool piece = cut_l || cut_r;
            const int64_t pslot = 2 * (int64_t)blockIdx.x + (cut_l ? 0 : 1);
            float* part = a.part + (pslot * TR + mt * 16) * HD;
            float2* stat = a.stat + pslot * TR + mt * 16;
            const float i0 = piece ? 1.f : l0 == 0.f ? 0.f : 1.f / l0;
            const float i1 = piece ? 1.f : l1 == 0.f ? 0.f : 1.f / l1;
            if (piece && t4 == 0) {
                stat[g] = make_float2(M0, l0);
                stat[g + 8] = make_float2(M1, l1);
            }
            // a row that sees nothing has no sum: zeros, whatever O holds
            auto put = [&](int row, int64_t off, bool on, int d, float4 v) {
                if (piece) *reinterpret_cast<float4*>(part + row * HD + d) = v;
                else if (on) store4<X, F>(a, v, off + d);
            };
            const bool on0 = g < wrows, on1 = g + 8 < wrows;
            if constexpr (F::kQ8) {
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    const float(&x)[4] = O[2 * c];
                    const float(&y)[4] = O[2 * c + 1];
                    put(g, off0, on0, 16 * c + 4 * t4,
                        make_float4(x[0] * i0, y[0] * i0, x[1] * i0, y[1] * i0));
                    if (two)
                        put(g + 8, off1, on1, 16 * c + 4 * t4,
                            make_float4(x[2] * i1, y[2] * i1, x[3] * i1, y[3] * i1));
                }
            } else {
                // two lanes exchange halves so that each stores 16 bytes of fp32
                const bool up = t4 & 1;
#pragma unroll
                for (int c = 0; c < NT / 2; ++c) {
                    const float(&x)[4] = O[2 * c];
                    const float(&y)[4] = O[2 * c + 1];
                    // even lanes take tile 2c, odd lanes tile 2c + 1
                    const float sa = up ? x[0] : y[0], sb = up ? x[1] : y[1];
                    const float ra = __shfl_xor_sync(0xffffffffu, sa, 1);
                    const float rb = __shfl_xor_sync(0xffffffffu, sb, 1);
                    const float4 v = up ? make_float4(ra * i0, rb * i0, y[0] * i0, y[1] * i0)
                                        : make_float4(x[0] * i0, x[1] * i0, ra * i0, rb * i0);
                    const int d = 16 * c + (up ? 8 : 0) + 4 * (t4 >> 1);
                    put(g, off0, on0, d, v);
                    const float sc = up ? x[2] : y[2], sd = up ? x[3] : y[3];
                    const float rc = __shfl_xor_sync(0xffffffffu, sc, 1);
                    const float rd = __shfl_xor_sync(0xffffffffu, sd, 1);
                    const float4 w = up ? make_float4(rc * i1, rd * i1, y[2] * i1, y[3] * i1)
                                        : make_float4(x[2] * i1, x[3] * i1, rc * i1, rd * i1);
                    if (two) put(g + 8, off1, on1, d, w);
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
    int cls;  // 0: 16 rows a tile, 1: 64, 2: as many as fit
    cudaStream_t st;
};

int page_map(CUtensorMap* m, const void* base, const ftc_kv_pages* c, int key_step, bool plain8);

// Shortest range of chunks worth a CTA of its own, in rounds of its groups.
constexpr int kLeastRounds = 2;

template <typename X, typename C, int HD, int MW, int NW>
int launch_cfg(const PagedJob& j) {
    using F = Cfg<X, C, HD, MW, NW>;
    auto fn = paged_mma<X, C, F>;
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

template <typename X, typename C, int HD, int MW, int NW>
PagedSet geom_cfg() {
    using F = Cfg<X, C, HD, MW, NW>;
    return {F::OCC * device_sms(), F::TR};
}

}  // namespace paged
}  // namespace ftc
