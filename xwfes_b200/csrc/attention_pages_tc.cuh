// attention_pages_tc.cuh -- the paged attention of long chunks with 16-bit
// queries on the tcgen05 tensor cores.
//
// A tile is 256 packed rows, two stages of 128; its keys come 128 at a time.
// Per stage and key chunk, S = Q K^T (128 x 128) and O += P V (128 x head_dim)
// accumulate in tensor memory: S 128 columns, the weights P written over it as
// 16-bit A operand, O head_dim columns.  One warp issues all MMAs, per chunk u
// and stage PV(u), then S(u + 1): the tensor cores work on one stage while the
// other's softmax runs, and PV(u) begins when half of its weights are there.
// MMAs of one warp run in order, which makes S(u + 1) after PV(u) safe on the
// same columns, and lets the softmax warps rescale O without a barrier of its
// own: S(u) has arrived, so PV(u - 1) is done, and PV(u) waits for this P.
// Rescaling is lazy: the reference maximum only moves when a score passes it by
// 2^8, which f16 weights leave room for (they sit 2^7 up).
//
// Warps: 0 brings K and V by TMA, one box per page (V as it lies in the cache:
// positions by head_dim, the MN-major B operand of PV); 1 issues MMAs; 4-7 and
// 8-11 are the softmax of the two stages, a thread per row, its 128 scores in
// registers (these warps get 216, the others 72); 2 and 3 turn 8-bit codes
// into f16 tiles, and in chunks where some row's mask hides something they take
// V elements that are not finite out (0 x inf would reach every row), which the
// rows that see them get back before the epilogue; between tiles each fetches the q rows
// of a stage.  8-bit scales stay in fp32: K's multiplies S, V's multiplies P,
// relative to the running maximum 2^E of those that the row sees (in a chunk
// that some row does not see whole, each thread looks over its own row's).
//
// What bounds it: per chunk and stage pair the tensor cores need 2048 clocks
// at head_dim 128 and the exponentials, 16 a clock, as many; both are busy for
// 53 % of the time (2048 bf16 rows of 32 heads on 16384 positions: 488 us, 1.06
// PFLOP/s).  A stage's softmax and its MMAs stand one after the other, two
// stages are what tensor memory holds at head_dim 128 (at 64, 128 columns and 90
// KB of shared memory are free and not used), its warps wait for tensor
// memory and barriers, and 44 to 72 bytes of registers spill.  Tried and not kept,
// with the time of the same call, then 520 us: two S
// buffers of 64 keys, scores a chunk early (820 us: what is done once per chunk
// weighs double); 16 warps, q fetched by two of their own (668 us); a part of
// the exponentials as polynomials on the FMA pipe (720 us: no one waits for the
// exponential unit); stage loops rolled (634 us); a shuffled, coalesced
// epilogue (552 us).
#pragma once

#include <climits>

#include "attention_pages.cuh"

namespace ftc {
namespace paged {

// Tiles of at most this many chunks are not cut when there is one for every
// CTA: a cut tile's second start and its join cost more than an uneven share
// (256 tiles: of 10 chunks 103 us cut, 90 whole; of 16, 107 and 94; of 18, 129
// and 113; of 5 to 32, 122 and 128).
constexpr int kWholeTile = 20;

template <typename X_, typename C_, int HD_>
struct TcCfg {
    using X = X_;
    using C = C_;
    static constexpr int HD = HD_, TR = 256, KS = 128;
    static constexpr bool kQ8 = sizeof(C) == 1;
    using OT = typename std::conditional<std::is_same<C, __nv_bfloat16>::value, __nv_bfloat16,
                                         __half>::type;
    static constexpr bool kHalf = std::is_same<OT, __half>::value;
    static constexpr bool kRowScale = kHalf && !std::is_same<X, __half>::value;
    static constexpr int SUB = KS * 128;           // 64 dimensions of 128 rows
    static constexpr int TILE = SUB * (HD / 64);   // K or V chunk or a stage's q, 16-bit
    // operand ring, K and V chunks in turn (16-bit: an even number of slots)
    static constexpr int NS = kQ8 ? (HD == 128 ? 3 : 4) : (HD == 128 ? 4 : 6);
    static constexpr int RAW = kQ8 ? KS * HD : 0;
    static constexpr int NR = 3;                   // slots of raw codes
    static constexpr int NSC = 3;
    static constexpr int NPREP = 2;
    static constexpr int OFF_RING = 0;
    static constexpr int OFF_Q = OFF_RING + NS * TILE;
    static constexpr int OFF_RAW = OFF_Q + 2 * TILE;
    static constexpr int OFF_SC = OFF_RAW + (kQ8 ? NR * RAW : 0);
    static constexpr int OFF_C = OFF_SC + NSC * (kQ8 ? 2 * KS * 4 : 0);
    static constexpr int OFF_BAR = OFF_C + (kRowScale ? 4 * TR * 4 : 0);
    static constexpr int SMEM = OFF_BAR + 1024 + 1024;
    static constexpr int THREADS = 384;
    // registers a thread: 384 x 168 at launch, then 128 x 72 + 256 x 216
    static constexpr int kRegsFew = 72, kRegsMany = 216;
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static_assert(NS * TILE >= Plan<TR, KS>::kSmem, "the plan's prefix sums fit in the ring");
};

__device__ __forceinline__ uint64_t f2u(uint32_t a, uint32_t b) {
    return (uint64_t)a | ((uint64_t)b << 32);
}
__device__ __forceinline__ void scale2f(float& a, float& b, uint64_t k) {
    const uint64_t v = f2mul(f2(a, b), k);
    a = f2lo(v);
    b = f2hi(v);
}
// (a, b) *= k
__device__ __forceinline__ void scale2(uint32_t& a, uint32_t& b, uint64_t k) {
    const uint64_t v = f2mul(f2u(a, b), k);
    a = (uint32_t)v;
    b = (uint32_t)(v >> 32);
}

// max of three, NaN if one of them is (an fmaxf chain would lose it).
__device__ __forceinline__ float max3n(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Bits below n, of 32.
__device__ __forceinline__ uint32_t low_bits(int n) {
    return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
}

// The 32 positions from key0 on that a row at `pos` sees, as bits; `mapped`:
// a bit per 16 of them.
__device__ __forceinline__ uint32_t seen_bits(const PagedArgs& a, int pos, int key0, int mapped) {
    const int hi = pos - key0 + 1;
    const uint32_t near = a.window > 0 ? ~low_bits(hi - a.window) | low_bits(a.n_sink - key0)
                                       : 0xFFFFFFFFu;
    return low_bits(hi) & near &
           ((mapped & 1 ? 0xFFFFu : 0u) | (mapped & 2 ? 0xFFFF0000u : 0u));
}

// Loads done: ties the registers to the wait, so that no use moves above it.
__device__ __forceinline__ void tmem_ld_done(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                   "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
        "%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
        "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

// Shared-memory descriptor of V as MN-major B operand, 128-byte swizzle: 64
// dimensions (128 bytes) of a position side by side, positions 128 bytes
// apart; leading offset = from one 64 dimensions to the next, stride offset =
// from 8 positions to the next 8.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(const void* tile, uint32_t lead) {
    const uint64_t addr = smem_u32(tile);
    uint64_t d = 0;
    d |= (addr >> 4) & 0x3FFFull;
    d |= (uint64_t)(lead >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= 1ull << 46;
    d |= 2ull << 61;
    return d;
}

// 1 in one lane of the warp, the same one every time.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(e));
    return e;
}

// A value every lane holds, as the compiler can know it.
__device__ __forceinline__ uint64_t uniform(uint64_t v) {
    const uint32_t lo = __shfl_sync(0xffffffffu, (uint32_t)v, 0);
    const uint32_t hi = __shfl_sync(0xffffffffu, (uint32_t)(v >> 32), 0);
    return (uint64_t)lo | ((uint64_t)hi << 32);
}

// The commit of sm100.cuh by the lane whose `lead` is 1.
__device__ __forceinline__ void commit_lead(uint64_t* bar, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
            smem_u32(bar)), "r"(lead)
        : "memory");
}

// Bits 15 and 31: the 16-bit value in that half is not finite (a full exponent
// field carries into the sign's place).
template <typename OT>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    constexpr bool half = std::is_same<OT, __half>::value;
    return ((w & (half ? 0x7C007C00u : 0x7F807F80u)) + (half ? 0x04000400u : 0x00800080u)) &
           0x80008000u;
}

// Whether every row of a tile sees all of the chunk from key0 on, mapped or not.
template <class F>
__device__ __forceinline__ bool covered(const PagedArgs& a, const TileWork<F::TR, F::KS>& tw,
                                        int key0) {
    return key0 + F::KS - 1 <= tw.p_first &&
           (a.window == 0 || tw.p_last - key0 < a.window || key0 + F::KS - 1 < a.n_sink);
}

// V elements that are not finite, of the positions that a row sees, added to
// 32 dimensions of its sum.  Chunks that all rows see whole went through the
// product as they are.
template <class F>
__device__ __noinline__ void add_odd(const PagedArgs& a, const PlanPos& p,
                                     const TileWork<F::TR, F::KS>& tw, int m, int pos, int d0,
                                     uint32_t (&s)[32]) {
    using OT = typename F::OT;
    for (int j = 0; j < m; ++j) {
        const int key0 = tw.key0(p.i + j);
        bool whole = covered<F>(a, tw, key0);
        for (int k = key0; whole && k < key0 + F::KS; k += a.b.page_size)
            whole = page_of(a.b, p.s, k) >= 0;
        if (whole) continue;
        int pg = -1;
        for (int key = key0; key < key0 + F::KS && key <= pos; ++key) {
            if (key % 16 == 0) pg = page_of(a.b, p.s, key);
            if (pg < 0 || !(a.window == 0 || pos - key < a.window || key < a.n_sink)) continue;
            const uint4* v = reinterpret_cast<const uint4*>(
                static_cast<const OT*>(a.v) + (int64_t)pg * a.b.page_stride +
                ((int64_t)p.kvh * a.b.page_size + (key & (a.b.page_size - 1))) * F::HD + d0);
            uint4 x4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x4[i] = v[i];
            const uint32_t* x = reinterpret_cast<const uint32_t*>(x4);
            uint32_t z = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) z |= not_finite<OT>(x[i]);
            if (z == 0) continue;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 y = unpack<OT>(x[i]);
                if (!(fabsf(y.x) < INFINITY))
                    s[2 * i] = __float_as_uint(__uint_as_float(s[2 * i]) + y.x);
                if (!(fabsf(y.y) < INFINITY))
                    s[2 * i + 1] = __float_as_uint(__uint_as_float(s[2 * i + 1]) + y.y);
            }
        }
    }
}

// One stage's q rows into the K-major operand tile by a warp, all of them in
// flight at once; where they become f16, a power of two per row brings the
// largest value to [2^14, 2^15) and goes to the score factor.
template <class F>
__device__ __forceinline__ void load_q(const PagedArgs& a, const PlanPos& p, int pr0, int rows,
                                       uint8_t* tile, float* sC) {
    using X = typename F::X;
    using OT = typename F::OT;
    constexpr int LPR = F::HD / 8;   // lanes to a row
    constexpr int RPI = 32 / LPR;    // rows a step
    const int lane = threadIdx.x & 31, c = lane % LPR;
    auto at = [&](int r) {
        return tile + (c / 8) * F::SUB + r * 128 + (((c % 8) ^ (r & 7)) << 4);
    };
#pragma unroll 2
    for (int r = lane / LPR; r < 128; r += RPI) {
        const int pr = pr0 + r;
        if (pr < rows) {
            const RowRef rr(a, p, pr);
            cp_async16(at(r), static_cast<const X*>(a.q) + (int64_t)(p.row + rr.tok) * a.q_stride +
                                  (int64_t)rr.head * F::HD + 8 * c);
        } else {
            *reinterpret_cast<uint4*>(at(r)) = make_uint4(0, 0, 0, 0);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if constexpr (F::kRowScale) {
        // (a lane converts the chunks that it brought)
#pragma unroll 4
        for (int r = lane / LPR; r < 128; r += RPI) {
            uint4 u = *reinterpret_cast<const uint4*>(at(r));
            uint32_t* x = reinterpret_cast<uint32_t*>(&u);
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                top = max(top, max((x[k] << 16) & 0x7FFF0000u, x[k] & 0x7FFF0000u));
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1)
                top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = top > 0 && top < 0x7F800000u ? (int)(top >> 23) - 141 : 0;
            const float fa = pow2(-e / 2), fb = pow2(-e - -e / 2);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 v = unpack<X>(x[k]);
                x[k] = pack<OT>(v.x * fa * fb, v.y * fa * fb);
            }
            if (c == 0) sC[r] = fmaxf(a.c * pow2(e / 2) * pow2(e - e / 2), 1e-38f);
            *reinterpret_cast<uint4*>(at(r)) = u;
        }
    }
}

template <int N>
__device__ __forceinline__ void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// The chunks of a CTA's share, one after another.
template <class F>
struct Walk {
    PlanPos p;
    int left, m, j;  // chunks to go, of this segment, done of it
    TileWork<F::TR, F::KS> tw;

    __device__ __forceinline__ Walk(const PagedArgs& a, const PlanPos& p0, int total)
        : p(p0), left(total), j(0), tw(a, p0.n, p0.len, p0.t) {
        m = min(tw.count - p.i, left);
    }
    __device__ __forceinline__ int key0() const { return tw.key0(p.i + j); }
    __device__ __forceinline__ bool first() const { return j == 0; }
    __device__ __forceinline__ void next(const PagedArgs& a) {
        --left;
        if (++j < m || left == 0) return;
        Plan<F::TR, F::KS>::next_tile(a, p);
        tw = TileWork<F::TR, F::KS>(a, p.n, p.len, p.t);
        m = min(tw.count, left);
        j = 0;
    }
};

template <class F>
__global__ void __launch_bounds__(F::THREADS, 1)
paged_tc(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
         const __grid_constant__ PagedArgs a, int least) {
    using X = typename F::X;
    using OT = typename F::OT;
    constexpr int HD = F::HD, TR = F::TR, KS = F::KS, NS = F::NS;
    using P = Plan<TR, KS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sRing = smem + F::OFF_RING;
    uint8_t* sQ = smem + F::OFF_Q;
    uint8_t* sRaw = smem + F::OFF_RAW;
    float* sScale = reinterpret_cast<float*>(smem + F::OFF_SC);  // [NSC][K, V][KS]
    float* sC = reinterpret_cast<float*>(smem + F::OFF_C);       // [4][2][128] score factors
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + F::OFF_BAR);  // 16-bit chunk landed
    uint64_t* ready = full + NS;            // converted; 16-bit: V looked over
    uint64_t* empty = ready + NS;           // its MMAs are done
    uint64_t* raw_full = empty + NS;
    uint64_t* raw_empty = raw_full + F::NR;
    uint64_t* sc_full = raw_empty + F::NR;  // flags and scales of a chunk
    uint64_t* sc_empty = sc_full + F::NSC;
    uint64_t* q_full = sc_empty + F::NSC;   // [stage] from here on
    uint64_t* q_empty = q_full + 2;
    uint64_t* s_full = q_empty + 2;
    uint64_t* p_half = s_full + 2;          // weights of keys 0-63
    uint64_t* p_full = p_half + 2;
    uint64_t* o_full = p_full + 2;
    uint64_t* o_empty = o_full + 2;
    uint64_t* drain = o_empty + 2;
    volatile int* dead = reinterpret_cast<volatile int*>(drain + 1);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(const_cast<int*>(dead) + 1);
    // [stage][4][2] the stage's segment (from 1 on) in which a preparing warp
    // took V elements out; no warp is four segments ahead of another
    volatile int* odd = dead + 2;
    int* sFlag = const_cast<int*>(dead) + 18;  // [NSC]
    PlanPos* sPos = reinterpret_cast<PlanPos*>(sFlag + F::NSC);
    static_assert((3 * NS + 2 * F::NR + 2 * F::NSC + 15) * 8 + 72 + 4 * F::NSC +
                          (int)sizeof(PlanPos) <= 1024, "control block");
    int64_t* sPre = reinterpret_cast<int64_t*>(sRing);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&ready[i], F::NPREP);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < F::NR; ++i) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], F::NPREP);
        }
        for (int i = 0; i < F::NSC; ++i) {
            mbar_init(&sc_full[i], 1);
            mbar_init(&sc_empty[i], 8 + F::NPREP);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_half[i], 4);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
            mbar_init(&o_empty[i], 4);
        }
        mbar_init(drain, 1);
        *dead = 0;
        for (int i = 0; i < 16; ++i) odd[i] = 0;
        mbar_fence_init();
    }
    if (!a.second) grid_dependency_wait();  // as paged_mma
    grid_launch_dependents();
    __syncthreads();

    int64_t tiles;
    int largest;
    const int64_t W = P::template scan<true>(a, sPre, tiles, largest);
    const int64_t L = plan_share(W, tiles, (int)gridDim.x, 1, least);
    int64_t u0 = min((int64_t)blockIdx.x * L, W), u1 = min(u0 + L, W);
    if (largest <= kWholeTile && tiles >= gridDim.x) {  // the ranges go to the nearest tile edges
        if (warp == 0) {
            const int64_t e0 = P::nearest_edge(a, sPre, u0, W);
            const int64_t e1 = P::nearest_edge(a, sPre, u1, W);
            if (lane == 0) sPre[kMaxSeqs + 3] = e0, sPre[kMaxSeqs + 4] = e1;
        }
        __syncthreads();
        u0 = sPre[kMaxSeqs + 3];
        u1 = sPre[kMaxSeqs + 4];
    }
    if (u0 >= u1) {
        if (threadIdx.x == 0) a.cut[blockIdx.x].pieces = 0;
        if (a.second) grid_dependency_wait();
        return;
    }
    const int total = (int)(u1 - u0);
    if (warp == 0) {
        const PlanPos p = P::locate(a, sPre, u0);
        if (lane == 0) *sPos = p;
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    fence_proxy_async_smem();  // the prefix sums are done with: the ring may be filled
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // columns: stage i's S (and P over it) at 128 i, its O at 256 + 128 i

    if (warp < 4) {
        regs_dec<F::kRegsFew>();
        Walk<F> wk(a, *sPos, total);
        if (warp == 0) {
            // ---------------------------------------------------- producer
            const int box = min(a.b.page_size, KS), boxes = KS / box;
            constexpr int NBOX = F::kQ8 ? 1 : HD / 64;  // 128-byte columns
            bool on = true;
            for (uint32_t u = 0; on && u < (uint32_t)total; ++u) {
                const int key0 = wk.key0();
                const int id = lane < boxes ? page_of(a.b, wk.p.s, key0 + lane * box) : -1;
                const int y = wk.p.kvh * a.b.page_size + (key0 & (a.b.page_size - 1));
                const unsigned mapped = __ballot_sync(0xffffffffu, id >= 0);
                const int ss = u % F::NSC;
                if (!ring_wait(&sc_empty[ss], ((u / F::NSC) & 1) ^ 1, dead)) break;
                if (lane == 0) {
                    int flag = 0;  // a bit per 16 positions
                    for (int b = 0; b < boxes; ++b)
                        if ((mapped >> b) & 1) flag |= ((1 << (box / 16)) - 1) << (b * box / 16);
                    sFlag[ss] = flag;
                    if constexpr (F::kQ8)
                        mbar_arrive_expect_tx(&sc_full[ss], __popc(mapped) * 2 * box * 4);
                    else mbar_arrive(&sc_full[ss]);
                }
                __syncwarp();
                if constexpr (F::kQ8) {
                    if (id >= 0) {
                        const int64_t src = (int64_t)id * a.b.scale_stride + y;
                        bulk_copy(sScale + (ss * 2 + 0) * KS + lane * box, a.ks + src, box * 4,
                                  &sc_full[ss]);
                        bulk_copy(sScale + (ss * 2 + 1) * KS + lane * box, a.vs + src, box * 4,
                                  &sc_full[ss]);
                    }
                }
#pragma unroll 1
                for (int v = 0; on && v < 2; ++v) {
                    const uint32_t t = 2 * u + v;
                    constexpr int N = F::kQ8 ? F::NR : NS;
                    constexpr int BYTES = F::kQ8 ? F::RAW : F::TILE;
                    const int s = t % N;
                    uint64_t* bar = F::kQ8 ? &raw_full[s] : &full[s];
                    on = ring_wait(F::kQ8 ? &raw_empty[s] : &empty[s], ((t / N) & 1) ^ 1, dead);
                    if (!on) break;
                    if (lane == 0) mbar_arrive_expect_tx(bar, BYTES);
                    __syncwarp();
                    const int b = lane / NBOX, col = lane % NBOX;
                    const int pg = __shfl_sync(0xffffffffu, id, b);
                    if (b < boxes)  // past the last page: zeros
                        tma_box((F::kQ8 ? sRaw : sRing) + s * BYTES + col * F::SUB +
                                    b * box * (F::kQ8 ? HD : 128),
                                v ? &tv : &tk, col * 64, y, pg < 0 ? a.b.n_pages : pg, bar);
                    __syncwarp();
                }
                wk.next(a);
            }
            if (*dead && lane == 0) {  // let issued copies land before the CTA leaves
                for (int par = 0; par < 2; ++par) {
                    for (int i = 0; i < F::NSC; ++i) mbar_wait(&sc_full[i], par);
                    for (int i = 0; i < (F::kQ8 ? F::NR : NS); ++i)
                        mbar_wait(F::kQ8 ? &raw_full[i] : &full[i], par);
                }
            }
        } else if (warp == 1) {
            // --------------------------------------------------------- MMA
            // The whole warp runs this; an elected lane issues a group of MMAs
            // in one branch (a predicate on each of them cost 4 %).
            constexpr uint32_t fmt = F::kHalf ? 0u : 1u;
            constexpr uint32_t id_s = idesc_f16(fmt, 128, KS);
            constexpr uint32_t id_o = idesc_f16(fmt, 128, HD) | (1u << 16);  // B is MN-major
            const uint32_t lead = elect_lane();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t dq0 = uniform(smem_desc_k_sw128(sQ));
            const uint64_t dk0 = uniform(smem_desc_k_sw128(sRing));
            const uint64_t dv0 = uniform(smem_desc_mn_sw128(sRing, F::SUB));
            uint32_t it = 0, np[2] = {0, 0}, no[2] = {0, 0};  // no: segments of a stage
            // slot of operand tile t once it is there, as descriptor offset
            auto operand = [&](uint32_t t, uint32_t& off) -> bool {
                const int s = t % NS;
                // ready of a 16-bit ring only counts V tiles (odd t, even NSL)
                uint64_t* b = F::kQ8 || (t & 1) ? &ready[s] : &full[s];
                if (!ring_wait(b, (t / NS) & 1, dead)) return false;
                tc_fence_after();
                off = __shfl_sync(0xffffffffu, (uint32_t)s * (F::TILE >> 4), 0);
                return true;
            };
            auto scores = [&](int i, uint32_t koff) {
                const uint64_t dq = dq0 + i * (F::TILE >> 4), dk = dk0 + koff;
                if (lead) {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const int o = (k / 4) * (F::SUB >> 4) + 2 * (k % 4);
                        umma_f16_ss(tm + i * 128, dq + o, dk + o, id_s, k != 0);
                    }
                    umma_commit(&s_full[i]);
                }
                __syncwarp();
            };
            PlanPos& p = wk.p;
            for (int left = total; left > 0;) {
                const TileWork<TR, KS> tw(a, p.n, p.len, p.t);
                const int m = min(tw.count - p.i, left);
                const int stages = p.n * a.gqa - p.t * TR > 128 ? 2 : 1;
                uint32_t koff, voff = 0;
                bool on = operand(2 * it, koff);
                for (int i = 0; on && i < stages; ++i) {
                    on = ring_wait(&q_full[i], no[i] & 1, dead);
                    if (!on) break;
                    tc_fence_after();
                    scores(i, koff);
                    if (m == 1) commit_lead(&q_empty[i], lead);
                }
                if (!on) break;
                commit_lead(&empty[2 * it % NS], lead);
                for (int j = 0; j < m; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (i >= stages) break;
                        on = ring_wait(&p_half[i], np[i] & 1, dead) &&
                             (i != 0 || operand(2 * (it + j) + 1, voff)) &&
                             (j != 0 || ring_wait(&o_empty[i], (no[i] & 1) ^ 1, dead));
                        if (!on) break;
                        tc_fence_after();
                        const uint64_t dv = dv0 + voff;
                        if (lead) {
#pragma unroll
                            for (int k = 0; k < KS / 32; ++k)
                                umma_f16_ts(tm + 256 + i * 128, tm + i * 128 + 8 * k, dv + k * 128,
                                            id_o, j != 0 || k != 0);
                        }
                        __syncwarp();
                        on = ring_wait(&p_full[i], np[i]++ & 1, dead);
                        if (!on) break;
                        tc_fence_after();
                        if (lead) {
#pragma unroll
                            for (int k = KS / 32; k < KS / 16; ++k)
                                umma_f16_ts(tm + 256 + i * 128, tm + i * 128 + 8 * k, dv + k * 128,
                                            id_o, 1);
                        }
                        __syncwarp();
                        if (j + 1 < m) {
                            on = i != 0 || operand(2 * (it + j + 1), koff);
                            if (!on) break;
                            scores(i, koff);
                            if (j + 2 == m) commit_lead(&q_empty[i], lead);
                        } else {
                            commit_lead(&o_full[i], lead);
                            ++no[i];
                        }
                    }
                    if (!on) break;
                    commit_lead(&empty[(2 * (it + j) + 1) % NS], lead);
                    if (j + 1 < m) commit_lead(&empty[2 * (it + j + 1) % NS], lead);
                }
                if (!on) break;
                it += m;
                left -= m;
                if (left > 0) P::next_tile(a, p);
            }
            if (*dead) {  // nothing of this CTA may be in flight when it leaves
                commit_lead(drain, lead);
                mbar_wait_warp(drain, 0);
            }
            __syncwarp();
        } else {
            // ------------------------------------------- operand preparation
            // and each of the two warps brings the q rows of a stage
            const int w = warp - 2;
            // segments, those with rows of this stage, and of the second
            uint32_t seg = 0, nq = 0, seg1 = 0;
            bool both = false;  // this one has
            for (uint32_t u = 0; u < (uint32_t)total; ++u) {
                if (wk.first()) {
                    const int pr0 = wk.p.t * TR + w * 128, rows = wk.p.n * a.gqa;
                    both = wk.p.t * TR + 128 < rows;
                    seg1 += both;
                    if (pr0 < rows) {
                        // (the last tile's scores are all done)
                        if (!ring_wait(&q_empty[w], (nq & 1) ^ 1, dead)) break;
                        ++nq;
                        load_q<F>(a, wk.p, pr0, rows, sQ + w * F::TILE,
                                  sC + ((seg & 3) * 2 + w) * 128);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&q_full[w]);
                    }
                    ++seg;
                }
                const int ss = u % F::NSC;
                ring_wait(&sc_full[ss], (u / F::NSC) & 1, dead);
                const int flag = sFlag[ss];
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_empty[ss]);
                if constexpr (F::kQ8) {
#pragma unroll 1
                    for (uint32_t t = 2 * u; t < 2 * u + 2; ++t) {
                        const int rs = t % F::NR, s = t % NS;
                        if (!ring_wait(&raw_full[rs], (t / F::NR) & 1, dead)) continue;
                        if (!ring_wait(&empty[s], ((t / NS) & 1) ^ 1, dead)) continue;
                        constexpr int LPR = HD / 16;       // lanes per row
                        constexpr int RPI = 32 / LPR;      // rows per step
                        constexpr int BATCH = 4;
                        const int c = lane % LPR;          // 16 codes of a row
                        const bool swap = (c >> 2) & 1;    // other bank half first
                        const uint8_t* src = sRaw + rs * F::RAW + 16 * c;
                        uint8_t* dst = sRing + s * F::TILE + (c >> 2) * F::SUB;
#pragma unroll 1
                        for (int r0 = w * (KS / F::NPREP) + lane / LPR;
                             r0 < (w + 1) * (KS / F::NPREP); r0 += BATCH * RPI) {
                            uint4 x[BATCH];
#pragma unroll
                            for (int i = 0; i < BATCH; ++i)
                                x[i] = *reinterpret_cast<const uint4*>(src + (r0 + i * RPI) * HD);
#pragma unroll
                            for (int i = 0; i < BATCH; ++i) {
                                const int r = r0 + i * RPI;
                                const uint32_t x0 = x[i].x ^ 0x80808080u;
                                const uint32_t x1 = x[i].y ^ 0x80808080u;
                                const uint32_t x2 = x[i].z ^ 0x80808080u;
                                const uint32_t x3 = x[i].w ^ 0x80808080u;
                                const uint4 lo = make_uint4(codes2<0x4140>(x0), codes2<0x4342>(x0),
                                                            codes2<0x4140>(x1), codes2<0x4342>(x1));
                                const uint4 hi = make_uint4(codes2<0x4140>(x2), codes2<0x4342>(x2),
                                                            codes2<0x4140>(x3), codes2<0x4342>(x3));
                                const int ch = 2 * (c & 3);
                                *reinterpret_cast<uint4*>(dst + r * 128 +
                                                          (((ch + swap) ^ (r & 7)) << 4)) =
                                    swap ? hi : lo;
                                *reinterpret_cast<uint4*>(dst + r * 128 +
                                                          (((ch + !swap) ^ (r & 7)) << 4)) =
                                    swap ? lo : hi;
                            }
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&ready[s]);
                            mbar_arrive(&raw_empty[rs]);
                        }
                    }
                } else {
                    const uint32_t t = 2 * u + 1;
                    const int s = t % NS;
                    const int key0 = wk.key0();
                    const bool whole = flag == 0xFF && covered<F>(a, wk.tw, key0);
                    if (ring_wait(&full[s], (t / NS) & 1, dead)) {
                        if (!whole) {
                            uint4* v = reinterpret_cast<uint4*>(sRing + s * F::TILE);
#pragma unroll 4
                            for (int q = w * 32 + lane; q < F::TILE / 16; q += 32 * F::NPREP) {
                                uint4 x4 = v[q];
                                uint32_t* x = reinterpret_cast<uint32_t*>(&x4);
                                uint32_t z = 0;
#pragma unroll
                                for (int i = 0; i < 4; ++i) z |= not_finite<OT>(x[i]);
                                if (z != 0) {
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const uint32_t b = not_finite<OT>(x[i]);
                                        x[i] &= ~((b & 0x8000u ? 0xFFFFu : 0u) |
                                                  (b & 0x80000000u ? 0xFFFF0000u : 0u));
                                    }
                                    v[q] = x4;
                                    odd[2 * (seg & 3) + w] = (int)seg;
                                    if (both) odd[8 + 2 * (seg1 & 3) + w] = (int)seg1;
                                }
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                        }
                        if (lane == 0) mbar_arrive(&ready[s]);
                    }
                }
                wk.next(a);
            }
        }
    } else {
        // --------------------------------------------------------- softmax
        regs_inc<F::kRegsMany>();
        const int st = warp >= 8 ? 1 : 0;
        const int r = (warp & 3) * 32 + lane;  // row of the stage, TMEM lane
        const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + st * 128;
        const uint32_t tO = tS + 256;
        uint32_t u = 0, sph = 0, no = 0, seg = 0;
        bool owner = false;
        PlanPos p = *sPos;
        for (int left = total; left > 0; ++seg) {
            const TileWork<TR, KS> tw(a, p.n, p.len, p.t);
            const int m = min(tw.count - p.i, left);
            const bool cut_l = p.i > 0, cut_r = p.i + m < tw.count;
            const int rows = p.n * a.gqa;
            const bool active = rows - p.t * TR > st * 128;
            const int pr = p.t * TR + st * 128 + r;  // packed row
            const bool live = pr < rows;
            const int tok = live ? pr / a.gqa : 0;
            const int h = p.kvh * a.gqa + pr - tok * a.gqa;
            const int pos = live ? p.len - p.n + tok : -1;
            float c = a.c;
            // positions of this warp's rows, for the mask tests
            const int wr = p.t * TR + st * 128 + (warp & 3) * 32;
            const int p_lo = p.len - p.n + min(wr, rows - 1) / a.gqa;
            const int p_hi = p.len - p.n + min(wr + 31, rows - 1) / a.gqa;
            constexpr float kUp = F::kHalf ? 7.f : 0.f;
            float M = -INFINITY;  // reference maximum (log2)
            int E = F::kQ8 ? -90 : 0;
            uint64_t l2 = 0;      // two partial sums of weights
            for (int j = 0; j < m; ++j, ++u) {
                const int ss = u % F::NSC;
                ring_wait(&sc_full[ss], (u / F::NSC) & 1, dead);
                if (active) {
                    const bool on = ring_wait(&s_full[st], sph & 1, dead);
                    ++sph;
                    if (!on) continue;
                    tc_fence_after();
                    uint32_t s[4][32];
#pragma unroll
                    for (int q = 0; q < 4; ++q) tmem_ld_32x32b_x32(tS + 32 * q, s[q]);
                    // (there are scores, so q and its factors were there; they
                    // stay for four segments, scores come a chunk early)
                    if (F::kRowScale && j == 0) c = sC[((seg & 3) * 2 + st) * 128 + r];
                    const int key0 = tw.key0(p.i + j);
                    const int flag = sFlag[ss];
                    const float4* ksc = reinterpret_cast<const float4*>(sScale + ss * 2 * KS);
                    const float4* vsc = ksc + KS / 4;
                    const bool whole = flag == 0xFF && key0 + KS - 1 <= p_lo &&
                                       (a.window == 0 || p_hi - key0 < a.window ||
                                        key0 + KS - 1 < a.n_sink);
#pragma unroll
                    for (int q = 0; q < 4; ++q) tmem_ld_done(s[q]);
                    // ---- the row's scores and their maximum
                    if constexpr (F::kQ8) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float4 k4 = ksc[i];
                            uint32_t* x = &s[i / 8][4 * (i % 8)];
                            scale2(x[0], x[1], f2(k4.x, k4.y));
                            scale2(x[2], x[3], f2(k4.z, k4.w));
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const uint32_t seen = seen_bits(a, pos, key0 + 32 * q, flag >> (2 * q));
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!((seen >> i) & 1)) s[q][i] = 0xFF800000u;
                        }
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            m4[q] = max3n(m4[q], __uint_as_float(s[q][i]),
                                          __uint_as_float(s[q][i + 1]));
                    const float mx = max3n(max3n(m4[0], m4[1], m4[2]), m4[3], m4[3]) * c;
                    int Et = E;
                    if constexpr (F::kQ8) {
                        // V's largest finite scale of the positions that this row sees
                        // (a hidden position may hold any): in a whole chunk of all
                        uint32_t top = 0;
                        auto take = [&](float v, bool on) {
                            const uint32_t b = __float_as_uint(fabsf(v));
                            if (on && b < 0x7F800000u) top = max(top, b);
                        };
                        if (whole) {
                            const float4 v4 = vsc[lane];
                            take(v4.x, true), take(v4.y, true);
                            take(v4.z, true), take(v4.w, true);
                            top = __reduce_max_sync(0xffffffffu, top);
                        } else {
#pragma unroll 1
                            for (int q = 0; q < 4; ++q) {
                                const uint32_t seen =
                                    seen_bits(a, pos, key0 + 32 * q, flag >> (2 * q));
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const float4 v4 = vsc[8 * q + i];
                                    take(v4.x, (seen >> (4 * i)) & 1);
                                    take(v4.y, (seen >> (4 * i)) & 2);
                                    take(v4.z, (seen >> (4 * i)) & 4);
                                    take(v4.w, (seen >> (4 * i)) & 8);
                                }
                            }
                        }
                        Et = max(E, min((int)(top >> 23) - 126, 126));
                    }
                    if (__any_sync(0xffffffffu, mx > M + 8.f || Et > E)) {
                        const float N = fmaxf(M, mx);
                        // (0 while nothing was seen; the accumulator is not set before j = 1)
                        const float f = M == -INFINITY ? 0.f : ex2(M - N + (float)(E - Et));
                        M = N;
                        E = Et;
                        l2 = f2mul(l2, f2(f, f));
                        if (j > 0) {
#pragma unroll 1
                            for (int q = 0; q < HD / 32; ++q) {
                                uint32_t o[32];
                                tmem_ld_32x32b_x32(tO + 32 * q, o);
                                tmem_ld_done(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tmem_st_x32(tO + 32 * q, o);
                            }
                        }
                    }
                    // ---- weights 2^(z - D), packed over the scores; a visible NaN
                    // makes all of them NaN
                    const float D = mx != mx ? mx
                                             : kUp - (M == -INFINITY ? 0.f : M) -
                                                   (float)(F::kQ8 ? E : 0);
                    const uint64_t c2 = f2(c, c), d2 = f2(D, D);
                    uint64_t lb = 0;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const uint64_t z0 = f2fma(f2u(s[q][i], s[q][i + 1]), c2, d2);
                            const uint64_t z1 = f2fma(f2u(s[q][i + 2], s[q][i + 3]), c2, d2);
                            float w0 = ex2(f2lo(z0)), w1 = ex2(f2hi(z0));
                            float w2 = ex2(f2lo(z1)), w3 = ex2(f2hi(z1));
                            l2 = f2add(l2, f2(w0, w1));
                            lb = f2add(lb, f2(w2, w3));
                            if constexpr (F::kQ8) {
                                const float4 v4 = vsc[8 * q + i / 4];
                                scale2f(w0, w1, f2(v4.x, v4.y));
                                scale2f(w2, w3, f2(v4.z, v4.w));
                            }
                            w[i / 2] = pack<OT>(w0, w1);
                            w[i / 2 + 1] = pack<OT>(w2, w3);
                        }
                        if (F::kQ8 && !whole) {  // a hidden position's scale may be anything
                            const uint32_t seen = seen_bits(a, pos, key0 + 32 * q, flag >> (2 * q));
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                w[i] &= ((seen >> (2 * i)) & 1 ? 0xFFFFu : 0u) |
                                        ((seen >> (2 * i)) & 2 ? 0xFFFF0000u : 0u);
                        }
                        tmem_st_x16(tS + 16 * q, w);
                        if (q & 1) {  // half of the keys: their products may begin
                            tmem_st_wait();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(q == 1 ? &p_half[st] : &p_full[st]);
                        }
                    }
                    l2 = f2add(l2, lb);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_empty[ss]);
            }

            // ---- the finished rows, or this piece of them
            if (active && ring_wait(&o_full[st], no++ & 1, dead)) {
                tc_fence_after();
                if constexpr (!F::kQ8) {
                    const volatile int* o2 = odd + 8 * st + 2 * (no & 3);
                    if (o2[0] == (int)no || o2[1] == (int)no) {
#pragma unroll 1
                        for (int q = 0; q < HD / 32; ++q) {
                            uint32_t s[32];
                            tmem_ld_32x32b_x32(tO + 32 * q, s);
                            tmem_ld_done(s);
                            if (live) add_odd<F>(a, p, tw, m, pos, 32 * q, s);
                            __syncwarp();
                            tmem_st_x32(tO + 32 * q, s);
                        }
                        tmem_st_wait();
                    }
                }
                const bool piece = cut_l || cut_r;
                const float l = f2lo(l2) + f2hi(l2);
                // nothing seen: zeros.  (Scores of -inf alone, and NaN: no zeros)
                if (M == -INFINITY && l == 0.f && sees_any<KS>(a, p, tw, m, pos)) M = -FLT_MAX;
                const float inv = piece ? 1.f : M == -INFINITY && l == l ? 0.f : 1.f / l;
                const int64_t pslot = 2 * (int64_t)blockIdx.x + (cut_l ? 0 : 1);
                float* part = a.part + (pslot * TR + st * 128 + r) * HD;
                if (piece)
                    a.stat[pslot * TR + st * 128 + r] =
                        make_float2(M + (float)(F::kQ8 ? E : 0), l);
                X* o = static_cast<X*>(a.out) + (int64_t)(p.row + tok) * a.out_stride +
                       (int64_t)h * HD;
#pragma unroll
                for (int q = 0; q < HD / 32; ++q) {
                    uint32_t s[32];
                    tmem_ld_32x32b_x32(tO + 32 * q, s);
                    tmem_ld_done(s);
                    if (piece) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4*>(part + 32 * q + i) =
                                make_uint4(s[i], s[i + 1], s[i + 2], s[i + 3]);
                    } else if (live) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t y[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                y[k] = pack<X>(__uint_as_float(s[i + 2 * k]) * inv,
                                               __uint_as_float(s[i + 2 * k + 1]) * inv);
                            *reinterpret_cast<uint4*>(o + 32 * q + i) =
                                make_uint4(y[0], y[1], y[2], y[3]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_empty[st]);
            }
            if (cut_r && !cut_l) {
                owner = true;
                if (threadIdx.x == 128) {
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
        if (!owner && threadIdx.x == 128) a.cut[blockIdx.x].pieces = 0;
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
    if (a.second) grid_dependency_wait();
}

template <typename X, typename C, int HD>
int launch_tc(const PagedJob& j) {
    using F = TcCfg<X, C, HD>;
    auto fn = paged_tc<F>;
    int rc = opt_in_smem(reinterpret_cast<const void*>(fn), F::SMEM,
                         "cudaFuncSetAttribute(paged_tc)");
    if (rc) return rc;
    CUtensorMap tk, tv;
    if ((rc = page_map(&tk, j.c->k, j.c, F::KS, true)) ||
        (rc = page_map(&tv, j.c->v, j.c, F::KS, true)))
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, tk, tv, j.a, 2);
    if (e != cudaSuccess) return cuda_error(e, "launch paged_tc");
    return FTC_OK;
}

}  // namespace paged
}  // namespace ftc
