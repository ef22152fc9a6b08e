// paged_plan.cuh -- how the paged attention kernels cut their work.
//
// The packed rows of a sequence and KV head are its new rows times the gqa
// query heads that share the KV head (row r: token r / gqa, head r % gqa); a
// tile is TR consecutive packed rows.  A tile's work is the list of key
// chunks (KS positions each, KS-aligned) that any of its rows sees: the chunks
// of the first n_sink positions, then those from the window's start to the
// last row's position.  All chunks of all tiles, in (sequence, KV head, tile)
// order, are one line of W units, and CTA b of G takes the units [b L, b L +
// L): every CTA gets the same work whatever the lengths (a tile's cut pieces
// are joined afterwards, in order).  The lengths are on the device, so each
// CTA works the plan out for itself: a thread per sequence, a scan, a search.
#pragma once

#include "kv_pages.cuh"
#include "sm100.cuh"

namespace ftc {

constexpr int kMaxSeqs = 2048;

// What joins a cut tile: written by the CTA that holds its start.
struct CutTile {
    int pieces;  // 0: this CTA starts no cut tile
    int row;     // first row of the sequence
    int kvh;
    int r0;      // first packed row of the tile
    int rows;    // its packed rows
};

struct PagedArgs {
    PageView b;
    const void* q;
    const void* v;         // the V pool
    void* out;
    const float *ks, *vs;  // 8-bit scales
    int64_t q_stride, out_stride;
    int n_head, gqa;
    int window, n_sink;    // window 0: none
    int min_rows, max_rows;  // sequences of this many packed rows are this launch's
    int second;            // the call's second launch (see paged_mma)
    float c;               // score scale * log2(e)
    float* part;           // cut tiles: [G][2][TR][HD] sums, then
    float2* stat;          // [G][2][TR] (maximum, sum of weights)
    CutTile* cut;           // [G]
};

// A tile and the chunks of it.
template <int TR, int KS>
struct TileWork {
    int n_sink_chunks, first, count;  // chunk i: i < n_sink_chunks ? i : first + i - n_sink_chunks
    int p_first, p_last;              // positions of the tile's first and last row

    __device__ __forceinline__ TileWork(const PagedArgs& a, int n, int len, int t) {
        const int rows = n * a.gqa;
        const int r1 = min((t + 1) * TR, rows) - 1;
        p_first = len - n + t * TR / a.gqa;
        p_last = len - n + r1 / a.gqa;
        const int cap = a.b.table_cols << a.b.page_shift;  // positions the table can name
        const int hi = min(p_last, cap - 1);
        // (rows before position 0 have no window; window may be INT_MAX)
        first = a.window > 0 ? max(max(p_first, 0) - a.window + 1, 0) / KS : 0;
        n_sink_chunks = a.window > 0
                            ? min((int)(((int64_t)min(a.n_sink, hi + 1) + KS - 1) / KS), first)
                            : 0;
        n_sink_chunks = max(n_sink_chunks, 0);
        const int own = hi < 0 ? 0 : max(hi / KS - first + 1, 0);
        count = max(n_sink_chunks + own, 1);  // a tile that sees nothing still stores its zeros
    }
    __device__ __forceinline__ int key0(int i) const {
        return (i < n_sink_chunks ? i : first + i - n_sink_chunks) * KS;
    }
};

// Where a CTA stands on the line of units.
struct PlanPos {
    int s, kvh, t;  // sequence, KV head, tile
    int i;          // chunk inside the tile
    int n, len, row;  // of the sequence
    int tiles;
};

template <int TR, int KS>
struct Plan {
    static constexpr int kSmem = (kMaxSeqs + 5) * 8;  // sums, and five more words

    // The sequence's rows for this launch: 0 tiles when it is another's.
    static __device__ __forceinline__ void load_seq(const PagedArgs& a, PlanPos& p) {
        seq_rows(a.b, p.s, p.row, p.n);
        p.len = seq_len(a.b, p.s);
        const int64_t rows = (int64_t)p.n * a.gqa;
        p.tiles = rows < a.min_rows || rows > a.max_rows ? 0 : (int)((rows + TR - 1) / TR);
    }

    // Chunks of all tiles of one KV head of a sequence, lanes of a warp
    // over the tiles; `most` grows to the largest tile that the lane sees.
    static __device__ __forceinline__ int64_t seq_chunks_warp(const PagedArgs& a,
                                                              const PlanPos& p, int& most) {
        int64_t w = 0;
        for (int t = threadIdx.x & 31; t < p.tiles; t += 32) {
            const int c = TileWork<TR, KS>(a, p.n, p.len, t).count;
            w += c;
            most = max(most, c);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        return w;
    }

    // Units before each sequence to pre[0 .. n_seqs) (shared memory), all
    // units returned, the tiles that they are of and, when asked for, the
    // largest tile's units; every thread of the CTA calls it.
    template <bool kLargest>
    static __device__ int64_t scan(const PagedArgs& a, int64_t* pre, int64_t& n_tiles,
                                   int& largest) {
        const int tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31;
        unsigned long long* tiles = reinterpret_cast<unsigned long long*>(pre + kMaxSeqs + 1);
        int* top = reinterpret_cast<int*>(pre + kMaxSeqs + 2);
        if (tid == 0) *tiles = 0, *top = 0;
        __syncthreads();
        int mine = 0, most = 0;
        for (int s = tid; s < a.b.n_seqs; s += nt) {
            PlanPos p;
            p.s = s;
            load_seq(a, p);
            mine += p.tiles;
            int64_t w = 0;
            if (p.tiles > 4) {
                w = -1;  // a warp's work, below
            } else {
                for (int t = 0; t < p.tiles; ++t) {
                    const int c = TileWork<TR, KS>(a, p.n, p.len, t).count;
                    w += c;
                    most = max(most, c);
                }
            }
            pre[s] = w;
        }
        if (mine) atomicAdd(tiles, (unsigned long long)mine);
        __syncthreads();
        for (int s = warp; s < a.b.n_seqs; s += nt >> 5) {
            if (pre[s] >= 0) continue;
            PlanPos p;
            p.s = s;
            load_seq(a, p);
            const int64_t w = seq_chunks_warp(a, p, most);
            __syncwarp();
            if (lane == 0) pre[s] = w;
        }
        if (kLargest && most) atomicMax(top, most);
        __syncthreads();
        int64_t* total = pre + kMaxSeqs;
        if (warp == 0) {
            int64_t sum = 0;
            for (int s0 = 0; s0 < a.b.n_seqs; s0 += 32) {
                const int s = s0 + lane;
                const int64_t w = s < a.b.n_seqs ? pre[s] * a.b.n_kv : 0;
                int64_t x = w;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                if (s < a.b.n_seqs) pre[s] = sum + x - w;
                sum += __shfl_sync(0xffffffffu, x, 31);
            }
            if (lane == 0) *total = sum;
        }
        __syncthreads();
        n_tiles = (int64_t)*tiles * a.b.n_kv;
        largest = kLargest ? *top : 0;
        return *total;
    }

    // The position of unit u (a whole warp calls it; u < all units).
    static __device__ PlanPos locate(const PagedArgs& a, const int64_t* pre, int64_t u) {
        const int lane = threadIdx.x & 31;
        int lo = 0, hi = a.b.n_seqs - 1;  // last s with pre[s] <= u
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= u) lo = mid;
            else hi = mid - 1;
        }
        PlanPos p;
        p.s = lo;
        load_seq(a, p);
        int most = 0;
        const int64_t per = p.tiles > 0 ? seq_chunks_warp(a, p, most) : 1;
        const int64_t rem = u - pre[lo];
        p.kvh = (int)(rem / per);
        int64_t left = rem - p.kvh * per;
        p.t = 0;
        p.i = 0;
        for (int t0 = 0; t0 < p.tiles; t0 += 32) {
            const int t = t0 + lane;
            const int64_t w = t < p.tiles ? TileWork<TR, KS>(a, p.n, p.len, t).count : 0;
            int64_t x = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, t < p.tiles && x > left);
            if (hit) {
                const int l = __ffs(hit) - 1;
                p.t = t0 + l;
                p.i = (int)(left - __shfl_sync(0xffffffffu, x - w, l));
                break;
            }
            left -= __shfl_sync(0xffffffffu, x, 31);
        }
        return p;
    }

    // The tile edge nearest to unit u of W (a whole warp calls it).
    static __device__ int64_t nearest_edge(const PagedArgs& a, const int64_t* pre, int64_t u,
                                           int64_t W) {
        if (u >= W) return W;
        const PlanPos p = locate(a, pre, u);
        const int c = TileWork<TR, KS>(a, p.n, p.len, p.t).count;
        return 2 * p.i < c ? u - p.i : u - p.i + c;
    }

    // To the first chunk of the next tile.
    static __device__ __forceinline__ void next_tile(const PagedArgs& a, PlanPos& p) {
        p.i = 0;
        if (++p.t < p.tiles) return;
        p.t = 0;
        if (++p.kvh < a.b.n_kv) return;
        p.kvh = 0;
        do {
            if (++p.s >= a.b.n_seqs) return;
            load_seq(a, p);
        } while (p.tiles == 0);
    }
};

// Units per CTA: an equal share of all, rounded up to `step`.  A share below
// `least` is raised to it (a shorter range costs more in joining than it
// saves), but not past a tile: with little work, CTAs of their own for the
// tiles beat one that takes several in turn (8 tiles of 60 positions: 21 us in
// shares of four tiles, 10 us one by one).
__device__ __forceinline__ int64_t plan_share(int64_t W, int64_t tiles, int G, int step,
                                              int least) {
    const int64_t per = (W + G - 1) / G;
    if (per >= least) return (per + step - 1) / step * step;
    const int64_t tile = (W + tiles - 1) / max(tiles, (int64_t)1);
    return max(per, min((int64_t)least, tile));
}

}  // namespace ftc
