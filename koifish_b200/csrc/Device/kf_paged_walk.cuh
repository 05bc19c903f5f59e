// kf_paged_walk.cuh -- how the attention kernels share a step over a cache in pages among their CTAs (attn_paged.cu, attn_paged_tc.cu).
//
// The new tokens of a sequence are cut into blocks of `tb`, a block's visible positions into tiles; the tiles of all blocks (and of plan.heads kv heads of each), one after the
// other, are cut into equal runs, so that every CTA has the same number of them whatever the lengths are.  A block that two or more runs share is a piece in each and is merged
// afterwards.
#pragma once
#include "kf_paged.cuh"
#include "kf_tc.cuh"

struct PagedPlan {  // kernel parameter
    int tb, group, window;  // tokens of a block; heads of a kv group; positions that a row sees at most (<= 0: all)
    int heads;              // kv heads that lie one after the other in the order of tiles (1: every CTA of a team has its own)
    int runs;               // runs at most
};
// the positions [lo, hi) that a row of block b may see, their first tile and how many tiles they touch
static inline __host__ __device__ int paged_block(int tile, int cap, int tb, int window, int n, int len, int b, int& lo, int& hi, int& kt0) {
    const int first = len - n + b * tb, last = len - n + (n < (b + 1) * tb ? n : (b + 1) * tb);  // positions of the block's rows: first .. last - 1
    hi  = last < cap ? last : cap;
    lo  = window > 0 && first >= window ? first - window + 1 : 0;
    kt0 = lo / tile;
    if (hi <= lo) {  // nothing to see: a tile without positions, so that the rows are written
        kt0 = 0, lo = hi = 0;
        return 1;
    }
    return (hi + tile - 1) / tile - kt0;
}
// tiles that a step can have at most
static inline long long paged_most(int tile, const KfPaged& pg, const PagedPlan& pl) {
    return ((long long)pg.M / pl.tb + pg.n_seq) * ((pg.cap + tile - 1) / tile + 1) * pl.heads;
}
#ifdef __CUDACC__
struct alignas(16) PagedPiece {
    int s, q0, n, len;          // sequence, its rows in the panel, its positions
    int t0, t1, lo, hi;         // tiles of this piece (t0 < 0: no more pieces); positions that a row of the block may see
    int b, head, whole, first;  // block; head of plan.heads; 1: all tiles of the block; run in which the block begins
    int last, pad[3];           // run in which it ends
};
// One warp's way through the sequences, 32 at a time: every lane holds one.
template <int TILE>
struct PagedWalk {
    const KfPaged pg;
    const PagedPlan pl;
    const int lane;
    int base, q0, n, len, nb;
    int units, inc, before = 0;  // tiles of the lane's sequence, of it and the lanes below, of the sequences before these 32
    __device__ __forceinline__ PagedWalk(const KfPaged& pg_, const PagedPlan& pl_, int lane_) : pg(pg_), pl(pl_), lane(lane_) {}
    static __device__ __forceinline__ int scan(int v, int lane) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        return v;
    }
    __device__ __forceinline__ int tiles(int n_, int len_, int b) const {
        int lo, hi, kt0;
        return paged_block(TILE, pg.cap, pl.tb, pl.window, n_, len_, b, lo, hi, kt0);
    }
    __device__ __forceinline__ void load(int base_) {
        base = base_, n = 0, nb = 0, units = 0;
        if (base + lane < pg.n_seq) {
            paged_seq(pg, base + lane, q0, n, len);
            if (n > 0) nb = n <= pl.tb ? 1 : (n + pl.tb - 1) / pl.tb, units = tiles(n, len, 0);
        }
        for (unsigned many = __ballot_sync(0xffffffffu, nb > 1); many; many &= many - 1) {  // the blocks of a sequence over the lanes
            const int l = __ffs(many) - 1, n_ = __shfl_sync(0xffffffffu, n, l), len_ = __shfl_sync(0xffffffffu, len, l), nb_ = __shfl_sync(0xffffffffu, nb, l);
            int sum = 0;
#pragma unroll 1
            for (int b = lane; b < nb_; b += 32) sum += tiles(n_, len_, b);
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == l) units = sum;
        }
        units *= pl.heads;
        inc = scan(units, lane);
    }
    __device__ __forceinline__ int total() const { return __shfl_sync(0xffffffffu, inc, 31); }
    // to the 32 sequences that hold tile u
    __device__ __forceinline__ void seek(const int* s_sum, int u) {
        const int wins = (pg.n_seq + 31) / 32;
#pragma unroll 1
        for (int w0 = 0; w0 < wins; w0 += 32) {
            const int v = w0 + lane < wins ? s_sum[w0 + lane] : 0, c = scan(v, lane);
            const unsigned hit = __ballot_sync(0xffffffffu, before + c > u);
            if (hit) {
                const int l = __ffs(hit) - 1;
                before += __shfl_sync(0xffffffffu, c - v, l);
                load((w0 + l) * 32);
                return;
            }
            before += __shfl_sync(0xffffffffu, c, 31);
        }
    }
    // the piece that starts at tile u and ends before tile end (u < end <= all tiles, u not before what was asked for last)
    __device__ __forceinline__ PagedPiece at(int u, int end, int run) {
        unsigned hit;
#pragma unroll 1
        while (!(hit = __ballot_sync(0xffffffffu, before + inc > u)) && base + 32 < pg.n_seq) {
            before += total();
            load(base + 32);
        }
        const int l = hit ? __ffs(hit) - 1 : 31;
        PagedPiece p;
        p.s = base + l, p.q0 = __shfl_sync(0xffffffffu, q0, l), p.n = __shfl_sync(0xffffffffu, n, l), p.len = __shfl_sync(0xffffffffu, len, l);
        const int nb_ = __shfl_sync(0xffffffffu, nb, l);
        int off       = u - before - __shfl_sync(0xffffffffu, inc - units, l);
        p.b = 0, p.head = 0;
        if (nb_ > 1) {
#pragma unroll 1
            for (int b0 = 0; b0 < nb_; b0 += 32) {
                const int t = b0 + lane < nb_ ? tiles(p.n, p.len, b0 + lane) * pl.heads : 0, c = scan(t, lane);
                const unsigned in = __ballot_sync(0xffffffffu, c > off);
                if (in) {
                    const int f = __ffs(in) - 1;
                    p.b = b0 + f, off -= __shfl_sync(0xffffffffu, c - t, f);
                    break;
                }
                off -= __shfl_sync(0xffffffffu, c, 31);
            }
        }
        int kt0;
        const int all = paged_block(TILE, pg.cap, pl.tb, pl.window, p.n, p.len, p.b, p.lo, p.hi, kt0);
        if (off >= all) p.head = off / all, off -= p.head * all;
        const int n_tiles = min(all - off, end - u);
        p.t0 = kt0 + off, p.t1 = p.t0 + n_tiles;
        p.whole = n_tiles == all;
        p.first = p.last = 0;
        if (!p.whole) p.first = (u - off) / run, p.last = (u - off + all - 1) / run;
        return p;
    }
};
// The pieces of a CTA's run: one warp works them out and hands them to the others, a few ahead of their use.  The others' code stays small that way: what a warp runs for the
// first time comes line by line from L2 or from memory, and that was most of a short call's time when each of them found its own pieces.
constexpr int kPieceSlots = 4;
struct PagedQueue {  // shared memory
    PagedPiece piece[kPieceSlots];
    uint64_t full[kPieceSlots], empty[kPieceSlots];
    int s_sum[256];  // tiles of every 32 sequences, from 33 on
    __device__ __forceinline__ void init(int readers) {  // one thread
        for (int i = 0; i < kPieceSlots; i++) mbar_init(&full[i], 1), mbar_init(&empty[i], readers);
    }
};
// Works the pieces of run `index` out.  From 33 sequences on all warps of the CTA count first, and meet behind it.
template <int TILE>
struct PagedPlanner {
    PagedWalk<TILE> walk;
    int u = 0, u0 = 0, u1 = 0, run = 1;
    uint32_t i = 0;
    bool more = true;
    PagedPiece pc;
    __device__ __forceinline__ PagedPlanner(const KfPaged& pg, const PagedPlan& pl, int lane) : walk(pg, pl, lane) {}
    static __device__ __noinline__ void count(const KfPaged& pg, const PagedPlan& pl, int* s_sum, int warp, int warps, int lane) {
        PagedWalk<TILE> walk(pg, pl, lane);
#pragma unroll 1
        for (int w = warp; w < (pg.n_seq + 31) / 32; w += warps) {
            walk.load(w * 32);
            if (lane == 31) s_sum[w] = walk.inc;
        }
    }
    __device__ __forceinline__ void start(const PagedQueue& qu, int index) {
        int W = 0;
        if (walk.pg.n_seq <= 32) {
            walk.load(0);
            W = walk.total();
        } else {
            for (int w = walk.lane; w < (walk.pg.n_seq + 31) / 32; w += 32) W += qu.s_sum[w];
            W = __reduce_add_sync(0xffffffffu, W);
        }
        run = max(1, (W + walk.pl.runs - 1) / walk.pl.runs);
        u = u0 = (int)min((long long)W, (long long)index * run), u1 = min(W, u + run);
        if (u < u1 && walk.pg.n_seq > 32) walk.seek(qu.s_sum, u);
        pc.last = 0;
    }
    // the next piece to the readers; false: there was none, which they have been told.  rec (or NULL): behind the last, the piece that later runs go on with, last 0
    // where there is none (for the kernel that merges them).  It stays unwritten when a wait runs out before
    __device__ __forceinline__ bool push(PagedQueue& qu, int index, PagedPiece* rec, volatile int* dead, const KfBound& bound) {
        if (!more) return false;
        more = u < u1;
        if (more) {
            pc = walk.at(u, u1, run);
            u += pc.t1 - pc.t0;
        } else {
            if (rec && walk.lane == 0) {
                if (u0 == u1 || pc.whole || pc.first != index || pc.last == index) pc.last = 0;
                rec[index] = pc;
            }
            pc.t0 = -1;
        }
        const uint32_t slot = i % kPieceSlots;
        if (!mbar_wait_warp(smem_u32(&qu.empty[slot]), ((i / kPieceSlots) & 1) ^ 1, dead, bound)) return more = false;
        if (walk.lane == 0) {
            qu.piece[slot] = pc;
            mbar_arrive(&qu.full[slot]);
        }
        i++;
        return more;
    }
};
// a reader's way through the pieces: false behind the last, or when a wait has run out (live)
struct PagedReader {
    uint32_t i = 0;
    __device__ __forceinline__ bool next(PagedQueue& qu, PagedPiece& pc, int lane, volatile int* dead, const KfBound& bound, bool& live) {
        const uint32_t slot = i % kPieceSlots;
        if (!(live = mbar_wait_warp(smem_u32(&qu.full[slot]), (i / kPieceSlots) & 1, dead, bound))) return false;
        pc = qu.piece[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&qu.empty[slot]);
        i++;
        return pc.t0 >= 0;
    }
};
#endif
