// kf_paged_walk.cuh -- how the attention kernels share a step over a cache in pages among their CTAs (attn_paged.cu, attn_paged_tc.cu).
#pragma once
#include "kf_paged.cuh"
#include "kf_tc.cuh"

// What an attention kernel takes of a step, and in which order.  The rows (new token, head of the kv group) of a sequence are cut into blocks of `rb`, a block's visible
// positions into tiles; the tiles of all blocks, one after the other, are cut into equal runs, so that every CTA has the same number of them whatever the lengths are.
// A block that two or more runs share is a piece in each and is merged afterwards.
struct PagedPlan {  // kernel parameter
    int rb, group, window, min_rows, max_rows;  // sequences with min_rows < rows <= max_rows
    int heads;                                  // kv heads that lie one after the other in the order of tiles (1: every CTA of a team has its own)
};
// the positions [lo, hi) that a row of block b may see, their first tile and how many tiles they touch
static inline __host__ __device__ int paged_block(int tile, int cap, const PagedPlan& pl, int n, int len, int b, int& lo, int& hi, int& kt0) {
    const int t_lo = b * pl.rb / pl.group, t_hi = ((n * pl.group < (b + 1) * pl.rb ? n * pl.group : (b + 1) * pl.rb) - 1) / pl.group;
    hi  = len - n + t_hi + 1 < cap ? len - n + t_hi + 1 : cap;
    lo  = pl.window > 0 && len - n + t_lo >= pl.window ? len - n + t_lo - pl.window + 1 : 0;
    kt0 = lo / tile;
    if (hi <= lo) {  // nothing to see: a tile without positions, so that the rows are written
        kt0 = 0, lo = hi = 0;
        return 1;
    }
    return (hi + tile - 1) / tile - kt0;
}
// tiles that a step can have at most
static inline long long paged_most(int tile, const KfPaged& pg, const PagedPlan& pl) {
    return ((long long)pg.M * pl.group / pl.rb + pg.n_seq) * ((pg.cap + tile - 1) / tile + 1) * pl.heads;
}
#ifdef __CUDACC__
struct PagedPiece {
    int s, q0, n, len, b;     // sequence, its rows in the panel, its positions; block
    int head;                 // of plan.heads
    int lo, hi;               // positions that a row of the block may see
    int t0, t1;               // tiles of this piece
    int u, tiles;             // first tile of the block and head in the order of all, and how many there are
};
// One warp's way through the sequences, 32 at a time: every lane holds one.
template <int TILE>
struct PagedWalk {  // plan.heads is counted in
    const KfPaged pg;
    const PagedPlan pl;
    const int lane;
    int base = 0, q0 = 0, n = 0, len = 0, nb = 0;
    int units = 0, inc = 0, before = 0;  // tiles of the lane's sequence, of it and the lanes below, of the sequences before these 32
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
        return paged_block(TILE, pg.cap, pl, n_, len_, b, lo, hi, kt0);
    }
    __device__ __noinline__ void load(int base_) {
        base = base_, n = 0, nb = 0, units = 0;
        if (base + lane < pg.n_seq) {
            paged_seq(pg, base + lane, q0, n, len);
            const int rows = n * pl.group;
            if (rows > pl.min_rows && rows <= pl.max_rows) nb = (rows + pl.rb - 1) / pl.rb;
        }
        if (nb == 1) units = tiles(n, len, 0);
        for (unsigned many = __ballot_sync(0xffffffffu, nb > 1); many; many &= many - 1) {  // the blocks of a sequence over the lanes
            const int l = __ffs(many) - 1, n_ = __shfl_sync(0xffffffffu, n, l), len_ = __shfl_sync(0xffffffffu, len, l), nb_ = __shfl_sync(0xffffffffu, nb, l);
            int sum = 0;
            for (int b = lane; b < nb_; b += 32) sum += tiles(n_, len_, b);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == l) units = sum;
        }
        units *= pl.heads;
        inc = scan(units, lane);
    }
    __device__ __forceinline__ int total() const { return __shfl_sync(0xffffffffu, inc, 31); }
    // the tiles of all sequences; from 33 sequences on behind paged_sums()
    __device__ __forceinline__ int count(const int* s_sum) {
        if (pg.n_seq <= 32) {
            load(0);
            return total();
        }
        int sum = 0;
        for (int w = lane; w < (pg.n_seq + 31) / 32; w += 32) sum += s_sum[w];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
    }
    // to the 32 sequences that hold tile u, behind count()
    __device__ __forceinline__ void seek(const int* s_sum, int u) {
        if (pg.n_seq <= 32) return;
        const int wins = (pg.n_seq + 31) / 32;
        before = 0;
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
    __device__ __forceinline__ PagedPiece at(int u, int end) {
        unsigned hit;
        while (!(hit = __ballot_sync(0xffffffffu, before + inc > u)) && base + 32 < pg.n_seq) {
            before += total();
            load(base + 32);
        }
        const int l = hit ? __ffs(hit) - 1 : 31;
        PagedPiece p;
        p.s = base + l, p.q0 = __shfl_sync(0xffffffffu, q0, l), p.n = __shfl_sync(0xffffffffu, n, l), p.len = __shfl_sync(0xffffffffu, len, l);
        const int nb_ = __shfl_sync(0xffffffffu, nb, l);
        int off = u - before - __shfl_sync(0xffffffffu, inc - units, l);
        p.b           = 0;
        if (nb_ > 1)
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
        int kt0;
        p.tiles = paged_block(TILE, pg.cap, pl, p.n, p.len, p.b, p.lo, p.hi, kt0);
        p.head  = pl.heads > 1 ? off / p.tiles : 0;
        off -= p.head * p.tiles;
        p.u  = u - off;
        p.t0 = kt0 + off, p.t1 = kt0 + min(p.tiles, off + (end - u));
        return p;
    }
};
// All warps of a CTA, from 33 sequences on: the tiles of every 32 of them (s_sum: 256 entries of shared memory)
template <int TILE>
__device__ __noinline__ void paged_sums(const KfPaged& pg, const PagedPlan& pl, int* s_sum, int warp, int warps, int lane) {
    PagedWalk<TILE> walk(pg, pl, lane);
    for (int w = warp; w < (pg.n_seq + 31) / 32; w += warps) {
        walk.load(w * 32);
        const int t = walk.total();
        if (lane == 0) s_sum[w] = t;
    }
}
// The pieces of a CTA's run: one warp works them out and hands them to the others, a few ahead of their use.  The others' code stays small that way: what a warp runs for the
// first time comes from L2 line by line, and that was most of a short call's time when each of them found its own pieces (a step of 64 sequences, 11 warps: 14 us until the first
// tile had landed).
constexpr int kPieceSlots = 4;
struct PagedQueue {  // shared memory
    uint64_t full[kPieceSlots], empty[kPieceSlots];
    PagedPiece piece[kPieceSlots];  // t0 < 0: no more
    int first[kPieceSlots], last[kPieceSlots];  // runs in which the piece's block begins and ends
    int s_sum[256];
    __device__ __forceinline__ void init(int readers) {  // one thread
        for (int i = 0; i < kPieceSlots; i++) mbar_init(&full[i], 1), mbar_init(&empty[i], readers);
    }
};
template <int TILE>
__device__ __noinline__ void paged_plan(PagedQueue& qu, const KfPaged& pg, const PagedPlan& pl, int runs, int min_run, int index, int lane, volatile int* dead, const KfBound& bound) {
    PagedWalk<TILE> walk(pg, pl, lane);
    const int W = walk.count(qu.s_sum), run = max(min_run, (W + runs - 1) / runs), u0 = (int)min((long long)W, (long long)index * run), u1 = min(W, u0 + run);
    if (u0 < u1) walk.seek(qu.s_sum, u0);
    int u = u0;
    for (uint32_t i = 0;; i++) {
        PagedPiece pc;
        pc.t0 = -1;
        const bool more = u < u1;
        if (more) {
            pc = walk.at(u, u1);
            u += pc.t1 - pc.t0;
        }
        const uint32_t slot = i % kPieceSlots;
        if (!mbar_wait_warp(smem_u32(&qu.empty[slot]), ((i / kPieceSlots) & 1) ^ 1, dead, bound)) return;
        if (lane == 0) {
            qu.piece[slot] = pc;
            if (more) qu.first[slot] = pc.u / run, qu.last[slot] = (pc.u + pc.tiles - 1) / run;
            mbar_arrive(&qu.full[slot]);
        }
        if (!more) return;
    }
}
// a reader's way through the pieces: false behind the last, or when a wait has run out (live)
struct PagedReader {
    uint32_t i = 0;
    int first, last;
    __device__ __forceinline__ bool next(PagedQueue& qu, PagedPiece& pc, int lane, volatile int* dead, const KfBound& bound, bool& live) {
        const uint32_t slot = i % kPieceSlots;
        if (!(live = mbar_wait_warp(smem_u32(&qu.full[slot]), (i / kPieceSlots) & 1, dead, bound))) return false;
        pc = qu.piece[slot], first = qu.first[slot], last = qu.last[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&qu.empty[slot]);
        i++;
        return pc.t0 >= 0;
    }
};
#endif
