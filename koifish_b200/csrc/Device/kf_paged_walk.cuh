// kf_paged_walk.cuh -- how the attention kernels share a step over a cache in pages among their CTAs (attn_paged.cu, attn_paged_tc.cu, attn_paged_q4.cu).
//
// The new tokens of a sequence are cut into blocks of `tb`, a block's visible positions into tiles; the tiles of all blocks (and of plan.heads kv heads of each), one after the
// other, are cut into equal runs, so that every CTA has the same number of them (or of units that tiles are worth) whatever the lengths are.  A block that two or more runs share is a
// piece in each and is merged afterwards.
#pragma once
#include "kf_paged.cuh"
#include "kf_tc.cuh"

struct PagedPlan {  // kernel parameter
    int tb, group, window;  // tokens of a block; heads of a kv group; positions that a row sees at most (<= 0: all)
    int heads;              // kv heads that lie one after the other in the order of tiles (1: every CTA of a team has its own)
    int runs;               // runs at most
    int first;              // with a window, positions from 0 on that stay visible
};
// The positions [lo, hi) that a row of block b may see, and with a window and first positions that lie apart from it [0, first) too; the first tile of [lo, hi), how many tiles
// of the first positions lie in front of it (ns), and how many tiles there are.
static inline __host__ __device__ int paged_block(int tile, int cap, int tb, int window, int first, int n, int len, int b, int& lo, int& hi, int& kt0, int& ns) {
    const int p0 = len - n + b * tb, p1 = len - n + (n < (b + 1) * tb ? n : (b + 1) * tb);  // positions of the block's rows: p0 .. p1 - 1
    hi = p1 < cap ? p1 : cap, ns = 0;
    lo = window > 0 && p0 >= window ? p0 - window + 1 : 0;
    if (window > 0) {
        const int f = first < hi ? first : hi;
        if (lo <= f) lo = 0;  // side by side
        else if (f > 0 && hi <= lo) lo = 0, hi = f;  // the window lies behind the table
        else if (f > 0) ns = (f + tile - 1) / tile;
    }
    kt0 = lo / tile;
    if (hi <= lo) {  // nothing to see: a tile without positions, so that the rows are written
        kt0 = 0, lo = hi = 0;
        return 1;
    }
    if (ns > kt0) ns = kt0;  // they end in the tile in which the window begins
    return (hi + tile - 1) / tile - kt0 + ns;
}
// tiles that a step can have at most
static inline long long paged_most(int tile, const KfPaged& pg, const PagedPlan& pl) {
    return ((long long)pg.M / pl.tb + pg.n_seq) * ((pg.cap + tile - 1) / tile + 1) * pl.heads;
}
#ifdef __CUDACC__
struct alignas(16) PagedPiece {
    int s, q0, n, len;          // sequence, its rows in the panel, its positions
    int t0, t1, lo, hi;         // tiles of this piece (t0 < 0: no more pieces), see tile(); positions that a row of the block may see
    int b, head, whole, first;  // block; head of plan.heads; 1: all tiles of the block; run in which the block begins
    int last;                   // run in which it ends
    int kt0, ns;                // first tile of [lo, hi); tiles of the first positions, which come before it
    int pad;
    // the tile of positions that index t stands for: those of the first positions have the ns indices in front of kt0
    __device__ __forceinline__ int tile(int t) const { return t < kt0 ? t - kt0 + ns : t; }
};
// What the runs are equal in: units.  A tile of a block that has `left` tokens from its first on is worth 2^tile() of them, a block kBlock beside its tiles.  Up to kFew tiles a run
// and up to 32 sequences each tile is one and a block none all the same.
struct EqualTiles {
    static constexpr int kMost = 1, kBlock = 0, kFew = 0;
    static __device__ __forceinline__ int tile(int left, int tb) { return 0; }
};
// One warp's way through the sequences, 32 at a time: every lane holds one.
template <int TILE, class Units = EqualTiles>
struct PagedWalk {
    const KfPaged pg;
    const PagedPlan pl;
    const int lane;
    int base, q0, n, len, nb;
    int units, inc, before = 0;  // of the lane's sequence, of it and the lanes below, of the sequences before these 32
    int took = 0;                // units of what at() found last
    bool equal = Units::kMost == 1;
    __device__ __forceinline__ PagedWalk(const KfPaged& pg_, const PagedPlan& pl_, int lane_) : pg(pg_), pl(pl_), lane(lane_) {}
    static __device__ __forceinline__ int scan(int v, int lane) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        return v;
    }
    __device__ __forceinline__ int cost(int n_, int len_, int b) const {  // units of a block
        int lo, hi, kt0, ns;
        return (paged_block(TILE, pg.cap, pl.tb, pl.window, pl.first, n_, len_, b, lo, hi, kt0, ns) << worth(n_, b)) + block();
    }
    __device__ __forceinline__ int worth(int n_, int b) const { return Units::kMost == 1 || equal ? 0 : Units::tile(n_ - b * pl.tb, pl.tb); }
    __device__ __forceinline__ int block() const { return Units::kMost == 1 || equal ? 0 : Units::kBlock; }
    // tiles of a block that begin in its first x units: the first one at 0, tile i at block() + (i << w)
    __device__ __forceinline__ int below(int x, int w) const { return Units::kMost == 1 ? x : x <= 0 ? 0 : 1 + (max(0, x - 1 - block()) >> w); }
    __device__ __forceinline__ void load(int base_) {
        base = base_, n = 0, nb = 0, units = 0;
        if (base + lane < pg.n_seq) {
            paged_seq(pg, base + lane, q0, n, len);
            if (n > 0) nb = n <= pl.tb ? 1 : (n + pl.tb - 1) / pl.tb, units = cost(n, len, 0);
        }
        for (unsigned many = __ballot_sync(0xffffffffu, nb > 1); many; many &= many - 1) {  // the blocks of a sequence over the lanes
            const int l = __ffs(many) - 1, n_ = __shfl_sync(0xffffffffu, n, l), len_ = __shfl_sync(0xffffffffu, len, l), nb_ = __shfl_sync(0xffffffffu, nb, l);
            int sum = 0;
#pragma unroll 1
            for (int b = lane; b < nb_; b += 32) sum += cost(n_, len_, b);
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == l) units = sum;
        }
        units *= pl.heads;
        inc = scan(units, lane);
    }
    __device__ __forceinline__ int total() const { return __shfl_sync(0xffffffffu, inc, 31); }
    // to the 32 sequences that hold unit u
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
    // The piece of run `index` of the tiles that begin in units u .. end - 1 (u < end <= all units, u not before what was asked for last), up to the block's end; runs have `run`
    // units.  Where tiles have several units and the run begins inside one, that may be none (t0 == t1).
    __device__ __forceinline__ PagedPiece at(int u, int end, int run, int index) {
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
                const int t = b0 + lane < nb_ ? cost(p.n, p.len, b0 + lane) * pl.heads : 0, c = scan(t, lane);
                const unsigned in = __ballot_sync(0xffffffffu, c > off);
                if (in) {
                    const int f = __ffs(in) - 1;
                    p.b = b0 + f, off -= __shfl_sync(0xffffffffu, c - t, f);
                    break;
                }
                off -= __shfl_sync(0xffffffffu, c, 31);
            }
        }
        const int all = paged_block(TILE, pg.cap, pl.tb, pl.window, pl.first, p.n, p.len, p.b, p.lo, p.hi, p.kt0, p.ns);
        const int w = worth(p.n, p.b), span = (all << w) + block();
        if (off >= span) p.head = off / span, off -= p.head * span;
        took = min(span - off, end - u);
        const int t0 = below(off, w), t1 = below(off + took, w);
        p.t0 = p.kt0 - p.ns + t0, p.t1 = p.kt0 - p.ns + t1;
        p.whole = t1 - t0 == all;
        p.first = p.last = 0;
        // a division where the block begins or its last tile does in another run
        if (!p.whole) p.first = off == 0 ? index : (u - off) / run, p.last = t1 == all ? index : (u - off + (all - 1 << w) + (all > 1 ? block() : 0)) / run;
        return p;
    }
};
// The pieces of a CTA's run: one warp works them out and hands them to the others, a few ahead of their use.  The others' code stays small that way: what a warp runs for the
// first time comes line by line from L2 or from memory, and that was most of a short call's time when each of them found its own pieces.
constexpr int kPieceSlots = 4;
struct PagedQueue {  // shared memory
    PagedPiece piece[kPieceSlots];
    uint64_t full[kPieceSlots], empty[kPieceSlots];
    int s_sum[256];  // units of every 32 sequences, from 33 on
    __device__ __forceinline__ void init(int readers) {  // one thread
        for (int i = 0; i < kPieceSlots; i++) mbar_init(&full[i], 1), mbar_init(&empty[i], readers);
    }
};
// Works the pieces of run `index` out.  From 33 sequences on all warps of the CTA count first, and meet behind it.
template <int TILE, class Units = EqualTiles>
struct PagedPlanner {
    PagedWalk<TILE, Units> walk;
    int u = 0, u0 = 0, u1 = 0, run = 1;
    uint32_t i = 0;
    bool more = true;
    PagedPiece pc;
    __device__ __forceinline__ PagedPlanner(const KfPaged& pg, const PagedPlan& pl, int lane) : walk(pg, pl, lane) {}
    static __device__ __noinline__ void count(const KfPaged& pg, const PagedPlan& pl, int* s_sum, int warp, int warps, int lane) {
        PagedWalk<TILE, Units> walk(pg, pl, lane);
#pragma unroll 1
        for (int w = warp; w < (pg.n_seq + 31) / 32; w += warps) {
            walk.load(w * 32);
            if (lane == 31) s_sum[w] = walk.inc;
        }
    }
    __device__ __forceinline__ void start(const PagedQueue& qu, int index) {
        int W = 0;
        if (walk.pg.n_seq <= 32) {
            walk.equal = true;
#pragma unroll 1
            while (true) {
                walk.load(0);
                W = walk.total();
                if (Units::kMost == 1 || !walk.equal || W <= Units::kFew * walk.pl.runs) break;
                walk.equal = false;
            }
        } else {
            for (int w = walk.lane; w < (walk.pg.n_seq + 31) / 32; w += 32) W += qu.s_sum[w];
            W = __reduce_add_sync(0xffffffffu, W);
        }
        run = max(Units::kMost == 1 || walk.equal ? 1 : Units::kMost + Units::kBlock, (W + walk.pl.runs - 1) / walk.pl.runs);  // a run inside a block has a tile that begins in it
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
            pc = walk.at(u, u1, run, index), u += walk.took;
            if (Units::kMost > 1 && pc.t0 == pc.t1) {  // the rest of a tile that began in the run before
                more = u < u1;
                if (more) pc = walk.at(u, u1, run, index), u += walk.took;
                else pc.last = 0;
            }
        }
        if (!more) {
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
