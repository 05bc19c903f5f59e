// kf_paged.cuh -- a step over a cache in pages, as the kernels see it (paged_append.cu, attn_paged.cu, attn_paged_tc.cu).
#pragma once
#include "kf_common.cuh"

struct KfPaged {  // kernel parameter
    const int32_t *table, *q_start, *len;
    int table_cols, n_seq, n_pages, page, cap /* positions a table holds */, M /* rows of the panel */;
};
// attn_paged_tc.cu: sequences with more than min_rows rows on tcgen05
int kf_attn_paged_tc(kf_ctx* ctx, const kf_paged_kv* kv, const KfPaged& pg, void* out, long long ldo, const void* q, long long ldq, int n_head, float scale, int window, int min_rows);
int kf_paged_check(kf_ctx* ctx, const kf_paged_kv* kv, int M, KfPaged* out);  // paged_append.cu: arguments that all of them share
static inline size_t kf_paged_stride(const kf_paged_kv* kv) { return kv->page_stride ? kv->page_stride : (size_t)kv->page_size * kv->n_kv * kv->head_dim; }

// What an attention kernel takes of a step, and in which order.  The rows (new token, head of the kv group) of a sequence are cut into blocks of `rb`, a block's visible
// positions into tiles; the tiles of all blocks, one after the other, are cut into equal runs, so that every CTA has the same number of them whatever the lengths are.
// A block that two or more runs share is a piece in each and is merged afterwards.
struct PagedPlan {  // kernel parameter
    int rb, group, window, min_rows, max_rows;  // sequences with min_rows < rows <= max_rows
    int heads;                                  // kv heads that lie one after the other in the order of tiles (1: every CTA of a team has its own)
};
// the positions [lo, hi) that a row of block b may see, their first tile and how many tiles they touch
static inline __host__ __device__ int paged_block(int tile, int cap, const PagedPlan& pl, int n, int len, int b, int& lo, int& hi, int& kt0) {
    const int t_lo = (int)((long long)b * pl.rb / pl.group), t_hi = (int)(((long long)n * pl.group < (long long)(b + 1) * pl.rb ? (long long)n * pl.group : (long long)(b + 1) * pl.rb) - 1) / pl.group;
    hi  = len - n + t_hi + 1 < cap ? len - n + t_hi + 1 : cap;
    lo  = pl.window > 0 && len - n + t_lo >= pl.window ? len - n + t_lo - pl.window + 1 : 0;
    kt0 = lo / tile;
    if (hi <= lo) {  // nothing to see: a tile without positions, so that the rows are written
        kt0 = 0, lo = hi = 0;
        return 1;
    }
    return (hi + tile - 1) / tile - kt0;
}
#ifdef __CUDACC__
// the pointers for use behind kf_grid_dependency_wait()
__device__ __forceinline__ KfPaged behind_wait(KfPaged p) {
    p.table = behind_wait(p.table), p.q_start = behind_wait(p.q_start), p.len = behind_wait(p.len);
    return p;
}
// page of position p >= 0 of sequence s, -1: not there
__device__ __forceinline__ int paged_page(const KfPaged& pg, int s, int p) {
    if (p >= pg.cap) return -1;
    const int e = pg.table[(size_t)s * pg.table_cols + p / pg.page];
    return e >= 0 && e < pg.n_pages ? e : -1;
}
// rows [q0, q0 + n) of sequence s in the panel, and its positions
__device__ __forceinline__ void paged_seq(const KfPaged& pg, int s, int& q0, int& n, int& len) {
    q0  = min(max(pg.q_start[s], 0), pg.M);
    n   = min(max(pg.q_start[s + 1], q0), pg.M) - q0;
    len = max(pg.len[s], 0);
}

struct PagedPiece {
    int s, q0, n, len, b;     // sequence, its rows in the panel, its positions; block
    int head;                 // of plan.heads
    int lo, hi;               // positions that a row of the block may see
    int t0, t1;               // tiles of this piece
    long long u;              // first tile of the block and head in the order of all, and how many there are
    int tiles;
};
// One warp's way through the sequences, 32 at a time: every lane holds one.
template <int TILE>
struct PagedWalk {  // plan.heads is counted in
    const KfPaged pg;
    const PagedPlan pl;
    const int lane;
    int base = 0, q0 = 0, n = 0, len = 0, nb = 0;
    long long units = 0, inc = 0, before = 0;  // tiles of the lane's sequence, of it and the lanes below, of the sequences before these 32
    __device__ __forceinline__ PagedWalk(const KfPaged& pg_, const PagedPlan& pl_, int lane_) : pg(pg_), pl(pl_), lane(lane_) {}
    static __device__ __forceinline__ long long scan(long long v, int lane) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long w = __shfl_up_sync(0xffffffffu, v, o);
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
            const long long rows = (long long)n * pl.group;
            if (rows > pl.min_rows && rows <= pl.max_rows) nb = (int)((rows + pl.rb - 1) / pl.rb);
        }
        if (nb == 1) units = tiles(n, len, 0);
        for (unsigned many = __ballot_sync(0xffffffffu, nb > 1); many; many &= many - 1) {  // the blocks of a sequence over the lanes
            const int l = __ffs(many) - 1, n_ = __shfl_sync(0xffffffffu, n, l), len_ = __shfl_sync(0xffffffffu, len, l), nb_ = __shfl_sync(0xffffffffu, nb, l);
            long long sum = 0;
            for (int b = lane; b < nb_; b += 32) sum += tiles(n_, len_, b);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == l) units = sum;
        }
        units *= pl.heads;
        inc = scan(units, lane);
    }
    __device__ __forceinline__ long long total() const { return __shfl_sync(0xffffffffu, inc, 31); }
    // all warps of a CTA: the tiles of all sequences.  s_sum: 256 entries of shared memory, used from 33 sequences on
    __device__ __forceinline__ long long count(long long* s_sum, int warp, int warps) {
        if (pg.n_seq <= 32) {
            load(0);
            return total();
        }
        const int wins = (pg.n_seq + 31) / 32;
        for (int w = warp; w < wins; w += warps) {
            load(w * 32);
            const long long t = total();
            if (lane == 0) s_sum[w] = t;
        }
        __syncthreads();
        long long sum = 0;
        for (int w = lane; w < wins; w += 32) sum += s_sum[w];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
    }
    // to the 32 sequences that hold tile u, behind count()
    __device__ __forceinline__ void seek(const long long* s_sum, long long u) {
        if (pg.n_seq <= 32) return;
        const int wins = (pg.n_seq + 31) / 32;
        before = 0;
        for (int w0 = 0; w0 < wins; w0 += 32) {
            const long long v = w0 + lane < wins ? s_sum[w0 + lane] : 0, c = scan(v, lane);
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
    __device__ __forceinline__ PagedPiece at(long long u, long long end) {
        unsigned hit;
        while (!(hit = __ballot_sync(0xffffffffu, before + inc > u)) && base + 32 < pg.n_seq) {
            before += total();
            load(base + 32);
        }
        const int l = hit ? __ffs(hit) - 1 : 31;
        PagedPiece p;
        p.s = base + l, p.q0 = __shfl_sync(0xffffffffu, q0, l), p.n = __shfl_sync(0xffffffffu, n, l), p.len = __shfl_sync(0xffffffffu, len, l);
        const int nb_ = __shfl_sync(0xffffffffu, nb, l);
        long long off = u - before - __shfl_sync(0xffffffffu, inc - units, l);
        p.b           = 0;
        if (nb_ > 1)
            for (int b0 = 0; b0 < nb_; b0 += 32) {
                const long long t = b0 + lane < nb_ ? (long long)tiles(p.n, p.len, b0 + lane) * pl.heads : 0, c = scan(t, lane);
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
        p.head  = pl.heads > 1 ? (int)(off / p.tiles) : 0;
        off -= (long long)p.head * p.tiles;
        p.u  = u - off;
        p.t0 = kt0 + (int)off, p.t1 = kt0 + (int)min((long long)p.tiles, off + (end - u));
        return p;
    }
};
#endif
