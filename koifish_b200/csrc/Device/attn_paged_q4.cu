// attn_paged_q4.cu -- attention of a step's rows over a cache in pages that is held in 4 bits (kf_paged_attention_q4).
//
//   out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q.k_j - m),  c = scale * log2(e),  over the positions j that the row sees;  k and v: step * (code - zero), groups of 32 dims
//
// What the groups share stays outside the products:
//   q . k_j             = sum_g kstep_jg * (sum_{d in g} q_d code_jd - kzero_jg * sum_{d in g} q_d)
//   sum_j w_j v_jd      = sum_j (w_j vstep_jg) * code_jd - sum_j (w_j vstep_jg) * vzero_jg
// so codes go into the matrix instructions as they are: 4 bits in an otherwise empty bf16 word are the number code * 2^-133 (in the next 4 bits code * 2^-129: subnormal numbers and
// the first normal ones are one ladder), and one AND makes an operand of two codes.  The other operands carry 2^60, accumulators 2^-73, and what is left is undone with the scale.
// w_j vstep_jg is rounded to bf16 once, and what multiplies the zeros is the same rounded number, so that its error is relative to v.
//   * S^T = K q^T: positions are the 16 rows of mma.sync, up to 8 (two times 8) rows of the block its columns; a lane's registers hold whole words of its position's codes.
//     The zeros are one more step of 16 per group, in which the sum of the group's q stands as three bf16 numbers.
//   * O^T = V^T P^T: dims are the rows; P goes from the scores' layout to the operand's by a transposition of 8 x 8 (movmatrix), and the zeros of group j are row j of a
//     fifth accumulator.
//   * A warp takes 32 positions (four units) of a tile of 128; a unit is contiguous (Q4Unit), so a tile is a bulk copy per page (or part of 8 .. 128 positions of it).
//   * A team of n_kv CTAs takes a run of tiles, a kv head each; runs are equal whatever the lengths are (PagedWalk), and a second kernel, launched behind, merges what several share.
// For up to 16 rows of a sequence and kv head (new tokens x heads of the group); more go to attn_paged_q4_tc.cu, where few rows take longer.  64 sequences of 400 .. 4000 positions, one
// token each, us here / there: 128 dims, up to 8 rows 56 .. 62 / 154, 9 .. 16 rows 105 .. 111 / 154; 64 dims 38 .. 43 and 61 .. 64 / 124.
// What bounds it: the computing warps' own way.  The 64 sequences (64 / 8 heads, 196 MB) take 62.5 us, 3.1 TB/s; 59.8 with nothing loaded, 45.6 with nothing computed.  16 positions of 128 dims and
// 8 rows are 307 instructions of a warp, 149 of them on the pipe of logic and shifts, 24 products.  No pipe is full (1.8 instructions a clock of 4, logic 42 %, products 26 %): there are two
// computing warps to a scheduler, and an instruction waits 1.2 clocks for the one before it and 0.9 for memory and barriers.  One sequence of 100000 positions (128 MB) 38.3 us, 3.3 TB/s (35.6, 30.0), of
// which 7 are the start, 4 the end and the merge; one of 1300 9.3, as long as issuing two launches takes from Python; 40 with a window of 1000 and 4 first positions 28.7.
// 9 .. 16 rows of 128 dims do not fit the 168 registers that ten warps on four schedulers leave a thread: 200 bytes of it are spilled; the other instances spill nothing.
// Not kept: three CTAs per SM (62 us, and more pieces to merge: 42 for the one of 100000), one of eight computing warps (80 and 47), the merge by the CTA that arrives last (44 for the one of 100000:
// a fence, an atomic and rounds of loads one behind the other).
#include <algorithm>

#include "kf_paged_walk.cuh"

namespace {
// computing warps; groups of 16 positions that a warp takes of a tile beside one another (one: 77 us for the 64 sequences above, two: 68, at the time); positions of a tile
constexpr int kWarps = 4, kSub = 2, kTok = 16 * kSub * kWarps, kMaxStages = 12;
constexpr float kSlack = 8.f;  // growth of a maximum, log2, that sums are not rescaled for

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// products of 16 rows, 16 steps and 8 columns: c + a b, and a b.  Not volatile, nor are the loads around them: the scheduler is to mix what is independent
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_new(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// a pair of zeros times 2^-kZeroLog2: the zeros' sums, of weights of up to 2^68 times values of up to 2^50, stay within 32 bits' range over any number of positions
constexpr int kZeroLog2 = 24;
__device__ __forceinline__ uint32_t smaller(uint32_t zeros) {
    constexpr uint32_t f = (127u - kZeroLog2) << 7;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(zeros) : "r"(zeros), "r"(f << 16 | f));
    return zeros;
}
// pairs of codes out of a word: nibbles (0, 4), (1, 5), (2, 6), (3, 7); the second and the fourth stand for 16 times their codes
__device__ __forceinline__ void codes(uint32_t w, uint32_t (&c)[4]) { c[0] = w & 0x000f000fu, c[1] = w & 0x00f000f0u, c[2] = (w >> 8) & 0x000f000fu, c[3] = (w >> 8) & 0x00f000f0u; }

struct Q4Args {  // kernel parameter
    const uint8_t* pool;
    long long page_stride;
    uint16_t* out;
    const uint16_t* q;
    float* ws;        // [CTA][2][rb][HD] sums, then as many (maximum, denominator) pairs, then what begins in a run and goes on behind it, per CTA
    float2* ws_ml;
    PagedPiece* rec;
    long long ldo, ldq;
    int n_kv;
    int box, stages;         // positions of a copy
    float sc2;               // scale * log2(e) * 2^73
};
__host__ __device__ constexpr int stage_bytes(int hd) { return kTok / 8 * Q4Unit(hd).bytes; }
__host__ __device__ constexpr int q_bytes(int hd, int nt) { return nt * 8 * hd * 2; }  // queries of a block, which there are two of
constexpr int rows_area(int hd, int rb) { return kWarps * rb * hd * 4; }

// positions that all rows of a block see: below `hi`, the first row's end, and from `lo` on, where the last row's window begins, or below `first`
struct Sure {
    int hi, lo, first;
    __device__ __forceinline__ Sure(const PagedPiece& pc, const PagedPlan& pl, int cap) {
        hi = min(pc.len - pc.n + pc.b * pl.tb + 1, cap), lo = pl.window > 0 ? pc.len - pc.n + min(pc.n, (pc.b + 1) * pl.tb) - pl.window : 0, first = pl.window > 0 ? pl.first : 0;
    }
};
__device__ __forceinline__ uint16_t* out_row(const Q4Args& a, const PagedPlan& pl, const PagedPiece& pc, int kvh, int r, int hd) {
    return a.out + (pc.q0 + pc.b * pl.tb + r / pl.group) * a.ldo + (long long)(kvh * pl.group + r % pl.group) * hd;
}
__device__ __forceinline__ void put_row(uint16_t* p, float4 v, float l, bool vec) {
    const float f      = l == 0.f ? 0.f : 1.f / l;
    const uint32_t lo = pack_bf16x2(v.x * f, v.y * f), hi = pack_bf16x2(v.z * f, v.w * f);
    if (vec) *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
    else p[0] = lo & 0xffff, p[1] = lo >> 16, p[2] = hi & 0xffff, p[3] = hi >> 16;
}

template <int HD, int NT, int OCC>
__global__ void __launch_bounds__((kWarps + 1) * 32, OCC)
    kf_attn_paged_q4_kernel(const __grid_constant__ Q4Args a, const __grid_constant__ KfPaged pg_, const __grid_constant__ PagedPlan pl, const __grid_constant__ KfBound bound) {
    constexpr Q4Unit un(HD);
    constexpr int G = un.groups, UNIT = un.bytes, STAGE = stage_bytes(HD), QB = q_bytes(HD, NT);
    extern __shared__ __align__(128) uint8_t ring[];
    uint8_t* s_q = ring + (size_t)a.stages * STAGE;              // [2][8 NT][HD] queries
    float* s_o   = reinterpret_cast<float*>(s_q + 2 * QB);       // [kWarps][rb][HD]
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], q_full[2], q_empty[2], meet_bar;
    __shared__ volatile int dead;
    __shared__ int s_there[kMaxStages];  // bit i: positions 8 i .. 8 i + 7 of the tile are there; bit 31: all are, and all rows of the block see them
    __shared__ PagedQueue qu;
    __shared__ float s_m[kWarps][8 * NT], s_l[kWarps][8 * NT];
    __shared__ uint4 s_qb[NT == 1 ? 1 : NT * G][32];  // 9 .. 16 rows: the operands of q, which the warps' registers do not hold beside the sums

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    if (tid == 0) {
        for (int s = 0; s < a.stages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], kWarps);
        for (int s = 0; s < 2; s++) mbar_init(&q_full[s], 1), mbar_init(&q_empty[s], kWarps);
        mbar_init(&meet_bar, kWarps);
        qu.init(kWarps);
        dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    kf_grid_launch_dependents();
    int team = (int)blockIdx.x / a.n_kv, kvh = (int)blockIdx.x % a.n_kv, teams = (int)gridDim.x / a.n_kv, n_box = kTok / a.box;
    asm volatile("" : "+r"(team), "+r"(kvh), "+r"(teams), "+r"(n_box));  // worked out ahead of the wait: divisions
    kf_grid_dependency_wait();  // queries, the new positions' codes, lengths and tables, workspace
    const KfPaged pg    = behind_wait(pg_);
    const uint16_t* q   = behind_wait(a.q);
    PagedPiece* rec = a.rec + kvh * teams;  // by team
    const int group = pl.group, rb = pl.tb * group;
    if (pg.n_seq > 32) {
        PagedPlanner<kTok>::count(pg, pl, qu.s_sum, warp, kWarps + 1, lane);
        __syncthreads();
    }
    PagedReader reader;
    PagedPiece pc;
    bool live = true;
    if (warp == kWarps) {
        // One warp works the pieces out and loads their tiles, up to a ring ahead of the others
        PagedPlanner<kTok> plan(pg, pl, lane);
        if (lane == 0) rec[team].last = 0;  // nothing to merge, should a wait run out before the end of the run is known
        plan.start(qu, team);
        if (bound.drop == (int)blockIdx.x + 1) {
            while (plan.push(qu, team, rec, &dead, bound)) {}
            return;
        }
        uint32_t st = 0, ph = 0, asked = 0, qn = 0;
        // A lane per box (page, or part of one) of several tiles: the pages of the next 32 boxes are looked up while those before are copied.  A look-up takes about as long as
        // a tile
        const int units = a.box / 8, ahead = 32 / n_box, bx = lane % n_box, mine = lane < ahead * n_box ? lane / n_box : 1 << 24;
        const uint32_t bytes = (uint32_t)(units * UNIT);
        uint8_t* dst         = ring + bx * units * UNIT;
        while (live && plan.push(qu, team, rec, &dead, bound)) {
            pc           = plan.pc;
            const int fs = pc.lo > 0 ? pl.first : 0;
            int next_row = 0;
            auto page_of = [&](int t) {
                const int p = pc.tile(t) * kTok + bx * a.box;
                return t < pc.t1 && p < pc.hi && (p + a.box > pc.lo || p < fs) ? paged_page(pg, pc.s, p, next_row) : -1;
            };
            const Sure sure(pc, pl, pg.cap);
            int next = page_of(pc.t0 + mine);
            // the block's queries, a token to a lane
            const int tok0 = pc.b * pl.tb, toks = min(pl.tb, pc.n - tok0);
            if (!(live = mbar_wait_warp(smem_u32(&q_empty[qn & 1]), ((qn >> 1) & 1) ^ 1, &dead, bound))) break;
            if (lane == 0) mbar_arrive_expect_tx(&q_full[qn & 1], (uint32_t)(toks * group * HD * 2));
            __syncwarp();
            if (lane < toks) bulk_load(s_q + (qn & 1) * QB + lane * group * HD * 2, q + (pc.q0 + tok0 + lane) * a.ldq + (long long)kvh * group * HD, (uint32_t)(group * HD * 2), &q_full[qn & 1]);
            __syncwarp();
            qn++;
            for (int t0 = pc.t0; live && t0 < pc.t1; t0 += ahead) {
                const int page = next, row = next_row, n = min(ahead, pc.t1 - t0);
                next = page_of(t0 + ahead + mine);
                const uint8_t* src   = a.pool + page * a.page_stride + ((long long)kvh * (pg.page / 8) + row / 8) * UNIT;
                const unsigned has = page >= 0 ? ((1u << units) - 1u) << (bx * units) : 0u;  // units of its tile that the lane brings
                for (int i = 0; i < n; i++) {
                    const unsigned there = __reduce_or_sync(0xffffffffu, mine == i ? has : 0u);
                    if (!(live = mbar_wait_warp(smem_u32(&empty[st]), ph ^ 1, &dead, bound))) break;
                    if (lane == 0) {
                        const int p0 = pc.tile(t0 + i) * kTok;
                        s_there[st]  = (int)(there == (1u << kTok / 8) - 1u && p0 + kTok <= sure.hi && (p0 >= sure.lo || p0 + kTok <= sure.first) ? there | 1u << 31 : there);
                        mbar_arrive_expect_tx(&full[st], (uint32_t)__popc(there) * UNIT);
                    }
                    __syncwarp();
                    if (mine == i && page >= 0) bulk_load(dst + st * STAGE, src, bytes, &full[st]);
                    __syncwarp();
                    asked++;
                    if (++st == (uint32_t)a.stages) st = 0, ph ^= 1;
                }
            }
        }
        // copies in flight write shared memory, which is another's once the CTA has ended, and where a wait has run out nobody else may have waited for them
        for (uint32_t k = qn > 2 ? qn - 2 : 0; k < qn; k++) mbar_drain(smem_u32(&q_full[k & 1]), (k >> 1) & 1, bound);
        for (uint32_t k = asked > (uint32_t)a.stages ? asked - a.stages : 0; k < asked; k++) mbar_drain(smem_u32(&full[k % a.stages]), (k / a.stages) & 1, bound);
        return;
    }
    const bool vec = ((uintptr_t)a.out & 7) == 0 && a.ldo % 4 == 0;
    uint32_t mph = 0, st = 0, ph = 0, qn = 0;
    auto meet = [&]() {  // all computing warps; bounded like every wait
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet_bar);
        live = mbar_wait_warp(smem_u32(&meet_bar), mph, &dead, bound) && live;
        mph ^= 1;
    };
    while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
        const int rows = min(pl.tb, pc.n - pc.b * pl.tb) * group, fs = pc.lo > 0 ? pl.first : 0;
        // The block's queries as B operands.  Slot pairs of a lane's words: entries (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16 of its 8 of every group, times 2^60; rows past the end: zero
        uint32_t qb[NT == 1 ? G : 1][4], qz[NT][NT == 1 ? G : 1][2];  // qz: minus the sum of q over a group, times 2^-73, as three numbers in the lanes t4 of the group's number
        uint32_t toks = 0;                 // tokens of the lane's columns, eight bits each
        if (!(live = mbar_wait_warp(smem_u32(&q_full[qn & 1]), (qn >> 1) & 1, &dead, bound))) break;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = n * 8 + g;
            const uint8_t* qp = s_q + (qn & 1) * QB + r * HD * 2;
            float mine = 0.f;
#pragma unroll
            for (int j = 0; j < G; j++) {
                uint4 w = *reinterpret_cast<const uint4*>(qp + (32 * j + 8 * t4) * 2);
                if (r >= rows) w = make_uint4(0u, 0u, 0u, 0u);
                const float e[8] = {bf16lo(w.x), bf16hi(w.x), bf16lo(w.y), bf16hi(w.y), bf16lo(w.z), bf16hi(w.z), bf16lo(w.w), bf16hi(w.w)};
                float sum = 0.f;
                uint32_t x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float f = i & 1 ? 0x1p56f : 0x1p60f;
                    x[i] = pack_bf16x2(e[i] * f, e[i + 4] * f);
                    if constexpr (NT == 1) qb[j][i] = x[i];
                    sum += e[i] + e[i + 4];
                }
                if (NT > 1 && warp == (n * G + j) % kWarps) s_qb[n * G + j][lane] = make_uint4(x[0], x[1], x[2], x[3]);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1), sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (t4 == j) mine = sum;
            }
            mine *= -0x1p-73f;
            const float hi = __bfloat162float(__float2bfloat16_rn(mine)), mid = __bfloat162float(__float2bfloat16_rn(mine - hi));
#pragma unroll
            for (int j = 0; j < (NT == 1 ? G : 1); j++)  // registers allow it for 8 rows; otherwise chosen as they are used
                qz[n][j][0] = NT == 2 || t4 == j ? pack_bf16x2(hi, mid) : 0u, qz[n][j][1] = NT == 2 || t4 == j ? pack_bf16x2(mine - hi - mid, 0.f) : 0u;
#pragma unroll
            for (int e = 0; e < 2; e++) toks |= (uint32_t)((n * 8 + 2 * t4 + e) / group) << (8 * (2 * n + e));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[qn & 1]);
        qn++;
        if (NT > 1) meet();
        if (!live) break;
        const Sure sure(pc, pl, pg.cap);
        float o[NT][G][2][4], oz[NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < G; j++)
#pragma unroll
                for (int i = 0; i < 8; i++) o[n][j][i >> 2][i & 3] = 0.f;
            oz[n][0] = oz[n][1] = oz[n][2] = oz[n][3] = 0.f;
            m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
        }
        const int place = pc.len - pc.n + pc.b * pl.tb;  // position of the block's first token
        for (int t = pc.t0; t < pc.t1; t++) {
            if (!(live = mbar_wait_warp(smem_u32(&full[st]), ph, &dead, bound))) break;
            const unsigned there_ = (unsigned)*(volatile int*)&s_there[st];
            const bool fine       = (int)there_ < 0;
            int tok0 = 0;  // this warp's positions and which of their units are there, where that is not all
            unsigned there = 0;
            bool any = true;
            if (!fine) {
                tok0  = pc.tile(t) * kTok + warp * 16 * kSub;
                there = (there_ >> (warp * 2 * kSub)) & ((1u << (2 * kSub)) - 1u);
                any   = there && tok0 < pc.hi && (tok0 + 16 * kSub > pc.lo || tok0 < fs);
            }
            if (any) {
                const uint8_t* u0 = ring + st * STAGE + warp * 2 * kSub * UNIT;  // their units
                const bool ragged = !fine && (there != (1u << (2 * kSub)) - 1u || tok0 + 16 * kSub > sure.hi || (tok0 < sure.lo && tok0 + 16 * kSub > sure.first));
                // ---- scores, transposed: rows are positions g of two units, columns the block's rows ----
                float sc[kSub][NT][4];
#pragma unroll
                for (int b = 0; b < kSub; b++) {
                    uint32_t kw[2][G], kz[2], ks[2][G / 2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint8_t* u = u0 + (2 * b + e) * UNIT;
                        words(u + lane * 4 * G, kw[e]), words(u + un.k_step() + g * 2 * G, ks[e]);
                        kz[e] = *reinterpret_cast<const uint16_t*>(u + un.k_zero() + (g * G + t4 % G) * 2) * 0x10001u;
                    }
                    const uint32_t az[4] = {kz[0], kz[1], kz[0], kz[1]};
#pragma unroll
                    for (int j = 0; j < G; j++) {
                        uint32_t c0[4], c1[4];
                        codes(kw[0][j], c0), codes(kw[1][j], c1);
                        const uint32_t a0[4] = {c0[0], c1[0], c0[1], c1[1]}, a1[4] = {c0[2], c1[2], c0[3], c1[3]};
                        const float s0 = half_of(ks[0][j / 2], j & 1), s1 = half_of(ks[1][j / 2], j & 1);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float acc[4];
                            if constexpr (NT == 1) {
                                mma_new(acc, az, qz[n][j][0], qz[n][j][1]);
                                mma(acc, a0, qb[j][0], qb[j][1]), mma(acc, a1, qb[j][2], qb[j][3]);
                            } else {
                                const uint4 x = s_qb[n * G + j][lane];
                                mma_new(acc, az, t4 == j ? qz[n][0][0] : 0u, t4 == j ? qz[n][0][1] : 0u);
                                mma(acc, a0, x.x, x.y), mma(acc, a1, x.z, x.w);
                            }
#pragma unroll
                            for (int i = 0; i < 4; i++) sc[b][n][i] = j == 0 ? (i < 2 ? s0 : s1) * acc[i] : fmaf(i < 2 ? s0 : s1, acc[i], sc[b][n][i]);
                        }
                    }
                }
                // ---- weights, times 2^60 ----
                unsigned ok = ~0u;  // bit 2 b + e: somebody may see the lane's position, and it is there
                if (ragged) {
#pragma unroll
                    for (int e = 0; e < 2 * kSub; e++) {
                        const int p = tok0 + 8 * e + g;
                        if (!(p < pc.hi && (p >= pc.lo || p < fs) && (there >> e & 1))) ok &= ~(1u << e);
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const int at = place + (int)(toks >> (8 * (2 * n + i)) & 255u);  // the column's position
                                if (!(ok >> e & 1) || p > at || (pl.window > 0 && p <= at - pl.window && p >= pl.first)) sc[e / 2][n][2 * (e & 1) + i] = -INFINITY;
                            }
                    }
                }
                float mx[NT][2];
                bool grown = false;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        mx[n][i] = fmaxf(sc[0][n][i], sc[0][n][2 + i]);
#pragma unroll
                        for (int b = 1; b < kSub; b++) mx[n][i] = fmaxf(mx[n][i], fmaxf(sc[b][n][i], sc[b][n][2 + i]));
                        mx[n][i] *= a.sc2;
                        grown |= mx[n][i] > m[n][i] + kSlack;
                    }
                if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float x = mx[n][i];
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4)), x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8)), x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                            x = fmaxf(x, m[n][i]);
                            const float f = ex2(m[n][i] - finite_or_0(x));
                            m[n][i] = x, l[n][i] *= f, oz[n][i] *= f, oz[n][2 + i] *= f;
#pragma unroll
                            for (int j = 0; j < G; j++) o[n][j][0][i] *= f, o[n][j][0][2 + i] *= f, o[n][j][1][i] *= f, o[n][j][1][2 + i] *= f;
                        }
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float base = 60.f - finite_or_0(m[n][i]);
#pragma unroll
                        for (int b = 0; b < kSub; b++) {
                            float(&p)[4] = sc[b][n];
                            p[i] = ex2(fmaf(p[i], a.sc2, base)), p[2 + i] = ex2(fmaf(p[2 + i], a.sc2, base));
                            l[n][i] += p[i] + p[2 + i];
                        }
                    }
                // ---- sums, transposed: rows are dims ----
#pragma unroll
                for (int b = 0; b < kSub; b++) {
                    uint32_t vs[2][G / 2], vw[2][G], vz[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint8_t* u = u0 + (2 * b + e) * UNIT;
                        words(u + un.v_code() + lane * 4 * G, vw[e]), words(u + un.v_step() + g * 2 * G, vs[e]);
                        vz[e] = smaller(*reinterpret_cast<const uint32_t*>(u + un.v_zero() + (g % G) * 16 + t4 * 4));  // positions 2 t4, 2 t4 + 1 of group g
                    }
                    if (ragged) {  // what no row sees need not be numbers
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            if (!(ok >> (2 * b + e) & 1)) {
#pragma unroll
                                for (int j = 0; j < G / 2; j++) vs[e][j] = 0u;
                            }
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const int pp = tok0 + 8 * (2 * b + e) + 2 * t4 + i;
                                if (!(pp < pc.hi && (pp >= pc.lo || pp < fs) && (there >> (2 * b + e) & 1))) vz[e] &= i ? 0x0000ffffu : 0xffff0000u;
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < G; j++) {
                        uint32_t c0[4], c1[4];
                        codes(__byte_perm(vw[0][j / 2], vw[0][G / 2 + j / 2], j & 1 ? 0x7632 : 0x5410), c0);
                        codes(__byte_perm(vw[1][j / 2], vw[1][G / 2 + j / 2], j & 1 ? 0x7632 : 0x5410), c1);
                        const uint32_t a0[4] = {c0[0], c0[1], c1[0], c1[1]}, a1[4] = {c0[2], c0[3], c1[2], c1[3]};
                        const uint32_t az[4] = {g == j ? vz[0] : 0u, 0u, g == j ? vz[1] : 0u, 0u};
                        const float s0 = half_of(vs[0][j / 2], j & 1), s1 = half_of(vs[1][j / 2], j & 1);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            const float(&p)[4] = sc[b][n];
                            const uint32_t b0 = transpose8x8(pack_bf16x2(p[0] * s0, p[1] * s0)), b1 = transpose8x8(pack_bf16x2(p[2] * s1, p[3] * s1));
                            mma(o[n][j][0], a0, b0, b1), mma(o[n][j][1], a1, b0, b1), mma(oz[n], az, b0, b1);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
            if (++st == (uint32_t)a.stages) st = 0, ph ^= 1;
        }
        if (!live) break;
        // ---- the warp's sums in rows; the zeros' sums of group j are in the lanes of row j ----
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float sum = l[n][i];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4), sum += __shfl_xor_sync(0xffffffffu, sum, 8), sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int r = n * 8 + 2 * t4 + i;
                if (g == 0) s_m[warp][r] = m[n][i], s_l[warp][r] = sum * 0x1p-60f;
#pragma unroll
                for (int j = 0; j < G; j++) {
                    const float z = __shfl_sync(0xffffffffu, oz[n][i], j * 4 + t4) * -__uint_as_float((127u - 60u + kZeroLog2) << 23);
                    if (r < rows)
                        *reinterpret_cast<float4*>(s_o + ((size_t)warp * rb + r) * HD + 32 * j + 4 * g) =
                            make_float4(fmaf(o[n][j][0][i], 0x1p73f, z), fmaf(o[n][j][0][2 + i], 0x1p69f, z), fmaf(o[n][j][1][i], 0x1p73f, z), fmaf(o[n][j][1][2 + i], 0x1p69f, z));
                }
            }
        meet();
        if (!live) break;
        // the warps' sums as one, in order: the result, or what is left for the merge -- a CTA has at most one piece that others have begun (slot 0) and one that others go on with (slot 1)
        const size_t slot = (size_t)blockIdx.x * 2 + (pc.first == team);
        for (int idx = tid; idx < rows * (HD / 4); idx += kWarps * 32) {
            const int r = idx / (HD / 4), c = idx % (HD / 4) * 4;
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) top = fmaxf(top, s_m[w][r]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f  = ex2(s_m[w][r] - finite_or_0(top));
                const float4 x = *reinterpret_cast<const float4*>(s_o + ((size_t)w * rb + r) * HD + c);
                sum = fmaf(s_l[w][r], f, sum);
                v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
            }
            if (pc.whole) put_row(out_row(a, pl, pc, kvh, r, HD) + c, v, sum, vec);
            else {
                __stcg(reinterpret_cast<float4*>(a.ws + (slot * rb + r) * HD + c), v);
                if (c == 0) __stcg(a.ws_ml + slot * rb + r, make_float2(top, sum));
            }
        }
        meet();  // the area belongs to the next piece
    }
}

// Blocks that several CTAs share: thread block (n, y) takes rows kMergeRows y .. of the one that begins in run n and goes on behind it, if there is one.  A row's pieces are spread over as many
// warps as there are for it, kAt on their way for each; these meet in order.  One row to 128 threads: 39.3 us for the sequence of 100000 positions; two rows to 256 39.6, all rows to 512 40.2.
constexpr int kMergeWarps = 4, kMergeRows = 1;
template <int HD>
__global__ void __launch_bounds__(kMergeWarps * 32) kf_attn_paged_q4_merge_kernel(const __grid_constant__ PagedPlan pl, const __grid_constant__ Q4Args a) {
    constexpr int VEC = HD / 4, kAt = 8, kSlots = kMergeWarps * 32 / VEC, kSpread = kSlots / kMergeRows;  // HD 64: half a warp to a row
    __shared__ float4 s_v[kSlots][VEC];
    __shared__ float2 s_ml[kSlots];
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();
    const int team = (int)blockIdx.x / a.n_kv, kvh = (int)blockIdx.x % a.n_kv, teams = (int)gridDim.x / a.n_kv;
    const PagedPiece pc = *behind_wait(a.rec + kvh * teams + team);
    const int rb = pl.tb * pl.group, rows = min(pl.tb, pc.n - pc.b * pl.tb) * pl.group, pieces = pc.last - team + 1;
    if (pc.last <= team || pc.last >= teams || (int)blockIdx.y * kMergeRows >= rows) return;  // last 0: nothing that goes on
    const int tid = threadIdx.x, slot = tid / VEC, c = tid % VEC * 4, r = blockIdx.y * kMergeRows + slot / kSpread, part = slot % kSpread;
    if (r < rows && part < pieces) {
        float top = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = part; i0 < pieces; i0 += kAt * kSpread) {
            float4 w[kAt];
            float2 ml[kAt];
#pragma unroll
            for (int k = 0; k < kAt; k++) {
                const int i = i0 + k * kSpread;
                if (i < pieces) {
                    const size_t row = (((size_t)(team + i) * a.n_kv + kvh) * 2 + (i == 0)) * rb + r;
                    w[k] = __ldcg(reinterpret_cast<const float4*>(a.ws + row * HD + c)), ml[k] = __ldcg(a.ws_ml + row);
                } else w[k] = make_float4(0.f, 0.f, 0.f, 0.f), ml[k] = make_float2(-INFINITY, 0.f);
            }
            float n = top;
#pragma unroll
            for (int k = 0; k < kAt; k++) n = fmaxf(n, ml[k].x);
            const float base = finite_or_0(n), f0 = ex2(top - base);
            top = n, sum *= f0, v.x *= f0, v.y *= f0, v.z *= f0, v.w *= f0;
#pragma unroll
            for (int k = 0; k < kAt; k++) {
                const float f = ex2(ml[k].x - base);
                sum = fmaf(ml[k].y, f, sum);
                v.x = fmaf(w[k].x, f, v.x), v.y = fmaf(w[k].y, f, v.y), v.z = fmaf(w[k].z, f, v.z), v.w = fmaf(w[k].w, f, v.w);
            }
        }
        s_v[slot][c / 4] = v;
        if (c == 0) s_ml[slot] = make_float2(top, sum);
    }
    __syncthreads();
    if (r >= rows || part != 0) return;
    const int n = min(kSpread, pieces);
    float top = -INFINITY, sum = 0.f;
    for (int k = 0; k < n; k++) top = fmaxf(top, s_ml[slot + k].x);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < n; k++) {
        const float f  = ex2(s_ml[slot + k].x - finite_or_0(top));
        const float4 x = s_v[slot + k][c / 4];
        sum = fmaf(s_ml[slot + k].y, f, sum);
        v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
    }
    put_row(out_row(a, pl, pc, kvh, r, HD) + c, v, sum, ((uintptr_t)a.out & 7) == 0 && a.ldo % 4 == 0);
}

template <int HD, int NT, int OCC>
int launch_q4(kf_ctx* ctx, const kf_paged_q4* kv, const KfPaged& pg, PagedPlan pl, Q4Args a, float scale) {
    constexpr int kStage = stage_bytes(HD);
    const int teams = std::max(1, OCC * ctx->sm_count / a.n_kv), grid = teams * a.n_kv, rb = pl.tb * pl.group;
    const size_t rows = (size_t)grid * 2 * rb;
    pl.runs = teams;
    KF_REQUIRE(ctx, paged_most(kTok, pg, pl) < 0x7fff0000, "as many tiles as M rows over full tables have");
    const int rc = kf_ensure_attn_ws(ctx, rows * (HD + 2) * sizeof(float) + 16 + grid * sizeof(PagedPiece));
    if (rc) return rc;
    a.box = 8;
    while (kTok % (2 * a.box) == 0 && kv->page_size % (2 * a.box) == 0) a.box *= 2;
    constexpr int kBytes = (224 / OCC - 4) * 1024;  // of shared memory for a CTA, its fixed part aside
    const int other      = 2 * q_bytes(HD, NT) + rows_area(HD, rb);
    a.stages             = std::min(kMaxStages, (kBytes - other) / kStage);
    const size_t smem    = (size_t)a.stages * kStage + other;
    a.ws = ctx->attn_ws, a.ws_ml = reinterpret_cast<float2*>(ctx->attn_ws + rows * HD), a.rec = reinterpret_cast<PagedPiece*>(ctx->attn_ws + (rows * (HD + 2) + 3) / 4 * 4);
    a.sc2     = scale * 1.4426950408889634f * 0x1p73f;
    auto kern = kf_attn_paged_q4_kernel<HD, NT, OCC>;
    static bool set[kf_ctx::kMaxDevices] = {};  // function attributes are per device
    if (!set[ctx->device]) {
        KF_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes));
        set[ctx->device] = true;
    }
    KF_CUDA(ctx, kf_launch_pdl(ctx, kern, dim3(grid), dim3((kWarps + 1) * 32), smem, a, pg, pl, KfBound{ctx->wait_flags + kWaitPaged, (unsigned)ctx->attn_wait_us, ctx->attn_drop}));
    KF_LAUNCH_CHECK(ctx);
    KF_CUDA(ctx, kf_launch_pdl(ctx, kf_attn_paged_q4_merge_kernel<HD>, dim3(grid, (rb + kMergeRows - 1) / kMergeRows), dim3(kMergeWarps * 32), 0, pl, a));
    KF_LAUNCH_CHECK(ctx);
    return KF_OK;
}
int check_args(kf_ctx* ctx, const kf_paged_q4* kv, const void* out, int ldo, const void* q, int ldq, int M, int n_head, float scale, int first, int max_q, KfPaged* pg) {
    if (!kv || !out || !q) return KF_ERR_BAD_ARG;
    const int rc = kf_paged_q4_check(ctx, kv, M, pg);
    if (rc) return rc;
    KF_REQUIRE(ctx, n_head >= 1 && n_head % kv->n_kv == 0 && n_head / kv->n_kv <= 64, "n_head a multiple of n_kv, at most 64 heads to a kv head");
    KF_REQUIRE(ctx, (long long)n_head * kv->head_dim <= ldq && (long long)n_head * kv->head_dim <= ldo, "rows as long as their heads");
    KF_REQUIRE(ctx, ((uintptr_t)q & 15) == 0 && ldq % 8 == 0, "q at 16 bytes, ldq a multiple of 8");
    KF_REQUIRE(ctx, ((uintptr_t)out & 1) == 0, "out at 2 bytes");
    KF_REQUIRE(ctx, (long long)M * (n_head / kv->n_kv) < 0x7fffff00, "rows");
    KF_REQUIRE(ctx, scale > 0.f && scale <= 0x1p20f && first >= 0 && max_q >= 0, "scale above 0, at most 2^20; first and max_q not negative");
    const size_t wide = (size_t)n_head * kv->head_dim * 2;
    KF_REQUIRE(ctx, out != q && !kf_rows_overlap(out, (size_t)ldo * 2, wide, q, (size_t)ldq * 2, wide, M), "the result over the queries");
    return KF_OK;
}
}  // namespace

extern "C" int kf_paged_attention_q4(kf_ctx* ctx, const kf_paged_q4* kv, void* out, int ldo, const void* q, int ldq, int M, int n_head, float scale, int window, int first, int max_q) {
    if (!ctx) return KF_ERR_BAD_ARG;
    KfPaged pg;
    int rc = check_args(ctx, kv, out, ldo, q, ldq, M, n_head, scale, first, max_q, &pg);
    if (!rc) rc = kf_wait_status(ctx);
    if (rc || M == 0) return rc;
    const int group = n_head / kv->n_kv, tokens = std::max(1, max_q);
    if (tokens * (long long)group > 16) return kf_attn_paged_q4_tc(ctx, kv, pg, out, ldo, q, ldq, n_head, scale, window, first);
    Q4Args a = {};
    a.pool = (const uint8_t*)kv->pool_dev, a.page_stride = (long long)kf_paged_q4_stride(kv), a.out = (uint16_t*)out, a.q = (const uint16_t*)q, a.ldo = ldo, a.ldq = ldq, a.n_kv = kv->n_kv;
    const PagedPlan pl{tokens, group, window, 1, 0, first};
    if (kv->head_dim == 128) return tokens * group <= 8 ? launch_q4<128, 1, 2>(ctx, kv, pg, pl, a, scale) : launch_q4<128, 2, 2>(ctx, kv, pg, pl, a, scale);
    return tokens * group <= 8 ? launch_q4<64, 1, 3>(ctx, kv, pg, pl, a, scale) : launch_q4<64, 2, 2>(ctx, kv, pg, pl, a, scale);
}
// The checks for tests on a host without a device
extern "C" int kf_paged_attention_q4_args(const kf_paged_q4* kv, const void* out, int ldo, const void* q, int ldq, int M, int n_head, float scale, int first, int max_q) {
    KfPaged pg;
    return check_args(nullptr, kv, out, ldo, q, ldq, M, n_head, scale, first, max_q, &pg);
}
