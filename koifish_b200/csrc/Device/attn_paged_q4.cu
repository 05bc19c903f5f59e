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
//   * A warp takes 16 positions (two units) of a tile of 64; a unit is contiguous (Q4Unit), so a tile is a bulk copy per page (or part of 8, 16, 32 or 64 positions of it).
#include <algorithm>

#include "kf_paged_finish.cuh"

namespace {
constexpr int kTok = 64, kWarps = 4, kMaxStages = 12;
constexpr float kSlack = 8.f;  // growth of a maximum, log2, that sums are not rescaled for

// bytes from global into shared memory, both at 16 bytes, a multiple of 16
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// pairs of codes out of a word: nibbles (0, 4), (1, 5), (2, 6), (3, 7); the second and the fourth stand for 16 times their codes
__device__ __forceinline__ void codes(uint32_t w, uint32_t (&c)[4]) { c[0] = w & 0x000f000fu, c[1] = w & 0x00f000f0u, c[2] = (w >> 8) & 0x000f000fu, c[3] = (w >> 8) & 0x00f000f0u; }

struct Q4Args {  // kernel parameter
    const uint8_t* pool;
    long long page_stride;
    uint16_t* out;
    const uint16_t* q;
    float* ws;
    float2* ws_ml;
    unsigned* cnt;
    long long ldo, ldq;
    int n_kv, parts, heads;  // a kv head's group in `parts` of up to `heads` heads, a CTA of the team each
    int box, stages;         // positions of a copy
    float sc2;               // scale * log2(e) * 2^73
};
__host__ __device__ constexpr int stage_bytes(int hd) { return kTok / 8 * Q4Unit(hd).bytes; }
constexpr int rows_area(int hd, int rb) { return kWarps * rb * hd * 4; }

template <int HD, int NT, int OCC>
__global__ void __launch_bounds__((kWarps + 2) * 32, OCC)
    kf_attn_paged_q4_kernel(const __grid_constant__ Q4Args a, const __grid_constant__ KfPaged pg_, const __grid_constant__ PagedPlan pl, const __grid_constant__ KfBound bound) {
    constexpr Q4Unit un(HD);
    constexpr int G = un.groups, UNIT = un.bytes, STAGE = stage_bytes(HD);
    extern __shared__ __align__(128) uint8_t ring[];
    float* s_o = reinterpret_cast<float*>(ring + (size_t)a.stages * STAGE);  // [kWarps][rb][HD]
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], meet_bar;
    __shared__ volatile int dead;
    __shared__ int s_there[kMaxStages], s_last;  // bit i: positions 8 i .. 8 i + 7 of the tile are there
    __shared__ PagedQueue qu;
    __shared__ float s_m[kWarps][16], s_l[kWarps][16];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    if (tid == 0) {
        for (int s = 0; s < a.stages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], kWarps);
        mbar_init(&meet_bar, kWarps);
        qu.init(kWarps + 1);
        dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();  // queries, the new positions' codes, lengths and tables, workspace
    const KfPaged pg    = behind_wait(pg_);
    const uint16_t* q   = behind_wait(a.q);
    const int mates = a.n_kv * a.parts, team = (int)blockIdx.x / mates, mate = (int)blockIdx.x % mates, kvh = mate / a.parts, h0 = mate % a.parts * a.heads;
    if (pg.n_seq > 32) {
        PagedPlanner<kTok>::count(pg, pl, qu.s_sum, warp, kWarps + 2, lane);
        __syncthreads();
    }
    if (warp == kWarps + 1) {
        PagedPlanner<kTok> plan(pg, pl, lane);
        plan.start(qu, team);
        while (plan.push(qu, team, nullptr, &dead, bound)) {}
        return;
    }
    PagedReader reader;
    PagedPiece pc;
    bool live = true;
    if (warp == kWarps) {
        if (bound.drop == (int)blockIdx.x + 1) return;
        uint32_t st = 0, ph = 0, asked = 0;
        const int n_box = kTok / a.box, bx = lane;  // a lane per box; bx >= n_box: none
        const uint32_t bytes = (uint32_t)(a.box / 8 * UNIT);
        while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
            const int fs = pc.lo > 0 ? pl.first : 0;
            int next_row = 0;
            auto page_of = [&](int t) {  // the page of this lane's box of tile t
                const int p = pc.tile(t) * kTok + bx * a.box;
                return t < pc.t1 && bx < n_box && p < pc.hi && (p + a.box > pc.lo || p < fs) ? paged_page(pg, pc.s, p, next_row) : -1;
            };
            int next = page_of(pc.t0);
            for (int t = pc.t0; live && t < pc.t1; t++) {
                const int page = next, row = next_row;
                next = page_of(t + 1);  // a tile ahead: the look-up takes as long as a tile
                const unsigned lanes = __ballot_sync(0xffffffffu, page >= 0);
                if (!(live = mbar_wait_warp(smem_u32(&empty[st]), ph ^ 1, &dead, bound))) break;
                if (lane == 0) {
                    unsigned there = 0;
                    for (int i = 0; i < kTok / 8; i++) there |= (lanes >> (i * 8 / a.box) & 1) << i;
                    s_there[st] = (int)there;
                    mbar_arrive_expect_tx(&full[st], (uint32_t)__popc(lanes) * bytes);
                }
                __syncwarp();
                if (page >= 0)
                    bulk_load(ring + (size_t)st * STAGE + bx * a.box / 8 * UNIT, a.pool + page * a.page_stride + ((long long)kvh * (pg.page / 8) + row / 8) * UNIT, bytes, &full[st]);
                __syncwarp();
                asked++;
                if (++st == (uint32_t)a.stages) st = 0, ph ^= 1;
            }
        }
        // copies in flight write shared memory, which is another's once the CTA has ended, and where a wait has run out nobody else may have waited for them
        for (uint32_t k = asked > (uint32_t)a.stages ? asked - a.stages : 0; k < asked; k++) mbar_drain(smem_u32(&full[k % a.stages]), (k / a.stages) & 1, bound);
        return;
    }
    const int group = pl.group, rb = pl.tb * a.heads, heads = min(a.heads, group - h0);
    const bool vec = ((uintptr_t)a.out & 7) == 0 && a.ldo % 4 == 0;
    uint32_t mph = 0, st = 0, ph = 0;
    auto meet = [&]() {  // all computing warps; bounded like every wait
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet_bar);
        live = mbar_wait_warp(smem_u32(&meet_bar), mph, &dead, bound) && live;
        mph ^= 1;
    };
    while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
        const int rows = min(pl.tb, pc.n - pc.b * pl.tb) * heads, fs = pc.lo > 0 ? pl.first : 0;
        // The block's queries as B operands.  Slot pairs of a lane's words: entries (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16 of its 8 of every group, times 2^60; rows past the end: zero
        uint32_t qb[NT][G][4], qz[NT][2];  // qz: minus the sum of q over group t4, times 2^-73, as three numbers
        int lim[NT][2], low[NT][2];        // what the lane's columns see: positions above `low`, or of the first, up to `lim`
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = n * 8 + g, tok = pc.b * pl.tb + r / heads;
            const uint16_t* qp = q + (pc.q0 + tok) * a.ldq + (long long)(kvh * group + h0 + r % heads) * HD;
            float mine = 0.f;
#pragma unroll
            for (int j = 0; j < G; j++) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (r < rows) w = *reinterpret_cast<const uint4*>(qp + 32 * j + 8 * t4);
                const float e[8] = {bf16lo(w.x), bf16hi(w.x), bf16lo(w.y), bf16hi(w.y), bf16lo(w.z), bf16hi(w.z), bf16lo(w.w), bf16hi(w.w)};
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float f = i & 1 ? 0x1p56f : 0x1p60f;
                    qb[n][j][i] = pack_bf16x2(e[i] * f, e[i + 4] * f);
                    sum += e[i] + e[i + 4];
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1), sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (t4 % G == j) mine = sum;
            }
            mine *= -0x1p-73f;
            const float hi = __bfloat162float(__float2bfloat16_rn(mine)), mid = __bfloat162float(__float2bfloat16_rn(mine - hi));
            qz[n][0] = t4 < G ? pack_bf16x2(hi, mid) : 0u, qz[n][1] = t4 < G ? pack_bf16x2(mine - hi - mid, 0.f) : 0u;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int tc = pc.b * pl.tb + (n * 8 + 2 * t4 + e) / heads;
                lim[n][e] = min(pc.len - pc.n + tc, pg.cap - 1), low[n][e] = pl.window > 0 ? pc.len - pc.n + tc - pl.window : -1;
            }
        }
        // positions that all rows see: below the first row's, and above the last row's window or of the first
        const int sure_hi = min(pc.len - pc.n + pc.b * pl.tb + 1, pg.cap), sure_lo = pl.window > 0 ? pc.len - pc.n + min(pc.n, (pc.b + 1) * pl.tb) - pl.window : 0;
        const int fw = pl.window > 0 ? pl.first : 0;
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
        for (int t = pc.t0; t < pc.t1; t++) {
            if (!(live = mbar_wait_warp(smem_u32(&full[st]), ph, &dead, bound))) break;
            const int tok0 = pc.tile(t) * kTok + warp * 16;  // this warp's 16 positions
            const unsigned there = ((unsigned)*(volatile int*)&s_there[st] >> (warp * 2)) & 3u;
            if (there && tok0 < pc.hi && (tok0 + 16 > pc.lo || tok0 < fs)) {
                const uint32_t u0 = smem_u32(ring + (size_t)st * STAGE + warp * 2 * UNIT);  // the two units
                const bool ragged = there != 3u || tok0 + 16 > sure_hi || (tok0 < sure_lo && tok0 + 16 > fw);
                // ---- scores, transposed: rows are positions g of both units, columns the block's rows ----
                float sc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; n++) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
                {
                    uint32_t kw[2][G], kz[2], ks[2][G / 2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t u = u0 + e * UNIT;
                        if constexpr (G == 4) lds128(u + lane * 16, kw[e]), lds64(u + un.k_step() + g * 8, ks[e]);
                        else {
                            lds64(u + lane * 8, kw[e]);
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(ks[e][0]) : "r"(u + un.k_step() + g * 4) : "memory");
                        }
                        uint16_t z;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(z) : "r"(u + un.k_zero() + (g * G + t4 % G) * 2) : "memory");
                        kz[e] = z | (uint32_t)z << 16;
                    }
                    const uint32_t az[4] = {kz[0], kz[1], kz[0], kz[1]};
#pragma unroll
                    for (int j = 0; j < G; j++) {
                        uint32_t c0[4], c1[4];
                        codes(kw[0][j], c0), codes(kw[1][j], c1);
                        const uint32_t a0[4] = {c0[0], c1[0], c0[1], c1[1]}, a1[4] = {c0[2], c1[2], c0[3], c1[3]};
                        const float s0 = j & 1 ? bf16hi(ks[0][j / 2]) : bf16lo(ks[0][j / 2]), s1 = j & 1 ? bf16hi(ks[1][j / 2]) : bf16lo(ks[1][j / 2]);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float acc[4] = {0.f, 0.f, 0.f, 0.f};
                            mma16816(acc, az, t4 == j ? qz[n][0] : 0u, t4 == j ? qz[n][1] : 0u);
                            mma16816(acc, a0, qb[n][j][0], qb[n][j][1]);
                            mma16816(acc, a1, qb[n][j][2], qb[n][j][3]);
                            sc[n][0] = fmaf(s0, acc[0], sc[n][0]), sc[n][1] = fmaf(s0, acc[1], sc[n][1]);
                            sc[n][2] = fmaf(s1, acc[2], sc[n][2]), sc[n][3] = fmaf(s1, acc[3], sc[n][3]);
                        }
                    }
                }
                // ---- weights, times 2^60 ----
                bool ok[2] = {true, true};  // somebody may see the lane's positions, and they are there
                if (ragged) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int p = tok0 + 8 * e + g;
                        ok[e] = p < pc.hi && (p >= pc.lo || p < fs) && (there >> e & 1);
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int i = 0; i < 2; i++)
                                if (!ok[e] || p > lim[n][i] || (p <= low[n][i] && p >= fw)) sc[n][2 * e + i] = -INFINITY;
                    }
                }
                bool grown = false;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) grown |= fmaxf(sc[n][i], sc[n][2 + i]) * a.sc2 > m[n][i] + kSlack;
                if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float mx = fmaxf(sc[n][i], sc[n][2 + i]) * a.sc2;
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4)), mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8)), mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            mx = fmaxf(mx, m[n][i]);
                            const float f = ex2(m[n][i] - finite_or_0(mx));
                            m[n][i] = mx, l[n][i] *= f, oz[n][i] *= f, oz[n][2 + i] *= f;
#pragma unroll
                            for (int j = 0; j < G; j++) o[n][j][0][i] *= f, o[n][j][0][2 + i] *= f, o[n][j][1][i] *= f, o[n][j][1][2 + i] *= f;
                        }
                }
                float p[NT][4];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float base = finite_or_0(m[n][i]) - 60.f;
                        p[n][i] = ex2(fmaf(sc[n][i], a.sc2, -base)), p[n][2 + i] = ex2(fmaf(sc[n][2 + i], a.sc2, -base));
                        l[n][i] += p[n][i] + p[n][2 + i];
                    }
                // ---- sums, transposed: rows are dims ----
                uint32_t vs[2][G / 2], vw[2][G], vz[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t u = u0 + e * UNIT;
                    if constexpr (G == 4) lds128(u + un.v_code() + lane * 16, vw[e]), lds64(u + un.v_step() + g * 8, vs[e]);
                    else {
                        lds64(u + un.v_code() + lane * 8, vw[e]);
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(vs[e][0]) : "r"(u + un.v_step() + g * 4) : "memory");
                    }
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(vz[e]) : "r"(u + un.v_zero() + (g % G) * 16 + t4 * 4) : "memory");  // positions 2 t4, 2 t4 + 1 of group g
                }
                if (ragged) {  // what no row sees need not be numbers
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        if (!ok[e]) {
#pragma unroll
                            for (int j = 0; j < G / 2; j++) vs[e][j] = 0u;
                        }
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int pp = tok0 + 8 * e + 2 * t4 + i;
                            if (!(pp < pc.hi && (pp >= pc.lo || pp < fs) && (there >> e & 1))) vz[e] &= i ? 0x0000ffffu : 0xffff0000u;
                        }
                    }
                }
#pragma unroll
                for (int w = 0; w < G / 2; w++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {  // group 2 w + h
                        const int j = 2 * w + h;
                        uint32_t c0[4], c1[4];
                        codes(__byte_perm(vw[0][w], vw[0][G / 2 + w], h ? 0x7632 : 0x5410), c0);
                        codes(__byte_perm(vw[1][w], vw[1][G / 2 + w], h ? 0x7632 : 0x5410), c1);
                        const uint32_t a0[4] = {c0[0], c0[1], c1[0], c1[1]}, a1[4] = {c0[2], c0[3], c1[2], c1[3]};
                        const uint32_t az[4] = {g == j ? vz[0] : 0u, 0u, g == j ? vz[1] : 0u, 0u};
                        const float s0 = h ? bf16hi(vs[0][w]) : bf16lo(vs[0][w]), s1 = h ? bf16hi(vs[1][w]) : bf16lo(vs[1][w]);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            const uint32_t b0 = transpose8x8(pack_bf16x2(p[n][0] * s0, p[n][1] * s0)), b1 = transpose8x8(pack_bf16x2(p[n][2] * s1, p[n][3] * s1));
                            mma16816(o[n][j][0], a0, b0, b1);
                            mma16816(o[n][j][1], a1, b0, b1);
                            mma16816(oz[n], az, b0, b1);
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
                    const float z = __shfl_sync(0xffffffffu, oz[n][i], j * 4 + t4) * -0x1p-60f;
                    if (r < rows)
                        *reinterpret_cast<float4*>(s_o + ((size_t)warp * rb + r) * HD + 32 * j + 4 * g) =
                            make_float4(fmaf(o[n][j][0][i], 0x1p73f, z), fmaf(o[n][j][0][2 + i], 0x1p69f, z), fmaf(o[n][j][1][i], 0x1p73f, z), fmaf(o[n][j][1][2 + i], 0x1p69f, z));
                }
            }
        meet();
        if (!live) break;
        auto out_row = [&](int r) {
            return a.out + (pc.q0 + pc.b * pl.tb + r / heads) * a.ldo + (long long)(kvh * group + h0 + r % heads) * HD;
        };
        paged_finish<HD, kWarps>(pc, PagedSums{team, mate, mates, a.ws, a.ws_ml, a.cnt}, rows, rb, s_o, s_m, s_l, &s_last, vec, live, out_row, meet);
        meet();  // the area belongs to the next piece
    }
}

template <int HD, int NT, int OCC>
int launch_q4(kf_ctx* ctx, const kf_paged_q4* kv, const KfPaged& pg, PagedPlan pl, Q4Args a, float scale) {
    const int mates = a.n_kv * a.parts, teams = std::max(1, OCC * ctx->sm_count / mates), grid = teams * mates, rb = pl.tb * a.heads;
    const size_t rows = (size_t)grid * 2 * rb;
    pl.runs = teams;
    KF_REQUIRE(ctx, paged_most(kTok, pg, pl) < 0x7fff0000, "as many tiles as M rows over full tables have");
    int rc = kf_ensure_attn_ws(ctx, rows * (HD + 2) * sizeof(float));
    if (!rc) rc = kf_ensure_attn_cnt(ctx, grid);
    if (rc) return rc;
    a.box = 8;
    while (a.box < kTok && kv->page_size % (2 * a.box) == 0) a.box *= 2;
    constexpr int kBytes = (224 / OCC - 4) * 1024;  // of shared memory for a CTA, its fixed part aside
    a.stages             = std::min(kMaxStages, (kBytes - rows_area(HD, rb)) / stage_bytes(HD));
    const size_t smem    = (size_t)a.stages * stage_bytes(HD) + rows_area(HD, rb);
    a.ws = ctx->attn_ws, a.ws_ml = reinterpret_cast<float2*>(ctx->attn_ws + rows * HD), a.cnt = ctx->attn_cnt;
    a.sc2     = scale * 1.4426950408889634f * 0x1p73f;
    auto kern = kf_attn_paged_q4_kernel<HD, NT, OCC>;
    static bool set[kf_ctx::kMaxDevices] = {};  // function attributes are per device
    if (!set[ctx->device]) {
        KF_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes));
        set[ctx->device] = true;
    }
    KF_CUDA(ctx, kf_launch_pdl(ctx, kern, dim3(grid), dim3((kWarps + 2) * 32), smem, a, pg, pl, KfBound{ctx->wait_flags + kWaitPaged, (unsigned)ctx->attn_wait_us, ctx->attn_drop}));
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
    const int group = n_head / kv->n_kv;
    Q4Args a = {};
    a.pool = (const uint8_t*)kv->pool_dev, a.page_stride = (long long)kf_paged_q4_stride(kv), a.out = (uint16_t*)out, a.q = (const uint16_t*)q, a.ldo = ldo, a.ldq = ldq, a.n_kv = kv->n_kv;
    a.parts = (group + 15) / 16, a.heads = (group + a.parts - 1) / a.parts;
    const int tokens = std::max(1, std::min(std::max(1, max_q), 16 / a.heads));
    const PagedPlan pl{tokens, group, window, 1, 0, first};
    if (kv->head_dim == 128) return tokens * a.heads <= 8 ? launch_q4<128, 1, 2>(ctx, kv, pg, pl, a, scale) : launch_q4<128, 2, 2>(ctx, kv, pg, pl, a, scale);
    return tokens * a.heads <= 8 ? launch_q4<64, 1, 3>(ctx, kv, pg, pl, a, scale) : launch_q4<64, 2, 2>(ctx, kv, pg, pl, a, scale);
}
// The checks for tests on a host without a device
extern "C" int kf_paged_attention_q4_args(const kf_paged_q4* kv, const void* out, int ldo, const void* q, int ldq, int M, int n_head, float scale, int first, int max_q) {
    KfPaged pg;
    return check_args(nullptr, kv, out, ldo, q, ldq, M, n_head, scale, first, max_q, &pg);
}
