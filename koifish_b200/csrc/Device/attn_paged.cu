// attn_paged.cu -- attention of a step's rows over a cache in pages (kf_paged_attention): the kernel for steps whose sequences have up to 16 rows a kv head (new tokens x heads
// of its group), and the choice between it and the one for more (attn_paged_tc.cu).
//
//   out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q.k_j - m),  c = scale * log2(e),  m the largest c q.k_j so far, over the positions j that the row sees
//
// Every cached row is read once per kv head for all rows of a block, so the bytes of the cache bound it; what matters is how many of them are on their way and that no SM
// runs dry.
//   * A team of n_kv CTAs takes a run of tiles of 64 positions, a kv head each, so that the rows of a position, which lie side by side, are read at about the same time.
//     The runs are equal whatever the sequences' lengths are (PagedWalk).
//   * One warp looks the pages up and loads tiles of K and V by TMA into a ring of stages; a tile is as many boxes as pages (or parts of 8, 16, 32 or 64 positions of
//     them) meet in it, each asked for by a lane of its own.  Boxes of pages that are not there are out of the tensor map's range and arrive as zeros.
//   * Four computing warps take a tile, 16 positions each; scores and P V on mma.sync with the block's rows as the 16 rows of the A operand.
//   * The piece that arrives last at its block merges all of them in order, a row to a warp with eight pieces on their way (sums by slices of the threads, maxima looked up
//     first: 17 us of 85 for one sequence at 100000 positions, 10 less here).
//   * Two CTAs of four warps per SM: one's merge runs beside the other's tiles.  (One CTA of eight: 166 against 111 us for 64 sequences, 89 against 76 for one.)
// Measured in a steady run (in brackets: a few dozen passes): 64 sequences of 400 .. 4000 positions, 8 kv heads (624 MB) 117 us, 5.3 TB/s (111 us, 5.6 TB/s); one of 100000
// positions (410 MB) 77 us, 5.3 TB/s (76 us); one of 1300 10.3 us, most of it the way from the lengths over the table to the first tile and the merge.
// Values behind a block's last position or before its window need not be numbers: their rows of V are zeroed in shared memory.
#include <algorithm>

#include "kf_paged_walk.cuh"

namespace {
constexpr int kTok = 64;

__device__ __forceinline__ void put4(uint16_t* p, float4 v, bool vec) {
    if (vec) *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    else p[0] = f32_to_bf16_bits(v.x), p[1] = f32_to_bf16_bits(v.y), p[2] = f32_to_bf16_bits(v.z), p[3] = f32_to_bf16_bits(v.w);
}

// Shared memory of one of two CTAs on an SM: a ring of stages (K and V tiles in turn) and the computing warps' sums.
constexpr int kWarps = 4, kComp = kWarps * 32, kMaxStages = 10, kSmemKB = 108;
constexpr int rows_area(int hd, int rb) { return kWarps * rb * hd * 4; }
constexpr int ring_stages(int hd, int rb) {
    const int fit = (kSmemKB * 1024 - rows_area(hd, rb)) / (kTok * hd * 2);
    return (fit < kMaxStages ? fit : kMaxStages) & ~1;
}
static_assert(ring_stages(128, 16) >= 4, "two tiles in flight");

template <int HD>
__global__ void __launch_bounds__((kWarps + 2) * 32, 2)
    kf_attn_paged_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, uint16_t* out, float* ws, float2* ws_ml, unsigned* cnt, const uint16_t* q,
                         const __grid_constant__ KfPaged pg_, const __grid_constant__ PagedPlan pl, long long ldo, long long ldq, int n_kv, int box /* positions */, int stages,
                         float sc2 /* scale * log2(e) */, const __grid_constant__ KfBound bound) {
    constexpr int PARTS = HD / 64, TILE = kTok * HD * 2, GROUP8 = PARTS * 1024;  // a tile lies as groups of 8 rows, each in parts of 64 dims (kf_tmap_pages)
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* s_o    = reinterpret_cast<float*>(ring + (size_t)stages * TILE);  // [kWarps][rb][HD]
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], meet_bar;
    __shared__ volatile int dead;
    __shared__ int s_there[kMaxStages], s_last;  // bit i: positions 8 i .. 8 i + 7 of the stage's K tile are there
    __shared__ PagedQueue qu;
    __shared__ float s_m[kWarps][16], s_l[kWarps][16];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    if (tid == 0) {
        for (int s = 0; s < stages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], 4);
        mbar_init(&meet_bar, kWarps);
        qu.init(kWarps + 1);
        dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&tm_k), tma_prefetch_map(&tm_v);
    }
    __syncthreads();
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();  // queries, the new positions' rows, lengths and tables, workspace
    const KfPaged pg = behind_wait(pg_);
    q                = behind_wait(q);
    const int team = (int)blockIdx.x / n_kv, kvh = (int)blockIdx.x % n_kv;
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
    uint32_t st = 0, ph = 0;  // ring position and its phase
    if (warp == kWarps) {
        if (bound.drop == (int)blockIdx.x + 1) return;
        uint32_t asked = 0;
        const int n_box = kTok / box, bx = lane;  // a lane per box; bx >= n_box: none
        while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
            int next_row = 0;
            auto page_of = [&](int t) {  // the page of this lane's box of tile t
                const int p = t * kTok + bx * box;
                return t < pc.t1 && bx < n_box && p < pc.hi && p + box > pc.lo ? paged_page(pg, pc.s, p, next_row) : -1;
            };
            int next = page_of(pc.t0);
            for (int t = pc.t0; live && t < pc.t1; t++) {
                const int page = next, row = next_row;
                next = page_of(t + 1);  // a tile ahead: the look-up takes as long as a tile
                const unsigned lanes = __ballot_sync(0xffffffffu, page >= 0);
                for (int kv = 0; kv < 2; kv++) {
                    if (!(live = mbar_wait_warp(smem_u32(&empty[st]), ph ^ 1, &dead, bound))) break;
                    if (lane == 0) {
                        unsigned there = 0;
                        for (int i = 0; i < kTok / 8; i++) there |= (lanes >> (i * 8 / box) & 1) << i;
                        s_there[st] = (int)there;
                        mbar_arrive_expect_tx(&full[st], TILE);
                    }
                    __syncwarp();
                    if (bx < n_box) tma_load_page(ring + (size_t)st * TILE + bx * box * (HD * 2), kv ? &tm_v : &tm_k, kvh * PARTS, page >= 0 ? row / 8 : 0, page >= 0 ? page : pg.n_pages, &full[st]);
                    __syncwarp();
                    asked++;
                    if (++st == (uint32_t)stages) st = 0, ph ^= 1;
                }
            }
        }
        // copies in flight write shared memory, which is another's once the CTA has ended, and where a wait has run out nobody else may have waited for them
        for (uint32_t k = asked > (uint32_t)stages ? asked - stages : 0; k < asked; k++) mbar_drain(smem_u32(&full[k % stages]), (k / stages) & 1, bound);
        return;
    }
    const int group = pl.group, rb = pl.tb * group;
    const bool vec = ((uintptr_t)out & 7) == 0 && ldo % 4 == 0;
    uint32_t mph = 0, done = 0;  // done: tiles of this CTA before the current piece
    auto meet = [&]() {  // all computing warps; bounded like every wait
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet_bar);
        live = mbar_wait_warp(smem_u32(&meet_bar), mph, &dead, bound) && live;
        mph ^= 1;
    };
    // 16-byte chunk c (0 .. HD / 8 - 1) of a row: part c / 8, chunk c % 8 swizzled by the row
    auto at = [](uint32_t base, int row, int c) { return base + (uint32_t)((row >> 3) * GROUP8 + (c >> 3) * 1024 + (row & 7) * 128 + (((c & 7) ^ (row & 7)) << 4)); };
    while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
        const int ntiles = pc.t1 - pc.t0, rows = min(pl.tb, pc.n - pc.b * pl.tb) * group;
        // the block's queries as A fragments (rows past its end are zero), and what its rows see: positions above `low` up to `lim`
        uint32_t qa[HD / 16][4];
        int lim[2], low[2];
        const uint32_t* qp[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = g + 8 * e, tok = pc.b * pl.tb + r / group;
            lim[e] = min(pc.len - pc.n + tok, pg.cap - 1), low[e] = pl.window > 0 ? pc.len - pc.n + tok - pl.window : -1;
            qp[e]  = reinterpret_cast<const uint32_t*>(q + (pc.q0 + tok) * ldq + (long long)(kvh * group + r % group) * HD);
        }
#pragma unroll
        for (int kc = 0; kc < HD / 16; kc++) {
            qa[kc][0] = g < rows ? qp[0][kc * 8 + t4] : 0u, qa[kc][2] = g < rows ? qp[0][kc * 8 + t4 + 4] : 0u;
            qa[kc][1] = g + 8 < rows ? qp[1][kc * 8 + t4] : 0u, qa[kc][3] = g + 8 < rows ? qp[1][kc * 8 + t4 + 4] : 0u;
        }
        // positions that all rows see: below the first row's, above the last row's window
        const int sure_hi = min(pc.len - pc.n + pc.b * pl.tb + 1, pg.cap), sure_lo = pl.window > 0 ? pc.len - pc.n + min(pc.n, (pc.b + 1) * pl.tb) - pl.window : 0;
        float o[HD / 8][4];
#pragma unroll
        for (int j = 0; j < HD / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
        for (int kt = 0; kt < ntiles; kt++) {
            const uint32_t n = 2 * (done + kt);
            const uint32_t sk = n % stages, pk = (n / stages) & 1, sv = (n + 1) % stages, pv = ((n + 1) / stages) & 1;
            if (!(live = mbar_wait_warp(smem_u32(&full[sk]), pk, &dead, bound))) break;
            const uint32_t kb = smem_u32(ring + (size_t)sk * TILE), vb = smem_u32(ring + (size_t)sv * TILE);
            const int tok0 = (pc.t0 + kt) * kTok + warp * 16;  // this warp's 16 positions
            const unsigned there = ((unsigned)*(volatile int*)&s_there[sk] >> (warp * 2)) & 3u;
            const bool mine = tok0 < pc.hi && tok0 + 16 > pc.lo && there;
            float sc[2][4];
#pragma unroll
            for (int j = 0; j < 2; j++) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
            if (mine) {
#pragma unroll
                for (int kc = 0; kc < HD / 16; kc++) {
                    uint32_t b[4];
                    ldsm4(b, at(kb, warp * 16 + (lane & 7) + (lane >> 4) * 8, kc * 2 + ((lane >> 3) & 1)));
                    mma16816(sc[0], qa[kc], b[0], b[1]);
                    mma16816(sc[1], qa[kc], b[2], b[3]);
                }
            }
            // a stage goes back when every ldmatrix of it has delivered: the matrix instructions behind them were issued with its registers
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[sk]);
            if (!(live = mbar_wait_warp(smem_u32(&full[sv]), pv, &dead, bound))) break;
            if (mine) {
                if (tok0 + 16 > sure_hi || tok0 < sure_lo || there != 3u) {
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int p = tok0 + j * 8 + 2 * t4 + (e & 1);
                            if (p > lim[e >> 1] || p <= low[e >> 1] || !(there >> j & 1)) sc[j][e] = -INFINITY;
                        }
                }
                if (tok0 + 16 > pc.hi || tok0 < pc.lo) {  // positions that no row sees: no value that might not be a number
                    for (int c = lane; c < 16 * (HD / 8); c += 32) {
                        const int r = c / (HD / 8), ch = c % (HD / 8), row = warp * 16 + r;
                        if (tok0 + r >= pc.hi || tok0 + r < pc.lo)
                            *reinterpret_cast<uint4*>(ring + (size_t)sv * TILE + (row >> 3) * GROUP8 + (ch >> 3) * 1024 + (row & 7) * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    // the stage is refilled by the asynchronous proxy later: these writes come before that
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                float mx_lo = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1])), mx_hi = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
                mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 1)), mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 2));
                mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 1)), mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 2));
                const float mn_lo = fmaxf(m_lo, mx_lo * sc2), mn_hi = fmaxf(m_hi, mx_hi * sc2);
                // where all scores so far are -inf their weights are 0
                const float b_lo = mn_lo == -INFINITY ? 0.f : mn_lo, b_hi = mn_hi == -INFINITY ? 0.f : mn_hi;
                const float c_lo = exp2f(m_lo - b_lo), c_hi = exp2f(m_hi - b_hi);
                m_lo = mn_lo, m_hi = mn_hi;
                float rs_lo = 0.f, rs_hi = 0.f;
                uint32_t pa[4];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float p0 = exp2f(fmaf(sc[j][0], sc2, -b_lo)), p1 = exp2f(fmaf(sc[j][1], sc2, -b_lo));
                    const float p2 = exp2f(fmaf(sc[j][2], sc2, -b_hi)), p3 = exp2f(fmaf(sc[j][3], sc2, -b_hi));
                    rs_lo += p0 + p1, rs_hi += p2 + p3;
                    pa[j * 2 + 0] = pack_bf16x2(p0, p1), pa[j * 2 + 1] = pack_bf16x2(p2, p3);
                }
                l_lo = l_lo * c_lo + rs_lo, l_hi = l_hi * c_hi + rs_hi;
                if (__any_sync(0xffffffffu, c_lo != 1.f || c_hi != 1.f)) {
#pragma unroll
                    for (int j = 0; j < HD / 8; j++) o[j][0] *= c_lo, o[j][1] *= c_lo, o[j][2] *= c_hi, o[j][3] *= c_hi;
                }
#pragma unroll
                for (int jp = 0; jp < HD / 16; jp++) {
                    uint32_t b[4];
                    ldsm4_t(b, at(vb, warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, jp * 2 + (lane >> 4)));
                    mma16816(o[2 * jp], pa, b[0], b[1]);
                    mma16816(o[2 * jp + 1], pa, b[2], b[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[sv]);
        }
        done += (uint32_t)ntiles;
        if (!live) break;
        // ---- merge the warps (fixed order) through shared memory ----
        l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1), l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
        l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1), l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
#pragma unroll
        for (int j = 0; j < HD / 8; j++) {
            float* r0 = s_o + ((size_t)warp * rb + g) * HD + j * 8 + 2 * t4;
            if (g < rows) *reinterpret_cast<float2*>(r0) = make_float2(o[j][0], o[j][1]);
            if (g + 8 < rows) *reinterpret_cast<float2*>(r0 + 8 * HD) = make_float2(o[j][2], o[j][3]);
        }
        if (t4 == 0) s_m[warp][g] = m_lo, s_m[warp][g + 8] = m_hi, s_l[warp][g] = l_lo, s_l[warp][g + 8] = l_hi;
        meet();
        if (!live) break;
        const bool whole = pc.whole;
        auto out_row = [&](int r) {
            return out + (pc.q0 + pc.b * pl.tb + r / group) * ldo + (long long)(kvh * group + r % group) * HD;
        };
        // partial sums: a CTA has at most one piece that others have begun (slot 0) and one that others go on with (slot 1)
        const int first = pc.first, last = pc.last;  // teams
        const size_t slot = (size_t)blockIdx.x * 2 + (first == team);
        for (int idx = tid; idx < rows * (HD / 4); idx += kComp) {
            const int r = idx / (HD / 4), c = idx % (HD / 4) * 4;
            float M_ = -INFINITY, L_ = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) M_ = fmaxf(M_, s_m[w][r]);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f  = s_m[w][r] == -INFINITY ? 0.f : exp2f(s_m[w][r] - M_);
                const float4 v = *reinterpret_cast<const float4*>(s_o + ((size_t)w * rb + r) * HD + c);
                L_ += s_l[w][r] * f;
                a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
            }
            if (whole) {
                const float i = L_ == 0.f ? 0.f : 1.f / L_;
                put4(out_row(r) + c, make_float4(a.x * i, a.y * i, a.z * i, a.w * i), vec);
            } else {
                __stcg(reinterpret_cast<float4*>(ws + (slot * rb + r) * HD + c), a);
                if (c == 0) __stcg(ws_ml + slot * rb + r, make_float2(M_, L_));
            }
        }
        if (!whole) {
            // ---- the piece that arrives last at its block merges all of them in order ----
            const int pieces = last - first + 1;
            auto slot_of = [&](int i) { return ((size_t)(first + i) * n_kv + kvh) * 2 + (i == 0); };
            __threadfence();
            meet();
            if (live && tid == 0) {
                unsigned* c = cnt + (size_t)first * n_kv + kvh;
                s_last      = atomicAdd(c, 1u) == (unsigned)(pieces - 1);
                if (s_last) *c = 0u;  // self-reset for the next launch
            }
            meet();
            if (live && s_last) {
                __threadfence();
                // a row to a warp (HD 64: the halves of the warp take every second piece), its pieces in order, kAt at a time and as many more on their way
                constexpr int VEC = HD / 4, LANES = 32 / VEC, kAt = 8;
                const int half = lane / VEC, c = lane % VEC * 4;
                for (int r = warp; r < rows; r += kWarps) {
                    float M_ = -INFINITY, L_ = 0.f;
                    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), v[kAt];
                    float2 ml[kAt];
                    auto ask = [&](int i0) {
#pragma unroll
                        for (int i = 0; i < kAt; i++) {
                            const int at    = i0 + i * LANES + half;
                            const size_t at_row = slot_of(min(at, pieces - 1)) * rb + r;
                            v[i]  = __ldcg(reinterpret_cast<const float4*>(ws + at_row * HD + c));
                            ml[i] = __ldcg(ws_ml + at_row);
                            if (at >= pieces) ml[i].x = -INFINITY;  // asked for twice, weighs nothing
                        }
                    };
                    ask(0);
                    for (int i0 = 0; i0 < pieces; i0 += kAt * LANES) {
                        float4 w[kAt];
                        float2 wl[kAt];
                        float n = M_;
#pragma unroll
                        for (int i = 0; i < kAt; i++) w[i] = v[i], wl[i] = ml[i], n = fmaxf(n, ml[i].x);
                        if (i0 + kAt * LANES < pieces) ask(i0 + kAt * LANES);
                        const float base = n == -INFINITY ? 0.f : n, f0 = exp2f(M_ - base);
                        M_ = n, L_ *= f0, a.x *= f0, a.y *= f0, a.z *= f0, a.w *= f0;
#pragma unroll
                        for (int i = 0; i < kAt; i++) {
                            const float f = exp2f(wl[i].x - base);
                            L_ = fmaf(wl[i].y, f, L_);
                            a.x = fmaf(w[i].x, f, a.x), a.y = fmaf(w[i].y, f, a.y), a.z = fmaf(w[i].z, f, a.z), a.w = fmaf(w[i].w, f, a.w);
                        }
                    }
                    if (LANES == 2) {  // the two halves' sums
                        const float Mo = __shfl_xor_sync(0xffffffffu, M_, 16), n = fmaxf(M_, Mo), base = n == -INFINITY ? 0.f : n, f = exp2f(M_ - base);
                        L_ *= f, a.x *= f, a.y *= f, a.z *= f, a.w *= f;
                        L_ += __shfl_xor_sync(0xffffffffu, L_, 16);
                        a.x += __shfl_xor_sync(0xffffffffu, a.x, 16), a.y += __shfl_xor_sync(0xffffffffu, a.y, 16);
                        a.z += __shfl_xor_sync(0xffffffffu, a.z, 16), a.w += __shfl_xor_sync(0xffffffffu, a.w, 16);
                    }
                    const float i = L_ == 0.f ? 0.f : 1.f / L_;
                    if (half == 0) put4(out_row(r) + c, make_float4(a.x * i, a.y * i, a.z * i, a.w * i), vec);
                }
            }
        }
        meet();  // the area belongs to the next piece
    }
}

// positions of a box: the largest power of two that divides a page, at most `most`
int box_of(int page, int most) {
    int b = 8;
    while (b < most && page % (2 * b) == 0) b *= 2;
    return b;
}

template <int HD>
int launch_few(kf_ctx* ctx, const kf_paged_kv* kv, const KfPaged& pg, PagedPlan pl, void* out, long long ldo, const void* q, long long ldq, float scale) {
    const int n_kv = kv->n_kv, teams = std::max(1, 2 * ctx->sm_count / n_kv), grid = teams * n_kv, box = box_of(kv->page_size, kTok), rb = pl.tb * pl.group;
    const size_t rows = (size_t)grid * 2 * rb;
    pl.runs = teams;
    KF_REQUIRE(ctx, paged_most(kTok, pg, pl) < 0x7fff0000, "as many tiles as M rows over full tables have");
    int rc = kf_ensure_attn_ws(ctx, rows * (HD + 2) * sizeof(float));
    if (!rc) rc = kf_ensure_attn_cnt(ctx, grid);
    if (rc) return rc;
    CUtensorMap tk, tv;
    const uint64_t stride = kf_paged_stride(kv) * 2;
    rc = kf_tmap_pages(ctx, &tk, kv->k_dev, (uint64_t)n_kv * HD, (uint64_t)kv->page_size, (uint64_t)kv->n_pages, stride, HD / 64, box);
    if (!rc) rc = kf_tmap_pages(ctx, &tv, kv->v_dev, (uint64_t)n_kv * HD, (uint64_t)kv->page_size, (uint64_t)kv->n_pages, stride, HD / 64, box);
    if (rc) return rc;
    const int stages  = ring_stages(HD, rb);
    const size_t smem = (size_t)stages * kTok * HD * 2 + rows_area(HD, rb) + 1024;
    auto kern         = kf_attn_paged_kernel<HD>;
    static bool set[kf_ctx::kMaxDevices] = {};  // function attributes are per device
    if (!set[ctx->device]) {
        KF_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (kSmemKB + 1) * 1024));
        set[ctx->device] = true;
    }
    KF_CUDA(ctx, kf_launch_pdl(ctx, kern, dim3(grid), dim3((kWarps + 2) * 32), smem, tk, tv, (uint16_t*)out, ctx->attn_ws, reinterpret_cast<float2*>(ctx->attn_ws + rows * HD),
                               ctx->attn_cnt, (const uint16_t*)q, pg, pl, ldo, ldq, n_kv, box, stages, scale * 1.4426950408889634f,
                               KfBound{ctx->wait_flags + kWaitPaged, (unsigned)ctx->attn_wait_us, ctx->attn_drop}));
    KF_LAUNCH_CHECK(ctx);
    return KF_OK;
}
}  // namespace

static int check_args(kf_ctx* ctx, const kf_paged_kv* kv, const void* out, int ldo, const void* q, int ldq, int M, int n_head, float scale, int max_q, KfPaged* pg) {
    if (!kv || !out || !q) return KF_ERR_BAD_ARG;
    const int rc = kf_paged_check(ctx, kv, M, pg);
    if (rc) return rc;
    KF_REQUIRE(ctx, n_head >= 1 && n_head % kv->n_kv == 0 && n_head / kv->n_kv <= 64, "n_head a multiple of n_kv, at most 64 heads to a kv head");
    KF_REQUIRE(ctx, (long long)n_head * kv->head_dim <= ldq && (long long)n_head * kv->head_dim <= ldo, "rows as long as their heads");
    KF_REQUIRE(ctx, ((uintptr_t)q & 15) == 0 && ldq % 8 == 0, "q at 16 bytes, ldq a multiple of 8");
    KF_REQUIRE(ctx, (long long)M * (n_head / kv->n_kv) < 0x7fffff00, "rows");
    KF_REQUIRE(ctx, out != q, "the result over the queries");
    KF_REQUIRE(ctx, scale > 0.f && scale < INFINITY && max_q >= 0, "scale above 0, max_q not negative");
    return KF_OK;
}
extern "C" int kf_paged_attention(kf_ctx* ctx, const kf_paged_kv* kv, void* out, int ldo, const void* q, int ldq, int M, int n_head, float scale, int window, int max_q) {
    if (!ctx) return KF_ERR_BAD_ARG;
    KfPaged pg;
    int rc = check_args(ctx, kv, out, ldo, q, ldq, M, n_head, scale, max_q, &pg);
    if (rc) return rc;
    const size_t wide = (size_t)n_head * kv->head_dim * 2;
    KF_REQUIRE(ctx, !kf_rows_overlap(out, (size_t)ldo * 2, wide, q, (size_t)ldq * 2, wide, M), "the result over a part of the queries");
    rc = kf_wait_status(ctx);
    if (rc || M == 0) return rc;
    const int group = n_head / kv->n_kv;
    // steps whose sequences have up to 16 rows a kv head (new tokens x heads of the group) here, others as a whole on tcgen05.  Single tokens alone, here / there: 64 ragged
    // sequences 112 / 158 us, one at 1300 positions 10.5 / 15.9; 16 sequences with two tokens of 8 heads 49 / 54.  For the single tokens of a step with chunks a second launch
    // was measured where their rows have few positions, and costs more than their row tiles (24 sequences, three of them with chunks, 64 dims, a window of 1000: 60 against 55
    // us; 16 x 5 drafted tokens, launched for nothing: 71 against 67).  Where they have many it would gain: the 64 sequences and a chunk of 512 behind 2000 positions
    // take 228 us, the two apart 112 + 67.
    const int tokens = std::max(1, max_q), few = 16 / group;
    if (tokens > few) return kf_attn_paged_tc(ctx, kv, pg, out, ldo, q, ldq, n_head, scale, window);
    const PagedPlan pl{tokens, group, window, 1, 0};
    return kv->head_dim == 128 ? launch_few<128>(ctx, kv, pg, pl, out, ldo, q, ldq, scale) : launch_few<64>(ctx, kv, pg, pl, out, ldo, q, ldq, scale);
}
// The checks and the blocks' arithmetic for tests on a host without a device
extern "C" int kf_paged_attention_args(const kf_paged_kv* kv, const void* out, int ldo, const void* q, int ldq, int M, int n_head, float scale, int max_q) {
    KfPaged pg;
    return check_args(nullptr, kv, out, ldo, q, ldq, M, n_head, scale, max_q, &pg);
}
extern "C" int kf_paged_attention_block(int tile, int cap, int tb, int window, int n, int len, int b, int* lo_hi_first) {
    int ns;
    return paged_block(tile, cap, tb, window, 0, n, len, b, lo_hi_first[0], lo_hi_first[1], lo_hi_first[2], ns);
}
extern "C" int kf_paged_attention_block_first(int tile, int cap, int tb, int window, int first, int n, int len, int b, int* lo_hi_first_ns) {
    return paged_block(tile, cap, tb, window, first, n, len, b, lo_hi_first_ns[0], lo_hi_first_ns[1], lo_hi_first_ns[2], lo_hi_first_ns[3]);
}
extern "C" int kf_paged_page_of(int page, int p) {
    KfPaged pg = {};
    pg.page    = page;
    kf_paged_divisor(&pg);
    return (int)((uint64_t)(uint32_t)p * pg.page_mul >> 32 >> pg.page_shift);
}
