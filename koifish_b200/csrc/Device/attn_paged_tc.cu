// attn_paged_tc.cu -- attention of sequences with many rows (chunks of prompts, drafts) over a cache in pages, on tcgen05 / TMEM / TMA.  Formulas: attn_paged.cu.
//
// A row tile is 128 rows: as many tokens as fit with all heads of their kv group, so that a tile of K and V serves all of them and few tokens still fill a tile.  A block
// is two row tiles.  Its visible positions go by in tiles of 128, and the two chains of scores -> weights -> sums fill each other's gaps: while the softmax warps of one turn
// scores into weights, the tensor cores work for the other.  The chains are the block's two row tiles, which share every tile of K and V -- or, where the block has one
// row tile only, its even and odd tiles of positions, whose sums meet in shared memory at the end.
//   warps 0-3 / 4-7  softmax of chain 0 / 1, thread = row: scores from tensor memory into registers, running maximum, weights as bf16 back over the first half of the scores
//   warp 8           matrix instructions of both chains in turn: S = Q K^T (both operands in shared memory), O += P V (P from tensor memory, V as it lies: MN-major)
//   warp 9 / 10      Q and K / V: page look-up and TMA, a box per page (or part of 8 .. 128 positions of it), each asked for by a lane of its own
//   warp 11          the pieces
// The tiles of all blocks and kv heads are cut into equal runs, one CTA each (PagedWalk).  Blocks that several CTAs share leave their sums in the workspace; a second
// kernel, launched behind, merges them in order.
// Sums are rescaled when a row's maximum has grown by more than 2^8 over the one they refer to (deferring it so is a published method of attention on this generation of tensor
// cores): until about 32 tiles have gone by nearly every tile brings one of a warp's rows a new maximum, and the rescaling stands in a chain's way (2048 tokens behind 8192, 32
// heads: 362 us rescaling whenever a maximum grows, 301 with the slack).  Weights up to 2^8 are rounded to bf16 like the others, and the denominator adds them as they are rounded: the error of a row that one weight carries cancels.  Relative to 64 bits, 512 tokens:
// 2.3e-3 flat and 1.8e-3 sharp (scores four times as large), 2.1e-3 and 1.7e-3 rescaling always, 2.3e-3 and 2.0e-3 with the unrounded weights in the denominator; the
// result's own rounding is 1.7e-3.
// What bounds it: a chain's way.  A tile takes it about 3600 clocks -- scores 512, from them to the first half of the weights 1500, to the second 900, sums behind these 256, the
// rest hand-overs -- while the tensor cores are busy for 2048 of both chains' clocks and the special-function units for as many.  Forming a quarter of the exponentials on the
// multiply-add units made it 5 % slower, an issuing warp for each chain 16 % (they fall into step).  Measured: that chunk 330 us in a steady run, 935 TFLOP/s
// under the power cap (290 us, 1070 TFLOP/s in a few dozen passes); 16 sequences of 500 .. 5000 positions with five drafted tokens of 40 heads 56 us, 3.2 TB/s, where the
// way of a tile of V through three stages adds to it.  Runs are equal in tiles, not in time: a tile of a block with two row tiles takes both chains a step, of another
// block half of one, so in steps that mix chunks and single tokens the CTAs end at different times.
// Rows of V that no row of the block sees are zeroed in shared memory, since they need not hold numbers; boxes of pages that are not there arrive as zeros.
// Every wait is bounded: when one runs out, `dead` ends all roles, copies and matrix instructions in flight are awaited and tensor memory is freed.
#include <algorithm>

#include "kf_paged_tc.cuh"

namespace {
constexpr int kMmaW = 8, kLoadK = 9, kLoadV = 10, kPlanW = 11, kThreads = 12 * 32, kMasks = 8;
template <int HD>
struct Cfg {
    static constexpr int kParts = HD / 64, kTile = kKV * HD * 2, kHalf = kKV * 128, kStagesK = HD == 128 ? 2 : 4, kStagesV = HD == 128 ? 3 : 6;
    static constexpr int kGroup = kParts * 1024;  // tiles of K and V lie as groups of 8 rows, each in parts of 64 dims (kf_tmap_pages); of Q as halves of 64 dims
    static constexpr size_t kSmem = (2 + kStagesK + kStagesV) * (size_t)kTile + 1024;
};
template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    kf_attn_paged_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                            const __grid_constant__ KfPaged pg_, const __grid_constant__ PagedPlan pl, const __grid_constant__ TcArgs a, const __grid_constant__ KfBound bound) {
    using C = Cfg<HD>;
    constexpr int kTile = C::kTile, kHalf = C::kHalf, kParts = C::kParts, kGroup = C::kGroup, kStagesK = C::kStagesK, kStagesV = C::kStagesV;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sq = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sk = sq + 2 * kTile;
    uint8_t* sv = sk + kStagesK * kTile;
    __shared__ uint64_t q_full, q_empty, k_full[kStagesK], k_empty[kStagesK], v_full[kStagesV], v_empty[kStagesV], v_land, s_full[2], p_full[2][kParts2], o_done[2], x_full, x_free, x_done, done_bar;
    __shared__ uint32_t tmem_base_smem;
    __shared__ volatile int dead;
    __shared__ volatile int s_there[kMasks];  // bit i: positions 8 i .. 8 i + 7 of a tile are there; by tile
    __shared__ PagedQueue qu;
    // chain 1's maximum and denominator, where the chains share a row tile: over the sequences' tiles, which are not looked at once the first piece is known
    float *s_m = reinterpret_cast<float*>(qu.s_sum), *s_l = s_m + kQ;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(&q_full, 1), mbar_init(&q_empty, 1), mbar_init(&v_land, 1), mbar_init(&done_bar, 1), mbar_init(&x_full, 4), mbar_init(&x_free, 4), mbar_init(&x_done, 4);
        for (int s = 0; s < kStagesK; s++) mbar_init(&k_full[s], 1), mbar_init(&k_empty[s], 1);
        for (int s = 0; s < kStagesV; s++) mbar_init(&v_full[s], 1), mbar_init(&v_empty[s], 1);
        for (int t = 0; t < 2; t++) {
            mbar_init(&s_full[t], 2), mbar_init(&o_done[t], 1);
            for (int k = 0; k < kParts2; k++) mbar_init(&p_full[t][k], 4);
        }
        qu.init(11);
        dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&tm_q), tma_prefetch_map(&tm_k), tma_prefetch_map(&tm_v);
    }
    if (warp == kMmaW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_smem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_smem;
    const int cta       = (int)blockIdx.x;
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();  // queries, cache rows, lengths and tables, workspace
    const KfPaged pg = behind_wait(pg_);
    if (pg.n_seq > 32) {
        PagedPlanner<kKV>::count(pg, pl, qu.s_sum, warp, kThreads / 32, lane);
        __syncthreads();
    }
    PagedReader reader;
    PagedPiece pc;
    bool live = true;

    if (warp < 8) {
        const int t = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t s_row = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(t * 128), o_row = tmem + ((uint32_t)(quad * 32) << 16) + 256u + (uint32_t)(t * HD);
        const uint32_t sfull = smem_u32(&s_full[t]), pfull = smem_u32(&p_full[t][0]), odone = smem_u32(&o_done[t]);
        const bool vec = ((uintptr_t)a.out & 15) == 0 && a.ldo % 8 == 0;
        const float sc2 = a.sc2;
        uint32_t cnt = 0, tile0 = 0, xph = 0;  // steps of this chain, tiles of this CTA before the piece, phases of the exchange
        while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
            const Steps st(pc, pl, a.tokens);
            const int steps = st.of(t), tok0 = pc.b * pl.tb + (st.pair ? t * a.tokens : 0);  // the row tile's first token
            const int tok = tok0 + row / pl.group;
            const bool mine = row < a.tokens * pl.group && tok < pc.n;
            const bool idle = !__any_sync(0xffffffffu, mine);
            const int pos = mine ? min(pc.len - pc.n + tok, pg.cap - 1) : -1, low = pl.window > 0 ? pc.len - pc.n + tok - pl.window : -1;  // sees (low, pos]
            // positions that all rows of the row tile see
            const int last = min(pc.n, tok0 + a.tokens) - 1, sure_hi = min(pc.len - pc.n + tok0 + 1, pg.cap), sure_lo = pl.window > 0 ? pc.len - pc.n + last - pl.window + 1 : 0;
            float m = -INFINITY;           // the maximum, times sc2, that the weights and O refer to
            unsigned long long l2 = 0ull;  // the denominator, even and odd positions apart
            for (int j = 0; j < steps; j++) {
                if (!(live = mbar_wait_warp(sfull, cnt & 1, &dead, bound))) break;
                if (idle) {  // what lies there is taken for the weights of rows that are nobody's
#pragma unroll
                    for (int k = 0; k < kParts2; k++)
                        if (lane == 0) mbar_arrive_a(pfull + 8 * k);
                    cnt++;
                    continue;
                }
                tc_fence_after();
                uint32_t s[kKV];
#pragma unroll
                for (int c = 0; c < 4; c++) ld32_async(s_row + 32 * c, s + 32 * c);
                const int p0 = (pc.t0 + st.tile(t, j)) * kKV;
                const unsigned there = (unsigned)s_there[(tile0 + st.tile(t, j)) % kMasks];
                wait_ld();
                if (p0 + kKV > sure_hi || p0 < sure_lo || there != 0xffffu) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {  // what the row sees of 32 positions, a bit each
                        const int hi = pos - p0 - 32 * c, lo = low - p0 - 32 * c;
                        uint32_t see = ((there >> (4 * c) & 15u) * 0x00204081u & 0x01010101u) * 255u;
                        see &= hi < 0 ? 0u : hi > 30 ? 0xffffffffu : (2u << hi) - 1u;
                        see &= lo < 0 ? 0xffffffffu : lo > 30 ? 0u : ~((2u << lo) - 1u);
#pragma unroll
                        for (int i = 0; i < 32; i++) s[32 * c + i] = see >> i & 1 ? s[32 * c + i] : 0xff800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kKV; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], __uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1]));
                const float mn = mine ? max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * sc2 : -INFINITY;  // nobody's rows hold what lay there: they have no say in a rescaling
                if (j == 0) {
                    m = mn;
                } else if (__any_sync(0xffffffffu, mn > m + kSlack)) {
                    const float n = fmaxf(m, mn), f = ex2(m - finite_or_0(n));
                    if (!(live = mbar_wait_warp(odone, (cnt - 1) & 1, &dead, bound))) break;  // the last O += P V is through
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_row + c, o);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st16(o_row + c, o);
                    }
                    wait_st();
                    l2 = mul2(l2, pack2(f, f)), m = n;
                }
                const float base = finite_or_0(m);
                const unsigned long long sc22 = pack2(sc2, sc2), nm2 = pack2(-base, -base);
#pragma unroll
                for (int c = 0; c < 4; c++) {  // a part's O += P V runs while the next one's weights are formed
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float2 x = unpack2(fma2(pack2(__uint_as_float(s[32 * c + 2 * i]), __uint_as_float(s[32 * c + 2 * i + 1])), sc22, nm2));
                        p[i] = pack_bf16x2(ex2(x.x), ex2(x.y));
                        l2   = add2(l2, pack2(bf16lo(p[i]), bf16hi(p[i])));  // the weights as they are used: a rounding that numerator and denominator share
                    }
                    tmem_st16(s_row + 16 * c, p);  // over scores, which are in registers
                    if ((c + 1) % (4 / kParts2) == 0) {
                        wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_a(pfull + 8 * (c / (4 / kParts2)));
                    }
                }
                cnt++;
            }
            if (live && steps > 0) live = mbar_wait_warp(odone, (cnt - 1) & 1, &dead, bound);
            if (!live) break;
            tc_fence_after();
            const float2 ll = unpack2(l2);
            float l = ll.x + ll.y, m2 = m;
            const bool whole = pc.whole, meet = !st.pair && st.n > 1;
            const size_t slot = ((size_t)cta * 2 + (pc.first == cta)) * 256 + (st.pair ? t * kQ : 0) + row;
            uint16_t* op = a.out + (pc.q0 + tok) * a.ldo + (long long)(pc.head * pl.group + row % pl.group) * HD;
            float f0 = 1.f, f1 = 0.f;
            constexpr int kCols = HD / 2;  // columns of an exchange: as many as the second Q tile, which such a block does not have, holds of 128 rows
            float4* xb = reinterpret_cast<float4*>(sq + kTile);
            for (int c0 = 0; live && c0 < HD; c0 += kCols) {
                if (meet && t == 1) {
                    if (!(live = mbar_wait_warp(smem_u32(&x_free), (xph & 1) ^ 1, &dead, bound))) break;  // what was there has been read
                    xph++;
                    if (c0 == 0) s_m[row] = m2, s_l[row] = l;
#pragma unroll 1
                    for (int c = 0; c < kCols; c += 32) {
                        uint32_t o[32];
                        ld32_async(o_row + c0 + c, o);
                        wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; i++) xb[(c / 4 + i) * kQ + row] = *reinterpret_cast<const float4*>(&o[4 * i]);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&x_full);
                    continue;
                }
                if (st.pair || t == 0) {
                    if (meet) {
                        if (!(live = mbar_wait_warp(smem_u32(&x_full), xph & 1, &dead, bound))) break;
                        xph++;
                        if (c0 == 0) {
                            const float mb = s_m[row], mm = fmaxf(m2, mb);
                            f0 = m2 == -INFINITY ? 0.f : ex2(m2 - mm), f1 = mb == -INFINITY ? 0.f : ex2(mb - mm);
                            l = l * f0 + s_l[row] * f1, m2 = mm;
                        }
                    }
                    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
                    for (int c = 0; c < kCols; c += 32) {
                        uint32_t o[32];
                        ld32_async(o_row + c0 + c, o);
                        wait_ld();
                        if (meet) {
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const float4 b = xb[(c / 4 + i) * kQ + row];
                                o[4 * i]     = __float_as_uint(fmaf(b.x, f1, __uint_as_float(o[4 * i]) * f0));
                                o[4 * i + 1] = __float_as_uint(fmaf(b.y, f1, __uint_as_float(o[4 * i + 1]) * f0));
                                o[4 * i + 2] = __float_as_uint(fmaf(b.z, f1, __uint_as_float(o[4 * i + 2]) * f0));
                                o[4 * i + 3] = __float_as_uint(fmaf(b.w, f1, __uint_as_float(o[4 * i + 3]) * f0));
                            }
                        }
                        if (!mine) continue;
                        if (whole) store_row(op + c0 + c, o, inv, vec);
                        else {
                            float4* w = reinterpret_cast<float4*>(a.ws + slot * HD + c0 + c);
#pragma unroll
                            for (int i = 0; i < 8; i++) __stcg(w + i, *reinterpret_cast<const float4*>(&o[4 * i]));
                        }
                    }
                    if (mine && !whole && c0 == 0) __stcg(a.ws_ml + slot, make_float2(m2, l));
                    if (meet) {
                        const bool over = c0 + kCols >= HD;
                        if (over) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the second Q tile may be the loader's next
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&x_free);
                        if (over && lane == 0) mbar_arrive(&x_done);
                    }
                }
            }
            if (!live) break;
            tc_fence_before();
            tile0 += st.n;
        }
    } else if (warp == kMmaW) {
        constexpr uint32_t id_s = make_idesc_bf16(128), id_o = make_idesc_bf16(HD) | (1u << 16);  // bit 16: B is MN-major
        const uint32_t q_addr = smem_u32(sq), k_addr = smem_u32(sk), v_addr = smem_u32(sv);
        uint32_t pos = 0, qn = 0, kseen = 0, vseen = 0, cnt[2] = {0, 0};  // tiles of the CTA before the piece, pieces, tiles that have landed, steps of the chains
        while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
            const Steps st(pc, pl, a.tokens);
            if (!(live = mbar_wait_warp(smem_u32(&q_full), qn & 1, &dead, bound))) break;
            for (int j = -1; live && j < st.of(0); j++)  // the sums of step j, the scores of step j + 1
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const bool sums = live && j >= 0 && j < st.of(t), scores = live && j + 1 < st.of(t);
                    const uint32_t iv = pos + st.tile(t, j), ik = pos + st.tile(t, j + 1), vs = iv % kStagesV, ks = ik % kStagesK;
                    // what the loaders bring is waited for first: the weights come last
                    if (scores && kseen <= ik) live = mbar_wait_warp(smem_u32(&k_full[ks]), (ik / kStagesK) & 1, &dead, bound), kseen = ik + 1;
                    if (live && sums) {
                        if (vseen <= iv) live = mbar_wait_warp(smem_u32(&v_full[vs]), (iv / kStagesV) & 1, &dead, bound), vseen = iv + 1;
                        const uint64_t vd = make_desc_kv<HD>(v_addr + vs * kTile);
#pragma unroll
                        for (int k = 0; k < kParts2; k++) {  // O_t += P_t V
                            live = live && mbar_wait_warp(smem_u32(&p_full[t][k]), cnt[t] & 1, &dead, bound);
                            tc_fence_after();
                            if (live)
#pragma unroll
                                for (int i = 0; i < 4 / kParts2; i++)
                                    umma_sums_x2<kGroup>(tmem + 256 + t * HD, tmem + t * 128 + k * (64 / kParts2) + i * 16, vd + (k * (4 / kParts2) + i) * (4 * kGroup / 16), id_o, j > 0 || k + i > 0);
                        }
                        if (live) umma_commit_a(smem_u32(&o_done[t]));
                        cnt[t]++;
                    }
                    if (live && scores) {  // S_t = Q K^T, behind the O above, which reads the weights from the same columns
                        tc_fence_after();
                        const uint32_t qd = q_addr + (st.pair ? t * kTile : 0), kd = k_addr + ks * kTile;
#pragma unroll
                        for (int k = 0; k < kParts; k++) umma_scores_x4(tmem + t * 128, make_desc_sw128(qd + k * kHalf), make_desc_kv<HD>(kd + k * 1024), id_s, k > 0);
                        umma_commit_a(smem_u32(&s_full[t]));
                        if (lane == 0) mbar_arrive(&s_full[t]);  // for what the loader wrote beside the tile
                    }
                    // tiles go back behind the last chain that reads them
                    if (live && sums && (t == 1 || !st.pair)) umma_commit_a(smem_u32(&v_empty[vs]));
                    if (live && scores && (t == 1 || !st.pair)) umma_commit_a(smem_u32(&k_empty[ks]));
                    if (live && t == 1 && j + 2 == st.of(0)) umma_commit_a(smem_u32(&q_empty));
                }
            pos += st.n, qn++;
        }
        // instructions in flight write tensor memory: waited for here, since where a wait has run out nobody else may have
        umma_commit_a(smem_u32(&done_bar));
        mbar_drain(smem_u32(&done_bar), 0, bound);
    } else if (warp == kPlanW) {
        PagedPlanner<kKV> plan(pg, pl, lane);
        if (lane == 0) a.rec[cta].last = 0;  // nothing to merge, should a wait run out before the end of the run is known
        plan.start(qu, cta);
        while (plan.push(qu, cta, a.rec, &dead, bound)) {}
    } else if (bound.drop != cta + 1) {
        // Q and K, or V
        const bool isv = warp == kLoadV;
        const uint32_t stages = isv ? kStagesV : kStagesK;
        const int n_box = kKV / a.box, bx = lane;  // a lane per box; bx >= n_box: none
        uint32_t pos = 0, landed = 0, qn = 0, xn = 0;  // tiles, ragged tiles, pieces, meetings that are over
        bool met = false;  // the chains meet over the piece before this one, and that has not been waited for
        while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
            const Steps st(pc, pl, a.tokens);
            const int head = pc.head;
            int next_row = 0;
            auto page_of = [&](int t) {  // the page of this lane's box of tile t
                const int p = t * kKV + bx * a.box;
                return t < pc.t1 && bx < n_box && p < pc.hi && p + a.box > pc.lo ? paged_page(pg, pc.s, p, next_row) : -1;
            };
            int next = page_of(pc.t0);
            if (!isv) {
                if (qn > 0) live = mbar_wait_warp(smem_u32(&q_empty), (qn - 1) & 1, &dead, bound);
                // the chains may still be meeting over the piece before, in the second Q tile
                if (live && met && st.pair) live = mbar_wait_warp(smem_u32(&x_done), xn++ & 1, &dead, bound), met = false;
                if (!live) break;
                if (lane == 0) {
                    const int tiles = st.pair ? 2 : 1;
                    mbar_arrive_expect_tx(&q_full, (uint32_t)(tiles * kParts * a.tokens * pl.group * 128));
                    for (int i = 0; i < tiles * kParts; i++) {
                        const int t = i / kParts, h = i % kParts;
                        tma_load_3d(sq + t * kTile + h * kHalf, &tm_q, h * 64, head * pl.group, pc.q0 + (pc.b * 2 + t) * a.tokens, &q_full);
                    }
                }
                __syncwarp();
                qn++;
            }
            for (int t = pc.t0; t < pc.t1; t++) {
                const uint32_t stage = pos % stages;
                const int page = next, row = next_row;
                next = page_of(t + 1);  // a tile ahead: the look-up takes its time
                const unsigned lanes = __ballot_sync(0xffffffffu, page >= 0);
                // ... which this warp has to have seen before the next meeting can be over (a wait tells a phase from the one before by one bit), for which a tile is missing yet
                if (met && t + 1 == pc.t1) {
                    if (!(live = mbar_wait_warp(smem_u32(&x_done), xn++ & 1, &dead, bound))) break;
                    met = false;
                }
                if (!(live = mbar_wait_warp(smem_u32(isv ? &v_empty[stage] : &k_empty[stage]), ((pos / stages) & 1) ^ 1, &dead, bound))) break;
                const bool ragged = isv && (t * kKV < pc.lo || (t + 1) * kKV > pc.hi);
                uint64_t* bar = !isv ? &k_full[stage] : ragged ? &v_land : &v_full[stage];
                uint8_t* dst  = (isv ? sv : sk) + stage * kTile;
                if (lane == 0) {
                    if (!isv) {
                        unsigned there = 0;
                        for (int i = 0; i < kKV / 8; i++) there |= (lanes >> (i * 8 / a.box) & 1) << i;
                        s_there[pos % kMasks] = (int)there;
                    }
                    mbar_arrive_expect_tx(bar, kTile);
                }
                __syncwarp();
                if (bx < n_box) tma_load_page(dst + bx * a.box * (HD * 2), isv ? &tm_v : &tm_k, head * kParts, page >= 0 ? row / 8 : 0, page >= 0 ? page : pg.n_pages, bar);
                __syncwarp();
                pos++;
                if (ragged) {
                    if (!(live = mbar_wait_warp(smem_u32(&v_land), landed++ & 1, &dead, bound))) break;
                    for (int i = lane; i < kKV * (HD / 8); i += 32) {
                        const int r = i / (HD / 8), c = i % (HD / 8), p = t * kKV + r;
                        if (p < pc.lo || p >= pc.hi) *reinterpret_cast<uint4*>(dst + (r >> 3) * kGroup + (c >> 3) * 1024 + (r & 7) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[stage]);
                }
            }
            met = !isv && !st.pair && st.n > 1;
        }
        // copies in flight write shared memory, which is another's once the CTA has ended: the same
        if (!isv && qn > 0) mbar_drain(smem_u32(&q_full), (qn - 1) & 1, bound);
        for (uint32_t k = pos > stages ? pos - stages : 0; k < pos; k++) mbar_drain(smem_u32(isv ? &v_full[k % stages] : &k_full[k % stages]), (k / stages) & 1, bound);
        if (isv && landed > 0) mbar_drain(smem_u32(&v_land), (landed - 1) & 1, bound);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaW) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int HD>
int launch_tc(kf_ctx* ctx, const kf_paged_kv* kv, const KfPaged& pg, void* out, long long ldo, const void* q, long long ldq, int n_head, float scale, int window) {
    const int n_kv = kv->n_kv, group = n_head / n_kv, tokens = kQ / group, grid = ctx->sm_count;
    int box = 8;
    while (box < kKV && kv->page_size % (2 * box) == 0) box *= 2;
    const PagedPlan pl{2 * tokens, group, window, n_kv, grid};
    const size_t rows = (size_t)grid * 2 * 256;
    KF_REQUIRE(ctx, paged_most(kKV, pg, pl) < 0x7fff0000, "as many tiles as M rows over full tables have");
    int rc = kf_ensure_attn_ws(ctx, rows * (HD + 2) * sizeof(float) + grid * sizeof(PagedPiece));
    CUtensorMap tq, tk, tv;
    const uint64_t stride = kf_paged_stride(kv) * 2;
    if (!rc) rc = kf_tmap_heads(ctx, &tq, q, HD, n_head, (uint64_t)pg.M, (uint64_t)ldq * 2, 64, group, tokens);
    if (!rc) rc = kf_tmap_pages(ctx, &tk, kv->k_dev, (uint64_t)n_kv * HD, (uint64_t)kv->page_size, (uint64_t)kv->n_pages, stride, HD / 64, box);
    if (!rc) rc = kf_tmap_pages(ctx, &tv, kv->v_dev, (uint64_t)n_kv * HD, (uint64_t)kv->page_size, (uint64_t)kv->n_pages, stride, HD / 64, box);
    if (rc) return rc;
    auto kern = kf_attn_paged_tc_kernel<HD>;
    static bool set[kf_ctx::kMaxDevices] = {};  // function attributes are per device
    if (!set[ctx->device]) {
        KF_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<HD>::kSmem));
        set[ctx->device] = true;
    }
    const TcArgs a{(uint16_t*)out, ctx->attn_ws, reinterpret_cast<float2*>(ctx->attn_ws + rows * HD), reinterpret_cast<PagedPiece*>(ctx->attn_ws + rows * (HD + 2)), ldo, tokens, box,
                   scale * 1.4426950408889634f};
    KF_CUDA(ctx, kf_launch_pdl(ctx, kern, dim3(grid), dim3(kThreads), Cfg<HD>::kSmem, tq, tk, tv, pg, pl, a, KfBound{ctx->wait_flags + kWaitPaged, (unsigned)ctx->attn_wait_us, ctx->attn_drop}));
    KF_LAUNCH_CHECK(ctx);
    KF_CUDA(ctx, kf_launch_pdl(ctx, kf_attn_paged_merge_kernel<HD>, dim3(grid, 256 / kMergeRows), dim3(256), 0, pl, a));
    KF_LAUNCH_CHECK(ctx);
    return KF_OK;
}
}  // namespace

int kf_attn_paged_tc(kf_ctx* ctx, const kf_paged_kv* kv, const KfPaged& pg, void* out, long long ldo, const void* q, long long ldq, int n_head, float scale, int window) {
    return kv->head_dim == 128 ? launch_tc<128>(ctx, kv, pg, out, ldo, q, ldq, n_head, scale, window)
                               : launch_tc<64>(ctx, kv, pg, out, ldo, q, ldq, n_head, scale, window);
}
