// attn_paged_q4_tc.cu -- attention of sequences with many rows (chunks of prompts, drafts) over a cache in pages that is held in 4 bits, on tcgen05 / TMEM.  The cache: attn_paged_q4.cu; row
// tiles, blocks and chains: attn_paged_tc.cu.
//
// Here the tiles of K and V for the matrix instructions are made on the SM: codes come as they lie (a bulk copy per page or part of it, keys and values at once) into a ring of raw tiles, and
// four warps expand them, step * code - step * zero in fp32 with one rounding to bf16, into the swizzled tiles that the bf16 kernel gets by TMA.  A code at bits 16 .. 19 of a word is the fp32
// number code * 2^-133, at bits 20 .. 23 code * 2^-129 (subnormal numbers and the first normal ones are one ladder), so a shift and an AND make the operand and one f32x2 multiply-add two
// entries; steps carry 2^73, so what is stored is 2^-60 of the entry, and the scale and the final division undo it.
//   warps 0-3 / 4-7  softmax of chain 0 / 1, thread = row.  128 registers a thread (15 warps) do not hold a row's 128 scores, so the first half is read twice: for the maximum, behind which the
//                    second half stays for its weights, and for its own weights, which come second
//   warp 8           matrix instructions of both chains in turn
//   warp 9           Q by TMA, raw tiles by bulk copies
//   warp 10          the pieces
//   warps 11-14      expansion: a unit of 8 positions at a time, K of a tile before V of it
// Rows of V that no row of the block sees, or whose page is not there, are written as zeros.
// Roundings: keys, values and weights to bf16 each, the roundings that reading the pages as bf16 and attending the result would have; denominators add the weights before their rounding (the
// rounded ones, as the bf16 kernel has them: 392 against 342 us for two more instructions a pair).  4.0e-3 of the result's norm from the formula in 64 bits, of which the result's own rounding is 1.7e-3
// (attn_paged_q4.cu, where only weights times steps are rounded, 2.3e-3).  fp16 operands would be nearer, but have to be brought into range by powers of two: found for whole tiles by another
// warp 496 against 366 us, drafts 91 against 61; for keys and q alone, found by the expanding warps, 384 against 326 and 72 against 57.
// What bounds it: the chains' way, as in attn_paged_tc.cu, and the expansion beside it.
//   * 2048 tokens behind 8192, 32 / 8 heads: 324 us, 870 TFLOP/s in a steady run under the power cap (354 us; bf16 335); 45 us less with nothing stored by the expanding warps.  A fifth of these 360
//     against 342 us, a tile of K ahead of the V before it 434.
//   * Where a tile has few rows, expansion and shared memory: 16 sequences of 500 .. 5000 positions with five drafted tokens of 40 / 8 heads 57 us, 1.85 a tile (K 0.64, V 0.70, 0.90 where the softmax
//     runs on the same scheduler).  The matrix operands read 770 clocks' worth of shared memory, the expansion 880; five, eight or eleven expanding warps make no difference there.
// Every wait is bounded: when one runs out, `dead` ends all roles, copies and matrix instructions in flight are awaited and tensor memory is freed.
#include <algorithm>

#include "kf_paged_tc.cuh"

namespace {
constexpr int kMmaW = 8, kLoadW = 9, kPlanW = 10, kExpW = 11, kExps = 4, kThreads = 15 * 32, kMasks = 16, kScale2 = 60;
template <int HD>
struct Cfg {
    static constexpr int kParts = HD / 64, kTile = kKV * HD * 2, kHalf = kKV * 128, kRaw = kKV / 8 * Q4Unit(HD).bytes;
    static constexpr int kStagesK = HD == 128 ? 1 : 2, kStagesV = HD == 128 ? 2 : 3, kStagesR = HD == 128 ? 3 : 6;
    static constexpr int kGroup = kParts * 1024;  // tiles of K and V lie as groups of 8 rows, each in parts of 64 dims; of Q as halves of 64 dims
    static constexpr size_t kSmem = (2 + kStagesK + kStagesV) * (size_t)kTile + kStagesR * (size_t)kRaw + 1024;
};
// What the runs are equal in.  A step of a block whose chains share their tiles (2.2 .. 2.7 us) is near two tiles of one whose chains take turns (1.6 .. 1.9 each), and what a block
// takes beside its tiles, queries, first scores and sums, is about as much (3.7 us): 16 sequences with five drafted tokens 57.3 us, 62.1 with runs equal in tiles, 24 sequences with
// three chunks and 64 dims 51.3 and 55.1.  A run must then be four units or more, which costs more than it gives where there are few tiles for all CTAs: 300 tokens of one
// sequence alone 20.3 us, 28.5 by units.  From 33 sequences on it is units in any case: how many tiles there are is known only behind the count, which adds up units, and counting both costs every
// step of many sequences 1 .. 5 us (40 x 60 tokens behind 100 .. 600 of 64 / 8 heads 110 us, 115.6).  That is the worse choice for few tiles of like blocks (in tiles / by units: 40 x 5 tokens behind
// 100 .. 250 of 40 / 8 heads 27.4 / 35.6, 33 x 30 behind 200 .. 500 of 16 / 4 29.3 / 32.0) and the better one where single tokens lie between them (27.9 / 25.7) or tiles are more (64 x 5 53.1 / 51.0).
struct ChainTiles {
    static constexpr int kMost = 2, kBlock = 2, kFew = 4;
    static __device__ __forceinline__ int tile(int left, int tb) { return left > tb / 2; }
};
struct Q4TcArgs {  // kernel parameter
    TcArgs t;
    const uint8_t* pool;
    long long page_stride;
};
// Keys or values of a unit and eight rows of a tile.  A lane takes the codes of one row that stand for eight dims of every group, as one word each: K dims 32 j + 8 t .. + 7, which it stores as
// 16 bytes, V dims 32 j + 4 t .. + 3 and 32 j + 16 + 4 t .. + 3, half words of two words in the unit, stored as 8 bytes each.  Lanes of four are rows 0, 4, 2, 6, 1, 5, 3, 7: those that store
// together meet all 32 banks.  The code is small for a reason: with two units unrolled beside one another, instructions had to be fetched again and again (2048 tokens behind 8192: 478 us
// against 405 one at a time).
template <int HD, bool is_v>
struct Eight {
    static constexpr int G = HD / 32;
    uint32_t w[G], s[G / 2];
    float z[G];
    static __device__ __forceinline__ int row(int lane) { return (lane & 4) | (lane >> 2 & 2) | lane >> 4; }
    __device__ __forceinline__ void load(const uint8_t* u, int lane) {
        constexpr Q4Unit un(HD);
        const int r = row(lane), t = lane & 3;
        if constexpr (is_v) {
            uint32_t x[G / 2], y[G / 2];
            const uint8_t* at = u + un.v_code() + t * (HD / 2) + (r >> 1) * (HD / 8) + (r & 1) * (HD / 16);
            words(at, x), words(at + 2 * HD, y), words(u + un.v_step() + r * 2 * G, s);
#pragma unroll
            for (int j = 0; j < G; j++) {
                w[j] = __byte_perm(x[j / 2], y[j / 2], j & 1 ? 0x7632 : 0x5410);
                z[j] = bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(u + un.v_zero() + j * 16 + r * 2));
            }
        } else {
            uint32_t x[G / 2];
            words(u + r * (HD / 2) + t * 4 * G, w), words(u + un.k_step() + r * 2 * G, s), words(u + un.k_zero() + r * 2 * G, x);
#pragma unroll
            for (int j = 0; j < G; j++) z[j] = half_of(x[j / 2], j & 1);
        }
    }
    __device__ __forceinline__ void hide() {  // rows that nobody sees become zeros, whatever their steps and zeros are
#pragma unroll
        for (int j = 0; j < G; j++) s[j / 2] = 0u, z[j] = 0.f;
    }
    __device__ __forceinline__ void store(uint8_t* rows, int lane) const {
        const int r = row(lane), t = lane & 3;
#pragma unroll
        for (int j = 0; j < G; j++) {
            // step * (2^73, 2^69) and minus step * zero * 2^-60 twice
            const float step = half_of(s[j / 2], j & 1), off = step * -0x1p-60f * z[j];
            const unsigned long long fa = pack2(step * 0x1p73f, step * 0x1p69f), fb = pack2(off, off);
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t x = i == 0 ? w[j] << 16 : i == 1 ? w[j] << 8 : i == 2 ? w[j] : w[j] >> 8;
                const float2 e   = unpack2(fma2(pack2(__uint_as_float(x & 0x000f0000u), __uint_as_float(x & 0x00f00000u)), fa, fb));
                v[i]             = pack_bf16x2(e.x, e.y);
            }
            uint8_t* at = rows + (j >> 1) * 1024 + r * 128;
            if (is_v) {
                *reinterpret_cast<uint2*>(at + (((4 * (j & 1) + (t >> 1)) ^ r) << 4) + (t & 1) * 8)     = make_uint2(v[0], v[1]);
                *reinterpret_cast<uint2*>(at + (((4 * (j & 1) + 2 + (t >> 1)) ^ r) << 4) + (t & 1) * 8) = make_uint2(v[2], v[3]);
            } else *reinterpret_cast<uint4*>(at + (((4 * (j & 1) + t) ^ r) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
    }
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    kf_attn_paged_q4_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ KfPaged pg_, const __grid_constant__ PagedPlan pl, const __grid_constant__ Q4TcArgs qa,
                               const __grid_constant__ KfBound bound) {
    using C = Cfg<HD>;
    constexpr int kTile = C::kTile, kHalf = C::kHalf, kParts = C::kParts, kGroup = C::kGroup, kStagesK = C::kStagesK, kStagesV = C::kStagesV, kStagesR = C::kStagesR, kRaw = C::kRaw;
    constexpr int UNIT = Q4Unit(HD).bytes;
    const TcArgs& a = qa.t;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sq = smem_raw + (-smem_u32(smem_raw) & 1023u);  // still an address in shared memory for the compiler
    uint8_t* sk = sq + 2 * kTile;
    uint8_t* sv = sk + kStagesK * kTile;
    uint8_t* sr = sv + kStagesV * kTile;
    __shared__ uint64_t q_full, q_empty, r_full[kStagesR], r_empty[kStagesR], k_full[kStagesK], k_empty[kStagesK], v_full[kStagesV], v_empty[kStagesV], s_full[2], p_full[2][kParts2], o_done[2],
        x_full, x_free, x_done, done_bar;
    __shared__ uint32_t tmem_base_smem;
    __shared__ volatile int dead;
    __shared__ volatile int s_there[kMasks];  // bit i: positions 8 i .. 8 i + 7 of a tile are there; by tile
    __shared__ PagedQueue qu;
    // chain 1's maximum and denominator, where the chains share a row tile: over the sequences' tiles, which are not looked at once the first piece is known
    float *s_m = reinterpret_cast<float*>(qu.s_sum), *s_l = s_m + kQ;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(&q_full, 1), mbar_init(&q_empty, 1), mbar_init(&done_bar, 1), mbar_init(&x_full, 4), mbar_init(&x_free, 4), mbar_init(&x_done, 4);
        for (int s = 0; s < kStagesR; s++) mbar_init(&r_full[s], 1), mbar_init(&r_empty[s], kExps);
        for (int s = 0; s < kStagesK; s++) mbar_init(&k_full[s], kExps), mbar_init(&k_empty[s], 1);
        for (int s = 0; s < kStagesV; s++) mbar_init(&v_full[s], kExps), mbar_init(&v_empty[s], 1);
        for (int t = 0; t < 2; t++) {
            mbar_init(&s_full[t], 2), mbar_init(&o_done[t], 1);
            for (int k = 0; k < kParts2; k++) mbar_init(&p_full[t][k], 4);
        }
        qu.init(10 + kExps);
        dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&tm_q);
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
    kf_grid_dependency_wait();  // queries, codes, lengths and tables, workspace
    const KfPaged pg = behind_wait(pg_);
    if (pg.n_seq > 32) {
        PagedPlanner<kKV, ChainTiles>::count(pg, pl, qu.s_sum, warp, kThreads / 32, lane);
        __syncthreads();
    }
    PagedReader reader;
    PagedPiece pc;
    bool live = true;

    // The order of the roles is that of their code: with the same instructions 2048 tokens behind 8192 take 326 us in this order and up to 349 in others, the planning code, which runs
    // once, in front of or between the loops (it is no function of its own, since the kernel's registers then pay for the call: 385)
    if (warp >= kExpW) {
        uint32_t pos = 0;
        while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
            const int fs = pc.lo > 0 ? pl.first : 0;
            for (int t = pc.t0; live && t < pc.t1; t++, pos++) {
                const uint32_t sr_ = pos % kStagesR, sk_ = pos % kStagesK, sv_ = pos % kStagesV;
                const int p0        = pc.tile(t) * kKV;
                if (!(live = mbar_wait_warp(smem_u32(&r_full[sr_]), (pos / kStagesR) & 1, &dead, bound))) break;
                const unsigned there = (unsigned)s_there[pos % kMasks];
                const uint8_t* raw   = sr + sr_ * kRaw;
                if (!(live = mbar_wait_warp(smem_u32(&k_empty[sk_]), ((pos / kStagesK) & 1) ^ 1, &dead, bound))) break;
#pragma unroll 1
                for (int u = warp - kExpW; u < kKV / 8; u += kExps) {
                    Eight<HD, false> x;
                    x.load(raw + u * UNIT, lane);
                    x.store(sk + sk_ * kTile + u * kGroup, lane);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read by the matrix instructions
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[sk_]);
                if (!(live = mbar_wait_warp(smem_u32(&v_empty[sv_]), ((pos / kStagesV) & 1) ^ 1, &dead, bound))) break;
#pragma unroll 1
                for (int u = warp - kExpW; u < kKV / 8; u += kExps) {
                    Eight<HD, true> x;
                    x.load(raw + u * UNIT, lane);
                    const int p = p0 + 8 * u;
                    if (!(there >> u & 1) || p + 8 > pc.hi || p < pc.lo) {
                        const int at = p + x.row(lane);
                        if (!(there >> u & 1) || at >= pc.hi || (at < pc.lo && at >= fs)) x.hide();
                    }
                    x.store(sv + sv_ * kTile + u * kGroup, lane);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[sv_]), mbar_arrive(&r_empty[sr_]);
            }
        }
    } else if (warp == kMmaW) {
        constexpr uint32_t id_s = make_idesc_bf16(128), id_o = make_idesc_bf16(HD) | (1u << 16);  // bit 16: B is MN-major
        const uint32_t q_addr = smem_u32(sq), k_addr = smem_u32(sk), v_addr = smem_u32(sv);
        uint32_t pos = 0, qn = 0, kseen = 0, vseen = 0, cnt[2] = {0, 0};  // tiles of the CTA before the piece, pieces, tiles that are expanded, steps of the chains
        while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
            const Steps st(pc, pl, a.tokens);
            if (!(live = mbar_wait_warp(smem_u32(&q_full), qn & 1, &dead, bound))) break;
            for (int j = -1; live && j < st.of(0); j++)  // the sums of step j, the scores of step j + 1
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const bool sums = live && j >= 0 && j < st.of(t), scores = live && j + 1 < st.of(t);
                    const uint32_t iv = pos + st.tile(t, j), ik = pos + st.tile(t, j + 1), vs = iv % kStagesV, ks = ik % kStagesK;
                    // what is expanded is waited for first: the weights come last
                    if (live && sums) {
                        if (vseen <= iv) live = mbar_wait_warp(smem_u32(&v_full[vs]), (iv / kStagesV) & 1, &dead, bound), vseen = iv + 1;
                        const uint64_t vd = make_desc_kv<HD>(v_addr + vs * kTile);
#pragma unroll
                        for (int k = kParts2 - 1; k >= 0; k--) {  // O_t += P_t V, the second part first
                            live = live && mbar_wait_warp(smem_u32(&p_full[t][k]), cnt[t] & 1, &dead, bound);
                            tc_fence_after();
                            if (live)
#pragma unroll
                                for (int i = 0; i < 4 / kParts2; i++)
                                    umma_sums_x2<kGroup>(tmem + 256 + t * HD, tmem + t * 128 + k * 64 + i * 16, vd + (k * (4 / kParts2) + i) * (4 * kGroup / 16), id_o,
                                                         j > 0 || k < kParts2 - 1 || i > 0);
                        }
                        if (live) umma_commit_a(smem_u32(&o_done[t]));
                        // the tile goes back behind the last chain that reads it, and ahead of the wait for the next one, which the same warps expand
                        if (live && (t == 1 || !st.pair)) umma_commit_a(smem_u32(&v_empty[vs]));
                        cnt[t]++;
                    }
                    if (live && scores && kseen <= ik) live = mbar_wait_warp(smem_u32(&k_full[ks]), (ik / kStagesK) & 1, &dead, bound), kseen = ik + 1;
                    if (live && scores) {  // S_t = Q K^T, behind the O above, which reads the weights from the same columns
                        tc_fence_after();
                        const uint32_t qd = q_addr + (st.pair ? t * kTile : 0), kd = k_addr + ks * kTile;
#pragma unroll
                        for (int k = 0; k < kParts; k++) umma_scores_x4(tmem + t * 128, make_desc_sw128(qd + k * kHalf), make_desc_kv<HD>(kd + k * 1024), id_s, k > 0);
                        umma_commit_a(smem_u32(&s_full[t]));
                        if (lane == 0) mbar_arrive(&s_full[t]);  // for what the loader wrote beside the tile
                    }
                    if (live && scores && (t == 1 || !st.pair)) umma_commit_a(smem_u32(&k_empty[ks]));
                    if (live && t == 1 && j + 2 == st.of(0)) umma_commit_a(smem_u32(&q_empty));
                }
            pos += st.n, qn++;
        }
        // instructions in flight write tensor memory: waited for here, since where a wait has run out nobody else may have
        umma_commit_a(smem_u32(&done_bar));
        mbar_drain(smem_u32(&done_bar), 0, bound);
    } else if (warp < 8) {
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
            const int pos = mine ? min(pc.len - pc.n + tok, pg.cap - 1) : -1, low = pl.window > 0 ? pc.len - pc.n + tok - pl.window : -1;  // sees (low, pos] and what is below `first`
            const int first = pl.window > 0 ? pl.first : 0;
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
                const int p0 = pc.tile(pc.t0 + st.tile(t, j)) * kKV;
                const unsigned there = (unsigned)s_there[(tile0 + st.tile(t, j)) % kMasks];
                const bool ragged = p0 + kKV > sure_hi || (p0 < sure_lo && p0 + kKV > first) || there != 0xffffu;
                auto hide = [&](uint32_t (&s)[32], int c) {  // what the row does not see of 32 positions
                    const int hi = pos - p0 - 32 * c, lo = low - p0 - 32 * c, fi = first - p0 - 32 * c;
                    uint32_t see = ((there >> (4 * c) & 15u) * 0x00204081u & 0x01010101u) * 255u;
                    see &= hi < 0 ? 0u : hi > 30 ? 0xffffffffu : (2u << hi) - 1u;
                    see &= (lo < 0 ? 0xffffffffu : lo > 30 ? 0u : ~((2u << lo) - 1u)) | (fi <= 0 ? 0u : fi > 31 ? 0xffffffffu : (1u << fi) - 1u);
#pragma unroll
                    for (int i = 0; i < 32; i++) s[i] = see >> i & 1 ? s[i] : 0xff800000u;
                };
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                auto most = [&](const uint32_t (&s)[32]) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], __uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1]));
                };
                uint32_t x[32], y[32];
                ld32_async(s_row, x), ld32_async(s_row + 32, y);
                wait_ld();
                if (ragged) hide(x, 0), hide(y, 1);
                most(x);
                ld32_async(s_row + 96, x);
                most(y);
                wait_ld();
                if (ragged) hide(x, 3);
                ld32_async(s_row + 64, y);
                most(x);
                wait_ld();
                if (ragged) hide(y, 2);
                most(y);
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
                auto weigh = [&](const uint32_t (&s)[32], uint32_t at) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float2 e = unpack2(fma2(pack2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), sc22, nm2));
                        const float w0 = ex2(e.x), w1 = ex2(e.y);
                        p[i] = pack_bf16x2(w0, w1);
                        l2   = add2(l2, pack2(w0, w1));
                    }
                    tmem_st16(at, p);
                };
                auto part_done = [&](int k) {
                    wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_a(pfull + 8 * k);
                };
                // the second half first, over its own scores; a part's O += P V runs while the next one's weights are formed
                weigh(y, s_row + 64);
                ld32_async(s_row, y);
                weigh(x, s_row + 80);
                ld32_async(s_row + 32, x);
                part_done(1);
                wait_ld();
                if (ragged) hide(y, 0), hide(x, 1);
                weigh(y, s_row);
                weigh(x, s_row + 16);
                part_done(0);
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
                    for (int c = 0; c < kCols && !idle; c += 32) {
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
                    const float inv = l == 0.f ? 0.f : 0x1p60f / l;
#pragma unroll 1
                    for (int c = 0; c < kCols && !idle; c += 32) {
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
    } else if (warp == kLoadW) {
        if (bound.drop != cta + 1) {
            // a lane per box (page, or part of one) of one or several tiles: the next 32 boxes are looked up while those before are copied
            const int n_box = kKV / a.box, units = a.box / 8, ahead = 32 / n_box, bx = lane % n_box, own = lane / n_box;
            const uint32_t bytes = (uint32_t)(units * UNIT);
            uint32_t pos = 0, qn = 0, xn = 0;  // tiles, pieces, meetings that are over
            bool met = false;                  // the chains meet over the piece before this one, and that has not been waited for
            while (live && reader.next(qu, pc, lane, &dead, bound, live)) {
                const Steps st(pc, pl, a.tokens);
                const int fs = pc.lo > 0 ? pl.first : 0;
                int next_row = 0;
                auto page_of = [&](int t) {
                    const int p = pc.tile(t) * kKV + bx * a.box;
                    return t < pc.t1 && p < pc.hi && (p + a.box > pc.lo || p < fs) ? paged_page(pg, pc.s, p, next_row) : -1;
                };
                int next = page_of(pc.t0 + own);
                if (qn > 0) live = mbar_wait_warp(smem_u32(&q_empty), (qn - 1) & 1, &dead, bound);
                // the chains may still be meeting over the piece before, in the second Q tile
                if (live && met && st.pair) live = mbar_wait_warp(smem_u32(&x_done), xn++ & 1, &dead, bound), met = false;
                if (!live) break;
                if (lane == 0) {
                    const int tiles = st.pair ? 2 : 1;
                    mbar_arrive_expect_tx(&q_full, (uint32_t)(tiles * kParts * a.tokens * pl.group * 128));
                    for (int i = 0; i < tiles * kParts; i++) {
                        const int t = i / kParts, h = i % kParts;
                        tma_load_3d(sq + t * kTile + h * kHalf, &tm_q, h * 64, pc.head * pl.group, pc.q0 + (pc.b * 2 + t) * a.tokens, &q_full);
                    }
                }
                __syncwarp();
                qn++;
                for (int t0 = pc.t0; live && t0 < pc.t1; t0 += ahead) {
                    const int page = next, row = next_row, n = min(ahead, pc.t1 - t0);
                    next = page_of(t0 + ahead + own);
                    const uint8_t* src = qa.pool + page * qa.page_stride + ((long long)pc.head * (pg.page / 8) + row / 8) * UNIT;
                    const unsigned has = page >= 0 ? ((1u << units) - 1u) << (bx * units) : 0u;  // units of its tile that the lane brings
                    for (int i = 0; i < n; i++) {
                        const uint32_t stage = pos % kStagesR;
                        const unsigned there = __reduce_or_sync(0xffffffffu, own == i ? has : 0u);
                        // ... which this warp has to have seen before the next meeting can be over (a wait tells a phase from the one before by one bit), for which a tile is missing yet
                        if (met && t0 + i + 1 == pc.t1) {
                            if (!(live = mbar_wait_warp(smem_u32(&x_done), xn++ & 1, &dead, bound))) break;
                            met = false;
                        }
                        if (!(live = mbar_wait_warp(smem_u32(&r_empty[stage]), ((pos / kStagesR) & 1) ^ 1, &dead, bound))) break;
                        if (lane == 0) {
                            s_there[pos % kMasks] = (int)there;
                            mbar_arrive_expect_tx(&r_full[stage], (uint32_t)__popc(there) * UNIT);
                        }
                        __syncwarp();
                        if (own == i && page >= 0) bulk_load(sr + stage * kRaw + bx * units * UNIT, src, bytes, &r_full[stage]);
                        __syncwarp();
                        pos++;
                    }
                }
                met = !st.pair && st.n > 1;
            }
            // copies in flight write shared memory, which is another's once the CTA has ended: the same
            if (qn > 0) mbar_drain(smem_u32(&q_full), (qn - 1) & 1, bound);
            for (uint32_t k = pos > kStagesR ? pos - kStagesR : 0; k < pos; k++) mbar_drain(smem_u32(&r_full[k % kStagesR]), (k / kStagesR) & 1, bound);
        }
    } else {
        PagedPlanner<kKV, ChainTiles> plan(pg, pl, lane);
        if (lane == 0) a.rec[cta].last = 0;  // nothing to merge, should a wait run out before the end of the run is known
        plan.start(qu, cta);
        while (plan.push(qu, cta, a.rec, &dead, bound)) {}
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaW) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int HD>
int launch_tc(kf_ctx* ctx, const kf_paged_q4* kv, const KfPaged& pg, void* out, long long ldo, const void* q, long long ldq, int n_head, float scale, int window, int first) {
    const int n_kv = kv->n_kv, group = n_head / n_kv, tokens = kQ / group, grid = ctx->sm_count;
    int box = 8;
    while (box < kKV && kv->page_size % (2 * box) == 0) box *= 2;
    const PagedPlan pl{2 * tokens, group, window, n_kv, grid, first};
    const size_t rows = (size_t)grid * 2 * 256;
    KF_REQUIRE(ctx, paged_most(kKV, pg, pl) * ChainTiles::kMost + ((long long)pg.M / pl.tb + pg.n_seq) * n_kv * ChainTiles::kBlock < 0x7fff0000, "as many tiles as M rows over full tables have");
    int rc = kf_ensure_attn_ws(ctx, rows * (HD + 2) * sizeof(float) + grid * sizeof(PagedPiece));
    CUtensorMap tq;
    if (!rc) rc = kf_tmap_heads(ctx, &tq, q, HD, n_head, (uint64_t)pg.M, (uint64_t)ldq * 2, 64, group, tokens);
    if (rc) return rc;
    auto kern = kf_attn_paged_q4_tc_kernel<HD>;
    static bool set[kf_ctx::kMaxDevices] = {};  // function attributes are per device
    if (!set[ctx->device]) {
        KF_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<HD>::kSmem));
        set[ctx->device] = true;
    }
    const Q4TcArgs a{TcArgs{(uint16_t*)out, ctx->attn_ws, reinterpret_cast<float2*>(ctx->attn_ws + rows * HD), reinterpret_cast<PagedPiece*>(ctx->attn_ws + rows * (HD + 2)), ldo, tokens, box,
                            scale * 1.4426950408889634f * 0x1p60f},
                     (const uint8_t*)kv->pool_dev, (long long)kf_paged_q4_stride(kv)};
    KF_CUDA(ctx, kf_launch_pdl(ctx, kern, dim3(grid), dim3(kThreads), Cfg<HD>::kSmem, tq, pg, pl, a, KfBound{ctx->wait_flags + kWaitPaged, (unsigned)ctx->attn_wait_us, ctx->attn_drop}));
    KF_LAUNCH_CHECK(ctx);
    KF_CUDA(ctx, kf_launch_pdl(ctx, kf_attn_paged_merge_kernel<HD, kScale2>, dim3(grid, 256 / kMergeRows), dim3(256), 0, pl, a.t));
    KF_LAUNCH_CHECK(ctx);
    return KF_OK;
}
}  // namespace

int kf_attn_paged_q4_tc(kf_ctx* ctx, const kf_paged_q4* kv, const KfPaged& pg, void* out, long long ldo, const void* q, long long ldq, int n_head, float scale, int window, int first) {
    return kv->head_dim == 128 ? launch_tc<128>(ctx, kv, pg, out, ldo, q, ldq, n_head, scale, window, first)
                               : launch_tc<64>(ctx, kv, pg, out, ldo, q, ldq, n_head, scale, window, first);
}
