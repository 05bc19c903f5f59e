// paged_read_q4.cu -- rows of K and V back out of a 4-bit cache in pages (kf_paged_read_q4).
//
//   x = step * (code - zero), in fp32, rounded once
//
// Every byte is read once and every entry written once, so HBM bounds it.  A warp takes four positions that lie side by side in the panel and one of K and V of one head at a time: eight (or four)
// lanes a row, eight bytes of codes each, so that four positions of one unit meet in whole sectors of V's codes, which lie by pairs of positions.
#include <algorithm>

#include "kf_paged.cuh"

namespace {
constexpr int kThreads = 256, kTokens = 16;  // of a block

struct ReadParams {
    void *k, *v;
    long long ldk, ldv;
    const uint8_t* pool;
    long long page_stride;
    int n_kv, rows_per_block;
    KfPaged pg;
};
__device__ __forceinline__ void put(uint16_t* p, const float (&x)[8], int n) {
#pragma unroll
    for (int i = 0; i < 8; i += 4)
        if (i < n) *reinterpret_cast<uint2*>(p + i) = make_uint2(pack_bf16x2(x[i], x[i + 1]), pack_bf16x2(x[i + 2], x[i + 3]));
}
__device__ __forceinline__ void put(float* p, const float (&x)[8], int n) {
#pragma unroll
    for (int i = 0; i < 8; i += 4)
        if (i < n) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
__device__ __forceinline__ void put1(uint16_t* p, float x) { *p = f32_to_bf16_bits(x); }
__device__ __forceinline__ void put1(float* p, float x) { *p = x; }

// VEC: rows of the results are aligned to four entries
template <int HD, typename Y, bool VEC>
__global__ void __launch_bounds__(kThreads) kf_paged_read_q4_kernel(const __grid_constant__ ReadParams p) {
    constexpr Q4Unit un(HD);
    constexpr int G = un.groups, LPR = 8, RPW = 32 / LPR, kWarps = kThreads / 32;  // lanes of a row: one for each g of V's codes
    __shared__ long long s_row[kTokens];  // a token's unit in the pool, -1: none
    __shared__ int s_in[kTokens];         // position in the unit; -1: the token belongs to no sequence
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, m0 = blockIdx.x * kTokens, nt = min(kTokens, p.pg.M - m0);
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();
    const KfPaged pg    = behind_wait(p.pg);
    const uint8_t* pool = behind_wait(p.pool);
    for (int t = warp; t < nt; t += kWarps) {
        const int s = paged_find_seq(pg, m0 + t, lane);
        long long row = -1;
        int in = 0;
        if (s >= 0) {
            int q0, n, len;
            paged_seq(pg, s, q0, n, len);
            const int at = len - n + (m0 + t - q0), page = at >= 0 ? paged_page(pg, s, at, in) : -1;
            if (page >= 0) row = page * p.page_stride + in / 8 * (long long)un.bytes;
        }
        if (lane == 0) s_row[t] = row, s_in[t] = s >= 0 ? in & 7 : -1;
    }
    __syncthreads();
    const int r0 = blockIdx.y * p.rows_per_block, r1 = min(2 * p.n_kv, r0 + p.rows_per_block), quads = (nt + RPW - 1) / RPW, u = lane % LPR;
    for (int x = warp; x < quads * (r1 - r0); x += kWarps) {
        const int t = x / (r1 - r0) * RPW + lane / LPR, r = r0 + x % (r1 - r0), head = r >> 1;
        const bool is_v = r & 1;
        if (t >= nt || s_in[t] < 0 || !(is_v ? p.v : p.k)) continue;
        Y* to = is_v ? (Y*)p.v + (m0 + t) * p.ldv + head * HD : (Y*)p.k + (m0 + t) * p.ldk + head * HD;
        const long long row = s_row[t];
        const int in        = s_in[t];
        const uint8_t* at   = pool + max(row, 0ll) + (long long)head * (pg.page / 8) * un.bytes;
        const uint16_t *steps = reinterpret_cast<const uint16_t*>(at + (is_v ? un.v_step() : un.k_step())) + in * G;
        const uint16_t *zeros = reinterpret_cast<const uint16_t*>(at + (is_v ? un.v_zero() : un.k_zero()));
#pragma unroll
        for (int w = 0; w < G / 2; w++) {  // a word a time
            // K: word w of the lane's G / 2 is entries 32 j + 8 t .. + 7, j = (u * G / 2 + w) % G, t = (u * G / 2 + w) / G; V: 4 entries of groups 2 w and 2 w + 1
            uint32_t c = 0;
            if (row >= 0) c = is_v ? *reinterpret_cast<const uint32_t*>(at + un.v_code() + u * (HD / 2) + (in >> 1) * (HD / 8) + (in & 1) * (HD / 16) + w * 4)
                                   : *reinterpret_cast<const uint32_t*>(at + in * (HD / 2) + (u * (G / 2) + w) * 4);
            const int ka = (u * (G / 2) + w) % G, kt = (u * (G / 2) + w) / G;
            float e[8];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int j      = is_v ? 2 * w + h : ka;
                const float step = row >= 0 ? bf16_bits_to_f32(steps[j]) : 0.f, zero = row >= 0 ? bf16_bits_to_f32(is_v ? zeros[j * 8 + in] : zeros[in * G + j]) : 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++) e[4 * h + i] = step * ((float)((c >> (16 * h + 4 * i)) & 15u) - zero);
            }
            const int d0 = is_v ? 64 * w + 4 * u : 32 * ka + 8 * kt, d1 = is_v ? d0 + 32 : d0 + 4;
            if (VEC) {
                put(to + d0, e, 4);
                const float f[8] = {e[4], e[5], e[6], e[7]};
                put(to + d1, f, 4);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) put1(to + d0 + i, e[i]), put1(to + d1 + i, e[4 + i]);
            }
        }
    }
}

template <int HD, typename Y>
int launch_read(kf_ctx* ctx, ReadParams& p, bool vec) {
    const int blocks = (p.pg.M + kTokens - 1) / kTokens, all = 2 * p.n_kv;
    const int parts  = std::max(1, std::min(all, 4 * ctx->sm_count / blocks));  // few tokens: their heads over several blocks
    p.rows_per_block = (all + parts - 1) / parts;
    const dim3 grid(blocks, (all + p.rows_per_block - 1) / p.rows_per_block);
    KF_CUDA(ctx, kf_launch_pdl(ctx, vec ? kf_paged_read_q4_kernel<HD, Y, true> : kf_paged_read_q4_kernel<HD, Y, false>, grid, dim3(kThreads), 0, p));
    KF_LAUNCH_CHECK(ctx);
    return KF_OK;
}
int read_args(kf_ctx* ctx, const kf_paged_q4* kv, const void* k, int ldk, const void* v, int ldv, int out_f32, int M, KfPaged* pg) {
    if (!kv || (!k && !v)) return KF_ERR_BAD_ARG;
    const int rc = kf_paged_q4_check(ctx, kv, M, pg);
    if (rc) return rc;
    const size_t size = out_f32 ? 4 : 2, wide = (size_t)kv->n_kv * kv->head_dim;
    KF_REQUIRE(ctx, out_f32 == 0 || out_f32 == 1, "out_f32 0 or 1");
    KF_REQUIRE(ctx, (!k || (long long)wide <= ldk) && (!v || (long long)wide <= ldv), "rows as long as their heads");
    KF_REQUIRE(ctx, (((uintptr_t)k | (uintptr_t)v) & (size - 1)) == 0, "results at their own alignment");
    KF_REQUIRE(ctx, !k || !v || !kf_rows_overlap(k, ldk * size, wide * size, v, ldv * size, wide * size, M), "keys over values");
    return KF_OK;
}
}  // namespace

extern "C" int kf_paged_read_q4(kf_ctx* ctx, const kf_paged_q4* kv, void* k, int ldk, void* v, int ldv, int out_f32, int M) {
    if (!ctx) return KF_ERR_BAD_ARG;
    ReadParams p = {};
    const int rc = read_args(ctx, kv, k, ldk, v, ldv, out_f32, M, &p.pg);
    if (rc || M == 0) return rc;
    p.k = k, p.v = v, p.ldk = ldk, p.ldv = ldv, p.pool = (const uint8_t*)kv->pool_dev, p.page_stride = (long long)kf_paged_q4_stride(kv), p.n_kv = kv->n_kv;
    const uintptr_t mask = out_f32 ? 15 : 7;
    const bool vec       = (((uintptr_t)k | (uintptr_t)v) & mask) == 0 && (!k || ldk % 4 == 0) && (!v || ldv % 4 == 0);
    if (kv->head_dim == 128) return out_f32 ? launch_read<128, float>(ctx, p, vec) : launch_read<128, uint16_t>(ctx, p, vec);
    return out_f32 ? launch_read<64, float>(ctx, p, vec) : launch_read<64, uint16_t>(ctx, p, vec);
}
// The checks for tests on a host without a device
extern "C" int kf_paged_read_q4_args(const kf_paged_q4* kv, const void* k, int ldk, const void* v, int ldv, int out_f32, int M) {
    KfPaged pg;
    return read_args(nullptr, kv, k, ldk, v, ldv, out_f32, M, &pg);
}
