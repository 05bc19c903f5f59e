// paged_read_q4.cu -- rows of K and V back out of a 4-bit cache in pages (kf_paged_read_q4).
//
//   x = step * (code - zero), in fp32, rounded once
//
// Every byte is read once and every entry written once, so HBM bounds it, and instructions are not far.  A warp takes eight positions that lie side by side in the panel, four lanes a row, and one of
// K and V of one head at a time: a unit, where the positions are one, in whole.  A lane has one word of eight codes for every group.  A code at bits 16 .. 19 of a word is the fp32 number
// code * 2^-133, at bits 20 .. 23 code * 2^-129 (subnormal numbers and the first normal ones are one ladder): a shift and an AND take the place of a conversion, and the multiply-add that brings
// it back to size takes the zero off with the rounding of code - zero.  Measured: 52184 positions of 8 heads of 128 (67 MB of codes, 214 MB of rows) 51.6 us, 5.4 TB/s, 0.84 of the copy rate;
// with conversions, a row a turn and sixteen tokens a block 80 us.
#include <algorithm>

#include "kf_paged.cuh"
#include "kf_tc.cuh"

namespace {
constexpr int kThreads = 256, kTokens = 8;  // of a block: a warp's

struct ReadParams {
    void *k, *v;
    long long ldk, ldv;
    const uint8_t* pool;
    long long page_stride;
    int n_kv, rows_per_block;
    KfPaged pg;
};
template <bool VEC>
__device__ __forceinline__ void put4(uint16_t* p, float2 a, float2 b) {
    if (VEC) *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(b.x, b.y));
    else p[0] = f32_to_bf16_bits(a.x), p[1] = f32_to_bf16_bits(a.y), p[2] = f32_to_bf16_bits(b.x), p[3] = f32_to_bf16_bits(b.y);
}
template <bool VEC>
__device__ __forceinline__ void put4(float* p, float2 a, float2 b) {
    if (VEC) *reinterpret_cast<float4*>(p) = make_float4(a.x, a.y, b.x, b.y);
    else p[0] = a.x, p[1] = a.y, p[2] = b.x, p[3] = b.y;
}

// VEC: rows of the results are aligned to four entries
template <int HD, typename Y, bool VEC>
__global__ void __launch_bounds__(kThreads) kf_paged_read_q4_kernel(const __grid_constant__ ReadParams p) {
    constexpr Q4Unit un(HD);
    constexpr int G = un.groups, kWarps = kThreads / 32;
    static_assert(kWarps == kTokens, "a warp looks a token up");
    __shared__ long long s_row[kTokens];  // a token's unit in the pool, -1: none
    __shared__ int s_in[kTokens];         // position in the unit; -1: the token belongs to no sequence
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, m0 = blockIdx.x * kTokens, nt = min(kTokens, p.pg.M - m0);
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();
    const KfPaged pg    = behind_wait(p.pg);
    const uint8_t* pool = behind_wait(p.pool);
    if (warp < nt) {
        const int s = paged_find_seq(pg, m0 + warp, lane);
        long long row = -1;
        int in = 0;
        if (s >= 0) {
            int q0, n, len;
            paged_seq(pg, s, q0, n, len);
            const int at = len - n + (m0 + warp - q0), page = at >= 0 ? paged_page(pg, s, at, in) : -1;
            if (page >= 0) row = page * p.page_stride + in / 8 * (long long)un.bytes;
        }
        if (lane == 0) s_row[warp] = row, s_in[warp] = s >= 0 ? in & 7 : -1;
    }
    __syncthreads();
    const int r0 = blockIdx.y * p.rows_per_block, r1 = min(2 * p.n_kv, r0 + p.rows_per_block), l = lane & 3, t = lane >> 2;
    if (t >= nt || s_in[t] < 0) return;
    const long long row = s_row[t], head_bytes = (long long)(pg.page / 8) * un.bytes;
    const int in        = s_in[t];
    for (int r = r0 + warp; r < r1; r += kWarps) {
        const int head  = r >> 1;
        const bool is_v = r & 1;
        if (!(is_v ? p.v : p.k)) continue;
        Y* to = is_v ? (Y*)p.v + (m0 + t) * p.ldv + head * HD : (Y*)p.k + (m0 + t) * p.ldk + head * HD;
        const uint8_t* at = pool + row + head * head_bytes;
        uint32_t w[G], s[G / 2], z[G];
        if (row < 0) {
#pragma unroll
            for (int j = 0; j < G; j++) w[j] = z[j] = s[j / 2] = 0u;
        } else if (is_v) {  // dims 32 j + 4 l .. + 3 and 32 j + 16 + 4 l .. + 3
            uint32_t x[G / 2], y[G / 2];
            const uint8_t* c = at + un.v_code() + l * (HD / 2) + (in >> 1) * (HD / 8) + (in & 1) * (HD / 16);
            words(c, x), words(c + 2 * HD, y), words(at + un.v_step() + in * 2 * G, s);
#pragma unroll
            for (int j = 0; j < G; j++) z[j] = *reinterpret_cast<const uint16_t*>(at + un.v_zero() + j * 16 + in * 2);
#pragma unroll
            for (int j = 0; j < G; j++) w[j] = __byte_perm(x[j / 2], y[j / 2], j & 1 ? 0x7632 : 0x5410);
        } else {  // dims 32 j + 8 l .. + 7
            uint32_t x[G / 2];
            words(at + in * (HD / 2) + l * 4 * G, w), words(at + un.k_step() + in * 2 * G, s), words(at + un.k_zero() + in * 2 * G, x);
#pragma unroll
            for (int j = 0; j < G; j++) z[j] = j & 1 ? x[j / 2] >> 16 : x[j / 2] & 0xffffu;
        }
        const int d0 = is_v ? 4 * l : 8 * l, d1 = is_v ? d0 + 16 : d0 + 4;
#pragma unroll
        for (int j = 0; j < G; j++) {
            const float step = j & 1 ? bf16hi(s[j / 2]) : bf16lo(s[j / 2]), zero = __uint_as_float(z[j] << 16);
            const unsigned long long up = pack2(0x1p127f, 0x1p123f), off = pack2(zero * -0x1p-6f, zero * -0x1p-6f), back = pack2(step, step), by = pack2(0x1p6f, 0x1p6f);
            float2 e[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t x = i == 0 ? w[j] << 16 : i == 1 ? w[j] << 8 : i == 2 ? w[j] : w[j] >> 8;
                // (code - zero) / 64, times 64, which is exact, times the step
                e[i] = unpack2(mul2(mul2(fma2(pack2(__uint_as_float(x & 0x000f0000u), __uint_as_float(x & 0x00f00000u)), up, off), by), back));
            }
            put4<VEC>(to + 32 * j + d0, e[0], e[1]), put4<VEC>(to + 32 * j + d1, e[2], e[3]);
        }
    }
}

template <int HD, typename Y>
int launch_read(kf_ctx* ctx, ReadParams& p, bool vec) {
    const int blocks = (p.pg.M + kTokens - 1) / kTokens, all = 2 * p.n_kv;
    const int parts  = std::max(1, std::min((all + 7) / 8, 16 * ctx->sm_count / blocks));  // few tokens: their heads over several blocks
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
