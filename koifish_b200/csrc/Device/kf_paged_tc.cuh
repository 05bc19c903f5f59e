// kf_paged_tc.cuh -- what the tcgen05 kernels for many rows over a cache in pages share (attn_paged_tc.cu, attn_paged_q4_tc.cu): tiles, the way of the chains through them, instructions of several
// steps, and the kernel that merges what several CTAs leave.
#pragma once
#include "kf_paged_walk.cuh"

#ifdef __CUDACC__
namespace {
constexpr float kSlack = 8.f;  // growth of a maximum, log2, that sums are not rescaled for
constexpr int kQ = 128, kKV = 128, kParts2 = 2 /* parts of a tile's weights */;
struct TcArgs {  // kernel parameter
    uint16_t* out;
    float* ws;        // [CTA][2][256][HD] sums, then as many (maximum, denominator) pairs, then what begins in a run and goes on behind it, per run
    float2* ws_ml;
    PagedPiece* rec;
    long long ldo;
    int tokens, box;  // tokens of a row tile; positions of a box
    float sc2;        // scale * log2(e)
};
// shared-memory descriptors of a K tile (K-major) and a V tile (MN-major: 64 dims side by side, then the next position's 128-byte row), SWIZZLE_128B: eight positions lie
// HD * 16 bytes behind the eight before (stride byte offset), V's second 64 dims 1024 bytes behind the first (leading byte offset)
template <int HD>
__device__ __forceinline__ uint64_t make_desc_kv(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | ((uint64_t)(1024 >> 4) << 16) | ((uint64_t)(HD * 16 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// four steps of 16 dims of scores: 32 bytes on in the swizzled rows of both operands each; one election for all of them
__device__ __forceinline__ void umma_scores_x4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "add.u64 a1, %1, 2;\n\tadd.u64 a2, %1, 4;\n\tadd.u64 a3, %1, 6;\n\t"
        "add.u64 b1, %2, 2;\n\tadd.u64 b2, %2, 4;\n\tadd.u64 b3, %2, 6;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, 1;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// two steps of 16 positions of sums: 8 tensor-memory columns of weights, 2 groups of 8 rows of V on
template <int GROUP>
__device__ __forceinline__ void umma_sums_x2(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b32 a1;\n\t.reg .b64 b1;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "add.u32 a1, %1, 8;\n\tadd.u64 b1, %2, %5;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "n"(2 * GROUP / 16)
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void store_row(uint16_t* p, const uint32_t (&o)[32], float f, bool vec) {
    if (vec) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = pack_bf16x2(__uint_as_float(o[8 * j + 2 * e]) * f, __uint_as_float(o[8 * j + 2 * e + 1]) * f);
            *reinterpret_cast<uint4*>(p + 8 * j) = make_uint4(v[0], v[1], v[2], v[3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; j++) p[j] = f32_to_bf16_bits(__uint_as_float(o[j]) * f);
    }
}
// the tiles of a piece as the chains take them
struct Steps {
    bool pair;  // two row tiles, which share the tiles; otherwise chain t takes every second one
    int n;      // tiles
    __device__ __forceinline__ Steps(const PagedPiece& pc, const PagedPlan& pl, int tokens) {
        pair = pc.n - pc.b * pl.tb > tokens;
        n    = pc.t1 - pc.t0;
    }
    __device__ __forceinline__ int of(int t) const { return pair ? n : (n + 1 - t) / 2; }              // steps of chain t
    __device__ __forceinline__ int tile(int t, int j) const { return pair ? j : 2 * j + t; }
};

// Blocks that several CTAs share: block (c, s) takes rows 32 s .. 32 s + 31 of the one that begins in run c and goes on behind it, if there is one.  A thread takes four entries
// of several rows, the pieces in order, the next one's on their way.
constexpr int kMergeRows = 32;
// SCALE2: the sums are 2^-SCALE2 of what they stand for
template <int HD, int SCALE2 = 0>
__global__ void __launch_bounds__(256) kf_attn_paged_merge_kernel(const __grid_constant__ PagedPlan pl, const __grid_constant__ TcArgs a) {
    constexpr int kStep = 256 / (HD / 4), kOwn = kMergeRows / kStep;  // rows side by side, rows of a thread
    const int tid = threadIdx.x, cta = blockIdx.x;
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();
    const PagedPiece pc = *behind_wait(a.rec + cta);
    const bool pair     = pc.n - pc.b * pl.tb > a.tokens;
    const int r0        = blockIdx.y * kMergeRows;
    if (pc.last <= cta || pc.last >= (int)gridDim.x || (r0 >= kQ && !pair)) return;  // last 0: nothing that goes on
    const int pieces = pc.last - cta + 1, c = tid % (HD / 4) * 4, rr = tid / (HD / 4);
    float m[kOwn], l[kOwn];
    float4 o[kOwn], v[kOwn];
    float2 ml[kOwn];
    auto ask = [&](int i) {
#pragma unroll
        for (int u = 0; u < kOwn; u++) {
            const size_t row = ((size_t)(cta + i) * 2 + (i == 0)) * 256 + r0 + rr + u * kStep;
            ml[u] = __ldcg(a.ws_ml + row), v[u] = __ldcg(reinterpret_cast<const float4*>(a.ws + row * HD + c));
        }
    };
    ask(0);
#pragma unroll
    for (int u = 0; u < kOwn; u++) m[u] = -INFINITY, l[u] = 0.f, o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i = 0; i < pieces; i++) {
        float4 w[kOwn];
        float2 wl[kOwn];
#pragma unroll
        for (int u = 0; u < kOwn; u++) w[u] = v[u], wl[u] = ml[u];
        if (i + 1 < pieces) ask(i + 1);
#pragma unroll
        for (int u = 0; u < kOwn; u++) {
            const float n = fmaxf(m[u], wl[u].x), f = ex2(m[u] - finite_or_0(n)), g = ex2(wl[u].x - finite_or_0(n));
            m[u] = n, l[u] = fmaf(l[u], f, wl[u].y * g);
            o[u].x = fmaf(o[u].x, f, w[u].x * g), o[u].y = fmaf(o[u].y, f, w[u].y * g), o[u].z = fmaf(o[u].z, f, w[u].z * g), o[u].w = fmaf(o[u].w, f, w[u].w * g);
        }
    }
    const bool vec = ((uintptr_t)a.out & 7) == 0 && a.ldo % 4 == 0;
#pragma unroll
    for (int u = 0; u < kOwn; u++) {
        const int r = r0 + rr + u * kStep, row = r % kQ, tok = pc.b * pl.tb + r / kQ * a.tokens + row / pl.group;
        if (row >= a.tokens * pl.group || tok >= pc.n) continue;  // its sums are whatever lay there
        const float inv = l[u] == 0.f ? 0.f : (SCALE2 ? __uint_as_float((127u + SCALE2) << 23) : 1.f) / l[u];
        uint16_t* op    = a.out + (pc.q0 + tok) * a.ldo + (long long)(pc.head * pl.group + row % pl.group) * HD + c;
        const uint32_t lo = pack_bf16x2(o[u].x * inv, o[u].y * inv), hi = pack_bf16x2(o[u].z * inv, o[u].w * inv);
        if (vec) *reinterpret_cast<uint2*>(op) = make_uint2(lo, hi);
        else op[0] = lo & 0xffff, op[1] = lo >> 16, op[2] = hi & 0xffff, op[3] = hi >> 16;
    }
}
}  // namespace
#endif
