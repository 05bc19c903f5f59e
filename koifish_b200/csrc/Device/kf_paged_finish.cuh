// kf_paged_finish.cuh -- the end of a piece in the attention kernels for few rows: the computing warps' sums become one, and a block's pieces its result.
#pragma once
#include "kf_paged_walk.cuh"

#ifdef __CUDACC__
namespace {
__device__ __forceinline__ void put4(uint16_t* p, float4 v, bool vec) {
    if (vec) *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    else p[0] = f32_to_bf16_bits(v.x), p[1] = f32_to_bf16_bits(v.y), p[2] = f32_to_bf16_bits(v.z), p[3] = f32_to_bf16_bits(v.w);
}
struct PagedSums {          // a CTA's place in the team and what the pieces leave for one another
    int team, mate, mates;  // team of this CTA, its number in it and how many there are
    float* ws;              // [CTA][2][rb][HD] sums
    float2* ws_ml;          // their maxima (log2) and denominators
    unsigned* cnt;          // [CTA] pieces that have arrived, 0 between launches
};
// s_o [WARPS][rb][HD], s_m and s_l [WARPS][16]: sums, maxima (log2) and denominators of the rows by warp, written and met over.  out_row(r): where row r goes.
// A CTA has at most one piece that others have begun (slot 0) and one that others go on with (slot 1); the piece that arrives last at its block merges all of them in order.
template <int HD, int WARPS, typename OutRow, typename Meet>
__device__ __forceinline__ void paged_finish(const PagedPiece& pc, const PagedSums& ps, int rows, int rb, const float* s_o, const float (*s_m)[16], const float (*s_l)[16], int* s_last, bool vec,
                                             bool& live, OutRow out_row, Meet meet) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int first = pc.first, last = pc.last;  // teams
    const size_t slot = ((size_t)ps.team * ps.mates + ps.mate) * 2 + (first == ps.team);
    for (int idx = tid; idx < rows * (HD / 4); idx += WARPS * 32) {
        const int r = idx / (HD / 4), c = idx % (HD / 4) * 4;
        float M_ = -INFINITY, L_ = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) M_ = fmaxf(M_, s_m[w][r]);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f  = s_m[w][r] == -INFINITY ? 0.f : exp2f(s_m[w][r] - M_);
            const float4 v = *reinterpret_cast<const float4*>(s_o + ((size_t)w * rb + r) * HD + c);
            L_ += s_l[w][r] * f;
            a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
        }
        if (pc.whole) {
            const float i = L_ == 0.f ? 0.f : 1.f / L_;
            put4(out_row(r) + c, make_float4(a.x * i, a.y * i, a.z * i, a.w * i), vec);
        } else {
            __stcg(reinterpret_cast<float4*>(ps.ws + (slot * rb + r) * HD + c), a);
            if (c == 0) __stcg(ps.ws_ml + slot * rb + r, make_float2(M_, L_));
        }
    }
    if (pc.whole) return;
    const int pieces = last - first + 1;
    auto slot_of = [&](int i) { return ((size_t)(first + i) * ps.mates + ps.mate) * 2 + (i == 0); };
    __threadfence();
    meet();
    if (live && tid == 0) {
        unsigned* c = ps.cnt + (size_t)first * ps.mates + ps.mate;
        *s_last     = atomicAdd(c, 1u) == (unsigned)(pieces - 1);
        if (*s_last) *c = 0u;  // self-reset for the next launch
    }
    meet();
    if (!live || !*s_last) return;
    __threadfence();
    // a row to a warp (HD 64: the halves of the warp take every second piece), its pieces in order, kAt at a time and as many more on their way
    constexpr int VEC = HD / 4, LANES = 32 / VEC, kAt = 8;
    const int half = lane / VEC, c = lane % VEC * 4;
    for (int r = warp; r < rows; r += WARPS) {
        float M_ = -INFINITY, L_ = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), v[kAt];
        float2 ml[kAt];
        auto ask = [&](int i0) {
#pragma unroll
            for (int i = 0; i < kAt; i++) {
                const int at        = i0 + i * LANES + half;
                const size_t at_row = slot_of(min(at, pieces - 1)) * rb + r;
                v[i]  = __ldcg(reinterpret_cast<const float4*>(ps.ws + at_row * HD + c));
                ml[i] = __ldcg(ps.ws_ml + at_row);
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
}  // namespace
#endif
