// paged_append.cu -- a step's keys and values into the pages of their sequences with the norm and the rotation of q and k on the way (kf_paged_append), and the
// rotation alone (kf_rope_axes).
//
//   y = x * rsqrt(mean(x^2) + eps) * w (per head; optional),  pair j: (a, b) -> amp * (a cos t - b sin t, b cos t + a sin t),  t = pos[axis[j]][row] * inv_freq[j]
//
// Every element is read once and written once, so HBM bounds the large calls and latency the small ones.  A block takes up to four tokens, whose rotations are worked out once
// for all their heads: t / pi in 64 bits, reduced to [-1, 1] there (a far position turns many times; its remainder in 32 bits would be off by more than the result's
// rounding), then sine and cosine in 32 bits.  A head's row is spread over 4, 8 or 16 lanes; a lane holds eight pairs, so both of a pair's entries are its own: 16 bytes of
// either half of the rotated part, or 32 bytes in a row where pairs lie side by side.  (With 16 bytes a lane and the other half from another lane by shuffles, one token a
// block: 8192 tokens of 64 + 8 + 8 heads with their norm 148 us, 16001 tokens of 40 heads 165 us; here 64 and 57, in a steady run 68 and 59, 4.9 and 5.5
// TB/s.)  What bounds it is how many bytes are on their way: four or five blocks per SM, a lane's next rows asked for before it works on its own.  With the norm: one row ahead
// and the weights in shared memory, five blocks (two rows, four blocks: 67 us; weights in registers, which spill: 76); without, two rows ahead (one: 61, three: 69).  The first
// rows are asked for before the positions are known: finding the sequence of a token, its page and its position are three dependent reads.  Few tokens are spread over blocks by
// heads.  Rows at any element, heads that are no multiple of 16 and, with pairs apart, rotated parts that are none go entry by entry: 16000 tokens of 16 heads of 72 83 us, 0.9 TB/s
// (of 80, whole lanes: 33 us, 2.5 TB/s); with 24 of 64 entries rotated 91 us.
//
// kf_paged_append_q4 writes rows of K and V as 4-bit codes with a step and a zero for every 32 entries (kf_device.h): the same kernel, whose finished rows of K and V go through shared memory so that
// two lanes hold a group.  8007 tokens of 64 + 8 + 8 heads with their norm, written and read back: 87 us, of which the quantisation is about 7 (divisions by the compiler: 22), reading back
// 14; 5000 tokens of 32 + 8 + 8 float heads with three axes 53.
#include <algorithm>
#include <type_traits>

#include "kf_paged.cuh"
#include "kf_tc.cuh"

namespace {
constexpr int kThreads = 256, kTokens = 4;  // of a block at most

struct RowsParams {
    const void *q, *k, *v;
    long long ldq, ldk, ldv, ldo;
    void* out;
    int nq, nkv /* 0: no cache */, hd, M, tokens, rows_per_block;  // tokens of a block and rows of each
    const double* freq;
    const int32_t *axis, *pos;
    long long pos_stride;
    int rot, layout, n_axes;
    float amp;
    const uint16_t *qw, *kw;
    float eps;
    uint16_t *kc, *vc;
    uint8_t* pool;          // the 4-bit cache's pages, instead
    long long page_stride;  // elements; of the 4-bit cache bytes
    KfPaged pg;
};

__device__ __forceinline__ float load1(const uint16_t* p) { return bf16_bits_to_f32(*p); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ void store1(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
// eight entries as they lie in memory, and as four pairs of floats
typedef unsigned long long f32x2;
template <typename X>
struct Raw;
template <>
struct Raw<uint16_t> {
    uint4 a;
    __device__ __forceinline__ void load(const uint16_t* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(f32x2 (&f)[4]) const { f[0] = pack2(bf16lo(a.x), bf16hi(a.x)), f[1] = pack2(bf16lo(a.y), bf16hi(a.y)), f[2] = pack2(bf16lo(a.z), bf16hi(a.z)), f[3] = pack2(bf16lo(a.w), bf16hi(a.w)); }
};
template <>
struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ void get(f32x2 (&f)[4]) const { f[0] = pack2(a.x, a.y), f[1] = pack2(a.z, a.w), f[2] = pack2(b.x, b.y), f[3] = pack2(b.z, b.w); }
};
__device__ __forceinline__ void store8(uint16_t* p, const f32x2 (&f)[4]) {
    const float2 a = unpack2(f[0]), b = unpack2(f[1]), c = unpack2(f[2]), d = unpack2(f[3]);
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(b.x, b.y), pack_bf16x2(c.x, c.y), pack_bf16x2(d.x, d.y));
}
__device__ __forceinline__ void store8(float* p, const f32x2 (&f)[4]) {
    const float2 a = unpack2(f[0]), b = unpack2(f[1]), c = unpack2(f[2]), d = unpack2(f[3]);
    reinterpret_cast<float4*>(p)[0] = make_float4(a.x, a.y, b.x, b.y), reinterpret_cast<float4*>(p)[1] = make_float4(c.x, c.y, d.x, d.y);
}

__device__ __forceinline__ uint16_t bf16_bits_up(float f) { return (uint16_t)((__float_as_uint(f) + 0xffffu) >> 16); }  // f >= 0
// the smallest and the largest of three; NaN if one of them is
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(a) : "f"(a), "f"(b), "f"(c));
    return a;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(a) : "f"(a), "f"(b), "f"(c));
    return a;
}
// A finished row of K or V into its unit of the 4-bit cache.  HD / 16 lanes side by side hold 16 entries each in `x`, entries 16 u .. 16 u + 15 in lane u; two lanes are a group.
// All lanes of the warp call it; `to` (NULL: nothing is written) is the unit, p the position in it.
template <int HD>
__device__ __forceinline__ void store_q4(uint8_t* to, int p, bool is_v, int u, const float (&x)[16]) {
    constexpr Q4Unit un(HD);
    constexpr int G = un.groups;
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 15; i += 2) lo = min3_nan(lo, x[i], x[i + 1]), hi = max3_nan(hi, x[i], x[i + 1]);
    lo = min3_nan(lo, x[15], __shfl_xor_sync(0xffffffffu, min3_nan(lo, x[15], x[15]), 1)), hi = max3_nan(hi, x[15], __shfl_xor_sync(0xffffffffu, max3_nan(hi, x[15], x[15]), 1));
    const float most  = max3_nan(hi, -lo, 0.f);
    const bool fine   = most < INFINITY;  // not NaN either
    const uint32_t sb = fine ? bf16_bits_up(fmaxf(__fdiv_rn(hi - lo, 15.f), most * (1.f / 2048.f))) : 0x7fffu;
    const float step  = fine && sb ? bf16_bits_to_f32(sb) : 1.f;
    const uint32_t zb = fine && sb ? f32_to_bf16_bits(__fdiv_rn(-lo, step)) : 0u;
    const float zero  = bf16_bits_to_f32(zb);
    // x / step, correctly rounded, so that a tie is a tie: with y = 1 / step correctly rounded and q = x y, q + (x - q step) y is (Markstein's theorem), away from the ends of the range
    f32x2 q[8];
    const bool mid = step > 0x1p-90f && step < 0x1p90f;
    if (__all_sync(0xffffffffu, mid)) {
        const float y   = __frcp_rn(step);
        const f32x2 y2  = pack2(y, y), s2 = pack2(-step, -step);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const f32x2 a = pack2(x[2 * i], x[2 * i + 1]), b = mul2(a, y2);
            q[i] = fma2(fma2(b, s2, a), y2, b);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = pack2(__fdiv_rn(x[2 * i], step), __fdiv_rn(x[2 * i + 1], step));
    }
    uint32_t c[2] = {0u, 0u};  // entries 8 e .. 8 e + 7
#pragma unroll
    for (int i = 7; i >= 0; i--) {
        const float2 t = unpack2(add2(q[i], pack2(zero, zero)));
        // kept to 0 .. 15 (NaN: 0); in front of 1.5 * 2^23 the nearest whole number, ties to even, is what is left in the lowest bits
        const float2 r = unpack2(add2(pack2(fminf(fmaxf(t.x, 0.f), 15.f), fminf(fmaxf(t.y, 0.f), 15.f)), pack2(12582912.f, 12582912.f)));
        c[i >> 2]      = c[i >> 2] << 8 | (__float_as_uint(r.y) & 15u) << 4 | (__float_as_uint(r.x) & 15u);
    }
    if (!fine) c[0] = c[1] = 0u;
    const int j = u >> 1;
    // Values: entries 4 g .. 4 g + 3 of two groups are a word.  The lanes that hold the same entries of the two (u and u ^ 2) exchange halves, so that each has two whole words, of the
    // first two of their four g in the lane of the even group, of the others in that of the odd one; with four groups (HD 128) the words of both halves of the row meet likewise.
    const bool odd      = j & 1;
    const uint32_t got  = __shfl_xor_sync(0xffffffffu, odd ? c[0] : c[1], 2), keep = odd ? c[1] : c[0];
    const uint32_t even = odd ? got : keep, other = odd ? keep : got;
    const uint32_t w0 = (even & 0xffffu) | other << 16, w1 = even >> 16 | (other & 0xffff0000u);
    const bool far      = u >> 2;
    const uint32_t give = HD == 128 ? __shfl_xor_sync(0xffffffffu, far ? w0 : w1, 4) : 0u, mine = far ? w1 : w0;
    if (!to) return;
    uint16_t *step_at, *zero_at;
    if (is_v) {
        const int g = (u & 1) * 4 + odd * 2;
        uint8_t* at = to + un.v_code() + (p >> 1) * (HD / 8) + (p & 1) * (HD / 16);
        if (HD == 128) *reinterpret_cast<uint2*>(at + (g + far) * (HD / 2)) = make_uint2(far ? give : mine, far ? mine : give);
        else *reinterpret_cast<uint32_t*>(at + g * (HD / 2)) = w0, *reinterpret_cast<uint32_t*>(at + (g + 1) * (HD / 2)) = w1;
        step_at = reinterpret_cast<uint16_t*>(to + un.v_step()) + p * G + j, zero_at = reinterpret_cast<uint16_t*>(to + un.v_zero()) + j * 8 + p;
    } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(to + p * (HD / 2));
        w[(u & 1) * 2 * G + j] = c[0], w[((u & 1) * 2 + 1) * G + j] = c[1];
        step_at = reinterpret_cast<uint16_t*>(to + un.k_step()) + p * G + j, zero_at = reinterpret_cast<uint16_t*>(to + un.k_zero()) + p * G + j;
    }
    if (!(u & 1)) *step_at = (uint16_t)sb, *zero_at = (uint16_t)zb;
}

// LPR: lanes to a row, eight pairs each; 0: rows at any element, or pairs that do not fall on whole lanes -- a warp per row, an entry or a pair per lane
// Q4: the cache is the 4-bit one, head_dim Q4 (0: bf16).  A finished row of K or V goes through shared memory there, so that a lane gets 16 entries side by side
template <typename X, typename Y, int LPR, bool NORM, int Q4 = 0>
__global__ void __launch_bounds__(kThreads, LPR == 0 ? 1 : Q4 ? 4 : NORM && sizeof(X) == 2 ? 5 : 4) kf_rows_kernel(const __grid_constant__ RowsParams p) {
    constexpr int kL = LPR ? LPR : 32, kGroups = kThreads / kL, kAhead = sizeof(X) == 4 || NORM ? 1 : 2;  // rows of a lane on their way beside those in its hands
    __shared__ alignas(16) float s_cos[kTokens][128], s_sin[kTokens][128];
    __shared__ long long s_row[kTokens];  // a token's row in the pools, -1: none
    __shared__ int s_at[kTokens];         // its position in the sequence
    __shared__ bool s_ours[kTokens];      // it belongs to a sequence
    __shared__ alignas(16) uint16_t s_w[NORM ? 2 : 1][256];  // norm weights of q and k
    __shared__ alignas(16) float s_cache[Q4 ? kThreads / kL : 1][Q4 ? Q4 + 4 : 1];
    __shared__ int s_in[kTokens];  // Q4: the position's row in its page
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = tid / kL, v = tid % kL, m0 = blockIdx.x * p.tokens, nt = min(p.tokens, p.M - m0);
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();  // the panel, positions, lengths and tables come from the kernels before us
    const X *q = behind_wait((const X*)p.q), *k = behind_wait((const X*)p.k), *vv = behind_wait((const X*)p.v);
    const KfPaged pg = behind_wait(p.pg);
    const int all = p.nq + 2 * p.nkv, r0 = blockIdx.y * p.rows_per_block, r1 = min(all, r0 + p.rows_per_block), half = p.rot / 2;
    auto src = [&](int t, int r) -> const X* {
        const long long m = m0 + t;
        return r < p.nq ? q + m * p.ldq + r * p.hd : r < p.nq + p.nkv ? k + m * p.ldk + (r - p.nq) * p.hd : vv + m * p.ldv + (r - p.nq - p.nkv) * p.hd;
    };
    // a lane's two runs of eight entries: the pairs' first and second entries, entries side by side, or behind the rotated part
    const int ea = p.layout && 8 * v < half ? 8 * v : p.layout ? p.rot + 16 * (v - half / 8) : 16 * v, eb = p.layout && 8 * v < half ? half + 8 * v : ea + 8;
    const bool lives = LPR && 16 * v < p.hd;
    Raw<X> ra[kAhead], rb[kAhead];
    // rows rb0 + grp, kGroups further on, ... of token t.  Q4: half a turn further in every other token, since rows of K and V, the last ones, take longer
    auto row_at = [&](int t, int rb0, int u) { return rb0 + (Q4 ? (grp + (t & 1) * (kGroups / 2)) % kGroups : grp) + u * kGroups; };
    auto fetch  = [&](int t, int rb0) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int r = row_at(t, rb0, u);
            if (lives && r < r1) {
                const X* from = src(t, r);
                ra[u].load(from + ea), rb[u].load(from + eb);
            }
        }
    };
    if (LPR) fetch(0, r0);
    if (p.nkv) {
        if (warp < nt) {
            const int s = paged_find_seq(pg, m0 + warp, lane);
            long long row = -1;
            int at = 0;
            if (s >= 0) {
                int q0, n, len, in = 0;
                paged_seq(pg, s, q0, n, len);
                at             = len - n + (m0 + warp - q0);
                const int page = at >= 0 ? paged_page(pg, s, at, in) : -1;
                if (page >= 0) row = page * p.page_stride + (Q4 ? in / 8 * (long long)Q4Unit(Q4).bytes : (long long)in * p.nkv * p.hd);
                if (Q4 && lane == 0) s_in[warp] = in;
            }
            if (lane == 0) s_row[warp] = row, s_at[warp] = at, s_ours[warp] = s >= 0;
        }
        __syncthreads();
    }
    if (NORM && LPR)
        for (int i = tid; i < 2 * p.hd; i += kThreads) {
            const uint16_t* w = i < p.hd ? p.qw : p.kw;
            if (w) s_w[i >= p.hd][i < p.hd ? i : i - p.hd] = w[i < p.hd ? i : i - p.hd];
        }
    for (int i = tid; i < nt * half; i += kThreads) {
        const int t = i / half, j = i - t * half, ax = p.axis ? p.axis[j] : 0;
        float sn = 0.f, cs = 1.f;
        if (ax >= 0 && ax < p.n_axes) {
            const double a = (double)(p.pos ? p.pos[ax * p.pos_stride + m0 + t] : s_at[t]) * p.freq[j] * 0.31830988618379067154;
            sincospif((float)(a - 2.0 * rint(0.5 * a)), &sn, &cs);
            cs *= p.amp, sn *= p.amp;
        }
        s_cos[t][j] = cs, s_sin[t][j] = sn;
    }
    __syncthreads();
    if constexpr (LPR != 0) {
        const bool turns = lives && 8 * v < half;
        for (int t = 0, rb0 = r0; t < nt;) {
            Raw<X> ca[kAhead], cb[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++) ca[u] = ra[u], cb[u] = rb[u];
            int tn = t, rn = rb0 + kAhead * kGroups;
            if (rn >= r1) tn++, rn = r0;
            if (tn < nt) fetch(tn, rn);  // the next rows are on their way meanwhile
            const bool ours  = !p.nkv || s_ours[t];
            const long long row = p.nkv ? s_row[t] : -1;
            Y* out           = (Y*)p.out + (m0 + t) * p.ldo;
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const int r = row_at(t, rb0, u);
                if (!ours || __all_sync(0xffffffffu, r >= r1)) break;
                const bool is_q = r < p.nq, is_v = r >= p.nq + p.nkv, live = lives && r < r1;
                f32x2 a[4], b[4];
                ca[u].get(a), cb[u].get(b);
                if (NORM) {
                    f32x2 s2 = 0ull;
#pragma unroll
                    for (int i = 0; i < 4; i++) s2 = fma2(a[i], a[i], fma2(b[i], b[i], s2));
                    const float2 s = unpack2(s2);
                    float ss       = live ? s.x + s.y : 0.f;
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    if ((is_q ? p.qw : p.kw) && !is_v) {
                        const float inv = rsqrtf(ss / (float)p.hd + p.eps);
                        const f32x2 iv  = pack2(inv, inv);
                        f32x2 g[4], h[4];
                        Raw<uint16_t> w[2];  // from shared memory: in registers they cost a block per SM
                        w[0].load(s_w[!is_q] + ea), w[1].load(s_w[!is_q] + eb);
                        w[0].get(g), w[1].get(h);
#pragma unroll
                        for (int i = 0; i < 4; i++) a[i] = mul2(mul2(a[i], iv), g[i]), b[i] = mul2(mul2(b[i], iv), h[i]);
                    }
                }
                if (!Q4 && !live) continue;
                if (turns && !is_v) {
                    if (p.layout) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float2 cc = *reinterpret_cast<const float2*>(&s_cos[t][8 * v + 2 * i]), sn = *reinterpret_cast<const float2*>(&s_sin[t][8 * v + 2 * i]);
                            const f32x2 c2 = pack2(cc.x, cc.y), e = a[i];
                            a[i] = fma2(b[i], pack2(-sn.x, -sn.y), mul2(e, c2)), b[i] = fma2(e, pack2(sn.x, sn.y), mul2(b[i], c2));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float2 e = unpack2(a[i]), f = unpack2(b[i]);
                            const float c0 = s_cos[t][8 * v + i], n0 = s_sin[t][8 * v + i], c1 = s_cos[t][8 * v + 4 + i], n1 = s_sin[t][8 * v + 4 + i];
                            if (8 * v + i < half) a[i] = pack2(e.x * c0 - e.y * n0, e.y * c0 + e.x * n0);
                            if (8 * v + 4 + i < half) b[i] = pack2(f.x * c1 - f.y * n1, f.y * c1 + f.x * n1);
                        }
                    }
                }
                if (Q4) {
                    if (is_q && live) {
                        Y* to = out + r * p.hd;
                        store8(to + ea, a), store8(to + eb, b);
                    }
                    if (!__any_sync(0xffffffffu, live && !is_q)) continue;
                    float* st = s_cache[grp];
                    store8(st + ea, a), store8(st + eb, b);
                    __syncwarp();
                    float x[16];
#pragma unroll
                    for (int i = 0; i < 4; i++) *reinterpret_cast<float4*>(&x[4 * i]) = *reinterpret_cast<const float4*>(st + 16 * v + 4 * i);
                    const int head = is_v ? r - p.nq - p.nkv : r - p.nq;
                    store_q4<Q4 ? Q4 : 128>(live && !is_q && row >= 0 ? p.pool + row + (long long)head * (pg.page / 8) * Q4Unit(Q4).bytes : nullptr, s_in[t] & 7, is_v, v, x);
                    __syncwarp();
                } else if (is_q) {
                    Y* to = out + r * p.hd;
                    store8(to + ea, a), store8(to + eb, b);
                } else if (row >= 0) {
                    uint16_t* to = is_v ? p.vc + row + (r - p.nq - p.nkv) * p.hd : p.kc + row + (r - p.nq) * p.hd;
                    store8(to + ea, a), store8(to + eb, b);
                }
            }
            t = tn, rb0 = rn;
        }
    } else {
        for (int x = grp; x < nt * (r1 - r0); x += kGroups) {  // a warp per row
            const int t = x / (r1 - r0), r = r0 + x % (r1 - r0);
            const bool is_q = r < p.nq, is_v = r >= p.nq + p.nkv;
            if (p.nkv && (!s_ours[t] || (!is_q && s_row[t] < 0))) continue;
            const X* in_row   = src(t, r);
            const uint16_t* w = is_v ? nullptr : is_q ? p.qw : p.kw;
            float inv = 1.f;
            if (w) {
                float ss = 0.f;
                for (int i = lane; i < p.hd; i += 32) ss = fmaf(load1(in_row + i), load1(in_row + i), ss);
                inv = rsqrtf(warp_sum(ss) / (float)p.hd + p.eps);
            }
            auto in     = [&](int i) { return w ? load1(in_row + i) * inv * bf16_bits_to_f32(w[i]) : load1(in_row + i); };
            Y* to       = (Y*)p.out + (m0 + t) * p.ldo + r * p.hd;
            uint16_t* c = is_q || Q4 ? nullptr : is_v ? p.vc + s_row[t] + (r - p.nq - p.nkv) * p.hd : p.kc + s_row[t] + (r - p.nq) * p.hd;
            auto put    = [&](int i, float y) {
                if (is_q) store1(to + i, y);
                else if (Q4) s_cache[grp][i] = y;
                else store1(c + i, y);
            };
            const int pairs = is_v ? 0 : half;
            for (int j = lane; j < pairs; j += 32) {
                const int ia = p.layout ? j : 2 * j, ib = p.layout ? j + half : 2 * j + 1;
                const float a = in(ia), b = in(ib), cs = s_cos[t][j], sn = s_sin[t][j];
                put(ia, a * cs - b * sn), put(ib, b * cs + a * sn);
            }
            for (int i = 2 * pairs + lane; i < p.hd; i += 32) put(i, in(i));
            if (Q4 && !is_q) {
                __syncwarp();
                const int u = min(lane, Q4 / 16 - 1), head = is_v ? r - p.nq - p.nkv : r - p.nq;
                float e[16];
                for (int i = 0; i < 16; i++) e[i] = s_cache[grp][16 * u + i];
                store_q4<Q4 ? Q4 : 128>(lane < Q4 / 16 ? p.pool + s_row[t] + (long long)head * (pg.page / 8) * Q4Unit(Q4).bytes : nullptr, s_in[t] & 7, is_v, lane & (Q4 / 16 - 1), e);
                __syncwarp();
            }
        }
    }
}

template <typename X, typename Y>
int launch_rows(kf_ctx* ctx, RowsParams& p, bool wide) {
    const int lpr = !wide ? 0 : p.hd <= 64 ? 4 : p.hd <= 128 ? 8 : 16, groups = kThreads / (lpr ? lpr : 32), all = p.nq + 2 * p.nkv;
    // many tokens: four to a block; few: their heads over several blocks, up to four blocks per SM
    p.tokens        = p.M >= 4 * kTokens * ctx->sm_count ? kTokens : 1;
    const int parts = std::max(1, std::min((all + groups - 1) / groups, 4 * ctx->sm_count / p.M));
    p.rows_per_block = ((all + parts - 1) / parts + groups - 1) / groups * groups;
    const dim3 grid((p.M + p.tokens - 1) / p.tokens, (all + p.rows_per_block - 1) / p.rows_per_block);
    auto pick = [&](auto normed) {
        constexpr bool N = decltype(normed)::value;
        if constexpr (std::is_same_v<Y, uint16_t>)  // finished queries are bf16
            if (p.pool) {
                if (p.hd == 64) return lpr ? kf_rows_kernel<X, Y, 4, N, 64> : kf_rows_kernel<X, Y, 0, N, 64>;
                return lpr ? kf_rows_kernel<X, Y, 8, N, 128> : kf_rows_kernel<X, Y, 0, N, 128>;
            }
        return lpr == 0 ? kf_rows_kernel<X, Y, 0, N> : lpr == 4 ? kf_rows_kernel<X, Y, 4, N> : lpr == 8 ? kf_rows_kernel<X, Y, 8, N> : kf_rows_kernel<X, Y, 16, N>;
    };
    auto kern = p.qw || p.kw ? pick(std::true_type()) : pick(std::false_type());
    KF_CUDA(ctx, kf_launch_pdl(ctx, kern, grid, dim3(kThreads), 0, p));
    KF_LAUNCH_CHECK(ctx);
    return KF_OK;
}
int rotation(kf_ctx* ctx, const kf_rotation* rot, int hd, int M, RowsParams* p) {
    p->amp = 1.f, p->n_axes = 1;
    if (!rot) return KF_OK;
    KF_REQUIRE(ctx, rot->rot_dims >= 0 && rot->rot_dims <= hd && rot->rot_dims % 2 == 0, "rot_dims: even, at most head_dim");
    KF_REQUIRE(ctx, (rot->layout == 0 || rot->layout == 1) && rot->n_axes >= 1 && rot->n_axes <= 8, "layout 0 or 1, 1 to 8 axes");
    KF_REQUIRE(ctx, rot->rot_dims == 0 || rot->inv_freq_dev, "frequencies");
    KF_REQUIRE(ctx, rot->pos_stride == 0 || rot->pos_stride >= (size_t)M, "pos_stride: at least a position per row");
    p->freq = rot->inv_freq_dev, p->axis = rot->axis_dev, p->pos = rot->pos_dev, p->pos_stride = (long long)(rot->pos_stride ? rot->pos_stride : (size_t)M);
    p->rot = rot->rot_dims, p->layout = rot->layout, p->n_axes = rot->n_axes, p->amp = rot->amp;
    return KF_OK;
}
bool whole_lanes(const RowsParams& p) { return p.hd % 16 == 0 && (p.layout == 0 || p.rot % 16 == 0); }
}  // namespace

// what the caches in bf16 and in 4 bits have in common
template <typename KV>
static int check_step(kf_ctx* ctx, const KV* kv, int M, KfPaged* out) {
    KF_REQUIRE(ctx, kv->table_dev && kv->q_start_dev && kv->len_dev, "table, starts and lengths");
    KF_REQUIRE(ctx, kv->head_dim == 64 || kv->head_dim == 128, "head_dim 64 or 128");
    KF_REQUIRE(ctx, kv->n_kv >= 1 && kv->n_kv <= 1024 && kv->n_pages >= 1 && kv->page_size >= 8 && kv->page_size % 8 == 0, "n_kv 1 .. 1024, page_size a multiple of 8");
    KF_REQUIRE(ctx, kv->table_cols >= 1 && (long long)kv->table_cols * kv->page_size <= 0x7fffffff - 256, "table_cols");
    KF_REQUIRE(ctx, kv->n_seq >= 1 && kv->n_seq <= 8192 && M >= 0, "n_seq 1 .. 8192");
    *out = KfPaged{kv->table_dev, kv->q_start_dev, kv->len_dev, kv->table_cols, kv->n_seq, kv->n_pages, kv->page_size, kv->table_cols * kv->page_size, M, 0, 0};
    kf_paged_divisor(out);
    return KF_OK;
}
int kf_paged_check(kf_ctx* ctx, const kf_paged_kv* kv, int M, KfPaged* out) {
    KF_REQUIRE(ctx, kv->k_dev && kv->v_dev, "cache");
    const int rc = check_step(ctx, kv, M, out);
    if (rc) return rc;
    KF_REQUIRE(ctx, kv->page_stride == 0 || (kv->page_stride % 8 == 0 && kv->page_stride >= (size_t)kv->page_size * kv->n_kv * kv->head_dim), "page_stride: a multiple of 8, at least a page");
    KF_REQUIRE(ctx, (((uintptr_t)kv->k_dev | (uintptr_t)kv->v_dev) & 15) == 0, "pages at 16 bytes");
    return KF_OK;
}
extern "C" size_t kf_paged_q4_page_bytes(int page_size, int n_kv, int head_dim) {
    return page_size >= 8 && page_size % 8 == 0 && n_kv >= 1 && (head_dim == 64 || head_dim == 128) ? (size_t)(page_size / 8) * n_kv * Q4Unit(head_dim).bytes : 0;
}
int kf_paged_q4_check(kf_ctx* ctx, const kf_paged_q4* kv, int M, KfPaged* out) {
    KF_REQUIRE(ctx, kv->pool_dev, "cache");
    const int rc = check_step(ctx, kv, M, out);
    if (rc) return rc;
    KF_REQUIRE(ctx, kv->page_stride == 0 || (kv->page_stride % 16 == 0 && kv->page_stride >= kf_paged_q4_page_bytes(kv->page_size, kv->n_kv, kv->head_dim)),
               "page_stride: a multiple of 16, at least a page");
    KF_REQUIRE(ctx, kv->page_stride < (1ull << 62), "page_stride");
    KF_REQUIRE(ctx, ((uintptr_t)kv->pool_dev & 15) == 0, "pages at 16 bytes");
    return KF_OK;
}

extern "C" int kf_rows_overlap(const void* a, size_t a_pitch, size_t a_wide, const void* b, size_t b_pitch, size_t b_wide, int M) {
    const long long d = (long long)((uintptr_t)b - (uintptr_t)a), ap = (long long)a_pitch, bp = (long long)b_pitch, aw = (long long)a_wide, bw = (long long)b_wide;
    if (M <= 0 || d >= (M - 1) * ap + aw || d + (M - 1) * bp + bw <= 0) return 0;
    // rows side by side in one panel have one pitch: then only the distance of two rows matters, and the first and the last row of a meet every distance there is
    for (long long i = 0; i < M; i += ap == bp && M > 1 ? M - 1 : 1) {
        const long long before = i * ap - d - bw, j = before < 0 ? 0 : before / bp + 1;  // the first row of b that ends behind the start of row i of a
        if (j < M && d + j * bp < i * ap + aw) return 1;
    }
    return 0;
}

static int check_cache(kf_ctx* ctx, const kf_paged_kv* kv, int M, KfPaged* out) { return kf_paged_check(ctx, kv, M, out); }
static int check_cache(kf_ctx* ctx, const kf_paged_q4* kv, int M, KfPaged* out) { return kf_paged_q4_check(ctx, kv, M, out); }
template <typename KV>
static int append_args(kf_ctx* ctx, const KV* kv, const kf_rotation* rot, const void* q_out, int ldqo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv,
                       int src_f32, int M, int n_head, RowsParams* p) {
    if (!kv || !q_out || !q || !k || !v) return KF_ERR_BAD_ARG;
    int rc = check_cache(ctx, kv, M, &p->pg);
    if (!rc) rc = rotation(ctx, rot, kv->head_dim, M, p);
    if (rc) return rc;
    const int hd = kv->head_dim;
    KF_REQUIRE(ctx, n_head >= 1 && (long long)n_head * hd <= ldq && (long long)n_head * hd <= ldqo && (long long)kv->n_kv * hd <= ldk && (long long)kv->n_kv * hd <= ldv,
               "rows as long as their heads");
    KF_REQUIRE(ctx, src_f32 == 0 || (src_f32 == 1 && q_out != q), "src_f32 0 or 1; float queries are not finished in place");
    KF_REQUIRE(ctx, q_out != q || ldqo == ldq, "in place: rows where they were");
    return KF_OK;
}
// the cache's own addresses are in p already
template <typename KV>
static int append(kf_ctx* ctx, RowsParams& p, const KV* kv, const kf_rotation* rot, void* q_out, int ldqo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, int src_f32,
                  int M, int n_head, const void* qnorm_w, const void* knorm_w, float eps) {
    const int rc = append_args(ctx, kv, rot, q_out, ldqo, q, ldq, k, ldk, v, ldv, src_f32, M, n_head, &p);
    if (rc) return rc;
    const int hd = kv->head_dim;
    if (M == 0) return KF_OK;
    const size_t per_in = src_f32 ? 4 : 2, q_wide = (size_t)n_head * hd, kv_wide = (size_t)kv->n_kv * hd;
    auto over = [&](const void* x, int ldx, size_t wide) { return kf_rows_overlap(q_out, (size_t)ldqo * 2, q_wide * 2, x, ldx * per_in, wide * per_in, M); };
    KF_REQUIRE(ctx, (q_out == q || !over(q, ldq, q_wide)) && !over(k, ldk, kv_wide) && !over(v, ldv, kv_wide), "the finished queries over a part of the panel");
    p.q = q, p.k = k, p.v = v, p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.out = q_out, p.ldo = ldqo, p.nq = n_head, p.nkv = kv->n_kv, p.hd = hd, p.M = M;
    p.qw = (const uint16_t*)qnorm_w, p.kw = (const uint16_t*)knorm_w, p.eps = eps;
    const int per = src_f32 ? 4 : 8;  // elements in 16 bytes
    const bool wide = whole_lanes(p) && (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)qnorm_w | (uintptr_t)knorm_w) & 15) == 0 && ldq % per == 0 &&
                      ldk % per == 0 && ldv % per == 0 && ldqo % 8 == 0;
    return src_f32 ? launch_rows<float, uint16_t>(ctx, p, wide) : launch_rows<uint16_t, uint16_t>(ctx, p, wide);
}
extern "C" int kf_paged_append(kf_ctx* ctx, const kf_paged_kv* kv, const kf_rotation* rot, void* q_out, int ldqo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv,
                               int src_f32, int M, int n_head, const void* qnorm_w, const void* knorm_w, float eps) {
    if (!ctx || !kv) return KF_ERR_BAD_ARG;
    RowsParams p = {};
    p.kc = (uint16_t*)kv->k_dev, p.vc = (uint16_t*)kv->v_dev, p.page_stride = (long long)kf_paged_stride(kv);
    return append(ctx, p, kv, rot, q_out, ldqo, q, ldq, k, ldk, v, ldv, src_f32, M, n_head, qnorm_w, knorm_w, eps);
}
extern "C" int kf_paged_append_q4(kf_ctx* ctx, const kf_paged_q4* kv, const kf_rotation* rot, void* q_out, int ldqo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv,
                                  int src_f32, int M, int n_head, const void* qnorm_w, const void* knorm_w, float eps) {
    if (!ctx || !kv) return KF_ERR_BAD_ARG;
    RowsParams p = {};
    p.pool = (uint8_t*)kv->pool_dev, p.page_stride = (long long)kf_paged_q4_stride(kv);
    return append(ctx, p, kv, rot, q_out, ldqo, q, ldq, k, ldk, v, ldv, src_f32, M, n_head, qnorm_w, knorm_w, eps);
}

static int rope_args(kf_ctx* ctx, const kf_rotation* rot, const void* out, int ldo, const void* x, int ldx, int f32, int M, int n_head, int hd, RowsParams* p) {
    if (!rot || !out || !x || !rot->pos_dev) return KF_ERR_BAD_ARG;
    KF_REQUIRE(ctx, hd >= 2 && hd <= 256 && n_head >= 1 && M >= 0 && (f32 == 0 || f32 == 1), "head_dim 2 .. 256, f32 0 or 1");
    const int rc = rotation(ctx, rot, hd, M, p);
    if (rc) return rc;
    KF_REQUIRE(ctx, (long long)n_head * hd <= ldx && (long long)n_head * hd <= ldo, "rows as long as their heads");
    KF_REQUIRE(ctx, out != x || ldo == ldx, "in place: rows where they were");
    return KF_OK;
}
extern "C" int kf_rope_axes(kf_ctx* ctx, const kf_rotation* rot, void* out, int ldo, const void* x, int ldx, int f32, int M, int n_head, int hd) {
    if (!ctx) return KF_ERR_BAD_ARG;
    RowsParams p = {};
    const int rc = rope_args(ctx, rot, out, ldo, x, ldx, f32, M, n_head, hd, &p);
    if (rc) return rc;
    if (M == 0) return KF_OK;
    const size_t size = f32 ? 4 : 2, wide_bytes = (size_t)n_head * hd * size;
    KF_REQUIRE(ctx, out == x || !kf_rows_overlap(out, ldo * size, wide_bytes, x, ldx * size, wide_bytes, M), "the result over a part of the panel");
    p.q = p.k = p.v = x, p.ldq = ldx, p.out = out, p.ldo = ldo, p.nq = n_head, p.hd = hd, p.M = M;
    const int per = f32 ? 4 : 8;
    const bool wide = whole_lanes(p) && (((uintptr_t)x | (uintptr_t)out) & 15) == 0 && ldx % per == 0 && ldo % per == 0;
    return f32 ? launch_rows<float, float>(ctx, p, wide) : launch_rows<uint16_t, uint16_t>(ctx, p, wide);
}
// The checks for tests on a host without a device
extern "C" int kf_paged_append_args(const kf_paged_kv* kv, const kf_rotation* rot, const void* q_out, int ldqo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv,
                                    int src_f32, int M, int n_head) {
    RowsParams p = {};
    return append_args(nullptr, kv, rot, q_out, ldqo, q, ldq, k, ldk, v, ldv, src_f32, M, n_head, &p);
}
extern "C" int kf_paged_append_q4_args(const kf_paged_q4* kv, const kf_rotation* rot, const void* q_out, int ldqo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv,
                                       int src_f32, int M, int n_head) {
    RowsParams p = {};
    return append_args(nullptr, kv, rot, q_out, ldqo, q, ldq, k, ldk, v, ldv, src_f32, M, n_head, &p);
}
extern "C" int kf_rope_axes_args(const kf_rotation* rot, const void* out, int ldo, const void* x, int ldx, int f32, int M, int n_head, int hd) {
    RowsParams p = {};
    return rope_args(nullptr, rot, out, ldo, x, ldx, f32, M, n_head, hd, &p);
}
