// paged_append.cu -- a step's keys and values into the pages of their sequences with the norm and the rotation of q and k on the way (kf_paged_append), and the
// rotation alone (kf_rope_axes).
//
//   y = x * rsqrt(mean(x^2) + eps) * w (per head; optional),  pair j: (a, b) -> amp * (a cos t - b sin t, b cos t + a sin t),  t = pos[axis[j]][row] * inv_freq[j]
//
// Every element is read once and written once, so HBM bounds the large calls and latency the small ones.  A block takes one token, whose rotation is worked out once for
// all its heads: t / pi in 64 bits, reduced to [-1, 1] there (a far position turns many times; its remainder in 32 bits would be off by more than the result's rounding),
// then sine and cosine in 32 bits.  A head's row is spread over 8, 16 or 32 lanes with eight entries each; the lane that holds a pair's other half is found by a shuffle,
// and a thread keeps its eight pairs' sines and cosines in registers for all the rows it takes.  The first rows are asked for before the position is known: finding the
// sequence of a token, its page and its position are three dependent reads.  Few tokens are spread over blocks by heads.
#include <algorithm>

#include "kf_paged.cuh"

namespace {
constexpr int kThreads = 256, kRows = 4;  // rows of a lane in flight

struct RowsParams {
    const void *q, *k, *v;
    long long ldq, ldk, ldv, ldo;
    void* out;
    int nq, nkv /* 0: no cache */, hd, M, rows_per_block;
    const double* freq;
    const int32_t *axis, *pos;
    long long pos_stride;
    int rot, layout, n_axes;
    float amp;
    const uint16_t *qw, *kw;
    float eps;
    uint16_t *kc, *vc;
    long long page_stride;
    KfPaged pg;
};

// the sequence that row m of the panel belongs to, -1: none.  One warp, 32 candidates at a time
__device__ __forceinline__ int find_seq(const KfPaged& pg, int m, int lane) {
    int lo = 0, size = pg.n_seq + 1;  // the number of starts at or before m is looked for
    while (true) {
        const int step = (size + 31) / 32, at = lo + lane * step;
        const int c = __popc(__ballot_sync(0xffffffffu, at < lo + size && pg.q_start[min(at, pg.n_seq)] <= m));
        if (c == 0) return -1;
        const int first = lo + (c - 1) * step;
        if (step == 1) return first < pg.n_seq ? first : -1;
        size = min(step, lo + size - first), lo = first;
    }
}

__device__ __forceinline__ float load1(const uint16_t* p) { return bf16_bits_to_f32(*p); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ void store1(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
// eight entries as they lie in memory
template <typename X>
struct Raw;
template <>
struct Raw<uint16_t> {
    uint4 a;
    __device__ __forceinline__ void load(const uint16_t* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        f[0] = bf16lo(a.x), f[1] = bf16hi(a.x), f[2] = bf16lo(a.y), f[3] = bf16hi(a.y), f[4] = bf16lo(a.z), f[5] = bf16hi(a.z), f[6] = bf16lo(a.w), f[7] = bf16hi(a.w);
    }
};
template <>
struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ void get(float (&f)[8]) const { f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w; }
};
__device__ __forceinline__ void store8(uint16_t* p, const float (&f)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]), reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// LPR: lanes to a row, eight entries each; 0: rows at any element, or pairs that do not fall on whole lanes -- a warp per row, an entry or a pair per lane
template <typename X, typename Y, int LPR>
__global__ void __launch_bounds__(kThreads) kf_rows_kernel(const __grid_constant__ RowsParams p) {
    constexpr int kL = LPR ? LPR : 32, kGroups = kThreads / kL;
    __shared__ float2 s_cs[128];
    const int tid = threadIdx.x, lane = tid & 31, grp = tid / kL, v = tid % kL, m = blockIdx.x;
    kf_grid_launch_dependents();
    kf_grid_dependency_wait();  // the panel, positions, lengths and tables come from the kernels before us
    const X *q = behind_wait((const X*)p.q) + m * p.ldq, *k = behind_wait((const X*)p.k) + m * p.ldk, *vv = behind_wait((const X*)p.v) + m * p.ldv;
    const KfPaged pg = behind_wait(p.pg);
    const int all = p.nq + 2 * p.nkv, r0 = blockIdx.y * p.rows_per_block, r1 = min(all, r0 + p.rows_per_block);
    auto src = [&](int r) -> const X* { return r < p.nq ? q + (long long)r * p.hd : r < p.nq + p.nkv ? k + (long long)(r - p.nq) * p.hd : vv + (long long)(r - p.nq - p.nkv) * p.hd; };
    Raw<X> raw[kRows];
    auto fetch = [&](int rb) {
#pragma unroll
        for (int u = 0; u < kRows; u++)
            if (rb + u * kGroups < r1 && v * 8 < p.hd) raw[u].load(src(rb + u * kGroups) + v * 8);
    };
    if (LPR) fetch(r0 + grp);

    int at = 0;            // position in the sequence
    long long row = -1;    // the token's row in the pools
    if (p.nkv) {
        const int s = find_seq(pg, m, lane);
        if (s < 0) return;  // padding
        int q0, n, len;
        paged_seq(pg, s, q0, n, len);
        at = len - n + (m - q0);
        int in         = 0;
        const int page = at >= 0 ? paged_page(pg, s, at, in) : -1;
        if (page >= 0) row = page * p.page_stride + (long long)in * p.nkv * p.hd;
    }
    for (int j = tid; j < p.rot / 2; j += kThreads) {
        const int ax = p.axis ? p.axis[j] : 0;
        float sn = 0.f, cs = 1.f;
        if (ax >= 0 && ax < p.n_axes) {
            const double t = (double)(p.pos ? p.pos[ax * p.pos_stride + m] : at) * p.freq[j] * 0.31830988618379067154;
            sincospif((float)(t - 2.0 * rint(0.5 * t)), &sn, &cs);
            cs *= p.amp, sn *= p.amp;
        }
        s_cs[j] = make_float2(cs, sn);
    }
    __syncthreads();
    const int half = p.rot / 2;
    Y* out         = (Y*)p.out + m * p.ldo;
    if constexpr (LPR != 0) {
        // this lane's pairs: entry i turns with cs[i] (layout 1), entries 2i and 2i + 1 with cs[i] (layout 0)
        float2 cs[8];
        const bool lower = 8 * v < half, turns = 8 * v < p.rot;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int j = p.layout ? (lower ? 8 * v + i : 8 * v - half + i) : 4 * v + i;
            cs[i]       = turns && j < half && (p.layout || i < 4) ? s_cs[j] : make_float2(1.f, 0.f);
        }
        const int mate = (lane & ~(LPR - 1)) | (p.layout && turns ? (lower ? v + half / 8 : v - half / 8) : v);
        uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
        if (p.qw && v * 8 < p.hd) wq = *reinterpret_cast<const uint4*>(p.qw + v * 8);
        if (p.kw && v * 8 < p.hd) wk = *reinterpret_cast<const uint4*>(p.kw + v * 8);
        for (int rb = r0 + grp; rb < r1 + grp; rb += kRows * kGroups) {  // the same number of turns for all lanes of a warp
            if (rb != r0 + grp) fetch(rb);
#pragma unroll
            for (int u = 0; u < kRows; u++) {
                const int r = rb + u * kGroups;
                if (__all_sync(0xffffffffu, r >= r1)) break;
                const bool is_q = r < p.nq, is_v = r >= p.nq + p.nkv, live = r < r1 && v * 8 < p.hd;
                float f[8];
                raw[u].get(f);
                const uint16_t* w = is_q ? p.qw : p.kw;
                if (p.qw || p.kw) {
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) ss = live ? fmaf(f[i], f[i], ss) : 0.f;
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    if (w && !is_v) {
                        const float inv = rsqrtf(ss / (float)p.hd + p.eps);
                        Raw<uint16_t> ww;
                        ww.a = is_q ? wq : wk;
                        float g[8];
                        ww.get(g);
#pragma unroll
                        for (int i = 0; i < 8; i++) f[i] = f[i] * inv * g[i];
                    }
                }
                float y[8];
                if (p.layout) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float other = __shfl_sync(0xffffffffu, f[i], mate);
                        y[i]              = !turns || is_v ? f[i] : lower ? f[i] * cs[i].x - other * cs[i].y : f[i] * cs[i].x + other * cs[i].y;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool t = !is_v && 8 * v + 2 * i < p.rot;
                        y[2 * i]     = t ? f[2 * i] * cs[i].x - f[2 * i + 1] * cs[i].y : f[2 * i];
                        y[2 * i + 1] = t ? f[2 * i + 1] * cs[i].x + f[2 * i] * cs[i].y : f[2 * i + 1];
                    }
                }
                if (!live) continue;
                if (is_q) store8(out + (long long)r * p.hd + v * 8, y);
                else if (row >= 0) store8((is_v ? p.vc + row + (long long)(r - p.nq - p.nkv) * p.hd : p.kc + row + (long long)(r - p.nq) * p.hd) + v * 8, y);
            }
        }
    } else {
        for (int r = r0 + grp; r < r1; r += kGroups) {  // a warp per row
            const bool is_q = r < p.nq, is_v = r >= p.nq + p.nkv;
            const X* x = src(r);
            if (!is_q && row < 0) continue;
            const uint16_t* w = is_v ? nullptr : is_q ? p.qw : p.kw;
            float inv = 1.f;
            if (w) {
                float ss = 0.f;
                for (int i = lane; i < p.hd; i += 32) ss = fmaf(load1(x + i), load1(x + i), ss);
                inv = rsqrtf(warp_sum(ss) / (float)p.hd + p.eps);
            }
            auto in  = [&](int i) { return w ? load1(x + i) * inv * bf16_bits_to_f32(w[i]) : load1(x + i); };
            uint16_t* c = is_q ? nullptr : is_v ? p.vc + row + (long long)(r - p.nq - p.nkv) * p.hd : p.kc + row + (long long)(r - p.nq) * p.hd;
            auto put = [&](int i, float y) {
                if (is_q) store1(out + (long long)r * p.hd + i, y);
                else store1(c + i, y);
            };
            const int pairs = is_v ? 0 : half;
            for (int j = lane; j < pairs; j += 32) {
                const int ia = p.layout ? j : 2 * j, ib = p.layout ? j + half : 2 * j + 1;
                const float a = in(ia), b = in(ib);
                const float2 t = s_cs[j];
                put(ia, a * t.x - b * t.y), put(ib, b * t.x + a * t.y);
            }
            for (int i = 2 * pairs + lane; i < p.hd; i += 32) put(i, in(i));
        }
    }
}

template <typename X, typename Y>
int launch_rows(kf_ctx* ctx, RowsParams& p, bool wide) {
    const int lpr = !wide ? 0 : p.hd <= 64 ? 8 : p.hd <= 128 ? 16 : 32, groups = kThreads / (lpr ? lpr : 32), all = p.nq + 2 * p.nkv;
    // few tokens: their heads over several blocks, up to four blocks per SM
    const int parts = std::max(1, std::min((all + groups - 1) / groups, 4 * ctx->sm_count / p.M));
    p.rows_per_block = ((all + parts - 1) / parts + groups - 1) / groups * groups;
    const dim3 grid(p.M, (all + p.rows_per_block - 1) / p.rows_per_block);
    auto kern = lpr == 0 ? kf_rows_kernel<X, Y, 0> : lpr == 8 ? kf_rows_kernel<X, Y, 8> : lpr == 16 ? kf_rows_kernel<X, Y, 16> : kf_rows_kernel<X, Y, 32>;
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
bool whole_lanes(const RowsParams& p) { return p.hd % 8 == 0 && (p.layout == 0 || p.rot % 16 == 0); }
}  // namespace

int kf_paged_check(kf_ctx* ctx, const kf_paged_kv* kv, int M, KfPaged* out) {
    KF_REQUIRE(ctx, kv->k_dev && kv->v_dev && kv->table_dev && kv->q_start_dev && kv->len_dev, "cache, table, starts and lengths");
    KF_REQUIRE(ctx, kv->head_dim == 64 || kv->head_dim == 128, "head_dim 64 or 128");
    KF_REQUIRE(ctx, kv->n_kv >= 1 && kv->n_kv <= 1024 && kv->n_pages >= 1 && kv->page_size >= 8 && kv->page_size % 8 == 0, "n_kv 1 .. 1024, page_size a multiple of 8");
    KF_REQUIRE(ctx, kv->table_cols >= 1 && (long long)kv->table_cols * kv->page_size <= 0x7fffffff - 256, "table_cols");
    KF_REQUIRE(ctx, kv->n_seq >= 1 && kv->n_seq <= 8192 && M >= 0, "n_seq 1 .. 8192");
    KF_REQUIRE(ctx, kv->page_stride == 0 || (kv->page_stride % 8 == 0 && kv->page_stride >= (size_t)kv->page_size * kv->n_kv * kv->head_dim), "page_stride: a multiple of 8, at least a page");
    KF_REQUIRE(ctx, (((uintptr_t)kv->k_dev | (uintptr_t)kv->v_dev) & 15) == 0, "pages at 16 bytes");
    *out = KfPaged{kv->table_dev, kv->q_start_dev, kv->len_dev, kv->table_cols, kv->n_seq, kv->n_pages, kv->page_size, kv->table_cols * kv->page_size, M, 0, 0};
    kf_paged_divisor(out);
    return KF_OK;
}

static int append_args(kf_ctx* ctx, const kf_paged_kv* kv, const kf_rotation* rot, const void* q_out, int ldqo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv,
                       int src_f32, int M, int n_head, RowsParams* p) {
    if (!kv || !q_out || !q || !k || !v) return KF_ERR_BAD_ARG;
    int rc = kf_paged_check(ctx, kv, M, &p->pg);
    if (!rc) rc = rotation(ctx, rot, kv->head_dim, M, p);
    if (rc) return rc;
    const int hd = kv->head_dim;
    KF_REQUIRE(ctx, n_head >= 1 && (long long)n_head * hd <= ldq && (long long)n_head * hd <= ldqo && (long long)kv->n_kv * hd <= ldk && (long long)kv->n_kv * hd <= ldv,
               "rows as long as their heads");
    KF_REQUIRE(ctx, src_f32 == 0 || (src_f32 == 1 && q_out != q), "src_f32 0 or 1; float queries are not finished in place");
    KF_REQUIRE(ctx, q_out != q || ldqo == ldq, "in place: rows where they were");
    return KF_OK;
}
extern "C" int kf_paged_append(kf_ctx* ctx, const kf_paged_kv* kv, const kf_rotation* rot, void* q_out, int ldqo, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv,
                               int src_f32, int M, int n_head, const void* qnorm_w, const void* knorm_w, float eps) {
    if (!ctx) return KF_ERR_BAD_ARG;
    RowsParams p = {};
    const int rc = append_args(ctx, kv, rot, q_out, ldqo, q, ldq, k, ldk, v, ldv, src_f32, M, n_head, &p);
    if (rc) return rc;
    const int hd = kv->head_dim;
    if (M == 0) return KF_OK;
    p.q = q, p.k = k, p.v = v, p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.out = q_out, p.ldo = ldqo, p.nq = n_head, p.nkv = kv->n_kv, p.hd = hd, p.M = M;
    p.qw = (const uint16_t*)qnorm_w, p.kw = (const uint16_t*)knorm_w, p.eps = eps;
    p.kc = (uint16_t*)kv->k_dev, p.vc = (uint16_t*)kv->v_dev, p.page_stride = (long long)kf_paged_stride(kv);
    const int per = src_f32 ? 4 : 8;  // elements in 16 bytes
    const bool wide = whole_lanes(p) && (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)qnorm_w | (uintptr_t)knorm_w) & 15) == 0 && ldq % per == 0 &&
                      ldk % per == 0 && ldv % per == 0 && ldqo % 8 == 0;
    return src_f32 ? launch_rows<float, uint16_t>(ctx, p, wide) : launch_rows<uint16_t, uint16_t>(ctx, p, wide);
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
extern "C" int kf_rope_axes_args(const kf_rotation* rot, const void* out, int ldo, const void* x, int ldx, int f32, int M, int n_head, int hd) {
    RowsParams p = {};
    return rope_args(nullptr, rot, out, ldo, x, ldx, f32, M, n_head, hd, &p);
}
