// kf_paged.cuh -- a step over a cache in pages, as the kernels see it (paged_append.cu, attn_paged.cu, attn_paged_tc.cu, and for 4 bits paged_read_q4.cu, attn_paged_q4.cu).
#pragma once
#include "kf_common.cuh"

struct KfPaged {  // kernel parameter
    const int32_t *table, *q_start, *len;
    int table_cols, n_seq, n_pages, page, cap /* positions a table holds */, M /* rows of the panel */;
    uint32_t page_mul;  // p / page = umulhi(p, page_mul) >> page_shift for 0 <= p < 2^31
    int page_shift;
};
// attn_paged_tc.cu: on tcgen05
int kf_attn_paged_tc(kf_ctx* ctx, const kf_paged_kv* kv, const KfPaged& pg, void* out, long long ldo, const void* q, long long ldq, int n_head, float scale, int window);
// attn_paged_q4_tc.cu: the same over the 4-bit cache
int kf_attn_paged_q4_tc(kf_ctx* ctx, const kf_paged_q4* kv, const KfPaged& pg, void* out, long long ldo, const void* q, long long ldq, int n_head, float scale, int window, int first);
// whether M rows of a_wide bytes from a on, a_pitch bytes apart, and M rows of b_wide bytes from b on have a byte in common (paged_append.cu)
extern "C" int kf_rows_overlap(const void* a, size_t a_pitch, size_t a_wide, const void* b, size_t b_pitch, size_t b_wide, int M);
int kf_paged_check(kf_ctx* ctx, const kf_paged_kv* kv, int M, KfPaged* out);  // paged_append.cu: arguments that all of them share
int kf_paged_q4_check(kf_ctx* ctx, const kf_paged_q4* kv, int M, KfPaged* out);
static inline size_t kf_paged_stride(const kf_paged_kv* kv) { return kv->page_stride ? kv->page_stride : (size_t)kv->page_size * kv->n_kv * kv->head_dim; }

// With l bits in page - 1: page_mul = ceil(2^(31 + l) / page) exceeds the quotient by less than page, so p * page_mul / 2^(31 + l) exceeds p / page by less than p / 2^(31 + l) < 1 / page
static inline void kf_paged_divisor(KfPaged* pg) {
    int l = 0;
    while ((1ll << l) < pg->page) l++;  // up to 31
    pg->page_mul = (uint32_t)(((1ull << (31 + l)) + pg->page - 1) / pg->page), pg->page_shift = l - 1;
}
// The 4-bit cache (kf_device.h): bytes of a unit, which is 8 positions of one head, and where its parts lie.  Codes are stored in the order in which the attention's matrix
// instructions take them: lane (g, t) of a warp, g = lane / 4, t = lane % 4, finds its operand of 8 positions as 16 (head_dim 64: 8) bytes at lane * 16 (* 8).
struct Q4Unit {
    int groups, codes, table, bytes;  // groups of 32 entries in a row; bytes of 8 rows of codes, of 8 x groups numbers, of the unit
    __host__ __device__ constexpr Q4Unit(int hd) : groups(hd / 32), codes(4 * hd), table(hd / 2), bytes(10 * hd) {}
    __host__ __device__ constexpr int k_step() const { return codes; }              // [8][groups]
    __host__ __device__ constexpr int k_zero() const { return codes + table; }      // [8][groups]
    __host__ __device__ constexpr int v_code() const { return codes + 2 * table; }
    __host__ __device__ constexpr int v_step() const { return 2 * codes + 2 * table; }  // [8][groups]
    __host__ __device__ constexpr int v_zero() const { return 2 * codes + 3 * table; }  // [groups][8]
};
static inline size_t kf_paged_q4_stride(const kf_paged_q4* kv) { return kv->page_stride ? kv->page_stride : kf_paged_q4_page_bytes(kv->page_size, kv->n_kv, kv->head_dim); }
#ifdef __CUDACC__
// the pointers for use behind kf_grid_dependency_wait()
__device__ __forceinline__ KfPaged behind_wait(KfPaged p) {
    p.table = behind_wait(p.table), p.q_start = behind_wait(p.q_start), p.len = behind_wait(p.len);
    return p;
}
// N words, aligned to as many (up to four)
template <int N>
__device__ __forceinline__ void words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else w[0] = *reinterpret_cast<const uint32_t*>(p);
}
__device__ __forceinline__ float half_of(uint32_t w, int h) { return h ? bf16hi(w) : bf16lo(w); }
// page of position p >= 0 of sequence s, -1: not there; row: of the position in its page
__device__ __forceinline__ int paged_page(const KfPaged& pg, int s, int p, int& row) {
    const int c = (int)(__umulhi((uint32_t)p, pg.page_mul) >> pg.page_shift);
    row         = p - c * pg.page;
    if (p >= pg.cap) return -1;
    const int e = pg.table[(size_t)s * pg.table_cols + c];
    return e >= 0 && e < pg.n_pages ? e : -1;
}
// rows [q0, q0 + n) of sequence s in the panel, and its positions
__device__ __forceinline__ void paged_seq(const KfPaged& pg, int s, int& q0, int& n, int& len) {
    q0  = min(max(pg.q_start[s], 0), pg.M);
    n   = min(max(pg.q_start[s + 1], q0), pg.M) - q0;
    len = max(pg.len[s], 0);
}
// the sequence that row m of the panel belongs to, -1: none.  One warp, 32 candidates at a time
__device__ __forceinline__ int paged_find_seq(const KfPaged& pg, int m, int lane) {
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
#endif
