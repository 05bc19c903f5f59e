// kf_paged.cuh -- a step over a cache in pages, as the kernels see it (paged_append.cu, attn_paged.cu, attn_paged_tc.cu).
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
// whether M rows of a_wide bytes from a on, a_pitch bytes apart, and M rows of b_wide bytes from b on have a byte in common (paged_append.cu)
extern "C" int kf_rows_overlap(const void* a, size_t a_pitch, size_t a_wide, const void* b, size_t b_pitch, size_t b_wide, int M);
int kf_paged_check(kf_ctx* ctx, const kf_paged_kv* kv, int M, KfPaged* out);  // paged_append.cu: arguments that all of them share
static inline size_t kf_paged_stride(const kf_paged_kv* kv) { return kv->page_stride ? kv->page_stride : (size_t)kv->page_size * kv->n_kv * kv->head_dim; }

// With l bits in page - 1: page_mul = ceil(2^(31 + l) / page) exceeds the quotient by less than page, so p * page_mul / 2^(31 + l) exceeds p / page by less than p / 2^(31 + l) < 1 / page
static inline void kf_paged_divisor(KfPaged* pg) {
    int l = 0;
    while ((1ll << l) < pg->page) l++;  // up to 31
    pg->page_mul = (uint32_t)(((1ull << (31 + l)) + pg->page - 1) / pg->page), pg->page_shift = l - 1;
}
#ifdef __CUDACC__
// the pointers for use behind kf_grid_dependency_wait()
__device__ __forceinline__ KfPaged behind_wait(KfPaged p) {
    p.table = behind_wait(p.table), p.q_start = behind_wait(p.q_start), p.len = behind_wait(p.len);
    return p;
}
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
#endif
