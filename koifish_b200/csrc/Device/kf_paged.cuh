// kf_paged.cuh -- a step over a cache in pages, as the kernels see it (paged_append.cu, attn_paged.cu, attn_paged_tc.cu).
#pragma once
#include "kf_common.cuh"

struct KfPaged {  // kernel parameter
    const int32_t *table, *q_start, *len;
    int table_cols, n_seq, n_pages, page, cap /* positions a table holds */, M /* rows of the panel */;
};
// attn_paged_tc.cu: sequences with more than min_rows rows on tcgen05
int kf_attn_paged_tc(kf_ctx* ctx, const kf_paged_kv* kv, const KfPaged& pg, void* out, long long ldo, const void* q, long long ldq, int n_head, float scale, int window, int min_rows);
int kf_paged_check(kf_ctx* ctx, const kf_paged_kv* kv, int M, KfPaged* out);  // paged_append.cu: arguments that all of them share
static inline size_t kf_paged_stride(const kf_paged_kv* kv) { return kv->page_stride ? kv->page_stride : (size_t)kv->page_size * kv->n_kv * kv->head_dim; }

#ifdef __CUDACC__
// the pointers for use behind kf_grid_dependency_wait()
__device__ __forceinline__ KfPaged behind_wait(KfPaged p) {
    p.table = behind_wait(p.table), p.q_start = behind_wait(p.q_start), p.len = behind_wait(p.len);
    return p;
}
// page of position p >= 0 of sequence s, -1: not there
__device__ __forceinline__ int paged_page(const KfPaged& pg, int s, int p) {
    if (p >= pg.cap) return -1;
    const int e = pg.table[(size_t)s * pg.table_cols + p / pg.page];
    return e >= 0 && e < pg.n_pages ? e : -1;
}
// rows [q0, q0 + n) of sequence s in the panel, and its positions
__device__ __forceinline__ void paged_seq(const KfPaged& pg, int s, int& q0, int& n, int& len) {
    q0  = min(max(pg.q_start[s], 0), pg.M);
    n   = min(max(pg.q_start[s + 1], q0), pg.M) - q0;
    len = max(pg.len[s], 0);
}
#endif
