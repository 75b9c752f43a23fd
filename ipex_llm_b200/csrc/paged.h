// paged.h -- what the kernels of the paged cache share (paged_cache.cu, paged_attention.cu, paged_prompt.cu).
// A cache is [pages][page_size][kv heads][D] with D contiguous and any strides; token p of request r lies in page table[r][p / page_size],
// row p % page_size.  Packed prompts are the same without pages: token p of request r is row cu[r] + p.
#pragma once
#include "lowbit_common.cuh"
#include "lowbit_internal.h"

namespace lowbit {

constexpr int CACHE_E5M2 = QT_FP8_E5M2;       // a cache's dtype: DT_F16, DT_BF16 (that of the queries) or this

struct PagedAttnArgs {
    const void* q; int64_t q_st, q_sh;                       // strides in elements: token, head
    const void *k, *v; int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;       // ... page, row, head
    const int32_t* table; int64_t table_stride; int width;   // [R][width]; NULL: packed prompts
    int n_pages, page_size;
    const int32_t *seq_lens, *cu;                            // [R] keys a request holds, its new tokens included (NULL: as many as it has queries); [R + 1]
    int R; int64_t T;
    void* out; int64_t o_st, o_sh;
    int Hq, Hkv, D, dtype, cache_dtype, causal;
    float scale_log2e;
    float* part; Waits waits;
};

// a request's tokens, whatever the lists on the device say: nothing outside q and the table is ever addressed
struct PagedReq { int64_t q0; int n, len; };
__device__ __forceinline__ PagedReq paged_req(const PagedAttnArgs& A, int r) {
    PagedReq q;
    const int64_t a = A.cu[r], b = A.cu[r + 1];
    q.q0 = a < 0 ? 0 : a > A.T ? A.T : a;
    const int64_t e = b < q.q0 ? q.q0 : b > A.T ? A.T : b;
    q.n = (int)(e - q.q0);
    if (A.table) {
        const int64_t held = A.seq_lens[r], most = (int64_t)A.width * A.page_size;
        q.len = (int)(held < 0 ? 0 : held > most ? most : held);
    } else q.len = q.n;
    return q;
}

}  // namespace lowbit
