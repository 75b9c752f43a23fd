// paged_attention.cu -- attention of the new tokens of many requests over a paged cache, and of packed prompts over themselves:
//   out[t][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - max),   j = the keys that token t of its request sees.
// Token i of a request's n new ones, which holds len, sees keys 0 .. len - n + i; a token that sees none gives zeros.
#include <type_traits>
#include "paged.h"

using namespace lowbit;

namespace lowbit {
namespace {

// a warp per (token, query head): one pass over the keys with the running maximum and sum
template <typename T, bool E5M2>
__global__ void __launch_bounds__(128) paged_attention_simple_kernel(const PagedAttnArgs A) {
    const int lane = threadIdx.x & 31;
    const int64_t w = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t t = w / A.Hq;
    const int h = (int)(w % A.Hq), hk = h / (A.Hq / A.Hkv);
    if (t >= A.T) return;
    int r = 0;
    PagedReq q;
    for (;; r++) {
        if (r == A.R) return;                                   // behind the last request
        q = paged_req(A, r);
        if (t >= q.q0 && t < q.q0 + q.n) break;
    }
    auto load = [&](const void* p, int64_t i) -> float {
        if (sizeof(T) == 2 && E5M2) return decode_e5m2(((const uint8_t*)p)[i]);
        if constexpr (std::is_same<T, __half>::value) return __half2float(((const __half*)p)[i]);
        else return __bfloat162float(((const __nv_bfloat16*)p)[i]);
    };
    float x[8], o[8], m = -INFINITY, sum = 0.0f;
    const int E = (A.D + 31) / 32;
    for (int e = 0; e < 8; e++) {
        const int d = lane + 32 * e;
        x[e] = 0.0f; o[e] = 0.0f;
        if (d < A.D) {
            const int64_t at = t * A.q_st + h * A.q_sh + d;
            if constexpr (std::is_same<T, __half>::value) x[e] = __half2float(((const __half*)A.q)[at]);
            else x[e] = __bfloat162float(((const __nv_bfloat16*)A.q)[at]);
        }
    }
    const int64_t i = t - q.q0, see = A.causal ? min((int64_t)q.len, q.len - q.n + i + 1) : q.len;
    for (int64_t j = 0; j < see; j++) {
        int64_t kb, vb;
        bool bad = false;
        if (A.table) {
            const int pg = A.table[r * A.table_stride + j / A.page_size], in = (int)(j % A.page_size);
            bad = pg < 0 || pg >= A.n_pages;
            kb = bad ? 0 : pg * A.k_sp + in * A.k_ss + hk * A.k_sh;
            vb = bad ? 0 : pg * A.v_sp + in * A.v_ss + hk * A.v_sh;
        } else {
            kb = (q.q0 + j) * A.k_ss + hk * A.k_sh;
            vb = (q.q0 + j) * A.v_ss + hk * A.v_sh;
        }
        float s = 0.0f;
        for (int e = 0; e < E; e++) { const int d = lane + 32 * e; if (d < A.D) s = fmaf(x[e], load(A.k, kb + d), s); }
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= A.scale_log2e;
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : exp2f(m - mn), p = s == -INFINITY ? 0.0f : exp2f(s - mn);
        sum = fmaf(sum, c, p);
        for (int e = 0; e < E; e++) { const int d = lane + 32 * e; if (d < A.D) o[e] = fmaf(p, bad ? NAN : load(A.v, vb + d), o[e] * c); }
        m = mn;
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    for (int e = 0; e < E; e++) {
        const int d = lane + 32 * e;
        if (d >= A.D) break;
        const int64_t at = t * A.o_st + h * A.o_sh + d;
        if constexpr (std::is_same<T, __half>::value) ((__half*)A.out)[at] = __float2half_rn(o[e] * inv);
        else ((__nv_bfloat16*)A.out)[at] = __float2bfloat16_rn(o[e] * inv);
    }
}

bool aligned(const void* p, int64_t a, int64_t b, int64_t c, int unit) { return !((uintptr_t)p & 15) && !((a | b | c) & (unit - 1)); }

// what both entry points refuse
int check(const PagedAttnArgs& A, const char* name) {
    if (!A.q || !A.k || !A.v || !A.cu || !A.out || A.R <= 0 || A.T < 0 || A.Hq <= 0 || A.Hkv <= 0 || A.Hq % A.Hkv || A.D <= 0 || A.D % 16 || A.D > 256 ||
        (A.dtype != DT_F16 && A.dtype != DT_BF16) || (A.cache_dtype != A.dtype && !(A.table && A.cache_dtype == CACHE_E5M2)) || !(A.scale_log2e > 0.0f) ||
        A.T * A.Hq > 0x7fffffffll) {
        set_error(LB_ERR_ARG, "%s: bad argument (R %d, T %lld, Hq %d, Hkv %d, D %d, dtype %d, cache dtype %d)", name, A.R, (long long)A.T, A.Hq, A.Hkv, A.D, A.dtype,
                  A.cache_dtype);
        return LB_ERR_ARG;
    }
    const int unit = A.cache_dtype == CACHE_E5M2 ? 16 : 8;
    if (!aligned(A.q, A.q_st, A.q_sh, 0, 8) || !aligned(A.out, A.o_st, A.o_sh, 0, 8) || !aligned(A.k, A.k_sp, A.k_ss, A.k_sh, unit) ||
        !aligned(A.v, A.v_sp, A.v_ss, A.v_sh, unit)) {
        set_error(LB_ERR_ARG, "%s: queries, keys, values and output must be 16-byte aligned (pointers and strides)", name);
        return LB_ERR_ARG;
    }
    return LB_OK;
}

int launch(const PagedAttnArgs& A, cudaStream_t st) {
    const int64_t warps = A.T * A.Hq;
    const dim3 grid((unsigned)((warps + 3) / 4));
    if (A.dtype == DT_F16) {
        if (A.cache_dtype == CACHE_E5M2) paged_attention_simple_kernel<__half, true><<<grid, 128, 0, st>>>(A);
        else paged_attention_simple_kernel<__half, false><<<grid, 128, 0, st>>>(A);
    } else {
        if (A.cache_dtype == CACHE_E5M2) paged_attention_simple_kernel<__nv_bfloat16, true><<<grid, 128, 0, st>>>(A);
        else paged_attention_simple_kernel<__nv_bfloat16, false><<<grid, 128, 0, st>>>(A);
    }
    note_launch();
    return check_launch();
}

}  // namespace
}  // namespace lowbit

extern "C" size_t lowbit_sdp_paged_workspace_size(int64_t T, int R, int Hq, int Hkv, int D, int64_t max_query) {
    (void)T; (void)R; (void)Hq; (void)Hkv; (void)D; (void)max_query;
    return 0;
}

extern "C" int lowbit_sdp_paged_cuda(const void* d_q, int q_dtype, const int64_t* q_strides, int64_t T, const void* d_k, const int64_t* k_strides,
                                     const void* d_v, const int64_t* v_strides, int cache_dtype, int n_pages, int page_size, const int32_t* d_table,
                                     int64_t table_stride, int width, const int32_t* d_seq_lens, const int32_t* d_cu_seqlens, int R, int Hq, int Hkv,
                                     int D, float scale, int64_t max_query, void* d_out, const int64_t* out_strides, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    reset_launch_count();
    (void)max_query; (void)workspace; (void)workspace_bytes;
    if (!d_table || !d_seq_lens || !q_strides || !k_strides || !v_strides || !out_strides || n_pages <= 0 || page_size <= 0 || width <= 0 || table_stride < width ||
        (int64_t)width * page_size > 0x7fffffffll) {
        set_error(LB_ERR_ARG, "lowbit_sdp_paged_cuda: bad argument (pages %d, page_size %d, width %d)", n_pages, page_size, width);
        return LB_ERR_ARG;
    }
    PagedAttnArgs A = {};
    A.q = d_q; A.q_st = q_strides[0]; A.q_sh = q_strides[1];
    A.k = d_k; A.k_sp = k_strides[0]; A.k_ss = k_strides[1]; A.k_sh = k_strides[2];
    A.v = d_v; A.v_sp = v_strides[0]; A.v_ss = v_strides[1]; A.v_sh = v_strides[2];
    A.table = d_table; A.table_stride = table_stride; A.width = width; A.n_pages = n_pages; A.page_size = page_size;
    A.seq_lens = d_seq_lens; A.cu = d_cu_seqlens; A.R = R; A.T = T;
    A.out = d_out; A.o_st = out_strides[0]; A.o_sh = out_strides[1];
    A.Hq = Hq; A.Hkv = Hkv; A.D = D; A.dtype = q_dtype; A.cache_dtype = cache_dtype; A.causal = 1;
    A.scale_log2e = scale * 1.4426950408889634f;
    if (const int rc = check(A, "lowbit_sdp_paged_cuda")) return rc;
    if (T == 0) return LB_OK;
    return launch(A, (cudaStream_t)stream);
}

extern "C" size_t lowbit_sdp_packed_workspace_size(int64_t T, int R, int Hq, int Hkv, int D, int64_t max_seqlen) {
    (void)T; (void)R; (void)Hq; (void)Hkv; (void)D; (void)max_seqlen;
    return 0;
}

extern "C" int lowbit_sdp_packed_cuda(const void* d_q, int dtype, const int64_t* q_strides, int64_t T, const void* d_k, const int64_t* k_strides,
                                      const void* d_v, const int64_t* v_strides, const int32_t* d_cu_seqlens, int R, int Hq, int Hkv, int D, float scale,
                                      int causal, int64_t max_seqlen, void* d_out, const int64_t* out_strides, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    reset_launch_count();
    (void)max_seqlen; (void)workspace; (void)workspace_bytes;
    if (!q_strides || !k_strides || !v_strides || !out_strides || T > 0x7fffffffll) {
        set_error(LB_ERR_ARG, "lowbit_sdp_packed_cuda: bad argument (T %lld)", (long long)T);
        return LB_ERR_ARG;
    }
    PagedAttnArgs A = {};
    A.q = d_q; A.q_st = q_strides[0]; A.q_sh = q_strides[1];
    A.k = d_k; A.k_ss = k_strides[0]; A.k_sh = k_strides[1];
    A.v = d_v; A.v_ss = v_strides[0]; A.v_sh = v_strides[1];
    A.page_size = 1;
    A.cu = d_cu_seqlens; A.R = R; A.T = T;
    A.out = d_out; A.o_st = out_strides[0]; A.o_sh = out_strides[1];
    A.Hq = Hq; A.Hkv = Hkv; A.D = D; A.dtype = dtype; A.cache_dtype = dtype; A.causal = causal ? 1 : 0;
    A.scale_log2e = scale * 1.4426950408889634f;
    if (const int rc = check(A, "lowbit_sdp_packed_cuda")) return rc;
    if (T == 0) return LB_OK;
    return launch(A, (cudaStream_t)stream);
}
