// paged_cache.cu -- the bookkeeping of a paged key/value cache on the GPU and the write into it.
//
// lowbit_paged_step_cuda: from what every request holds (tokens in the cache) and brings (new tokens) the pages that it still needs, taken
// off a stack of free ones; its row of the block table; and for every new token its position and its slot (page * page_size + row).  With
//   need_r = ceil((held_r + new_r) / page_size) - ceil(held_r / page_size)      and      before_r = sum of need over the requests in front,
// request r's i-th new page is free[count - 1 - (before_r + i)], so a token's slot follows from two prefix sums and nobody waits for a
// neighbour's page.
#include "paged.h"

using namespace lowbit;

namespace lowbit {
namespace {

struct StepArgs {
    const int32_t *fresh, *held; int R;
    int32_t* table; int64_t table_stride; int width;
    const int32_t* pages; int n_pages; const int32_t* count; int32_t* left;
    int page_size; int64_t n_tokens;
    int32_t *cu, *seq_lens; int64_t *positions, *slots; int32_t* missing;
};

constexpr int STEP_THREADS = 1024;

__device__ __forceinline__ int pages_of(int64_t tokens, int page) { return (int)((tokens + page - 1) / page); }

// inclusive sums of two values over the block; `total` those of the whole block
__device__ __forceinline__ void block_scan2(int64_t& a, int& b, int64_t* wa, int* wb, int64_t& ta, int& tb) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, a, d);
        const int y = __shfl_up_sync(0xffffffffu, b, d);
        if (lane >= d) { a += x; b += y; }
    }
    __syncthreads();
    if (lane == 31) { wa[warp] = a; wb[warp] = b; }
    __syncthreads();
    int64_t pa = 0; int pb = 0;
    ta = 0; tb = 0;
    for (int w = 0; w < warps; w++) {
        if (w < warp) { pa += wa[w]; pb += wb[w]; }
        ta += wa[w]; tb += wb[w];
    }
    a += pa; b += pb;
}

// one block: the requests in rounds of a thread each; a request's tokens and pages by a warp
__global__ void __launch_bounds__(STEP_THREADS) paged_step_kernel(const StepArgs A) {
    __shared__ int64_t wa[32];
    __shared__ int wb[32];
    const int lane = threadIdx.x & 31;
    const int count = max(0, min(*A.count, A.n_pages));
    int64_t tokens = 0;
    int taken = 0, lost = 0;
    if (threadIdx.x == 0) A.cu[0] = 0;
    for (int r0 = 0; r0 < A.R; r0 += blockDim.x) {
        const int r = r0 + threadIdx.x;
        const int held = r < A.R ? max(A.held[r], 0) : 0, fresh = r < A.R ? max(A.fresh[r], 0) : 0;
        const int had = min(pages_of(held, A.page_size), A.width), all = pages_of((int64_t)held + fresh, A.page_size), want = min(all, A.width);
        int64_t tok = fresh, tt;
        int need = max(want - had, 0), nt;
        const int mine = need, over = r < A.R ? max(all - A.width, 0) : 0;
        block_scan2(tok, need, wa, wb, tt, nt);
        const int64_t tok0 = tokens + tok - fresh;
        const int page0 = taken + need - mine;
        if (r < A.R) {
            A.cu[r + 1] = (int32_t)(tok0 + fresh);
            A.seq_lens[r] = held + fresh;
        }
        lost += over;
        // the warp's requests one after the other
        for (int l = 0; l < 32; l++) {
            const int rr = r0 + (int)(threadIdx.x & ~31u) + l;
            if (rr >= A.R) break;
            const int h = __shfl_sync(0xffffffffu, held, l), f = __shfl_sync(0xffffffffu, fresh, l), hd = __shfl_sync(0xffffffffu, had, l), n = __shfl_sync(0xffffffffu, mine, l),
                      p0 = __shfl_sync(0xffffffffu, page0, l);
            const int64_t t0 = __shfl_sync(0xffffffffu, tok0, l);
            int32_t* row = A.table + rr * A.table_stride;
            auto page = [&](int i) { const int at = count - 1 - (p0 + i); return at >= 0 ? A.pages[at] : -1; };      // the i-th new one
            for (int i = lane; i < n; i += 32) row[hd + i] = page(i);
            for (int i = lane; i < f; i += 32) {
                if (t0 + i >= A.n_tokens) break;
                const int64_t p = (int64_t)h + i;
                const int64_t c = p / A.page_size;
                const int pg = c >= A.width ? -1 : c < hd ? row[c] : page((int)c - hd);
                A.positions[t0 + i] = p;
                A.slots[t0 + i] = pg >= 0 ? (int64_t)pg * A.page_size + p % A.page_size : -1;
            }
        }
        tokens += tt; taken += nt;
    }
    for (int64_t t = tokens + threadIdx.x; t < A.n_tokens; t += blockDim.x) { A.positions[t] = 0; A.slots[t] = -1; }
    int64_t none = 0, tt; int all_lost;
    __syncthreads();
    block_scan2(none, lost, wa, wb, tt, all_lost);
    if (threadIdx.x == 0) {
        *A.missing = max(taken - count, 0) + all_lost;
        *A.left = max(count - taken, 0);
    }
}

// rows that are done give back every page that they hold, in the order of the table, and forget them
__global__ void __launch_bounds__(STEP_THREADS) paged_release_kernel(const uint8_t* done, int R, int32_t* table, int64_t table_stride, int width,
                                                                     int32_t* pages, int n_pages, int32_t* count) {
    __shared__ int64_t wa[32];
    __shared__ int wb[32];
    int top = max(0, min(*count, n_pages));
    for (int r = 0; r < R; r++) {
        if (!done[r]) continue;
        int32_t* row = table + r * table_stride;
        for (int c0 = 0; c0 < width; c0 += blockDim.x) {
            const int c = c0 + threadIdx.x;
            const int page = c < width ? row[c] : -1;
            const int is = page >= 0;
            int64_t none = 0, tt;
            int at = is, total;
            block_scan2(none, at, wa, wb, tt, total);
            if (is && top + at - 1 < n_pages) pages[top + at - 1] = page;
            if (c < width) row[c] = -1;
            top = min(top + total, n_pages);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) *count = top;
}

// ------------------------------------------------------------------ rotary embedding and the write into the slots
struct AppendArgs {
    void* qkv; int64_t st; int64_t T; int Hq, Hkv, D, R;
    const void *cos, *sin; int cs_dtype; int64_t cs_row; int64_t n_pos;
    const int64_t *positions, *slots;
    uint8_t *kc, *vc; int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;
    int64_t n_slots; int page_size;
};
__device__ __forceinline__ float table_at(const void* p, int dtype, int64_t i) {
    return dtype == DT_F32 ? ((const float*)p)[i] : dtype == DT_F16 ? __half2float(((const __half*)p)[i]) : __bfloat162float(((const __nv_bfloat16*)p)[i]);
}
template <typename T> struct Act;
template <> struct Act<__half> {
    __device__ static float get(__half x) { return __half2float(x); }
    __device__ static __half put(float x) { return __float2half_rn(x); }
};
template <> struct Act<__nv_bfloat16> {
    __device__ static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
    __device__ static __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};
__device__ __forceinline__ uint8_t to_e5m2(float x) { return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E5M2); }

// element of a head and its partner by one thread
template <typename T, bool E5M2>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs A) {
    const int half = A.R / 2, per = half + (A.D - A.R), heads = A.Hq + 2 * A.Hkv;
    const int64_t total = A.T * heads * per;
    for (int64_t idx = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; idx < total; idx += (int64_t)gridDim.x * blockDim.x) {
        const int i = (int)(idx % per), h = (int)(idx / per % heads);
        const int64_t t = idx / ((int64_t)per * heads);
        T* row = (T*)A.qkv + t * A.st + (int64_t)h * A.D;
        const int e0 = i < half ? i : A.R + i - half, e1 = i < half ? i + half : e0;
        T x0 = row[e0], x1 = row[e1];
        if (i < half && h < A.Hq + A.Hkv) {
            int64_t p = A.positions[t];
            p = p < 0 ? 0 : p < A.n_pos ? p : A.n_pos - 1;
            const float c = table_at(A.cos, A.cs_dtype, p * A.cs_row + i), s = table_at(A.sin, A.cs_dtype, p * A.cs_row + i);
            const float a = Act<T>::get(x0), b = Act<T>::get(x1);
            x0 = Act<T>::put(fmaf(a, c, -b * s));
            x1 = Act<T>::put(fmaf(b, c, a * s));
            row[e0] = x0;
            row[e1] = x1;
        }
        if (h < A.Hq) continue;
        const int64_t slot = A.slots[t];
        if (slot < 0 || slot >= A.n_slots) continue;                 // a padded token, or one that got no page
        const bool is_k = h < A.Hq + A.Hkv;
        const int hk = h - A.Hq - (is_k ? 0 : A.Hkv);
        const int64_t pg = slot / A.page_size, in = slot % A.page_size;
        const int64_t at = is_k ? pg * A.k_sp + in * A.k_ss + hk * A.k_sh : pg * A.v_sp + in * A.v_ss + hk * A.v_sh;
        if (E5M2) {
            uint8_t* d = (is_k ? A.kc : A.vc) + at;
            d[e0] = to_e5m2(Act<T>::get(x0));
            d[e1] = to_e5m2(Act<T>::get(x1));
        } else {
            T* d = (T*)(is_k ? A.kc : A.vc) + at;
            d[e0] = x0;
            d[e1] = x1;
        }
    }
}

}  // namespace
}  // namespace lowbit

extern "C" int lowbit_paged_step_cuda(const int32_t* d_new, const int32_t* d_held, int R, int32_t* d_table, int64_t table_stride, int width,
                                      const int32_t* d_free_pages, int n_pages, const int32_t* d_free_count, int32_t* d_free_left, int page_size,
                                      int64_t n_tokens, int32_t* d_cu_seqlens, int32_t* d_seq_lens, int64_t* d_positions, int64_t* d_slots,
                                      int32_t* d_missing, void* stream) {
    reset_launch_count();
    if (!d_new || !d_held || !d_table || !d_free_pages || !d_free_count || !d_free_left || !d_cu_seqlens || !d_seq_lens || !d_missing ||
        (n_tokens > 0 && (!d_positions || !d_slots)) || R <= 0 || width <= 0 || table_stride < width || n_pages <= 0 || page_size <= 0 || n_tokens < 0) {
        set_error(LB_ERR_ARG, "lowbit_paged_step_cuda: bad argument (R %d, width %d, pages %d, page_size %d, tokens %lld)", R, width, n_pages, page_size,
                  (long long)n_tokens);
        return LB_ERR_ARG;
    }
    const StepArgs A = {d_new, d_held, R, d_table, table_stride, width, d_free_pages, n_pages, d_free_count, d_free_left, page_size, n_tokens,
                        d_cu_seqlens, d_seq_lens, d_positions, d_slots, d_missing};
    paged_step_kernel<<<1, STEP_THREADS, 0, (cudaStream_t)stream>>>(A);
    note_launch();
    return check_launch();
}

extern "C" int lowbit_paged_release_cuda(const uint8_t* d_done, int R, int32_t* d_table, int64_t table_stride, int width, int32_t* d_free_pages,
                                         int n_pages, int32_t* d_free_count, void* stream) {
    reset_launch_count();
    if (!d_done || !d_table || !d_free_pages || !d_free_count || R <= 0 || width <= 0 || table_stride < width || n_pages <= 0) {
        set_error(LB_ERR_ARG, "lowbit_paged_release_cuda: bad argument (R %d, width %d, pages %d)", R, width, n_pages);
        return LB_ERR_ARG;
    }
    paged_release_kernel<<<1, STEP_THREADS, 0, (cudaStream_t)stream>>>(d_done, R, d_table, table_stride, width, d_free_pages, n_pages, d_free_count);
    note_launch();
    return check_launch();
}

extern "C" int lowbit_paged_rope_append_cuda(void* d_qkv, int dtype, int64_t token_stride, int64_t T, int Hq, int Hkv, int D, int rotary_dim,
                                             const void* d_cos, const void* d_sin, int cs_dtype, int64_t cs_row_stride, int64_t n_positions,
                                             const int64_t* d_positions, const int64_t* d_slots, void* d_k_cache, const int64_t* k_strides,
                                             void* d_v_cache, const int64_t* v_strides, int cache_dtype, int n_pages, int page_size, void* stream) {
    reset_launch_count();
    if (!d_qkv || !d_slots || !d_k_cache || !d_v_cache || !k_strides || !v_strides || (dtype != DT_F16 && dtype != DT_BF16) ||
        (cache_dtype != dtype && cache_dtype != CACHE_E5M2) || T < 0 || Hq < 0 || Hkv <= 0 || D <= 0 || rotary_dim < 0 || rotary_dim > D || (rotary_dim & 1) ||
        (rotary_dim > 0 && (!d_cos || !d_sin || !d_positions || cs_dtype < 0 || cs_dtype > 2 || cs_row_stride < rotary_dim / 2 || n_positions <= 0)) ||
        n_pages <= 0 || page_size <= 0 || token_stride < (int64_t)(Hq + 2 * Hkv) * D) {
        set_error(LB_ERR_ARG, "lowbit_paged_rope_append_cuda: bad argument (T %lld, Hq %d, Hkv %d, D %d, rotary %d, dtype %d, cache dtype %d)", (long long)T, Hq,
                  Hkv, D, rotary_dim, dtype, cache_dtype);
        return LB_ERR_ARG;
    }
    if (T == 0) return LB_OK;
    AppendArgs A = {d_qkv, token_stride, T, Hq, Hkv, D, rotary_dim, d_cos, d_sin, cs_dtype, cs_row_stride, n_positions, d_positions, d_slots,
                    (uint8_t*)d_k_cache, (uint8_t*)d_v_cache, k_strides[0], k_strides[1], k_strides[2], v_strides[0], v_strides[1], v_strides[2],
                    (int64_t)n_pages * page_size, page_size};
    const int64_t total = T * (Hq + 2 * Hkv) * (D - rotary_dim / 2);
    const int64_t want = (total + 255) / 256, most = (int64_t)sm_count() * 8;
    const dim3 grid((unsigned)(want < most ? want : most));
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F16) {
        if (cache_dtype == CACHE_E5M2) paged_append_kernel<__half, true><<<grid, 256, 0, st>>>(A);
        else paged_append_kernel<__half, false><<<grid, 256, 0, st>>>(A);
    } else {
        if (cache_dtype == CACHE_E5M2) paged_append_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(A);
        else paged_append_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(A);
    }
    note_launch();
    return check_launch();
}
