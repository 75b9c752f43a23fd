// paged_cache.cu -- the bookkeeping of a paged key/value cache on the GPU and the write into it.
//
// lowbit_paged_step_cuda: from what every request holds (tokens in the cache) and brings (new tokens) the pages that it still needs, taken
// off a stack of free ones; its row of the block table; and for every new token its position and its slot (page * page_size + row).  With
//   need_r = ceil((held_r + new_r) / page_size) - ceil(held_r / page_size)      and      before_r = sum of need over the requests in front,
// request r's i-th new page is free[count - 1 - (before_r + i)], so a token's slot follows from two prefix sums and nobody waits for a
// neighbour's page.  What the table names behind held_r is written over, not looked at: such pages (a step that ran short and is repeated, tokens that a
// request drops) go back first (lowbit_paged_release_behind_cuda).
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
    int lost_most;                                            // pages behind the table's width that a request counts at most: the sum stays in 32 bits
};

constexpr int STEP_THREADS = 1024;

constexpr int64_t MOST = 0x7fffffff;

__device__ __forceinline__ int pages_of(int64_t tokens, int page) {
    return tokens <= MOST ? (int)(((uint32_t)tokens + (uint32_t)page - 1u) / (uint32_t)page) : (int)min((tokens + page - 1) / page, MOST);
}

// inclusive sums of three values over the block; t*: those of the whole block
struct Three { int64_t a; int b, c; };
__device__ __forceinline__ Three block_scan3(Three x, Three* warps, Three& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t a = __shfl_up_sync(0xffffffffu, x.a, d);
        const int b = __shfl_up_sync(0xffffffffu, x.b, d), c = __shfl_up_sync(0xffffffffu, x.c, d);
        if (lane >= d) { x.a += a; x.b += b; x.c += c; }
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    // every warp sums the warps' totals for itself
    Three w = lane < n ? warps[lane] : Three{0, 0, 0}, s = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t a = __shfl_up_sync(0xffffffffu, s.a, d);
        const int b = __shfl_up_sync(0xffffffffu, s.b, d), c = __shfl_up_sync(0xffffffffu, s.c, d);
        if (lane >= d) { s.a += a; s.b += b; s.c += c; }
    }
    total = {__shfl_sync(0xffffffffu, s.a, 31), __shfl_sync(0xffffffffu, s.b, 31), __shfl_sync(0xffffffffu, s.c, 31)};
    x.a += __shfl_sync(0xffffffffu, s.a - w.a, warp);
    x.b += __shfl_sync(0xffffffffu, s.b - w.b, warp);
    x.c += __shfl_sync(0xffffffffu, s.c - w.c, warp);
    return x;
}
// the last entry of the ascending list first[0 .. n) that is at most x (first[0] is)
__device__ __forceinline__ int last_at_most(const int64_t* first, int n, int64_t x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ int last_at_most(const int* first, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One block, or a cluster of them for many tokens.  Every block sums over all requests for itself, a round of a thread each; the round's tokens
// and new pages are then dealt to the cluster's threads, who find their request in the sums.  What a token's slot needs of pages that
// the step itself hands out comes from the stack, so nobody waits for the table.  The count of free pages is read by all before the first
// block writes it (it may be written in place): that is what the cluster is for.
// What bounds it: the launch and two passes of dependent loads.  32 requests with a token each 3.1 us; 500 requests, 19000 tokens 8.0 us, most of it
// the search of every token for its request.
__global__ void __launch_bounds__(STEP_THREADS) paged_step_kernel(const StepArgs A) {
    __shared__ Three sums[32];
    __shared__ int64_t first[STEP_THREADS];
    __shared__ int page0[STEP_THREADS], holds[STEP_THREADS], has[STEP_THREADS];
    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
    const int me = (int)rank * blockDim.x + threadIdx.x, all = (int)blocks * blockDim.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int count = max(0, min(*A.count, A.n_pages));
    if (blocks > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    int64_t tokens = 0;
    int taken = 0, over = 0;
    if (me == 0) A.cu[0] = 0;
    for (int r0 = 0; r0 < A.R; r0 += blockDim.x) {
        const int r = r0 + threadIdx.x, in_round = min((int)blockDim.x, A.R - r0);
        const int held = r < A.R ? max(A.held[r], 0) : 0, fresh = r < A.R ? max(A.fresh[r], 0) : 0;
        const int had = min(pages_of(held, A.page_size), A.width), all_pages = pages_of((int64_t)held + fresh, A.page_size);
        const int need = max(min(all_pages, A.width) - had, 0);
        const int lost = r < A.R ? min(max(all_pages - A.width, 0) - max(pages_of(held, A.page_size) - A.width, 0), A.lost_most) : 0;
        Three total;
        const Three x = block_scan3({fresh, need, lost}, sums, total);
        first[threadIdx.x] = tokens + x.a - fresh;
        page0[threadIdx.x] = x.b - need;
        holds[threadIdx.x] = held;
        has[threadIdx.x] = had;
        if (r < A.R && rank == 0) {
            A.cu[r + 1] = (int32_t)min(tokens + x.a, MOST);             // what 32 bits cannot say is their largest, and behind every row
            A.seq_lens[r] = (int32_t)min((int64_t)held + fresh, MOST);
        }
        __syncthreads();
        // page i of the round's new ones
        auto page = [&](int i) { const int at = count - 1 - (taken + i); return at >= 0 ? A.pages[at] : -1; };
        for (int i = me; i < total.b; i += all) {
            const int k = last_at_most(page0, in_round, i);
            A.table[(r0 + k) * A.table_stride + has[k] + i - page0[k]] = page(i);
        }
        const int64_t end = min(tokens + total.a, A.n_tokens);
        for (int64_t t = tokens + me; t < end; t += all) {
            const int k = last_at_most(first, in_round, t);
            const int64_t p = holds[k] + (t - first[k]);
            const int c = p < 1ll << 31 ? (int)((uint32_t)p / (uint32_t)A.page_size) : A.width;
            const int in = p < 1ll << 31 ? (int)((uint32_t)p % (uint32_t)A.page_size) : 0;
            const int pg = c >= A.width ? -1 : c < has[k] ? A.table[(r0 + k) * A.table_stride + c] : page(page0[k] + c - has[k]);
            A.positions[t] = p;
            A.slots[t] = pg >= 0 ? (int64_t)pg * A.page_size + in : -1;
        }
        tokens += total.a; taken += total.b; over += total.c;
        __syncthreads();
    }
    for (int64_t t = tokens + me; t < A.n_tokens; t += all) { A.positions[t] = 0; A.slots[t] = -1; }
    if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    else __syncthreads();
    if (me == 0) {
        *A.missing = (int32_t)min((int64_t)max(taken - count, 0) + over, MOST);
        *A.left = max(count - taken, 0);
    }
}

// rows that are done give back every page that they hold, in the order of the table, and forget them; with `held` those behind its tokens
__global__ void __launch_bounds__(STEP_THREADS) paged_release_kernel(const uint8_t* done, const int32_t* held, int page_size, int R, int32_t* table, int64_t table_stride,
                                                                     int width, int32_t* pages, int n_pages, int32_t* count) {
    __shared__ Three sums[32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    int top = max(0, min(*count, n_pages));
    for (int r = 0; r < R; r++) {
        if (!done[r]) continue;
        int32_t* row = table + r * table_stride;
        for (int c0 = held ? min(pages_of(max(held[r], 0), page_size), width) : 0; c0 < width; c0 += blockDim.x) {
            const int c = c0 + threadIdx.x;
            const int page = c < width ? row[c] : -1;
            Three total;
            const Three x = block_scan3({0, page >= 0, 0}, sums, total);
            if (page >= 0 && top + x.b - 1 < n_pages) pages[top + x.b - 1] = page;
            if (c < width) row[c] = -1;
            top = min(top + total.b, n_pages);
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

// an element of a head and its partner by one thread: whatever lies on no 16 bytes
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

// The same for rows on 16 bytes: 16 elements a thread, two runs of 8 that are each other's partners (rotated heads), or of one piece.  A head's
// tables are read once a head, from L1.  What bounds it: DRAM, 8000 tokens of 32 / 8 heads (217 MB) in 35.6 us, 6.1 TB/s.  The kernel of a pair a
// thread, half precision into e5m2: 32 tokens 2.8 us for 2.2, 256 tokens 7.7 for 2.7, 8000 tokens 202 for 35.
template <typename T, bool E5M2, typename C>
__global__ void __launch_bounds__(256) paged_append_vec_kernel(const AppendArgs A) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t per_head = (uint32_t)A.D / 16, heads = (uint32_t)(A.Hq + 2 * A.Hkv), per = per_head * heads, total = (uint32_t)A.T * per;
    const int half = A.R / 2;
    for (uint32_t idx = blockIdx.x * 256u + threadIdx.x; idx < total; idx += gridDim.x * 256u) {
        const uint32_t t = idx / per, in = idx - t * per;
        const int h = (int)(in / per_head), i = (int)(in - (uint32_t)h * per_head) * 8;       // 8 elements from i and, rotated, from i + half
        const bool turn = i < half, keeps = h < A.Hq + A.Hkv;                                  // queries and keys rotate
        if (!turn && h < A.Hq) continue;
        const int e0 = turn ? i : A.R + 2 * (i - half), e1 = turn ? i + half : e0 + 8;
        T* const row = (T*)A.qkv + t * A.st + (int64_t)h * A.D;
        T x0[8], x1[8];
        *reinterpret_cast<uint4*>(x0) = *reinterpret_cast<const uint4*>(row + e0);
        *reinterpret_cast<uint4*>(x1) = *reinterpret_cast<const uint4*>(row + e1);
        if (turn && keeps) {
            int64_t p = A.positions[t];
            p = p < 0 ? 0 : p < A.n_pos ? p : A.n_pos - 1;
            C c[8], s[8];
#pragma unroll
            for (int z = 0; z < (int)sizeof(C) / 2; z++) {
                reinterpret_cast<uint4*>(c)[z] = reinterpret_cast<const uint4*>((const C*)A.cos + p * A.cs_row + i)[z];
                reinterpret_cast<uint4*>(s)[z] = reinterpret_cast<const uint4*>((const C*)A.sin + p * A.cs_row + i)[z];
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float a = Act<T>::get(x0[e]), b = Act<T>::get(x1[e]), cf = (float)c[e], sf = (float)s[e];
                x0[e] = Act<T>::put(fmaf(a, cf, -b * sf));
                x1[e] = Act<T>::put(fmaf(b, cf, a * sf));
            }
            *reinterpret_cast<uint4*>(row + e0) = *reinterpret_cast<const uint4*>(x0);
            *reinterpret_cast<uint4*>(row + e1) = *reinterpret_cast<const uint4*>(x1);
        }
        if (h < A.Hq) continue;
        const int64_t slot = A.slots[t];
        if (slot < 0 || slot >= A.n_slots) continue;
        const int hk = h - A.Hq - (keeps ? 0 : A.Hkv);
        const int64_t pg = slot < 1ll << 31 ? (int64_t)((uint32_t)slot / (uint32_t)A.page_size) : slot / A.page_size, rw = slot - pg * A.page_size;
        const int64_t at = keeps ? pg * A.k_sp + rw * A.k_ss + hk * A.k_sh : pg * A.v_sp + rw * A.v_ss + hk * A.v_sh;
        if (E5M2) {
            uint8_t* const d = (keeps ? A.kc : A.vc) + at;
            uint8_t q0[8], q1[8];
#pragma unroll
            for (int e = 0; e < 8; e++) { q0[e] = to_e5m2(Act<T>::get(x0[e])); q1[e] = to_e5m2(Act<T>::get(x1[e])); }
            *reinterpret_cast<uint2*>(d + e0) = *reinterpret_cast<const uint2*>(q0);
            *reinterpret_cast<uint2*>(d + e1) = *reinterpret_cast<const uint2*>(q1);
        } else {
            T* const d = (T*)(keeps ? A.kc : A.vc) + at;
            *reinterpret_cast<uint4*>(d + e0) = *reinterpret_cast<const uint4*>(x0);
            *reinterpret_cast<uint4*>(d + e1) = *reinterpret_cast<const uint4*>(x1);
        }
    }
}
template <typename T, bool E5M2> void append_vec(const AppendArgs& A, unsigned grid, cudaStream_t st) {
    const bool on = launch_overlaps(st);
    if (A.R == 0 || A.cs_dtype == DT_F32) launch_behind(paged_append_vec_kernel<T, E5M2, float>, dim3(grid), 256, 0, st, on, A);
    else if (A.cs_dtype == DT_F16) launch_behind(paged_append_vec_kernel<T, E5M2, __half>, dim3(grid), 256, 0, st, on, A);
    else launch_behind(paged_append_vec_kernel<T, E5M2, __nv_bfloat16>, dim3(grid), 256, 0, st, on, A);
}

// ------------------------------------------------------------------ the same with a norm of every query and key head in front of the rotation
//   y = x w / sqrt(mean x^2 + eps), then y cos + rot(y) sin: one rounding, of the result
struct NormArgs { AppendArgs a; const void *qw, *kw; int w_dtype; float eps; };

// a head by a warp: whatever lies on no 16 bytes
template <typename T, bool E5M2>
__global__ void __launch_bounds__(256) paged_norm_append_kernel(const NormArgs N) {
    const AppendArgs& A = N.a;
    const int half = A.R / 2, per = half + (A.D - A.R), heads = A.Hq + 2 * A.Hkv, lane = threadIdx.x & 31;
    const int64_t total = A.T * heads;
    for (int64_t idx = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; idx < total; idx += ((int64_t)gridDim.x * blockDim.x) >> 5) {
        const int h = (int)(idx % heads);
        const int64_t t = idx / heads;
        T* const row = (T*)A.qkv + t * A.st + (int64_t)h * A.D;
        const bool keeps = h < A.Hq + A.Hkv;                   // queries and keys
        float inv = 1.0f;
        if (keeps) {
            float sum = 0.0f;
            for (int e = lane; e < A.D; e += 32) { const float x = Act<T>::get(row[e]); sum = fmaf(x, x, sum); }
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            inv = rsqrtf(sum / A.D + N.eps);
        }
        const void* const w = h < A.Hq ? N.qw : N.kw;
        int64_t p = A.R > 0 ? A.positions[t] : 0;
        p = p < 0 ? 0 : p < A.n_pos ? p : A.n_pos - 1;
        const int64_t slot = A.kc && h >= A.Hq ? A.slots[t] : -1;
        const bool kept = slot >= 0 && slot < A.n_slots;
        const int hk = h - A.Hq - (keeps ? 0 : A.Hkv);
        const int64_t pg = kept ? slot / A.page_size : 0, in = kept ? slot % A.page_size : 0;
        const int64_t at = keeps ? pg * A.k_sp + in * A.k_ss + hk * A.k_sh : pg * A.v_sp + in * A.v_ss + hk * A.v_sh;
        for (int i = lane; i < per; i += 32) {
            const int e0 = i < half ? i : A.R + i - half, e1 = i < half ? i + half : e0;
            T x0 = row[e0], x1 = row[e1];
            if (keeps) {
                const float a = Act<T>::get(x0) * inv * table_at(w, N.w_dtype, e0), b = Act<T>::get(x1) * inv * table_at(w, N.w_dtype, e1);
                const float c = i < half ? table_at(A.cos, A.cs_dtype, p * A.cs_row + i) : 1.0f, s = i < half ? table_at(A.sin, A.cs_dtype, p * A.cs_row + i) : 0.0f;
                x0 = Act<T>::put(i < half ? fmaf(a, c, -b * s) : a);
                x1 = Act<T>::put(i < half ? fmaf(b, c, a * s) : a);
                row[e0] = x0;
                row[e1] = x1;
            }
            if (!kept) continue;
            if (E5M2) {
                uint8_t* const d = (keeps ? A.kc : A.vc) + at;
                d[e0] = to_e5m2(Act<T>::get(x0));
                d[e1] = to_e5m2(Act<T>::get(x1));
            } else {
                T* const d = (T*)(keeps ? A.kc : A.vc) + at;
                d[e0] = x0;
                d[e1] = x1;
            }
        }
        __syncwarp();
    }
}

// Rows on 16 bytes: 16 elements a thread as in paged_append_vec_kernel, LANES (a power of two from D / 16 on) threads a head, whose squares meet by
// shuffles.  Memory bounds it: 8001 tokens of 32 + 8 + 8 heads of 128, 217 MB, in 39.7 us (5.5 TB/s); 32 tokens 3.0 us.  Blocks an SM: 4, 5, 8, 16, one a piece:
// 42.3, 39.7, 45.2, 44.6, 51.0 us (each fills its table of weights first).
template <typename T, bool E5M2, typename C, int LANES>
__global__ void __launch_bounds__(256) paged_norm_append_vec_kernel(const NormArgs N) {
    const AppendArgs& A = N.a;
    extern __shared__ __align__(16) float norm_w[];            // [2][D]
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    for (int i = threadIdx.x; i < 2 * A.D; i += 256) norm_w[i] = table_at(i < A.D ? N.qw : N.kw, N.w_dtype, i < A.D ? i : i - A.D);
    __syncthreads();
    const uint32_t heads = (uint32_t)(A.Hq + 2 * A.Hkv), per = heads * LANES, total = (uint32_t)A.T * per;
    const int half = A.R / 2;
    const float over = 1.0f / A.D;
    for (uint32_t base = blockIdx.x * 256u; base < total; base += gridDim.x * 256u) {
        const uint32_t idx = base + threadIdx.x, t = idx / per, in = idx - t * per;
        const int h = (int)(in / LANES), i = (int)(in % LANES) * 8;                            // 8 elements from i and, rotated, from i + half
        const bool live = idx < total && 2 * i < A.D, turn = i < half, keeps = h < A.Hq + A.Hkv;
        const int e0 = turn ? i : A.R + 2 * (i - half), e1 = turn ? i + half : e0 + 8;
        T* const row = (T*)A.qkv + t * A.st + (int64_t)h * A.D;
        T x0[8], x1[8];
        int64_t p = 0, slot = -1;                              // asked for with the row: they lead to other loads
        if (live) {
            *reinterpret_cast<uint4*>(x0) = *reinterpret_cast<const uint4*>(row + e0);
            *reinterpret_cast<uint4*>(x1) = *reinterpret_cast<const uint4*>(row + e1);
            if (turn && keeps) p = A.positions[t];
            if (h >= A.Hq && A.kc) slot = A.slots[t];
        }
        float sum = 0.0f;
        if (live && keeps) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float a = Act<T>::get(x0[e]), b = Act<T>::get(x1[e]);
                sum = fmaf(a, a, sum);
                sum = fmaf(b, b, sum);
            }
        }
#pragma unroll
        for (int d = LANES / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (!live) continue;
        if (keeps) {
            const float inv = rsqrtf(fmaf(sum, over, N.eps));
            const float* const w = norm_w + (h < A.Hq ? 0 : A.D);
            float a[8], b[8];
#pragma unroll
            for (int e = 0; e < 8; e++) { a[e] = Act<T>::get(x0[e]) * inv * w[e0 + e]; b[e] = Act<T>::get(x1[e]) * inv * w[e1 + e]; }
            if (turn) {
                p = p < 0 ? 0 : p < A.n_pos ? p : A.n_pos - 1;
                C c[8], s[8];
#pragma unroll
                for (int z = 0; z < (int)sizeof(C) / 2; z++) {
                    reinterpret_cast<uint4*>(c)[z] = reinterpret_cast<const uint4*>((const C*)A.cos + p * A.cs_row + i)[z];
                    reinterpret_cast<uint4*>(s)[z] = reinterpret_cast<const uint4*>((const C*)A.sin + p * A.cs_row + i)[z];
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float cf = (float)c[e], sf = (float)s[e];
                    x0[e] = Act<T>::put(fmaf(a[e], cf, -b[e] * sf));
                    x1[e] = Act<T>::put(fmaf(b[e], cf, a[e] * sf));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) { x0[e] = Act<T>::put(a[e]); x1[e] = Act<T>::put(b[e]); }
            }
            *reinterpret_cast<uint4*>(row + e0) = *reinterpret_cast<const uint4*>(x0);
            *reinterpret_cast<uint4*>(row + e1) = *reinterpret_cast<const uint4*>(x1);
        }
        if (slot < 0 || slot >= A.n_slots) continue;
        const int hk = h - A.Hq - (keeps ? 0 : A.Hkv);
        const int64_t pg = slot < 1ll << 31 ? (int64_t)((uint32_t)slot / (uint32_t)A.page_size) : slot / A.page_size, rw = slot - pg * A.page_size;
        const int64_t at = keeps ? pg * A.k_sp + rw * A.k_ss + hk * A.k_sh : pg * A.v_sp + rw * A.v_ss + hk * A.v_sh;
        if (E5M2) {
            uint8_t* const d = (keeps ? A.kc : A.vc) + at;
            uint8_t q0[8], q1[8];
#pragma unroll
            for (int e = 0; e < 8; e++) { q0[e] = to_e5m2(Act<T>::get(x0[e])); q1[e] = to_e5m2(Act<T>::get(x1[e])); }
            *reinterpret_cast<uint2*>(d + e0) = *reinterpret_cast<const uint2*>(q0);
            *reinterpret_cast<uint2*>(d + e1) = *reinterpret_cast<const uint2*>(q1);
        } else {
            T* const d = (T*)(keeps ? A.kc : A.vc) + at;
            *reinterpret_cast<uint4*>(d + e0) = *reinterpret_cast<const uint4*>(x0);
            *reinterpret_cast<uint4*>(d + e1) = *reinterpret_cast<const uint4*>(x1);
        }
    }
}
template <typename T, bool E5M2, typename C> void norm_append_lanes(const NormArgs& N, int lanes, unsigned grid, cudaStream_t st) {
    const bool on = launch_overlaps(st);
    const size_t smem = 2 * N.a.D * sizeof(float);
    if (lanes <= 4) launch_behind(paged_norm_append_vec_kernel<T, E5M2, C, 4>, dim3(grid), 256, smem, st, on, N);
    else if (lanes == 8) launch_behind(paged_norm_append_vec_kernel<T, E5M2, C, 8>, dim3(grid), 256, smem, st, on, N);
    else launch_behind(paged_norm_append_vec_kernel<T, E5M2, C, 16>, dim3(grid), 256, smem, st, on, N);
}
template <typename T, bool E5M2> void norm_append_vec(const NormArgs& N, int lanes, unsigned grid, cudaStream_t st) {
    if (N.a.R == 0 || N.a.cs_dtype == DT_F32) norm_append_lanes<T, E5M2, float>(N, lanes, grid, st);
    else if (N.a.cs_dtype == DT_F16) norm_append_lanes<T, E5M2, __half>(N, lanes, grid, st);
    else norm_append_lanes<T, E5M2, __nv_bfloat16>(N, lanes, grid, st);
}

}  // namespace
}  // namespace lowbit

extern "C" int lowbit_paged_step_cuda(const int32_t* d_new, const int32_t* d_held, int R, int32_t* d_table, int64_t table_stride, int width,
                                      const int32_t* d_free_pages, int n_pages, const int32_t* d_free_count, int32_t* d_free_left, int page_size,
                                      int64_t n_tokens, int32_t* d_cu_seqlens, int32_t* d_seq_lens, int64_t* d_positions, int64_t* d_slots,
                                      int32_t* d_missing, void* stream) {
    reset_launch_count();
    if (!d_new || !d_held || !d_table || !d_free_pages || !d_free_count || !d_free_left || !d_cu_seqlens || !d_seq_lens || !d_missing ||
        (n_tokens > 0 && (!d_positions || !d_slots)) || R <= 0 || width <= 0 || table_stride < width || n_pages <= 0 || page_size <= 0 || n_tokens < 0 ||
        (int64_t)R * width > 0x7fffffffll) {                            // pages are counted in 32 bits
        set_error(LB_ERR_ARG, "lowbit_paged_step_cuda: bad argument (R %d, width %d, pages %d, page_size %d, tokens %lld)", R, width, n_pages, page_size,
                  (long long)n_tokens);
        return LB_ERR_ARG;
    }
    const StepArgs A = {d_new, d_held, R, d_table, table_stride, width, d_free_pages, n_pages, d_free_count, d_free_left, page_size, n_tokens,
                        d_cu_seqlens, d_seq_lens, d_positions, d_slots, d_missing, 0x7fffffff / R};
    // A block for a decode step, a cluster of eight (the most that any device takes) for more tokens; blocks of 1024 threads where requests or
    // tokens are many.  One block / eight, of 256 threads: 32 requests with a token each 3.1 / 3.5 us, 4 with 800 tokens in all 4.5 / 3.6, 16
    // with 5000 14 / 4.8; of 1024: 500 requests with a token each 4.5 / 4.7, 19000 tokens 27 / 8.4.  256 / 1024 threads, eight blocks: 5000 tokens 4.8 /
    // 5.0, 7000 5.5 / 5.0, 8000 6.1 / 5.2; one block: 256 requests 3.3 / 4.2, 257 4.6 / 4.2, 500 5.0 / 4.4.  Near the borders, one block / eight: 400 tokens of one or 4
    // requests 3.5 / 3.6, of 100 4.0 / 3.4, 600 of 4 4.0 / 3.5, of 100 4.7 / 3.4.
    const bool many = n_tokens > 512, wide = R > 256 || n_tokens > 6000;
    cudaStream_t st = (cudaStream_t)stream;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(many ? 8 : 1);
    cfg.blockDim = dim3(wide ? STEP_THREADS : 256);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {many ? 8u : 1u, 1u, 1u};
    cfg.attrs = at;
    cfg.numAttrs = add_overlap(at, 1, launch_overlaps(st));
    cudaLaunchKernelEx(&cfg, paged_step_kernel, A);
    note_launch();
    return check_launch();
}

static int release(const char* name, const uint8_t* d_done, const int32_t* d_held, int page_size, int R, int32_t* d_table, int64_t table_stride, int width, int32_t* d_free_pages,
                   int n_pages, int32_t* d_free_count, void* stream) {
    reset_launch_count();
    if (!d_done || !d_table || !d_free_pages || !d_free_count || R <= 0 || width <= 0 || table_stride < width || n_pages <= 0 || page_size <= 0) {
        set_error(LB_ERR_ARG, "%s: bad argument (R %d, width %d, pages %d, page_size %d)", name, R, width, n_pages, page_size);
        return LB_ERR_ARG;
    }
    launch_behind(paged_release_kernel, dim3(1), STEP_THREADS, 0, (cudaStream_t)stream, launch_overlaps((cudaStream_t)stream), d_done, d_held, page_size, R, d_table, table_stride,
                  width, d_free_pages, n_pages, d_free_count);
    note_launch();
    return check_launch();
}

extern "C" int lowbit_paged_release_cuda(const uint8_t* d_done, int R, int32_t* d_table, int64_t table_stride, int width, int32_t* d_free_pages,
                                         int n_pages, int32_t* d_free_count, void* stream) {
    return release("lowbit_paged_release_cuda", d_done, nullptr, 1, R, d_table, table_stride, width, d_free_pages, n_pages, d_free_count, stream);
}

extern "C" int lowbit_paged_release_behind_cuda(const uint8_t* d_done, const int32_t* d_held, int R, int32_t* d_table, int64_t table_stride, int width,
                                                int page_size, int32_t* d_free_pages, int n_pages, int32_t* d_free_count, void* stream) {
    if (!d_held) page_size = 0;                                        // refused
    return release("lowbit_paged_release_behind_cuda", d_done, d_held, page_size, R, d_table, table_stride, width, d_free_pages, n_pages, d_free_count, stream);
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
    cudaStream_t st = (cudaStream_t)stream;
    const int64_t chunks = T * (Hq + 2 * Hkv) * (D / 16), table = rotary_dim == 0 ? 0 : cs_dtype == DT_F32 ? 3 : 7;
    if (D % 16 == 0 && rotary_dim % 16 == 0 && chunks < 1ll << 31 && !((uintptr_t)d_qkv & 15) && !(token_stride & 7) &&
        !(((uintptr_t)d_k_cache | (uintptr_t)d_v_cache) & (cache_dtype == CACHE_E5M2 ? 7 : 15)) &&
        !((k_strides[0] | k_strides[1] | k_strides[2] | v_strides[0] | v_strides[1] | v_strides[2]) & 7) &&
        (rotary_dim == 0 || (!(((uintptr_t)d_cos | (uintptr_t)d_sin) & 15) && !(cs_row_stride & table)))) {
        // five blocks an SM, as many as are resident; eight: 41 us where this takes 35.6 (8000 tokens, 32 / 8 heads)
        const int64_t want = (chunks + 255) / 256, most = (int64_t)sm_count() * 5;
        const unsigned grid = (unsigned)(want < most ? want : most);
        if (dtype == DT_F16) cache_dtype == CACHE_E5M2 ? append_vec<__half, true>(A, grid, st) : append_vec<__half, false>(A, grid, st);
        else cache_dtype == CACHE_E5M2 ? append_vec<__nv_bfloat16, true>(A, grid, st) : append_vec<__nv_bfloat16, false>(A, grid, st);
        note_launch();
        return check_launch();
    }
    const int64_t total = T * (Hq + 2 * Hkv) * (D - rotary_dim / 2);
    const int64_t want = (total + 255) / 256, most = (int64_t)sm_count() * 8;
    const dim3 grid((unsigned)(want < most ? want : most));
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

extern "C" int lowbit_paged_norm_rope_append_cuda(void* d_qkv, int dtype, int64_t token_stride, int64_t T, int Hq, int Hkv, int D, int rotary_dim,
                                                  const void* d_q_weight, const void* d_k_weight, int w_dtype, float eps, const void* d_cos, const void* d_sin, int cs_dtype,
                                                  int64_t cs_row_stride, int64_t n_positions, const int64_t* d_positions, const int64_t* d_slots, void* d_k_cache,
                                                  const int64_t* k_strides, void* d_v_cache, const int64_t* v_strides, int cache_dtype, int n_pages, int page_size,
                                                  void* stream) {
    reset_launch_count();
    const bool cached = d_k_cache != nullptr;
    if (!d_qkv || !d_q_weight || !d_k_weight || w_dtype < 0 || w_dtype > 2 || !(eps >= 0.0f) || (dtype != DT_F16 && dtype != DT_BF16) || T < 0 || Hq < 0 || Hkv < 0 || Hq + Hkv <= 0 || D <= 0 ||
        rotary_dim < 0 || rotary_dim > D || (rotary_dim & 1) ||
        (rotary_dim > 0 && (!d_cos || !d_sin || !d_positions || cs_dtype < 0 || cs_dtype > 2 || cs_row_stride < rotary_dim / 2 || n_positions <= 0)) ||
        token_stride < (int64_t)(Hq + 2 * Hkv) * D || cached != (d_v_cache != nullptr) ||
        (cached && (!d_slots || !k_strides || !v_strides || (cache_dtype != dtype && cache_dtype != CACHE_E5M2) || Hkv <= 0 || n_pages <= 0 || page_size <= 0))) {
        set_error(LB_ERR_ARG, "lowbit_paged_norm_rope_append_cuda: bad argument (T %lld, Hq %d, Hkv %d, D %d, rotary %d, dtype %d, cache dtype %d)", (long long)T, Hq,
                  Hkv, D, rotary_dim, dtype, cache_dtype);
        return LB_ERR_ARG;
    }
    if (T == 0) return LB_OK;
    const int64_t none[3] = {0, 0, 0};
    if (!cached) { k_strides = v_strides = none; n_pages = page_size = 1; cache_dtype = dtype; }
    const NormArgs N = {{d_qkv, token_stride, T, Hq, Hkv, D, rotary_dim, d_cos, d_sin, cs_dtype, cs_row_stride, n_positions, d_positions, d_slots,
                         (uint8_t*)d_k_cache, (uint8_t*)d_v_cache, k_strides[0], k_strides[1], k_strides[2], v_strides[0], v_strides[1], v_strides[2],
                         (int64_t)n_pages * page_size, page_size}, d_q_weight, d_k_weight, w_dtype, eps};
    cudaStream_t st = (cudaStream_t)stream;
    int lanes = 4;
    while (lanes * 16 < D) lanes *= 2;
    const int64_t threads = T * (Hq + 2 * Hkv) * lanes, table = rotary_dim == 0 ? 0 : cs_dtype == DT_F32 ? 3 : 7;
    const bool e5m2 = cache_dtype == CACHE_E5M2;
    if (D % 16 == 0 && D <= 256 && rotary_dim % 16 == 0 && threads < 1ll << 31 && !((uintptr_t)d_qkv & 15) && !(token_stride & 7) &&
        !(((uintptr_t)d_k_cache | (uintptr_t)d_v_cache) & (e5m2 ? 7 : 15)) &&
        !((k_strides[0] | k_strides[1] | k_strides[2] | v_strides[0] | v_strides[1] | v_strides[2]) & 7) &&
        (rotary_dim == 0 || (!(((uintptr_t)d_cos | (uintptr_t)d_sin) & 15) && !(cs_row_stride & table)))) {
        const int64_t want = (threads + 255) / 256, most = (int64_t)sm_count() * 5;
        const unsigned grid = (unsigned)(want < most ? want : most);
        if (dtype == DT_F16) e5m2 ? norm_append_vec<__half, true>(N, lanes, grid, st) : norm_append_vec<__half, false>(N, lanes, grid, st);
        else e5m2 ? norm_append_vec<__nv_bfloat16, true>(N, lanes, grid, st) : norm_append_vec<__nv_bfloat16, false>(N, lanes, grid, st);
        note_launch();
        return check_launch();
    }
    const int64_t want = (T * (Hq + 2 * Hkv) + 7) / 8, most = (int64_t)sm_count() * 8;
    const dim3 grid((unsigned)(want < most ? want : most));
    if (dtype == DT_F16) {
        if (e5m2) paged_norm_append_kernel<__half, true><<<grid, 256, 0, st>>>(N);
        else paged_norm_append_kernel<__half, false><<<grid, 256, 0, st>>>(N);
    } else {
        if (e5m2) paged_norm_append_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(N);
        else paged_norm_append_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(N);
    }
    note_launch();
    return check_launch();
}
