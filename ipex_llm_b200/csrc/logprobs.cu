// logprobs.cu -- what a row of logits says about its tokens, and the gradient of that.  With z the row divided by the temperature:
//   log p_i = z_i - log sum_j exp z_j,      H = - sum_j p_j log p_j,      the k largest logits in order, the lower index first where two are equal;
//   dL/dz_i = sum_m g_m [i = i_m] - p_i (sum_m g_m + g_H (log p_i + H))    over the given token and the alternatives m.
// One pass over the row: exponentials and their sums in 32 bits relative to a maximum that runs along.  The k largest cost that pass nothing but a maximum
// a thread: at least k elements are not below the k-th largest of the threads' maxima, so the k largest lie in the strips of the threads whose
// maximum reaches it, some k of them, and those are read again from L2.
#include "lowbit_common.cuh"
#include "lowbit_internal.h"

using namespace lowbit;

namespace lowbit {
namespace {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_MOST = 32, LP_ROOM = 512;
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;

struct LogprobArgs {
    const void* logits; int64_t row; int64_t rows; int V;
    const int64_t* tokens; float c, by;                       // c = log2 e / temperature, by = 1 / temperature
    int k;
    float *logp, *entropy; int64_t* ids; float* top; float4* stats;
};
// A row's stats, for the gradient: ref and m of an element's exponent u = (x - ref) c - m, base 2 (ref is 0 but in rows whose products pass 32 bits);
// the sum of the powers; the mean of the exponents under them

template <typename T> struct Vec;                              // 16 bytes of logits
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4& w, float (&x)[4]) { x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w); }
};
template <> struct Vec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(v + i)); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(v[i] << 16); x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u); }
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// a reference for exponents, the sum of powers, and of powers x exponents, relative to it; the largest logit
struct Sums {
    float m, s, d, big;
    __device__ __forceinline__ void add(const Sums& o) {
        const float to = fmaxf(m, o.m);
        const float a = m == to ? 0.0f : m - to, b = o.m == to ? 0.0f : o.m - to;
        const float wa = ex2(a), wb = ex2(b);
        // a side that holds nothing has m = -inf: weight 0
        d = (s == 0.0f ? 0.0f : wa * fmaf(s, a, d)) + (o.s == 0.0f ? 0.0f : wb * fmaf(o.s, b, o.d));
        s = (s == 0.0f ? 0.0f : wa * s) + (o.s == 0.0f ? 0.0f : wb * o.s);
        m = to;
        big = fmaxf(big, o.big);
    }
};

// order of the alternatives: larger value first, then lower index.  -0 equals 0; key 0 is nobody's
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.0f), o = (int)b < 0 ? ~b : b | 0x80000000u;
    return (uint64_t)o << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

// one value a lane, sorted over the warp, the largest in lane 0
template <typename K> __device__ __forceinline__ K sort32(K x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int step = size >> 1; step; step >>= 1) {
            const K y = __shfl_xor_sync(0xffffffffu, x, step);
            const bool down = (lane & size) == 0 || size == 32, low = (lane & step) == 0;
            x = (x > y) == (down == low) ? x : y;
        }
    return x;
}
// the 32 largest of two sorted lists, sorted
template <typename K> __device__ __forceinline__ K merge32(K x, K y) {
    const int lane = threadIdx.x & 31;
    y = __shfl_xor_sync(0xffffffffu, y, 31);
    x = x > y ? x : y;
#pragma unroll
    for (int step = 16; step; step >>= 1) {
        const K z = __shfl_xor_sync(0xffffffffu, x, step);
        x = (x > z) == ((lane & step) == 0) ? x : z;
    }
    return x;
}

// the elements of a row that block `rank` of `blocks` takes: a strip of whole 16-byte pieces, the ends that lie on none to the first and last block
template <typename T> struct Strip {
    const T* row; int head, first, last, tail, V;              // elements [0, head) and [tail, V) one by one, pieces [first, last) from `head` on
    __device__ __forceinline__ Strip(const T* r, int V_, int rank, int blocks) : row(r), V(V_) {
        constexpr int N = Vec<T>::N;
        head = min((int)((16 - ((uintptr_t)r & 15)) & 15) / (int)sizeof(T), V_);
        const int pieces = (V_ - head) / N, each = (pieces + blocks - 1) / blocks;
        first = min(rank * each, pieces);
        last = min(first + each, pieces);
        tail = rank == blocks - 1 ? head + pieces * N : V_;
        if (rank != 0) head = -head;                           // not ours, but where the pieces begin
    }
    __device__ __forceinline__ int base() const { return head < 0 ? -head : head; }
    __device__ __forceinline__ uint4 piece(int i) const { return *reinterpret_cast<const uint4*>(row + base() + (int64_t)i * Vec<T>::N); }
    // this thread's element of the ends, -1: none (up to 7 + 7)
    __device__ __forceinline__ int end_of(int t) const {
        const int h = max(head, 0);
        return t < h ? t : t - h < V - tail ? tail + t - h : -1;
    }
};
template <typename T> __device__ __forceinline__ float one(const T* p) { return to_float<T>(*p); }

// the k-th largest of the threads' values: a lower bound of the k-th largest element
__device__ __forceinline__ float kth_of_threads(float x, int k, uint32_t (*lists)[32], float* out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t b = __float_as_uint(x + 0.0f);
    uint32_t key = sort32((int)b < 0 ? ~b : b | 0x80000000u);
    lists[warp][lane] = key;
#pragma unroll
    for (int n = LP_WARPS / 2; n; n >>= 1) {
        __syncthreads();
        if (warp < n) {
            key = merge32(key, lists[warp + n][lane]);
            lists[warp][lane] = key;
        }
    }
    if (warp == 0 && lane == k - 1) *out = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    __syncthreads();
    return *out;
}

// blocks of a cluster share a row.  What bounds it: see the launch below
template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS) token_logprobs_kernel(const LogprobArgs A) {
    constexpr int N = Vec<T>::N;
    __shared__ Sums warps[LP_WARPS];
    __shared__ __align__(16) Sums mine;                        // read by the cluster's first block
    __shared__ Sums total;
    __shared__ uint64_t found[TOP ? LP_ROOM : 1];
    __shared__ uint64_t lists[TOP ? LP_WARPS : 1][32];
    __shared__ uint64_t best[32];                              // as `mine`
    __shared__ float level;
    __shared__ int n_found;
    __shared__ uint32_t owners[LP_WARPS];
    __shared__ uint8_t owner[LP_THREADS];
    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
    const int64_t r = blockIdx.x / blocks;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const T* const row = (const T*)A.logits + r * A.row;
    const Strip<T> strip(row, A.V, (int)rank, (int)blocks);
    const float c = A.c;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    // ---- the pass
    Sums x = {-INFINITY, 0.0f, 0.0f, -INFINITY};
    auto take = [&](const float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i += 2) x.big = max3(x.big, v[i], v[i + 1]);
        // the reference follows where an exponent would pass 2^20 of it: sums of powers up to that are as exact as those up to 1
        const float top = x.big * c;
        if (top > x.m + 20.0f) {
            const float a = x.m - top, w = ex2(a);
            x.d = x.s == 0.0f ? 0.0f : w * fmaf(x.s, a, x.d);
            x.s = x.s == 0.0f ? 0.0f : w * x.s;
            x.m = top;
        }
        const float ref = x.m == -INFINITY ? 0.0f : x.m;       // nothing but -inf so far
        float s0 = 0.0f, s1 = 0.0f, d0 = 0.0f, d1 = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float a = fmaf(v[i], c, -ref), b = fmaf(v[i + 1], c, -ref), ea = ex2(a), eb = ex2(b);
            s0 += ea; s1 += eb;
            d0 = fmaf(ea, fmaxf(a, -300.0f), d0);              // a power of 0 adds 0, not 0 x inf
            d1 = fmaf(eb, fmaxf(b, -300.0f), d1);
        }
        x.s += s0 + s1;
        x.d += d0 + d1;
    };
    constexpr int AHEAD = 4;
    for (int i = strip.first + t; i < strip.last; i += AHEAD * LP_THREADS) {
        uint4 w[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++)
            if (i + a * LP_THREADS < strip.last) w[a] = strip.piece(i + a * LP_THREADS);
#pragma unroll
        for (int a = 0; a < AHEAD; a++)
            if (i + a * LP_THREADS < strip.last) { float v[N]; Vec<T>::get(w[a], v); take(v); }
    }
    const int end = strip.end_of(t);
    if (end >= 0) {
        float v[N];
        v[0] = one(row + end);
#pragma unroll
        for (int e = 1; e < N; e++) v[e] = -INFINITY;
        take(v);
    }

    // ---- the block's sums, and the cluster's
    const float own_big = x.big;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        Sums o = {__shfl_xor_sync(0xffffffffu, x.m, d), __shfl_xor_sync(0xffffffffu, x.s, d), __shfl_xor_sync(0xffffffffu, x.d, d), __shfl_xor_sync(0xffffffffu, x.big, d)};
        // in the order of the lanes on both sides, so that both hold the same
        Sums lo = lane & d ? o : x, hi = lane & d ? x : o;
        lo.add(hi);
        x = lo;
    }
    if (lane == 0) warps[warp] = x;
    if (t == 0) n_found = 0;
    if (!TOP) __syncthreads();

    if (TOP) {
        // ---- the strips in which the k largest lie, read again
        const float floor_ = kth_of_threads(own_big, A.k, reinterpret_cast<uint32_t(*)[32]>(&lists[0][0]), &level);
        const uint32_t own = __ballot_sync(0xffffffffu, own_big >= floor_);
        if (lane == 0) owners[warp] = own;
        __syncthreads();
        int strips = 0, before = 0;
#pragma unroll
        for (int w = 0; w < LP_WARPS; w++) { const int c_ = __popc(owners[w]); strips += c_; before += w < warp ? c_ : 0; }
        if (own >> lane & 1) owner[before + __popc(own & ((1u << lane) - 1u))] = (uint8_t)t;
        __syncthreads();
        auto note = [&](float v, int at) {
            if (v >= floor_) {
                const int slot = atomicAdd(&n_found, 1);       // their order does not matter: they are sorted
                if (slot < LP_ROOM) found[slot] = key_of(v, (uint32_t)at);
            }
        };
        const int deep = (strip.last - strip.first + LP_THREADS - 1) / LP_THREADS;             // pieces of a strip
        for (int i = t; i < strips * deep; i += AHEAD * LP_THREADS) {
            uint4 w[AHEAD];
            int p[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) {
                const int u = i + a * LP_THREADS, s = u / deep;
                p[a] = s < strips ? strip.first + owner[s] + (u - s * deep) * LP_THREADS : strip.last;
                if (p[a] < strip.last) w[a] = strip.piece(p[a]);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
                if (p[a] < strip.last) {
                    float v[N];
                    Vec<T>::get(w[a], v);
#pragma unroll
                    for (int e = 0; e < N; e++) note(v[e], strip.base() + p[a] * N + e);
                }
        }
        if (end >= 0) note(one(row + end), end);
        __syncthreads();
        const int n = n_found;
        uint64_t key = 0;
        if (n <= LP_ROOM) {
            for (int b = 32 * warp; b < n; b += LP_THREADS) key = merge32(key, sort32(b + lane < n ? found[b + lane] : (uint64_t)0));
        } else {
            // too many equal ones, or the largest lie in few strips: every warp keeps its 32 largest of the whole strip as it goes along
            auto keep = [&](float v, int at, bool there) {
                const uint64_t mine_ = there && v == v ? key_of(v, (uint32_t)at) : (uint64_t)0;
                uint64_t last = __shfl_sync(0xffffffffu, key, 31);
                for (uint32_t c_ = __ballot_sync(0xffffffffu, mine_ > last); c_; c_ &= c_ - 1) {
                    const uint64_t cand = __shfl_sync(0xffffffffu, mine_, __ffs(c_) - 1);
                    const uint64_t up = __shfl_up_sync(0xffffffffu, key, 1);
                    const int place = __popc(__ballot_sync(0xffffffffu, key > cand));
                    key = lane < place ? key : lane == place ? cand : up;
                }
            };
            for (int p0 = strip.first + 32 * warp; p0 < strip.last; p0 += LP_THREADS) {
                const int p = p0 + lane;
                float v[N];
                Vec<T>::get(strip.piece(min(p, strip.last - 1)), v);
#pragma unroll 1
                for (int e = 0; e < N; e++) {
                    float u = v[0];
#pragma unroll
                    for (int q = 1; q < N; q++) u = e == q ? v[q] : u;
                    keep(u, strip.base() + p * N + e, p < strip.last);
                }
            }
            if (warp == 0) {
                const int at = strip.end_of(lane);
                keep(at >= 0 ? one(row + at) : 0.0f, at, at >= 0);
            }
        }
        if (n > 32) {                                          // else the first warp has them all
            lists[warp][lane] = key;
#pragma unroll
            for (int h = LP_WARPS / 2; h; h >>= 1) {
                __syncthreads();
                if (warp < h) {
                    key = merge32(key, lists[warp + h][lane]);
                    lists[warp][lane] = key;
                }
            }
        }
        if (warp == 0) best[lane] = key;
    }
    if (t == 0) {
        for (int w = 1; w < LP_WARPS; w++) x.add(warps[w]);
        mine = x;
    }
    __syncthreads();
    if (blocks > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (rank == 0) {
        // the first block's first warp: the others' sums and lists, in their order
        uint64_t key = 0;
        if (warp == 0) {
            const uint32_t at_mine = (uint32_t)__cvta_generic_to_shared(&mine), at_best = (uint32_t)__cvta_generic_to_shared(&best[lane]);
            Sums all = mine;
            if (TOP) key = best[lane];
            for (uint32_t b = 1; b < blocks; b++) {
                uint32_t p;
                Sums o;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(at_mine), "r"(b));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o.m), "=f"(o.s), "=f"(o.d), "=f"(o.big) : "r"(p) : "memory");
                all.add(o);
                if (TOP) {
                    uint64_t other;
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(at_best), "r"(b));
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(other) : "r"(p) : "memory");
                    key = merge32(key, other);
                }
            }
            if (lane == 0) total = all;
        }
        __syncthreads();
        Sums all = total;
        float ref = 0.0f;
        if (!(fabsf(all.m) < 16777216.0f)) {
            // the products have lost the logits' differences, or passed 32 bits: the row once more, the largest logit taken off first.  A row of the
            // type's lowest value is even; one of -inf alone, or with inf in it, has no probabilities
            ref = all.big;
            float s = fabsf(ref) < INFINITY ? 0.0f : NAN, d = 0.0f;
            for (int j = t; j < A.V; j += LP_THREADS) {
                const float a = (one(row + j) - ref) * c, e = ex2(a);
                s += e;
                d = fmaf(e, fmaxf(a, -300.0f), d);
            }
#pragma unroll
            for (int h = 16; h; h >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, h); d += __shfl_xor_sync(0xffffffffu, d, h); }
            if (lane == 0) warps[warp] = {0.0f, s, d, ref};
            __syncthreads();
            all = {0.0f, 0.0f, 0.0f, ref};
            for (int w = 0; w < LP_WARPS; w++) { all.s += warps[w].s; all.d += warps[w].d; }
        }
        const float log2s = log2f(all.s);
        auto logp = [&](float v) {
            const float u = fmaf(v - ref, c, -all.m);
            // the type's lowest value: base e has room for what base 2 has not
            return u == -INFINITY ? fmaf(v - ref, A.by, -(all.m + log2s) * LP_LN2) : (u - log2s) * LP_LN2;
        };
        if (t == 0) {
            const int64_t token = A.tokens[r];
            A.logp[r] = token >= 0 && token < A.V ? logp(one(row + token)) : 0.0f;
            A.entropy[r] = (log2s - all.d / all.s) * LP_LN2;
            if (A.stats) A.stats[r] = make_float4(ref, all.m, all.s, all.d / all.s);
        }
        if (TOP && t < A.k) {
            const uint32_t id = key_index(key);
            A.ids[r * A.k + t] = key ? (int64_t)id : -1;       // a row with fewer numbers than that
            A.top[r * A.k + t] = key ? logp(one(row + id)) : NAN;
        }
    }
    __syncwarp();
    if (blocks > 1) {                                          // nobody leaves while the first block reads its sums
        asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    }
}

// ------------------------------------------------------------------ the gradient
struct LogprobGradArgs {
    const void* logits; int64_t row; int64_t rows; int V;
    const int64_t* tokens; float c, by;                        // by = 1 / temperature
    int k;
    const int64_t* ids;
    const float *g_logp, *g_entropy, *g_top;                   // NULL: zero
    const float4* stats;
    void* grad; int64_t grad_row;
    int chunk, chunks;                                         // elements of a block; blocks of a row
};

template <typename T> __device__ __forceinline__ void pack(const float (&x)[Vec<T>::N], uint4& w);
template <> __device__ __forceinline__ void pack<float>(const float (&x)[4], uint4& w) { w = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])); }
template <> __device__ __forceinline__ void pack<__half>(const float (&x)[8], uint4& w) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w = *reinterpret_cast<const uint4*>(h);
}
template <> __device__ __forceinline__ void pack<__nv_bfloat16>(const float (&x)[8], uint4& w) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w = *reinterpret_cast<const uint4*>(h);
}

// a piece of a row a block; the elements that the row's tokens name are written over at the end, by a thread each
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) token_logprobs_grad_kernel(const LogprobGradArgs A) {
    constexpr int N = Vec<T>::N;
    __shared__ int64_t ids[LP_MOST + 1];
    __shared__ float gs[LP_MOST + 1];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int64_t r = blockIdx.x / A.chunks;
    const int t = threadIdx.x, from = (int)(blockIdx.x - r * A.chunks) * A.chunk, to = min(from + A.chunk, A.V);
    const T* const row = (const T*)A.logits + r * A.row;
    T* const out = (T*)A.grad + r * A.grad_row;
    if (t <= A.k) {
        const int64_t id = t == 0 ? A.tokens[r] : A.ids[r * A.k + t - 1];
        const float g = t == 0 ? (A.g_logp ? A.g_logp[r] : 0.0f) : A.g_top ? A.g_top[r * A.k + t - 1] : 0.0f;
        const bool there = id >= 0 && id < A.V;
        ids[t] = there ? id : -1;
        gs[t] = there ? g : 0.0f;
    }
    const float4 st = A.stats[r];
    const float gh = A.g_entropy ? A.g_entropy[r] : 0.0f;
    __syncthreads();
    float total = 0.0f;
    for (int j = 0; j <= A.k; j++) total += gs[j];
    // log p + H = (u - mean u) ln 2, so that dL/dx = 2^u (a + b u)
    const float scale = -A.by / st.z, b = scale * gh * LP_LN2, a = scale * (total - gh * LP_LN2 * st.w);
    auto at = [&](float x) {
        const float u = fmaf(x - st.x, A.c, -st.y);
        return ex2(u) * fmaf(b, fmaxf(u, -300.0f), a);         // a power of 0 gives 0, not 0 x inf
    };
    const int head = (int)((16 - ((uintptr_t)(row + from) & 15)) & 15) / (int)sizeof(T);
    int i = from;
    if ((((uintptr_t)row ^ (uintptr_t)out) & 15) == 0) {
        const int begin = min(from + head, to), pieces = (to - begin) / N;
        const uint4* const src = reinterpret_cast<const uint4*>(row + begin);
        uint4* const dst = reinterpret_cast<uint4*>(out + begin);
        if (t < begin - from) out[from + t] = from_float<T>(at(one(row + from + t)));
        auto piece = [&](uint4 w) {
            float x[N];
            Vec<T>::get(w, x);
#pragma unroll
            for (int e = 0; e < N; e++) x[e] = at(x[e]);
            pack<T>(x, w);
            return w;
        };
        constexpr int AHEAD = 4;
        int p = t;
        for (; p + (AHEAD - 1) * LP_THREADS < pieces; p += AHEAD * LP_THREADS) {
            uint4 w[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; q++) w[q] = src[p + q * LP_THREADS];
#pragma unroll
            for (int q = 0; q < AHEAD; q++) dst[p + q * LP_THREADS] = piece(w[q]);
        }
        for (; p < pieces; p += LP_THREADS) dst[p] = piece(src[p]);
        i = begin + pieces * N;
    }
    for (int j = i + t; j < to; j += LP_THREADS) out[j] = from_float<T>(at(one(row + j)));
    __syncthreads();
    if (t <= A.k && ids[t] >= from && ids[t] < to) {
        float g = 0.0f;
        bool first = true;
        for (int j = 0; j <= A.k; j++)
            if (ids[j] == ids[t]) { g += gs[j]; first &= j >= t; }
        if (first) out[ids[t]] = from_float<T>(fmaf(g, A.by, at(one(row + ids[t]))));
    }
}

bool bad_logits(const char* name, const void* logits, int dtype, int64_t row_stride, int64_t rows, int64_t V, const void* tokens, float temperature, int k) {
    const bool bad = !logits || dtype < 0 || dtype > 2 || rows < 0 || V <= 0 || V > 0x7fff0000ll || row_stride < V || !tokens || !(temperature > 0.0f) || !(temperature < INFINITY) ||
                     k < 0 || k > LP_MOST || k > V || rows > 0x3ffffffll || ((uintptr_t)logits & (dtype == DT_F32 ? 3 : 1));
    if (bad) set_error(LB_ERR_ARG, "%s: bad argument (rows %lld, vocabulary %lld, dtype %d, top_k %d)", name, (long long)rows, (long long)V, dtype, k);
    return bad;
}

template <typename T> int logprobs_launch(const LogprobArgs& A, cudaStream_t st) {
    // blocks of a row: as many as are resident at once, five an SM, each with a piece a thread at least
    int64_t blocks = A.rows < 5ll * sm_count() ? 5ll * sm_count() / A.rows : 1;
    if (blocks > 8) blocks = 8;
    if (blocks > A.V / (LP_THREADS * Vec<T>::N)) blocks = A.V / (LP_THREADS * Vec<T>::N);
    if (blocks < 1) blocks = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(A.rows * blocks));
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)blocks, 1u, 1u};
    cfg.attrs = at;
    cfg.numAttrs = add_overlap(at, 1, launch_overlaps(st));
    if (A.k) cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, A);
    else cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, A);
    note_launch();
    return check_launch();
}

template <typename T> int grad_launch(LogprobGradArgs A, cudaStream_t st) {
    // a block's piece: some 16 of 16 bytes a thread; whole pieces, so that only a row's ends lie on none
    A.chunk = LP_THREADS * Vec<T>::N * 8;
    A.chunks = (A.V + A.chunk - 1) / A.chunk;
    launch_behind(token_logprobs_grad_kernel<T>, dim3((unsigned)(A.rows * A.chunks)), LP_THREADS, 0, st, launch_overlaps(st), A);
    note_launch();
    return check_launch();
}

}  // namespace
}  // namespace lowbit

extern "C" int lowbit_token_logprobs_cuda(const void* d_logits, int dtype, int64_t row_stride, int64_t rows, int64_t V, const int64_t* d_tokens, float temperature, int top_k,
                                          float* d_logprobs, float* d_entropy, int64_t* d_top_ids, float* d_top_logprobs, float* d_stats, void* stream) {
    reset_launch_count();
    const char* const name = "lowbit_token_logprobs_cuda";
    if (rows == 0) return LB_OK;
    if (bad_logits(name, d_logits, dtype, row_stride, rows, V, d_tokens, temperature, top_k)) return LB_ERR_ARG;
    if (!d_logprobs || !d_entropy || (top_k && (!d_top_ids || !d_top_logprobs)) || ((uintptr_t)d_stats & 15)) {
        set_error(LB_ERR_ARG, "%s: an output is missing or off its alignment", name);
        return LB_ERR_ARG;
    }
    const LogprobArgs A = {d_logits, row_stride, rows, (int)V, d_tokens, LP_LOG2E / temperature, 1.0f / temperature, top_k, d_logprobs, d_entropy, d_top_ids, d_top_logprobs, (float4*)d_stats};
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == DT_F32 ? logprobs_launch<float>(A, st) : dtype == DT_F16 ? logprobs_launch<__half>(A, st) : logprobs_launch<__nv_bfloat16>(A, st);
}

extern "C" int lowbit_token_logprobs_grad_cuda(const void* d_logits, int dtype, int64_t row_stride, int64_t rows, int64_t V, const int64_t* d_tokens, float temperature, int top_k,
                                               const int64_t* d_top_ids, const float* d_g_logprobs, const float* d_g_entropy, const float* d_g_top, const float* d_stats,
                                               void* d_grad, int64_t grad_row_stride, void* stream) {
    reset_launch_count();
    const char* const name = "lowbit_token_logprobs_grad_cuda";
    if (rows == 0) return LB_OK;
    if (bad_logits(name, d_logits, dtype, row_stride, rows, V, d_tokens, temperature, top_k)) return LB_ERR_ARG;
    const int64_t chunk = LP_THREADS * 8 * (dtype == DT_F32 ? 4 : 8);
    if (!d_stats || ((uintptr_t)d_stats & 15) || !d_grad || ((uintptr_t)d_grad & (dtype == DT_F32 ? 3 : 1)) || grad_row_stride < V || (top_k && !d_top_ids) ||
        rows * ((V + chunk - 1) / chunk) > 0x7fffffffll) {
        set_error(LB_ERR_ARG, "%s: bad argument (rows %lld, vocabulary %lld, gradient stride %lld)", name, (long long)rows, (long long)V, (long long)grad_row_stride);
        return LB_ERR_ARG;
    }
    const LogprobGradArgs A = {d_logits, row_stride, rows, (int)V, d_tokens, LP_LOG2E / temperature, 1.0f / temperature, top_k, d_top_ids, d_g_logprobs, d_g_entropy, d_g_top,
                               (const float4*)d_stats, d_grad, grad_row_stride, 0, 0};
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == DT_F32 ? grad_launch<float>(A, st) : dtype == DT_F16 ? grad_launch<__half>(A, st) : grad_launch<__nv_bfloat16>(A, st);
}
