// logprobs.cu -- what a row of logits says about its tokens, and the gradient of that.  With z the row divided by the temperature:
//   log p_i = z_i - log sum_j exp z_j,      H = - sum_j p_j log p_j,      the k largest logits in order, the lower index first where two are equal;
//   dL/dz_i = sum_m g_m [i = i_m] - p_i (sum_m g_m + g_H (log p_i + H))    over the given token and the alternatives m.
// One pass over the row: exponentials and their sums in 32 bits relative to a maximum that runs along.  The k largest cost that pass nothing but a maximum
// a thread: at least k elements are not below the k-th largest of the threads' maxima, so the k largest lie in the strips of the threads whose
// maximum reaches it, some k of them, and those are read again from L2.  Where masks leave too few numbers for that, all strips are.
#include "lowbit_common.cuh"
#include "lowbit_internal.h"

using namespace lowbit;

namespace lowbit {
namespace {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_MOST = 32, LP_ROOM = 512, LP_RESIDENT = 5;
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;

struct LogprobArgs {
    const void* logits; int64_t row; int64_t rows; int V;
    const int64_t* tokens; float c, by;                       // c = log2 e / temperature, by = 1 / temperature
    int k;
    float *logp, *entropy; int64_t* ids; float* top; float4* stats;
};
// A row's stats, for the gradient: ref and m of an element's exponent u = (x - ref) c - m, base 2 (ref is 0 but in rows whose products pass 32 bits);
// the sum of the powers; the mean of the exponents under them

// 16 bytes of logits.  floored: none below kFloor, so that the product of a power of 0 with its exponent is 0; fp16 has no number that is low enough at
// every temperature, and its exponents are bounded one by one (kBound)
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static constexpr float kFloor = -1e30f;
    static constexpr bool kBound = false;
    static __device__ __forceinline__ void get(const uint4& w, float (&x)[4]) { x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w); }
    static __device__ __forceinline__ void floored(const uint4& w, float (&x)[4]) {
        get(w, x);
#pragma unroll
        for (int i = 0; i < 4; i++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(x[i]) : "f"(kFloor));
    }
};
template <> struct Vec<__half> {
    static constexpr int N = 8;
    static constexpr float kFloor = -INFINITY;
    static constexpr bool kBound = true;
    static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(v + i)); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ void floored(const uint4& w, float (&x)[8]) { get(w, x); }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr float kFloor = -0x1.92p99f;               // -1e30 in its 16 bits, 0xf149
    static constexpr bool kBound = false;
    static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(v[i] << 16); x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ void floored(uint4 w, float (&x)[8]) {
        uint32_t* const v[4] = {&w.x, &w.y, &w.z, &w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(*v[i]) : "r"(0xf149f149u));
        get(w, x);
    }
};

// two 32-bit numbers by one instruction
struct Two { uint64_t v; };
__device__ __forceinline__ Two two(float a, float b) { Two r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void apart(Two x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ Two fma(Two a, Two b, Two c) { Two r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ Two add(Two a, Two b) { Two r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }

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

// a reference for exponents, the sum of powers, and of powers x exponents, relative to it
struct __align__(16) Sums { float m, s, d; };
// those of the first `lanes` (a power of two) lanes together, in every one of them the same
__device__ __forceinline__ Sums together(Sums x, int lanes) {
    float m = x.m;
    for (int d = lanes / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    // a lane that holds nothing has m = -inf, and one whose weight is 0 holds nothing that counts, but for NaN
    const float a = x.m - m, w = x.m == -INFINITY ? 0.0f : ex2(a);
    x.d = w == 0.0f ? 0.0f : w * fmaf(x.s, a, x.d);
    x.s = w != 0.0f ? w * x.s : x.s == x.s ? 0.0f : x.s;
    for (int d = lanes / 2; d; d >>= 1) {
        x.s += __shfl_xor_sync(0xffffffffu, x.s, d);
        x.d += __shfl_xor_sync(0xffffffffu, x.d, d);
    }
    x.m = m;
    return x;
}

// order of the alternatives: larger value first, then lower index.  -0 equals 0; key 0 is nobody's
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.0f), o = (int)b < 0 ? ~b : b | 0x80000000u;
    return (uint64_t)o << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float key_value(uint64_t k) { const uint32_t o = (uint32_t)(k >> 32); return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
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

// a value that k threads reach at least, and so k elements: the least of the k / full-th largest values (rounded up) of the first `full` warps
__device__ __forceinline__ float reached_by(float x, int k, int full, uint32_t* warps) {
    if (full == 0) return -INFINITY;
    const int lane = threadIdx.x & 31;
    const uint32_t b = __float_as_uint(x + 0.0f);
    uint32_t key = (int)b < 0 ? ~b : b | 0x80000000u, top = 0;
    for (int left = (k + full - 1) / full; left; left--) {
        top = __reduce_max_sync(0xffffffffu, key);
        const uint32_t has = __ballot_sync(0xffffffffu, key == top);
        if (lane == __ffs(has) - 1) key = 0;
    }
    if (lane == 0) warps[threadIdx.x >> 5] = top;
    __syncthreads();
    uint32_t least = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < LP_WARPS; w++) least = w < full ? min(least, warps[w]) : least;
    return __uint_as_float(least & 0x80000000u ? least & 0x7fffffffu : ~least);
}

// Blocks of a cluster share a row; the first one finishes it.
// What bounds it: instructions and memory alike where rows are many (4001 rows of 32000 bf16 logits, 256 MB: 51 us, 5.0 TB/s, at
// 31.5 million instructions of warps; 63 us at 51 million, before two exponents went by one instruction and the
// floor was one maximum of two), and for few what comes behind the pass: 256 rows of 128256 with 20 alternatives take 26.9 us, 16 of them the pass, the rest
// the threshold, the strips and the sorts, some 7000 cycles, one after the other.  One row of 32000: 6.3 us.
// 256 rows of 128256 of which masks leave 100 tokens or fewer: 164 us with 20 alternatives, 18 with none.
template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, LP_RESIDENT) token_logprobs_kernel(const LogprobArgs A) {
    constexpr int N = Vec<T>::N;
    __shared__ Sums warps[LP_WARPS];
    __shared__ Sums mine;                                      // read by the cluster's first block
    __shared__ uint64_t found[TOP ? LP_ROOM : 1];
    __shared__ uint64_t lists[TOP ? LP_WARPS : 1][32];
    __shared__ uint64_t best[32];                              // as `mine`
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

    int64_t token = -1;                                        // the first thread's, asked for ahead: it leads to another load
    float token_logit = 0.0f;
    if (rank == 0 && t == 0) {
        token = A.tokens[r];
        if (token >= 0 && token < A.V) token_logit = one(row + token);
        else token = -1;
    }
    // ---- the pass
    float m = -INFINITY, big = -INFINITY;                      // the reference; this thread's largest logit
    Two sum = two(0.0f, 0.0f), dot = sum;                      // of powers, and of powers x exponents
    const Two c2 = two(c, c);
    auto follow = [&]() {
        // the reference follows where an exponent would pass 2^4 of it: rarely, and what the sums lose by it is four bits of their distance from 1
        const float top = big * c;
        if (top > m + 4.0f && big > Vec<T>::kFloor) {
            const float a = m - top, w = ex2(a);
            if (w == 0.0f) {
                // nothing that counts so far.  (The exponents of logits beyond 2^24 have lost their differences: whatever they gave goes, but for NaN)
                float p, q;
                apart(sum, p, q);
                sum = two(p == p ? 0.0f : p, q == q ? 0.0f : q);
                dot = two(0.0f, 0.0f);
            } else {
                const Two w2 = two(w, w);
                dot = fma(w2, fma(sum, two(a, a), dot), two(0.0f, 0.0f));
                sum = fma(w2, sum, two(0.0f, 0.0f));
            }
            m = top;
        }
        return m == -INFINITY ? 0.0f : -m;                     // nothing above the floor so far
    };
    auto take = [&](const float* v, int n) {                   // n: a constant
#pragma unroll
        for (int i = 0; i < n; i += 2) big = max3(big, v[i], v[i + 1]);
        const float r0 = follow();
        const Two ref = two(r0, r0);
#pragma unroll
        for (int i = 0; i < n; i += 2) {
            Two u = fma(two(v[i], v[i + 1]), c2, ref);
            float a, b;
            apart(u, a, b);
            const Two e = two(ex2(a), ex2(b));
            if (Vec<T>::kBound) u = two(fmaxf(a, -300.0f), fmaxf(b, -300.0f));
            sum = add(sum, e);
            dot = fma(e, u, dot);
        }
    };
    constexpr int AHEAD = 4;
    int next = strip.first + t;
#pragma unroll 1
    for (; next + (AHEAD - 1) * LP_THREADS < strip.last; next += AHEAD * LP_THREADS) {
        uint4 w[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) w[a] = strip.piece(next + a * LP_THREADS);
#pragma unroll
        for (int a = 0; a < AHEAD; a += 2) {
            float v[2 * N];
            Vec<T>::floored(w[a], *reinterpret_cast<float(*)[N]>(v));
            Vec<T>::floored(w[a + 1], *reinterpret_cast<float(*)[N]>(v + N));
            take(v, 2 * N);
        }
    }
    {
        // what is left of the pieces, asked for at once
        uint4 w[AHEAD - 1];
#pragma unroll
        for (int a = 0; a < AHEAD - 1; a++)
            if (next + a * LP_THREADS < strip.last) w[a] = strip.piece(next + a * LP_THREADS);
#pragma unroll 1
        for (int a = 0; a < AHEAD - 1; a++) {
            if (next + a * LP_THREADS >= strip.last) break;
            float v[N];
            Vec<T>::floored(a == 0 ? w[0] : a == 1 ? w[1] : w[2], v);
            take(v, N);
        }
    }
    const int end = strip.end_of(t);
    if (end >= 0) {
        float v = one(row + end);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(Vec<T>::kFloor));
        big = fmaxf(big, v);
        const float u = fmaf(v, c, follow()), e = ex2(u);
        sum = add(sum, two(e, 0.0f));
        dot = add(dot, two(e * (Vec<T>::kBound ? fmaxf(u, -300.0f) : u), 0.0f));
    }

    // ---- the block's sums, and the cluster's
    Sums x = {m, 0.0f, 0.0f};
    {
        float a, b;
        apart(sum, a, b);
        x.s = a + b;
        apart(dot, a, b);
        x.d = a + b;
    }
    x = together(x, 32);
    if (lane == 0) warps[warp] = x;
    if (t == 0) n_found = 0;

    if (TOP) {
        // ---- the strips in which the k largest lie, read again
        const float reached = reached_by(big, A.k, min(strip.last - strip.first, LP_THREADS) / 32, owners);
        const float floor_ = reached > Vec<T>::kFloor ? reached : -INFINITY;                   // what is below the floor was read as that
        __syncthreads();                                       // everybody has read the warps' values
        const uint32_t own = __ballot_sync(0xffffffffu, big >= floor_);
        if (lane == 0) owners[warp] = own;
        __syncthreads();
        int strips = 0, before = 0;
#pragma unroll
        for (int w = 0; w < LP_WARPS; w++) { const int c_ = __popc(owners[w]); strips += c_; before += w < warp ? c_ : 0; }
        if (own >> lane & 1) owner[before + __popc(own & ((1u << lane) - 1u))] = (uint8_t)t;
        __syncthreads();
        auto note = [&](int at) {
            const int slot = atomicAdd(&n_found, 1);           // their order does not matter: they are sorted
            if (slot < LP_ROOM) found[slot] = key_of(one(row + at), (uint32_t)at);
        };
        const int deep = (strip.last - strip.first + LP_THREADS - 1) / LP_THREADS;             // pieces of a strip
#pragma unroll 1
        for (int i = t; i < strips * deep; i += 2 * LP_THREADS) {
            uint4 w[2];
            int p[2];
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const int u = i + a * LP_THREADS, s = u / deep;
                p[a] = s < strips ? strip.first + owner[s] + (u - s * deep) * LP_THREADS : strip.last;
                if (p[a] < strip.last) w[a] = strip.piece(p[a]);
            }
            uint32_t hits = 0;
#pragma unroll
            for (int a = 0; a < 2; a++)
                if (p[a] < strip.last) {
                    float v[N];
                    Vec<T>::get(w[a], v);
#pragma unroll
                    for (int e = 0; e < N; e++) hits |= v[e] >= floor_ ? 1u << (8 * a + e) : 0u;
                }
#pragma unroll 1
            for (; hits; hits &= hits - 1) {
                const int e = __ffs(hits) - 1;
                note(strip.base() + (e < 8 ? p[0] : p[1]) * N + (e & 7));
            }
        }
        if (end >= 0 && one(row + end) >= floor_) note(end);
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
        // the lists of as many warps as have one, to the first
        const int n_lists = n <= LP_ROOM ? min((n + 31) / 32, LP_WARPS) : LP_WARPS;
        if (n_lists > 1) {
            lists[warp][lane] = key;
            __syncthreads();
            if (warp == 0)
                for (int w = 1; w < n_lists; w++) key = merge32(key, lists[w][lane]);
        }
        if (warp == 0) best[lane] = key;
    } else __syncthreads();
    if (warp == 0) {
        x = together(lane < LP_WARPS ? warps[lane] : Sums{-INFINITY, 0.0f, 0.0f}, LP_WARPS);
        if (lane == 0) mine = x;
    }
    __syncthreads();
    if (blocks > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (rank == 0) {
        // the first block: the others' sums and lists, a warp each
        uint64_t key = 0;
        Sums all = mine;
        if (blocks > 1) {
            if (warp < (int)blocks) {
                const uint32_t at_mine = (uint32_t)__cvta_generic_to_shared(&mine), at_best = (uint32_t)__cvta_generic_to_shared(&best[lane]);
                uint32_t p;
                if (lane == 0) {
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(at_mine), "r"(warp));
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(all.m), "=f"(all.s) : "r"(p) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1 + 8];" : "=f"(all.d) : "r"(p) : "memory");
                    warps[warp] = all;
                }
                if (TOP) {
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(at_best), "r"(warp));
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(p) : "memory");
                    lists[warp][lane] = key;
                }
            }
            __syncthreads();
            if (TOP) {
#pragma unroll
                for (int h = 4; h; h >>= 1) {
                    if (warp < h && warp + h < (int)blocks) {
                        key = merge32(key, lists[warp + h][lane]);
                        lists[warp][lane] = key;
                    }
                    __syncthreads();
                }
            }
            all = together(lane < (int)blocks ? warps[lane] : Sums{-INFINITY, 0.0f, 0.0f}, LP_WARPS);
            all = {__shfl_sync(0xffffffffu, all.m, 0), __shfl_sync(0xffffffffu, all.s, 0), __shfl_sync(0xffffffffu, all.d, 0)};
        } else if (TOP) key = best[lane];
        float ref = 0.0f;
        if (!(fabsf(all.m) < 16777216.0f)) {
            // the products have lost the logits' differences, or passed 32 bits: the row twice more, the largest logit taken off first.  A row of the
            // type's lowest value is even; one of -inf alone, or with inf in it, has no probabilities
            for (int j = t; j < A.V; j += LP_THREADS) ref = j == t ? one(row + j) : fmaxf(ref, one(row + j));
            if (t >= A.V) ref = -INFINITY;
#pragma unroll
            for (int h = 16; h; h >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, h));
            __syncthreads();                                   // everybody has read the warps' sums
            if (lane == 0) warps[warp].m = ref;
            __syncthreads();
            for (int w = 0; w < LP_WARPS; w++) ref = fmaxf(ref, warps[w].m);
            float s = fabsf(ref) < INFINITY ? 0.0f : NAN, d = 0.0f;
            for (int j = t; j < A.V; j += LP_THREADS) {
                const float a = (one(row + j) - ref) * c, e = ex2(a);
                s += e;
                d = fmaf(e, fmaxf(a, -300.0f), d);
            }
#pragma unroll
            for (int h = 16; h; h >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, h); d += __shfl_xor_sync(0xffffffffu, d, h); }
            __syncthreads();                                   // everybody has read the warps' sums
            if (lane == 0) warps[warp] = {0.0f, s, d};
            __syncthreads();
            all = {0.0f, 0.0f, 0.0f};
            for (int w = 0; w < LP_WARPS; w++) { all.s += warps[w].s; all.d += warps[w].d; }
        }
        const float log2s = log2f(all.s);
        auto logp = [&](float v) {
            const float d = v - ref, u = fmaf(d, c, -all.m);
            if (u > -INFINITY || u != u) return (u - log2s) * LP_LN2;
            // the type's lowest value: base e has room for what base 2 has not, and the quotients by the temperature for what their difference has not
            return (d > -INFINITY ? d * A.by : fmaf(v, A.by, -(ref * A.by))) - (all.m + log2s) * LP_LN2;
        };
        if (t == 0) {
            A.logp[r] = token >= 0 ? logp(token_logit) : 0.0f;
            A.entropy[r] = (log2s - all.d / all.s) * LP_LN2;
            if (A.stats) A.stats[r] = make_float4(ref, all.m, all.s, all.d / all.s);
        }
        if (TOP && t < A.k) {
            A.ids[r * A.k + t] = key ? (int64_t)key_index(key) : -1;       // a row with fewer numbers than that
            A.top[r * A.k + t] = key ? logp(key_value(key)) : NAN;
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

// A piece of a row a block; the elements that the row's tokens name are written over at the end, by a thread each.  It reads the logits once and writes their
// gradient: 4001 rows of 32000 bf16 logits, 512 MB in all, 79 us, 6.5 TB/s.
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
    const bool bad = !logits || dtype < 0 || dtype > 2 || rows < 0 || V <= 0 || V > 0x7fff0000ll || row_stride < V || !tokens || !(temperature >= 0.99e-7f) || !(temperature <= 1.01e7f) ||
                     k < 0 || k > LP_MOST || k > V || rows > 0x3ffffffll || ((uintptr_t)logits & (dtype == DT_F32 ? 3 : 1));
    if (bad) set_error(LB_ERR_ARG, "%s: bad argument (rows %lld, vocabulary %lld, dtype %d, top_k %d)", name, (long long)rows, (long long)V, dtype, k);
    return bad;
}

template <typename T> int logprobs_launch(const LogprobArgs& A, cudaStream_t st) {
    // blocks of a row, each with a piece a thread at least: of the numbers with which all are resident at once the one that leaves the fewest places empty
    // (256 rows of 128256 by 1, 2, 3 and 4 blocks: 39, 27, 29 and 36 us)
    int64_t blocks = 1, most = A.V / (LP_THREADS * Vec<T>::N);
    double best = 0.0;
    for (int64_t b = 1; b <= 8 && (b == 1 || b <= most) && (b == 1 || A.rows * b <= (int64_t)LP_RESIDENT * sm_count()); b++) {
        const int64_t n = A.rows * b, deep = (n + sm_count() - 1) / sm_count();
        const double used = (double)n / (double)(deep * sm_count());
        if (used >= best) { best = used; blocks = b; }
    }
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
    // a block's piece: 8 of 16 bytes a thread; whole pieces, so that only a row's ends lie on none
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
