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

// Probabilities are kept relative to a reference that follows a row's maximum when that grew by more than 2^P_GROW, and in fp16 2^P_LIFT above their
// place (the division by their sum, which has it too, takes it out): a ratio to the reference from 2^-25 to 2^4 is a normal number, below that the
// two parts that enter the product share fp16's last bit, 2^-24, so that a key is off by at most 2^-36 of the reference.  Without, a key 2^-14 below the
// largest lost bits and one 2^-25 below all of them, while the sum counted both.  bf16 has the range of 32 bits.
constexpr float P_GROW = 4.0f, P_LIFT = 11.0f;                // 2^(4 + 11) < 65504

// two values rounded to 16 bits, and what that left.  bf16 by the multiply-add that takes a 16-bit factor, without unpacking (a chunk of 512 behind 16000
// keys 181 us, 188 without); fp16's conversions cost nothing more as they are
template <bool BF> __device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    if (BF) asm("{\n\t.reg .b16 p, q, m;\n\t.reg .f32 a, b;\n\t"
                "cvt.rn.bf16x2.f32 %0, %3, %2;\n\t"
                "mov.b32 {p, q}, %0;\n\t"
                "mov.b16 m, 0xbf80;\n\t"
                "fma.rn.f32.bf16 a, p, m, %2;\n\t"
                "fma.rn.f32.bf16 b, q, m, %3;\n\t"
                "cvt.rn.bf16x2.f32 %1, b, a;\n\t}" : "=&r"(hi), "=r"(lo) : "f"(x), "f"(y));
    else {
        const __half2 h = __floats2half2_rn(x, y);
        const __half2 l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
        hi = *reinterpret_cast<const uint32_t*>(&h);
        lo = *reinterpret_cast<const uint32_t*>(&l);
    }
}

// a request's tokens, whatever the lists on the device say: nothing outside q and the table is ever addressed
struct PagedReq { int64_t q0; int n, len; };
__device__ __forceinline__ PagedReq paged_req(const PagedAttnArgs& A, int r) {
    PagedReq q;
    const int64_t a = A.cu[r], b = A.cu[r + 1];
    q.q0 = a < 0 ? 0 : a > A.T ? A.T : a;
    const int64_t e = b < q.q0 ? q.q0 : b > A.T ? A.T : b;
    q.n = (int)(e - q.q0);
    if (A.table) {
        // tokens behind row T are not there, and the others see what they would with them
        const int64_t held = A.seq_lens[r] - (b > A.T ? b - (a > A.T ? a : A.T) : 0), most = (int64_t)A.width * A.page_size;
        // more than its row of the table can name: every token sees the first key without a page
        const int64_t len = held > most ? most + q.n : held;
        q.len = (int)(len < 0 ? 0 : len > 0x7fffffff ? 0x7fffffff : len);
    } else q.len = q.n;
    return q;
}

// the page of a request's key, -1 behind the table's width
__device__ __forceinline__ int paged_page(const PagedAttnArgs& A, int r, int key) {
    const int c = key / A.page_size;
    return c < A.width ? A.table[r * A.table_stride + c] : -1;
}

// paged_prompt.cu: requests with more than `above` rows (new tokens x heads of a group) a kv head
int paged_prompt_max_group(int D);
size_t paged_prompt_part_bytes(int D);
int paged_prompt_launch(PagedAttnArgs A, int above, cudaStream_t st);

// ---- work in equal shares.  The tiles of all units (a request's kv head; or a block of its rows on one) lie behind one another, n of them
// in all, and block c of C takes tiles c n / C .. (c + 1) n / C: whatever the lengths, every block reads as many.  A unit whose tiles
// lie in several blocks leaves its sums there, each block's slot 1 for a unit that began in it and slot 0 for one that did not, and a note
// in the block that it began in; the merge adds them up in the order of the keys.
// Divisions are written out in 32 bits: a 64-bit one is a call, and a kernel that calls anything keeps the registers of its launch
// (setmaxnreg is ignored).
__device__ __forceinline__ uint64_t div_small(uint64_t n, uint32_t d, uint32_t& rem) {      // d < 2^16, 16 bits at a time
    uint64_t q = 0;
    uint32_t r = 0;
#pragma unroll
    for (int i = 48; i >= 0; i -= 16) {
        const uint32_t x = r << 16 | ((uint32_t)(n >> i) & 0xffffu);
        q = q << 16 | x / d;
        r = x % d;
    }
    rem = r;
    return q;
}
__device__ __forceinline__ int64_t share_begin(int64_t n, int c, int C) {
    if (n < 1 << 20) return (uint32_t)n * (uint32_t)c / (uint32_t)C;                        // C is at most some thousands
    uint32_t rem;
    const uint64_t q = div_small((uint64_t)n, (uint32_t)C, rem);
    return (int64_t)q * c + rem * (uint32_t)c / (uint32_t)C;
}
__device__ __forceinline__ int share_of(int64_t tile, int64_t n, int C) {                   // the block that takes a tile
    int c = min(C - 1, (int)(__fdividef((float)tile, (float)n) * (float)C));
    while (c > 0 && share_begin(n, c, C) > tile) c--;
    while (c + 1 < C && share_begin(n, c + 1, C) <= tile) c++;
    return c;
}
__device__ __forceinline__ int div_few(int64_t x, int64_t y, int64_t& rem) {                // a quotient of a few thousand at most
    int q = (int)__fdividef((float)x, (float)y);
    while (q > 0 && q * y > x) q--;
    while ((q + 1) * y <= x) q++;
    rem = x - q * y;
    return q;
}

// blocks that share n places: none takes fewer than `least`
__device__ __forceinline__ int sharers(int64_t n, int least, int C) { return n < (int64_t)least * C ? max((int)n / least, 1) : C; }

// Of block c: the unit that began in it and goes on in others, to block `end`.  Rows are (token, head of the group).  The merge could find all
// this out from the lists, but starts when the block's registers are free, and then every clock counts
struct __align__(16) SplitNote { int rows, hk, end, unused; int64_t q0, unused2; };     // rows 0: there is none
// b of the unit's tiles were in block c
__device__ __forceinline__ SplitNote split_note(int rows, int hk, int64_t q0, int b, int tiles, int64_t all, int c, int C) {
    return {rows, hk, share_of(share_begin(all, c + 1, C) - b + tiles - 1, all, C), 0, q0, 0};
}

// sum over the block before this thread, and of all of it
__device__ __forceinline__ int64_t block_before(int64_t x, int64_t* warps, int64_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = (blockDim.x + 31) >> 5;
    int64_t s = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, s, d);
        if (lane >= d) s += y;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < n; w++) {
        if (w < warp) before += warps[w];
        total += warps[w];
    }
    return before + s - x;
}
// the whole block: tiles of all requests (count(r) of request r), and the request that holds tile `pick(total)` with the tiles before it.
// Two walks over the requests when they are more than the threads; one loop for both, since a block waits for this code to be fetched
// before its first copy
template <typename Count, typename Pick>
__device__ __forceinline__ int64_t find_tile(int R, Count count, Pick pick, int64_t* warps, int* r_out, int64_t* before_out) {
    int64_t all = 0, sum = 0, want = -1;
    const bool twice = R > (int)blockDim.x;
#pragma unroll 1
    for (int walk = twice ? 0 : 1; walk < 2; walk++) {
        sum = 0;
#pragma unroll 1
        for (int r0 = 0; r0 < R; r0 += blockDim.x) {
            const int r = r0 + threadIdx.x;
            int64_t total;
            const int64_t mine = r < R ? count(r) : 0;
            const int64_t first = sum + block_before(mine, warps, total);
            sum += total;
            if (!twice && sum > 0) want = pick(sum);
            if (mine > 0 && first <= want && want < first + mine) { *r_out = r; *before_out = first; }
        }
        all = sum;
        if (walk == 0 && all > 0) want = pick(all);
    }
    __syncthreads();
    return all;
}

}  // namespace lowbit
