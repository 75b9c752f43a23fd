// paged_prompt.cu -- attention of many rows: chunks of prompts over a paged cache, and packed prompts over themselves.
//
// A unit is NT tiles of 128 rows of one kv head; a request's rows there are (new token, head of the group), tokens first, so that all heads
// that share a kv head share every key that is read.  Keys come in tiles of 128:
//   S_t = Q_t . K^T   tcgen05.mma M = 128, N = 128, both operands in shared memory, S in tensor memory (lane = row);
//   softmax           four warps a tile, a thread per row: the maximum in one reading of the row's 128 scores, exp2 in another, 64 in registers at
//                     a time, P back into tensor memory over S;
//   O_t += P_t . V    A operand = P in tensor memory, B operand = V as it lies in the cache (rows = keys: the MN-major descriptor).
// Warps 0 .. 4 NT - 1: softmax; the next four copy keys and values into a ring of 128-byte swizzled tiles (TMA, a box per run of rows in a page;
// rows behind the last key and pages without boxes by cp.async; e5m2 bytes spread to fp16 in their slot); the next one issues the MMAs and owns the
// tensor memory.
// Two tiles alternate: one's products run while the other is in its softmax.  The blocks share the key tiles of all units equally (paged.h).
// P enters P . V as two 16-bit values, the second with what the rounding of the first left, and both multiply V: only the result is rounded
// (fp16's range: P_LIFT in paged.h).  With one value an output added up to sqrt(2) of the error that rounding the output alone leaves; one value / two: the 8
// prompts below 223 / 268 us, the long one 545 / 690, the chunk 155 / 181.
// What bounds it: a tile's chain in a step of 256 rows and 128 keys, 5200 clocks: its softmax 3400 (maximum 570, exponentials and both parts of P 2800, while the
// other tile's warps are in theirs), P V of the last 64 keys 790, Q K of the next ones 790; 32768 exponentials need 2048 clocks of a step, the MMAs of both
// tiles 6 x 512 (tensor pipe 48 %, issue slots 46 %).  8 prompts of 200 to 4000 tokens, 32 heads on 8, bf16: 268 us, 564 TFLOP/s, each product counted once; one
// of 8000, 32 heads, fp16: 690 us, 760 TFLOP/s (820 us in a long loop, under the power cap); 512 tokens behind 16000 keys, 32 on 8, bf16: 181 us, 752 TFLOP/s,
// over e5m2 pages 272 us.  With TMA / without: 269 / 291, 698 / 746, 181 / 261 us.
#include <string.h>
#include "paged.h"
#include "tc_common.cuh"

using namespace lowbit;
using namespace lowbit::gemmtc;

namespace lowbit {
namespace {

constexpr int PR_KEYS = 128;

template <int DP, bool E5M2> struct Prompt {
    static constexpr int NT = DP == 256 ? 1 : 2, kRows = 128 * NT;
    static constexpr int kTile = 128 * DP * 2, kSlots = DP == 256 ? 2 : DP == 128 ? 4 : 8;
    static constexpr int kWarps = 4 * NT + 8;
    static constexpr int kStageAt = (NT + kSlots) * kTile + 512;
    static constexpr int kSmem = 1024 + kStageAt + 4 * NT * 4096;          // 4 KB a softmax warp for results on their way out
    // registers a thread: softmax, copies, MMAs (the launch's are 128 or 168)
    static constexpr int kSoftRegs = NT == 2 ? 152 : 232, kCopyRegs = NT == 2 ? 104 : 144, kMmaRegs = NT == 2 ? 104 : 128;
    static constexpr int64_t kPart = (int64_t)NT * 128 * (DP + 2);     // floats of a slot: [t][DP / 4][128] float4, [t][128] float2
};

__device__ __forceinline__ void tmem_ld32x(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16x(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16x(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// A operand in tensor memory
__device__ __forceinline__ void umma_ts_w(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void sts4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
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
template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// ------------------------------------------------------------------ the units and their key tiles
// sum of floor((a i + b) / 128) over i = 0 .. n - 1, by the Euclidean exchange of a and the divisor; the first step, by 128, needs no division
__device__ __forceinline__ int64_t floor_sum128(uint32_t n, uint32_t a, uint32_t b) {
    if (n == 0) return 0;
    int64_t s = (int64_t)n * (n - 1) / 2 * (a >> 7) + (int64_t)n * (b >> 7);
    a &= 127u; b &= 127u;
    uint32_t y = a * n + b, m = 128;                                   // at most the tokens of a request
    while (y >= m) {
        n = y / m;
        b = y - n * m;
        const uint32_t h = m; m = a; a = h;
        const uint32_t qa = a / m, qb = b / m;
        s += (int64_t)n * (n - 1) / 2 * qa + (int64_t)n * qb;
        a -= qa * m;
        b -= qb * m;
        y = a * n + b;
    }
    return s;
}
// What a unit costs beside its key tiles (queries, result, a pipeline that drains), in tiles: shares are taken of places, PR_EXTRA of them in
// front of a unit's tiles, so that blocks with many short prompts are not the last.  0 / 1 / 2 / 3: the 8 prompts above 377 / 291 / 269 / 270 us, 7
// of 17 to 300 tokens 26.4 / 19.4 / 18.6 / 18.0, 40 requests with chunks to 300 and tokens over e5m2 pages 129 / 111 / 113 / 118
constexpr int PR_EXTRA = 2;
// A unit of up to so many key tiles is never split: it is the block's in whose share it begins.  A part costs a store and a load of its 32-bit
// sums (128 KB a unit) and its merge, more than such a unit is worth.  0 / 2 / 4 / 8: 7 prompts of 17 to 300 tokens 22.1 / 18.6 / 18.6 / 18.7 us, 8
// of 400 60 / 61 / 54 / 54, 20 of 500 143 / 144 / 131 / 131, one of 2000 with 4 heads on one 29.7 / 29.8 / 32.0 / 40.8, the 40 requests 113 / 113 / 113 / 121
constexpr int PR_WHOLE = 4;
struct Units {
    int n, units, tpu, causal, off, len;                      // new tokens, units, tokens of a unit; keys before the first new token
    __device__ __forceinline__ Units(const PagedReq& q, int group, int rows, int causal_, int above) {
        tpu = rows / group;
        causal = causal_;
        n = (int64_t)q.n * group > above ? q.n : 0;
        units = n > 0 ? (n - 1) / tpu + 1 : 0;
        len = q.len;
        off = q.len - q.n;
    }
    // key tiles of unit u: one at least, so that rows without keys are written too
    __device__ __forceinline__ int tiles(int u) const {
        const int end = causal ? off + min((u + 1) * tpu, n) : len;
        return end <= PR_KEYS ? 1 : (end - 1) / PR_KEYS + 1;
    }
    // places of the first u units
    __device__ __forceinline__ int64_t before(int u) const { return tiles_before(u) + (int64_t)min(u, units) * PR_EXTRA; }
    __device__ __forceinline__ int64_t tiles_before(int u) const {
        if (u <= 0) return 0;
        if (!causal) return (int64_t)u * tiles(0);
        const int last = u >= units ? tiles(units - 1) : 0;            // which may have fewer tokens
        if (u >= units) u = units - 1;
        // those whose last token has at most PR_KEYS keys count one each: (i + 1) tpu + off <= PR_KEYS
        const int room = PR_KEYS - off, ones = room < tpu ? 0 : min(u, room / tpu);
        return last + ones + floor_sum128(u - ones, tpu, (uint32_t)off + (uint32_t)(ones + 1) * tpu + PR_KEYS - 1);
    }
};
// a block's way through its share: pieces of units, key tiles a .. b - 1 of unit (r, hk, u)
struct PromptAt {
    PagedReq q; int r, hk, u, units, tpu, a, b, tiles, left;
    __device__ __forceinline__ bool piece(const PagedAttnArgs& A, int group, int rows, int above, int place) {
        const Units w(q, group, rows, A.causal, above);
        tiles = w.tiles(u);
        const int rest = tiles + PR_EXTRA - place, take = tiles <= PR_WHOLE ? rest : min(rest, left);
        left -= take;
        a = max(place - PR_EXTRA, 0);
        b = max(place + take - PR_EXTRA, 0);
        return a < b && (place == 0 || tiles > PR_WHOLE);
    }
    __device__ __forceinline__ bool next(const PagedAttnArgs& A, int group, int rows, int above) {
        while (left > 0) {
            if (++u >= units) {
                u = 0;
                if (++hk >= A.Hkv) {
                    hk = 0;
                    do {
                        if (++r >= A.R) return false;
                        q = paged_req(A, r);
                        units = Units(q, group, rows, A.causal, above).units;
                    } while (units == 0);
                }
            }
            if (piece(A, group, rows, above, 0)) return true;
        }
        return false;
    }
    // key tiles that the rows of tile t need, and whether the piece has any of them
    __device__ __forceinline__ int tiles_of(const PagedAttnArgs& A, int group, int t) const {
        const int first = u * tpu, end = min(first + tpu, q.n);
        if (128 * t / group >= end - first) return 0;
        const int last = min(first + (128 * t + 127) / group + 1, end);
        const int keys = A.causal ? q.len - q.n + last : q.len;
        return keys <= 0 ? 0 : (keys - 1) / PR_KEYS + 1;
    }
};
// places that a block takes at least.  1 / 3 / 6: a prompt of 2000 tokens, 4 heads on one 33.2 / 32.0 / 34.3 us, seven of 17 to 300 tokens 18.7 / 18.6 / 26.6, one of
// 100, 8 heads, 13.3 / 12.6 / 18.3
constexpr int PR_LEAST = 3;

// the whole block: where place `pick` of all lies (`place` of its unit); `all` = places of all units
template <typename Pick>
__device__ __forceinline__ int64_t open_share(const PagedAttnArgs& A, int group, int rows, int above, Pick pick, int64_t* scan, int* found_r, int64_t* found_before, PromptAt& at, int& place) {
    int64_t want = 0;
    const int64_t all = find_tile(A.R, [&](int r) { const Units w(paged_req(A, r), group, rows, A.causal, above); return w.before(w.units) * A.Hkv; },
                                  [&](int64_t n) { return want = pick(n); }, scan, found_r, found_before);
    if (all == 0 || want < 0) return all;
    at.r = *found_r;
    at.q = paged_req(A, at.r);
    const Units w(at.q, group, rows, A.causal, above);
    at.units = w.units;
    at.tpu = w.tpu;
    const int64_t per = w.before(w.units), x = want - *found_before;
    int64_t y;
    at.hk = div_few(x, per, y);
    // the last unit that begins at y or before.  Places up to unit u grow with u^2: the 32 units around the root of that are looked at first,
    // one a lane, and 32 places of what is left at a time if it is none of them
    int lo = 0, hi = w.units, from = 0, step = 1;                      // before(lo) <= y < before(hi)
    int64_t reached = 0;                                               // before(lo)
    if (hi > 32) {
        const float q = A.causal ? w.tpu / 256.0f : 0.0f, l = PR_EXTRA + 0.5f + (A.causal ? (w.off + 0.5f * w.tpu) / PR_KEYS : (float)w.tiles(0) - 0.5f);
        const float root = q > 0.0f ? (sqrtf(fmaxf(l * l + 4.0f * q * (float)y, 0.0f)) - l) / (2.0f * q) : (float)y / l;
        from = max(0, min(hi - 32, (int)root - 16));
    }
#pragma unroll 1
    do {
        const int u = from + step * (int)(threadIdx.x & 31);
        const int64_t mine = w.before(u);
        const uint32_t yes = __ballot_sync(0xffffffffu, u < hi && mine <= y);
        if (yes) {
            const int l = 31 - __clz(yes);
            lo = from + step * l;
            reached = __shfl_sync(0xffffffffu, mine, l);
            if (l < 31) hi = min(hi, lo + step);
        } else hi = from;
        from = lo;
        step = (hi - lo + 31) / 32;
    } while (hi - lo > 1);
    at.u = lo;
    place = (int)(y - reached);
    return all;
}

template <int DP, bool E5M2> __device__ __forceinline__ SplitNote* prompt_notes(const PagedAttnArgs& A, int C) { return reinterpret_cast<SplitNote*>(A.part + C * 2 * Prompt<DP, E5M2>::kPart); }

// keys and values in the order of their tensor maps: [D][rows of a page][heads][pages], or [D][heads][tokens]
struct PromptMaps { CUtensorMap k, v; };

template <int DP, bool BF, bool E5M2, bool PAGED>
__global__ void __launch_bounds__((Prompt<DP, E5M2>::kWarps * 32), 1) paged_prompt_kernel(const PagedAttnArgs A, const __grid_constant__ PromptMaps M, int box, int above) {
    using P = Prompt<DP, E5M2>;
    constexpr int NT = P::NT, SLOTS = P::kSlots, TILE = P::kTile, HALF = 128 * 128;        // a tile is halves of 64 columns
    constexpr bool MBF = BF && !E5M2;                                 // type in the products: fp16 over e5m2
    extern __shared__ uint8_t pr_raw[];
    __shared__ int64_t scan[32];
    __shared__ int found_r;
    __shared__ int64_t found_before;
    const uint32_t base = (smem_u32(pr_raw) + 1023u) & ~1023u;
    const uint32_t qs = base, ring = base + NT * TILE, bars = ring + SLOTS * TILE;
    auto kv_full = [&](int s) { return bars + s * 8; };
    auto kv_empty = [&](int s) { return bars + 64 + s * 8; };
    auto s_full = [&](int t) { return bars + 128 + t * 8; };
    auto p_full = [&](int t, int c) { return bars + 144 + (2 * t + c) * 8; };              // P of 64 keys
    auto pv_done = [&](int t) { return bars + 176 + t * 8; };
    auto q_full = [&](int t) { return bars + 192 + t * 8; };
    auto o_free = [&](int t) { return bars + 208 + t * 8; };
    const uint32_t drained = bars + 224, tmem_slot = bars + 232;
    constexpr uint32_t TMEM_COLS = 512;                                // S_t at 128 t, O_t at 128 NT + DP t
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int group = A.Hq / A.Hkv;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; s++) { mbar_init(kv_full(s), 4); mbar_init(kv_empty(s), 1); }
        for (int t = 0; t < 2; t++) {
            mbar_init(s_full(t), 1); mbar_init(p_full(t, 0), 4); mbar_init(p_full(t, 1), 4); mbar_init(pv_done(t), 1);
            mbar_init(q_full(t), 4); mbar_init(o_free(t), 4);
        }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4 * NT + 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (A.D < DP) {                                                    // columns behind D are never copied to
        for (uint32_t i = threadIdx.x * 16; i < (uint32_t)((NT + SLOTS) * TILE); i += blockDim.x * 16) sts4(base + i, 0u, 0u, 0u, 0u);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    PromptAt at;
    int C = gridDim.x, issued = 0, place = 0;
    const int c = blockIdx.x;
    const int64_t all = open_share(A, group, P::kRows, above, [&](int64_t n) { C = sharers(n, PR_LEAST, gridDim.x); return c < C ? share_begin(n, c, C) : -1; }, scan, &found_r,
                                   &found_before, at, place);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
    // not before every block holds its columns: a dependent that allocates in front of its wait must find nobody who still wants some
    asm volatile("griddepcontrol.launch_dependents;");
    at.left = all > 0 && c < C ? (int)(share_begin(all, c + 1, C) - share_begin(all, c, C)) : 0;
    const bool any = at.left > 0 && (at.piece(A, group, P::kRows, above, place) || at.next(A, group, P::kRows, above));

    if (warp < 4 * NT) {
        // ================= softmax: thread = row =================
        regs_inc<P::kSoftRegs>();
        const int t = warp >> 2, quarter = warp & 3, r = 32 * quarter + lane;
        const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
        const uint32_t st = tmem + lanes + t * 128, ot = tmem + lanes + NT * 128 + t * DP;
        const uint32_t stage = base + P::kStageAt + warp * 4096;
        uint32_t steps = 0;                                            // key tiles so far
        float mul = A.scale_log2e;
        // the unit's queries into tile t: the products that read the last ones are done
        auto queries = [&](const PromptAt& w) {
            const int row = 128 * t + r, first = w.u * w.tpu, token = first + row / group;
            const bool live = row < w.tpu * group && token < w.q.n;
            const int64_t from = live ? (w.q.q0 + token) * A.q_st + (int64_t)(w.hk * group + row % group) * A.q_sh : -1;
            const uint32_t dst = qs + t * TILE;
            if (BF && E5M2) {
                // bf16 enters as fp16, divided by a power of two that brings the row's largest value to 2^14: exact but for what lies 2^-28
                // below it (fp16's last bit, 2^-24), where a 32-bit sum with that value ends too
                const uint4* p = reinterpret_cast<const uint4*>((const uint16_t*)A.q + (live ? from : 0));
                uint32_t big = 0;
                for (int i = 0; i < A.D / 8; i++) {
                    const uint4 w4 = live ? p[i] : make_uint4(0, 0, 0, 0);
                    const uint32_t v[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) big = max(big, max(v[e] & 0x7fffu, (v[e] >> 16) & 0x7fffu));
                }
                const int ex = (int)(big >> 7) - 127 - 14, e2 = big >= 0x7f80u || big == 0u ? 0 : ex < -100 ? -100 : ex;
                const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
                mul = A.scale_log2e * __uint_as_float((uint32_t)(127 + e2) << 23);
                for (int i = 0; i < A.D / 8; i++) {
                    const uint4 w4 = live ? p[i] : make_uint4(0, 0, 0, 0);
                    uint32_t v[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = h2u(__floats2half2_rn(__uint_as_float(v[e] << 16) * down, __uint_as_float(v[e] & 0xffff0000u) * down));
                    sts4(dst + (i >> 3) * HALF + r * 128 + (((i & 7) ^ (r & 7)) << 4), v[0], v[1], v[2], v[3]);
                }
            } else {
                constexpr int CH = DP / 8, RP = 32 / CH;               // 16-byte pieces of a row, rows a pass
#pragma unroll 4
                for (int i = 0; i < 32 / RP; i++) {
                    const int l = i * RP + lane / CH, piece = lane % CH, rr = 32 * quarter + l;
                    const int64_t o = __shfl_sync(0xffffffffu, from, l);
                    if (piece * 8 < A.D) cp16(dst + (piece >> 3) * HALF + rr * 128 + (((piece & 7) ^ (rr & 7)) << 4), (const uint16_t*)A.q + (o < 0 ? 0 : o) + piece * 8, o < 0 ? 0u : 16u);
                }
            }
        };
        auto hand_over = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full(t));
        };
        // whether the piece has keys for this tile: else nobody waits for its queries
        auto needed = [&](const PromptAt& w) { return min(w.b, w.tiles_of(A, group, t)) > w.a; };
        if (any) {
            if (needed(at)) { queries(at); hand_over(); }
            for (bool more = true; more;) {
                const int row = 128 * t + r, first = at.u * at.tpu, token = first + row / group;
                const bool live = row < at.tpu * group && token < at.q.n;
                const int off = at.q.len - at.q.n;
                const int n_vis = !live ? 0 : A.causal ? off + token + 1 : at.q.len;       // keys the row sees
                // keys below: every row of the warp sees them (rows behind the unit's are nobody's)
                const int plain_end = A.causal ? off + first + (128 * t + 32 * quarter) / group + 1 : at.q.len;
                const int end = min(at.b, at.tiles_of(A, group, t));
                const bool some = end > at.a, from_start = at.a == 0, whole = from_start && at.b == at.tiles;
                const int64_t oi = live ? (at.q.q0 + token) * A.o_st + (int64_t)(at.hk * group + row % group) * A.o_sh : -1;
                float top = -INFINITY, sum = 0.0f;              // the reference, as a score
                const int start = at.a;
                more = at.next(A, group, P::kRows, above);             // in the time that the first scores take
                const bool coming = more && needed(at);                // the next piece's queries
                for (int j = start; j < end; j++, steps++) {
                    if (!mbar_wait_lim(s_full(t), steps & 1, A.waits)) goto done;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    // 64 scores in registers at a time, by loops that are not unrolled: the roles share an instruction cache, and this one in a
                    // row, three loads instead of four, took 640 us where they took 553 (8000 tokens, 32 heads, P of one part)
                    const bool plain = j < plain_end / PR_KEYS;
                    const int left = n_vis - j * PR_KEYS;
                    float x[64], m0, m1, m2, m3;
                    auto load = [&](int h) {
                        tmem_ld32x(st + 64 * h, x);
                        tmem_ld32x(st + 64 * h + 32, x + 32);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (!plain) {
#pragma unroll
                            for (int i = 0; i < 64; i++) x[i] = 64 * h + i < left ? x[i] : -INFINITY;
                        }
                    };
                    m0 = m1 = m2 = m3 = -INFINITY;
#pragma unroll 1
                    for (int h = 0; h < 2; h++) {
                        load(h);
#pragma unroll
                        for (int i = 0; i < 64; i += 8) { m0 = max3(m0, x[i], x[i + 1]); m1 = max3(m1, x[i + 2], x[i + 3]); m2 = max3(m2, x[i + 4], x[i + 5]); m3 = max3(m3, x[i + 6], x[i + 7]); }
                    }
                    const float mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
                    const bool grow = (mx - top) * mul > (MBF ? 6.0f : P_GROW);    // -inf: any visible key; bf16 has room for more
                    if (__any_sync(0xffffffffu, grow)) {
                        const float top_new = grow ? mx : top;
                        if (j > start) {
                            // the P . V before this Q . K is done: O is at rest
                            const float corr = grow ? ex2((top - top_new) * mul) : 1.0f;
                            sum *= corr;
#pragma unroll 1
                            for (int i = 0; i < DP; i += 16) {
                                float o[16];
                                tmem_ld16x(ot + i, o);
                                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                                for (int e = 0; e < 16; e++) o[e] *= corr;
                                tmem_st16x(ot + i, reinterpret_cast<const uint32_t*>(o));
                            }
                        }
                        top = top_new;
                    }
                    // the multiply-add's two terms are each rounded once: 2^-8 apart up to 2^16.  Beyond, scores lose the reference first, exactly or nearly
                    const float m_ref = top == -INFINITY ? 0.0f : top * mul;
                    const bool steep = fabsf(m_ref) > 65536.0f, any_steep = __any_sync(0xffffffffu, steep);
                    const float shift = (MBF ? 0.0f : P_LIFT) - (steep ? 0.0f : m_ref);
                    float a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
                    // P of 32 keys goes where their scores were: the high parts to the first 16 columns, what their rounding left to the others
                    auto exponentials = [&](int h) {
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            uint32_t hi[16], lo[16];
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                const float* const s = x + 32 * c + 2 * i;
                                const float p0 = ex2(fmaf(s[0], mul, shift)), p1 = ex2(fmaf(s[1], mul, shift)), p2 = ex2(fmaf(s[2], mul, shift)), p3 = ex2(fmaf(s[3], mul, shift));
                                a0 += p0; a1 += p1; a2 += p2; a3 += p3;
                                split2<MBF>(p0, p1, hi[i], lo[i]);
                                split2<MBF>(p2, p3, hi[i + 1], lo[i + 1]);
                            }
                            tmem_st16x(st + 64 * h + 32 * c, hi);
                            tmem_st16x(st + 64 * h + 32 * c + 16, lo);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_full(t, h));
                    };
#pragma unroll 1
                    for (int h = 0; h < 2; h++) {
                        load(h);
                        if (any_steep) {
#pragma unroll
                            for (int i = 0; i < 64; i++) x[i] -= steep ? top : 0.0f;
                        }
                        exponentials(h);
                    }
                    sum += (a0 + a1) + (a2 + a3);
                }
                const float m_ref = top * mul;
                if (coming) queries(at);                               // the last product with the old ones is done
                if (some) {
                    if (!mbar_wait_lim(pv_done(t), (steps - 1) & 1, A.waits)) goto done;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                if (coming) hand_over();
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;                 // a row without a key gives zeros
                float* const part = A.part + ((int64_t)c * 2 + (from_start ? 1 : 0)) * P::kPart;
#pragma unroll 1
                for (int i = 0; i < DP; i += 64) {
                    float o[64];
                    if (some) {
                        tmem_ld32x(ot + i, o);
                        tmem_ld32x(ot + i + 32, o + 32);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    } else {
#pragma unroll
                        for (int e = 0; e < 64; e++) o[e] = 0.0f;
                    }
                    if (whole) {
                        // through shared memory, so that a store writes four rows of 128 bytes and not 32 of 16
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            sts4(stage + lane * 128 + ((e ^ (lane & 7)) << 4), pack2<BF>(o[8 * e] * inv, o[8 * e + 1] * inv), pack2<BF>(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                                 pack2<BF>(o[8 * e + 4] * inv, o[8 * e + 5] * inv), pack2<BF>(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
                        __syncwarp();
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const int l = 4 * e + (lane >> 3), piece = lane & 7;
                            const int64_t to = __shfl_sync(0xffffffffu, oi, l);
                            if (to >= 0 && i + 8 * piece < A.D) *reinterpret_cast<uint4*>((uint16_t*)A.out + to + i + 8 * piece) = lds128(stage + l * 128 + ((piece ^ (l & 7)) << 4));
                        }
                    } else if (some) {
                        float4* p = reinterpret_cast<float4*>(part) + (int64_t)(t * (DP / 4) + i / 4) * 128 + r;
#pragma unroll
                        for (int e = 0; e < 16; e++) p[e * 128] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                    __syncwarp();
                }
                if (!whole) reinterpret_cast<float2*>(part + (int64_t)NT * 128 * DP)[t * 128 + r] = make_float2(m_ref, sum);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (some && lane == 0) mbar_arrive(o_free(t));
            }
        }
    } else if (warp < 4 * NT + 4) {
        // ================= keys and values into the ring =================
        regs_dec<P::kCopyRegs>();
        const int w0 = 32 * (warp - 4 * NT);                           // this warp's rows of a tile: lane = row
        constexpr int CH = E5M2 ? DP / 16 : DP / 8, RP = 32 / CH, PASSES = 32 / RP;
        const int live = A.D * (E5M2 ? 1 : 2) / 16, piece = lane % CH;
        const bool notes = threadIdx.x == 4 * NT * 32;
        if (notes) prompt_notes<DP, E5M2>(A, gridDim.x)[c].rows = 0;
        int j = at.a;
        int64_t ko = 0, vo = 0;
        uint32_t state = 0;                                            // of this lane's key: none, there, in no page
        int page = 0, at_page = 0, at_row = 0, at_head = 0;
        bool more = any;
        auto ask = [&]() {
            const int64_t key = (int64_t)j * PR_KEYS + w0 + lane;
            if (PAGED && more && key < at.q.len) page = paged_page(A, at.r, (int)key);
        };
        bool more_keys = any, over = false;                            // tiles behind the one that was placed; behind the last item
        auto where = [&]() {                                           // this lane's key lies, and on to the next tile
            const int64_t key = (int64_t)j * PR_KEYS + w0 + lane;
            const bool here = key < at.q.len;
            if (PAGED) {
                const bool bad = here && (page < 0 || page >= A.n_pages);
                const int row = (int)key % A.page_size;
                state = here ? bad ? 2u : 1u : 0u;
                at_page = page; at_row = row; at_head = at.hk;
                ko = state == 1 ? page * A.k_sp + row * A.k_ss + at.hk * A.k_sh : 0;
                vo = state == 1 ? page * A.v_sp + row * A.v_ss + at.hk * A.v_sh : 0;
            } else {
                state = here ? 1u : 0u;
                at_row = (int)(at.q.q0 + key); at_head = at.hk;
                ko = here ? (at.q.q0 + key) * A.k_ss + at.hk * A.k_sh : 0;
                vo = here ? (at.q.q0 + key) * A.v_ss + at.hk * A.v_sh : 0;
            }
            if (notes && j == 0 && at.b < at.tiles)
                prompt_notes<DP, E5M2>(A, gridDim.x)[c] = split_note(min(at.tpu, at.q.n - at.u * at.tpu) * group, at.hk, at.q.q0 + at.u * at.tpu, at.b, at.tiles, all, c, C);
            if (++j >= at.b) {
                more = at.next(A, group, P::kRows, above);
                j = at.a;
            }
            more_keys = more;
            ask();
        };
        uint32_t left = any ? A.waits.limit < 0 ? (uint32_t)(share_begin(all, c + 1, C) - share_begin(all, c, C)) : 0xffffffffu : 0u;      // items, two a tile
        uint32_t item = 0;
        ask();
        if (E5M2) {
            // Bytes come by cp.async into the slot that their halves will fill, AHEAD items early, and a warp spreads its 32 rows in place.  (Loads
            // into registers an item ahead: the shuffles of addresses waited for them, 2700 clocks an item.)  A slot becomes free once the
            // item behind its own is there, so two of the ring are never ahead.
            constexpr int AHEAD = SLOTS - 2;
            const uint32_t raw = w0 * 128 + lane * 16;                 // pieces of the warp's rows in a line, 4 KB a half
            auto issue = [&]() {
                if (!over && left > 0) {
                    const int s = issued % SLOTS;
                    const bool is_v = issued & 1;
                    if (!is_v) where();
                    else over = !more_keys;
                    if (!mbar_wait_lim(kv_empty(s), ((issued / SLOTS) & 1) ^ 1, A.waits)) return false;
                    const uint8_t* const src = (const uint8_t*)(is_v ? A.v : A.k);
#pragma unroll
                    for (int i = 0; i < PASSES; i++) {
                        const int l = i * RP + lane / CH;
                        const int64_t o = __shfl_sync(0xffffffffu, is_v ? vo : ko, l);
                        const uint32_t of = __shfl_sync(0xffffffffu, state, l), to = ring + s * TILE + (i >> 3) * HALF + (i & 7) * 512 + raw;
                        if (of == 2 && is_v) sts4(to, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);       // no such page: not a number
                        else if (piece < live) cp16(to, src + o + piece * 16, of == 1 ? 16u : 0u);
                    }
                    issued++;
                    left--;
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                return true;
            };
#pragma unroll 1
            for (int i = 0; i < AHEAD; i++)
                if (!issue()) goto done;
            for (;; item++) {
                if (!issue()) goto done;
                if ((int)item == issued) break;
                asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
                __syncwarp();
                const int s = item % SLOTS;
                const uint32_t slot = ring + s * TILE, dst = slot + (piece >> 2) * HALF;
                const int c0 = 2 * (piece & 3);
                uint4 x[PASSES];
#pragma unroll
                for (int i = 0; i < PASSES; i++) {
                    x[i] = lds128(slot + (i >> 3) * HALF + (i & 7) * 512 + raw);
                    if (piece >= live) x[i] = make_uint4(0, 0, 0, 0);  // columns behind D
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < PASSES; i++) {                     // e5m2 is the upper byte of fp16
                    const int rr = w0 + i * RP + lane / CH;
                    const uint32_t a = dst + rr * 128 + ((c0 ^ (rr & 7)) << 4), b = dst + rr * 128 + (((c0 + 1) ^ (rr & 7)) << 4);
                    sts4(a, __byte_perm(x[i].x, 0u, 0x1404u), __byte_perm(x[i].x, 0u, 0x3424u), __byte_perm(x[i].y, 0u, 0x1404u), __byte_perm(x[i].y, 0u, 0x3424u));
                    sts4(b, __byte_perm(x[i].z, 0u, 0x1404u), __byte_perm(x[i].z, 0u, 0x3424u), __byte_perm(x[i].w, 0u, 0x1404u), __byte_perm(x[i].w, 0u, 0x3424u));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(kv_full(s));
            }
        } else {
            // a warp's 32 rows: boxes of rows that lie in one page by TMA (box: 8, 16 or 32 rows; 0: the layout allows none), in the order of
            // the ring.  What may not reach a product, values behind the last key, is written as zeros: such rows are copied one by one
            for (; !over && left > 0; item++, left--) {
                const int s = item % SLOTS;
                const bool is_v = item & 1;
                issued = item;
                if (!is_v) where();
                else over = !more_keys;
                if (!mbar_wait_lim(kv_empty(s), ((item / SLOTS) & 1) ^ 1, A.waits)) goto done;
                const uint32_t dst = ring + s * TILE;
                if (box && (!is_v || __all_sync(0xffffffffu, state == 1))) {
                    const bool first = lane % box == 0 && state == 1;  // keys: whatever else lies in the box is masked
                    const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, first)) * box * (DP * 2);
                    if (lane == 0) {
                        if (bytes) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(kv_full(s)), "r"(bytes) : "memory");
                        else mbar_arrive(kv_full(s));
                    }
                    __syncwarp();
                    if (first) {
#pragma unroll
                        for (int h = 0; h < DP / 64; h++) {
                            const uint32_t to = dst + h * HALF + (w0 + lane) * 128;
                            if (PAGED) asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                                                    ::"r"(to), "l"(is_v ? &M.v : &M.k), "r"(64 * h), "r"(at_row), "r"(at_head), "r"(at_page), "r"(kv_full(s)) : "memory");
                            else asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                              ::"r"(to), "l"(is_v ? &M.v : &M.k), "r"(64 * h), "r"(at_head), "r"(at_row), "r"(kv_full(s)) : "memory");
                        }
                    }
                    __syncwarp();
                    continue;
                }
                const uint16_t* const src = (const uint16_t*)(is_v ? A.v : A.k);
#pragma unroll 8
                for (int i = 0; i < PASSES; i++) {
                    const int l = i * RP + lane / CH, rr = w0 + l;
                    const int64_t o = __shfl_sync(0xffffffffu, is_v ? vo : ko, l);
                    const uint32_t of = __shfl_sync(0xffffffffu, state, l), a = dst + (piece >> 3) * HALF + rr * 128 + (((piece & 7) ^ (rr & 7)) << 4);
                    if (piece < live) {
                        if (PAGED && of == 2 && is_v) sts4(a, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);     // no such page: not a number
                        else cp16(a, src + o + piece * 8, of == 1 ? 16u : 0u);
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(kv_full(s));
            }
            issued = item;
        }
    } else {
        regs_dec<P::kMmaRegs>();
        if (warp == 4 * NT + 4 && any) {
            // ================= MMA issuer: the whole warp runs the loop, one elected lane issues =================
            const uint32_t leader = elect_leader();
            // c F32, a / b fp16 or bf16, M = 128; S: N = 128, both operands K-major; O: N = DP, A in TMEM, B (values) MN-major (bit 16)
            const uint32_t id = (1u << 4) | (MBF ? (1u << 7) | (1u << 10) : 0u) | ((128u >> 4) << 24);
            const uint32_t id_s = id | ((128u >> 3) << 17), id_o = id | (((uint32_t)DP >> 3) << 17) | (1u << 16);
            uint32_t steps[2] = {0, 0}, turns[2] = {0, 0};              // key tiles, and pieces with any, of a tile so far
            uint32_t item = 0;                                         // of the piece's first keys
            auto slot = [&](uint32_t i) { return ring + i % SLOTS * TILE; };
            auto arrived = [&](uint32_t i) { return mbar_wait_lim(kv_full(i % SLOTS), (i / SLOTS) & 1, A.waits); };
            auto scores = [&](int t, uint32_t i) {
                const uint64_t qd = make_desc(qs + t * TILE), kd = make_desc(slot(i));
#pragma unroll
                for (int k = 0; k < DP / 16; k++) {
                    const uint64_t step = (uint64_t)(((k >> 2) * HALF + (k & 3) * 32) >> 4);
                    umma_f16_w(tmem + t * 128, qd + step, kd + step, id_s, k > 0 ? 1u : 0u, leader);
                }
                umma_commit_w(s_full(t), leader);
            };
            auto values = [&](int t, uint32_t i, int h, bool fresh) {   // 64 keys
                // V tile: element (d, key) at half(d / 64), row key: LBO = the next 64 d, SBO = the next 8 keys; 16 keys a step
                const uint64_t vd = (make_desc(slot(i)) & ~((uint64_t)0x3fff << 16)) | ((uint64_t)(HALF >> 4) << 16);
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int l = 0; l < 2; l++)                        // P's high and low parts
                        umma_ts_w(tmem + NT * 128 + t * DP, tmem + t * 128 + h * 64 + (k >> 1) * 32 + l * 16 + (k & 1) * 8, vd + (uint64_t)(((4 * h + k) * 2048) >> 4), id_o, fresh && h == 0 && k == 0 && l == 0 ? 0u : 1u, leader);
            };
            for (;;) {
                // lane 0's, so that the compiler knows them to be the warp's: operands that it takes for a lane's own cost a move per MMA
                auto warps_own = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
                const int a = warps_own(at.a), b = warps_own(at.b);
                const int end[2] = {warps_own(min(b, at.tiles_of(A, group, 0))), NT == 2 ? warps_own(min(b, at.tiles_of(A, group, 1))) : 0};
                if (!arrived(item)) goto done;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if (end[t] <= a) continue;
                    if (!mbar_wait_lim(q_full(t), turns[t] & 1, A.waits)) goto done;
                    if (steps[t] > 0 && !mbar_wait_lim(pv_done(t), (steps[t] - 1) & 1, A.waits)) goto done;      // S and P share their columns
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    scores(t, item);
                }
                umma_commit_w(kv_empty(item % SLOTS), leader);
                for (int j = a; j < b; j++, item += 2) {
                    if (!arrived(item + 1)) goto done;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        if (j >= end[t]) continue;
                        if (j == a && turns[t]++ > 0 && !mbar_wait_lim(o_free(t), turns[t] & 1, A.waits)) goto done;
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            if (!mbar_wait_lim(p_full(t, h), steps[t] & 1, A.waits)) goto done;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            values(t, item + 1, h, j == a);
                        }
                        umma_commit_w(pv_done(t), leader);
                        steps[t]++;
                        if (j + 1 < end[t]) {
                            if (!arrived(item + 2) || !mbar_wait_lim(pv_done(t), (steps[t] - 1) & 1, A.waits)) goto done;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            scores(t, item + 2);
                        }
                    }
                    umma_commit_w(kv_empty((item + 1) % SLOTS), leader);
                    if (j + 1 < b) {
                        if (!arrived(item + 2)) goto done;
                        umma_commit_w(kv_empty((item + 2) % SLOTS), leader);
                    }
                }
                if (!at.next(A, group, P::kRows, above)) break;
            }
        }
    }
done:
    asm volatile("cp.async.wait_all;" ::: "memory");                   // behind a wait that ran out copies may still be under way
    __syncwarp();
    if (!E5M2 && warp >= 4 * NT && warp < 4 * NT + 4) drain_ring(issued, SLOTS, kv_full, A.waits);
    if (warp == 4 * NT + 4) {
        // ... and MMAs: nobody leaves their memory
        const uint32_t leader = elect_leader();
        umma_commit_w(drained, leader);
        mbar_wait_lim(drained, 0u, Waits{A.waits.word, kWaitCycles});
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 4 * NT + 4) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// the units that began in block c and went on in others: their parts in the order of the keys.  A thread per row, a quarter of the columns a block
template <int DP, bool BF, bool E5M2>
__global__ void __launch_bounds__((Prompt<DP, E5M2>::kRows)) paged_prompt_merge_kernel(const PagedAttnArgs A, int blocks) {
    using P = Prompt<DP, E5M2>;
    const int group = A.Hq / A.Hkv, c = blockIdx.x, t = threadIdx.x >> 7, r = threadIdx.x & 127, row = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const SplitNote note = prompt_notes<DP, E5M2>(A, blocks)[c];
    if (row >= note.rows) return;
    const int end = note.end;
    auto slot = [&](int b) { return A.part + ((int64_t)b * 2 + (b == c ? 1 : 0)) * P::kPart; };
    auto stat = [&](int b) { return reinterpret_cast<const float2*>(slot(b) + (int64_t)P::NT * 128 * DP)[t * 128 + r]; };
    float top = -INFINITY, total = 0.0f;
    for (int b = c; b <= end; b++) top = fmaxf(top, stat(b).x);
    for (int b = c; b <= end; b++) {
        const float2 s = stat(b);
        if (s.y != 0.0f) total = fmaf(s.x == -INFINITY ? s.y : ex2(s.x - top), s.y, total);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t* const dst = (uint16_t*)A.out + (note.q0 + row / group) * A.o_st + (int64_t)(note.hk * group + row % group) * A.o_sh;
    constexpr int PER = DP / 4;                                        // columns of this block
    const int d0 = blockIdx.y * PER;
    float x[PER] = {};
    for (int b = c; b <= end; b++) {
        const float2 s = stat(b);
        if (s.y == 0.0f) continue;                                     // no key for this row: nothing was stored
        const float w = s.x == -INFINITY ? s.y : ex2(s.x - top);
        const float4* p = reinterpret_cast<const float4*>(slot(b)) + (int64_t)(t * (DP / 4) + d0 / 4) * 128 + r;
#pragma unroll
        for (int i = 0; i < PER / 4; i++) {
            const float4 y = p[i * 128];
            x[4 * i] = fmaf(w, y.x, x[4 * i]); x[4 * i + 1] = fmaf(w, y.y, x[4 * i + 1]); x[4 * i + 2] = fmaf(w, y.z, x[4 * i + 2]); x[4 * i + 3] = fmaf(w, y.w, x[4 * i + 3]);
        }
    }
#pragma unroll
    for (int i = 0; i < PER; i += 8)
        if (d0 + i < A.D)
            *reinterpret_cast<uint4*>(dst + d0 + i) = make_uint4(pack2<BF>(x[i] * inv, x[i + 1] * inv), pack2<BF>(x[i + 2] * inv, x[i + 3] * inv),
                                                                 pack2<BF>(x[i + 4] * inv, x[i + 5] * inv), pack2<BF>(x[i + 6] * inv, x[i + 7] * inv));
}

// boxes of 64 elements x `box` rows: rows that are a multiple of it apart never share one with another page; 0 rows where the strides of a
// tensor map cannot say it (a broadcast dimension) or a page's rows are no multiple of 8
int prompt_maps(const PagedAttnArgs& A, PromptMaps* M, int* box) {
    *box = 0;
    memset(M, 0, sizeof(*M));
    const int rows = A.table ? (A.page_size & -A.page_size) : 32;
    if (rows < 8) return LB_OK;
    EncodeTiledFn enc = encode_fn();
    if (!enc) { set_error(LB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver"); return LB_ERR_CUDA; }
    const int b = rows < 32 ? rows : 32;
    for (int i = 0; i < 2; i++) {
        const cuuint64_t ss = (cuuint64_t)(i ? A.v_ss : A.k_ss) * 2, sh = (cuuint64_t)(i ? A.v_sh : A.k_sh) * 2, sp = (cuuint64_t)(i ? A.v_sp : A.k_sp) * 2;
        const cuuint64_t dims[4] = {(cuuint64_t)A.D, (cuuint64_t)(A.table ? A.page_size : A.Hkv), (cuuint64_t)(A.table ? A.Hkv : A.T), (cuuint64_t)A.n_pages};
        const cuuint64_t strides[3] = {A.table ? ss : sh, A.table ? sh : ss, sp};
        const cuuint32_t boxes[4] = {64, A.table ? (cuuint32_t)b : 1u, A.table ? 1u : (cuuint32_t)b, 1}, unit[4] = {1, 1, 1, 1};
        const int rank = A.table ? 4 : 3;
        for (int d = 1; d < rank; d++)
            if (strides[d - 1] == 0 || strides[d - 1] >= ((cuuint64_t)1 << 40)) return LB_OK;
        auto encode = [&] { return enc(i ? &M->v : &M->k, A.dtype == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                                       const_cast<void*>(i ? A.v : A.k), dims, strides, boxes, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE); };
        CUresult r = encode();
        if (r == CUDA_ERROR_INVALID_CONTEXT) {                         // a thread before its first runtime call: bind its device's context
            int dev = 0;
            cudaGetDevice(&dev);
            cudaSetDevice(dev);
            r = encode();
        }
        if (r != CUDA_SUCCESS) { set_error(LB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r); return LB_ERR_CUDA; }
    }
    *box = b;
    return LB_OK;
}

template <int DP, bool BF, bool E5M2, bool PAGED> int launch(const PagedAttnArgs& A, int above, cudaStream_t st) {
    using P = Prompt<DP, E5M2>;
    static bool configured[64] = {};                                   // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        cudaFuncSetAttribute(paged_prompt_kernel<DP, BF, E5M2, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kSmem);
        configured[dev & 63] = true;
    }
    const int C = sm_count();
    PromptMaps M;
    int box = 0;
    if (!E5M2) {
        if (const int rc = prompt_maps(A, &M, &box)) return rc;
    }
    launch_behind(paged_prompt_kernel<DP, BF, E5M2, PAGED>, dim3((unsigned)C), P::kWarps * 32, P::kSmem, st, launch_overlaps(st), A, M, box, above);
    note_launch();
    // overlaps in a recorded step too: every block waits first, and none releases before it ends (lowbit_internal.h)
    launch_behind(paged_prompt_merge_kernel<DP, BF, E5M2>, dim3((unsigned)C, 4), P::kRows, 0, st, true, A, C);
    note_launch();
    return check_launch();
}
template <int DP> int launch_types(const PagedAttnArgs& A, int above, cudaStream_t st) {
    if (!A.table) return A.dtype == DT_BF16 ? launch<DP, true, false, false>(A, above, st) : launch<DP, false, false, false>(A, above, st);
    if (A.cache_dtype == CACHE_E5M2) return A.dtype == DT_BF16 ? launch<DP, true, true, true>(A, above, st) : launch<DP, false, true, true>(A, above, st);
    return A.dtype == DT_BF16 ? launch<DP, true, false, true>(A, above, st) : launch<DP, false, false, true>(A, above, st);
}

}  // namespace

int paged_prompt_max_group(int D) { return D <= 128 ? 256 : 128; }
size_t paged_prompt_part_bytes(int D) {
    const int64_t floats = D <= 64 ? Prompt<64, false>::kPart : D <= 128 ? Prompt<128, false>::kPart : Prompt<256, false>::kPart;
    return (size_t)sm_count() * (2 * floats * sizeof(float) + sizeof(SplitNote));
}
int paged_prompt_launch(PagedAttnArgs A, int above, cudaStream_t st) {
    if (const int rc = make_waits(&A.waits, kWaitCycles)) return rc;
    return A.D <= 64 ? launch_types<64>(A, above, st) : A.D <= 128 ? launch_types<128>(A, above, st) : launch_types<256>(A, above, st);
}

}  // namespace lowbit
