// paged_attention.cu -- attention of the new tokens of many requests over a paged cache, and of packed prompts over themselves:
//   out[t][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - max),   j = the keys that token t of its request sees.
// Token i of a request's n new ones, which holds len, sees keys 0 .. len - n + i; a token that sees none gives zeros.
#include <string.h>
#include "paged.h"
#include "tc_common.cuh"

using namespace lowbit;
using namespace lowbit::gemmtc;

namespace lowbit {
namespace {

// ------------------------------------------------------------------ few rows (decoding): at most 16 rows = new tokens x heads of a group
// One pass over the keys: a warp takes 16 or 32 of a tile, S = Q . K^T and O += P . V by mma.sync m16n8k16 with the running maximum and sum of its
// keys in registers; the warps' sums meet once a unit.  16 rows do not fill a tcgen05 tile (128), and what bounds the kernel is what it reads:
// 100 requests of 200 to 8000 bf16 keys, 64 heads on 8, in 124 us (6.1 TB/s), 64 requests of 100 to 16000 e5m2 keys, 32 on 8, in 84.7 us (4.8 TB/s;
// there the two computing warps of a scheduler wait for the fixed latencies of their chains: issue slots 44 % busy, tensor pipe 31 %, DRAM 72 %).
// P enters the product as a 16-bit value and what its rounding left, two rows of one MMA or two MMAs, so that only the result is rounded
// (fp16's range: P_LIFT in paged.h).
// At most 16 rows, the MMA's.  This kernel / that of many rows (paged_prompt.cu), 64 requests of 1000 keys on 8 heads, with 4, 8, 12 and 16 rows: bf16 52, 53,
// 58, 59 / 97 us, e5m2 43, 44, 57, 58 / 134 to 137; one of 8000 with 16 rows 19 / 39, e5m2 19 / 43.  From 17 rows on there is the other alone: 64 requests with
// 20 to 48 rows 105 to 107, e5m2 146 to 148, so that one row more than 16 costs as much as 30.
constexpr int FEW_ROWS = 16;

template <int DP, bool E5M2> struct Few {
    static constexpr int kWarps = DP == 256 ? 4 : 8, kStages = DP == 64 ? 6 : 3;
    static constexpr int kKeys = E5M2 ? 32 : 16;                      // a warp's keys of a tile
    static constexpr int kTile = kWarps * kKeys;
    static constexpr int kRow = DP * (E5M2 ? 1 : 2);                  // bytes
    static constexpr int kHalf = kKeys * kRow, kStage = 2 * kHalf;    // keys, values
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kSums = kWarps * 8 * DP * 4, kSmem = kRing + kSums + kWarps * FEW_ROWS * 8;
    static constexpr int kPart = FEW_ROWS * DP + 2 * FEW_ROWS;        // floats of a slot
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t a, uint32_t x) { asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(x) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
    return r;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
    return r;
}
template <bool TRANS> __device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    if (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
    else asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
template <bool BF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF) asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                         : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool BF> __device__ __forceinline__ float unpack16(uint32_t w, int hi) {
    if (BF) return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return hi ? __high2float(h) : __low2float(h);
}
__device__ __forceinline__ uint32_t pack_half(float x, float y) { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool BF> __device__ __forceinline__ void store4(uint16_t* p, const float4& x, float by) {
    uint2 w;
    if (BF) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x.x * by, x.y * by), b = __floats2bfloat162_rn(x.z * by, x.w * by);
        w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else w = make_uint2(pack_half(x.x * by, x.y * by), pack_half(x.z * by, x.w * by));
    *reinterpret_cast<uint2*>(p) = w;
}

// a request's tiles on one kv head: none where its rows are another kernel's, one where it has no keys (its rows become zeros)
__device__ __forceinline__ int few_tiles(const PagedReq& q, int group, int tile) {
    if (q.n <= 0 || (int64_t)q.n * group > FEW_ROWS) return 0;
    return q.len > 0 ? (q.len - 1) / tile + 1 : 1;
}

// What a unit costs beside its keys (queries, the warps' sums, the result), in tiles: shares are taken of places, FEW_EXTRA of them in front of
// a unit's tiles, so that blocks with many short requests are not the last.  0 / 1 / 2 / 3: the 64 e5m2 requests above 124 / 102 / 85 / 88 us, the 100 of bf16
// 148 / 129 / 124 / 126, one token over 4000 e5m2 keys 18.3 / 17.1 / 16.9 / 17.8
constexpr int FEW_EXTRA = 2;
// Places that a block takes at least.  1 / 2 / 3: one request of 8000 bf16 keys, 16 heads on one, 25.5 / 17.3 / 16.3 us, of e5m2 20.4 / 16.2 / 17.9, of 500 e5m2 keys,
// 32 heads, 10.4 / 10.6 / 11.7
constexpr int FEW_LEAST = 2;
// where a block is in its share: request, kv head, tile of that head, and the end of the piece that it takes of them
struct FewAt {
    PagedReq q; int r, hk, tile, end, tiles, left;
    __device__ __forceinline__ bool piece(int place) {
        const int take = min(tiles + FEW_EXTRA - place, left);
        left -= take;
        tile = max(place - FEW_EXTRA, 0);
        end = max(place + take - FEW_EXTRA, 0);
        return tile < end;
    }
    __device__ __forceinline__ bool next(const PagedAttnArgs& A, int group, int tile_keys) {
        if (++tile < end) return true;
        while (left > 0) {
            if (++hk >= A.Hkv) {
                hk = 0;
                do {
                    if (++r >= A.R) return false;
                    q = paged_req(A, r);
                    tiles = few_tiles(q, group, tile_keys);
                } while (tiles == 0);
            }
            if (piece(0)) return true;
        }
        return false;
    }
    __device__ __forceinline__ bool last() const { return tile + 1 == end; }
};
__device__ __forceinline__ int64_t few_places(const PagedReq& q, const PagedAttnArgs& A, int group, int tile) {
    const int tiles = few_tiles(q, group, tile);
    return tiles ? (int64_t)(tiles + FEW_EXTRA) * A.Hkv : 0;
}
template <int DP, bool E5M2> __device__ __forceinline__ SplitNote* few_notes(const PagedAttnArgs& A, int C) { return reinterpret_cast<SplitNote*>(A.part + (int64_t)C * 2 * Few<DP, E5M2>::kPart); }
// the whole block: where its share begins; false: it has none
__device__ __forceinline__ bool few_open(const PagedAttnArgs& A, int group, int tile, int c, int& C, int64_t* scan, int* found_r, int64_t* found_before, FewAt& at, int64_t& all) {
    all = find_tile(A.R, [&](int r) { return few_places(paged_req(A, r), A, group, tile); },
                    [&](int64_t n) { C = sharers(n, FEW_LEAST, C); return c < C ? share_begin(n, c, C) : -1; }, scan, found_r, found_before);
    if (all == 0 || c >= C) return false;
    const int64_t first = share_begin(all, c, C), last = share_begin(all, c + 1, C);
    if (first == last) return false;
    at.r = *found_r;
    at.q = paged_req(A, at.r);
    at.tiles = few_tiles(at.q, group, tile);
    at.left = (int)(last - first);
    int64_t place;
    at.hk = div_few(first - *found_before, at.tiles + FEW_EXTRA, place);
    return at.piece((int)place) || at.next(A, group, tile);
}

// Where a 16-byte piece of a row lies, in bytes.  Copied by TMA (rows of a page in one box): halves of 128 bytes a row, swizzled 128 bytes
// wide (64-byte rows: 64).  Copied by cp.async, in a warp's own 16 or 32 rows: keys so that 8 rows x 16 bytes (ldmatrix) or rows g and pieces t
// (e5m2) meet every bank once, values so that rows 2 t do.
template <int DP, bool E5M2, bool TMA> struct FewAtSmem {
    using F = Few<DP, E5M2>;
    static constexpr int CH = F::kRow / 16;
    __device__ static __forceinline__ uint32_t tma(int row, int piece) {
        if (CH == 4) return (uint32_t)(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
        return (uint32_t)((piece >> 3) * (F::kTile * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
    }
    __device__ static __forceinline__ uint32_t key(int row, int piece) {
        if (TMA) return tma(row, piece);
        return (uint32_t)(row * F::kRow + ((E5M2 ? (CH >= 8 ? piece ^ ((row & 1) << 2) : piece) : piece ^ (row & 7)) << 4));
    }
    __device__ static __forceinline__ uint32_t value(int row, int piece) {
        if (TMA) return tma(row, piece);
        const int turn = !E5M2 ? row & 7 : CH == 4 ? (row >> 1) & 3 : CH == 8 ? row & 6 : ((row >> 1) & 1) | (row & 4);
        return (uint32_t)(row * F::kRow + ((piece ^ turn) << 4));
    }
};

// a warp's part of a unit: its queries as A fragments, the running maxima and sums of rows g and g + 8 (EIGHT: no unit has more than 8, and rows
// 8 .. 15 of the products hold the probabilities' low parts), the weighted values
template <int DP, bool BF, bool E5M2, bool TMA, bool EIGHT> struct FewWarp {
    using F = Few<DP, E5M2>;
    using At = FewAtSmem<DP, E5M2, TMA>;
    static constexpr bool MBF = BF && !E5M2;                          // type in the products: fp16 over e5m2
    static constexpr int NT = F::kKeys / 8, H = EIGHT ? 1 : 2;
    uint32_t qf[DP / 16][4];
    float factor[2], m[2], sum[2], o[DP / 8][4];                       // factor: scale x log2 e (x what a row was divided by)
    int see[2], rows;

    __device__ __forceinline__ void begin(const PagedAttnArgs& A, const PagedReq& q, int hk, int group, int g, int t) {
        rows = q.n * group;
        if (EIGHT) {
#pragma unroll
            for (int k = 0; k < DP / 16; k++) qf[k][1] = qf[k][3] = 0u;
        }
#pragma unroll
        for (int h = 0; h < H; h++) {
            const int row = g + 8 * h, token = row / group;
            see[h] = row < rows ? q.len - q.n + token + 1 : 0;
            const uint16_t* p = (const uint16_t*)A.q + (q.q0 + token) * A.q_st + (int64_t)(hk * group + row % group) * A.q_sh;
            factor[h] = A.scale_log2e;
            if (E5M2) {
                // k-step (c, s) of lane t holds elements 64 c + 16 t + 4 s .. + 3, the order in which a lane reads a key's bytes
                uint32_t big = 0;
#pragma unroll
                for (int cc = 0; cc < DP / 64; cc++) {
                    const int d = 64 * cc + 16 * t;
                    uint4 x = make_uint4(0, 0, 0, 0), y = x;
                    if (row < rows && d < A.D) { x = *reinterpret_cast<const uint4*>(p + d); y = *reinterpret_cast<const uint4*>(p + d + 8); }
                    const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        qf[4 * cc + e / 2][h + 2 * (e & 1)] = w[e];
                        big = max(big, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
                    }
                }
                if (BF) {
                    // bf16 enters as fp16, divided by a power of two that brings the row's largest value to 2^14: exact but for what lies 2^-28
                    // below it (fp16's last bit, 2^-24), where a 32-bit sum with that value ends too
                    big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                    big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                    const int ex = (int)(big >> 7) - 127 - 14, e = big >= 0x7f80u || big == 0u ? 0 : ex < -100 ? -100 : ex;
                    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                    factor[h] *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                    for (int k = 0; k < DP / 16; k++)
#pragma unroll
                        for (int z = 0; z < 2; z++) {
                            const uint32_t w = qf[k][h + 2 * z];
                            qf[k][h + 2 * z] = pack_half(unpack16<true>(w, 0) * down, unpack16<true>(w, 1) * down);
                        }
                }
            } else {
#pragma unroll
                for (int k = 0; k < DP / 16; k++)
#pragma unroll
                    for (int z = 0; z < 2; z++) {
                        const int d = 16 * k + 8 * z + 2 * t;
                        qf[k][h + 2 * z] = row < rows && d < A.D ? *reinterpret_cast<const uint32_t*>(p + d) : 0u;
                    }
            }
            m[h] = -INFINITY; sum[h] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < DP / 8; u++) o[u][0] = o[u][1] = o[u][2] = o[u][3] = 0.0f;
    }

    // 16 or 32 keys from key0 on, in rows row0 .. of the tiles at ks and vs; `len`: values behind it are whatever was there (TMA)
    __device__ __forceinline__ void keys(uint32_t ks, uint32_t vs, int row0, int key0, int len, int g, int t, int lane) {
        float s[NT][4];
#pragma unroll
        for (int j = 0; j < NT; j++) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
        if (E5M2) {
#pragma unroll
            for (int cc = 0; cc < DP / 64; cc++) {
                uint32_t x[NT][4];
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const uint4 w = lds16(ks + At::key(row0 + 8 * j + g, 4 * cc + t));
                    x[j][0] = w.x; x[j][1] = w.y; x[j][2] = w.z; x[j][3] = w.w;
                }
#pragma unroll
                for (int k = 0; k < 4; k++)                            // e5m2 is the upper byte of fp16
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        mma<false>(s[j], qf[4 * cc + k][0], qf[4 * cc + k][1], qf[4 * cc + k][2], qf[4 * cc + k][3], __byte_perm(x[j][k], 0u, 0x1404u),
                                   __byte_perm(x[j][k], 0u, 0x3424u));
            }
        } else {
            // even and odd steps on sums of their own: an accumulator is free again only after some 20 clocks
            float s1[NT][4];
#pragma unroll
            for (int j = 0; j < NT; j++) s1[j][0] = s1[j][1] = s1[j][2] = s1[j][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < DP / 16; k += 2) {
                uint32_t b[4], d[4];
                ldsm4<false>(b, ks + At::key(row0 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                ldsm4<false>(d, ks + At::key(row0 + (lane & 7) + ((lane >> 4) << 3), 2 * k + 2 + ((lane >> 3) & 1)));
                mma<MBF>(s[0], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[0], b[1]);
                mma<MBF>(s[1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[2], b[3]);
                mma<MBF>(s1[0], qf[k + 1][0], qf[k + 1][1], qf[k + 1][2], qf[k + 1][3], d[0], d[1]);
                mma<MBF>(s1[1], qf[k + 1][0], qf[k + 1][1], qf[k + 1][2], qf[k + 1][3], d[2], d[3]);
            }
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[j][e] += s1[j][e];
        }
        // a row of nobody (see = 0) has no scores; rows of a request see keys up to their own, the first one the fewest
        const int first = key0 + 2 * t;
        float mx[H];
        bool grow = false;
#pragma unroll
        for (int h = 0; h < H; h++) {
            mx[h] = -INFINITY;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float& x = s[j][2 * h + e];
                    x = first + 8 * j + e < see[h] ? x * factor[h] : -INFINITY;
                    mx[h] = fmaxf(mx[h], x);
                }
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            grow |= mx[h] > m[h] + P_GROW;                             // -inf: any key
        }
        // the reference follows the maximum when that grew by more than 2^P_GROW: probabilities up to that are as exact as those up to 1
        if (__any_sync(0xffffffffu, grow)) {
            float corr[2];
#pragma unroll
            for (int h = 0; h < H; h++) {
                const float to = mx[h] > m[h] + P_GROW ? mx[h] : m[h];
                corr[h] = m[h] == to ? 1.0f : ex2(m[h] - to);
                m[h] = to;
                sum[h] *= corr[h];
            }
            if (EIGHT) corr[1] = corr[0];
#pragma unroll
            for (int u = 0; u < DP / 8; u++) { o[u][0] *= corr[0]; o[u][1] *= corr[0]; o[u][2] *= corr[1]; o[u][3] *= corr[1]; }
        }
        uint32_t hi[NT][H], lo[NT][H];
#pragma unroll
        for (int h = 0; h < H; h++) {
            const float shift = (MBF ? 0.0f : P_LIFT) - (m[h] == -INFINITY ? 0.0f : m[h]);
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const float x = ex2(s[j][2 * h] + shift), y = ex2(s[j][2 * h + 1] + shift);
                sum[h] += x + y;
                split2<MBF>(x, y, hi[j][h], lo[j][h]);
            }
        }
        // probabilities as two 16-bit values each; up to 8 rows the low parts are the products' other 8 rows, at no cost
        auto values = [&](int j, float (&acc)[4], uint32_t b0, uint32_t b1) {
            if constexpr (EIGHT) mma<MBF>(acc, hi[2 * j][0], lo[2 * j][0], hi[2 * j + 1][0], lo[2 * j + 1][0], b0, b1);
            else {
                mma<MBF>(acc, lo[2 * j][0], lo[2 * j][1], lo[2 * j + 1][0], lo[2 * j + 1][1], b0, b1);
                mma<MBF>(acc, hi[2 * j][0], hi[2 * j][1], hi[2 * j + 1][0], hi[2 * j + 1][1], b0, b1);
            }
        };
        const bool cut = TMA && key0 + F::kKeys > len;                 // values behind the last key do not reach a product
#pragma unroll
        for (int j = 0; j < NT / 2; j++) {                             // 16 keys
            if (E5M2) {
                // column tile u holds elements (DP / 8) n + u, n = 0 .. 7: a lane's bytes of a row lie together
                constexpr int B = DP / 8, W = B / 4;
                uint32_t x[4][W];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int row = 16 * j + 2 * t + (k & 1) + 8 * (k >> 1);
                    if (B == 8) {
                        const uint2 w = lds8(vs + At::value(row0 + row, g >> 1) + 8 * (g & 1));
                        x[k][0] = w.x; x[k][1] = w.y;
                    } else {
#pragma unroll
                        for (int z = 0; z < B / 16; z++) {
                            const uint4 w = lds16(vs + At::value(row0 + row, g * (B / 16) + z));
                            x[k][(4 * z) % W] = w.x; x[k][(4 * z + 1) % W] = w.y; x[k][(4 * z + 2) % W] = w.z; x[k][(4 * z + 3) % W] = w.w;
                        }
                    }
                    if (cut && key0 + row >= len) {
#pragma unroll
                        for (int z = 0; z < W; z++) x[k][z] = 0u;
                    }
                }
#pragma unroll
                for (int u = 0; u < DP / 8; u += 2) {
                    const uint32_t sel = u & 2 ? 0x7362u : 0x5140u;
                    const uint32_t p = __byte_perm(x[0][u / 4], x[1][u / 4], sel), q = __byte_perm(x[2][u / 4], x[3][u / 4], sel);
                    values(j, o[u], __byte_perm(p, 0u, 0x1404u), __byte_perm(q, 0u, 0x1404u));
                    values(j, o[u + 1], __byte_perm(p, 0u, 0x3424u), __byte_perm(q, 0u, 0x3424u));
                }
            } else {
                uint32_t keep[2];                                      // of keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const int left = len - key0 - 2 * t - 8 * z;
                    keep[z] = left >= 2 ? 0xffffffffu : left == 1 ? 0x0000ffffu : 0u;
                }
#pragma unroll
                for (int u = 0; u < DP / 8; u += 2) {
                    uint32_t b[4];
                    ldsm4<true>(b, vs + At::value(row0 + 16 * j + (lane & 15), u + (lane >> 4)));
                    if (cut) { b[0] &= keep[0]; b[1] &= keep[1]; b[2] &= keep[0]; b[3] &= keep[1]; }
                    values(j, o[u], b[0], b[1]);
                    values(j, o[u + 1], b[2], b[3]);
                }
            }
        }
    }

    // the unit's last tile here: the warps' sums to one, divided and stored, or left for the merge.  All NW warps; sync: a barrier of theirs
    template <typename Sync>
    __device__ __forceinline__ void finish(const PagedAttnArgs& A, const PagedReq& q, int hk, int group, bool whole, float* part, float* sums, float2* stats, int warp, int lane,
                                           Sync sync) {
        constexpr int NW = F::kWarps;
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int h = 0; h < H; h++) {
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
            if (t == 0) stats[warp * FEW_ROWS + g + 8 * h] = make_float2(m[h], sum[h]);
        }
        for (int h = 0; h < (EIGHT || rows <= 8 ? 1 : 2); h++) {
            float* const mine = sums + (warp * 8 + g) * DP;
#pragma unroll
            for (int u = 0; u < DP / 8; u++) {
                const float x = EIGHT ? o[u][0] + o[u][2] : h ? o[u][2] : o[u][0], y = EIGHT ? o[u][1] + o[u][3] : h ? o[u][3] : o[u][1];
                if (E5M2) { mine[2 * t * (DP / 8) + u] = x; mine[(2 * t + 1) * (DP / 8) + u] = y; }
                else *reinterpret_cast<float2*>(mine + 8 * u + 2 * t) = make_float2(x, y);
            }
            sync();
            for (int row = 8 * h + warp; row < rows && row < 8 * h + 8; row += NW) {
                float top = -INFINITY, total = 0.0f, weight[NW];
#pragma unroll
                for (int w = 0; w < NW; w++) top = fmaxf(top, stats[w * FEW_ROWS + row].x);
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const float2 st = stats[w * FEW_ROWS + row];
                    weight[w] = st.x == -INFINITY ? (st.y == 0.0f ? 0.0f : st.y) : ex2(st.x - top);
                    total += weight[w] * st.y;
                }
                const float inv = total == 0.0f ? 0.0f : 1.0f / total;
                const int token = row / group;
                uint16_t* const dst = (uint16_t*)A.out + (q.q0 + token) * A.o_st + (int64_t)(hk * group + row % group) * A.o_sh;
                for (int d = 4 * lane; d < DP; d += 128) {
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < NW; w++) {
                        const float4 y = *reinterpret_cast<const float4*>(sums + (w * 8 + row - 8 * h) * DP + d);
                        x.x = fmaf(weight[w], y.x, x.x); x.y = fmaf(weight[w], y.y, x.y); x.z = fmaf(weight[w], y.z, x.z); x.w = fmaf(weight[w], y.w, x.w);
                    }
                    if (whole) {
                        if (d < A.D) store4<BF>(dst + d, x, inv);
                    } else *reinterpret_cast<float4*>(part + row * DP + d) = x;
                }
                if (!whole && lane == 0) *reinterpret_cast<float2*>(part + FEW_ROWS * DP + 2 * row) = make_float2(top, total);
            }
            sync();
        }
    }
};

// Every warp copies its own keys: page sizes that TMA has no box for (no multiple of 8 rows, or a stride of 0).  Where both serve: one token over 4000 e5m2
// keys 20.4 us for 16.9, the 64 requests 125 for 85, the 100 requests 173 for 124
template <int DP, bool BF, bool E5M2>
__global__ void __launch_bounds__((Few<DP, E5M2>::kWarps * 32), 1) paged_few_kernel(const PagedAttnArgs A) {
    using F = Few<DP, E5M2>;
    using W = FewWarp<DP, BF, E5M2, false, false>;
    constexpr int ST = F::kStages, KW = F::kKeys, CH = F::kRow / 16;
    extern __shared__ __align__(128) uint8_t few_smem[];
    __shared__ int64_t scan[32];
    __shared__ int found_r;
    __shared__ int64_t found_before;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = A.Hq / A.Hkv;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int c = blockIdx.x;
    int C = gridDim.x;
    FewAt at;                                                          // of the products
    int64_t all;
    SplitNote* const note = few_notes<DP, E5M2>(A, gridDim.x) + c;
    if (threadIdx.x == 0) note->rows = 0;
    if (!few_open(A, group, F::kTile, c, C, scan, &found_r, &found_before, at, all)) return;
    FewAt in = at;                                                     // of the copies
    bool to_copy = true;

    const uint32_t ring = smem_addr(few_smem) + warp * ST * F::kStage;
    float* const sums = reinterpret_cast<float*>(few_smem + F::kRing);                       // [warp][8][DP]
    float2* const stats = reinterpret_cast<float2*>(few_smem + F::kRing + F::kSums);         // [warp][16]
    // columns behind D stay zero: they are never copied to
    if (A.D < DP) {
        for (int i = lane; i < ST * F::kStage / 16; i += 32) sts16(ring + 16 * i, 0u);
        __syncwarp();
    }
    const int live = A.D * (E5M2 ? 1 : 2) / 16;                        // 16-byte pieces of a row
    // the page of this lane's key in the copies' tile, one tile ahead of its copies
    int page = 0;
    auto key_of = [&](const FewAt& w) { return w.tile * F::kTile + warp * KW + (KW == 32 ? lane : lane & 15); };
    auto ask = [&]() {
        const int key = key_of(in);
        if (to_copy && key < in.q.len) page = paged_page(A, in.r, key);
    };
    auto copy = [&](int stage) {
        if (!to_copy) return;
        const uint32_t dst = ring + stage * F::kStage;
        const int key = key_of(in);
        const bool here = key < in.q.len, bad = here && (page < 0 || page >= A.n_pages);
        if (__any_sync(0xffffffffu, here)) {
            const int row = key % A.page_size;
            const int64_t ko = here && !bad ? page * A.k_sp + row * A.k_ss + in.hk * A.k_sh : 0, vo = here && !bad ? page * A.v_sp + row * A.v_ss + in.hk * A.v_sh : 0;
            const uint32_t state = here ? bad ? 2u : 1u : 0u;
#pragma unroll
            for (int i = 0; i < KW * CH / 32; i++) {
                const int r = (i * 32 + lane) / CH, piece = lane % CH;
                const int64_t kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
                const uint32_t s = __shfl_sync(0xffffffffu, state, r);
                if (piece < live) {
                    const uint32_t bytes = s == 1 ? 16u : 0u;
                    cp16(dst + W::At::key(r, piece), (const uint8_t*)A.k + kr * (E5M2 ? 1 : 2) + piece * 16, bytes);
                    if (s == 2) sts16(dst + F::kHalf + W::At::value(r, piece), E5M2 ? 0x7f7f7f7fu : 0x7fff7fffu);      // no such page: not a number
                    else cp16(dst + F::kHalf + W::At::value(r, piece), (const uint8_t*)A.v + vr * (E5M2 ? 1 : 2) + piece * 16, bytes);
                }
            }
        }
        to_copy = in.next(A, group, F::kTile);
        ask();
    };
    ask();
    for (int s = 0; s < ST - 1; s++) {
        copy(s);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    W w;
    bool begun = false, from_start = false, more = true;
    for (int i = 0; more; i++) {
        copy((i + ST - 1) % ST);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (!begun) {
            begun = true;
            from_start = at.tile == 0;
            if (from_start && at.end < at.tiles && threadIdx.x == 0) *note = split_note(at.q.n * group, at.hk, at.q.q0, at.end, at.tiles, all, c, C);
            w.begin(A, at.q, at.hk, group, g, t);
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        __syncwarp();
        const int key0 = at.tile * F::kTile + warp * KW;
        const uint32_t ks = ring + i % ST * F::kStage;
        if (key0 < at.q.len) w.keys(ks, ks + F::kHalf, 0, key0, at.q.len, g, t, lane);
        __syncwarp();
        if (!at.last()) { at.tile++; continue; }
        w.finish(A, at.q, at.hk, group, from_start && at.end == at.tiles, A.part + ((int64_t)c * 2 + (from_start ? 1 : 0)) * F::kPart, sums, stats, warp, lane,
                 [] { __syncthreads(); });
        begun = false;
        more = at.next(A, group, F::kTile);
    }
}

// keys and values: [D][rows of a page][heads][pages]
struct FewMaps { CUtensorMap k, v; };

// Four warps more fetch whole tiles by TMA, a box of 8 to 32 rows of a page a lane: a warp issues one in 80 to 95 clocks, and a tile of pages of 16
// rows takes 32 of them (one warp for all: 3100 clocks a tile, 2360 for the products)
template <int DP, bool BF, bool E5M2, bool EIGHT>
__global__ void __launch_bounds__((Few<DP, E5M2>::kWarps * 32 + 128), 1) paged_few_tma_kernel(const PagedAttnArgs A, const __grid_constant__ FewMaps M, int box) {
    using F = Few<DP, E5M2>;
    constexpr int NW = F::kWarps, ST = F::kRing / (F::kStage * NW), KW = F::kKeys, HALVES = F::kRow <= 128 ? 1 : F::kRow / 128, WIDE = F::kRow < 128 ? F::kRow : 128;
    constexpr int TILE = F::kTile * F::kRow;                           // bytes of a tile's keys
    extern __shared__ uint8_t few_raw[];
    __shared__ int64_t scan[32];
    __shared__ int found_r;
    __shared__ int64_t found_before;
    __shared__ __align__(8) uint64_t bars[2 * ST];
    __shared__ __align__(16) uint32_t bad_boxes[ST][4];
    __shared__ volatile int gave_up;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = A.Hq / A.Hkv;
    const uint32_t ring = (smem_addr(few_raw) + 1023u) & ~1023u;
    auto full = [&](int s) { return smem_addr(bars + s); };
    auto empty = [&](int s) { return smem_addr(bars + ST + s); };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < ST; s++) { mbar_init(full(s), 4); mbar_init(empty(s), NW); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const int c = blockIdx.x;
    int C = gridDim.x;
    FewAt at;
    int64_t all;
    const bool notes = threadIdx.x == NW * 32;
    SplitNote* const note = few_notes<DP, E5M2>(A, gridDim.x) + c;
    if (notes) note->rows = 0;
    if (!few_open(A, group, F::kTile, c, C, scan, &found_r, &found_before, at, all)) return;
    if (warp >= NW) {
        // ================= the copies: this warp's boxes of a tile =================
        const int boxes = F::kTile / box, own = max(boxes / 4, 1), mine = own * (warp - NW) + lane, most = A.waits.limit < 0 ? at.left / 2 : 0x7fffffff;
        const bool some = lane < own && mine < boxes;
        int page = 0, issued = 0;
        bool more = true;
        auto ask = [&]() {
            const int key = at.tile * F::kTile + mine * box;
            if (more && some && key < at.q.len) page = paged_page(A, at.r, key);
        };
        ask();
        for (; more && issued < most; issued++) {
            const int s = issued % ST;
            if (!mbar_wait_lim(empty(s), ((issued / ST) & 1) ^ 1, A.waits)) break;
            const int key = at.tile * F::kTile + mine * box;
            const bool here = some && key < at.q.len, good = here && page >= 0 && page < A.n_pages;
            const uint32_t bad = __ballot_sync(0xffffffffu, here && !good), bytes = __popc(__ballot_sync(0xffffffffu, good)) * box * (HALVES * WIDE * 2);
            if (lane == 0) {
                bad_boxes[s][warp - NW] = bad << own * (warp - NW);
                if (bytes) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full(s)), "r"(bytes) : "memory");
                else mbar_arrive(full(s));
            }
            __syncwarp();
            if (good) {
                const int row = key % A.page_size;
                const uint32_t dst = ring + s * (2 * TILE) + mine * box * WIDE;
#pragma unroll
                for (int v = 0; v < 2; v++)
#pragma unroll
                    for (int h = 0; h < HALVES; h++)
                        asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                                     ::"r"(dst + v * TILE + h * (F::kTile * 128)), "l"(v ? &M.v : &M.k), "r"(h * (E5M2 ? 128 : 64)), "r"(row), "r"(at.hk), "r"(page), "r"(full(s)) : "memory");
            }
            if (notes && at.tile == 0 && at.end < at.tiles) *note = split_note(at.q.n * group, at.hk, at.q.q0, at.end, at.tiles, all, c, C);
            __syncwarp();
            more = at.next(A, group, F::kTile);
            ask();
        }
        // nobody leaves while copies are under way
        drain_ring(issued, ST, full, A.waits);
    } else {
        float* const sums = reinterpret_cast<float*>(few_raw + (ring - smem_addr(few_raw)) + F::kRing);
        float2* const stats = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(sums) + F::kSums);
        FewWarp<DP, BF, E5M2, true, EIGHT> w;
        bool begun = false, from_start = false, more = true;
        for (int i = 0; more; i++) {
            const int s = i % ST;
            if (!begun) {
                begun = true;
                from_start = at.tile == 0;
                w.begin(A, at.q, at.hk, group, g, t);
            }
            // a wait that ran out in one warp ends them all; they go through the motions, because they meet at barriers
            if (!__any_sync(0xffffffffu, gave_up) && !mbar_wait_lim(full(s), (i / ST) & 1, A.waits)) gave_up = 1;
            const int key0 = at.tile * F::kTile + warp * KW;
            const uint32_t ks = ring + s * (2 * TILE);
            if (key0 < at.q.len) {
                w.keys(ks, ks + TILE, warp * KW, key0, at.q.len, g, t, lane);
                const uint4 bad = *reinterpret_cast<const uint4*>(bad_boxes[s]);
                if ((bad.x | bad.y | bad.z | bad.w) >> (warp * KW / box) & ((1u << ((KW + box - 1) / box)) - 1)) w.sum[0] = w.sum[EIGHT ? 0 : 1] = NAN;       // no such page
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(s));
            if (!at.last()) { at.tile++; continue; }
            w.finish(A, at.q, at.hk, group, from_start && at.end == at.tiles, A.part + ((int64_t)c * 2 + (from_start ? 1 : 0)) * F::kPart, sums, stats, warp, lane,
                     [] { asm volatile("barrier.sync 1, %0;" ::"n"(NW * 32) : "memory"); });
            begun = false;
            more = at.next(A, group, F::kTile);
        }
    }
    __syncthreads();
}

// the units that began in block c and went on in others: their parts in the order of the keys, a row a warp
template <int DP, bool BF, bool E5M2>
__global__ void __launch_bounds__(128) paged_few_merge_kernel(const PagedAttnArgs A) {
    using F = Few<DP, E5M2>;
    const int group = A.Hq / A.Hkv, c = blockIdx.x, row = 4 * blockIdx.y + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const SplitNote note = few_notes<DP, E5M2>(A, gridDim.x)[c];
    if (row >= note.rows) return;
    const int end = note.end, hk = note.hk;
    auto slot = [&](int b) { return A.part + ((int64_t)b * 2 + (b == c ? 1 : 0)) * F::kPart; };
    float top = -INFINITY, total = 0.0f;
    for (int b = c + lane; b <= end; b += 32)
        top = fmaxf(top, slot(b)[FEW_ROWS * DP + 2 * row]);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    float4 x[DP > 128 ? 2 : 1];
#pragma unroll
    for (int z = 0; z < (DP > 128 ? 2 : 1); z++) x[z] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int b0 = c; b0 <= end; b0 += 32) {
        // a lane finds a part's weight, and all add up its values
        float mine = 0.0f, part_sum = 0.0f;
        if (b0 + lane <= end) {
            const float2 st = *reinterpret_cast<const float2*>(slot(b0 + lane) + FEW_ROWS * DP + 2 * row);
            mine = st.x == -INFINITY ? (st.y == 0.0f ? 0.0f : st.y) : ex2(st.x - top);
            part_sum = st.y;
        }
#pragma unroll 8
        for (int k = 0; k < 32 && b0 + k <= end; k++) {
            const float w = __shfl_sync(0xffffffffu, mine, k);
            total = fmaf(w, __shfl_sync(0xffffffffu, part_sum, k), total);
            const float* const p = slot(b0 + k);
#pragma unroll
            for (int z = 0; z < (DP > 128 ? 2 : 1); z++) {
                const int d = 4 * lane + 128 * z;
                if (d >= DP) continue;
                const float4 y = *reinterpret_cast<const float4*>(p + row * DP + d);
                x[z].x = fmaf(w, y.x, x[z].x); x[z].y = fmaf(w, y.y, x[z].y); x[z].z = fmaf(w, y.z, x[z].z); x[z].w = fmaf(w, y.w, x[z].w);
            }
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t* const dst = (uint16_t*)A.out + (note.q0 + row / group) * A.o_st + (int64_t)(hk * group + row % group) * A.o_sh;
#pragma unroll
    for (int z = 0; z < (DP > 128 ? 2 : 1); z++) {
        const int d = 4 * lane + 128 * z;
        if (d < A.D) store4<BF>(dst + d, x[z], inv);
    }
}

bool aligned(const void* p, int64_t a, int64_t b, int64_t c, int unit) { return !((uintptr_t)p & 15) && !((a | b | c) & (unit - 1)); }

// what both entry points refuse
int check(const PagedAttnArgs& A, const char* name) {
    if (!A.q || !A.k || !A.v || !A.cu || !A.out || A.R <= 0 || A.T < 0 || A.Hq <= 0 || A.Hkv <= 0 || A.Hq % A.Hkv || A.Hq / A.Hkv > paged_prompt_max_group(A.D) || A.D <= 0 || A.D % 16 || A.D > 256 ||
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

// boxes of up to 32 rows; 0 rows where a page's rows are no multiple of 8 or a stride is none of a tensor map's
template <int DP, bool E5M2> int few_maps(const PagedAttnArgs& A, FewMaps* M, int* box) {
    using F = Few<DP, E5M2>;
    *box = 0;
    memset(M, 0, sizeof(*M));
    const int rows = A.page_size & -A.page_size, b = rows < 32 ? rows : 32;
    if (b < 8) return LB_OK;
    EncodeTiledFn enc = encode_fn();
    if (!enc) { set_error(LB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver"); return LB_ERR_CUDA; }
    const cuuint64_t size = E5M2 ? 1 : 2;
    for (int i = 0; i < 2; i++) {
        const cuuint64_t strides[3] = {(cuuint64_t)(i ? A.v_ss : A.k_ss) * size, (cuuint64_t)(i ? A.v_sh : A.k_sh) * size, (cuuint64_t)(i ? A.v_sp : A.k_sp) * size};
        const cuuint64_t dims[4] = {(cuuint64_t)A.D, (cuuint64_t)A.page_size, (cuuint64_t)A.Hkv, (cuuint64_t)A.n_pages};
        const cuuint32_t boxes[4] = {(cuuint32_t)((F::kRow < 128 ? F::kRow : 128) / size), (cuuint32_t)b, 1, 1}, unit[4] = {1, 1, 1, 1};
        for (const cuuint64_t st : strides)
            if (st == 0 || st >= ((cuuint64_t)1 << 40)) return LB_OK;
        auto encode = [&] { return enc(i ? &M->v : &M->k, E5M2 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : A.dtype == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(i ? A.v : A.k), dims, strides, boxes, unit,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, F::kRow < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, F::kRow >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : F::kRow == 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B,
                                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE); };
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

template <int DP, bool BF, bool E5M2> int few_launch(PagedAttnArgs A, bool eight, cudaStream_t st) {
    using F = Few<DP, E5M2>;
    static bool configured[64] = {};                                   // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        cudaFuncSetAttribute(paged_few_kernel<DP, BF, E5M2>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
        cudaFuncSetAttribute(paged_few_tma_kernel<DP, BF, E5M2, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem + 1024);
        cudaFuncSetAttribute(paged_few_tma_kernel<DP, BF, E5M2, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem + 1024);
        configured[dev & 63] = true;
    }
    const int C = sm_count();
    FewMaps M;
    int box = 0;
    if (const int rc = few_maps<DP, E5M2>(A, &M, &box)) return rc;
    if (box) {
        if (const int rc = make_waits(&A.waits, kWaitCycles)) return rc;
        launch_behind(eight ? paged_few_tma_kernel<DP, BF, E5M2, true> : paged_few_tma_kernel<DP, BF, E5M2, false>, dim3((unsigned)C), F::kWarps * 32 + 128, F::kSmem + 1024, st,
                      launch_overlaps(st), A, M, box);
    } else launch_behind(paged_few_kernel<DP, BF, E5M2>, dim3((unsigned)C), F::kWarps * 32, F::kSmem, st, launch_overlaps(st), A);
    note_launch();
    // overlaps in a recorded step too: every block waits first, and none releases before it ends (lowbit_internal.h)
    launch_behind(paged_few_merge_kernel<DP, BF, E5M2>, dim3((unsigned)C, FEW_ROWS / 4), 128, 0, st, true, A);
    note_launch();
    return check_launch();
}
template <int DP> int few_launch_types(const PagedAttnArgs& A, bool eight, cudaStream_t st) {
    if (A.cache_dtype == CACHE_E5M2) return A.dtype == DT_BF16 ? few_launch<DP, true, true>(A, eight, st) : few_launch<DP, false, true>(A, eight, st);
    return A.dtype == DT_BF16 ? few_launch<DP, true, false>(A, eight, st) : few_launch<DP, false, false>(A, eight, st);
}
size_t few_part_bytes(int D) {
    const int dp = D <= 64 ? 64 : D <= 128 ? 128 : 256;
    return (size_t)sm_count() * (2 * (FEW_ROWS * dp + 2 * FEW_ROWS) * sizeof(float) + sizeof(SplitNote));
}

}  // namespace
}  // namespace lowbit

extern "C" size_t lowbit_sdp_paged_workspace_size(int64_t T, int R, int Hq, int Hkv, int D, int64_t max_query) {
    (void)R;
    if (D <= 0 || D > 256) return 0;
    if (max_query > T) max_query = T;
    const size_t few = few_part_bytes(D);
    return Hkv > 0 && max_query * (Hq / Hkv) <= FEW_ROWS ? few : few + paged_prompt_part_bytes(D);
}

extern "C" int lowbit_sdp_paged_cuda(const void* d_q, int q_dtype, const int64_t* q_strides, int64_t T, const void* d_k, const int64_t* k_strides,
                                     const void* d_v, const int64_t* v_strides, int cache_dtype, int n_pages, int page_size, const int32_t* d_table,
                                     int64_t table_stride, int width, const int32_t* d_seq_lens, const int32_t* d_cu_seqlens, int R, int Hq, int Hkv,
                                     int D, float scale, int64_t max_query, void* d_out, const int64_t* out_strides, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    reset_launch_count();
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
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < lowbit_sdp_paged_workspace_size(T, R, Hq, Hkv, D, max_query)) {
        set_error(LB_ERR_WORKSPACE, "lowbit_sdp_paged_cuda: a 16-byte aligned workspace of lowbit_sdp_paged_workspace_size() bytes is needed");
        return LB_ERR_WORKSPACE;
    }
    A.part = (float*)workspace;
    if (max_query > T) max_query = T;
    cudaStream_t st = (cudaStream_t)stream;
    // no unit has more than 8 rows: the other 8 of the MMA carry what rounding P left.  Else / so: one token over 4000 e5m2 keys 19.1 / 16.9 us, the 64
    // requests 104 / 85, the 100 requests 126 / 124
    const bool eight = max_query * (Hq / Hkv) <= 8;
    if (const int rc = D <= 64 ? few_launch_types<64>(A, eight, st) : D <= 128 ? few_launch_types<128>(A, eight, st) : few_launch_types<256>(A, eight, st)) return rc;
    if (max_query * (Hq / Hkv) <= FEW_ROWS) return LB_OK;
    A.part = (float*)((uint8_t*)workspace + few_part_bytes(D));
    return paged_prompt_launch(A, FEW_ROWS, st);
}

extern "C" size_t lowbit_sdp_packed_workspace_size(int64_t T, int R, int Hq, int Hkv, int D, int64_t max_seqlen) {
    (void)T; (void)R; (void)Hq; (void)Hkv; (void)max_seqlen;
    return D > 0 && D <= 256 ? paged_prompt_part_bytes(D) : 0;
}

extern "C" int lowbit_sdp_packed_cuda(const void* d_q, int dtype, const int64_t* q_strides, int64_t T, const void* d_k, const int64_t* k_strides,
                                      const void* d_v, const int64_t* v_strides, const int32_t* d_cu_seqlens, int R, int Hq, int Hkv, int D, float scale,
                                      int causal, int64_t max_seqlen, void* d_out, const int64_t* out_strides, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    reset_launch_count();
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
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < lowbit_sdp_packed_workspace_size(T, R, Hq, Hkv, D, max_seqlen)) {
        set_error(LB_ERR_WORKSPACE, "lowbit_sdp_packed_cuda: a 16-byte aligned workspace of lowbit_sdp_packed_workspace_size() bytes is needed");
        return LB_ERR_WORKSPACE;
    }
    A.part = (float*)workspace;
    return paged_prompt_launch(A, 0, (cudaStream_t)stream);
}
