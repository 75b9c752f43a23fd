// lora.cu -- low-rank adapters of many requests beside a projection that all share:
//   out[t] += scale_l (x[t] A_l^T) B_l^T,      l = the adapter of the token's request (none: the row stays as it is).
//
// A cluster takes up to 64 rows of one adapter, wherever they lie.  Few tokens: it takes a tile of packed rows, finds the tile's requests in the list, and the different
// adapters among its rows are dealt to the clusters that share the tile.  Many: a launch in front orders all rows by their adapters.  So an adapter that requests
// have in common is read once for 64 rows of theirs.  For each:
//   every block multiplies its share of the inner dimension, h = x A^T in 32 bits;
//   the blocks add up their parts, a share of the rows each, and hand the sums to all through their shared memories;
//   every block multiplies its share of the columns, h B^T, and adds that to `out`, rounded once.
// Few tokens take one launch of that.  Many take one for each product, with h as two 16-bit values in memory between them: it costs little
// beside `out`, each kernel has the registers that its product wants, and a tile's columns are dealt as finely as fills the device.
// mma.sync m16n8k16: a tcgen05 tile wants 128 rows of one adapter, and x and B would have to pass through shared memory in its layout, the adapters' rows gathered.  In decode
// steps and mixed ones an adapter has some 1 to 64 rows.  In prompts it has thousands: at rank 32 the second product is little more than the copy of `out`; at rank
// 128 the first product, whose warps each read operands of their own, bounds the call (12000 tokens of K 4096 and N 896 148 us, 21 for their bytes), and a
// form for pieces of 128 rows that all warps share is not built.
// What the operator cannot do without is to read x and out, to write out, and the adapters' A and B once.
//
// Measured, times without the launch's share on the host.  One token of K 4096 and N 4096 at rank 16: 6.5 us, the latency of five dependent trips to memory and
// the cluster's two meetings.  64 tokens of 32 adapters at rank 16, 15.4 MB: 12.3 us, the same.
// 882 rows of 40 requests, K 4096 and N 11008 at rank 64, 69 MB: 40.3 us, 7 + 15 + 22.  11849 rows, N 14336 at rank 32, 628 MB: 140 us, 7 + 36 + 101.
// The second product's launch there copies `out`, which alone takes 88 us; 57 % of what a SM's shared memory and L1 can move in that time is h, read
// for 32 columns at a time, and `out` on its way through.
#include <type_traits>
#include "lowbit_common.cuh"
#include "lowbit_internal.h"

using namespace lowbit;

namespace lowbit {
namespace {

constexpr int LORA_THREADS = 256, LORA_WARPS = 8, LORA_SPLITS = 8;

struct LoraArgs {
    const void* x; int64_t x_st; int64_t T; int K;
    const void* a; int64_t a_st;                               // [adapters][splits][rank][K]
    const void* b; int64_t b_st;                               // [adapters][columns][rank]
    const float* scales; int adapters;
    const int32_t *ids, *cu; int R;                            // requests
    void* out; int64_t o_st;
    int rank, n_splits, together;                              // splits whose products with A are computed at once
    // of more launches: the pieces (adapter, first of its rows in the order of adapters, how many, 0), the rows in that order, h and what undoes its powers of
    // two between the products, blocks of a piece in the second product
    int4* pieces; int32_t* order; int32_t* lists; uint16_t* h; float* back; int shares;
    int first[LORA_SPLITS + 1];                                // columns in front of a split
};

template <bool BF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF) asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                         : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same from zero
template <bool BF> __device__ __forceinline__ void mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF) asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                         : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
template <bool BF> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    if (BF) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF> __device__ __forceinline__ float2 unpack2(uint32_t w) {
    if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// two 16-bit values plus two of 32 bits, rounded once, by the addition that takes a 16-bit term
template <bool BF> __device__ __forceinline__ uint32_t add2(uint32_t v, float x, float y) {
    float a, b;
    if (BF) asm("{\n\t.reg .b16 p, q;\n\tmov.b32 {p, q}, %2;\n\tadd.rn.f32.bf16 %0, p, %3;\n\tadd.rn.f32.bf16 %1, q, %4;\n\t}" : "=f"(a), "=f"(b) : "r"(v), "f"(x), "f"(y));
    else asm("{\n\t.reg .b16 p, q;\n\tmov.b32 {p, q}, %2;\n\tadd.rn.f32.f16 %0, p, %3;\n\tadd.rn.f32.f16 %1, q, %4;\n\t}" : "=f"(a), "=f"(b) : "r"(v), "f"(x), "f"(y));
    return pack2<BF>(a, b);
}

// the blocks of a cluster meet; what they wrote, to one another too, is seen by all
__device__ __forceinline__ void meet(uint32_t blocks) {
    if (blocks == 1) { __syncthreads(); return; }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t shared_of(uint32_t at, uint32_t block) {
    uint32_t p;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(at), "r"(block));
    return p;
}

constexpr int TM = 64;                                         // rows of a tile

// the different adapters among a tile's rows, and the rows of each, one behind the other
struct __align__(16) Tile {
    int id[TM];                                                // of the request that begins in a row; -2: none does
    int n, adapter[TM], first[TM + 1];
    int row[TM];
};
struct Rows { int row[TM]; };                                  // of a piece
// the whole block; ends behind a barrier
__device__ __forceinline__ void find_adapters(const LoraArgs& A, int64_t t0, Tile& tile) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < TM) tile.id[threadIdx.x] = -2;
    __syncthreads();
    const int64_t end = min((int64_t)A.cu[A.R], A.T);          // rows behind it are nobody's
    auto begin = [&](int r, int64_t a, int64_t b) {
        const int id = A.ids[r];
        if (a < b && b > t0 && a < t0 + TM) tile.id[max(a - t0, (int64_t)0)] = id >= 0 && id < A.adapters ? id : -1;
    };
    bool rises = true;
    for (int r = threadIdx.x; r < A.R; r += LORA_THREADS) {
        const int a = A.cu[r], b = A.cu[r + 1];
        rises &= a <= b;
        begin(r, a, b);
    }
    if (!__syncthreads_and(rises)) {                           // a list that goes back names no row twice: a request has what lies behind all in front of it
        if (threadIdx.x < TM) tile.id[threadIdx.x] = -2;
        __syncthreads();
        if (threadIdx.x == 0)
            for (int r = 0, most = A.cu[0]; r < A.R; r++) {
                most = max(most, A.cu[r]);
                begin(r, most, A.cu[r + 1]);
            }
        __syncthreads();
    }
    if (threadIdx.x < 32) {
        // of rows `lane` and `lane` + 32: what began last
        int v[2] = {tile.id[lane], tile.id[lane + 32]};
        const uint32_t under = (1u << lane) - 1u, upto = under | 1u << lane;
        const uint32_t low = __ballot_sync(0xffffffffu, v[0] != -2), high = __ballot_sync(0xffffffffu, v[1] != -2);
        const int last = __shfl_sync(0xffffffffu, v[0], low ? 31 - __clz(low) : 0);
        const int v0 = __shfl_sync(0xffffffffu, v[0], low & upto ? 31 - __clz(low & upto) : lane), v1 = __shfl_sync(0xffffffffu, v[1], high & upto ? 31 - __clz(high & upto) : lane);
        v[0] = t0 + lane < end ? v0 : -1;
        v[1] = t0 + lane + 32 < end ? (high & upto ? v1 : last) : -1;
        int n = 0, at = 0;
        for (;;) {
            const uint32_t left = __ballot_sync(0xffffffffu, v[0] >= 0), more = __ballot_sync(0xffffffffu, v[1] >= 0);
            if (!(left | more)) break;
            const int id = left ? __shfl_sync(0xffffffffu, v[0], __ffs(left) - 1) : __shfl_sync(0xffffffffu, v[1], __ffs(more) - 1);
            const uint32_t here = __ballot_sync(0xffffffffu, v[0] == id), there = __ballot_sync(0xffffffffu, v[1] == id);
            if (v[0] == id) { tile.row[at + __popc(here & under)] = lane; v[0] = -1; }
            if (v[1] == id) { tile.row[at + __popc(here) + __popc(there & under)] = lane + 32; v[1] = -1; }
            if (lane == 0) { tile.adapter[n] = id; tile.first[n] = at; }
            at += __popc(here) + __popc(there);
            n++;
        }
        if (lane == 0) { tile.n = n; tile.first[n] = at; }
    }
    __syncthreads();
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
    return r;
}

// Shared memory: two stages of 4 KB a warp, in which every lane finds what it asked for itself (so nobody waits for a neighbour), and in their place the
// sums of the warps on their way together; h as two 16-bit values; the block's part of h.  The first product takes 32 tokens at a time, 64 in a launch of
// its own, whose stages are of 6 KB: A is read half as often.
struct Lora {
    static constexpr int kStage = 8 * 512, kRing = LORA_WARPS * 2 * kStage, kRingFirst = LORA_WARPS * 2 * 12 * 512;
    static constexpr int kRingWide = LORA_WARPS * TM * (64 + 4) * 4;                           // 64 rows of A at a time: the sums are larger than the stages
    static __host__ __device__ int steps(int rank) { return (rank + 15) / 16; }
    // h as the second product's A operand: for each split, step of 16 and tile of 16 tokens 16 bytes a lane of high parts, then of low parts
    static constexpr int kFrag = 1024, kStep = TM / 16 * kFrag;
    static int parts(int rank, int together) { return TM * together * rank * 4; }
    static int smem(int rank, int together) { return kRing + together * steps(rank) * kStep; }
};

// First product: A operand 32 rows of the adapter, B operand 8 tokens, both from global memory, 16 bytes a lane: eight neighbours of a row are two steps' k
// = 2t, 2t + 1, 2t + 8, 2t + 9 of lane t, in the same order on both sides.  The eight warps share K; with more than 32 rows of A groups
// of them take 32 rows each in the one launch, and their warps share K.
// Second: A operand h of 16 tokens as two 16-bit values each, the second with what rounding the first left: 2^-16 of h stays out in bf16, 2^-22 in fp16, beside `out`'s
// rounding of 2^-8 and 2^-11.  fp16's lie a power of two off, which brings the row's largest to 2^14.  B operand 8 columns; column 2t + e of n-tile j is column 8t + 2j + e of the warp's 32, so that a lane
// holds 16 bytes of a row of `out`.  STEPS: of 16 in the rank, B in registers; 0: any number, B as it comes.  With an even number a lane reads 16 bytes of B, in the first product's order
// of two steps' k.  (The first product alone: 4 for up to 4.)
enum { LORA_BOTH, LORA_FIRST, LORA_WIDE, LORA_SECOND };                                      // WIDE: the first where A has more than 32 rows, 64 of them at a time
template <bool BF, int STEPS, int DO>
__global__ void __launch_bounds__(LORA_THREADS, DO == LORA_WIDE ? 1 : 2) lora_kernel(const LoraArgs A) {
    using L = Lora;
    constexpr bool WIDE = STEPS == 2 || STEPS == 4;
    constexpr bool FIRST = DO == LORA_FIRST || DO == LORA_WIDE;
    // of the first product: tiles of 8 tokens and of 16 rows of A; a warp's stores of sums meet every bank once
    constexpr int NT = FIRST ? 8 : 4, TOKS = 8 * NT, MT = DO == LORA_WIDE ? 4 : 2, ROWS = 16 * MT, PITCH = ROWS + 4, STAGE = (NT + 2 * MT) * 512;
    constexpr int RING = DO == LORA_WIDE ? L::kRingWide : FIRST ? L::kRingFirst : L::kRing;
    static_assert(RING >= LORA_WARPS * 2 * STAGE && RING >= LORA_WARPS * TOKS * PITCH * 4, "the stages fit, and the sums");
    __shared__ std::conditional_t<DO == LORA_BOTH, Tile, Rows> tile;
    __shared__ float back[TM][LORA_SPLITS];                    // what undoes a row's power of two
    extern __shared__ __align__(128) uint8_t lora_smem[];
    uint32_t rank = blockIdx.x % A.shares, blocks = A.shares;
    if (DO != LORA_SECOND) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
    }
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t t0 = DO == LORA_BOTH ? (int64_t)(blockIdx.x / blocks) * TM : 0;
    const int steps = STEPS && !FIRST ? STEPS : L::steps(A.rank);
    float* const sums = reinterpret_cast<float*>(lora_smem);
    float* const part = reinterpret_cast<float*>(lora_smem + RING + (FIRST ? 0 : A.together * steps * L::kStep));
    const uint32_t smem = (uint32_t)__cvta_generic_to_shared(lora_smem), ring = smem + warp * 2 * L::kStage + lane * 16, ring1 = smem + warp * 2 * STAGE + lane * 16, hs = smem + L::kRing;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    int4 piece = {};
    int n_adapters = 1;
    if constexpr (DO == LORA_BOTH) {
        find_adapters(A, t0, tile);
        n_adapters = tile.n;
    } else {
        piece = A.pieces[blockIdx.x / blocks];
        if (piece.z == 0) return;                              // the whole cluster
        if (threadIdx.x < TM) tile.row[threadIdx.x] = A.order[piece.y + min((int)threadIdx.x, piece.z - 1)];
        __syncthreads();
    }
    const int chunks = (A.K + 31) / 32, each = (chunks + (int)blocks - 1) / (int)blocks, from = min((int)rank * each, chunks), to = min(from + each, chunks);
    for (int j = DO == LORA_BOTH ? blockIdx.y : 0; j < n_adapters; j += gridDim.y) {
        int id = piece.x, count = piece.z;
        const int* row_of = tile.row;
        if constexpr (DO == LORA_BOTH) {
            id = tile.adapter[j];
            count = tile.first[j + 1] - tile.first[j];
            row_of += tile.first[j];
        }
        const float scale = A.scales[id];
        const int s_from = FIRST ? blockIdx.y * A.together : 0, s_step = FIRST ? gridDim.y * A.together : A.together;
        for (int s0 = s_from; s0 < A.n_splits; s0 += s_step) {
            const int n_here = min(A.together, A.n_splits - s0), rows = n_here * A.rank;
            const uint4* const w = (const uint4*)((const uint16_t*)A.a + id * A.a_st + (int64_t)s0 * A.rank * A.K);
            // ---- h of this block's share of K.  Rows behind the last, of A and of x, are read as the last ones: nobody looks at what they give
            const int groups = FIRST ? 1 : rows > 2 * ROWS ? 4 : rows > ROWS ? 2 : 1, of_group = LORA_WARPS / groups, nth = warp & (of_group - 1);
            for (int rows0 = 0, i0 = 0; DO != LORA_SECOND && rows0 < rows; i0 = i0 + TOKS < count ? i0 + TOKS : 0, rows0 += i0 ? 0 : ROWS * groups) {
                const int row0 = rows0 + warp / of_group * ROWS, m_end = min(MT, (rows - row0 + 15) / 16), n_end = min(NT, (count - i0 + 7) / 8);
                const int last = m_end > 0 ? to : from;        // nothing for a group behind the last row
                float acc[MT][NT][4] = {};
                uint32_t xs[NT], ws[MT][2];                    // in 16 bytes, of this lane's rows
                const uint4* const x = (const uint4*)((const uint16_t*)A.x + t0 * A.x_st);
#pragma unroll
                for (int n = 0; n < NT; n++) xs[n] = (uint32_t)(row_of[min(i0 + 8 * n + g, count - 1)] * (A.x_st / 8));
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int h = 0; h < 2; h++) ws[m][h] = (uint32_t)min(row0 + 16 * m + 8 * h + g, rows - 1) * (uint32_t)(A.K / 8);
                auto ask = [&](int c, int stage) {
                    const bool in = c < last && 32 * c + 8 * t < A.K;
                    const uint32_t k = in ? 4 * c + t : 0, at = ring1 + stage * STAGE;
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        if (n < n_end) cp16(at + n * 512, x + (xs[n] + k), in);
#pragma unroll
                    for (int m = 0; m < MT; m++)
                        if (m < m_end) {
                            cp16(at + (NT + 2 * m) * 512, w + (ws[m][0] + k), in);
                            cp16(at + (NT + 2 * m + 1) * 512, w + (ws[m][1] + k), in);
                        }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
                __syncthreads();                               // what was in the ring's place is read
                ask(from + nth, 0);
                ask(from + nth + of_group, 1);
                int stage = 0;
#pragma unroll 1
                for (int c = from + nth; c < last; c += of_group, stage ^= 1) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    const uint32_t at = ring1 + stage * STAGE;
                    uint4 wr[MT][2];
#pragma unroll
                    for (int m = 0; m < MT; m++)
                        if (m < m_end) { wr[m][0] = lds16(at + (NT + 2 * m) * 512); wr[m][1] = lds16(at + (NT + 2 * m + 1) * 512); }
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        if (n < n_end) {
                            const uint4 xr = lds16(at + n * 512);
#pragma unroll
                            for (int m = 0; m < MT; m++)
                                if (m < m_end) mma<BF>(acc[m][n], wr[m][0].x, wr[m][1].x, wr[m][0].y, wr[m][1].y, xr.x, xr.y);
#pragma unroll
                            for (int m = 0; m < MT; m++)
                                if (m < m_end) mma<BF>(acc[m][n], wr[m][0].z, wr[m][1].z, wr[m][0].w, wr[m][1].w, xr.z, xr.w);
                        }
                    ask(c + 2 * of_group, stage);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncthreads();                               // everybody is through with the ring
#pragma unroll
                for (int n = 0; n < NT; n++)
                    if (n < n_end) {
#pragma unroll
                        for (int m = 0; m < MT; m++)
                            if (m < m_end) {
#pragma unroll
                                for (int e = 0; e < 4; e++) sums[(warp * TOKS + 8 * n + 2 * t + (e & 1)) * PITCH + 16 * m + g + 8 * (e >> 1)] = acc[m][n][e];
                            }
                    }
                __syncthreads();
#pragma unroll 1
                for (int i = threadIdx.x; i < TOKS * ROWS / 4 * groups; i += LORA_THREADS) {
                    const int tok = i / (ROWS / 4) & (TOKS - 1), group = i / (TOKS * ROWS / 4), in = i % (ROWS / 4) * 4, row = rows0 + group * ROWS + in;
                    if (i0 + tok < count && row < rows) {
                        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                        for (int v = 0; v < LORA_WARPS; v++) {
                            if (v >= of_group) break;
                            const float4 p = *reinterpret_cast<const float4*>(sums + ((group * of_group + v) * TOKS + tok) * PITCH + in);
                            s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
                        }
                        *reinterpret_cast<float4*>(part + (i0 + tok) * rows + row) = s;
                    }
                }
            }
            if (DO != LORA_SECOND) meet(blocks);
            else __syncthreads();                              // what was in the ring's and h's place is read
            // ---- this block's share of the columns, 32 a warp: where its groups lie, and what it asks for ahead.  Rows and columns behind the last are read
            // as the last ones, and not written
            const uint16_t* const wb = (const uint16_t*)A.b + id * A.b_st;
            struct Group {
                int s, before, groups, grp, c0, c_end;
                __device__ __forceinline__ bool settle(const LoraArgs& A, int s0, int n_here) {
                    while (grp - before >= groups) {
                        before += groups;
                        if (++s >= n_here) return false;
                        groups = (A.first[s0 + s + 1] - A.first[s0 + s] + 31) / 32;
                    }
                    c0 = A.first[s0 + s] + 32 * (grp - before);
                    c_end = A.first[s0 + s + 1];
                    return true;
                }
            };
            const int m_tiles = (count + 15) / 16;
            uint32_t row_at[TM / 8];                           // rows 8 i + g of the adapter's, in 16 bytes from t0 on
#pragma unroll
            for (int i = 0; i < TM / 8; i++) row_at[i] = (uint32_t)(row_of[min(8 * i + g, count - 1)] * A.o_st / 8);
            uint4* const out = reinterpret_cast<uint4*>((uint16_t*)A.out + t0 * A.o_st);
            Group ahead = {0, 0, (A.first[s0 + 1] - A.first[s0] + 31) / 32, (int)rank * LORA_WARPS + warp, 0, 0};
            bool more = !FIRST && ahead.settle(A, s0, n_here);
            auto ask_out = [&](int stage) {
                if (more) {
                    const uint4* const from = out + min(ahead.c0 + 8 * t, ahead.c_end - 8) / 8;
#pragma unroll
                    for (int m = 0; m < TM / 16; m++)
                        if (m < m_tiles) {
                            cp16(ring + stage * L::kStage + 2 * m * 512, from + row_at[2 * m], true);
                            cp16(ring + stage * L::kStage + (2 * m + 1) * 512, from + row_at[2 * m + 1], true);
                        }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            ask_out(0);
            // ---- the blocks' parts together: a warp takes a row of the tile in one split
            const uint32_t at_part = (uint32_t)__cvta_generic_to_shared(part), at_back = (uint32_t)__cvta_generic_to_shared(&back[0][0]);
            constexpr int Z = STEPS ? 1 : 4;                   // pairs `lane`, `lane` + 32, ...
            auto place = [&](int tok, int s, float2 (&h)[Z]) {
                float big = 0.0f, down = 1.0f;
#pragma unroll
                for (int z = 0; z < Z; z++) {
                    h[z].x *= scale;
                    h[z].y *= scale;
                    big = fmaxf(big, fmaxf(fabsf(h[z].x), fabsf(h[z].y)));
                }
                const uint32_t others = DO == LORA_BOTH ? blocks : 1;
                if (!BF) {
#pragma unroll
                    for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
                    const int e = (int)(__float_as_uint(big) >> 23) - 127 - 14, use = big > 0.0f && big < INFINITY ? max(e, -100) : 0;
                    const float up = __uint_as_float((uint32_t)(127 + use) << 23);
                    down = __uint_as_float((uint32_t)(127 - use) << 23);
                    if (FIRST) {
                        if (lane == 0) A.back[(int64_t)(piece.y + tok) * A.n_splits + s0 + s] = up;
                    } else if (lane < (int)others) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(shared_of(at_back + (tok * LORA_SPLITS + s) * 4, lane)), "f"(up) : "memory");
                }
#pragma unroll
                for (int z = 0; z < Z; z++) {
                    const int r = 2 * lane + 64 * z;
                    if (r >= 16 * steps) continue;
                    const float x = h[z].x * down, y = h[z].y * down;
                    const uint32_t hi = pack2<BF>(x, y);
                    const float2 f = unpack2<BF>(hi);
                    const uint32_t lo = pack2<BF>(fabsf(f.x) < INFINITY ? x - f.x : 0.0f, fabsf(f.y) < INFINITY ? y - f.y : 0.0f);
                    if (FIRST) {
                        uint16_t* const to = A.h + (int64_t)(piece.y + tok) * (A.n_splits * 32 * steps) + (s0 + s) * 32 * steps + r;
                        *reinterpret_cast<uint32_t*>(to) = hi;
                        *reinterpret_cast<uint32_t*>(to + 16 * steps) = lo;
                    } else {
                        const uint32_t at = hs + (s * steps + (WIDE ? r / 32 * 2 + (r >> 2 & 1) : r / 16)) * L::kStep + tok / 16 * L::kFrag +
                                            ((tok & 7) * 4 + (WIDE ? r / 8 & 3 : r / 4 & 3)) * 16 + (tok & 8) + (r & 2) * 2;
#pragma unroll 8
                        for (uint32_t b = 0; b < blocks; b++) {
                            const uint32_t p = shared_of(at, b);
                            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(p), "r"(hi) : "memory");
                            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(p + L::kFrag / 2), "r"(lo) : "memory");
                        }
                    }
                }
            };
            if constexpr (DO == LORA_SECOND) {
                // 16 bytes, a row's eight neighbours, a thread: two lanes' share of a fragment, or a lane's of two
                const int pieces = n_here * steps * 4;         // of a row: two of high parts, two of low ones a step
                for (int i = threadIdx.x; i < count * pieces; i += LORA_THREADS) {
                    const int tok = i / pieces, in = i - tok * pieces, s = in / (4 * steps), half = in / (2 * steps) & 1, r = in % (2 * steps) * 8;
                    const uint4 v = *reinterpret_cast<const uint4*>(A.h + (int64_t)(piece.y + tok) * (A.n_splits * 32 * steps) + s0 * 32 * steps + in * 8);
                    const uint32_t at = hs + (s * steps + (WIDE ? r / 32 * 2 : r / 16)) * L::kStep + tok / 16 * L::kFrag + half * (L::kFrag / 2) +
                                        ((tok & 7) * 4 + (WIDE ? r / 8 & 3 : r / 4 & 2)) * 16 + (tok & 8);
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(v.x), "r"(v.y) : "memory");
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + (WIDE ? L::kStep : 16)), "r"(v.z), "r"(v.w) : "memory");
                }
                if (!BF)
                    for (int i = threadIdx.x; i < count * n_here; i += LORA_THREADS) back[i / n_here][i % n_here] = A.back[(int64_t)(piece.y + i / n_here) * A.n_splits + s0 + i % n_here];
            } else {
                for (int i = (int)rank + warp * (int)blocks; i < count * n_here; i += LORA_WARPS * (int)blocks) {
                    const int tok = i % count, s = i / count;
                    float2 h[Z];
#pragma unroll
                    for (int z = 0; z < Z; z++) {
                        h[z] = make_float2(0.0f, 0.0f);
                        const int r = 2 * lane + 64 * z;
                        if (r < A.rank) {
                            const uint32_t at = at_part + (tok * rows + s * A.rank + r) * 4;
#pragma unroll 8
                            for (uint32_t b = 0; b < blocks; b++) {
                                float2 p;
                                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(p.x), "=f"(p.y) : "r"(shared_of(at, b)) : "memory");
                                h[z].x += p.x;
                                h[z].y += p.y;
                            }
                        }
                    }
                    place(tok, s, h);
                }
            }
            if (FIRST) {
                meet(blocks);                                  // the parts are read: they may be written again, and their block may leave
                continue;
            }
            const int off = (8 * (g >> 1) + (g & 1)) * A.rank + (WIDE ? 8 : 4) * t;            // this lane's rows of B are 2 n further on
            // step `st`, or, WIDE, that and the next
            auto fetch = [&](const Group& of, int st, uint2 (*br)[4]) {
                const uint16_t* const p = wb + (int64_t)of.c0 * A.rank + 16 * st;
                auto take = [&](int n, bool there) {
                    if constexpr (WIDE) {
                        const uint4 v = there ? *reinterpret_cast<const uint4*>(p + (off + 2 * n * A.rank)) : make_uint4(0, 0, 0, 0);
                        br[0][n] = make_uint2(v.x, v.y);
                        br[1][n] = make_uint2(v.z, v.w);
                    } else br[0][n] = there ? *reinterpret_cast<const uint2*>(p + (off + 2 * n * A.rank)) : make_uint2(0, 0);
                };
                if (of.c0 + 32 <= of.c_end && 16 * st + (WIDE ? 32 : 16) <= A.rank) {
#pragma unroll
                    for (int n = 0; n < 4; n++) take(n, true);
                } else {
#pragma unroll
                    for (int n = 0; n < 4; n++) take(n, of.c0 + 8 * (g >> 1) + 2 * n + (g & 1) < of.c_end && 16 * st + (WIDE ? 8 : 4) * t < A.rank);
                }
            };
            uint2 br[STEPS ? STEPS : 2][4];
            if (!STEPS && more) fetch(ahead, 0, br);
            if (STEPS && more) {
#pragma unroll
                for (int st = 0; st < STEPS; st += WIDE ? 2 : 1) fetch(ahead, st, br + st);
            }
            if (DO == LORA_BOTH) meet(blocks);
            else __syncthreads();
#pragma unroll 1
            for (int stage = 0; more; stage ^= 1) {
                const Group now = ahead;
                ahead.grp += (int)blocks * LORA_WARPS;
                more = ahead.settle(A, s0, n_here);
                ask_out(stage ^ 1);
                const int col = now.c0 + 8 * t;
                uint4* const to = out + col / 8;
                const uint32_t h0 = hs + now.s * steps * L::kStep + lane * 16, o0 = ring + stage * L::kStage;
                const int rows_here = col < now.c_end ? count - g : 0;
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                // 16 tokens at a time; what the next ones need of h is asked for behind the products, ahead of what is done with them.  With B as it comes 32
                constexpr int P = STEPS ? 1 : 2;
                constexpr bool EARLY = STEPS == 1 || STEPS == 2;                                    // four steps of h and of B are more than the registers hold
                constexpr int S = EARLY ? STEPS : 1;
                uint4 hi[S][P], lo[S][P];
                auto ask_h = [&](int m, int st, uint4 (&hi_)[P], uint4 (&lo_)[P]) {
#pragma unroll
                    for (int q = 0; q < P; q++)
                        if (m + q < m_tiles) {
                            const uint32_t h = h0 + st * L::kStep + (m + q) * L::kFrag;
                            hi_[q] = lds16(h);
                            lo_[q] = lds16(h + L::kFrag / 2);
                        }
                };
                if constexpr (EARLY) {
#pragma unroll
                    for (int st = 0; st < STEPS; st++) ask_h(0, st, hi[st], lo[st]);
                }
#pragma unroll
                for (int m = 0; m < TM / 16; m += P) {
                    if (m >= m_tiles) break;
                    uint4 o[P][2];
#pragma unroll
                    for (int q = 0; q < P; q++)
#pragma unroll
                        for (int h = 0; h < 2; h++) o[q][h] = lds16(o0 + (2 * (m + q) + h) * 512);
                    float acc[P][4][4];
                    auto products = [&](const uint4 (&hi_)[P], const uint4 (&lo_)[P], const uint2 (&b)[4], bool first) {
#pragma unroll
                        for (int q = 0; q < P; q++)
                            if (m + q < m_tiles) {
#pragma unroll
                                for (int n = 0; n < 4; n++) {
                                    if (first) mma0<BF>(acc[q][n], lo_[q].x, lo_[q].z, lo_[q].y, lo_[q].w, b[n].x, b[n].y);
                                    else mma<BF>(acc[q][n], lo_[q].x, lo_[q].z, lo_[q].y, lo_[q].w, b[n].x, b[n].y);
                                }
#pragma unroll
                                for (int n = 0; n < 4; n++) mma<BF>(acc[q][n], hi_[q].x, hi_[q].z, hi_[q].y, hi_[q].w, b[n].x, b[n].y);
                            }
                    };
                    if constexpr (STEPS > 0) {
#pragma unroll
                        for (int st = 0; st < STEPS; st++) {
                            if (!EARLY) ask_h(m, st, hi[0], lo[0]);
                            products(hi[EARLY ? st : 0], lo[EARLY ? st : 0], br[st], st == 0);
                        }
                        if (m + 1 < m_tiles && m + 1 < TM / 16) {
                            if constexpr (EARLY) {
#pragma unroll
                                for (int st = 0; st < STEPS; st++) ask_h(m + 1, st, hi[st], lo[st]);
                            }
                        } else if (more) {                     // the products have B: the next group's
#pragma unroll
                            for (int st = 0; st < STEPS; st += WIDE ? 2 : 1) fetch(ahead, st, br + st);
                        }
                    } else {
                        if (m > 0) fetch(now, 0, br);
                        auto step = [&](int st, int at, bool first) {
                            if (st + 1 < steps) fetch(now, st + 1, br + (at ^ 1));
                            ask_h(m, st, hi[0], lo[0]);
                            products(hi[0], lo[0], br[at], first);
                        };
                        step(0, 0, true);
#pragma unroll 1
                        for (int st = 1; st < steps; st += 2) {
                            step(st, 1, false);
                            if (st + 1 < steps) step(st + 1, 0, false);
                        }
                        if (m + P >= m_tiles && more) fetch(ahead, 0, br);
                    }
#pragma unroll
                    for (int q = 0; q < P; q++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int i = 16 * (m + q) + 8 * h;
                            if (i >= rows_here) continue;
                            uint32_t v[4] = {o[q][h].x, o[q][h].y, o[q][h].z, o[q][h].w};
                            const float up = BF ? 1.0f : back[i + g][now.s];
#pragma unroll
                            for (int n = 0; n < 4; n++)
                                v[n] = add2<BF>(v[n], BF ? acc[q][n][2 * h] : acc[q][n][2 * h] * up, BF ? acc[q][n][2 * h + 1] : acc[q][n][2 * h + 1] * up);
                            to[row_at[2 * (m + q) + h]] = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    }
}

// ------------------------------------------------------------------ many tokens: the rows ordered by their adapters
constexpr int SORT_THREADS = 512, SORT_HERE = 4096;            // adapters whose lists lie in shared memory
template <bool MOST> __device__ __forceinline__ int scan(int x, int* warps, int& all) {        // inclusive sums, or maxima, over the block; all: of the whole block
    auto both = [](int a, int b) { return MOST ? max(a, b) : a + b; };
    constexpr int none = MOST ? (int)0x80000000 : 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x = both(x, y);
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    int w = lane < SORT_THREADS / 32 ? warps[lane] : none;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, d);
        if (lane >= d) w = both(w, y);
    }
    all = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    return both(x, warp ? before : none);
}
// One block: rows counted by adapter, a place for each adapter's, the pieces of 64, the rows written to their places.  In which order the rows of an adapter lie is
// chance, and nothing depends on it: a row's sums are its own.  Rows [row0, row0 + rows) count from 0; n_pieces: room for pieces.  It waits for barriers and for
// memory, some 6 us (1024 threads one more); 882 rows of 40 requests and 12 adapters become 23 pieces, of which tiles of neighbours' rows had some 50.
__global__ void __launch_bounds__(SORT_THREADS, 1) lora_order_kernel(const LoraArgs A, int64_t row0, int rows, int n_pieces) {
    __shared__ int warps[32];
    __shared__ int here[2][SORT_HERE];
    __shared__ int few[SORT_THREADS], few_n[SORT_THREADS], few_at[SORT_THREADS];               // stretches of rows: for a warp each from the front, for the block from the back
    __shared__ int n_few, n_more;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int* const place = A.adapters <= SORT_HERE ? here[0] : A.lists;                           // rows of an adapter, then where they begin
    int* const before = A.adapters <= SORT_HERE ? here[1] : A.lists + A.adapters;              // pieces of the adapters in front
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    for (int a = t; a < A.adapters; a += SORT_THREADS) place[a] = 0;
    const int64_t end = min((int64_t)A.cu[A.R], row0 + rows);
    // of request r0 + t: adapter, first row and number of rows; `seen`: where the requests in front end.  A list that goes back names no row twice
    int id = -1, lo = 0, n = 0;
    auto look = [&](int r0, int& seen) {
        const int r = r0 + t;
        const int c = r < A.R ? A.cu[r] : (int)0x80000000;
        const int64_t to = r < A.R ? min((int64_t)A.cu[r + 1], end) : 0;
        id = r < A.R ? A.ids[r] : -1;
        int all;
        const int most = scan<true>(c, warps, all);
        const int64_t from = max((int64_t)max(most, seen), row0);
        seen = max(seen, all);
        if (id < 0 || id >= A.adapters || from >= to) { id = -1; n = 0; }
        else { lo = (int)(from - row0); n = (int)(to - from); }
    };
    int seen = (int)0x80000000;
    __syncthreads();
    for (int r0 = 0; r0 < A.R; r0 += SORT_THREADS) {
        look(r0, seen);
        // one addition for the requests of an adapter in a warp
        if (r0 + 32 * warp >= A.R) continue;
        const uint32_t same = __match_any_sync(0xffffffffu, id);
        const int sum = __reduce_add_sync(same, n);
        if (id >= 0 && lane == __ffs(same) - 1) atomicAdd(place + id, sum);
    }
    __syncthreads();
    int row_at = 0, piece_at = 0;
    for (int a0 = 0; a0 < A.adapters; a0 += SORT_THREADS) {
        const int a = a0 + t, c = a < A.adapters ? place[a] : 0, p = (c + TM - 1) / TM;
        int all_rows, all_pieces;
        const int r = scan<false>(c, warps, all_rows), q = scan<false>(p, warps, all_pieces);
        if (a < A.adapters) { place[a] = row_at + r - c; before[a] = piece_at + q - p; }
        row_at += all_rows;
        piece_at += all_pieces;
    }
    __syncthreads();
    for (int i = t; i < n_pieces; i += SORT_THREADS) {
        int4 piece = make_int4(0, 0, 0, 0);
        if (i < piece_at) {
            int a = 0, last = A.adapters - 1;                  // the last adapter with no more pieces in front
            while (a < last) {
                const int mid = (a + last + 1) >> 1;
                if (before[mid] <= i) a = mid;
                else last = mid - 1;
            }
            const int first = place[a] + TM * (i - before[a]), stop = a + 1 < A.adapters ? place[a + 1] : row_at;
            piece = make_int4(a, first, min(TM, stop - first), 0);
        }
        A.pieces[i] = piece;
    }
    seen = (int)0x80000000;
    for (int r0 = 0; r0 < A.R; r0 += SORT_THREADS) {
        __syncthreads();
        if (t == 0) n_few = n_more = 0;
        if (A.R > SORT_THREADS) look(r0, seen);
        __syncthreads();
        if (r0 + 32 * warp < A.R) {
            const uint32_t same = __match_any_sync(0xffffffffu, id);
            const int sum = __reduce_add_sync(same, n), leader = __ffs(same) - 1;
            int at = id >= 0 && lane == leader ? atomicAdd(place + id, sum) : 0;
            at = __shfl_sync(0xffffffffu, at, leader);
#pragma unroll
            for (int l = 0; l < 31; l++) {
                const int v = __shfl_sync(0xffffffffu, n, l);
                if (l < lane && same >> l & 1) at += v;
            }
            if (n <= 4) {
                for (int k = 0; k < n; k++) A.order[at + k] = lo + k;
            } else {
                const int e = n <= 1024 ? atomicAdd(&n_few, 1) : SORT_THREADS - 1 - atomicAdd(&n_more, 1);
                few[e] = lo; few_n[e] = n; few_at[e] = at;
            }
        }
        __syncthreads();
        for (int e = warp; e < n_few; e += SORT_THREADS / 32)
            for (int k = lane; k < few_n[e]; k += 32) A.order[few_at[e] + k] = few[e] + k;
        for (int e = SORT_THREADS - n_more; e < SORT_THREADS; e++)
            for (int k = t; k < few_n[e]; k += SORT_THREADS) A.order[few_at[e] + k] = few[e] + k;
    }
}

// One launch or three.  One has a cluster for each adapter of a tile: where these are more than the device takes at once three take less time, and where they are few and
// a cluster's columns many.  K 4096, N 4096, rank 16: 64 tokens of 32 adapters 12 us by one, 17 by three; 256 of 8 9 and 16; 150 of 30 31 and 17; 256 of 64 111 and 25.
// N 22016: 16 tokens of one adapter 12 and 13, 64 24 and 18; at rank 64 22 and 16, 51 and 27; at rank 128 4 tokens 49 and 27, 64 124 and 53.
// K 14336, N 4096, 64 tokens at rank 64: 39 and 32, at rank 16 16 and 22.
constexpr int LORA_BLOCKS = 8;                                 // of a cluster: the most that any device takes
int64_t lora_tile_adapters(int adapters, int R) { const int64_t most = adapters < R ? adapters : R; return most < TM ? most : TM; }
// splits that share a reading of x: 128 rows of A at most (their parts and h fill what shared memory two blocks of an SM have), or one split
int lora_together(int rank, int n_splits) { return n_splits * rank <= 128 ? n_splits : rank >= 128 ? 1 : 128 / rank; }
bool lora_many(int64_t T, int64_t K, int64_t N, int rank, int n_splits, int adapters, int R) {
    const int together = lora_together(rank, n_splits);
    const bool alone = together * rank > 64;                                                   // a block fills its SM's shared memory
    const int64_t blocks = (T + TM - 1) / TM * lora_tile_adapters(adapters, R) * LORA_BLOCKS, places = (alone ? 1ll : 2ll) * sm_count();
    if (blocks > places) return true;
    // groups of columns a warp, by what one costs: itself, its tokens, its steps; and 32 k's of 32 rows of A and 32 tokens by what they cost beside those.  With half the
    // device busy only large ranks are worth the launches
    const int64_t tokens = T / (adapters < R ? adapters : R), each = tokens < 1 ? 1 : tokens < TM ? tokens : TM, much = 400ll * LORA_BLOCKS * LORA_WARPS;
    const int64_t work = N / 32 * (each + 16 + 4 * Lora::steps(rank)) + K / 32 * ((n_splits * rank + 31) / 32) * ((each + 31) / 32) * 8;
    return 2 * blocks <= places ? work >= much : Lora::steps(rank) >= 4 && work >= (alone ? much : much * 3 / 2);
}
// pieces that T rows of R requests may have: of whole 64, and one of every adapter
int64_t lora_pieces(int64_t T, int adapters, int R) { int64_t most = adapters < R ? adapters : R; if (most > T) most = T; return T / TM + most; }
size_t lora_lists_bytes(int64_t T, int adapters, int R) {
    return (size_t)lora_pieces(T, adapters, R) * sizeof(int4) + ((size_t)T + (adapters > SORT_HERE ? 2 * (size_t)adapters : 0) + 3) / 4 * 16;
}

template <bool BF, int STEPS> int lora_launch(LoraArgs A, int64_t row0, cudaStream_t st) {
    A.together = lora_together(A.rank, A.n_splits);
    static bool configured[64] = {};                           // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        cudaFuncSetAttribute(lora_kernel<BF, STEPS, LORA_BOTH>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lora::smem(256, 1) + Lora::parts(256, 1));
        cudaFuncSetAttribute(lora_kernel<BF, 4, LORA_FIRST>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lora::kRingFirst + Lora::parts(32, 1));
        cudaFuncSetAttribute(lora_kernel<BF, STEPS ? 4 : 0, LORA_WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lora::kRingWide + Lora::parts(256, 1));
        cudaFuncSetAttribute(lora_kernel<BF, STEPS, LORA_SECOND>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lora::smem(256, 1));
        configured[dev & 63] = true;
    }
    const bool many = A.pieces != nullptr;
    const bool on = launch_overlaps(st);
    // clusters of tiles, and those that share a tile's adapters: twice as many as a tile has on average, since neighbours' differ; those that find none leave at
    // once.  Or of pieces
    const int64_t tiles = many ? lora_pieces(A.T, A.adapters, A.R) : (A.T + TM - 1) / TM;
    int64_t some = 1 + (int64_t)A.R * TM * 2 / A.T;
    if (some > lora_tile_adapters(A.adapters, A.R)) some = lora_tile_adapters(A.adapters, A.R);
    // splits one after the other share a reading of x, or, where there is room for their clusters, each has its own
    if (many) some = 1;
    if (many && tiles * LORA_BLOCKS * A.n_splits <= (A.rank > 32 ? 1ll : 2ll) * sm_count()) { A.together = 1; some = A.n_splits; }
    // 64 rows of A at a time by a block that has its SM to itself: more work for what it reads, one pass for ranks up to 64.  Rank 128, K 4096, N 896: 12000 tokens 148 us
    // and 192 by 32 rows at a time, 3000 83 and 108, 600 50 and 54; rank 64, K 11008, N 4096: 175 and 215, 74 and 79, 39 and 39
    const bool wide = many && A.together * A.rank > 32;
    // blocks of a cluster, which share the inner dimension (and the columns): 8 (one token 7.1 us, by 4, 2 and 1 8.8, 11.8 and
    // 17.1; 64 tokens 13.2, and 14.3, 19.2, 28.1), fewer where the pieces fill the device: at 32 rows of A 11849 tokens by 2 blocks of a piece 141 us, by
    // 4 143, by 8 152.  At 64 as many as the device takes at once (882 tokens of 40 requests by 5 blocks 41 us, by 7 49), two at least (12000 by one 154, 148)
    int blocks = LORA_BLOCKS;
    if (wide) {
        while (blocks > 2 && tiles * some * blocks > sm_count()) blocks--;
    } else
        while (many && blocks > 1 && tiles * blocks >= 4ll * sm_count()) blocks /= 2;
    if (many) {
        launch_behind(lora_order_kernel, dim3(1), SORT_THREADS, 0, st, on, A, row0, (int)A.T, (int)tiles);
        note_launch();
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * blocks), (unsigned)some);
    cfg.blockDim = dim3(LORA_THREADS);
    cfg.dynamicSmemBytes = (size_t)(wide ? Lora::kRingWide : many ? Lora::kRingFirst : Lora::smem(A.rank, A.together)) + Lora::parts(A.rank, A.together);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)blocks, 1u, 1u};
    cfg.attrs = at;
    cfg.numAttrs = add_overlap(at, 1, on);
    A.shares = 1;
    cudaLaunchKernelEx(&cfg, wide ? lora_kernel<BF, STEPS ? 4 : 0, LORA_WIDE> : many ? lora_kernel<BF, 4, LORA_FIRST> : lora_kernel<BF, STEPS, LORA_BOTH>, A);
    note_launch();
    if (many) {
        A.together = lora_together(A.rank, A.n_splits);
        // blocks of a piece's columns: eight an SM's two places (11849 rows by 8 shares of a piece 147 us, by 4 150, by 16 173, in an earlier form), none with fewer than three groups a
        // warp, which would read h more often than it uses it
        const int64_t want = 8ll * sm_count() / tiles, room = A.first[A.n_splits] / (32 * LORA_WARPS * 3);
        A.shares = (int)(want < 8 ? 8 : want);
        if (A.shares > room) A.shares = (int)room;
        if (A.shares < 1) A.shares = 1;
        launch_behind(lora_kernel<BF, STEPS, LORA_SECOND>, dim3((unsigned)(tiles * A.shares)), LORA_THREADS, (size_t)Lora::smem(A.rank, A.together), st, on, A);
        note_launch();
    }
    return check_launch();
}

// B in registers for the ranks that adapters mostly have; other steps would cost a kernel each for less
template <bool BF> int lora_steps(const LoraArgs& A, int64_t row0, cudaStream_t st) {
    return A.rank <= 16 ? lora_launch<BF, 1>(A, row0, st) : A.rank <= 32 ? lora_launch<BF, 2>(A, row0, st) : A.rank <= 64 && A.rank > 48 ? lora_launch<BF, 4>(A, row0, st)
                                                                                                                  : lora_launch<BF, 0>(A, row0, st);
}

}  // namespace
}  // namespace lowbit

extern "C" size_t lowbit_lora_workspace_size(int64_t T, int K, int64_t N, int rank, int n_splits, int adapters, int R) {
    if (T <= 0 || K <= 0 || N <= 0 || rank <= 0 || n_splits <= 0 || adapters <= 0 || R <= 0 || !lora_many(T, K, N, rank, n_splits, adapters, R)) return 0;
    return lora_lists_bytes(T, adapters, R) + (size_t)T * n_splits * (Lora::steps(rank) * 64 + sizeof(float));
}

extern "C" int lowbit_lora_add_cuda(const void* d_x, int64_t x_stride, int dtype, int64_t T, int K, const void* d_a, int64_t a_stride, const void* d_b, int64_t b_stride,
                                    int rank, const float* d_scales, int adapters, const int32_t* d_ids, const int32_t* d_cu_seqlens, int R, const int* splits, int n_splits,
                                    void* d_out, int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    reset_launch_count();
    const char* const name = "lowbit_lora_add_cuda";
    bool bad = !d_x || !d_a || !d_b || !d_scales || !d_ids || !d_cu_seqlens || !d_out || !splits || (dtype != DT_F16 && dtype != DT_BF16) || T < 0 || T > 0x7fffffffll || K <= 0 ||
               K % 8 || K > 1 << 20 || rank <= 0 || rank % 8 || rank > 256 || adapters <= 0 || R <= 0 || n_splits <= 0 || n_splits > LORA_SPLITS || x_stride < K;
    int64_t N = 0;
    for (int i = 0; !bad && i < n_splits; i++) { bad = splits[i] <= 0 || splits[i] % 8; N += splits[i]; }
    bad = bad || N > 0x7fffff00ll || out_stride < N || a_stride < (int64_t)n_splits * rank * K || b_stride < N * rank || out_stride > 1 << 29 || x_stride > 1 << 29;
    if (bad) {
        set_error(LB_ERR_ARG, "%s: bad argument (T %lld, K %d, N %lld, rank %d, adapters %d, requests %d, splits %d, dtype %d)", name, (long long)T, K, (long long)N, rank, adapters, R,
                  n_splits, dtype);
        return LB_ERR_ARG;
    }
    if ((((uintptr_t)d_x | (uintptr_t)d_a | (uintptr_t)d_b | (uintptr_t)d_out) & 15) || ((x_stride | a_stride | b_stride | out_stride) & 7)) {
        set_error(LB_ERR_ARG, "%s: activations, weights and output must be 16-byte aligned (pointers and strides)", name);
        return LB_ERR_ARG;
    }
    if (T == 0) return LB_OK;
    const size_t need = lowbit_lora_workspace_size(T, K, N, rank, n_splits, adapters, R);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) {
        set_error(LB_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of lowbit_lora_workspace_size() bytes is needed", name);
        return LB_ERR_WORKSPACE;
    }
    LoraArgs A = {d_x, x_stride, T, K, d_a, a_stride, d_b, b_stride, d_scales, adapters, d_ids, d_cu_seqlens, R, d_out, out_stride, rank, n_splits, 0,
                  nullptr, nullptr, nullptr, nullptr, nullptr, 0, {}};
    for (int i = 0; i < n_splits; i++) A.first[i + 1] = A.first[i] + splits[i];
    cudaStream_t st = (cudaStream_t)stream;
    if (!need) return dtype == DT_BF16 ? lora_steps<true>(A, 0, st) : lora_steps<false>(A, 0, st);
    uint8_t* const w = (uint8_t*)workspace;
    A.pieces = (int4*)w;
    A.order = (int32_t*)(w + lora_pieces(T, adapters, R) * sizeof(int4));
    A.lists = A.order + T;
    A.h = (uint16_t*)(w + lora_lists_bytes(T, adapters, R));
    A.back = (float*)(A.h + T * n_splits * Lora::steps(rank) * 32);
    // a row's offset has 32 bits, in 16 bytes: as many rows at a time as that reaches
    const int64_t stride = x_stride > out_stride ? x_stride : out_stride;
    int64_t rows = (1ll << 35) / stride / TM * TM;             // 64 at least
    for (int64_t row0 = 0; row0 < T; row0 += rows) {
        LoraArgs part = A;
        part.T = T - row0 < rows ? T - row0 : rows;
        part.x = (const uint16_t*)d_x + row0 * x_stride;
        part.out = (uint16_t*)d_out + row0 * out_stride;
        if (const int rc = dtype == DT_BF16 ? lora_steps<true>(part, row0, st) : lora_steps<false>(part, row0, st)) return rc;
    }
    return LB_OK;
}
