// lora.cu -- low-rank adapters of many requests beside a projection that all share:
//   out[t] += scale_l (x[t] A_l^T) B_l^T,      l = the adapter of the token's request (none: the row stays as it is).
//
// One launch.  A cluster takes a tile of packed rows, whoever they belong to: it finds the tile's requests in the list, and the different adapters among
// its rows are dealt to the clusters that share the tile.  So an adapter that neighbours have in common is read once for them, and nobody sorts.  For each:
//   every block multiplies its share of the inner dimension, h = x A^T in 32 bits;
//   the blocks add up their parts, a share of the rows each, and hand the sums to all through their shared memories;
//   every block multiplies its share of the columns, h B^T, and adds that to `out`, rounded once.
// mma.sync m16n8k16: rank and tokens are far below a tcgen05 tile, and what bounds the kernel is what it reads and writes (x; out, twice).
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
    int first[LORA_SPLITS + 1];                                // columns in front of a split
};

template <bool BF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF) asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                         : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// the different adapters among a tile's rows, and the rows of each
template <int TM> struct Tile {
    int id[TM];
    int n, adapter[TM];
    uint64_t rows[TM];
};
// the whole block; ends behind a barrier
template <int TM> __device__ __forceinline__ void find_adapters(const LoraArgs& A, int64_t t0, Tile<TM>& tile) {
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < TM; i += LORA_THREADS) tile.id[i] = -1;
    __syncthreads();
    for (int r = threadIdx.x; r < A.R; r += LORA_THREADS) {
        const int64_t a = max((int64_t)A.cu[r], t0), b = min(min((int64_t)A.cu[r + 1], A.T), t0 + TM);
        const int id = A.ids[r];
        if (a < b && id >= 0 && id < A.adapters)
            for (int64_t t = a; t < b; t++) tile.id[t - t0] = id;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        // rows `lane` and, of tiles with more, `lane` + 32
        int v[2] = {lane < TM ? tile.id[lane] : -1, TM > 32 ? tile.id[lane + 32 < TM ? lane + 32 : 0] : -1};
        int n = 0;
#pragma unroll
        for (int h = 0; h < (TM > 32 ? 2 : 1); h++)
            for (uint32_t left = __ballot_sync(0xffffffffu, v[h] >= 0); left; left = __ballot_sync(0xffffffffu, v[h] >= 0)) {
                const int id = __shfl_sync(0xffffffffu, v[h], __ffs(left) - 1);
                const uint32_t low = __ballot_sync(0xffffffffu, v[0] == id), high = __ballot_sync(0xffffffffu, v[1] == id);
                if (lane == 0) { tile.adapter[n] = id; tile.rows[n] = (uint64_t)high << 32 | low; }
                if (v[0] == id) v[0] = -1;
                if (v[1] == id) v[1] = -1;
                n++;
            }
        if (lane == 0) tile.n = n;
    }
    __syncthreads();
}

// Sizes of a tile of TM rows: warps in KG groups of the inner dimension and TG of the rows, 16 MT rows of A at a time
template <int TM> struct Lora {
    static constexpr int TG = TM > 16 ? 2 : 1, KG = LORA_WARPS / TG, NT = TM / 8 / TG, MT = TM > 16 ? 2 : 4, ROWS = 16 * MT;
    static constexpr int PITCH = ROWS + 4;                     // a warp's stores of sums meet every bank once
    static constexpr int kSums = KG * TM * PITCH * 4;
    static __host__ __device__ int steps(int rank) { return (rank + 15) / 16; }
    // bytes of a row of h: 16 a step and split, 4 rows on different banks
    static __host__ __device__ int pitch(int rank, int together) { const int n = steps(rank) * together; return 32 * n + (n & 1 ? 0 : 32); }
    static __host__ __device__ int parts(int rank, int together) { const int h = 2 * TM * pitch(rank, together); return h > kSums ? h : kSums; }
    static __host__ __device__ int smem(int rank, int together) { return parts(rank, together) + TM * together * rank * 4; }
};

// First product: A operand 16 MT rows of the adapter, B operand 8 tokens, both from global memory, 16 bytes a lane: eight neighbours of a row are two
// steps' k = 2t, 2t + 1, 2t + 8, 2t + 9 of lane t, in the same order on both sides.
// Second: A operand h of 16 tokens as two 16-bit values each, the second with what rounding the first left, so that only `out` is rounded; fp16's lie a power
// of two off, which brings the row's largest to 2^14.  B operand 8 columns; column 2t + e of n-tile j is column 8t + 2j + e of the warp's 32, so that a lane
// holds 16 bytes of a row of `out`.
template <bool BF, int TM>
__global__ void __launch_bounds__(LORA_THREADS, 2) lora_kernel(const LoraArgs A) {
    using L = Lora<TM>;
    constexpr int NT = L::NT, MT = L::MT, ROWS = L::ROWS;
    __shared__ Tile<TM> tile;
    __shared__ float back[TM][LORA_SPLITS];                    // what undoes a row's power of two
    extern __shared__ __align__(16) uint8_t lora_smem[];
    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int kg = warp / L::TG, n0 = warp % L::TG * NT;       // this warp's part of the first product
    const int64_t t0 = (int64_t)(blockIdx.x / blocks) * TM;
    const int steps = L::steps(A.rank), pitch = L::pitch(A.rank, A.together);
    float* const sums = reinterpret_cast<float*>(lora_smem);  // [KG][TM][PITCH], and h behind it in the same place
    float* const part = reinterpret_cast<float*>(lora_smem + L::parts(A.rank, A.together));
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    find_adapters<TM>(A, t0, tile);
    const int chunks = (A.K + 31) / 32, each = (chunks + (int)blocks - 1) / (int)blocks, from = min((int)rank * each, chunks), to = min(from + each, chunks);
    for (int j = blockIdx.y; j < tile.n; j += gridDim.y) {
        const uint64_t mask = tile.rows[j];
        const int id = tile.adapter[j];
        const float scale = A.scales[id];
        for (int s0 = 0; s0 < A.n_splits; s0 += A.together) {
            const int n_here = min(A.together, A.n_splits - s0), rows = n_here * A.rank;
            const uint16_t* const w = (const uint16_t*)A.a + id * A.a_st + (int64_t)s0 * A.rank * A.K;
            // ---- h of this block's share of K
            for (int row0 = 0; row0 < rows; row0 += ROWS) {
                float acc[MT][NT][4] = {};
#pragma unroll 2
                for (int c = from + kg; c < to; c += L::KG) {
                    const int k = 32 * c + 8 * t;
                    const bool in = k < A.K;
                    uint4 wr[MT][2], xr[NT];
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int row = row0 + 16 * m + 8 * h + g;
                            wr[m][h] = in && row < rows ? *reinterpret_cast<const uint4*>(w + (int64_t)row * A.K + k) : make_uint4(0, 0, 0, 0);
                        }
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const int64_t tok = t0 + 8 * (n0 + n) + g;
                        xr[n] = in && tok < A.T && (mask >> (8 * (n0 + n)) & 0xff) ? *reinterpret_cast<const uint4*>((const uint16_t*)A.x + tok * A.x_st + k) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        if (mask >> (8 * (n0 + n)) & 0xff) {
#pragma unroll
                            for (int m = 0; m < MT; m++)
                                if (row0 + 16 * m < rows) {
                                    mma<BF>(acc[m][n], wr[m][0].x, wr[m][1].x, wr[m][0].y, wr[m][1].y, xr[n].x, xr[n].y);
                                    mma<BF>(acc[m][n], wr[m][0].z, wr[m][1].z, wr[m][0].w, wr[m][1].w, xr[n].z, xr[n].w);
                                }
                        }
                }
                __syncthreads();                               // what was in the sums' place is read
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sums[(kg * TM + 8 * (n0 + n) + 2 * t + (e & 1)) * L::PITCH + 16 * m + g + 8 * (e >> 1)] = acc[m][n][e];
                __syncthreads();
                for (int i = threadIdx.x; i < TM * ROWS; i += LORA_THREADS) {
                    const int tok = i / ROWS, row = i % ROWS;
                    if ((mask >> tok & 1) && row0 + row < rows) {
                        float s = 0.0f;
#pragma unroll
                        for (int v = 0; v < L::KG; v++) s += sums[(v * TM + tok) * L::PITCH + row];
                        part[tok * rows + row0 + row] = s;
                    }
                }
            }
            meet(blocks);
            // ---- the blocks' parts together: a warp takes a row of the tile in one split
            const uint32_t at_part = (uint32_t)__cvta_generic_to_shared(part), at_h = (uint32_t)__cvta_generic_to_shared(lora_smem), at_back = (uint32_t)__cvta_generic_to_shared(&back[0][0]);
            for (int i = (int)rank + warp * (int)blocks; i < TM * n_here; i += LORA_WARPS * (int)blocks) {
                const int tok = i % TM, s = i / TM;
                if (!(mask >> (tok & ~15) & 0xffff)) continue;
                const bool live = mask >> tok & 1;
                float2 h[4];                                   // pairs `lane`, `lane` + 32, ...
                float big = 0.0f;
#pragma unroll
                for (int z = 0; z < 4; z++) {
                    h[z] = make_float2(0.0f, 0.0f);
                    const int r = 2 * lane + 64 * z;
                    if (live && r < A.rank) {
                        const uint32_t at = at_part + (tok * rows + s * A.rank + r) * 4;
                        for (uint32_t b = 0; b < blocks; b++) {
                            float2 p;
                            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(p.x), "=f"(p.y) : "r"(shared_of(at, b)) : "memory");
                            h[z].x += p.x;
                            h[z].y += p.y;
                        }
                        h[z].x *= scale;
                        h[z].y *= scale;
                        big = fmaxf(big, fmaxf(fabsf(h[z].x), fabsf(h[z].y)));
                    }
                }
                float down = 1.0f;
                if (!BF) {
#pragma unroll
                    for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
                    const int e = (int)(__float_as_uint(big) >> 23) - 127 - 14, use = big > 0.0f && big < INFINITY ? max(e, -100) : 0;
                    down = __uint_as_float((uint32_t)(127 - use) << 23);
                    if (lane < (int)blocks)
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(shared_of(at_back + (tok * LORA_SPLITS + s) * 4, lane)), "f"(__uint_as_float((uint32_t)(127 + use) << 23)) : "memory");
                }
#pragma unroll
                for (int z = 0; z < 4; z++) {
                    const int r = 2 * lane + 64 * z;
                    if (r >= 16 * steps) continue;
                    const float x = h[z].x * down, y = h[z].y * down;
                    const uint32_t hi = pack2<BF>(x, y);
                    const float2 f = unpack2<BF>(hi);
                    const uint32_t lo = pack2<BF>(fabsf(f.x) < INFINITY ? x - f.x : 0.0f, fabsf(f.y) < INFINITY ? y - f.y : 0.0f);
                    const uint32_t at = at_h + tok * pitch + s * steps * 32 + 2 * r;
                    for (uint32_t b = 0; b < blocks; b++) {
                        const uint32_t p = shared_of(at, b);
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(p), "r"(hi) : "memory");
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(p + TM * pitch), "r"(lo) : "memory");
                    }
                }
            }
            meet(blocks);
            // ---- this block's share of the columns, 32 a warp
            const uint16_t* const wb = (const uint16_t*)A.b + id * A.b_st;
            int s = 0, before = 0, groups = (A.first[s0 + 1] - A.first[s0] + 31) / 32;         // of the splits in front, and of this one
            for (int grp = (int)rank * LORA_WARPS + warp;; grp += (int)blocks * LORA_WARPS) {
                while (s < n_here && grp - before >= groups) {
                    before += groups;
                    s++;
                    if (s < n_here) groups = (A.first[s0 + s + 1] - A.first[s0 + s] + 31) / 32;
                }
                if (s >= n_here) break;
                const int c0 = A.first[s0 + s] + 32 * (grp - before), c_end = A.first[s0 + s + 1], col = c0 + 8 * t;
                constexpr int MP = TM > 16 ? 2 : 1;            // tiles of 16 rows at a time
#pragma unroll 1
                for (int m0 = 0; m0 < TM / 16; m0 += MP) {
                    const uint32_t some = (uint32_t)(mask >> (16 * m0)) & (MP == 2 ? 0xffffffffu : 0xffffu);
                    if (!some) continue;
                    uint4 o[MP][2];
#pragma unroll
                    for (int m = 0; m < MP; m++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int tok = 16 * m + 8 * h + g;
                            if ((some >> tok & 1) && col < c_end) o[m][h] = *reinterpret_cast<const uint4*>((const uint16_t*)A.out + (t0 + 16 * m0 + tok) * A.o_st + col);
                        }
                    float acc[MP][4][4] = {};
                    for (int st = 0; st < steps; st++) {
                        uint2 br[4];
                        const int r = 16 * st + 4 * t;
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            const int cc = c0 + 8 * (g >> 1) + 2 * n + (g & 1);
                            br[n] = cc < c_end && r < A.rank ? *reinterpret_cast<const uint2*>(wb + (int64_t)cc * A.rank + r) : make_uint2(0, 0);
                        }
#pragma unroll
                        for (int m = 0; m < MP; m++)
                            if (some >> (16 * m) & 0xffff) {
                                const uint8_t* const h = lora_smem + (16 * (m0 + m) + g) * pitch + s * steps * 32 + 32 * st + 8 * t;
                                const uint2 a = *reinterpret_cast<const uint2*>(h), b = *reinterpret_cast<const uint2*>(h + 8 * pitch);
                                const uint2 c = *reinterpret_cast<const uint2*>(h + TM * pitch), d = *reinterpret_cast<const uint2*>(h + (TM + 8) * pitch);
#pragma unroll
                                for (int n = 0; n < 4; n++) {
                                    mma<BF>(acc[m][n], c.x, d.x, c.y, d.y, br[n].x, br[n].y);
                                    mma<BF>(acc[m][n], a.x, b.x, a.y, b.y, br[n].x, br[n].y);
                                }
                            }
                    }
#pragma unroll
                    for (int m = 0; m < MP; m++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int tok = 16 * m + 8 * h + g;
                            if (!(some >> tok & 1) || col >= c_end) continue;
                            uint32_t v[4] = {o[m][h].x, o[m][h].y, o[m][h].z, o[m][h].w};
                            const float up = BF ? 1.0f : back[16 * m0 + tok][s];
#pragma unroll
                            for (int n = 0; n < 4; n++) {
                                const float2 f = unpack2<BF>(v[n]);
                                v[n] = pack2<BF>(fmaf(acc[m][n][2 * h], up, f.x), fmaf(acc[m][n][2 * h + 1], up, f.y));
                            }
                            *reinterpret_cast<uint4*>((uint16_t*)A.out + (t0 + 16 * m0 + tok) * A.o_st + col) = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                }
            }
        }
    }
}

template <bool BF, int TM> int lora_launch(LoraArgs A, cudaStream_t st) {
    using L = Lora<TM>;
    // splits that share a reading of x: 128 rows of A at most, or one split
    A.together = A.n_splits * A.rank <= 128 ? A.n_splits : A.rank >= 128 ? 1 : 128 / A.rank;
    static bool configured[64] = {};                           // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        cudaFuncSetAttribute(lora_kernel<BF, TM>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem(256, 1));
        configured[dev & 63] = true;
    }
    const int64_t tiles = (A.T + TM - 1) / TM;
    // clusters that share a tile's adapters: as many as a tile has on average
    int64_t some = 1 + (int64_t)A.R * TM / A.T, most = TM < A.R ? TM : A.R;
    if (most > A.adapters) most = A.adapters;
    if (most > 16) most = 16;
    const int blocks = 8;                                      // of a cluster: the most that any device takes
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * blocks), (unsigned)(some < most ? some : most));
    cfg.blockDim = dim3(LORA_THREADS);
    cfg.dynamicSmemBytes = (size_t)L::smem(A.rank, A.together);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)blocks, 1u, 1u};
    cfg.attrs = at;
    cfg.numAttrs = add_overlap(at, 1, launch_overlaps(st));
    cudaLaunchKernelEx(&cfg, lora_kernel<BF, TM>, A);
    note_launch();
    return check_launch();
}

}  // namespace
}  // namespace lowbit

extern "C" int lowbit_lora_add_cuda(const void* d_x, int64_t x_stride, int dtype, int64_t T, int K, const void* d_a, int64_t a_stride, const void* d_b, int64_t b_stride,
                                    int rank, const float* d_scales, int adapters, const int32_t* d_ids, const int32_t* d_cu_seqlens, int R, const int* splits, int n_splits,
                                    void* d_out, int64_t out_stride, void* stream) {
    reset_launch_count();
    const char* const name = "lowbit_lora_add_cuda";
    bool bad = !d_x || !d_a || !d_b || !d_scales || !d_ids || !d_cu_seqlens || !d_out || !splits || (dtype != DT_F16 && dtype != DT_BF16) || T < 0 || T > 0x7fffffffll || K <= 0 ||
               K % 8 || K > 0x7fffff00 || rank <= 0 || rank % 8 || rank > 256 || adapters <= 0 || R <= 0 || n_splits <= 0 || n_splits > LORA_SPLITS || x_stride < K;
    int64_t N = 0;
    for (int i = 0; !bad && i < n_splits; i++) { bad = splits[i] <= 0 || splits[i] % 8; N += splits[i]; }
    bad = bad || N > 0x7fffff00ll || out_stride < N || a_stride < (int64_t)n_splits * rank * K || b_stride < N * rank;
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
    LoraArgs A = {d_x, x_stride, T, K, d_a, a_stride, d_b, b_stride, d_scales, adapters, d_ids, d_cu_seqlens, R, d_out, out_stride, rank, n_splits, 0, {}};
    for (int i = 0; i < n_splits; i++) A.first[i + 1] = A.first[i] + splits[i];
    cudaStream_t st = (cudaStream_t)stream;
    if (T <= 256) return dtype == DT_BF16 ? lora_launch<true, 16>(A, st) : lora_launch<false, 16>(A, st);
    return dtype == DT_BF16 ? lora_launch<true, 64>(A, st) : lora_launch<false, 64>(A, st);
}
