// lora.cu -- low-rank adapters of many requests beside a projection that all share:
//   out[t] += scale_l (x[t] A_l^T) B_l^T,      l = the adapter of the token's request (none: the row stays as it is).
// Two launches.  shrink: h = x A^T in 32 bits, the inner dimension dealt to KS blocks that leave a part each; expand: the parts added up in their order,
// times the scale, and the product with B added to `out`, rounded once.
//
// Both work on tiles of packed rows, whoever they belong to: a block finds the tile's requests in the list, and the different adapters among its rows are
// dealt to the blocks that share the tile.  So an adapter that neighbours have in common is read once for them, and nobody sorts.
// mma.sync m16n8k16: rank and tokens are far below a tcgen05 tile, and what bounds both is what they read and write (x; out, twice).
#include "lowbit_common.cuh"
#include "lowbit_internal.h"

using namespace lowbit;

namespace lowbit {
namespace {

constexpr int LORA_THREADS = 128, LORA_WARPS = 4, LORA_SPLITS = 8;
constexpr int LORA_COLUMNS = 128;                              // of a block of expand: 32 a warp

struct LoraArgs {
    const void* x; int64_t x_st; int64_t T; int K;
    const void* a; int64_t a_st;                               // [adapters][rows][K]
    const void* b; int64_t b_st;                               // [adapters][columns][rank]
    const float* scales; int adapters;
    const int32_t *ids, *cu; int R;                            // requests
    void* out; int64_t o_st;
    int rows, rank;                                            // rows = splits x rank
    float* part; int KS, chunks;                               // parts; 32-element chunks of K in one
    int n_splits, first[LORA_SPLITS + 1], blocks[LORA_SPLITS + 1];       // columns, and blocks of columns, in front of a split
};

template <bool BF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF) asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                         : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
        if (a < b) {
            const int id = A.ids[r];
            if (id >= 0 && id < A.adapters)
                for (int64_t t = a; t < b; t++) tile.id[t - t0] = id;
        }
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

// ------------------------------------------------------------------ h = x A^T
// A operand: 16 MT rows of the adapter; B operand: 8 tokens.  Both from global memory, 16 bytes a lane: eight neighbours of a row are the two steps' k
// = 2t, 2t + 1, 2t + 8, 2t + 9 of lane t, in the same order on both sides.  Warps take 32-element chunks in turn and meet in shared memory.
template <bool BF, int TM, int MT>
__global__ void __launch_bounds__(LORA_THREADS) lora_shrink_kernel(const LoraArgs A) {
    constexpr int NT = TM / 8, ROWS = 16 * MT, PITCH = ROWS + 1;
    __shared__ Tile<TM> tile;
    __shared__ float sums[LORA_WARPS][TM][PITCH];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int passes = (A.rows + ROWS - 1) / ROWS, ks = blockIdx.z / passes, row0 = (int)(blockIdx.z % passes) * ROWS;
    const int64_t t0 = (int64_t)blockIdx.x * TM;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    find_adapters<TM>(A, t0, tile);
    const int from = ks * A.chunks, to = min(from + A.chunks, (A.K + 31) / 32);
    for (int j = blockIdx.y; j < tile.n; j += gridDim.y) {
        const uint64_t mask = tile.rows[j];
        const uint16_t* const w = (const uint16_t*)A.a + tile.adapter[j] * A.a_st;
        float acc[MT][NT][4] = {};
        for (int c = from + warp; c < to; c += LORA_WARPS) {
            const int k = 32 * c + 8 * t;
            const bool in = k < A.K;
            uint4 wr[MT][2], xr[NT];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int row = row0 + 16 * m + 8 * h + g;
                    wr[m][h] = in && row < A.rows ? *reinterpret_cast<const uint4*>(w + (int64_t)row * A.K + k) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
            for (int n = 0; n < NT; n++)
                if (mask >> (8 * n) & 0xff) {
                    const int64_t tok = t0 + 8 * n + g;
                    xr[n] = in && tok < A.T ? *reinterpret_cast<const uint4*>((const uint16_t*)A.x + tok * A.x_st + k) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
            for (int n = 0; n < NT; n++)
                if (mask >> (8 * n) & 0xff) {
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        mma<BF>(acc[m][n], wr[m][0].x, wr[m][1].x, wr[m][0].y, wr[m][1].y, xr[n].x, xr[n].y);
                        mma<BF>(acc[m][n], wr[m][0].z, wr[m][1].z, wr[m][0].w, wr[m][1].w, xr[n].z, xr[n].w);
                    }
                }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
            if (mask >> (8 * n) & 0xff) {
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sums[warp][8 * n + 2 * t + (e & 1)][16 * m + g + 8 * (e >> 1)] = acc[m][n][e];
            }
        __syncthreads();
        for (int i = threadIdx.x; i < TM * ROWS; i += LORA_THREADS) {
            const int tok = i / ROWS, row = i % ROWS;
            if ((mask >> tok & 1) && row0 + row < A.rows) {
                float s = sums[0][tok][row];
#pragma unroll
                for (int v = 1; v < LORA_WARPS; v++) s += sums[v][tok][row];
                A.part[((int64_t)ks * A.T + t0 + tok) * A.rows + row0 + row] = s;
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ out += scale h B^T
template <bool BF> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    if (BF) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF> __device__ __forceinline__ float2 unpack2(uint32_t w) {
    if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// A operand: h of 16 tokens as two 16-bit values each, the second with what rounding the first left, so that only `out` is rounded; fp16's lie a power of
// two off, which brings the row's largest to 2^14.  B operand: 8 columns.  Column 2t + e of n-tile j is column 8t + 2j + e of the warp's 32, so that
// a lane holds 16 bytes of a row of `out`.
template <bool BF, int TM>
__global__ void __launch_bounds__(LORA_THREADS) lora_expand_kernel(const LoraArgs A) {
    constexpr int MT = TM / 16;
    __shared__ Tile<TM> tile;
    __shared__ float back[TM];                                 // what undoes a row's power of two
    extern __shared__ __align__(16) uint8_t lora_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t t0 = (int64_t)blockIdx.y * TM;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    int split = 0;
    while (split + 1 < A.n_splits && (int)blockIdx.x >= A.blocks[split + 1]) split++;
    const int c0 = A.first[split] + ((int)blockIdx.x - A.blocks[split]) * LORA_COLUMNS + 32 * warp, c_end = A.first[split + 1];
    const int steps = (A.rank + 15) / 16, pitch = 32 * steps + (steps & 1 ? 0 : 32);       // bytes of a row of h: 16 a step, 4 rows on different banks
    find_adapters<TM>(A, t0, tile);
    for (int j = blockIdx.z; j < tile.n; j += gridDim.z) {
        const uint64_t mask = tile.rows[j];
        const int id = tile.adapter[j];
        const float scale = A.scales[id];
        // a warp a row: the parts' sum, as two values
        for (int tok = warp; tok < TM; tok += LORA_WARPS) {
            if (!(mask >> (tok & ~15) & 0xffff)) continue;
            const bool live = mask >> tok & 1;
            uint8_t* const hi = lora_smem + tok * pitch;
            uint8_t* const lo = hi + TM * pitch;
            float down = 1.0f;
            if (!BF && live) {
                float big = 0.0f;
                for (int r = lane; r < A.rank; r += 32) {
                    float h = 0.0f;
                    for (int ks = 0; ks < A.KS; ks++) h += A.part[((int64_t)ks * A.T + t0 + tok) * A.rows + split * A.rank + r];
                    big = fmaxf(big, fabsf(h * scale));
                }
#pragma unroll
                for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
                const int e = (int)(__float_as_uint(big) >> 23) - 127 - 14;
                const int use = big > 0.0f && big < INFINITY ? max(e, -100) : 0;
                down = __uint_as_float((uint32_t)(127 - use) << 23);
                if (lane == 0) back[tok] = __uint_as_float((uint32_t)(127 + use) << 23);
            }
            for (int r = 2 * lane; r < 16 * steps; r += 64) {
                float h[2] = {0.0f, 0.0f};
                if (live && r < A.rank)
                    for (int ks = 0; ks < A.KS; ks++) {
                        const float2 p = *reinterpret_cast<const float2*>(A.part + ((int64_t)ks * A.T + t0 + tok) * A.rows + split * A.rank + r);
                        h[0] += p.x;
                        h[1] += p.y;
                    }
                h[0] *= scale * down;
                h[1] *= scale * down;
                const uint32_t w = pack2<BF>(h[0], h[1]);
                const float2 f = unpack2<BF>(w);
                *reinterpret_cast<uint32_t*>(hi + 2 * r) = w;
                *reinterpret_cast<uint32_t*>(lo + 2 * r) = pack2<BF>(fabsf(f.x) < INFINITY ? h[0] - f.x : 0.0f, fabsf(f.y) < INFINITY ? h[1] - f.y : 0.0f);
            }
        }
        __syncthreads();
        if (c0 < c_end) {
            float acc[MT][4][4] = {};
            const uint16_t* const w = (const uint16_t*)A.b + id * A.b_st;
            for (int s = 0; s < steps; s++) {
                uint2 br[4];
                const int r = 16 * s + 4 * t;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const int col = c0 + 8 * (g >> 1) + 2 * n + (g & 1);
                    br[n] = col < c_end && r < A.rank ? *reinterpret_cast<const uint2*>(w + (int64_t)col * A.rank + r) : make_uint2(0, 0);
                }
#pragma unroll
                for (int m = 0; m < MT; m++)
                    if (mask >> (16 * m) & 0xffff) {
                        const uint8_t* const h = lora_smem + (16 * m + g) * pitch + 32 * s + 8 * t;
                        const uint2 a = *reinterpret_cast<const uint2*>(h), b = *reinterpret_cast<const uint2*>(h + 8 * pitch);
                        const uint2 c = *reinterpret_cast<const uint2*>(h + TM * pitch), d = *reinterpret_cast<const uint2*>(h + (TM + 8) * pitch);
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            mma<BF>(acc[m][n], c.x, d.x, c.y, d.y, br[n].x, br[n].y);
                            mma<BF>(acc[m][n], a.x, b.x, a.y, b.y, br[n].x, br[n].y);
                        }
                    }
            }
            const int col = c0 + 8 * t;
            if (col < c_end) {
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int tok = 16 * m + 8 * h + g;
                        if (!(mask >> tok & 1)) continue;
                        uint4* const p = reinterpret_cast<uint4*>((uint16_t*)A.out + (t0 + tok) * A.o_st + col);
                        const uint4 v = *p;
                        uint32_t o[4] = {v.x, v.y, v.z, v.w};
                        const float up = BF ? 1.0f : back[tok];
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            const float2 f = unpack2<BF>(o[n]);
                            o[n] = pack2<BF>(fmaf(acc[m][n][2 * h], up, f.x), fmaf(acc[m][n][2 * h + 1], up, f.y));
                        }
                        *p = make_uint4(o[0], o[1], o[2], o[3]);
                    }
            }
        }
        __syncthreads();
    }
}

// how a call is dealt out
struct LoraPlan { int tile, adapters, mt, passes, KS, chunks; int64_t tiles; };
LoraPlan lora_plan(int64_t T, int K, int rows, int R, int adapters) {
    LoraPlan p;
    p.tile = T > 256 ? 64 : 16;
    p.tiles = (T + p.tile - 1) / p.tile;
    // blocks that share a tile's adapters: as many as a tile has on average
    int64_t some = 1 + (int64_t)R * p.tile / T, most = p.tile < R ? p.tile : R;
    if (most > adapters) most = adapters;
    if (most > 16) most = 16;
    p.adapters = (int)(some < most ? some : most);
    p.mt = rows > 16 ? 2 : 1;
    p.passes = (rows + 16 * p.mt - 1) / (16 * p.mt);
    const int chunks = (K + 31) / 32;
    const int64_t blocks = p.tiles * p.adapters * p.passes, want = 4ll * sm_count();
    int64_t ks = (want + blocks - 1) / blocks;
    if (ks > 16) ks = 16;
    if (ks > (chunks + 7) / 8) ks = (chunks + 7) / 8;          // two chunks a warp
    p.chunks = (int)((chunks + ks - 1) / ks);
    p.KS = (chunks + p.chunks - 1) / p.chunks;
    return p;
}

template <bool BF, int TM> void shrink(const LoraArgs& A, const LoraPlan& p, cudaStream_t st) {
    const dim3 grid((unsigned)p.tiles, (unsigned)p.adapters, (unsigned)(p.KS * p.passes));
    if (p.mt == 1) launch_behind(lora_shrink_kernel<BF, TM, 1>, grid, LORA_THREADS, 0, st, launch_overlaps(st), A);
    else launch_behind(lora_shrink_kernel<BF, TM, 2>, grid, LORA_THREADS, 0, st, launch_overlaps(st), A);
}
template <bool BF, int TM> int lora_launch(const LoraArgs& A, const LoraPlan& p, cudaStream_t st) {
    const int steps = (A.rank + 15) / 16, pitch = 32 * steps + (steps & 1 ? 0 : 32);
    const size_t smem = (size_t)2 * TM * pitch;
    static bool configured[64] = {};                           // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        cudaFuncSetAttribute(lora_expand_kernel<BF, TM>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * TM * (32 * 16 + 32));
        configured[dev & 63] = true;
    }
    shrink<BF, TM>(A, p, st);
    note_launch();
    launch_behind(lora_expand_kernel<BF, TM>, dim3((unsigned)A.blocks[A.n_splits], (unsigned)p.tiles, (unsigned)p.adapters), LORA_THREADS, smem, st, launch_overlaps(st), A);
    note_launch();
    return check_launch();
}

}  // namespace
}  // namespace lowbit

extern "C" size_t lowbit_lora_workspace_size(int64_t T, int K, int rows, int R, int adapters) {
    if (T <= 0 || K <= 0 || rows <= 0 || R <= 0 || adapters <= 0) return 0;
    return (size_t)lora_plan(T, K, rows, R, adapters).KS * T * rows * sizeof(float);
}

extern "C" int lowbit_lora_add_cuda(const void* d_x, int64_t x_stride, int dtype, int64_t T, int K, const void* d_a, int64_t a_stride, const void* d_b, int64_t b_stride,
                                    int rank, const float* d_scales, int adapters, const int32_t* d_ids, const int32_t* d_cu_seqlens, int R, const int* splits, int n_splits,
                                    void* d_out, int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    reset_launch_count();
    const char* const name = "lowbit_lora_add_cuda";
    bool bad = !d_x || !d_a || !d_b || !d_scales || !d_ids || !d_cu_seqlens || !d_out || !splits || (dtype != DT_F16 && dtype != DT_BF16) || T < 0 || T > 65535ll * 64 || K <= 0 ||
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
    const int rows = n_splits * rank;
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < lowbit_lora_workspace_size(T, K, rows, R, adapters)) {
        set_error(LB_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of lowbit_lora_workspace_size() bytes is needed", name);
        return LB_ERR_WORKSPACE;
    }
    const LoraPlan p = lora_plan(T, K, rows, R, adapters);
    LoraArgs A = {d_x, x_stride, T, K, d_a, a_stride, d_b, b_stride, d_scales, adapters, d_ids, d_cu_seqlens, R, d_out, out_stride, rows, rank, (float*)workspace, p.KS, p.chunks};
    A.n_splits = n_splits;
    for (int i = 0; i < n_splits; i++) {
        A.first[i + 1] = A.first[i] + splits[i];
        A.blocks[i + 1] = A.blocks[i] + (splits[i] + LORA_COLUMNS - 1) / LORA_COLUMNS;
    }
    cudaStream_t st = (cudaStream_t)stream;
    if (p.tile == 16) return dtype == DT_BF16 ? lora_launch<true, 16>(A, p, st) : lora_launch<false, 16>(A, p, st);
    return dtype == DT_BF16 ? lora_launch<true, 64>(A, p, st) : lora_launch<false, 64>(A, p, st);
}
