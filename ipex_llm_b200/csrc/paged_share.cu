// paged_share.cu -- pages of the cache that several rows of the block table name: forking a request, copying pages, giving them back, and moving those
// in use to the front.
//
// shared[p] counts the rows beyond the first that name page p.  A fork names its parent's full pages (one more each) and gets a page of its own for
// the tokens behind them, so a page that anybody writes to is named by one row.  A row that goes takes its counts with it, and the last one gives
// the page back.  All results are whole numbers that do not depend on the order in which threads run.
#include "paged.h"

using namespace lowbit;

namespace lowbit {
namespace {

constexpr int SHARE_THREADS = 1024, SHARE_WARPS = SHARE_THREADS / 32;
constexpr int SHARE_DEEP = 8;                                  // entries of a row that a lane reads at a time: what follows waits for memory once for all

// the blocks of a cluster meet; what they wrote is seen by all
__device__ __forceinline__ void meet(uint32_t blocks) {
    if (blocks == 1) { __syncthreads(); return; }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t x; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(x)); return x; }
__device__ __forceinline__ uint32_t cluster_blocks() { uint32_t x; asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(x)); return x; }

// inclusive sum over the block; all: of the whole block
__device__ __forceinline__ int block_sum(int x, int* warps, int& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    int w = warps[lane];                                       // 32 warps
    const int own = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, d);
        if (lane >= d) w += y;
    }
    all = __shfl_sync(0xffffffffu, w, 31);
    return x + __shfl_sync(0xffffffffu, w - own, warp);
}

// ------------------------------------------------------------------ fork
struct ForkArgs {
    const int32_t *parents, *children; int F;
    int32_t* lens; int32_t* table; int64_t table_stride; int R, width;
    const int32_t* pages; int n_pages; const int32_t* count; int32_t* left;
    int32_t* shared; int page_size;
    int32_t *src, *dst, *missing;
};

// Every block finds for itself which forks need a page (a round of a thread each), then a warp takes a fork at a time.  The count is read by all, and may
// be written in place: by the one block that there is, or (`last` false) by a launch behind.
__global__ void __launch_bounds__(SHARE_THREADS, 1) paged_fork_kernel(const ForkArgs A, bool last) {
    __shared__ int warps[32];
    __shared__ int fresh[SHARE_THREADS];                       // the page of each of these forks, -1: none to be had, -2: it needs none
    const int rank = blockIdx.x, blocks = gridDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int count = max(0, min(*A.count, A.n_pages));
    int taken = 0;
    for (int f0 = 0; f0 < A.F; f0 += SHARE_THREADS) {
        const int f = f0 + threadIdx.x;
        bool need = false;
        if (f < A.F) {
            const int par = A.parents[f], ch = A.children[f];
            if (par >= 0 && par < A.R && ch >= 0 && ch < A.R && par != ch) {
                const int held = max(A.lens[par], 0), full = held / A.page_size;
                need = full < A.width && full * A.page_size != held;
            }
        }
        int total;
        const int at = count - (taken + block_sum(need, warps, total));
        __syncthreads();
        fresh[threadIdx.x] = !need ? -2 : at >= 0 ? A.pages[at] : -1;
        taken += total;
        __syncthreads();
        // lens of parents are read above and below, and children's written below: no row is both
        for (int i = warp * blocks + rank; i < min(SHARE_THREADS, A.F - f0); i += blocks * SHARE_WARPS) {
            const int par = A.parents[f0 + i], ch = A.children[f0 + i], page = fresh[i];
            if (par < 0 || par >= A.R || ch < 0 || ch >= A.R || par == ch) {
                if (lane == 0) A.src[f0 + i] = A.dst[f0 + i] = -1;
                continue;
            }
            const int held = max(A.lens[par], 0), full = min(held / A.page_size, A.width);
            const int32_t* const from = A.table + par * A.table_stride;
            int32_t* const to = A.table + ch * A.table_stride;
            for (int c0 = lane; c0 < A.width; c0 += 32 * SHARE_DEEP) {
                int p[SHARE_DEEP];
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++) p[u] = c0 + 32 * u <= full && c0 + 32 * u < A.width ? from[c0 + 32 * u] : -1;
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++) {
                    const int c = c0 + 32 * u;
                    if (c >= A.width) continue;
                    if (c < full && p[u] >= 0 && p[u] < A.n_pages) atomicAdd(A.shared + p[u], 1);
                    to[c] = c < full ? p[u] : c == full && page != -2 ? page : -1;
                    if (c == full) A.src[f0 + i] = page != -2 ? p[u] : -1;
                }
            }
            if (lane == 0) {
                if (full == A.width) A.src[f0 + i] = -1;
                A.dst[f0 + i] = page != -2 ? page : -1;
                A.lens[ch] = A.lens[par];
            }
        }
        __syncthreads();
    }
    if (!last) {
        if (rank == 0 && threadIdx.x == 0) *A.missing = taken; // for the launch behind
    } else if (threadIdx.x == 0) {                             // behind the barrier: everybody has read the count
        *A.left = max(count - taken, 0);
        *A.missing = max(taken - count, 0);
    }
}
__global__ void paged_fork_count_kernel(const int32_t* count_at, int n_pages, int32_t* left, int32_t* missing) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int count = max(0, min(*count_at, n_pages)), taken = *missing;
    *left = max(count - taken, 0);
    *missing = max(taken - count, 0);
}

// ------------------------------------------------------------------ release
struct ShareReleaseArgs {
    const uint8_t* done; const int32_t* held; int page_size;
    int R; int32_t* table; int64_t table_stride; int width;
    int32_t* pages; int n_pages; int32_t* count; int32_t* shared;
    int32_t* times; int32_t* first; int32_t* gives;            // scratch: [pages], [pages], [stretches + 1]
};
constexpr int SHARE_STRETCH = 32 * SHARE_DEEP;                 // columns of a row that a warp takes at a time
inline int64_t share_stretches(int R, int width) { return (int64_t)R * ((width + SHARE_STRETCH - 1) / SHARE_STRETCH); }

// Rows that are done give up what they name (behind `held` tokens): page p, named `times` in all, goes onto the stack where that is more than shared[p],
// in the order of the entries that name it first.  A warp a stretch of a row, four times: places cleared, names counted, pages settled and those of a stretch counted, pages
// written.  One block does all four (PART -1); where there is more to do each is a launch over the whole device, and the count's place is the launch's behind that reads it.
template <int PART>
__global__ void __launch_bounds__(SHARE_THREADS, 1) paged_share_release_kernel(const ShareReleaseArgs A) {
    __shared__ int warps[32];
    __shared__ int before[SHARE_THREADS];
    const int lane = threadIdx.x & 31, blocks = gridDim.x, me = (threadIdx.x >> 5) * blocks + blockIdx.x, all = blocks * SHARE_WARPS;
    const int of_row = (A.width + SHARE_STRETCH - 1) / SHARE_STRETCH, stretches = A.R * of_row;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int count = max(0, min(*A.count, A.n_pages));
    // what stretch s gives up: f(its row, this lane's first column, its pages, SHARE_DEEP a lane, -1 what is none, the first column that goes); whole warps
    auto each = [&](int s, auto&& f) {
        const int r = s / of_row, c = (s - r * of_row) * SHARE_STRETCH + lane;
        if (!A.done[r]) return;
        const int from = A.held ? (int)min((int64_t)A.width, ((int64_t)max(A.held[r], 0) + A.page_size - 1) / A.page_size) : 0;
        const int32_t* const row = A.table + r * A.table_stride;
        int p[SHARE_DEEP];
#pragma unroll
        for (int u = 0; u < SHARE_DEEP; u++) p[u] = c + 32 * u >= from && c + 32 * u < A.width ? row[c + 32 * u] : -1;
#pragma unroll
        for (int u = 0; u < SHARE_DEEP; u++) p[u] = p[u] < A.n_pages ? p[u] : -1;
        f(r, c, p, from);
    };
    using Pages = const int (&)[SHARE_DEEP];
    if (PART == 0 && A.n_pages <= A.R * A.width) {             // all places: without a look at the table
        for (int p = (int)(blockIdx.x * SHARE_THREADS + threadIdx.x); p < A.n_pages; p += blocks * SHARE_THREADS) { A.times[p] = 0; A.first[p] = 0x7fffffff; }
        return;
    }
    if (PART < 0 || PART == 0) {
        for (int s = me; s < stretches; s += all)
            each(s, [&](int, int, Pages p, int) {
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++)
                    if (p[u] >= 0) { A.times[p[u]] = 0; A.first[p[u]] = 0x7fffffff; }
            });
    }
    if (PART < 0) __syncthreads();
    if (PART < 0 || PART == 1) {
        for (int s = me; s < stretches; s += all)
            each(s, [&](int r, int c, Pages p, int) {
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++)
                    if (p[u] >= 0) { atomicAdd(A.times + p[u], 1); atomicMin(A.first + p[u], r * A.width + c + 32 * u); }
            });
    }
    if (PART < 0) __syncthreads();
    if (PART < 0 || PART == 2) {
        for (int s = me; s < stretches; s += all) {
            int n = 0;
            each(s, [&](int r, int c, Pages p, int) {
                // the entry that names its page first settles the page: `times` is from now on by how many more that was given up than shared says
                bool mine[SHARE_DEEP];
                int more[SHARE_DEEP];
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++) mine[u] = p[u] >= 0 && A.first[p[u]] == r * A.width + c + 32 * u;
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++) more[u] = mine[u] ? A.times[p[u]] - A.shared[p[u]] : 0;
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++) {
                    if (mine[u]) { A.times[p[u]] = more[u]; A.shared[p[u]] = max(-more[u], 0); }
                    n += __popc(__ballot_sync(0xffffffffu, more[u] > 0));
                }
            });
            if (lane == 0) A.gives[s] = n;
        }
    }
    if (PART < 0) __syncthreads();
    if (PART >= 0 && PART != 3) return;
    int top = count;
    for (int s0 = 0; s0 < stretches; s0 += SHARE_THREADS) {
        const int n = s0 + (int)threadIdx.x < stretches ? A.gives[s0 + threadIdx.x] : 0;
        int total;
        const int sum = block_sum(n, warps, total);
        __syncthreads();
        before[threadIdx.x] = top + sum - n;
        __syncthreads();
        // stretches as they were dealt above
        for (int s = s0 + (me - s0 % all + all) % all; s < min(s0 + SHARE_THREADS, stretches); s += all) {
            int at = before[s - s0];
            each(s, [&](int r, int c, Pages p, int from) {
                int32_t* const row = A.table + r * A.table_stride;
                int first[SHARE_DEEP], times[SHARE_DEEP];
                bool goes[SHARE_DEEP];
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++) { first[u] = p[u] >= 0 ? A.first[p[u]] : -1; times[u] = p[u] >= 0 ? A.times[p[u]] : 0; }
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++) goes[u] = first[u] == r * A.width + c + 32 * u && times[u] > 0;
#pragma unroll
                for (int u = 0; u < SHARE_DEEP; u++) {
                    const uint32_t yes = __ballot_sync(0xffffffffu, goes[u]);
                    const int slot = at + __popc(yes & ((1u << lane) - 1u));
                    if (goes[u] && slot < A.n_pages) A.pages[slot] = p[u];
                    if (c + 32 * u >= from && c + 32 * u < A.width) row[c + 32 * u] = -1;
                    at += __popc(yes);
                }
            });
        }
        top += total;
        __syncthreads();
    }
    // the count may be read by other blocks yet: the sum of what was given goes where the launch behind finds it
    if (blockIdx.x == 0 && threadIdx.x == 0) *(PART < 0 ? A.count : A.gives + stretches) = min(top, A.n_pages);
}
__global__ void paged_share_count_kernel(const int32_t* top, int32_t* count) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    *count = *top;
}

// ------------------------------------------------------------------ compact
struct CompactArgs {
    const int32_t* table; int64_t table_stride; int R, width;
    const int32_t* pages; int n_pages; const int32_t* count; const int32_t* shared;
    int32_t *table_out, *pages_out, *count_out, *shared_out, *src, *dst;
    int32_t *state, *to, *free_up, *used_up;                   // scratch, [pages] each
};
// entries of the ascending list that are below x
__device__ __forceinline__ int below(const int32_t* list, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] < x) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Free pages in ascending order against used ones in descending order, as long as the free one lies in front: move i goes from the i-th of these to the
// i-th of those.  Pages that are neither in the table nor on the stack stay.  The stack's lowest page comes off first.  HERE: one block, the scratch in
// shared memory (a table of 2240 entries and 1365 pages 12 us, 16 with it in memory); else a cluster's blocks share it in memory.
template <bool HERE>
__global__ void __launch_bounds__(SHARE_THREADS, 1) paged_compact_kernel(const CompactArgs A) {
    extern __shared__ int32_t compact_here[];
    int32_t* const state = HERE ? compact_here : A.state;
    int32_t* const goes_to = HERE ? compact_here + A.n_pages : A.to;
    int32_t* const free_up = HERE ? compact_here + 2 * A.n_pages : A.free_up;
    int32_t* const used_up = HERE ? compact_here + 3 * A.n_pages : A.used_up;
    __shared__ int warps[32];
    __shared__ int totals[2];                                  // of this block's pages: free, used
    __shared__ int moves;
    const uint32_t rank = cluster_rank(), blocks = cluster_blocks();
    const int me = (int)rank * SHARE_THREADS + threadIdx.x, all = (int)blocks * SHARE_THREADS;
    const int entries = A.R * A.width;                         // up to 2^30
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int count = max(0, min(*A.count, A.n_pages));
    auto entry = [&](int e) { const int r = e / A.width; return A.table[r * A.table_stride + (e - r * A.width)]; };
    auto is_page = [&](int p) { return p >= 0 && p < A.n_pages; };
    for (int p = me; p < A.n_pages; p += all) { state[p] = 0; goes_to[p] = p; }
    meet(blocks);
    for (int i = me; i < A.n_pages; i += all) { const int p = A.pages[i]; if (i < count && is_page(p)) atomicOr(state + p, 1); }
    for (int e = me; e < entries; e += all) { const int p = entry(e); if (is_page(p)) atomicOr(state + p, 2); }
    meet(blocks);
    // both lists: this block's pages lie behind those of the blocks in front
    const int each = (A.n_pages + (int)blocks - 1) / (int)blocks, begin = min((int)rank * each, A.n_pages), end = min(begin + each, A.n_pages);
    int free_at = 0, used_at = 0, F = 0, U = 0;
    if (!HERE) {
        int n_free = 0, n_used = 0;
        for (int p0 = begin; p0 < end; p0 += SHARE_THREADS) {
            const int p = p0 + threadIdx.x, s = p < end ? state[p] : 0;
            n_free += __syncthreads_count(s == 1);
            n_used += __syncthreads_count(s & 2);
        }
        if (threadIdx.x == 0) { totals[0] = n_free; totals[1] = n_used; }
        meet(blocks);
        for (uint32_t b = 0; b < blocks; b++) {
            uint32_t at;
            int f, u;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(totals)), "r"(b));
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(f) : "r"(at) : "memory");
            asm volatile("ld.shared::cluster.s32 %0, [%1 + 4];" : "=r"(u) : "r"(at) : "memory");
            if (b < rank) { free_at += f; used_at += u; }
            F += f; U += u;
        }
    }
    for (int p0 = begin; p0 < end; p0 += SHARE_THREADS) {
        const int p = p0 + threadIdx.x, s = p < end ? state[p] : 0;
        int total;
        const int both = block_sum((s == 1 ? 1 : 0) + (s & 2 ? 1 << 16 : 0), warps, total);     // up to 1024 each
        if (s == 1) free_up[free_at + (both & 0xffff) - 1] = p;
        if (s & 2) used_up[used_at + (both >> 16) - 1] = p;
        free_at += total & 0xffff;
        used_at += total >> 16;
    }
    if (HERE) { F = free_at; U = used_at; }
    meet(blocks);
    if (threadIdx.x == 0) {
        int lo = 0, hi = min(F, U);                            // the first pair that does not move
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (free_up[mid] < used_up[U - 1 - mid]) lo = mid + 1;
            else hi = mid;
        }
        moves = lo;
    }
    __syncthreads();
    const int m = moves;
    for (int i = me; i < A.n_pages; i += all) {
        const int a = i < m ? free_up[i] : -1, b = i < m ? used_up[U - 1 - i] : -1;
        A.src[i] = b;
        A.dst[i] = a;
        if (i < m) goes_to[b] = a;
        // the stack, from its highest page down: free pages that stay free, and the vacated ones
        if (i >= m && i < F) {
            const int p = free_up[i];
            A.pages_out[F - 1 - (i - m) - below(used_up + U - m, m, p)] = p;
        }
        if (i < m) {
            const int p = used_up[U - m + i];
            A.pages_out[F - 1 - i - below(free_up + m, F - m, p)] = p;
        }
        if (i >= F) A.pages_out[i] = -1;
        if (A.shared_out) {
            const int s = state[i];                          // a page of nobody keeps its count
            int x = A.shared[i];
            // where page i's contents come from: nothing new, the page that moved here, or it has moved away
            if (s == 1) { const int k = below(free_up, F, i); if (k < m) x = A.shared[used_up[U - 1 - k]]; }
            else if (s & 2) { const int k = U - 1 - below(used_up, U, i); if (k < m) x = 0; }
            A.shared_out[i] = x;
        }
    }
    if (me == 0) *A.count_out = F;
    meet(blocks);
    for (int e = me; e < entries; e += all) {
        const int p = entry(e);
        A.table_out[e] = is_page(p) ? goes_to[p] : p;
    }
}

// ------------------------------------------------------------------ copies
constexpr int COPY_CACHES = 256, COPY_THREADS = 256, COPY_DEEP = 8;
struct CopyArgs {
    const int32_t *src, *dst; int n; int n_caches, n_pages;
    int64_t page_stride, page_bytes;                           // bytes
    int pieces; int64_t piece_bytes;                           // of a page
    uint8_t* caches[COPY_CACHES];
};
// page src[i] to page dst[i] of every cache: a piece of a page a block at a time, 128 bytes a thread in flight (268 MB in 43.7 us, 6.1 TB/s; with 64 in flight 49).
// Entries of -1 are looked at for every piece of every cache: 50000 of them and 64 caches take 1740 us
template <typename U>
__global__ void __launch_bounds__(COPY_THREADS) paged_copy_kernel(const __grid_constant__ CopyArgs A) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int64_t per = (int64_t)A.n_caches * A.pieces, items = per * A.n;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int i = (int)(item / per), in = (int)(item - i * per), cache = in / A.pieces, piece = in - cache * A.pieces;
        const int a = A.src[i], b = A.dst[i];
        if (a < 0 || a >= A.n_pages || b < 0 || b >= A.n_pages) continue;
        const int64_t at = piece * A.piece_bytes;
        const int n = (int)(min(A.piece_bytes, A.page_bytes - at) / (int64_t)sizeof(U));
        const U* const from = reinterpret_cast<const U*>(A.caches[cache] + a * A.page_stride + at);
        U* const to = reinterpret_cast<U*>(A.caches[cache] + b * A.page_stride + at);
        for (int e = threadIdx.x; e < n; e += COPY_DEEP * COPY_THREADS) {
            U x[COPY_DEEP];
#pragma unroll
            for (int k = 0; k < COPY_DEEP; k++)
                if (e + k * COPY_THREADS < n) x[k] = from[e + k * COPY_THREADS];
#pragma unroll
            for (int k = 0; k < COPY_DEEP; k++)
                if (e + k * COPY_THREADS < n) to[e + k * COPY_THREADS] = x[k];
        }
    }
}

// Entries of the table beyond which a launch over the device, or a cluster, takes less time than one block.  Latency bounds all of it: every trip to memory waits for
// the last.  300 forks of rows of up to 486 pages and the release of them: 200 us by a block, 55 by a cluster of eight, 20 over the device (seven launches); 4 forks of rows of 114: 6.0 by
// a block, 6.3 by a cluster.  Releases by a block with eight entries a lane at a time 45 us, with one 70, with four 52, with sixteen no less.
constexpr int64_t SHARE_MANY = 8192;
// blocks over the whole device, of rows by warps
int wide_grid(int64_t rows) { return rows < sm_count() ? (int)rows : sm_count(); }

// of a list: a step beyond its end stays in 32 bits
constexpr int SHARE_MOST = 1 << 30;
bool bad_table(const void* table, int64_t stride, int R, int width) { return !table || R <= 0 || width <= 0 || stride < width || (int64_t)R * width > SHARE_MOST; }

}  // namespace
}  // namespace lowbit

extern "C" int lowbit_paged_fork_cuda(const int32_t* d_parents, const int32_t* d_children, int F, int32_t* d_lens, int32_t* d_table, int64_t table_stride, int R, int width,
                                      const int32_t* d_free_pages, int n_pages, const int32_t* d_free_count, int32_t* d_free_left, int32_t* d_shared, int page_size,
                                      int32_t* d_src, int32_t* d_dst, int32_t* d_missing, void* stream) {
    reset_launch_count();
    if (!d_parents || !d_children || F <= 0 || F > SHARE_MOST || !d_lens || bad_table(d_table, table_stride, R, width) || !d_free_pages || n_pages <= 0 || n_pages > SHARE_MOST || !d_free_count || !d_free_left || !d_shared ||
        page_size <= 0 || !d_src || !d_dst || !d_missing) {
        set_error(LB_ERR_ARG, "lowbit_paged_fork_cuda: bad argument (forks %d, R %d, width %d, pages %d, page_size %d)", F, R, width, n_pages, page_size);
        return LB_ERR_ARG;
    }
    const ForkArgs A = {d_parents, d_children, F, d_lens, d_table, table_stride, R, width, d_free_pages, n_pages, d_free_count, d_free_left, d_shared, page_size, d_src, d_dst,
                        d_missing};
    cudaStream_t st = (cudaStream_t)stream;
    const bool many = (int64_t)F * width > SHARE_MANY;
    launch_behind(paged_fork_kernel, dim3((unsigned)(many ? wide_grid(F) : 1)), SHARE_THREADS, 0, st, launch_overlaps(st), A, !many);
    note_launch();
    if (many) {
        launch_behind(paged_fork_count_kernel, dim3(1), 1, 0, st, launch_overlaps(st), d_free_count, n_pages, d_free_left, d_missing);
        note_launch();
    }
    return check_launch();
}

extern "C" size_t lowbit_paged_share_release_workspace_size(int n_pages, int R, int width) {
    return n_pages > 0 && R > 0 && width > 0 ? ((size_t)n_pages * 2 + share_stretches(R, width) + 1) * sizeof(int32_t) : 0;
}

extern "C" int lowbit_paged_share_release_cuda(const uint8_t* d_done, const int32_t* d_held, int page_size, int R, int32_t* d_table, int64_t table_stride, int width,
                                               int32_t* d_free_pages, int n_pages, int32_t* d_free_count, int32_t* d_shared, void* workspace, size_t workspace_bytes,
                                               void* stream) {
    reset_launch_count();
    if (!d_done || bad_table(d_table, table_stride, R, width) || !d_free_pages || n_pages <= 0 || n_pages > SHARE_MOST || !d_free_count || !d_shared || (d_held && page_size <= 0)) {
        set_error(LB_ERR_ARG, "lowbit_paged_share_release_cuda: bad argument (R %d, width %d, pages %d, page_size %d)", R, width, n_pages, page_size);
        return LB_ERR_ARG;
    }
    if (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < lowbit_paged_share_release_workspace_size(n_pages, R, width)) {
        set_error(LB_ERR_WORKSPACE, "lowbit_paged_share_release_cuda: a workspace of lowbit_paged_share_release_workspace_size() bytes is needed");
        return LB_ERR_WORKSPACE;
    }
    int32_t* const w = (int32_t*)workspace;
    const ShareReleaseArgs A = {d_done, d_held, page_size, R, d_table, table_stride, width, d_free_pages, n_pages, d_free_count, d_shared, w, w + n_pages, w + 2 * (int64_t)n_pages};
    cudaStream_t st = (cudaStream_t)stream;
    if ((int64_t)R * width <= SHARE_MANY) {
        launch_behind(paged_share_release_kernel<-1>, dim3(1), SHARE_THREADS, 0, st, launch_overlaps(st), A);
        note_launch();
        return check_launch();
    }
    const dim3 grid((unsigned)wide_grid(share_stretches(R, width)));
    launch_behind(paged_share_release_kernel<0>, grid, SHARE_THREADS, 0, st, launch_overlaps(st), A);
    launch_behind(paged_share_release_kernel<1>, grid, SHARE_THREADS, 0, st, launch_overlaps(st), A);
    launch_behind(paged_share_release_kernel<2>, grid, SHARE_THREADS, 0, st, launch_overlaps(st), A);
    launch_behind(paged_share_release_kernel<3>, grid, SHARE_THREADS, 0, st, launch_overlaps(st), A);
    launch_behind(paged_share_count_kernel, dim3(1), 1, 0, st, launch_overlaps(st), A.gives + share_stretches(R, width), d_free_count);
    for (int i = 0; i < 5; i++) note_launch();
    return check_launch();
}

extern "C" size_t lowbit_paged_compact_workspace_size(int n_pages) { return n_pages > 0 ? (size_t)n_pages * 4 * sizeof(int32_t) : 0; }

extern "C" int lowbit_paged_compact_cuda(const int32_t* d_table, int64_t table_stride, int R, int width, const int32_t* d_free_pages, int n_pages, const int32_t* d_free_count,
                                         const int32_t* d_shared, int32_t* d_table_out, int32_t* d_free_pages_out, int32_t* d_free_count_out, int32_t* d_shared_out,
                                         int32_t* d_src, int32_t* d_dst, void* workspace, size_t workspace_bytes, void* stream) {
    reset_launch_count();
    if (bad_table(d_table, table_stride, R, width) || !d_free_pages || n_pages <= 0 || n_pages > SHARE_MOST || !d_free_count || !d_table_out || !d_free_pages_out || !d_free_count_out ||
        (d_shared != nullptr) != (d_shared_out != nullptr) || !d_src || !d_dst) {
        set_error(LB_ERR_ARG, "lowbit_paged_compact_cuda: bad argument (R %d, width %d, pages %d)", R, width, n_pages);
        return LB_ERR_ARG;
    }
    if (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < lowbit_paged_compact_workspace_size(n_pages)) {
        set_error(LB_ERR_WORKSPACE, "lowbit_paged_compact_cuda: a workspace of lowbit_paged_compact_workspace_size() bytes is needed");
        return LB_ERR_WORKSPACE;
    }
    int32_t* const w = (int32_t*)workspace;
    const CompactArgs A = {d_table, table_stride, R, width, d_free_pages, n_pages, d_free_count, d_shared, d_table_out, d_free_pages_out, d_free_count_out, d_shared_out, d_src, d_dst,
                           w, w + n_pages, w + 2 * (int64_t)n_pages, w + 3 * (int64_t)n_pages};
    const bool many = (int64_t)R * width + n_pages > SHARE_MANY;
    static bool configured[64] = {};                           // the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        cudaFuncSetAttribute(paged_compact_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(SHARE_MANY * 4 * sizeof(int32_t)));
        configured[dev & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(many ? 8 : 1);                          // a cluster of eight is the most that any device takes
    cfg.blockDim = dim3(SHARE_THREADS);
    cfg.dynamicSmemBytes = many ? 0 : lowbit_paged_compact_workspace_size(n_pages);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {many ? 8u : 1u, 1u, 1u};
    cfg.attrs = at;
    cfg.numAttrs = add_overlap(at, 1, launch_overlaps((cudaStream_t)stream));
    cudaLaunchKernelEx(&cfg, many ? paged_compact_kernel<false> : paged_compact_kernel<true>, A);
    note_launch();
    return check_launch();
}

extern "C" int lowbit_paged_copy_cuda(const int32_t* d_src, const int32_t* d_dst, int n, void* const* caches, int n_caches, int n_pages, int64_t page_stride_bytes,
                                      int64_t page_bytes, void* stream) {
    reset_launch_count();
    if (n < 0 || n_caches < 0 || (n > 0 && (!d_src || !d_dst)) || (n_caches > 0 && !caches) || n_pages <= 0 || page_bytes <= 0 || page_stride_bytes < page_bytes) {
        set_error(LB_ERR_ARG, "lowbit_paged_copy_cuda: bad argument (copies %d, caches %d, pages %d, %lld bytes every %lld)", n, n_caches, n_pages, (long long)page_bytes,
                  (long long)page_stride_bytes);
        return LB_ERR_ARG;
    }
    if (n == 0) return LB_OK;
    cudaStream_t st = (cudaStream_t)stream;
    for (int c0 = 0; c0 < n_caches; c0 += COPY_CACHES) {
        CopyArgs A;
        A.src = d_src; A.dst = d_dst; A.n = n; A.n_pages = n_pages; A.page_stride = page_stride_bytes; A.page_bytes = page_bytes;
        A.n_caches = n_caches - c0 < COPY_CACHES ? n_caches - c0 : COPY_CACHES;
        uintptr_t low = (uintptr_t)(page_stride_bytes | page_bytes);
        for (int c = 0; c < A.n_caches; c++) {
            if (!caches[c0 + c]) { set_error(LB_ERR_ARG, "lowbit_paged_copy_cuda: cache %d is missing", c0 + c); return LB_ERR_ARG; }
            A.caches[c] = (uint8_t*)caches[c0 + c];
            low |= (uintptr_t)caches[c0 + c];
        }
        const bool wide = !(low & 15);
        A.piece_bytes = (int64_t)COPY_THREADS * COPY_DEEP * (wide ? 16 : 1);
        const int64_t pieces = (page_bytes + A.piece_bytes - 1) / A.piece_bytes;
        if (pieces * A.n_caches > 0x7fffffffll) { set_error(LB_ERR_ARG, "lowbit_paged_copy_cuda: a page of %lld bytes", (long long)page_bytes); return LB_ERR_ARG; }
        A.pieces = (int)pieces;
        const int64_t items = pieces * A.n_caches * n, most = (int64_t)sm_count() * 8;
        const dim3 grid((unsigned)(items < most ? items : most));
        launch_behind(wide ? paged_copy_kernel<uint4> : paged_copy_kernel<uint8_t>, grid, COPY_THREADS, 0, st, launch_overlaps(st), A);
        note_launch();
        if (const int rc = check_launch()) return rc;
    }
    return LB_OK;
}
