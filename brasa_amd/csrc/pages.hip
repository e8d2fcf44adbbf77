// Bookkeeping of the paged KV cache's pages: forking and freeing of sequences, reserving positions
// (allocation and copy on write), compaction.
//
// A table row lists a sequence's pages (-1: none), ref[p] counts the rows' entries that name page p.
// All of it is whole numbers, and every choice goes by order (lowest free page, first owner), so the
// results do not depend on how the atomics of a launch interleave.
//
// Bound: latency for the tables (a few thousand entries; one workgroup walks them, so that no launch
// waits for another), HBM for the pages that move.
#include "paged.hpp"

namespace brasa {
namespace {

constexpr int kPagesThreads = 1024;
constexpr int kPagesWaves = kPagesThreads / 64;

// exclusive sum over the workgroup's threads; `sum` is the total. s: kPagesWaves + 1 ints of LDS.
__device__ __forceinline__ int block_scan(int x, int* s, int& sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int incl = wave_scan(x);
    __syncthreads();  // s is free
    if (lane == 63) s[wave] = incl;
    __syncthreads();
    if (wave == 0) {
        const int w = lane < kPagesWaves ? s[lane] : 0;
        const int i = wave_scan(w);
        if (lane < kPagesWaves) s[lane] = i - w;
        if (lane == kPagesWaves - 1) s[kPagesWaves] = i;
    }
    __syncthreads();
    sum = s[kPagesWaves];
    return s[wave] + incl - x;
}

__device__ __forceinline__ void copy_ints(int* dst, const int* src, long long n) {
    if (dst == src) return;
    for (long long i = threadIdx.x; i < n; i += kPagesThreads) dst[i] = src[i];
}

// ---- fork ---------------------------------------------------------------------------------------
struct ForkArgs {
    const int* parent;
    const int* table;
    const int* len;
    int* table_out;
    int* len_out;
    int* ref;
    int n, width, pages;
};

// entries [i0, n * width) by `step`: row i takes row parent[i]; the old row's pages lose an owner,
// the new one's gain one
__device__ __forceinline__ void fork_entries(const ForkArgs& a, long long i0, long long step) {
    const long long all = (long long)a.n * a.width;
    for (long long i = i0; i < all; i += step) {
        const int row = (int)(i / a.width), col = (int)(i - (long long)row * a.width);
        int parent = a.parent[row];
        if (parent < 0 || parent >= a.n) parent = -1;
        const int old = a.table[i];
        const int now = parent < 0 ? -1 : a.table[(long long)parent * a.width + col];
        a.table_out[i] = now;
        if (col == 0) a.len_out[row] = parent < 0 ? 0 : a.len[parent];
        if (parent == row) continue;
        if (old >= 0 && old < a.pages) atomicAdd(a.ref + old, -1);
        if (now >= 0 && now < a.pages) atomicAdd(a.ref + now, 1);
    }
}

__global__ void __launch_bounds__(kPagesThreads)
fork_small_kernel(ForkArgs a, const int* ref_in) {
    copy_ints(a.ref, ref_in, a.pages);
    __threadfence();
    __syncthreads();
    fork_entries(a, threadIdx.x, kPagesThreads);
}
__global__ void __launch_bounds__(256)
fork_kernel(ForkArgs a) {
    fork_entries(a, (long long)blockIdx.x * 256 + threadIdx.x, (long long)gridDim.x * 256);
}
__global__ void __launch_bounds__(256)
copy_ints_kernel(int* dst, const int* src, int n) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) dst[i] = src[i];
}

// ---- the moves of pages -----------------------------------------------------------------------
// The workspace of reserve and compact: the moves' count, then the lists.
struct MoveList {
    int* count;
    int* src;
    int* dst;
    int* held;   // live positions of the page (kPage: all)
    int* tmp;    // reserve: claims and first claim of each page; compact: unused
    int* free_ids;
    uint8_t* take;
};

// One head's page (8 KB each of K and V) per workgroup and step: 16-byte pieces, all of a step's
// loads in flight at once.
__global__ void __launch_bounds__(256)
move_pages_kernel(PoolArgs p, MoveList m, bool whole) {
    const int heads = p.layers * p.hkv;
    const long long units = (long long)*m.count * heads;
    for (long long w = blockIdx.x; w < units; w += gridDim.x) {
        const int i = (int)(w / heads), lh = (int)(w % heads);
        const int layer = lh / p.hkv, kh = lh % p.hkv;
        const int bytes = (whole ? kPage : m.held[i]) * kDim;
        const size_t src = ((size_t)layer * p.pages + m.src[i]) * p.hkv + kh;
        const size_t dst = ((size_t)layer * p.pages + m.dst[i]) * p.hkv + kh;
        u32x4 x[4];
        const int off[2] = {16 * (int)threadIdx.x, 16 * (int)threadIdx.x + 4096};
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (off[j] < bytes) {
                x[j] = *reinterpret_cast<const u32x4*>(p.k + src * kTileBytes8 + off[j]);
                x[2 + j] = *reinterpret_cast<const u32x4*>(p.v + src * kTileBytes8 + off[j]);
            }
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (off[j] < bytes) {
                *reinterpret_cast<u32x4*>(p.k + dst * kTileBytes8 + off[j]) = x[j];
                *reinterpret_cast<u32x4*>(p.v + dst * kTileBytes8 + off[j]) = x[2 + j];
            }
        if (threadIdx.x == 0) p.kx[dst] = p.kx[src];
        if (threadIdx.x == 64) p.vx[dst] = p.vx[src];
    }
}

// ---- reserve ------------------------------------------------------------------------------------
struct ReserveArgs {
    const int* add;
    const int* table;
    const int* len;
    const int* ref;
    int* table_out;
    int* ref_out;
    int* status;
    int n, width, pages;
    MoveList m;
};

// Calls f(valid, row, block, len, claim number) in rounds of the whole workgroup, the claims in order:
// blocks [len / 64, (len + add) / 64 up) of each row with add > 0.
template <typename F>
__device__ __forceinline__ void for_claims(const ReserveArgs& a, int* s_scan, int* s_end, F f) {
    long long base = 0;
    for (int r0 = 0; r0 < a.n; r0 += kPagesThreads) {
        const int r = r0 + threadIdx.x;
        int c = 0;
        if (r < a.n && a.add[r] > 0) {
            const int len = max(a.len[r], 0);
            c = max(min((int)(((long long)len + a.add[r] + kPage - 1) / kPage), a.width) - len / kPage, 0);
        }
        int sum;
        const int excl = block_scan(c, s_scan, sum);
        s_end[threadIdx.x] = excl + c;
        __syncthreads();
        const int rows = min(a.n - r0, kPagesThreads);
        for (int i0 = 0; i0 < sum; i0 += kPagesThreads) {
            const int i = i0 + threadIdx.x;
            int lo = 0, hi = rows - 1;  // the first row whose claims end past i
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (s_end[mid] > i) hi = mid;
                else lo = mid + 1;
            }
            const int row = r0 + lo;
            const int len = i < sum ? max(a.len[row], 0) : 0;
            const int block = len / kPage + i - (lo ? s_end[lo - 1] : 0);
            f(i < sum, row, block, len, base + i);
        }
        base += sum;
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kPagesThreads)
reserve_kernel(ReserveArgs a) {
    __shared__ int s_scan[kPagesWaves + 1];
    __shared__ int s_end[kPagesThreads];
    __shared__ int s_moves, s_refused;
    int* count = a.m.tmp;
    int* first = a.m.tmp + a.pages;
    auto page_of = [&](int row, int block) {
        const int e = a.table[(size_t)row * a.width + block];
        return e >= 0 && e < a.pages ? e : -1;
    };
    if (threadIdx.x == 0) s_moves = s_refused = 0;
    __syncthreads();
    copy_ints(a.table_out, a.table, (long long)a.n * a.width);
    copy_ints(a.ref_out, a.ref, a.pages);
    for (int r = threadIdx.x; r < a.n; r += kPagesThreads)
        if (a.add[r] > 0 && (long long)max(a.len[r], 0) + a.add[r] > (long long)a.width * kPage)
            s_refused = 1;  // more than the row's table holds
    // claims of each page that is claimed, and the first of them
    for_claims(a, s_scan, s_end, [&](bool on, int row, int block, int, long long) {
        const int e = on ? page_of(row, block) : -1;
        if (e >= 0) {
            count[e] = 0;
            first[e] = 0x7fffffff;
        }
    });
    __threadfence();
    __syncthreads();
    for_claims(a, s_scan, s_end, [&](bool on, int row, int block, int, long long i) {
        const int e = on ? page_of(row, block) : -1;
        if (e >= 0) {
            atomicAdd(count + e, 1);
            atomicMin(first + e, (int)i);
        }
    });
    __threadfence();
    __syncthreads();
    int need = 0;
    for_claims(a, s_scan, s_end, [&](bool on, int row, int block, int, long long i) {
        const int e = on ? page_of(row, block) : -1;
        bool take = on;
        // every owner claims it: the first keeps it
        if (e >= 0)
            take = !(a.ref[e] <= __hip_atomic_load(count + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) &&
                     __hip_atomic_load(first + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)i);
        if (on) a.m.take[i] = take;
        need += take;
    });
    int all;
    block_scan(need, s_scan, all);
    // the lowest free pages, as many as are needed
    int found = 0;
    for (int p0 = 0; p0 < a.pages && found < all; p0 += kPagesThreads) {
        const int p = p0 + threadIdx.x;
        const bool free = p < a.pages && a.ref[p] <= 0;
        int sum;
        const int at = found + block_scan(free, s_scan, sum);
        if (free && at < all) a.m.free_ids[at] = p;
        found += sum;
    }
    __threadfence();
    __syncthreads();
    const bool fits = found >= all && !s_refused;
    if (threadIdx.x == 0) {
        a.status[0] = fits ? all : 0;
        a.status[1] = s_refused ? -1 : max(all - found, 0);
    }
    if (fits) {
        int before = 0;
        for_claims(a, s_scan, s_end, [&](bool on, int row, int block, int len, long long i) {
            const bool take = on && a.m.take[i];
            int sum;
            const int rank = before + block_scan(take, s_scan, sum);
            before += sum;
            if (!take) return;
            const int e = page_of(row, block);
            const int page = a.m.free_ids[rank];
            a.ref_out[page] = 1;
            if (e >= 0) {
                atomicAdd(a.ref_out + e, -1);
                if (len > block * kPage) {  // the rows it holds are copied
                    const int k = atomicAdd(&s_moves, 1);
                    a.m.src[k] = e;
                    a.m.dst[k] = page;
                    a.m.held[k] = len - block * kPage;
                }
            }
            a.table_out[(size_t)row * a.width + block] = page;
        });
    }
    __syncthreads();
    if (threadIdx.x == 0) *a.m.count = s_moves;
}

// ---- compact ------------------------------------------------------------------------------------
struct CompactArgs {
    const int* table;
    const int* ref;
    int* table_out;
    int* ref_out;
    int* live;
    int n, width, pages;
    MoveList m;  // tmp: the new id of each page that moves
};

__global__ void __launch_bounds__(kPagesThreads)
compact_kernel(CompactArgs a) {
    __shared__ int s_scan[kPagesWaves + 1];
    int mine = 0, live;
    for (int p = threadIdx.x; p < a.pages; p += kPagesThreads) mine += a.ref[p] > 0;
    block_scan(mine, s_scan, live);
    int moves = 0, holes = 0;
    for (int p0 = 0; p0 < a.pages; p0 += kPagesThreads) {
        const int p = p0 + threadIdx.x;
        const bool used = p < a.pages && a.ref[p] > 0;
        int sum;
        // pages in use at or past `live` go down, free ones below it are filled
        const int at = block_scan(p >= live ? used : (p < a.pages && !used) << 16, s_scan, sum);
        if (p < a.pages && p >= live && used) a.m.src[moves + (at & 0xffff)] = p;
        if (p < a.pages && p < live && !used) a.m.dst[holes + (at >> 16)] = p;
        moves += sum & 0xffff;
        holes += sum >> 16;
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        *a.m.count = moves;
        *a.live = live;
    }
    for (int k = threadIdx.x; k < moves; k += kPagesThreads) a.m.tmp[a.m.src[k]] = a.m.dst[k];
    copy_ints(a.ref_out, a.ref, a.pages);
    __syncthreads();
    for (int k = threadIdx.x; k < moves; k += kPagesThreads) {
        const int s = a.m.src[k], d = a.m.dst[k];
        a.ref_out[d] = a.ref[s];
        a.ref_out[s] = 0;
    }
}

__global__ void __launch_bounds__(256)
remap_kernel(CompactArgs a) {
    const int live = *a.live;
    const long long all = (long long)a.n * a.width;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const int e = a.table[i];
        a.table_out[i] = e >= live && e < a.pages ? a.m.tmp[e] : e;
    }
}

size_t ints(size_t n) { return (n * sizeof(int) + 255) / 256 * 256; }

MoveList carve(void* ws, int n, int pages) {
    uint8_t* w = static_cast<uint8_t*>(ws);
    MoveList m;
    auto take = [&](size_t count) {
        int* p = reinterpret_cast<int*>(w);
        w += ints(count);
        return p;
    };
    const size_t most = (size_t)std::max(n, pages);
    m.count = take(1);
    m.src = take(most);
    m.dst = take(most);
    m.held = take(most);
    m.tmp = take(2 * (size_t)pages);
    m.free_ids = take(pages);
    m.take = w;
    return m;
}

int launch_moves(const PoolArgs& pool, const MoveList& m, long long most, bool whole, hipStream_t stream) {
    const long long units = most * pool.layers * pool.hkv;
    const unsigned grid = (unsigned)std::min<long long>(std::max<long long>(units, 1), 2048);
    hipLaunchKernelGGL(move_pages_kernel, dim3(grid), dim3(256), 0, stream, pool, m, whole);
    return check_launch("move_pages_kernel");
}

}  // namespace

size_t kv_pages_workspace_len(int pages, int n, int width) {
    return ints(1) + 3 * ints(std::max(n, pages)) + ints(2 * (size_t)pages) + ints(pages) +
           ((size_t)n * width + 255) / 256 * 256;
}

int kv_pages_fork_launch(const int* parent, const int* table, const int* len, const int* ref,
                         int* table_out, int* len_out, int* ref_out, int n, int width, int pages,
                         hipStream_t stream) {
    ForkArgs a{parent, table, len, table_out, len_out, ref_out, n, width, pages};
    const long long all = (long long)n * width;
    if (all <= 16384 && pages <= 16384) {
        hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kPagesThreads), 0, stream, a, ref);
        return check_launch("fork_small_kernel");
    }
    if (ref_out != ref) {
        hipLaunchKernelGGL(copy_ints_kernel, dim3(std::min((pages + 255) / 256, 1024)), dim3(256), 0, stream,
                           ref_out, ref, pages);
        const int st = check_launch("copy_ints_kernel");
        if (st != BRASA_OK) return st;
    }
    hipLaunchKernelGGL(fork_kernel, dim3((unsigned)std::min<long long>((all + 255) / 256, 2048)), dim3(256), 0,
                       stream, a);
    return check_launch("fork_kernel");
}

int kv_pages_reserve_launch(const PoolArgs& pool, const int* add, const int* table, const int* len,
                            const int* ref, int* table_out, int* ref_out, int* status, int n, int width,
                            void* ws, hipStream_t stream) {
    ReserveArgs a{add, table, len, ref, table_out, ref_out, status, n, width, pool.pages,
                  carve(ws, n, pool.pages)};
    hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kPagesThreads), 0, stream, a);
    const int st = check_launch("reserve_kernel");
    if (st != BRASA_OK) return st;
    return launch_moves(pool, a.m, n, false, stream);
}

int kv_pages_compact_launch(const PoolArgs& pool, const int* table, const int* ref, int* table_out,
                            int* ref_out, int* live, int n, int width, void* ws, hipStream_t stream) {
    CompactArgs a{table, ref, table_out, ref_out, live, n, width, pool.pages, carve(ws, n, pool.pages)};
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kPagesThreads), 0, stream, a);
    int st = check_launch("compact_kernel");
    if (st != BRASA_OK) return st;
    const long long all = (long long)n * width;
    if (all > 0) {
        hipLaunchKernelGGL(remap_kernel, dim3((unsigned)std::min<long long>((all + 255) / 256, 2048)), dim3(256),
                           0, stream, a);
        st = check_launch("remap_kernel");
        if (st != BRASA_OK) return st;
    }
    return launch_moves(pool, a.m, pool.pages / 2, true, stream);
}

}  // namespace brasa
