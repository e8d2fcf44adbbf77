// Bookkeeping of the paged KV cache's pages: forking and freeing of sequences, reserving positions
// (allocation and copy on write), compaction.
//
// A table row lists a sequence's pages (-1: none), ref[p] counts the rows' entries that name page p.
// All of it is whole numbers, and every choice goes by order (lowest free page, first owner), so the
// results do not depend on how the atomics of a launch interleave.
//
// Bound: latency for the tables (a few thousand entries), HBM for the pages that move. What has an order
// is decided by one workgroup in one launch, with its lists in LDS where they fit; what has none
// (copies of tables and counts, edits, moves) is spread over the chip. 128 sequences of 100 to 4000
// positions: fork 2.0 + 3.2 us, reserve 4.6 + 5.5; compaction of 1000 pages in 12 layers (364 of them
// move) 4.9 us of decisions and 150 of copies, 4.7 TB/s in and out, as an ordinary copy.
#include "paged.hpp"

namespace brasa {
namespace {

constexpr int kPagesThreads = 1024;
constexpr int kPagesWaves = kPagesThreads / 64;

// exclusive sum over the workgroup's threads; `sum` is the total. s: kPagesWaves ints of LDS, free
// again after the next barrier.
__device__ __forceinline__ int across_waves(int mine, int* s, int& sum) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __syncthreads();  // s is free
    if (lane == 0) s[wave] = mine;
    __syncthreads();
    static_assert(kPagesWaves == 16, "a row of 16 lanes scans the waves");
    int w = s[lane & 15];
    w += __builtin_amdgcn_update_dpp(0, w, 0x111, 0xF, 0xF, true);
    w += __builtin_amdgcn_update_dpp(0, w, 0x112, 0xF, 0xF, true);
    w += __builtin_amdgcn_update_dpp(0, w, 0x114, 0xF, 0xF, true);
    w += __builtin_amdgcn_update_dpp(0, w, 0x118, 0xF, 0xF, true);
    sum = __builtin_amdgcn_readlane(w, 15);
    return __builtin_amdgcn_readlane(w, wave) - mine;
}
__device__ __forceinline__ int block_scan(int x, int* s, int& sum) {
    const int incl = wave_scan(x);
    return across_waves(__builtin_amdgcn_readlane(incl, 63), s, sum) + incl - x;
}
// the same for truth values
__device__ __forceinline__ int block_rank(bool on, int* s, int& sum) {
    const unsigned long long b = __builtin_amdgcn_ballot_w64(on);
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
    return across_waves(__builtin_popcountll(b), s, sum) + before;
}
// Workgroup barrier after which the workgroup's earlier global stores and atomics have reached the L2,
// where its later atomics and device-scope loads see them.
__device__ __forceinline__ void stores_barrier() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}
__device__ __forceinline__ int ld_l2(const int* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// dst = src by `threads` threads, this one the tid-th, eight loads in flight
__device__ __forceinline__ void copy_ints(int* dst, const int* src, long long n, int tid, int threads) {
    if (dst == src) return;
    for (long long i = tid; i < n; i += 8LL * threads) {
        int x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = i + (long long)j * threads < n ? src[i + (long long)j * threads] : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + (long long)j * threads < n) dst[i + (long long)j * threads] = x[j];
    }
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

// Rows row0, row0 + rows, ...; a wave per row, a lane per entry, kForkRows rows' loads in flight
// together. Row i takes row parent[i]; the old row's pages lose an owner, the new one's gain one.
constexpr int kForkRows = 2;
__device__ __forceinline__ void fork_rows(const ForkArgs& a, int row0, int rows) {
    const int lane = threadIdx.x & 63;
    for (int i0 = row0; i0 < a.n; i0 += rows * kForkRows) {
        int parent[kForkRows];
#pragma unroll
        for (int j = 0; j < kForkRows; ++j) {
            const int i = i0 + j * rows;
            const int p = i < a.n ? a.parent[i] : -1;
            parent[j] = p < 0 || p >= a.n ? -1 : p;
        }
        for (int c0 = 0; c0 < a.width; c0 += 64) {
            const int col = c0 + lane;
            int old[kForkRows], now[kForkRows];
#pragma unroll
            for (int j = 0; j < kForkRows; ++j) {
                const int i = i0 + j * rows;
                old[j] = i < a.n && col < a.width ? a.table[(size_t)i * a.width + col] : -1;
                now[j] = parent[j] >= 0 && col < a.width ? a.table[(size_t)parent[j] * a.width + col] : -1;
            }
#pragma unroll
            for (int j = 0; j < kForkRows; ++j) {
                const int i = i0 + j * rows;
                if (i >= a.n) break;
                if (col < a.width) a.table_out[(size_t)i * a.width + col] = now[j];
                if (parent[j] == i) continue;
                if (old[j] >= 0 && old[j] < a.pages) atomicAdd(a.ref + old[j], -1);
                if (now[j] >= 0 && now[j] < a.pages) atomicAdd(a.ref + now[j], 1);
            }
        }
#pragma unroll
        for (int j = 0; j < kForkRows; ++j) {
            const int i = i0 + j * rows;
            if (i < a.n && lane == 0) a.len_out[i] = parent[j] < 0 ? 0 : a.len[parent[j]];
        }
    }
}

__global__ void __launch_bounds__(kPagesThreads)
fork_small_kernel(ForkArgs a, const int* ref_in) {
    copy_ints(a.ref, ref_in, a.pages, threadIdx.x, kPagesThreads);
    stores_barrier();
    fork_rows(a, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kPagesWaves);
}
__global__ void __launch_bounds__(256)
fork_kernel(ForkArgs a) {
    fork_rows(a, __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), gridDim.x * 4);
}
__global__ void __launch_bounds__(256)
copy_ints_kernel(int* dst, const int* src, int n) {
    copy_ints(dst, src, n, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ---- the moves of pages -----------------------------------------------------------------------
// The workspace of reserve and compact: what the first launch decides and the second carries out.
struct MoveList {
    int* count;     // [0] moves, [1] edits
    int* src;       // moves: page src to dst, its first `held` positions
    int* dst;
    int* held;
    int* entry;     // reserve, edits: table entry, its new page (and the one it held, or -1)
    int* page;
    int* was;
    int* tmp;       // reserve: claims and first claim of each page; compact: new ids
    int* free_ids;
    uint8_t* take;
};

// One head's page (8 KB each of K and V) per workgroup and step: 16-byte pieces, all of a step's
// loads in flight at once.
__device__ __forceinline__ void move_pages(const PoolArgs& p, const MoveList& m, bool whole) {
    const int heads = p.layers * p.hkv;
    const long long units = (long long)m.count[0] * heads;
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
    PoolArgs p;
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

// The claims of a row: blocks [len / 64, (len + add) / 64 up), none where add <= 0.
__device__ __forceinline__ int row_claims(const ReserveArgs& a, int len, int add) {
    if (add <= 0) return 0;
    return max(min((int)(((long long)len + add + kPage - 1) / kPage), a.width) - len / kPage, 0);
}
__device__ __forceinline__ int owned_page(const ReserveArgs& a, size_t entry) {
    const int e = a.table[entry];
    return e >= 0 && e < a.pages ? e : -1;
}
// Claim k of `rows` rows whose claims end at s_end[row]: its row (the first whose claims end past k)
// and its place among the row's.
__device__ __forceinline__ int claim_row(const int* s_end, int rows, int k, int& nth) {
    int lo = 0, hi = rows - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (s_end[mid] > k) hi = mid;
        else lo = mid + 1;
    }
    nth = k - (lo ? s_end[lo - 1] : 0);
    return lo;
}
// What one granted claim changes: the second launch's edit, and a move where the page it leaves
// holds positions of the row.
__device__ __forceinline__ void grant(const ReserveArgs& a, int k, int entry, int page, int was, int held,
                                      int* s_moves) {
    a.m.entry[k] = entry;
    a.m.page[k] = page;
    a.m.was[k] = was;
    if (was >= 0 && held > 0) {
        const int i = atomicAdd(s_moves, 1);
        a.m.src[i] = was;
        a.m.dst[i] = page;
        a.m.held[i] = held;
    }
}

// Calls f(valid, row, block, len, claim number) in rounds of the whole workgroup, the claims in order.
template <typename F>
__device__ __forceinline__ void for_claims(const ReserveArgs& a, int* s_scan, int* s_end, F f) {
    int base = 0;
    for (int r0 = 0; r0 < a.n; r0 += kPagesThreads) {
        const int r = r0 + threadIdx.x;
        const int c = r < a.n ? row_claims(a, max(a.len[r], 0), a.add[r]) : 0;
        int sum;
        const int excl = block_scan(c, s_scan, sum);
        s_end[threadIdx.x] = excl + c;
        __syncthreads();
        const int rows = min(a.n - r0, kPagesThreads);
        for (int i0 = 0; i0 < sum; i0 += kPagesThreads) {
            const int i = i0 + threadIdx.x;
            int nth;
            const int row = r0 + claim_row(s_end, rows, i, nth);
            const int len = i < sum ? max(a.len[row], 0) : 0;
            f(i < sum, row, len / kPage + nth, len, base + i);
        }
        base += sum;
        __syncthreads();
    }
}

// The general path: any number of rows and claims, in rounds of the workgroup, with the claims of each
// page counted in the workspace.
__device__ __forceinline__ void reserve_many(const ReserveArgs& a, bool refused, int* s_scan, int* s_end,
                                             int* s_moves) {
    int* count = a.m.tmp;
    int* first = a.m.tmp + a.pages;
    for_claims(a, s_scan, s_end, [&](bool on, int row, int block, int, int) {
        const int e = on ? owned_page(a, (size_t)row * a.width + block) : -1;
        if (e >= 0) {
            count[e] = 0;
            first[e] = 0x7fffffff;
        }
    });
    stores_barrier();
    for_claims(a, s_scan, s_end, [&](bool on, int row, int block, int, int i) {
        const int e = on ? owned_page(a, (size_t)row * a.width + block) : -1;
        if (e >= 0) {
            atomicAdd(count + e, 1);
            atomicMin(first + e, i);
        }
    });
    stores_barrier();
    int need = 0;
    for_claims(a, s_scan, s_end, [&](bool on, int row, int block, int, int i) {
        const int e = on ? owned_page(a, (size_t)row * a.width + block) : -1;
        // every owner claims it: the first keeps it
        const bool keeps = e >= 0 && a.ref[e] <= ld_l2(count + e) && ld_l2(first + e) == i;
        if (on) a.m.take[i] = !keeps;
        need += on && !keeps;
    });
    int all;
    block_scan(need, s_scan, all);
    // the lowest free pages, as many as are needed
    int found = 0;
    for (int p0 = 0; p0 < a.pages && found < all; p0 += kPagesThreads) {
        const int p = p0 + threadIdx.x;
        const bool free = p < a.pages && a.ref[p] <= 0;
        int sum;
        const int at = found + block_rank(free, s_scan, sum);
        if (free && at < all) a.m.free_ids[at] = p;
        found += sum;
    }
    stores_barrier();
    const bool fits = found >= all && !refused;
    if (threadIdx.x == 0) {
        a.status[0] = fits ? all : 0;
        a.status[1] = refused ? -1 : max(all - found, 0);
        a.m.count[1] = fits ? all : 0;
    }
    if (!fits) return;
    int before = 0;
    for_claims(a, s_scan, s_end, [&](bool on, int row, int block, int len, int i) {
        const bool take = on && a.m.take[i];
        int sum;
        const int rank = before + block_rank(take, s_scan, sum);
        before += sum;
        if (!take) return;
        const int entry = row * a.width + block;
        grant(a, rank, entry, ld_l2(a.m.free_ids + rank), owned_page(a, entry), len - block * kPage, s_moves);
    });
}

// Up to kPagesThreads rows and claims, as in a decode step: a claim per thread, the claims of a page
// counted in a hash table in LDS, free pages listed in LDS.
constexpr int kHash = 4 * kPagesThreads;  // slots: at most a quarter is taken, so a probe ends
struct ReserveLds {
    int scan[kPagesWaves];
    int end[kPagesThreads];
    int key[kHash], count[kHash], first[kHash];
    int free_ids[kPagesThreads];
    int moves, refused;
};

__device__ __forceinline__ void reserve_few(const ReserveArgs& a, ReserveLds& s, int claims, bool refused,
                                            int free0) {
    const int k = threadIdx.x;
    const bool on = k < claims;
    int nth, entry = 0, held = 0, e = -1;
    {
        const int row = claim_row(s.end, a.n, k, nth);
        if (on) {
            const int len = max(a.len[row], 0);
            entry = row * a.width + len / kPage + nth;
            held = nth ? 0 : len % kPage;
            e = owned_page(a, entry);
        }
    }
    const int owners = e >= 0 ? a.ref[e] : 0;
    int slot = -1;
    if (e >= 0) {
        slot = (int)((uint32_t)e * 2654435761u >> 20) & (kHash - 1);
        while (true) {
            const int was = atomicCAS(&s.key[slot], -1, e);
            if (was == -1 || was == e) break;
            slot = (slot + 1) & (kHash - 1);
        }
        atomicAdd(&s.count[slot], 1);
        atomicMin(&s.first[slot], k);
    }
    __syncthreads();
    // every owner claims it: the first keeps it
    const bool take = on && !(e >= 0 && owners <= s.count[slot] && s.first[slot] == k);
    int all;
    const int rank = block_rank(take, s.scan, all);
    int found = 0;
    for (int p0 = 0; p0 < a.pages && found < all; p0 += kPagesThreads) {
        const int p = p0 + threadIdx.x;
        const bool free = p < a.pages && (p0 ? a.ref[p] : free0) <= 0;
        int sum;
        const int at = found + block_rank(free, s.scan, sum);
        if (free && at < all) s.free_ids[at] = p;
        found += sum;
    }
    __syncthreads();
    const bool fits = found >= all && !refused;
    if (threadIdx.x == 0) {
        a.status[0] = fits ? all : 0;
        a.status[1] = refused ? -1 : max(all - found, 0);
        a.m.count[1] = fits ? all : 0;
    }
    if (fits && take) grant(a, rank, entry, s.free_ids[rank], e, held, &s.moves);
}

// Workgroup 0 decides; the others copy the table and the counts meanwhile.
__global__ void __launch_bounds__(kPagesThreads)
reserve_kernel(ReserveArgs a) {
    __shared__ ReserveLds s;
    if (blockIdx.x > 0) {
        const int tid = (blockIdx.x - 1) * kPagesThreads + threadIdx.x, threads = (gridDim.x - 1) * kPagesThreads;
        copy_ints(a.table_out, a.table, (long long)a.n * a.width, tid, threads);
        copy_ints(a.ref_out, a.ref, a.pages, tid, threads);
        return;
    }
    const int free0 = threadIdx.x < a.pages ? a.ref[threadIdx.x] : 1;
    if (threadIdx.x == 0) s.moves = s.refused = 0;
    for (int i = threadIdx.x; i < kHash; i += kPagesThreads) {
        s.key[i] = -1;
        s.count[i] = 0;
        s.first[i] = 0x7fffffff;
    }
    __syncthreads();
    int claims = 0;
    for (int r0 = 0; r0 < a.n; r0 += kPagesThreads) {
        const int r = r0 + threadIdx.x;
        const int len = r < a.n ? max(a.len[r], 0) : 0, add = r < a.n ? a.add[r] : 0;
        if (add > 0 && (long long)len + add > (long long)a.width * kPage) s.refused = 1;  // past the row's table
        const int c = row_claims(a, len, add);
        int sum;
        const int excl = block_scan(c, s.scan, sum);
        s.end[threadIdx.x] = excl + c;
        claims += sum;
    }
    __syncthreads();
    const bool refused = s.refused;
    if (a.n <= kPagesThreads && claims <= kPagesThreads) reserve_few(a, s, claims, refused, free0);
    else reserve_many(a, refused, s.scan, s.end, &s.moves);
    __syncthreads();
    if (threadIdx.x == 0) a.m.count[0] = s.moves;
}

__global__ void __launch_bounds__(256)
reserve_apply_kernel(ReserveArgs a) {
    const int edits = a.m.count[1];
    for (int i = blockIdx.x * 256 + threadIdx.x; i < edits; i += gridDim.x * 256) {
        const int was = a.m.was[i], page = a.m.page[i];
        a.table_out[a.m.entry[i]] = page;
        a.ref_out[page] = 1;
        if (was >= 0) atomicAdd(a.ref_out + was, -1);
    }
    move_pages(a.p, a.m, false);
}

// ---- compact ------------------------------------------------------------------------------------
struct CompactArgs {
    PoolArgs p;
    const int* table;
    const int* ref;
    int* table_out;
    int* ref_out;
    int* live;
    int n, width, pages;
    MoveList m;  // tmp: the new id of each page at or past *live
};

__global__ void __launch_bounds__(kPagesThreads)
compact_kernel(CompactArgs a) {
    __shared__ int s_scan[kPagesWaves];
    const int ref0 = threadIdx.x < a.pages ? a.ref[threadIdx.x] : 0;
    int mine = ref0 > 0, live;
    for (int p = kPagesThreads + threadIdx.x; p < a.pages; p += kPagesThreads) mine += a.ref[p] > 0;
    block_scan(mine, s_scan, live);
    int moves = 0, holes = 0;
    for (int p0 = 0; p0 < a.pages; p0 += kPagesThreads) {
        const int p = p0 + threadIdx.x;
        const bool used = p < a.pages && (p0 ? a.ref[p] : ref0) > 0;
        int sum;
        // pages in use at or past `live` go down, free ones below it are filled
        const int at = block_scan(p >= live ? used : (p < a.pages && !used) << 16, s_scan, sum);
        if (p < a.pages && p >= live) {
            if (used) a.m.src[moves + (at & 0xffff)] = p;
            else a.m.tmp[p] = p;  // an entry that names a free page stays as it is
        }
        if (p < a.pages && p < live && !used) a.m.dst[holes + (at >> 16)] = p;
        moves += sum & 0xffff;
        holes += sum >> 16;
    }
    copy_ints(a.ref_out, a.ref, a.pages, threadIdx.x, kPagesThreads);
    if (threadIdx.x == 0) {
        a.m.count[0] = moves;
        *a.live = live;
    }
    stores_barrier();
    for (int k = threadIdx.x; k < moves; k += kPagesThreads) {
        const int s = ld_l2(a.m.src + k), d = ld_l2(a.m.dst + k);
        a.m.tmp[s] = d;
        a.ref_out[d] = a.ref[s];
        a.ref_out[s] = 0;
    }
}

__global__ void __launch_bounds__(256)
compact_apply_kernel(CompactArgs a) {
    const int live = *a.live;
    const long long all = (long long)a.n * a.width;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const int e = a.table[i];
        a.table_out[i] = e >= live && e < a.pages ? a.m.tmp[e] : e;
    }
    move_pages(a.p, a.m, true);
}

size_t ints(size_t n) { return (n * sizeof(int) + 255) / 256 * 256; }

// most: moves (compact: of pages; reserve: one per row); claims: entries of the table, or pages
MoveList carve(void* ws, int n, int width, int pages) {
    uint8_t* w = static_cast<uint8_t*>(ws);
    MoveList m;
    auto take = [&](size_t count) {
        int* p = reinterpret_cast<int*>(w);
        w += ints(count);
        return p;
    };
    const size_t most = (size_t)std::max(n, pages);
    const size_t edits = std::min((size_t)n * width, (size_t)pages);  // an edit takes a page
    m.count = take(2);
    m.src = take(most);
    m.dst = take(most);
    m.held = take(most);
    m.entry = take(edits);
    m.page = take(edits);
    m.was = take(edits);
    m.tmp = take(2 * (size_t)pages);
    m.free_ids = take(pages);
    m.take = w;
    return m;
}

// workgroups of a launch that has `units` pieces of work at most
unsigned grid_of(long long units) { return (unsigned)std::min<long long>(std::max<long long>(units, 1), 16384); }

}  // namespace

size_t kv_pages_workspace_len(int pages, int n, int width) {
    const size_t edits = std::min((size_t)n * width, (size_t)pages);
    return ints(2) + 3 * ints(std::max(n, pages)) + 3 * ints(edits) + ints(2 * (size_t)pages) + ints(pages) +
           ((size_t)n * width + 255) / 256 * 256;
}

int kv_pages_fork_launch(const int* parent, const int* table, const int* len, const int* ref,
                         int* table_out, int* len_out, int* ref_out, int n, int width, int pages,
                         hipStream_t stream) {
    ForkArgs a{parent, table, len, table_out, len_out, ref_out, n, width, pages};
    // One workgroup's one launch for a few rows (60 entries: 2.4 us against 2.2 + 3.0), two launches of
    // many from there on (8064 entries: 11.2 us against 2.2 + 3.2).
    if ((long long)n * width <= 2048 && pages <= 16384) {
        hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kPagesThreads), 0, stream, a, ref);
        return check_launch("fork_small_kernel");
    }
    if (ref_out != ref) {
        hipLaunchKernelGGL(copy_ints_kernel, dim3(grid_of((pages + 2047) / 2048)), dim3(256), 0, stream,
                           ref_out, ref, pages);
        const int st = check_launch("copy_ints_kernel");
        if (st != BRASA_OK) return st;
    }
    hipLaunchKernelGGL(fork_kernel, dim3(grid_of((n + 3) / 4)), dim3(256), 0, stream, a);
    return check_launch("fork_kernel");
}

int kv_pages_reserve_launch(const PoolArgs& pool, const int* add, const int* table, const int* len,
                            const int* ref, int* table_out, int* ref_out, int* status, int n, int width,
                            void* ws, hipStream_t stream) {
    ReserveArgs a{pool, add, table, len, ref, table_out, ref_out, status, n, width, pool.pages,
                  carve(ws, n, width, pool.pages)};
    long long copies = 0;
    if (table_out != table) copies += (long long)n * width;
    if (ref_out != ref) copies += pool.pages;
    const unsigned others = copies ? grid_of((copies + 8 * kPagesThreads - 1) / (8 * kPagesThreads)) : 0;
    hipLaunchKernelGGL(reserve_kernel, dim3(1 + others), dim3(kPagesThreads), 0, stream, a);
    const int st = check_launch("reserve_kernel");
    if (st != BRASA_OK) return st;
    hipLaunchKernelGGL(reserve_apply_kernel, dim3(grid_of((long long)n * pool.layers * pool.hkv)), dim3(256), 0,
                       stream, a);
    return check_launch("reserve_apply_kernel");
}

int kv_pages_compact_launch(const PoolArgs& pool, const int* table, const int* ref, int* table_out,
                            int* ref_out, int* live, int n, int width, void* ws, hipStream_t stream) {
    CompactArgs a{pool, table, ref, table_out, ref_out, live, n, width, pool.pages,
                  carve(ws, n, width, pool.pages)};
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kPagesThreads), 0, stream, a);
    const int st = check_launch("compact_kernel");
    if (st != BRASA_OK) return st;
    const long long units = (long long)(pool.pages / 2) * pool.layers * pool.hkv;
    hipLaunchKernelGGL(compact_apply_kernel, dim3(grid_of(std::max(units, ((long long)n * width + 255) / 256))),
                       dim3(256), 0, stream, a);
    return check_launch("compact_apply_kernel");
}

}  // namespace brasa
