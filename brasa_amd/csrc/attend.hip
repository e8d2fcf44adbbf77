// Attention of new rows, one or many for each sequence, over the paged 8-bit cache, with the pages that
// a group of sequences shares read and multiplied once for all of the group's rows.
//
// o[t, h] = sum_j p_j v_j / sum_j p_j over the positions j <= the row's own, p_j = exp(q . k_j / sqrt(128)).
// The sums over two sets of positions join as (m, l, acc) pairs: with m = max(m1, m2), l = l1 2^(m1 - m)
// + l2 2^(m2 - m), and acc alike. So a row's positions may be cut anywhere, and the rows of several
// sequences may stand together in one product where they read the same pages.
//
// A column is a (row, query head) of a KV head; a tile is up to 32 columns over a run of pages of one table
// row, the work of one wave. The rows of a group's sequences that have too few for a tile of their own
// make prefix tiles over the shared pages, and each sequence's rows tiles over its other pages. All
// tiles of a KV head stand in one line by their pages, and wave w takes the w-th equal run of it, so
// that every CU has the same work whatever the lengths, which only the device knows. The plan kernel
// lays the line out once a step, every layer's launch walks it; a tile that a run's border cuts, or
// whose sequence has a prefix tile, leaves (m, l, acc) in the workspace and a second launch joins them
// in order, so the result does not depend on timing.
//
// Bound, 32 query heads over 8: for prompts and chunks the matrix cores and the vector instructions beside them
// (4988 rows over up to 13K positions, 333 GFLOP, each product twice: 670 us, 0.50 PFLOP/s, where a large product reaches 1.2;
// the short form 493, 0.68). For a step's single rows latency: four rows over 16K shared positions (33 MB) take 14.4 us, of
// which the six half pages of a wave are half and the loads header -> page ids and Q -> codes -> sums, each a
// trip of 0.6 to 1.5 us, the rest; 64 sequences behind 8192 shared positions (71 MB) 41 to 43 us, 32 to 34 in the short form.
#include <climits>
#include <type_traits>

#include "paged.hpp"

namespace brasa {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kCols = 32;     // columns of a tile
constexpr int kRuns = 2048;   // waves of a launch: two per SIMD
// Pages whose time a tile costs beside its own. 32 heads over 8, us a layer with its share of the plan: with 6 eight
// sequences of 4 to 5K positions take 22.8, 32 behind 4096 shared ones 23.3, a batch of 64 behind 8192 46.0, drafts 40.6; with
// 4 23.8, 23.8, 45.8 and 40.4, with 8 23.7, 24.9, 46.7 and 41.7, with 2 24.4, 23.1, 45.3 and 42.9.
constexpr int kOver = 6;
// Length of a run in a line of `total` pages cut into at most `runs`: one wave per SIMD while that leaves it up to
// kLongRun pages, and else two waves. A wave more costs its way to the first product, 4 us, and its parts their
// joining; with more waves than SIMDs but fewer than two each, most wait for few. (32 heads over 8. Two waves throughout: four
// rows over 16K positions 20.8 us a layer in place of 18.2, a batch of 64 48.9 in place of 46.0, drafts 43.0 in place of
// 40.6; one throughout: prompts 354 in place of 335, chunks 717 in place of 673.)
constexpr int kLongRun = 48;
__device__ __forceinline__ long long run_pages(long long total, int runs) {
    const long long half = (total + runs / 2 - 1) / (runs / 2);
    return half <= kLongRun ? half : (total + runs - 1) / runs;
}

struct Tile {
    int seq;          // table row whose pages it reads
    int row0;         // own tile: the sequence's first packed row; prefix tile: the group's first, or offset in the row list
    int col0, cols;   // its columns among the sequence's, or the group's
    int b0, b1;       // pages
    int pos0;         // own tile: position of the sequence's first new row
    int kind;         // TileKind
    long long start;  // of its pages in the line
    int base, parts;  // partials: columns base + part * cols + column; parts of it
    int run0;         // run of its first part
    int ptile, pcol;  // prefix tile and its column where the tile's first column continues; -1: none
    int index;        // its own
};
static_assert(sizeof(Tile) == 64, "a tile is one line");
// kInRow: a prefix tile whose group's sharing rows are all packed behind each other (a load less before Q's).
// kOnce: the tile holds all columns of its sequence or group, and its pages pass the caches by (four rows over 16K positions
// 18.2 us a layer in place of 19.5, eight sequences of 4 to 5K 22.8 in place of 25.0, a batch of 64 46.0 in place of 47.1; for
// all tiles prompts take 371 in place of 335, chunks 821 in place of 673). (Another sequence may name the same pages, where it
// is in no group, has positions below the group's prefix or just a tile's columns: its tile reads them from HBM too.)
enum TileKind { kPrefix = 1, kDirect = 2, kBad = 4, kInRow = 8, kOnce = 16 };

// Columns whose parts a workgroup of the merge joins: `many` of one tile, which continue in one prefix tile or in none.
struct Join {
    int base, parts, cols;     // own parts: columns base + part * cols + column
    int pbase, pparts, pcols;  // the prefix tile's
    int row0, col0, many;      // columns from col0 on of the sequence whose first packed row is row0
    int lanes;                 // of a column: 32 or all
    int unused0, unused1;
};
static_assert(sizeof(Join) % 16 == 0, "read in wide pieces");
// Half a wave has eight parts on their way at once, and up to 32 of a column in four turns; more take the workgroup. The
// joining takes 4.0 us for four rows over 16K positions (about 80 parts a column), 5.1 for a batch of 64 (8 to 30), 19 to 22 for
// prompts (2 or 3). With half waves throughout the four rows' pass of 36 layers takes 904 us in place of 657, with workgroups the
// prompts' 401 in place of 335.
__host__ __device__ constexpr int join_lanes(int parts) { return parts <= 32 ? 32 : kThreads; }

// Where the plan and the partials stand in the workspace.
struct Places {
    size_t tiles, rows, ml, acc, bytes;
    long long cap;  // columns of partials, for each KV head
};
struct Layout : Places {
    size_t starts, merges;      // where hkv alone says
    size_t seqs, first, group;  // the plan's own lists
    int runs, max_tiles, max_merges;
};

struct Header {
    int magic, n, tokens, width, hq, hkv, runs, tiles, merges;
    long long size, total;  // of a run, of the line
    Places at;
};
constexpr int kMagic = 0x61747031;

// A sequence and a group as the plan sees them.
struct PlanSeq {
    int c0, rows;  // its packed rows
    int pos;       // of the first; -1: there is no page for it
    int group;     // whose prefix it may share; -1: none
    int scol;      // columns of such sequences before it
};
struct PlanGroup {
    int s0, s1;      // its sequences
    int lead, many;  // the first of those that may share its prefix, and how many
    int pages;       // of its prefix
    int end;         // packed row behind theirs
};

__host__ __device__ constexpr size_t up256(size_t x) { return (x + 255) / 256 * 256; }

constexpr size_t kStarts = up256(sizeof(Header));
__host__ __device__ constexpr size_t merges_at(int runs) { return kStarts + up256(sizeof(Tile) * (size_t)runs); }

Layout layout(int n, int groups, int tokens, int hq, int hkv) {
    Layout l;
    const long long g = hq / hkv, cols = (long long)tokens * g, seqs = std::min(n, tokens);
    // columns of sequences that may share: each has fewer than a tile's
    const long long shared = groups ? std::min(cols, seqs * (kCols - 1)) : 0;
    l.runs = std::max(kRuns / hkv, kWaves);
    l.max_tiles = (int)(seqs + cols / kCols + (groups ? std::min((long long)groups, seqs) + shared / kCols : 0));
    // all shared columns, and those of the tiles that a run's border cuts; each column once
    l.max_merges = (int)std::min(shared + (long long)l.runs * std::min((long long)kCols, cols), cols);
    // shared columns once in each of the two tiles, and for each border a tile's columns once or twice
    l.cap = 2 * shared + 2LL * l.runs * std::min((long long)kCols, cols);
    size_t at = up256(sizeof(Header));
    auto take = [&](size_t bytes) {
        const size_t a = at;
        at += up256(bytes);
        return a;
    };
    l.starts = take(sizeof(Tile) * (size_t)l.runs);  // (at kStarts)
    l.merges = take(sizeof(Join) * (size_t)l.max_merges);
    l.tiles = take(sizeof(Tile) * (size_t)l.max_tiles);
    l.seqs = take(sizeof(PlanSeq) * (size_t)n);
    l.first = take(4 * ((size_t)groups + n + 1));
    l.group = take(sizeof(PlanGroup) * (size_t)groups);
    l.rows = take(groups ? 4 * (size_t)tokens : 0);
    l.ml = take(8 * (size_t)l.cap * hkv);
    l.acc = take(4 * kDim * (size_t)l.cap * hkv);
    l.bytes = at;
    return l;
}

// ---- the plan -----------------------------------------------------------------------------------
//
// One workgroup: sequences, then groups and sequences again (how many tiles each has), then the tiles, a
// thread for each of them. Bound: the latency of that chain of loads and scans, once a step.
struct PlanArgs {
    Header* head;
    Tile* start;  // [runs]: the tile where each run starts
    Tile* tile;
    Join* merge;
    PlanSeq* seq;
    int* first;  // [groups + n + 1]: first tile of each group's prefix, then of each sequence
    PlanGroup* grp;
    int* rows;  // packed rows of the sequences that may share, in order
    int n, groups, width, tokens, hq, hkv, per_row, runs;
    Places at;
};

// exclusive sum over a workgroup of W waves of values up to 2^62; s: W of LDS
template <int W>
__device__ __forceinline__ long long block_scan64(long long x, long long* s, long long& sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    long long incl = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const long long y = __shfl_up(incl, d);
        if (lane >= d) incl += y;
    }
    __syncthreads();  // s is free
    if (lane == 63) s[wave] = incl;
    __syncthreads();
    long long before = 0;
    sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const long long y = s[w];
        if (w < wave) before += y;
        sum += y;
    }
    return before + incl - x;
}
// inclusive maximum over the workgroup and `before`; `all`: of the whole workgroup
template <int W>
__device__ __forceinline__ int block_max(int x, int before, int* s, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = max(x, before);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x = max(x, y);
    }
    __syncthreads();  // s is free
    if (lane == 63) s[wave] = x;
    __syncthreads();
    all = before;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int y = s[w];
        if (w < wave) x = max(x, y);
        all = max(all, y);
    }
    return x;
}
// x / d for 0 <= x < 2^52, d > 0, with inv = 1.0 / d
__device__ __forceinline__ long long div_by(long long x, long long d, double inv) {
    long long q = (long long)((double)x * inv);
    q -= q * d > x;
    q += (q + 1) * d <= x;
    return q;
}
// IN_LDS: the lists of sequences and groups fit the LDS (up to kPlanLds of each); else they stand in the
// workspace, and every look at one costs a trip to the L2 (64 sequences in one group 15.9 us in place of 11.8).
// Up to kPlanFew sequences and tiles take as many threads, whose scans wait for four waves only (the same 64 in 8.7
// us; one sequence 5.2 in place of 8.2, 24 sequences' drafts 9.2 in place of 11.9).
constexpr int kPlanLds = 1024, kPlanFew = 256;
template <bool IN_LDS, int THREADS>
__global__ void __launch_bounds__(THREADS)
attend_plan_kernel(const int* cu, const int* pos, const int* group, const int* prefix, int n, int groups, PlanArgs a) {
    constexpr int kInLds = !IN_LDS ? 1 : std::min(THREADS, kPlanLds), W = THREADS / 64;
    __shared__ PlanSeq s_seq[kInLds];
    __shared__ PlanGroup s_grp[kInLds];
    __shared__ int s_first[2 * kInLds + 1];
    PlanSeq* const seqs = IN_LDS ? s_seq : a.seq;
    PlanGroup* const grps = IN_LDS ? s_grp : a.grp;
    int* const firsts = IN_LDS ? s_first : a.first;
    // (within the workgroup, but past its L1 where they stand in the workspace)
    auto ld_l2 = [](const int* p) { return IN_LDS ? *p : brasa::ld_l2(p); };
    auto st_l2 = [](int* p, int x) {
        if (IN_LDS) *p = x;
        else __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    __shared__ long long s_scan[W];
    __shared__ int s_scan32[W];
    __shared__ Tile s_tile[THREADS];  // one a thread
    __shared__ int s_unit[THREADS];   // first unit of each tile's columns to join
    const int tid = threadIdx.x;
    const int per_row = a.per_row;
    // (the first of each list at once: what follows then waits for one trip to memory, not for three)
    struct In {
        int cu0, cu1, pos;
    };
    struct InGroup {
        int s0, s1, prefix;
    };
    auto load_in = [&](int i) { return i < n ? In{cu[i], cu[i + 1], pos[i]} : In{0, 0, -1}; };
    auto load_group = [&](int g) { return g < groups ? InGroup{group[g], group[g + 1], prefix[g]} : InGroup{0, 0, 0}; };
    const In in0 = load_in(tid);
    const InGroup group0 = load_group(tid);

    // ---- groups: runs of sequences, in order and apart ------------------------------------------
    for (int g0 = 0, before = 0; g0 < a.groups; g0 += THREADS) {
        const int g = g0 + tid;
        int all;
        const InGroup in = g0 ? load_group(g) : group0;
        const int s0 = block_max<W>(min(max(in.s0, 0), a.n), before, s_scan32, all);
        const int s1 = max(s0, min(max(in.s1, 0), a.n));
        before = all;
        if (g < a.groups) {
            st_l2(&grps[g].s0, s0);
            st_l2(&grps[g].s1, s1);
            st_l2(&grps[g].lead, a.n);
            st_l2(&grps[g].many, 0);
            st_l2(&grps[g].end, 0);
            st_l2(&grps[g].pages, min(max(in.prefix, 0) / kPage, a.width));
        }
    }
    if (a.groups) stores_barrier();
    auto prefix_pages = [&](int g) { return ld_l2(&grps[g].pages); };

    // ---- sequences: their rows, in order and apart, and who may share a prefix --------------------
    int scols = 0;
    for (int i0 = 0, before = 0; i0 < a.n; i0 += THREADS) {
        const int i = i0 + tid;
        int all;
        const In in = i0 ? load_in(i) : in0;
        const int c0 = block_max<W>(min(max(in.cu0, 0), a.tokens), before, s_scan32, all);
        before = all;
        PlanSeq s;
        s.c0 = c0;
        s.rows = max(min(max(in.cu1, 0), a.tokens) - c0, 0);
        s.pos = in.pos;
        if (s.pos >= a.width * kPage) s.pos = -1;
        s.group = -1;
        int cols = 0;
        // (whose rows all stand behind the prefix, and do not fill a tile)
        if (a.groups && s.rows > 0 && s.rows < kCols && s.rows * per_row < kCols) {
            int lo = 0, hi = a.groups;  // the last group that starts at or before i
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (ld_l2(&grps[mid].s0) <= i) lo = mid;
                else hi = mid;
            }
            if (ld_l2(&grps[lo].s0) <= i && i < ld_l2(&grps[lo].s1)) {
                const int pages = prefix_pages(lo);
                if (pages > 0 && s.pos >= pages * kPage) {
                    s.group = lo;
                    cols = s.rows * per_row;
                    atomicMin(&grps[lo].lead, i);
                    atomicAdd(&grps[lo].many, 1);
                    atomicMax(&grps[lo].end, c0 + s.rows);
                }
            }
        }
        if (a.groups) {
            int sum;
            s.scol = scols + block_scan<W>(cols, s_scan32, sum);
            scols += sum;
            // (the rows of one that turns out to be alone in its group are listed, and not used)
            for (int r = 0; cols && r < s.rows; ++r) a.rows[s.scol / per_row + r] = s.c0 + r;
        }
        if (i < a.n) {
            st_l2(&seqs[i].c0, s.c0);
            st_l2(&seqs[i].rows, s.rows);
            st_l2(&seqs[i].pos, s.pos);
            st_l2(&seqs[i].group, s.group);
            st_l2(&seqs[i].scol, s.scol);
        }
    }
    stores_barrier();
    auto load_seq = [&](int i) {
        PlanSeq s = {ld_l2(&seqs[i].c0), ld_l2(&seqs[i].rows), ld_l2(&seqs[i].pos), ld_l2(&seqs[i].group), 0};
        if (s.group >= 0) {
            if (ld_l2(&grps[s.group].many) < 2) s.group = -1;
            else s.scol = ld_l2(&seqs[i].scol);
        }
        return s;
    };
    // columns of a group's sharing sequences, and how many there are before them in the list
    auto group_cols = [&](int g, int& col0) {
        if (ld_l2(&grps[g].many) < 2) return 0;
        const int s0 = ld_l2(&grps[g].s0), s1 = ld_l2(&grps[g].s1);
        col0 = ld_l2(&seqs[s0].scol);
        return (s1 < a.n ? ld_l2(&seqs[s1].scol) : scols) - col0;
    };

    // ---- how many tiles each has ------------------------------------------------------------------
    int ntiles = 0;
    const int entries = a.groups + a.n;
    for (int e0 = 0; e0 < entries; e0 += THREADS) {
        const int e = e0 + tid;
        int tiles = 0, col0;
        if (e < a.groups) tiles = (group_cols(e, col0) + kCols - 1) / kCols;
        else if (e < entries) tiles = (int)(((long long)ld_l2(&seqs[e - a.groups].rows) * per_row + kCols - 1) / kCols);
        int sum;
        const int at = ntiles + block_scan<W>(tiles, s_scan32, sum);
        ntiles += sum;
        if (e < entries) st_l2(firsts + e, at);
    }
    if (tid == 0) st_l2(firsts + entries, ntiles);
    stores_barrier();

    auto make_tile = [&](int at) {
        int lo = 0, hi = entries;  // the last group or sequence that starts at or before `at`: one with tiles
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (ld_l2(firsts + mid) <= at) lo = mid;
            else hi = mid;
        }
        Tile t;
        t.col0 = (at - ld_l2(firsts + lo)) * kCols;
        t.ptile = t.pcol = -1;
        if (lo < a.groups) {
            int col0;
            const int cols = group_cols(lo, col0);
            t.kind = kPrefix;
            t.seq = ld_l2(&grps[lo].lead);
            const int r0 = ld_l2(&seqs[t.seq].c0);
            if ((ld_l2(&grps[lo].end) - r0) * (long long)per_row == cols) {
                t.kind |= kInRow;
                t.row0 = r0;
            } else {
                t.row0 = col0 / per_row;
            }
            t.cols = min(cols - t.col0, kCols);
            if (cols <= kCols) t.kind |= kOnce;
            t.b0 = 0;
            t.b1 = prefix_pages(lo);
            t.pos0 = 0;
        } else {
            const int i = lo - a.groups;
            const PlanSeq s = load_seq(i);
            t.kind = (s.pos < 0 ? kBad : 0) | ((long long)s.rows * per_row <= kCols ? kOnce : 0);
            t.seq = i;
            t.row0 = s.c0;
            t.cols = (int)min((long long)s.rows * per_row - t.col0, (long long)kCols);
            t.b0 = s.group >= 0 ? prefix_pages(s.group) : 0;
            // (a sequence without a place gets one page, not read, whose tile writes NaN)
            const int last = (t.col0 + t.cols - 1) / per_row;
            t.b1 = s.pos < 0 ? 1 : min((int)(((long long)s.pos + last) / kPage) + 1, a.width);
            t.pos0 = s.pos;
            if (s.group >= 0) {
                int gcol0 = 0;
                group_cols(s.group, gcol0);
                t.ptile = ld_l2(firsts + s.group) + (s.scol - gcol0) / kCols;
                t.pcol = (s.scol - gcol0) % kCols;
            }
        }
        t.index = at;
        return t;
    };

    // ---- the line's length, and that of a run -----------------------------------------------------
    long long mine = 0, total;
    Tile t = {};
    for (int i = tid; i < ntiles; i += THREADS) {
        t = make_tile(i);
        mine += kOver + t.b1 - t.b0;
    }
    const long long before = block_scan64<W>(mine, s_scan, total);
    const long long size = run_pages(total, a.runs);
    const double inv = 1.0 / (double)size;

    // ---- the tiles, and the tile where each run starts ----------------------------------------------
    const bool one_round = ntiles <= THREADS;
    long long line = 0, cols = 0;
    for (int t0 = 0; t0 < ntiles; t0 += THREADS) {
        const int at = t0 + tid, many = min(ntiles - t0, THREADS);
        const bool on = at < ntiles;
        if (on && !one_round) t = make_tile(at);  // (else it is at hand)
        const long long len = on ? t.b1 - t.b0 : 0, line0 = line;
        long long sum = total;
        t.start = (one_round ? before : line + block_scan64<W>(on ? len + kOver : 0, s_scan, sum)) + kOver;
        line += sum;
        t.run0 = (int)div_by(t.start, size, inv);
        const int last = on ? (int)div_by(t.start + len - 1, size, inv) : 0;
        t.parts = last - t.run0 + 1;
        if (!(t.kind & kPrefix) && t.ptile < 0 && t.parts == 1) t.kind |= kDirect;
        const long long part_cols = on && !(t.kind & kDirect) ? (long long)t.cols * t.parts : 0;
        t.base = (int)(cols + block_scan64<W>(part_cols, s_scan, sum));
        cols += sum;
        if (on) s_tile[tid] = t;
        __syncthreads();
        // (through the LDS: written by their threads, 64 lines an instruction, and a tile of many runs by one thread, both
        // took 13 of 29 thousand cycles for drafts)
        for (int k = tid; k < 4 * many; k += THREADS)
            reinterpret_cast<u32x4*>(a.tile + t0)[k] = reinterpret_cast<const u32x4*>(s_tile)[k];
        const int w1 = (int)div_by(line + size - 1, size, inv);
        for (int w = (int)div_by(line0 + size - 1, size, inv) + tid; w < w1; w += THREADS) {
            int lo = 0, hi = many - 1;  // the first tile that ends behind the run's start
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (s_tile[mid].start + (s_tile[mid].b1 - s_tile[mid].b0) > w * size) hi = mid;
                else lo = mid + 1;
            }
            a.start[w] = s_tile[lo];
        }
    }
    if (!one_round) stores_barrier();

    // ---- the columns to join ----------------------------------------------------------------------
    // A tile's columns in its first prefix tile, or all (side 0), and those in the next one.
    auto join_of = [&](const Tile& x, int side) {
        const int border = x.ptile >= 0 ? min(kCols - x.pcol, x.cols) : x.cols, c0 = side ? border : 0;
        Join j = {};
        j.base = x.base + c0;
        j.parts = x.parts;
        j.cols = x.cols;
        j.row0 = x.row0;
        j.col0 = x.col0 + c0;
        j.many = side ? x.cols - border : border;
        if (x.ptile >= 0 && j.many > 0) {
            const int pt = x.ptile + side;
            j.pparts = one_round ? s_tile[pt].parts : brasa::ld_l2(&a.tile[pt].parts);
            j.pcols = one_round ? s_tile[pt].cols : brasa::ld_l2(&a.tile[pt].cols);
            j.pbase = (one_round ? s_tile[pt].base : brasa::ld_l2(&a.tile[pt].base)) + (side ? 0 : x.pcol);
        }
        j.lanes = join_lanes(j.parts + j.pparts);
        return j;
    };
    auto units_of = [](const Join& j) { return (j.many * j.lanes + kThreads - 1) / kThreads; };
    int merges = 0;
    for (int t0 = 0; t0 < ntiles; t0 += THREADS) {
        const int many = min(ntiles - t0, THREADS);
        int units = 0, sum;
        if (tid < many) {
            if (!one_round) t = a.tile[t0 + tid];
            if (!(t.kind & (kPrefix | kDirect))) units = units_of(join_of(t, 0)) + units_of(join_of(t, 1));
        }
        s_unit[tid] = block_scan<W>(units, s_scan32, sum);
        __syncthreads();
        for (int u = tid; u < sum; u += THREADS) {
            int lo = 0, hi = many;  // the last tile that starts at or before u: one with units
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (s_unit[mid] <= u) lo = mid;
                else hi = mid;
            }
            const Tile x = one_round ? s_tile[lo] : a.tile[t0 + lo];
            Join j = join_of(x, 0);
            int r = u - s_unit[lo];
            if (r >= units_of(j)) {
                r -= units_of(j);
                j = join_of(x, 1);
            }
            const int each = kThreads / j.lanes;
            j.base += r * each;
            j.pbase += r * each;
            j.col0 += r * each;
            j.many = min(j.many - r * each, each);
            a.merge[merges + u] = j;
        }
        merges += sum;
    }
    if (tid == 0) {
        a.head->magic = kMagic;
        a.head->n = a.n;
        a.head->tokens = a.tokens;
        a.head->width = a.width;
        a.head->hq = a.hq;
        a.head->hkv = a.hkv;
        a.head->runs = a.runs;
        a.head->tiles = ntiles;
        a.head->merges = merges;
        a.head->size = size;
        a.head->total = line;
        a.head->at.tiles = a.at.tiles;
        a.head->at.rows = a.at.rows;
        a.head->at.ml = a.at.ml;
        a.head->at.acc = a.at.acc;
        a.head->at.bytes = a.at.bytes;
        a.head->at.cap = a.at.cap;
    }
}

// ---- tiles --------------------------------------------------------------------------------------
//
// A wave holds 32 columns and takes 32 keys (half a page) at a time, on its own: no wave waits for another.
// K's and V's codes are copied into the wave's LDS, one half page ahead, in pieces of 16 bytes (a vector
// memory instruction costs a CU about 20 cycles whatever its width, and V by 4 bytes a lane, as its
// operand wants them, took 16 for a half page: 410 of 560 us of a pass were loads). Rows are swizzled:
// 16-byte piece c of row r stands in place c ^ (r & 7), so that rows are read and transposed without
// bank conflicts. K's codes are converted exactly (an e4m3 value is an f16 value) into the A operand of
// S^T = K Q^T on 32x32x16 f16 MFMAs. S^T's layout is the B operand of O^T += V^T P^T: lane (c, h) holds
// keys 16 st + 8 (j / 4) + 4 h + j % 4 of column c, j < 8, and V's rows stand in LDS in that order, so that
// ds_read_b64_tr_b8 gives a lane eight keys of one dim at once.
//
// ws, hkv and runs are kernel arguments of their own, before the others: such ones are in scalar registers when a
// wave starts, and the header and the run's tile need not wait for the rest (0.3 us).
struct AttendArgs {
    uint8_t* ws;
    size_t ws_len;
    const float* q;
    PoolArgs p;  // of one layer
    const int* table;
    void* o;
    int n, width, tokens, hq, per_row, o_f16;
};
struct AttendCall {  // the kernels' arguments as they stand in memory
    uint8_t* ws;
    int hkv, runs;
    AttendArgs a;
};
// The workspace's header and the parts it names.
struct Plan {
    Header head;
    float* ml;
    float* acc;
    bool fits;  // it is a plan of this call's sizes
};
__device__ __forceinline__ Plan load_plan(const uint8_t* ws, const AttendArgs& a) {
    Plan p;
    p.head = *reinterpret_cast<const Header*>(ws);
    const Header& h = p.head;
    p.fits = h.magic == kMagic && h.n == a.n && h.tokens == a.tokens && h.width == a.width && h.hq == a.hq &&
             h.hkv == a.p.hkv && h.at.bytes <= a.ws_len;
    p.ml = reinterpret_cast<float*>(a.ws + h.at.ml);
    p.acc = reinterpret_cast<float*>(a.ws + h.at.acc);
    return p;
}

template <typename T>
__device__ __forceinline__ T load_line(const T* p) {
    union {
        T t;
        uint32_t w[sizeof(T) / 4];
    } u;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) u.w[i] = ((Scalar<uint32_t>)(uintptr_t)p)[i];
    return u.t;
}

__device__ __forceinline__ f32x16 mfma32(half8v a, half8v b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// e4m3 codes 0, 1 (2, 3) of a word -> f16 values, exact
__device__ __forceinline__ half2v f16_of_lo(uint32_t w) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}
__device__ __forceinline__ half2v f16_of_hi(uint32_t w) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
}
__device__ __forceinline__ half8v join(half2v a, half2v b, half2v c, half2v d) {
    return half8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// x and y as f16 halves hi + lo (up to 2^-22 of each)
__device__ __forceinline__ void split(float x, float y, half2v& hi, half2v& lo) {
    hi = half2v{(_Float16)x, (_Float16)y};
    // (kept as one register: the remainders are then mixed FMAs of it, not conversions made again)
    asm volatile("" : "+v"(hi));
    lo = half2v{(_Float16)fmaf((float)hi.x, -1.0f, x), (_Float16)fmaf((float)hi.y, -1.0f, y)};
}
// 0x80 in the places of a word's NaN codes
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// over the two lanes c, c + 32 of a column
__device__ __forceinline__ float max_h(float x) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ __forceinline__ float sum_h(float x) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return __int_as_float(b[0]) + __int_as_float(b[1]);
}
// weight of a part whose largest score is m in a sum whose largest is top (no key: m = -inf)
__device__ __forceinline__ float part_weight(float m, float top) {
    return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}
// x times 1 / l, in o's type
template <bool F16>
__device__ __forceinline__ void write_o(void* o, size_t at, f32x4 x, float inv) {
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = x[e] * inv;
    if (F16) {
        u32x2 w = {f2h(y[0]) | (uint32_t)f2h(y[1]) << 16, f2h(y[2]) | (uint32_t)f2h(y[3]) << 16};
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(o) + at) = w;
    } else {
        *reinterpret_cast<f32x4*>(static_cast<float*>(o) + at) = y;
    }
}

// Keeps what is written before it before what is written after: the products below stand among the vector
// instructions that run beside them.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// Half a page's codes from p on (this lane's share of it) into the LDS at `to`, whole: K's row r to row r.
// NT: they pass the caches by, for pages that no other tile reads.
#define COPY_KEYS(NT)                                            \
    asm volatile(                                                \
        "s_mov_b32 %0, m0\n\t"                                   \
        "s_mov_b32 m0, %2\n\t"                                   \
        "s_nop 2\n\t"                                            \
        "global_load_lds_dwordx4 %1, off" NT "\n\t"              \
        "global_load_lds_dwordx4 %1, off offset:1024" NT "\n\t"  \
        "global_load_lds_dwordx4 %1, off offset:2048" NT "\n\t"  \
        "global_load_lds_dwordx4 %1, off offset:3072" NT "\n\t"  \
        "s_mov_b32 m0, %0"                                       \
        : "=&s"(saved)                                           \
        : "v"(p), "s"(to)                                        \
        : "memory")
__device__ __forceinline__ void copy_keys(const uint8_t* p, uint32_t to, bool once) {
    uint32_t saved;
    if (once) COPY_KEYS(" nt");
    else COPY_KEYS("");
}
#undef COPY_KEYS
// V's row of key 16 st + 8 (j / 4) + 4 h + j % 4 to row 16 st + 8 h + j (an instruction's offset counts in
// memory and in LDS; the second half's 512 bytes in memory are 1024 in LDS).
#define COPY_VALUES(NT)                                          \
    asm volatile(                                                \
        "s_mov_b32 %0, m0\n\t"                                   \
        "s_mov_b32 m0, %2\n\t"                                   \
        "s_nop 2\n\t"                                            \
        "global_load_lds_dwordx4 %1, off" NT "\n\t"              \
        "global_load_lds_dwordx4 %1, off offset:2048" NT "\n\t"  \
        "s_mov_b32 m0, %3\n\t"                                   \
        "s_nop 2\n\t"                                            \
        "global_load_lds_dwordx4 %1, off offset:512" NT "\n\t"   \
        "global_load_lds_dwordx4 %1, off offset:2560" NT "\n\t"  \
        "s_mov_b32 m0, %0"                                       \
        : "=&s"(saved)                                           \
        : "v"(p), "s"(to), "s"(to + 512)                         \
        : "memory")
__device__ __forceinline__ void copy_values(const uint8_t* p, uint32_t to, bool once) {
    uint32_t saved;
    if (once) COPY_VALUES(" nt");
    else COPY_VALUES("");
}
#undef COPY_VALUES
// 16 bytes a lane from p into the LDS at `to`, one lane's behind another's.
__device__ __forceinline__ void copy_rows(const float* p, uint32_t to) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 2\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(p), "s"(to)
        : "memory");
}
typedef int i32x2 __attribute__((ext_vector_type(2)));
// eight codes of one dim -> f16 values
__device__ __forceinline__ half8v value_op(i32x2 w) {
    return join(f16_of_lo(w.x), f16_of_hi(w.x), f16_of_lo(w.y), f16_of_hi(w.y));
}
// V^T P^T of 32 keys added to acc (rows 32 t .. + 32 of V^T in acc[t]): the operand of each product is made while
// the one before it runs.
template <bool EXACT>
__device__ __forceinline__ void add_pv(const i32x2 (&v)[2][4], const half8v (&hi)[2], const half8v (&lo)[2],
                                       f32x16 (&acc)[4]) {
    half8v now = value_op(v[0][0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int st = i >> 2, t = i & 3;
        acc[t] = mfma32(now, hi[st], acc[t]);
        if constexpr (EXACT) acc[t] = mfma32(now, lo[st], acc[t]);
        in_order();
        if (i < 7) now = value_op(v[(i + 1) >> 2][(i + 1) & 3]);
        in_order();
    }
}

// Q of a wave's columns as the B operands of S^T = K Q^T: f16 values, and what they leave over, as f16 values
// too (EXACT: 22 bits together, as the paged decode takes them) or, where the caller asks for fewer bits, as e4m3 codes of 2^11
// times it (15 bits, at half the matrix cores' time, and K's codes are the other operand as they are).
template <bool EXACT>
struct QueryOps {
    half8v hi[8];
    half8v lo[EXACT ? 8 : 1];
    i32x8 lo8[EXACT ? 1 : 2];
};
constexpr int kLoScale = 127 - 11;  // 2^-11 as an exponent byte
__device__ __forceinline__ half8v key_op(const u32x4 (&kw)[4], int i) {
    const uint32_t w0 = kw[i >> 1][2 * (i & 1)], w1 = kw[i >> 1][2 * (i & 1) + 1];
    return join(f16_of_lo(w0), f16_of_hi(w0), f16_of_lo(w1), f16_of_hi(w1));
}
// S^T of 32 keys, and beside it `work(0)` .. `work(9)`, vector instructions that do not depend on it.
template <bool EXACT, typename W>
__device__ __forceinline__ f32x16 scores(const u32x4 (&kw)[4], const QueryOps<EXACT>& q, W work) {
    f32x16 s;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = 0.0f;
    half8v now, next;
    if constexpr (!EXACT) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4 a = kw[2 * i], b = kw[2 * i + 1];
            const i32x8 k = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
            s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, q.lo8[i], s, 0, 0, 0, 127, 0, kLoScale);
            in_order();
            if (i == 1) now = key_op(kw, 0);
            work(i);
            in_order();
        }
    } else {
        now = key_op(kw, 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s = mfma32(now, q.hi[i], s);
        if constexpr (EXACT) s = mfma32(now, q.lo[i], s);
        in_order();
        if (i < 7) next = key_op(kw, i + 1);
        work(i + 2);
        in_order();
        now = next;
    }
    return s;
}

// A half page that not all columns see whole: V's rows behind the last key that any sees become zeros in
// LDS (whatever stands there), and NaN values that some columns see and others do not become 0 there and
// NaN in the sums of the columns that see them. `last1`, `last`: the last key that any column, and this
// lane's, sees, from the half page's first on. Rare: one or two half pages of a sequence.
__device__ __forceinline__ uint64_t hidden_rows(uint8_t* v, int* first, int last1) {
    const int lane = threadIdx.x & 63;
    // two lanes a row, four pieces of 16 bytes each
    const int row = lane >> 1, j = row & 7;
    const int key = 16 * (row >> 4) + 8 * (j >> 2) + 4 * (row >> 3 & 1) + (j & 3);
    u32x4* at = reinterpret_cast<u32x4*>(v + row * kDim + 64 * (lane & 1));
    first[lane] = first[lane + 64] = 64;  // (no key)
    uint32_t nans = 0;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        u32x4 w = at[i];
        if (key > last1) w = u32x4{0, 0, 0, 0};
        const int dim = 16 * ((4 * (lane & 1) + i) ^ j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t n = nan_codes(w[e]);
            nans |= n;
#pragma unroll 1
            for (int b = 0; n && b < 4; ++b)
                if (n >> 8 * b & 0x80u) atomicMin(&first[dim + 4 * e + b], key);
            w[e] &= ~((n >> 7) * 0xffu);
        }
        at[i] = w;
    }
    return __builtin_amdgcn_ballot_w64(nans != 0);
}
__device__ __forceinline__ void hide_values(uint8_t* v, int* first, int last1, int last, f32x16 (&acc)[4]) {
    if (!hidden_rows(v, first, last1)) return;
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (first[32 * (i >> 2) + 8 * (i & 3) + 4 * h + r] <= min(last, 63)) acc[i >> 2][4 * (i & 3) + r] = NAN;
        in_order();
    }
}

template <bool EXACT, bool F16>
__global__ void __launch_bounds__(kThreads, 2)
attend_kernel(uint8_t* ws, int hkv, int runs, AttendArgs a) {
    constexpr int kHalf = 32 * kDim;  // codes of half a page
    // a wave's: V's two halves, K's; before them Q's rows and behind them the result's, 512 bytes a column
    __shared__ __attribute__((aligned(16))) uint8_t s_kv[kWaves][4 * kHalf];
    static_assert(4 * kHalf == kCols * 4 * kDim, "32 columns of f32");
    __shared__ __attribute__((aligned(16))) int s_nan[kWaves][kDim];  // first key with a NaN value, for each dim
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, h = lane >> 5;
    const int kh = blockIdx.x % hkv, run = blockIdx.x / hkv * kWaves + wave;
    // The arguments and the header are read again where they are needed: held in scalar registers over
    // the loop they would crowd out its own.
    auto args = [] { return (Scalar<AttendArgs>)(again(__builtin_amdgcn_kernarg_segment_ptr()) + offsetof(AttendCall, a)); };
    auto header = [&] { return (Scalar<Header>)(uintptr_t)args()->ws; };
    // (a run's first tile comes with the header, before it is known to be one)
    Tile t = load_line(reinterpret_cast<const Tile*>(ws + kStarts) + min(run, runs - 1));
    {
        const Plan plan = load_plan(ws, a);
        if (!plan.fits || run >= plan.head.runs || run * plan.head.size >= plan.head.total) return;
    }

    while (true) {
        // ---- this run's pages of the tile ------------------------------------------------------------
        const int ti = t.index;
        int p0, p1, row0, col0, cols, pos0, kind, part0;
        const int* ids;
        {
            const auto g = args();
            const auto hd = header();
            const long long lo = run * hd->size, end = min(lo + hd->size, (long long)hd->total);
            if (t.start >= end) break;
            p0 = t.b0 + (int)max(lo - t.start, 0LL);
            p1 = min(t.b0 + (int)min(end - t.start, (long long)INT_MAX / 2), t.b1);
            ids = g->table + (size_t)t.seq * g->width;
            row0 = t.row0;
            col0 = t.col0;
            cols = t.cols;
            pos0 = t.pos0;
            kind = t.kind;
            part0 = t.base + (run - t.run0) * cols;
        }
        if (p0 < p1) {
        const bool nowhere = kind & kBad, once = kind & kOnce;

        // this lane's share of a half page's copies, and where it reads them
        const uint32_t j8 = lane >> 3, piece = ((lane & 7) ^ j8) * 16;
        const uint32_t k_from = j8 * kDim + piece, v_from = 1024 * (j8 >> 2) + kDim * (j8 & 3) + piece;
        const uint32_t k_at = c * kDim + ((h ^ (c & 7)) * 16), jv = (lane & 15) >> 1;
        const uint32_t v_at = (8 * h + jv) * kDim + 8 * (lane & 1) + ((((lane >> 4) & 1) ^ jv) * 16);
        const uint32_t k_lds = __builtin_amdgcn_readfirstlane(lds_addr(s_kv[wave]) + 2 * kHalf);
        const uint32_t v_lds = __builtin_amdgcn_readfirstlane(lds_addr(s_kv[wave]));
        auto load_k = [&](uint32_t tile, int half) {
            copy_keys(a.p.k + (size_t)tile * kTileBytes8 + half * kHalf + k_from, k_lds + half * kHalf, once);
        };
        auto load_v = [&](uint32_t tile, int half) {
            copy_values(a.p.v + (size_t)tile * kTileBytes8 + half * kHalf + v_from, v_lds + half * kHalf, once);
        };
        // Pages 64 at a time, a lane each: their tiles (page 0's in the place of one that is not there), which
        // are there, and their scale bytes. (Through the scalar cache they would have every LDS read wait
        // for them: both count in one counter, and scalar loads return in any order.)
        uint32_t tile_of_lane, kx_of_lane, vx_of_lane;
        uint64_t are_there;
        auto look_up = [&](int id) {  // of this lane's page
            const bool there = id >= 0 && id < a.p.pages;
            tile_of_lane = (uint32_t)(there ? id : 0) * a.p.hkv + kh;  // (a layer has at most 2^31 of them)
            are_there = __builtin_amdgcn_ballot_w64(there);
            kx_of_lane = a.p.kx[tile_of_lane];
            vx_of_lane = a.p.vx[tile_of_lane];
        };
        int looked_up = p0;  // the first of the 64
        const int first_id = nowhere ? 0 : ids[min(p0 + lane, p1 - 1)];  // (one without a place: page 0, not used)
        uint32_t tile;

        // ---- Q: hi and lo parts of q / sqrt(128) * log2 e, each column's exponent taken out ------------
        int limit;  // the last position this lane's column sees
        QueryOps<EXACT> q;
        int qx;
        {
            const auto g = args();
            const int cc = min(c, cols - 1);  // (lanes past the last column repeat it)
            const int col = col0 + cc, local = col / g->per_row;
            int row = row0 + local;
            if ((kind & (kPrefix | kInRow)) == kPrefix) row = reinterpret_cast<const int*>(g->ws + header()->at.rows)[row];
            const int q_row = row * g->hq + kh * g->per_row + col - local * g->per_row;
            limit = kind & kPrefix ? INT_MAX : nowhere ? -1 : pos0 + local;
            // Q's rows, two an instruction, as K's and V's codes: 16-byte piece p of column c in place p ^ c. (By lanes,
            // as the operands want them, an instruction touches 64 lines; with eight waves on a CU Q then took 7600
            // cycles of a tile, and so 4400.)
            const float* const qs = g->q;
            int slot = c ^ h;
            asm volatile("" : "+v"(slot));  // (or sixteen of them are kept over the tiles)
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) {
                if (2 * i >= cols) break;
                const int r0 = __builtin_amdgcn_readlane(q_row, 2 * i), r1 = __builtin_amdgcn_readlane(q_row, 2 * i + 1);
                copy_rows(qs + (size_t)(h ? r1 : r0) * kDim + 4 * (slot ^ 2 * i), v_lds + 1024 * i);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            // step s holds dims 32 (s / 2) + 16 h + 8 (s % 2) .. + 8, as K's 16-byte pieces do
            const uint32_t q_at = cc * 4 * kDim + 16 * (4 * h ^ cc);
            f32x4 raw[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
                raw[i] = *reinterpret_cast<const f32x4*>(&s_kv[wave][q_at ^ 16 * (8 * (i >> 2) + 2 * ((i >> 1) & 1) + (i & 1))]);
            // Q here, then the first page's copies on their way, then the work on Q under them. (The compiler
            // does not count the copies: a wait for an earlier load would be one for them too.)
#pragma unroll
            for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(raw[i]));
            in_order();
            look_up(first_id);
            tile = __builtin_amdgcn_readlane(tile_of_lane, 0);
            load_k(tile, 0);
            load_k(tile, 1);
            load_v(tile, 0);
            in_order();
            constexpr float kScale = 0.08838834764831845f * kLog2e;
            float qmax = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                qmax = fmaxf(fmaxf(qmax, fabsf(raw[i][0])), fabsf(raw[i][1]));
                qmax = fmaxf(fmaxf(qmax, fabsf(raw[i][2])), fabsf(raw[i][3]));
            }
            qmax = max_h(qmax) * kScale;
            // the row's largest to [2^8, 2^9) (below 2^-112 it stays less: every score is 0 there)
            qx = max((int)(__float_as_uint(qmax) >> 23) - 127 - 8, -120);
            const float up = ldexpf(kScale, -qx), up11 = up * 0x1p11f;
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                half2v u[4], w[4];
                float rest[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x0 = raw[2 * s + (j >> 1)][2 * (j & 1)], x1 = raw[2 * s + (j >> 1)][2 * (j & 1) + 1];
                    split(x0 * up, x1 * up, u[j], w[j]);
                    if constexpr (!EXACT) {  // (times 2^11: exact)
                        rest[2 * j] = fmaf((float)u[j].x, -0x1p11f, x0 * up11);
                        rest[2 * j + 1] = fmaf((float)u[j].y, -0x1p11f, x1 * up11);
                    }
                }
                q.hi[s] = join(u[0], u[1], u[2], u[3]);
                if constexpr (EXACT) {
                    q.lo[s] = join(w[0], w[1], w[2], w[3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        int word = __builtin_amdgcn_cvt_pk_fp8_f32(rest[4 * j], rest[4 * j + 1], 0, false);
                        word = __builtin_amdgcn_cvt_pk_fp8_f32(rest[4 * j + 2], rest[4 * j + 3], word, true);
                        q.lo8[s >> 2][2 * (s & 3) + j] = word;
                    }
                }
            }
            in_order();
            asm volatile("" : "+v"(kx_of_lane), "+v"(vx_of_lane));
        }
        // the least and the largest position that a column of this wave sees
        int lim0 = limit, lim1 = limit;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            lim0 = min(lim0, __shfl_xor(lim0, d));
            lim1 = max(lim1, __shfl_xor(lim1, d));
        }
        lim0 = __builtin_amdgcn_readfirstlane(lim0);
        lim1 = __builtin_amdgcn_readfirstlane(lim1);

        float m_used = -INFINITY, lsum = 0.0f;
        f32x16 acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
        int vref = 0;     // this lane's column of acc stands in units of 2^(vref - 127)

        u32x4 kw[4];    // key c, dims 32 i + 16 h .. + 16
        i32x2 vw[2][4]; // keys 16 st + 8 (j / 4) + 4 h + j % 4 of dim 32 t + c at [st][t]
        auto read_k = [&](int half) {
#pragma unroll
            for (int i = 0; i < 4; ++i) kw[i] = *reinterpret_cast<const u32x4*>(&s_kv[wave][(2 + half) * kHalf + (k_at ^ 32 * i)]);
        };
        auto read_v = [&](int half) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                vw[i >> 2][i & 3] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (__attribute__((address_space(3))) i32x2*)&s_kv[wave][half * kHalf + 2048 * (i >> 2) + (v_at ^ 32 * (i & 3))]);
        };
        if (!nowhere) {
            int page = p0;
            uint32_t tile_next = tile;
            int kx = __builtin_amdgcn_readlane(kx_of_lane, 0), vx = __builtin_amdgcn_readlane(vx_of_lane, 0);
            bool there = are_there & 1;
            vref = vx;
            // the scores of the half page at hand: of key k0 + 8 q + 4 h + r and column c, in units of
            // log2 and of 2^(qx + kx - 127)
            wait_vmcnt<8>();
            read_k(0);
            f32x16 s = scores(kw, q, [](int) {});

            // One half page: its weights, the scores of the next, and its share of the sums. K of the half
            // after the next and V of the next go on their way first: into the places of what has been used.
            auto half_page = [&](auto HALF, bool more) {
                constexpr int half = HALF;
                const int k0 = page * kPage + 32 * half;
                if (half == 0) {
                    if (more) load_k(tile_next, 0);
                    load_v(tile, 1);
                    if (more) wait_vmcnt<8>();
                    else wait_vmcnt<4>();
                } else if (more) {
                    load_k(tile_next, 1);
                    load_v(tile_next, 0);
                    wait_vmcnt<8>();
                } else {
                    wait_vmcnt<0>();
                }
                // (behind the last page K is an earlier one's, and its scores are not used)
                read_k(half ^ 1);
                // (past the clamp every score is 0, or so far from the next that one key takes all)
                const float sc = ldexpf(1.0f, min(max(qx + kx - 127, -126), 127));
                if (!there) lsum = limit >= page * kPage ? NAN : lsum;
                if (k0 + 31 > lim0) {  // some column does not see all of these keys
                    // (keys counted from k0 + 4 h, so that they are constants)
                    const int last = limit - k0 - 4 * h;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (8 * (i >> 2) + (i & 3) > last) s[i] = -INFINITY;
                    hide_values(&s_kv[wave][half * kHalf], s_nan[wave], lim1 - k0, limit - k0, acc);
                }
                float top = fmaxf(fmaxf(s[12], s[13]), fmaxf(s[14], s[15]));
#pragma unroll
                for (int i = 0; i < 12; i += 3) top = fmaxf(top, fmaxf(fmaxf(s[i], s[i + 1]), s[i + 2]));
                // Two reference points of each column, both powers of two: m_used for l, which moves when the largest
                // score has grown by 2^8 past it, and m_used + vref for acc, which moves when a weight times its page's
                // V scale has. So a key's f16 weight, p = 2^(score - m_used + 7 - less), keeps its bits wherever
                // its part of the sum is not far below the largest part, whatever scales the other pages have; p stays
                // below 2^15, and its bias of 2^7 keeps small p out of f16's subnormals.
                int less = vref - vx;
                if (__builtin_amdgcn_ballot_w64(top * sc > m_used + (float)(8 + min(less, 0)))) {
                    top = max_h(top) * sc;
                    const bool grow = top > m_used + 8.0f;
                    const float m = grow ? floorf(top) : m_used;
                    const int by = grow ? (int)fminf(m - m_used, 1000.0f) : 0;  // (from -inf: both sums are 0)
                    const int before = vref - by;
                    const float over = top - m;
                    vref = over + (float)(vx - 8) > (float)before ? vx + (int)floorf(over) : before;
                    m_used = m;
                    lsum *= ldexpf(1.0f, -by);
                    const float f = ldexpf(1.0f, before - vref);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i] *= f;
                    less = vref - vx;
                }
                // (from 2^40 on every p is 0 in f16; the limit is for l's sake)
                less = min(less, 64);
                // (a column that has seen no key yet: its scores are all -inf, and p 0)
                const float mb = m_used == -INFINITY ? 0.0f : (float)(7 - less) - m_used;
                in_order();
                f32x16 next;
                float p[16], psum = 0.0f;
                half8v ph[2], pl[2];
                auto weigh = [&](int i) {
                    p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], sc, mb));
                };
                auto pack = [&](int i) {  // weights 2 i, 2 i + 1
                    half2v u, w;
                    if constexpr (EXACT) {
                        split(p[2 * i], p[2 * i + 1], u, w);
                        pl[i >> 2][2 * (i & 3)] = w.x;
                        pl[i >> 2][2 * (i & 3) + 1] = w.y;
                    } else {
                        u = half2v{(_Float16)p[2 * i], (_Float16)p[2 * i + 1]};
                    }
                    ph[i >> 2][2 * (i & 3)] = u.x;
                    ph[i >> 2][2 * (i & 3) + 1] = u.y;
                    psum += p[2 * i];
                    psum += p[2 * i + 1];
                };
                read_v(half);
                next = scores(kw, q, [&](int i) {
                    if (i < 2) {
                        if constexpr (!EXACT) {
                            weigh(4 * i);
                            weigh(4 * i + 1);
                            weigh(4 * i + 2);
                            weigh(4 * i + 3);
                        }
                    } else if constexpr (EXACT) {
                        weigh(2 * i - 4);
                        weigh(2 * i - 3);
                        pack(i - 2);
                    } else {
                        weigh(6 + i);
                        pack(i - 2);
                    }
                });
                // (here, among the products, not sunk behind the branch below)
                asm volatile("" : "+v"(ph[0]), "+v"(ph[1]), "+v"(psum));
                lsum = fmaf(psum, ldexpf(1.0f, less), lsum);
                in_order();
                add_pv<EXACT>(vw, ph, pl, acc);
                s = next;
            };
            while (true) {
                const bool more = page + 1 < p1;
                if (more) {
                    if (page + 1 - looked_up == 64) {
                        looked_up += 64;
                        look_up(ids[min(looked_up + lane, p1 - 1)]);
                        asm volatile("" : "+v"(kx_of_lane), "+v"(vx_of_lane));  // (waited for here, not on every page)
                    }
                    tile_next = __builtin_amdgcn_readlane(tile_of_lane, page + 1 - looked_up);
                }
                half_page(std::integral_constant<int, 0>{}, more);
                half_page(std::integral_constant<int, 1>{}, more);
                if (!more) break;
                ++page;
                tile = tile_next;
                kx = __builtin_amdgcn_readlane(kx_of_lane, page - looked_up);
                vx = __builtin_amdgcn_readlane(vx_of_lane, page - looked_up);
                there = are_there >> (page - looked_up) & 1;
            }
        } else {
            wait_vmcnt<0>();  // (no copy outlives the workgroup)
        }
        // (a row past the table's width has no page)
        const auto g = args();
        if (nowhere || (!(kind & kPrefix) && limit >= g->width * kPage)) lsum = NAN;
        lsum = sum_h(lsum);
        const float unit = ldexpf(1.0f, vref - 127);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= unit;

        // ---- out: to o, or to the parts. The lane holds dims 32 t + 8 q + 4 h + r of its column -------------
        // and the rows leave through the LDS, two an instruction (straight from the lanes an instruction would touch
        // 64 lines, as Q's would).
        const bool direct = kind & kDirect;
        if (direct) {
            const float inv = 1.0f / lsum;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] *= inv;
        }
        uint32_t o_at = c * 4 * kDim + 16 * (h ^ c), piece_at = h * 4 * kDim + 16 * (h ^ c);
        asm volatile("" : "+v"(o_at), "+v"(piece_at));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const f32x16& x = acc[i >> 2];
            const int r = 4 * (i & 3);
            *reinterpret_cast<f32x4*>(&s_kv[wave][o_at ^ 16 * (8 * (i >> 2) + 2 * (i & 3))]) = f32x4{x[r], x[r + 1], x[r + 2], x[r + 3]};
        }
        asm volatile("" ::: "memory");
        auto column = [&](int i) {  // columns 2 i, 2 i + 1: this lane's piece
            return *reinterpret_cast<const f32x4*>(&s_kv[wave][(piece_at ^ 32 * i) + 8 * kDim * i]);
        };
        if (direct) {
            const int col = col0 + c, local = col / g->per_row;  // (a prefix tile is never direct)
            const int o_row = (row0 + local) * g->hq + kh * g->per_row + col - local * g->per_row;
            void* const o = g->o;
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) {
                if (2 * i >= cols) break;
                const int r0 = __builtin_amdgcn_readlane(o_row, 2 * i), r1 = __builtin_amdgcn_readlane(o_row, 2 * i + 1);
                const f32x4 x = column(i);
                if (2 * i + h < cols) write_o<F16>(o, (size_t)(h ? r1 : r0) * kDim + 4 * c, x, 1.0f);
            }
        } else {
            const auto hd = header();
            const size_t part = (size_t)kh * hd->at.cap + part0;
            float* to = reinterpret_cast<float*>(g->ws + hd->at.acc) + part * kDim + 4 * lane;
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) {
                if (2 * i >= cols) break;
                const f32x4 x = column(i);
                if (2 * i + h < cols) *reinterpret_cast<f32x4*>(to + 2 * kDim * i) = x;
            }
            if (lane < cols) *reinterpret_cast<f32x2*>(reinterpret_cast<float*>(g->ws + hd->at.ml) + 2 * (part + lane)) = f32x2{m_used, lsum};
        }
        }
        const auto hd = header();
        if (ti + 1 >= hd->tiles) break;
        t = load_line(reinterpret_cast<const Tile*>(args()->ws + hd->at.tiles) + ti + 1);
    }
}

// ---- parts into rows ----------------------------------------------------------------------------
//
// Half a wave per column, or a workgroup where it has many parts: each half wave joins them all, or every
// eighth, 16 bytes of their sums a lane and eight parts on their way at once, and then the halves theirs.
// Bound: the chain header -> unit -> parts -> o, and for prompts the parts' bytes.
__global__ void __launch_bounds__(kThreads)
attend_merge_kernel(uint8_t* ws, int hkv, int runs, AttendArgs a) {
    __shared__ __attribute__((aligned(16))) float s_x[kWaves][kDim];
    __shared__ f32x2 s_ml[kWaves];
    const Join* units = reinterpret_cast<const Join*>(ws + merges_at(runs));
    const int kh = blockIdx.x % hkv, e0 = blockIdx.x / hkv, es = gridDim.x / hkv;
    // (the first unit comes with the header, before it is known to be one)
    Join j = load_line(units + e0);
    const Plan plan = load_plan(ws, a);
    const Header& head = plan.head;
    const int lane = threadIdx.x & 63, h = lane >> 5, d = 4 * (lane & 31);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (!plan.fits) {  // of another step's sizes, or none: no row is left looking like a result
        const size_t all = (size_t)a.tokens * a.hq * kDim;
        for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (size_t)gridDim.x * kThreads) {
            if (a.o_f16) static_cast<uint16_t*>(a.o)[i] = 0x7e00;
            else static_cast<float*>(a.o)[i] = NAN;
        }
        return;
    }
    const float* ml = plan.ml + 2 * (size_t)kh * head.at.cap;
    const float* sums = plan.acc + (size_t)kh * head.at.cap * kDim + d;
    for (int e = e0; e < head.merges; e += es) {
        if (e != e0) j = load_line(units + e);
        // this half wave's column, and its first part
        const int half = 2 * wave + h, step = j.lanes / 32;
        const int c = j.lanes == 32 ? half : 0, first = half & (step - 1);
        const int parts = c < j.many ? j.pparts + j.parts : 0;
        float m = -INFINITY, l = 0.0f;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i0 = first; i0 < parts; i0 += 8 * step) {
            f32x4 y[8];
            f32x2 w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int i = min(i0 + k * step, parts - 1);
                const int p = c + (i < j.pparts ? j.pbase + i * j.pcols : j.base + (i - j.pparts) * j.cols);
                w[k] = *reinterpret_cast<const f32x2*>(ml + 2 * (size_t)p);
                y[k] = *reinterpret_cast<const f32x4*>(sums + (size_t)p * kDim);
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, w[k][0]);
            const float before = part_weight(m, top);
            l *= before;
            x *= before;
            m = top;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (i0 + k * step >= parts) break;
                // (a part without a key holds zeros, and a sum that is 0 or NaN)
                const float f = part_weight(w[k][0], m);
                l = fmaf(w[k][1], f, l);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = fmaf(y[k][r], f, x[r]);
            }
        }
        if (j.lanes > 32) {  // the halves, and the waves
            const float top = max_h(m), f = part_weight(m, top);
            l = sum_h(l * f);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = sum_h(x[r] * f);
            m = top;
            if (h == 0) *reinterpret_cast<f32x4*>(&s_x[wave][d]) = x;
            if (lane == 0) s_ml[wave] = f32x2{m, l};
            __syncthreads();
            m = s_ml[0][0];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_ml[w][0]);
            l = 0.0f;
            x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = part_weight(s_ml[w][0], m);
                l = fmaf(s_ml[w][1], f, l);
                const f32x4 y = *reinterpret_cast<const f32x4*>(&s_x[w][d]);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = fmaf(y[r], f, x[r]);
            }
            __syncthreads();  // the LDS is free for the next unit
        }
        if (c < j.many && first == 0) {
            const int col = j.col0 + c, local = col / a.per_row;
            const size_t o = ((size_t)(j.row0 + local) * a.hq + kh * a.per_row + col - local * a.per_row) * kDim + d;
            if (a.o_f16) write_o<true>(a.o, o, x, 1.0f / l);
            else write_o<false>(a.o, o, x, 1.0f / l);
        }
    }
}

}  // namespace

size_t attend_workspace_len(int n, int groups, int tokens, int hq, int hkv) {
    return layout(n, groups, tokens, hq, hkv).bytes;
}

int attend_plan_launch(const int* cu, const int* pos, const int* group, const int* prefix, int groups, int n,
                       int width, int tokens, int hq, int hkv, void* ws, hipStream_t stream) {
    const Layout l = layout(n, groups, tokens, hq, hkv);
    uint8_t* w = static_cast<uint8_t*>(ws);
    PlanArgs a = {};
    a.head = reinterpret_cast<Header*>(w);
    a.start = reinterpret_cast<Tile*>(w + l.starts);
    a.tile = reinterpret_cast<Tile*>(w + l.tiles);
    a.merge = reinterpret_cast<Join*>(w + l.merges);
    a.seq = reinterpret_cast<PlanSeq*>(w + l.seqs);
    a.first = reinterpret_cast<int*>(w + l.first);
    a.grp = reinterpret_cast<PlanGroup*>(w + l.group);
    a.rows = reinterpret_cast<int*>(w + l.rows);
    a.n = n;
    a.groups = groups;
    a.width = width;
    a.tokens = tokens;
    a.hq = hq;
    a.hkv = hkv;
    a.per_row = hq / hkv;
    a.runs = l.runs;
    a.at = l;
    const bool few = n <= kPlanFew && groups <= kPlanFew && l.max_tiles <= kPlanFew;
    auto kernel = few                                       ? attend_plan_kernel<true, kPlanFew>
                  : n <= kPlanLds && groups <= kPlanLds ? attend_plan_kernel<true, kScanThreads>
                                                        : attend_plan_kernel<false, kScanThreads>;
    hipLaunchKernelGGL(kernel, dim3(1), dim3(few ? kPlanFew : kScanThreads), 0, stream, cu, pos, group, prefix, n,
                       groups, a);
    return check_launch("attend_plan_kernel");
}

int attend_launch(const float* q, const PoolArgs& pool, const int* table, int width, int n, int tokens,
                  void* ws, size_t ws_len, void* o, int o_f16, int exact, int hq, hipStream_t stream) {
    const Layout l = layout(n, n, tokens, hq, pool.hkv);  // (the most entries: the plan's may have fewer groups)
    AttendArgs a = {};
    a.ws = static_cast<uint8_t*>(ws);
    a.ws_len = ws_len;
    a.q = q;
    a.p = pool;
    a.table = table;
    a.o = o;
    a.n = n;
    a.width = width;
    a.tokens = tokens;
    a.hq = hq;
    a.per_row = hq / pool.hkv;
    a.o_f16 = o_f16;
    auto kernel = !o_f16 ? attend_kernel<true, false> : exact ? attend_kernel<true, true> : attend_kernel<false, true>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((l.runs + kWaves - 1) / kWaves * pool.hkv)), dim3(kThreads), 0, stream,
                       a.ws, pool.hkv, l.runs, a);
    const int st = check_launch("attend_kernel");
    if (st != BRASA_OK) return st;
    // a workgroup for each unit of a KV head, up to eight per CU
    const int wgs = std::max(std::min(l.max_merges, 2048 / pool.hkv), 1);
    hipLaunchKernelGGL(attend_merge_kernel, dim3((unsigned)(wgs * pool.hkv)), dim3(kThreads), 0, stream, a.ws,
                       pool.hkv, l.runs, a);
    return check_launch("attend_merge_kernel");
}

}  // namespace brasa
