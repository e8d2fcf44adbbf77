// The maps of a step's packed rows, built on the device from its requests' lengths, and the pages that
// groups of sequences share.
//
// cu[i] = sum of add[j], j < i; row t of sequence i (cu[i] <= t < cu[i + 1]) stands at position
// len[i] + t - cu[i], in slot table[i][position / 64] * 64 + position % 64. Whole numbers throughout.
//
// Bound: latency (a launch, the lengths, a scan, the table's entries): 64 sequences of one row take 3.1 us, a
// thousand with 72K rows 5.3 (16 bytes a row). The pages that two groups of 32 share 6.2 us.
#include <climits>

#include "paged.hpp"

namespace brasa {
namespace {

// a + b up to a cap, for a, b in [0, 2^30], whose sum may be 2^31: associative, so scans may group the terms at will
__device__ __forceinline__ int add_cap(int a, int b, int cap) { return (int)min((unsigned)a + (unsigned)b, (unsigned)cap); }

struct RowsArgs {
    const int* add;
    const int* len;
    const int* table;
    int* cu;
    int* lk;
    int* seq;
    int* pos;
    int* slot;
    int n, width, pages, tokens;
    int per;  // sequences of a thread
};

__device__ __forceinline__ int added(const RowsArgs& a, int i) {
    return a.len[i] < 0 ? 0 : min(max(a.add[i], 0), a.tokens);
}

// Every workgroup scans all sequences' counts (thread i those from i * per on), finds the sequence of
// each of its rows in the scan, and writes its share of cu and lk.
__global__ void __launch_bounds__(kScanThreads)
kv_rows_kernel(RowsArgs a) {
    __shared__ int s_first[kScanThreads];  // first row of each thread's sequences
    __shared__ int s_wave[kScanWaves];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i0 = min((int)threadIdx.x * a.per, a.n), i1 = min(i0 + a.per, a.n);
    int mine = 0;
    for (int i = i0; i < i1; ++i) mine = add_cap(mine, added(a, i), a.tokens);
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int x = __shfl_up(incl, d);
        if (lane >= d) incl = add_cap(incl, x, a.tokens);
    }
    int excl = __shfl_up(incl, 1);
    if (lane == 0) excl = 0;
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w) before = add_cap(before, s_wave[w], a.tokens);
    const int first = add_cap(before, excl, a.tokens);
    s_first[threadIdx.x] = first;
    if (threadIdx.x % gridDim.x == blockIdx.x) {
        int at = first;
        for (int i = i0; i < i1; ++i) {
            const int next = add_cap(at, added(a, i), a.tokens);
            if (a.cu) a.cu[i] = at;
            if (a.lk) a.lk[i] = (int)min((long long)max(a.len[i], 0) + next - at, (long long)INT_MAX);
            at = next;
            if (a.cu && i == a.n - 1) a.cu[a.n] = at;
        }
    }
    if (!a.seq && !a.pos && !a.slot) return;
    __syncthreads();
    for (long long t0 = (long long)blockIdx.x * kScanThreads; t0 < a.tokens; t0 += (long long)gridDim.x * kScanThreads) {
        const long long tt = t0 + threadIdx.x;
        if (tt >= a.tokens) break;
        const int t = (int)tt;
        // the last thread whose first row is at or before t; of several, the last: the others have no rows
        int lo = 0;
#pragma unroll
        for (int step = kScanThreads / 2; step; step /= 2)
            if (s_first[lo + step] <= t) lo += step;
        int seq = lo * a.per, at = s_first[lo];
        const int end = min(seq + a.per, a.n);
        while (seq < end) {
            const int rows = added(a, seq);
            if (t - at < rows) break;
            at += rows;  // (at most t)
            ++seq;
        }
        int pos = -1, slot = -1;
        if (seq < end) {
            pos = (int)min((long long)a.len[seq] + t - at, (long long)INT_MAX);
            if (pos < a.width * kPage) {
                const int page = a.table[(size_t)seq * a.width + pos / kPage];
                if (page >= 0 && page < a.pages) slot = page * kPage + pos % kPage;
            }
        } else {
            seq = -1;
        }
        if (a.seq) a.seq[t] = seq;
        if (a.pos) a.pos[t] = pos;
        if (a.slot) a.slot[t] = slot;
    }
}

// ---- shared pages -------------------------------------------------------------------------------
struct SharedArgs {
    const int* table;
    const int* len;
    const int* group;
    int* prefix;
    int n, width, pages;
};

// A workgroup per group: the first row with positions leads; the others' entries are compared with its, four
// rows a wave, 256 entries at a time, up to the least difference found so far. Bound: the chain group ->
// lengths -> entries.
constexpr int kRowsAtOnce = 4;
__global__ void __launch_bounds__(kScanThreads)
kv_pages_shared_kernel(SharedArgs a) {
    __shared__ int s_lead, s_live, s_run;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = blockIdx.x;
    const int r0 = min(max(a.group[g], 0), a.n), r1 = min(max(a.group[g + 1], r0), a.n);
    if (threadIdx.x == 0) {
        s_lead = a.n;
        s_live = 0;
        s_run = a.width;
    }
    __syncthreads();
    int lead = a.n, live = 0, run = a.width;
    for (int i = r0 + (int)threadIdx.x; i < r1; i += kScanThreads) {
        const int len = a.len[i];
        if (len <= 0) continue;
        lead = min(lead, i);
        ++live;
        run = min(run, len / kPage);
    }
    if (live) {
        atomicMin(&s_lead, lead);
        atomicAdd(&s_live, live);
        atomicMin(&s_run, run);
    }
    __syncthreads();
    lead = s_lead;
    live = s_live;
    if (live > 1) {
        const int* want = a.table + (size_t)lead * a.width;
        for (int i0 = r0 + wave; i0 < r1; i0 += kRowsAtOnce * kScanWaves) {
            int len[kRowsAtOnce];
            const int* row[kRowsAtOnce];
#pragma unroll
            for (int r = 0; r < kRowsAtOnce; ++r) {
                const int i = min(i0 + r * kScanWaves, r1 - 1);  // (the last once more is no other answer)
                len[r] = a.len[i];
                row[r] = a.table + (size_t)i * a.width;
            }
            // (another wave's lower bound is only a shorter way: the least of all is the same)
            for (int c0 = 0; c0 < *(volatile int*)&s_run; c0 += 256) {
                int x[4], y[kRowsAtOnce][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = min(c0 + 64 * j + lane, a.width - 1);
                    x[j] = want[c];
#pragma unroll
                    for (int r = 0; r < kRowsAtOnce; ++r) y[r][j] = row[r][c];
                }
                int at = a.width;
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    bool other = x[j] < 0 || x[j] >= a.pages;
#pragma unroll
                    for (int r = 0; r < kRowsAtOnce; ++r) other |= len[r] > 0 && x[j] != y[r][j];
                    const uint64_t others = __builtin_amdgcn_ballot_w64(other);
                    if (others) at = c0 + 64 * j + __builtin_ctzll(others);
                }
                if (at < a.width) {
                    if (lane == 0) atomicMin(&s_run, at);
                    break;
                }
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) a.prefix[g] = live > 1 ? s_run * kPage : 0;
}

}  // namespace

int kv_rows_launch(const int* add, const int* len, const int* table, int* cu, int* lk, int* seq, int* pos,
                   int* slot, int n, int width, int pages, int tokens, hipStream_t stream) {
    RowsArgs a{add, len, table, cu, lk, seq, pos, slot, n, width, pages, tokens,
               (n + kScanThreads - 1) / kScanThreads};
    // one workgroup for each 1024 rows up to one per CU: every one of them scans the lengths
    const int grid = std::min(std::max((tokens + kScanThreads - 1) / kScanThreads, 1), 256);
    hipLaunchKernelGGL(kv_rows_kernel, dim3(grid), dim3(kScanThreads), 0, stream, a);
    return check_launch("kv_rows_kernel");
}

int kv_pages_shared_launch(const int* table, const int* len, const int* group, int groups, int* prefix, int n,
                           int width, int pages, hipStream_t stream) {
    SharedArgs a{table, len, group, prefix, n, width, pages};
    hipLaunchKernelGGL(kv_pages_shared_kernel, dim3(groups), dim3(kScanThreads), 0, stream, a);
    return check_launch("kv_pages_shared_kernel");
}

}  // namespace brasa
