// The 8-bit paged KV cache: its writer and the decode attention that reads it.
#include "paged.hpp"

namespace brasa {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));

// ---- store ------------------------------------------------------------------------------------
//
// Row t of the packed new rows belongs to sequence i with cu[i] <= t < cu[i + 1] and goes to
// position pos[i] + t - cu[i]. A block (page) and head is written by one workgroup, K and V by one
// each: it holds the block's new rows in registers, takes their largest magnitude, the scale
// from it (and from the block's scale, where earlier rows of the block stay), rounds those
// earlier rows to a larger scale, and writes the codes.
//
// Bound: HBM at 4 bytes in and 1 out a value for prompts (7K rows of 8 heads 14.2 us, 5.1 TB/s); a
// decode step's few rows are bound by the chain cu / pos -> page id -> scale -> codes (64 sequences
// 4.9 us in the kernel, 7.8 from call to call).
constexpr int kStoreThreads = 256;

struct StoreArgs {
    PoolArgs p;  // of one layer
    const float* k;
    const float* v;
    const int* cu;
    const int* pos;
    const int* table;
    int n, width, tokens;
    int item0;  // first item of the launch
};

// the blocks that sequence i's new rows touch: [first, first + count)
__device__ __forceinline__ int touched_blocks(const StoreArgs& a, int i, int& c0, int& c1, int& pos) {
    c0 = min(max(a.cu[i], 0), a.tokens);
    c1 = min(max(a.cu[i + 1], c0), a.tokens);
    pos = a.pos[i];
    // (a negative position, or one past what the table can hold, has no block)
    if (c1 == c0 || pos < 0 || pos >= a.width * kPage) return 0;
    return min((pos + (c1 - c0) - 1) / kPage, a.width - 1) - pos / kPage + 1;
}

__global__ void __launch_bounds__(kStoreThreads)
store_paged_kernel(StoreArgs a) {
    const int lane = threadIdx.x & 63;
    const int item = a.item0 + blockIdx.x / a.p.hkv, kh = blockIdx.x % a.p.hkv;
    const bool is_v = blockIdx.y;

    // the sequence and block of this item: every wave walks the sequences' block counts, 64 at a
    // time
    int seq = -1, before = 0;
    for (int i0 = 0; i0 < a.n; i0 += 64) {
        int c0, c1, pos, nb = 0;
        if (i0 + lane < a.n) nb = touched_blocks(a, i0 + lane, c0, c1, pos);
        const int incl = wave_scan(nb) + before;
        const unsigned long long past = __builtin_amdgcn_ballot_w64(incl > item);
        if (past) {
            const int l = __builtin_ctzll(past);
            seq = i0 + l;
            before = __shfl(incl - nb, l);
            break;
        }
        before = __shfl(incl, 63);
    }
    if (seq < 0) return;  // the grid's bound is loose
    seq = __builtin_amdgcn_readfirstlane(seq);
    int c0, c1, pos;
    touched_blocks(a, seq, c0, c1, pos);
    const int block = pos / kPage + item - before;
    const int page = a.table[(size_t)seq * a.width + block];
    if (page < 0 || page >= a.p.pages) return;
    // slots [s0, s1) of the block are new, [0, s0) hold earlier rows
    const int s0 = max(pos - block * kPage, 0);
    const int s1 = min(pos + (c1 - c0) - block * kPage, kPage);
    const size_t tile = (size_t)page * a.p.hkv + kh;
    uint8_t* codes = (is_v ? a.p.v : a.p.k) + tile * kTileBytes8;
    uint8_t* scale = (is_v ? a.p.vx : a.p.kx) + tile;
    const int row0 = c0 + block * kPage - pos;  // the packed row of slot 0
    const float* src = (is_v ? a.v : a.k) + kh * kDim + 4 * (threadIdx.x & 31);

    const int old = s0 > 0 ? *scale : 0;
    f32x4 x[8];
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int s = 8 * j + (threadIdx.x >> 5);
        x[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (s >= s0 && s < s1)
            x[j] = *reinterpret_cast<const f32x4*>(src + (size_t)(row0 + s) * a.p.hkv * kDim);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float m = fabsf(x[j][e]);
            amax = fmaxf(amax, m < INFINITY ? m : 0.0f);  // NaN and inf take no part in the scale
        }
    __shared__ float s_max[kStoreThreads / 64];
#pragma unroll
    for (int d = 32; d; d /= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
    if (lane == 0) s_max[threadIdx.x >> 6] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStoreThreads / 64; ++w) amax = fmaxf(amax, s_max[w]);
    const int ex = max(e4m3_scale(amax), old);

    if (s0 > 0 && ex > old) {
        // the earlier rows, rounded to the larger scale (exact but where they leave e4m3's normal
        // range)
        for (int i = threadIdx.x; i < s0 * (kDim / 4); i += kStoreThreads) {
            uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
            const uint32_t c = *w;
            float y[4];
            y[0] = __builtin_amdgcn_cvt_f32_fp8(c, 0);
            y[1] = __builtin_amdgcn_cvt_f32_fp8(c, 1);
            y[2] = __builtin_amdgcn_cvt_f32_fp8(c, 2);
            y[3] = __builtin_amdgcn_cvt_f32_fp8(c, 3);
#pragma unroll
            for (int e = 0; e < 4; ++e)  // (a NaN code keeps its sign too)
                if ((c >> 8 * e & 0x7fu) == 0x7fu) y[e] = __uint_as_float(0x7fc00000u | (c >> 8 * e << 24 & 0x80000000u));
            *w = e4m3_quad(y, old - ex);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int s = 8 * j + (threadIdx.x >> 5);
        if (s >= s0 && s < s1) {
            const float y[4] = {x[j][0], x[j][1], x[j][2], x[j][3]};
            reinterpret_cast<uint32_t*>(codes)[s * (kDim / 4) + (threadIdx.x & 31)] = e4m3_quad(y, 127 - ex);
        }
    }
    // (every thread that needed the old scale has read it before the barrier above)
    if (threadIdx.x == 0) *scale = (uint8_t)ex;
}

// ---- decode -----------------------------------------------------------------------------------
//
// o[i, h] = sum_j p_j v_j / sum_j p_j over the lk[i] keys of sequence i, p_j = exp(q . k_j / sqrt(128)).
//
// Bound: where a launch has a few pages for every wave, the loads of its 256 bytes of codes per (key, KV
// head): 5.0 TB/s, of 6.05 that the f16 decode of a ragged batch reads at. The vector units are 23 % busy
// then and the matrix cores 6 %; waves wait for data 35 % and to issue 45 % of their time. Else the
// chain lengths -> page ids -> codes -> merge. The pages of all sequences stand in
// one line, and workgroup w of a head takes the w-th equal run of them, so every CU reads the same
// number whatever the lengths, which only the device knows. A run's pieces of one sequence are its
// segments; a segment that is not the whole sequence leaves (m, l, sums) in the workspace, and
// the last workgroup of a sequence to arrive merges them in order (a fixed order: the result does
// not depend on who arrives last). A few sequences are cut into parts of their own instead, one
// a workgroup, and short ones are left whole.
//
// A wave takes every kWaves-th page of a segment, all of it in registers, the next page's codes loaded as
// soon as this one's are used. S^T = K Q^T on 16x16x32 f16 MFMAs: K's codes are converted exactly (an
// e4m3 value is an f16 value) right from the loaded 16-byte pieces; columns 0 .. 7 hold the f16 hi
// halves of the heads' q, columns 15 .. 8 the lo halves (22 bits together), so one MFMA does both
// and a mirrored addition joins them. Both lanes of a head then hold its scores of four keys of each 16,
// which is the layout P^T needs for O^T = V^T P^T, again hi halves in one lane and lo halves in the other.
// V's operand needs eight keys of one dim in a lane: the lane loads 8 bytes of each of its eight
// keys' rows (dims 8 i .. 8 i + 7 of lane row i) and byte permutes pair the keys before the
// conversion, so neither K nor V goes through LDS. The blocks' scales are exponents: K's is
// folded into the exponential's argument, V's multiplies the page's sum.
//
// Measured at 32 heads over 8: one sequence of 257 keys 8.0 us, 4096 13.1, 16384 15.5 (a layer of
// many, 2.2 TB/s), 32768 23.3 (2.9); 64 sequences of 300 to 16000 111 us (5.0 TB/s); 200 of 300 to 1000
// 63 us (3.8). A group of 16 heads reads its pages once for each 8: 128 heads over 8 take 23.0 us at
// 16384 and 186 us for the batch (64 over 8: 17.9 and 115). Where the 15 us at 16384 go: 2 until a wave's
// first page is asked for, 7 for the codes (32 workgroups of 8 pages a head), 1.5 for the waves' sums, parts
// and arrivals, 4 for the last workgroup's merge, whose one CU has 64 KB of parts to fetch. Two workgroups
// per CU, 256 registers a wave: with 256 or 1024 workgroups in place of 512 the batch takes 123 and 120
// us in place of 111, with 256 of eight waves 116 (which take 32768 keys in 21.5 us, 16384 in 15.4). Runs
// of 12 or 16 pages in place of kMinPages = 8 take 16384 keys in 16.5 and 18.7 us, 4096 in 15.1 and 17.9,
// 32768 in 25.3 and 21.8.
constexpr int kWaves = 4;
constexpr int kDecThreads = 64 * kWaves;
constexpr int kMaxCols = 8;      // query heads of a workgroup
constexpr int kSlots = 512;      // workgroups of a launch: two per CU
constexpr int kMinPages = 8;     // pages of a run that may split a sequence (two per wave)
constexpr int kWholePages = 12;  // pages of a sequence that is not worth splitting
constexpr int kPartBytes = kMaxCols * (kDim + 2) * 4;  // a part: (m, l) of each column, then its sums
constexpr int kCounterStride = 16;  // words between two arrival counters

struct DecodePagedArgs {
    const float* q;
    PoolArgs p;  // of one layer
    const int* table;
    const int* lk;
    void* o;
    float* part;
    unsigned* ctr;
    int n, width, hq, group, runs, o_f16, part_bytes;
};

__device__ __forceinline__ f32x4 mfma16(half8v a, half8v b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// 4 codes -> 4 f16 values, exact
__device__ __forceinline__ half2v f16_of_lo(uint32_t w) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}
__device__ __forceinline__ half2v f16_of_hi(uint32_t w) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
}
__device__ __forceinline__ half8v join(half2v a, half2v b, half2v c, half2v d) {
    return half8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// This lane's half of x = hi + lo (up to 2^-22 of x): hi where less = 0, lo where it is -1.
__device__ __forceinline__ half2v half_of(float x, float y, float less) {
    x = as_f32(x);
    y = as_f32(y);
    const half2v hi = {(_Float16)x, (_Float16)y};
    return half2v{(_Float16)fmaf((float)hi.x, less, x), (_Float16)fmaf((float)hi.y, less, y)};
}
// x plus that of column 15 - c: the same bits in both. (as_f32 keeps the addition here, where
// row_mirror folds into it; sunk into a later block it would leave its move behind.)
__device__ __forceinline__ float add_mirror(float x) {
    return as_f32(x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xF, 0xF, true)));
}
// over the four lanes c, c + 16, c + 32, c + 48 of a column
__device__ __forceinline__ float max_u(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    x = fmaxf(__int_as_float(a[0]), __int_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ __forceinline__ float sum_u(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    x = __int_as_float(a[0]) + __int_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return __int_as_float(b[0]) + __int_as_float(b[1]);
}
// pages of a sequence of lk keys in the line of pages: at least one, so that a sequence without
// keys has a workgroup that writes its zeros, and a length the table cannot hold one that
// writes its NaN
__device__ __forceinline__ int line_pages(int lk, int width) {
    return lk <= 0 || lk > width * kPage ? 1 : (lk + kPage - 1) / kPage;
}
// Parts cross XCDs: stores written through, loads past the L2 (sc1; the arrival counter orders
// them), through a buffer descriptor of the workspace's parts and byte offsets into it.
constexpr int kSc1 = 16;
typedef __amdgpu_buffer_rsrc_t Parts;
__device__ __forceinline__ void st_part(Parts p, int at, f32x4 x) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), p, at, 0, kSc1);
}
__device__ __forceinline__ void st_part2(Parts p, int at, float x, float y) {
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(x), __float_as_uint(y)}, p, at, 0, kSc1);
}
__device__ __forceinline__ f32x4 ld_part(Parts p, int at) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(p, at, 0, kSc1));
}
__device__ __forceinline__ f32x2 ld_part2(Parts p, int at) {
    return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(p, at, 0, kSc1));
}

// weight of a part whose largest score is m in a sum whose largest is top (a part without a key has
// m = -inf)
__device__ __forceinline__ float part_weight(float m, float top) {
    return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

// x / l of four dims (no key: l = 0 and zeros; a NaN l stays one)
__device__ __forceinline__ void write_o(const DecodePagedArgs& a, size_t at, f32x4 x, float l) {
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = l == 0.0f ? 0.0f : x[e] / l;
    if (a.o_f16) {
        u32x2 w = {f2h(y[0]) | (uint32_t)f2h(y[1]) << 16, f2h(y[2]) | (uint32_t)f2h(y[3]) << 16};
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.o) + at) = w;
    } else {
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.o) + at) = y;
    }
}

// A wave's page in registers: 8 KB each of K and V.
struct PageK {
    u32x4 w[4][2];  // key 16 T + c, bytes 64 hh + 16 u .. + 16
    int x;          // scale byte
};
struct PageV {
    u32x2 w[4][4];  // key 16 T + 4 u + r, bytes 8 c .. + 8
    int x;
};

__global__ void __launch_bounds__(kDecThreads, 2)
decode_paged_kernel(DecodePagedArgs a) {
    __shared__ __attribute__((aligned(16))) float s_acc[kWaves][kMaxCols][kDim];  // or the parts' weights
    __shared__ __attribute__((aligned(16))) f32x4 s_sum[kDecThreads];
    __shared__ float s_m[kWaves][kMaxCols], s_l[kWaves][kMaxCols];
    __shared__ unsigned s_last;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, u = lane >> 4;
    const float less = c < kMaxCols ? 0.0f : -1.0f;  // columns of hi halves, then of lo halves
    const int kh = blockIdx.x % a.p.hkv, run = blockIdx.x / a.p.hkv;
    const int h0 = kh * a.group + blockIdx.y * kMaxCols;          // first query head
    const int cols = min(a.group - (int)blockIdx.y * kMaxCols, kMaxCols);
    const int head_of_lane = h0 + min(c < kMaxCols ? c : 15 - c, cols - 1);

    // ---- this workgroup's run of the line of pages -------------------------------------------
    const int lk0 = lane < a.n ? a.lk[lane] : 0;
    const int np0 = lane < a.n ? line_pages(lk0, a.width) : 0;
    const int incl0 = wave_scan(np0);
    int total = __builtin_amdgcn_readlane(incl0, 63);
    bool lengthy = __builtin_amdgcn_ballot_w64(np0 > kWholePages);  // a sequence worth splitting
    if (a.n > 64) {
        int more = 0, most = 0;
        for (int i = 64 + lane; i < a.n; i += 64) {
            const int np = line_pages(a.lk[i], a.width);
            more += np;
            most = max(most, np);
        }
        total += __builtin_amdgcn_readlane(wave_scan(more), 63);
        lengthy |= (bool)__builtin_amdgcn_ballot_w64(most > kWholePages);
    }
    // Few pages, in sequences of few: a run takes the sequences that start in it, whole (128 sequences of
    // 100 keys 19.0 us cut into runs of kMinPages, 13.7 in runs of 4).
    const bool whole_only = total <= a.runs * kMinPages && !lengthy;
    const int size = max((total + a.runs - 1) / a.runs, whole_only ? (total + a.n - 1) / a.n : kMinPages);
    // Few sequences: each is cut into parts of its own, `cut` pages or a little less, and a run is one
    // part; the line is one of parts. With more of them that would leave runs idle or uneven.
    int cut = 0, incl1 = incl0, np1 = np0;
    if (!whole_only && a.n <= 64 && a.n <= a.runs / 4) {
        cut = size;
        while (true) {
            np1 = (np0 + cut - 1) / cut;
            incl1 = wave_scan(np1);
            total = __builtin_amdgcn_readlane(incl1, 63);
            if (total <= a.runs) break;
            cut += (cut + 7) / 8;  // (every sequence whole is n <= runs parts)
        }
    }
    const int run_size = cut ? 1 : size;
    int at = run * run_size;
    const int end = min(at + run_size, total);
    if (at >= end) return;
    int seq = 0, seq_at = 0;  // the sequence that holds page (or part) `at`, and its first in the line
    for (int i0 = 0; i0 < a.n; i0 += 64) {
        const int np = i0 == 0 ? np1 : i0 + lane < a.n ? line_pages(a.lk[i0 + lane], a.width) : 0;
        const int incl = (i0 == 0 ? incl1 : wave_scan(np)) + seq_at;
        const unsigned long long past = __builtin_amdgcn_ballot_w64(incl > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            seq = i0 + l;
            seq_at = __builtin_amdgcn_readlane(incl - np, l);
            break;
        }
        seq_at = __builtin_amdgcn_readlane(incl, 63);
    }
    auto keys_of = [&](int i) { return i < 64 ? __builtin_amdgcn_readlane(lk0, i) : a.lk[i]; };
    if (whole_only && seq_at < at) {  // that one is the run's before
        seq_at += line_pages(keys_of(seq), a.width);
        ++seq;
        at = seq_at;
        if (at >= end) return;
    }

    // ---- a segment: pages [b0, b1) of a sequence of np --------------------------------------------
    struct Segment {
        int seq, np, lk, b0, b1, blast;
        bool whole, bad;  // bad: a length or page that is not there, the output is NaN
    };
    auto segment = [&](int seq, int seq_at, int at) {
        Segment g;
        const int lk = keys_of(seq);
        const bool bad_len = lk < 0 || lk > a.width * kPage;
        g.seq = seq;
        g.np = line_pages(lk, a.width);
        g.lk = bad_len ? 0 : lk;
        if (cut) {  // part at - seq_at of the sequence's, as equal as they can be
            const int parts = __builtin_amdgcn_readlane(np1, seq), i = at - seq_at;
            const int each = g.np / parts, more = g.np - each * parts;
            g.b0 = i * each + min(i, more);
            g.b1 = g.b0 + each + (i < more ? 1 : 0);
        } else {
            g.b0 = at - seq_at;
            g.b1 = whole_only ? g.np : min(end - seq_at, g.np);
        }
        g.blast = g.lk > 0 ? g.b1 : 0;  // no keys: no pages
        g.whole = g.b0 == 0 && g.b1 == g.np;
        g.bad = bad_len;
        return g;
    };
    PageK k;
    PageV v;
    f32x4 qraw[4][2];
    int next_id = 0;  // the next page's id, loaded a page ahead of its codes
    // a page that is not there reads page 0 in its place
    auto tile_of = [&](int page, bool& bad) {
        const bool there = page >= 0 && page < a.p.pages;
        bad |= !there;
        return (size_t)(there ? page : 0) * a.p.hkv + kh;
    };
    auto load_k = [&](size_t tile) {
        const uint8_t* p = a.p.k + tile * kTileBytes8 + c * kDim + 16 * u;
#pragma unroll
        for (int T = 0; T < 4; ++T)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
                k.w[T][hh] = *reinterpret_cast<const u32x4*>(p + 16 * T * kDim + 64 * hh);
        k.x = a.p.kx[tile];
    };
    auto load_v = [&](size_t tile) {
        const uint8_t* p = a.p.v + tile * kTileBytes8 + 4 * u * kDim + 8 * c;
#pragma unroll
        for (int T = 0; T < 4; ++T)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                v.w[T][r] = *reinterpret_cast<const u32x2*>(p + (16 * T + r) * kDim);
        v.x = a.p.vx[tile];
    };
    // Q and this wave's first page on their way, Q ahead: it would wait behind the page.
    // k-step t = 2 hh + j holds dims 64 hh + 16 u + 8 j .. + 8, as K's 16-byte loads do
    auto begin = [&](Segment& g, const int* ids) {
        const int b = g.b0 + wave;
        int id = 0;
        if (b < g.blast) {
            id = ids[b];
            if (b + kWaves < g.blast) next_id = ids[b + kWaves];
        }
        const float* qrow = a.q + ((size_t)g.seq * a.hq + head_of_lane) * kDim + 16 * u;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                qraw[t][e] = *reinterpret_cast<const f32x4*>(qrow + 64 * (t >> 1) + 8 * (t & 1) + 4 * e);
        __builtin_amdgcn_sched_barrier(0);
        if (b < g.blast) {
            const size_t tile = tile_of(id, g.bad);
            load_k(tile);
            load_v(tile);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    while (true) {
        Segment g = segment(seq, seq_at, at);
        const int* ids = a.table + (size_t)g.seq * a.width;
        const int lk = g.lk, blast = g.blast;
        begin(g, ids);

        // ---- Q: this lane's halves of q / sqrt(128) * log2 e, its exponent taken out -------------
        half8v q[4];
        int qx;
        {
            const float scale = 0.08838834764831845f * kLog2e;
            float x[4][8];
            float qmax = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[t][e] = as_f32(qraw[t][e >> 2][e & 3] * scale);
                    qmax = fmaxf(qmax, fabsf(x[t][e]));
                }
            qmax = max_u(qmax);
            qx = (int)(__float_as_uint(qmax) >> 23) - 127 - 8;  // the row's largest to [2^8, 2^9)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                half2v h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    h[e] = half_of(ldexpf(x[t][2 * e], -qx), ldexpf(x[t][2 * e + 1], -qx), less);
                q[t] = join(h[0], h[1], h[2], h[3]);
            }
        }

        float m_used = -INFINITY, lsum = 0.0f;
        f32x4 acc[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

        size_t next = 0;
        for (int b = g.b0 + wave; b < blast; b += kWaves) {
            const bool more = b + kWaves < blast;
            // ---- scores: key 16 T + 4 u + r of head c, in units of log2 ---------------------------
            f32x4 s[4];
#pragma unroll
            for (int T = 0; T < 4; ++T) {
                s[T] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t w0 = k.w[T][t >> 1][2 * (t & 1)], w1 = k.w[T][t >> 1][2 * (t & 1) + 1];
                    const half8v ka = join(f16_of_lo(w0), f16_of_hi(w0), f16_of_lo(w1), f16_of_hi(w1));
                    s[T] = mfma16(ka, q[t], s[T]);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) s[T][r] = add_mirror(s[T][r]);  // q's hi + lo halves
            }
            // 2^sx times the products of the codes and the scaled q. (Past the clamp every score is
            // 0, or so far from the next that one key takes all.)
            const float sc = ldexpf(1.0f, min(max(qx + k.x - 127, -127), 127));
            // the next page's K takes this one's registers, its V later V's: a wave always has a
            // load on its way
            __builtin_amdgcn_sched_barrier(0);
            if (more) {
                next = tile_of(next_id, g.bad);
                load_k(next);
            }
            __builtin_amdgcn_sched_barrier(0);
            const int left = lk - b * kPage;  // live keys of the page
            if (left < kPage) {  // the codes behind the last key may be anything, NaN too
#pragma unroll
                for (int T = 0; T < 4; ++T)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool live = 16 * T + 4 * u + r < left;
                        s[T][r] = live ? s[T][r] : -INFINITY;
                        v.w[T][r] = live ? v.w[T][r] : u32x2{0, 0};
                    }
            }
            float tmax = -INFINITY;
#pragma unroll
            for (int T = 0; T < 4; ++T)
#pragma unroll
                for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, s[T][r]);
            tmax = max_u(tmax) * sc;
            // a reference point that moves only when the maximum has grown by 2^8: p stays below
            // 2^15 with the bias of 2^7 that keeps the lo halves of small p out of f16's subnormals
            const bool grow = tmax > m_used + 8.0f;
            if (__builtin_amdgcn_ballot_w64(grow)) {
                const float alpha = grow ? __builtin_amdgcn_exp2f(m_used - tmax) : 1.0f;
                if (grow) m_used = tmax;
                lsum *= alpha;
#pragma unroll
                for (int t = 0; t < 8; ++t) acc[t] *= alpha;
            }
            half8v p[2];
            const float mb = 7.0f - m_used;
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                half2v h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int T = 2 * st + (e >> 1), r = 2 * (e & 1);
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[T][r], sc, mb));
                    const float p1 = __builtin_amdgcn_exp2f(fmaf(s[T][r + 1], sc, mb));
                    lsum += p0 + p1;
                    h[e] = half_of(p0, p1, less);
                }
                p[st] = join(h[0], h[1], h[2], h[3]);
            }
            const float vs = ldexpf(1.0f, v.x - 127);
            // ---- O^T += V^T P^T: tile t's rows are dims 8 i + t ------------------------------------
#pragma unroll
            for (int t2 = 0; t2 < 4; ++t2) {  // tiles 2 t2, 2 t2 + 1
                f32x4 pv[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
                const int d = t2 >> 1;
                const uint32_t by = 2 * (t2 & 1);
                const uint32_t sel = by | (4 + by) << 8 | (by + 1) << 16 | (5 + by) << 24;
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    half2v x0[4], x1[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int T = 2 * st + (e >> 1), r = 2 * (e & 1);
                        const uint32_t w = __builtin_amdgcn_perm(v.w[T][r + 1][d], v.w[T][r][d], sel);
                        x0[e] = f16_of_lo(w);
                        x1[e] = f16_of_hi(w);
                    }
                    const half8v v0 = join(x0[0], x0[1], x0[2], x0[3]);
                    const half8v v1 = join(x1[0], x1[1], x1[2], x1[3]);
                    pv[0] = mfma16(v0, p[st], pv[0]);
                    pv[1] = mfma16(v1, p[st], pv[1]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[2 * t2 + j][r] = fmaf(pv[j][r], vs, acc[2 * t2 + j][r]);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (more) {
                load_v(next);
                if (b + 2 * kWaves < blast) next_id = ids[b + 2 * kWaves];
            }
        }

        // ---- the waves' states into one ----------------------------------------------------------
        if (g.bad) lsum = NAN;
        lsum = sum_u(lsum);
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[t][r] = add_mirror(acc[t][r]);  // P's hi + lo halves
        if (c < cols) {
            if (u == 0) {
                s_m[wave][c] = m_used;
                s_l[wave][c] = lsum;
            }
            // the lane holds dims 32 u + 8 r + t of its head
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < 8; t += 4)
                    *reinterpret_cast<f32x4*>(&s_acc[wave][c][32 * u + 8 * r + t]) =
                        f32x4{acc[t][r], acc[t + 1][r], acc[t + 2][r], acc[t + 3][r]};
        }
        __syncthreads();
        const size_t out0 = ((size_t)g.seq * a.hq + h0) * kDim;
        const size_t plane = (size_t)blockIdx.y * a.runs;  // of this chunk of columns
        const Parts parts_at = __builtin_amdgcn_make_buffer_rsrc(a.part, 0, a.part_bytes, 0x00027000);
        auto part_of = [&](int r, int second) {
            return (int)(((plane + r) * a.p.hkv + kh) * 2 + second) * kPartBytes;
        };
        constexpr int kSums = 2 * kMaxCols * 4;  // where a part's sums start
        for (int i = threadIdx.x; i < cols * (kDim / 4); i += kDecThreads) {
            const int col = i / (kDim / 4), d = 4 * (i % (kDim / 4));
            float m = s_m[0][col];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_m[w][col]);
            float l = 0.0f;
            f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                // a wave without a page has m = -inf, l = 0 (or NaN for a page that is not there)
                const float f = part_weight(s_m[w][col], m);
                l += s_m[w][col] == -INFINITY ? s_l[w][col] : s_l[w][col] * f;
                const f32x4 y = *reinterpret_cast<const f32x4*>(&s_acc[w][col][d]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = fmaf(y[e], f, x[e]);
            }
            if (g.whole) {
                write_o(a, out0 + 4 * i, x, l);
            } else {
                const int p = part_of(run, at == run * run_size ? 0 : 1);
                st_part(parts_at, p + kSums + 16 * i, x);
                if (d == 0) st_part2(parts_at, p + 8 * col, m, l);
            }
        }
        if (!g.whole) {
            // ---- the last segment of the sequence to arrive merges all of them ------------------
            const int r0 = seq_at / run_size;
            const int parts = cut ? __builtin_amdgcn_readlane(np1, seq) : (seq_at + g.np - 1) / size - r0 + 1;
            const int first = seq_at == r0 * run_size ? 0 : 1;  // a run's parts: its first segment's, then another
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (threadIdx.x == 0) {
                unsigned* ctr = a.ctr + ((plane + r0) * a.p.hkv + kh) * kCounterStride;
                s_last = atomicInc(ctr, parts - 1) == (unsigned)(parts - 1);
            }
            __syncthreads();
            if (s_last) {
                // A thread sums four dims over the parts; where the columns leave threads over,
                // these share the parts. The first loads go out before the weights are known.
                constexpr int kAhead = 16;  // parts whose loads are in flight together
                const int chunks = cols * (kDim / 4);
                const int share = kDecThreads / chunks;
                const int i = threadIdx.x % chunks, g = threadIdx.x / chunks;
                const int col = i / (kDim / 4);
                f32x4 w[kAhead];
                auto load = [&](int r) {
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) {
                        const int rj = min(r + j * share, parts - 1);
                        w[j] = ld_part(parts_at, part_of(r0 + rj, rj ? 0 : first) + kSums + 16 * i);
                    }
                };
                // (m, l) of this wave's first column's parts go ahead of the sums
                f32x2 ml = ld_part2(parts_at, part_of(r0 + min(lane, parts - 1), lane ? 0 : first) + 8 * min(wave, cols - 1));
                __builtin_amdgcn_sched_barrier(0);
                load(g);
                __builtin_amdgcn_sched_barrier(0);
                // weights: a wave per column, a lane per part
                float* s_w = &s_acc[0][0][0];  // [column][part]
                for (int cw = wave; cw < cols; cw += kWaves) {
                    if (cw != wave) ml = ld_part2(parts_at, part_of(r0 + min(lane, parts - 1), lane ? 0 : first) + 8 * cw);
                    float m = lane < parts ? ml[0] : -INFINITY, l = 0.0f;
                    for (int r = lane + 64; r < parts; r += 64)
                        m = fmaxf(m, ld_part2(parts_at, part_of(r0 + r, 0) + 8 * cw)[0]);
#pragma unroll
                    for (int d = 32; d; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
                    for (int r = lane; r < parts; r += 64) {
                        if (r >= 64) ml = ld_part2(parts_at, part_of(r0 + r, 0) + 8 * cw);
                        const float f = part_weight(ml[0], m);
                        s_w[cw * parts + r] = f;
                        l += ml[0] == -INFINITY ? ml[1] : ml[1] * f;
                    }
#pragma unroll
                    for (int d = 32; d; d /= 2) l += __shfl_xor(l, d);
                    if (lane == 0) s_l[0][cw] = l;
                }
                __syncthreads();
                f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int r = g; r < parts; r += share * kAhead) {
                    if (r != g) load(r);
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) {
                        if (r + j * share >= parts) continue;
                        const float f = s_w[col * parts + r + j * share];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = fmaf(w[j][e], f, x[e]);
                    }
                }
                if (share > 1) {
                    s_sum[threadIdx.x] = x;
                    __syncthreads();
                    for (int j = 1; j < share && threadIdx.x < chunks; ++j) x += s_sum[threadIdx.x + j * chunks];
                }
                if (threadIdx.x < chunks) write_o(a, out0 + 4 * i, x, s_l[0][col]);
            }
        }
        if (cut) return;
        at = seq_at + g.b1;
        if (at >= end) return;
        __syncthreads();  // the LDS is free for the next segment
        ++seq;
        seq_at = at;
    }
}

int decode_runs(int hkv, int chunks) { return std::max(kSlots / (hkv * chunks), 1); }

}  // namespace

int store_paged_launch(const PoolArgs& pool, const float* k, const float* v, const int* cu,
                       const int* pos, const int* table, int n, int width, int tokens,
                       hipStream_t stream) {
    StoreArgs a{pool, k, v, cu, pos, table, n, width, tokens, 0};
    // blocks touched: a sequence of r rows touches (r - 1) / 64 + 2 at most
    const long long m = std::min(n, tokens);
    const long long items = (tokens - m) / kPage + 2 * m;
    // A launch of 2^32 threads or more runs fewer, without an error: at most 2^31 in each.
    const long long most = (1LL << 31) / kStoreThreads / pool.hkv;
    for (long long i = 0; i < items; i += most) {
        a.item0 = (int)i;
        hipLaunchKernelGGL(store_paged_kernel, dim3((unsigned)(std::min(items - i, most) * pool.hkv), 2),
                           dim3(kStoreThreads), 0, stream, a);
        const int st = check_launch("store_paged_kernel");
        if (st != BRASA_OK) return st;
    }
    return BRASA_OK;
}

// The workspace: arrival counters, then two parts for each workgroup. The counters take the same room
// whatever the heads (hkv * chunks is at most 1024 where hq is), so that calls of other heads on one
// workspace leave them alone.
constexpr size_t kCounterBytes = 1024 * kCounterStride * sizeof(unsigned);
static size_t decode_paged_wgs(int hq, int hkv) {
    const int chunks = (hq / hkv + kMaxCols - 1) / kMaxCols;
    return (size_t)chunks * decode_runs(hkv, chunks) * hkv;
}
size_t decode_paged_workspace_len(int hq, int hkv) {
    const size_t wgs = decode_paged_wgs(hq, hkv);
    return kCounterBytes + wgs * 2 * kPartBytes;
}

int decode_paged_launch(const float* q, const PoolArgs& pool, const int* table, int width,
                        const int* lk, int n, void* ws, void* o, int o_f16, int hq,
                        hipStream_t stream) {
    DecodePagedArgs a;
    a.q = q;
    a.p = pool;
    a.table = table;
    a.lk = lk;
    a.o = o;
    a.n = n;
    a.width = width;
    a.hq = hq;
    a.group = hq / pool.hkv;
    a.o_f16 = o_f16;
    const int chunks = (a.group + kMaxCols - 1) / kMaxCols;
    a.runs = decode_runs(pool.hkv, chunks);
    const size_t wgs = decode_paged_wgs(hq, pool.hkv);
    a.ctr = static_cast<unsigned*>(ws);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kCounterBytes);
    a.part_bytes = (int)(wgs * 2 * kPartBytes);
    hipLaunchKernelGGL(decode_paged_kernel, dim3((unsigned)(a.runs * pool.hkv), chunks), dim3(kDecThreads),
                       0, stream, a);
    return check_launch("decode_paged_kernel");
}

}  // namespace brasa
