// What the kernels of the paged 8-bit KV cache share: its layout and its e4m3 conversions.
//
// One layer of a pool holds `pages` pages; a page holds kPage positions of every KV head. Codes are
// [page][kv head][position in page][128] e4m3 bytes, K and V apart, so a head's page is one run of
// 8 KB that a wave reads in whole lines. Scales are one byte x per (page, head): a code c stands
// for e4m3(c) * 2^(x - 127).
#pragma once

#include "common.hpp"

namespace brasa {

constexpr int kPage = BRASA_KV_PAGE;        // positions of a page
constexpr int kTileBytes8 = kPage * kDim;   // codes of one head's page

// ---- wave64 helpers -------------------------------------------------------------------------
// inclusive sum over the lanes of a wave: within rows of 16 (row_shr), then row 0 into 1 and 2 into
// 3 (row_bcast 15), then the lower half into the upper (row_bcast 31)
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}

// ---- scalar loads -------------------------------------------------------------------------------
// Memory that no kernel of the launch writes, read through the scalar cache: uniform values that arrive
// without a place among the vector loads in flight.
template <typename T>
using Scalar = const __attribute__((address_space(4))) T*;
template <typename T>
__device__ __forceinline__ Scalar<T> scalar(const T* p) { return (Scalar<T>)(uintptr_t)p; }
// The same pointer, which the compiler does not know to be the same: what is read through it is read again.
template <typename T>
__device__ __forceinline__ uintptr_t again(T p) {
    uintptr_t x = (uintptr_t)p;
    asm volatile("" : "+s"(x));
    return x;
}

// ---- workgroup scans, of 1024 threads unless W says otherwise ------------------------------------------------------------
constexpr int kScanThreads = 1024;
constexpr int kScanWaves = kScanThreads / 64;

// exclusive sum over the threads of a workgroup of W waves; `sum` is the total. s: W ints of LDS, free
// again after the next barrier.
template <int W = kScanWaves>
__device__ __forceinline__ int across_waves(int mine, int* s, int& sum) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __syncthreads();  // s is free
    if (lane == 0) s[wave] = mine;
    __syncthreads();
    static_assert(W <= 16, "a row of 16 lanes scans the waves");
    int w = s[lane & (W - 1)];
    w += __builtin_amdgcn_update_dpp(0, w, 0x111, 0xF, 0xF, true);
    if (W > 2) w += __builtin_amdgcn_update_dpp(0, w, 0x112, 0xF, 0xF, true);
    if (W > 4) w += __builtin_amdgcn_update_dpp(0, w, 0x114, 0xF, 0xF, true);
    if (W > 8) w += __builtin_amdgcn_update_dpp(0, w, 0x118, 0xF, 0xF, true);
    sum = __builtin_amdgcn_readlane(w, W - 1);
    return __builtin_amdgcn_readlane(w, wave) - mine;
}
template <int W = kScanWaves>
__device__ __forceinline__ int block_scan(int x, int* s, int& sum) {
    const int incl = wave_scan(x);
    return across_waves<W>(__builtin_amdgcn_readlane(incl, 63), s, sum) + incl - x;
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

// ---- new rows -----------------------------------------------------------------------------------
// Packed new rows and where they go: sequence i's rows cu[i] .. cu[i + 1] to positions pos[i], ...
struct NewRows {
    const int* cu;
    const int* pos;
    const int* table;
    int n, width, tokens;
};

// how many blocks a sequence's rows [c0, c1) touch from position pos on: [pos / kPage, + count)
__device__ __forceinline__ int touched_blocks(const NewRows& a, int c0, int c1, int pos) {
    // (a negative position, or one past what the table can hold, has no block)
    if (c1 == c0 || pos < 0 || pos >= a.width * kPage) return 0;
    return min((pos + (c1 - c0) - 1) / kPage, a.width - 1) - pos / kPage + 1;
}
// inclusive maximum over the lanes of a wave
__device__ __forceinline__ int wave_max(int x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x = max(x, y);
    }
    return x;
}

// The item-th block of all that new rows touch: its page, its slots [s0, s1) that are new, and the
// packed row of its slot 0. Every wave walks the sequences' block counts, 64 at a time. False: there
// is no such block, or it has no page. APART: bounds out of order are raised to the largest before them, so
// that no row is in two blocks, for rows that are rewritten in place; else each sequence's are clamped alone.
struct TouchedBlock {
    int page, s0, s1, row0;
};
template <bool APART>
__device__ __forceinline__ bool touched_block(const NewRows& a, int item, int pages, TouchedBlock& t) {
    const int lane = threadIdx.x & 63;
    int seq = -1, before = 0, top = 0, c0 = 0, c1 = 0, pos = 0;
    for (int i0 = 0; i0 < a.n; i0 += 64) {
        int nb = 0;
        const int i = i0 + lane;
        if (i < a.n) {
            c0 = min(max(a.cu[i], 0), a.tokens);
            c1 = min(max(a.cu[i + 1], 0), a.tokens);
            pos = a.pos[i];
        }
        if (APART && __builtin_amdgcn_ballot_w64(i < a.n && (c0 < top || c1 < c0))) c0 = max(wave_max(c0), top);
        c1 = max(c1, c0);
        if (APART) top = __builtin_amdgcn_readlane(c1, 63);  // (where another round follows, all lanes have a sequence)
        if (i < a.n) nb = touched_blocks(a, c0, c1, pos);
        const int incl = wave_scan(nb) + before;
        const unsigned long long past = __builtin_amdgcn_ballot_w64(incl > item);
        if (past) {
            const int l = __builtin_ctzll(past);
            seq = i0 + l;
            before = __builtin_amdgcn_readlane(incl - nb, l);
            c0 = __builtin_amdgcn_readlane(c0, l);
            c1 = __builtin_amdgcn_readlane(c1, l);
            pos = __builtin_amdgcn_readlane(pos, l);
            break;
        }
        before = __builtin_amdgcn_readlane(incl, 63);
    }
    if (seq < 0) return false;  // the grid's bound is loose
    const int block = pos / kPage + item - before;
    t.page = a.table[(size_t)seq * a.width + block];
    if (t.page < 0 || t.page >= pages) return false;
    t.s0 = max(pos - block * kPage, 0);
    t.s1 = min(pos + (c1 - c0) - block * kPage, kPage);
    t.row0 = c0 + block * kPage - pos;
    return true;
}

// Blocks that new rows can touch: a sequence of r rows touches (r - 1) / 64 + 2 at most.
inline long long most_blocks(int n, int tokens) {
    const long long m = std::min(n, tokens);
    return (tokens - m) / kPage + 2 * m;
}

// ---- e4m3 -----------------------------------------------------------------------------------
// The scale byte of a block by its largest finite magnitude: the least x >= 0 with
// amax <= 448 * 2^(x - 127). 448 = 1.75 * 2^8, so amax = m 2^a (1 <= m < 2) takes a - 8, and one
// more where m > 1.75; whole-number arithmetic on the bits, without a rounding.
__device__ __forceinline__ int e4m3_scale(float amax) {
    const uint32_t b = __float_as_uint(amax);
    return max((int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
}

// Four values x * 2^shift (of magnitude <= 448, or not finite: the NaN code with x's sign) as e4m3
// bytes, rounded to nearest even (v_cvt_pk_fp8_f32; half a step, 2^-4 relative, is the cache
// type's own precision).
__device__ __forceinline__ uint32_t e4m3_quad(const float (&x)[4], int shift) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = ldexpf(x[e], shift);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    uint32_t c = (uint32_t)w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (!(fabsf(x[e]) < INFINITY))
            c = (c & ~(0xffu << 8 * e)) | (0x7fu | (__float_as_uint(x[e]) >> 24 & 0x80u)) << 8 * e;
    return c;
}

// The codes of a block's slots [0, s0), rounded to a scale 2^-shift as large (exact but where they leave
// e4m3's normal range), by a workgroup of THREADS.
template <int THREADS>
__device__ __forceinline__ void rescale_rows(uint8_t* codes, int s0, int shift) {
    for (int i = threadIdx.x; i < s0 * (kDim / 4); i += THREADS) {
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
        *w = e4m3_quad(y, shift);
    }
}

}  // namespace brasa
