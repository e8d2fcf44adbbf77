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

}  // namespace brasa
