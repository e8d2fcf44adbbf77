// C ABI of libbrasa_attn.so: argument validation mirroring the reference's asserts, the error
// plumbing, and the device plumbing of brasa_hip_rt.h. Kernels live in kv.hip, decode.hip and
// prefill.hip.
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <vector>

#include "../../include/brasa_hip_rt.h"
#include "common.hpp"

namespace brasa {

int store_kv_launch(int kv, const float* src, void* dst, size_t n, hipStream_t stream);
int dequant_q8_launch(const void* src, float* dst, size_t rows, hipStream_t stream);
int fill_u8_launch(void* dst, uint8_t value, size_t bytes, hipStream_t stream);
int fill_normal_launch(float* out, size_t n, uint64_t seed, float scale, hipStream_t stream);
int decode_launch(const float* q, const void* k, const void* v, float* partials, void* o,
                  int o_f16, int hq, int hkv, int lk, int kv, bool per_head, hipStream_t stream);
int decode_noalloc_launch(const float* q, const void* k, const void* v, void* o, int o_f16,
                          int hq, int hkv, int lk, int kv, hipStream_t stream);
int rms_norm_launch(const float* x, const float* w, float* out, size_t rows, size_t n, float eps,
                    hipStream_t stream);
int rope_neox_launch(float* x, const float* cos_t, const float* sin_t, size_t tokens,
                     size_t heads, size_t dim, size_t pos0, hipStream_t stream);
int qk_norm_rope_store_launch(int kv, float* q, float* k, const float* v, const float* qn,
                              const float* kn, float eps, const float* cos_t, const float* sin_t,
                              void* kdst, void* vdst, size_t tokens, size_t hq, size_t hkv,
                              size_t pos0, hipStream_t stream);
void rope_table_host(double theta, size_t dim, size_t max_pos, float* cos_out, float* sin_out);
int decode_batch_launch(const float* q, const void* const* k, const void* const* v,
                        const int* lk, int n, float* partials, void* o, int o_f16, int hq,
                        int hkv, int kv, bool per_head, hipStream_t stream);
int prefill_launch(const float* q, const void* k, const void* v, void* o, int tokens, int hq,
                   int hkv, int pos0, int kv, int precision, bool caller_ws, void* ws,
                   size_t ws_len, hipStream_t stream, const int* layout = nullptr);
size_t prefill_workspace_len(int tokens, int hq, int hkv, int pos0, int kv, int precision,
                             size_t* required);
void prefill_release_workspaces();
int packed_launch(const float* q, const void* k, const void* v, void* o, const int* cu, int n, int tokens,
                  int hq, int hkv, int kv, int precision, hipStream_t stream);
int store_paged_launch(const PoolArgs& pool, const float* k, const float* v, const int* cu,
                       const int* pos, const int* table, int n, int width, int tokens,
                       hipStream_t stream);
size_t decode_paged_workspace_len(int hq, int hkv);
int decode_paged_launch(const float* q, const PoolArgs& pool, const int* table, int width,
                        const int* lk, int n, void* ws, void* o, int o_f16, int hq,
                        hipStream_t stream);
size_t kv_pages_workspace_len(int pages, int n, int width);
int kv_pages_fork_launch(const int* parent, const int* table, const int* len, const int* ref,
                         int* table_out, int* len_out, int* ref_out, int n, int width, int pages,
                         hipStream_t stream);
int kv_pages_reserve_launch(const PoolArgs& pool, const int* add, const int* table, const int* len,
                            const int* ref, int* table_out, int* ref_out, int* status, int n, int width,
                            void* ws, hipStream_t stream);
int kv_pages_compact_launch(const PoolArgs& pool, const int* table, const int* ref, int* table_out,
                            int* ref_out, int* live, int n, int width, void* ws, hipStream_t stream);

namespace {
thread_local char g_err[512] = "";
}

int set_error(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return set_error(BRASA_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
    return BRASA_OK;
}

static int hip_ok(hipError_t e, const char* what) {
    if (e != hipSuccess) return set_error(BRASA_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
    return BRASA_OK;
}

static inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

static bool valid_kv(int kv) {
    return kv == BRASA_KV_F32 || kv == BRASA_KV_F16 || kv == BRASA_KV_Q8_0;
}

// Largest sizes the kernels index with 32-bit integers.
static constexpr size_t kMaxPositions = (size_t)1 << 30;
static constexpr size_t kMaxHeads = 1024;
static constexpr size_t kMaxSeqs = 65536;  // (a workgroup walks them to find its own)
static constexpr size_t kMaxPages = (size_t)1 << 24;

}  // namespace brasa

using namespace brasa;

extern "C" {

size_t brasa_decode_partials_len(size_t hq, size_t lk) {
    return hq * ((lk + BRASA_DECODE_CHUNK - 1) / BRASA_DECODE_CHUNK) * 130;
}

size_t brasa_kv_capacity(size_t ctx) {
    return (ctx + BRASA_KV_ALIGN - 1) / BRASA_KV_ALIGN * BRASA_KV_ALIGN;
}

size_t brasa_kv_cache_len(size_t layers, size_t ctx, size_t hkv, size_t dim) {
    return layers * brasa_kv_capacity(ctx) * hkv * dim;
}

size_t brasa_kv_offset(size_t layer, size_t ctx, size_t hkv, size_t dim, size_t pos) {
    return (layer * brasa_kv_capacity(ctx) + pos) * hkv * dim;
}

int brasa_gqa_supported(size_t hq, size_t hkv) {
    if (hkv == 0 || hq % hkv != 0) return 0;
    const size_t g = hq / hkv;
    return g == 1 || g == 2 || g == 4 || g == 8;
}

size_t brasa_kv_bytes(int kv, size_t n) {
    switch (kv) {
        case BRASA_KV_F32: return n * 4;
        case BRASA_KV_F16: return n * 2;
        case BRASA_KV_Q8_0:
            if (n % kDim != 0) {
                set_error(BRASA_ERR_SHAPE, "KV Q8: rows of %d values (n = %zu)", kDim, n);
                return 0;
            }
            return n / kDim * kQ8Row;
    }
    set_error(BRASA_ERR_ARG, "invalid kv type %d", kv);
    return 0;
}

int brasa_store_kv(int kv, const float* src, void* dst, size_t n, void* stream) {
    g_err[0] = 0;
    if (!valid_kv(kv)) return set_error(BRASA_ERR_ARG, "store_kv: invalid kv type %d", kv);
    if (n == 0) return BRASA_OK;
    if (!src || !dst) return set_error(BRASA_ERR_ARG, "store_kv: null pointer");
    if (kv == BRASA_KV_Q8_0 && n % kDim != 0)  // lib.rs:1039
        return set_error(BRASA_ERR_SHAPE, "KV Q8: rows of %d values (n = %zu)", kDim, n);
    return store_kv_launch(kv, src, dst, n, as_stream(stream));
}

int brasa_dequantize_kv_q8(const void* src, float* dst, size_t rows, void* stream) {
    g_err[0] = 0;
    if (rows == 0) return BRASA_OK;
    if (!src || !dst) return set_error(BRASA_ERR_ARG, "dequantize_kv_q8: null pointer");
    return dequant_q8_launch(src, dst, rows, as_stream(stream));
}

// Shape checks of the decode entry points (lib.rs:1074-1080 / 1128-1135). partials == nullptr
// with noalloc: the library's fixed scratch array is used instead of the caller's.
static int decode_common(const float* q, const void* k, const void* v, float* partials,
                         size_t partials_len, void* o, int o_dtype, brasa_attn_shape s,
                         void* stream, bool per_head, bool noalloc = false) {
    g_err[0] = 0;
    if (!valid_kv(s.kv)) return set_error(BRASA_ERR_ARG, "decode: invalid kv type %d", s.kv);
    if (o_dtype != BRASA_OUT_F32 && o_dtype != BRASA_OUT_F16)
        return set_error(BRASA_ERR_ARG, "decode: invalid output dtype %d", o_dtype);
    // lib.rs:1074-1080 / 1128-1135
    if (s.tokens != 1) return set_error(BRASA_ERR_SHAPE, "decode_attention is for one token");
    if (s.dim != (size_t)kDim)
        return set_error(BRASA_ERR_SHAPE, "decode_attention requires head_dim 128");
    if (s.hkv == 0 || s.hq % s.hkv != 0)
        return set_error(BRASA_ERR_SHAPE, "hq must be a multiple of hkv");
    if (s.hq > kMaxHeads || s.pos0 + 1 > kMaxPositions)
        return set_error(BRASA_ERR_SHAPE, "decode: shape too large");
    const size_t lk = s.pos0 + 1;
    if (!noalloc && partials_len < brasa_decode_partials_len(s.hq, lk))
        return set_error(BRASA_ERR_SCRATCH, "decode scratch too small (%zu < %zu floats)",
                         partials_len, brasa_decode_partials_len(s.hq, lk));
    if (!per_head && !brasa_gqa_supported(s.hq, s.hkv))
        return set_error(BRASA_ERR_UNSUPPORTED,
                         "decode_attention_lanes: GQA group %zu not compiled", s.hq / s.hkv);
    if (!q || !k || !v || (!partials && !noalloc) || !o)
        return set_error(BRASA_ERR_ARG, "decode: null pointer");
    if (noalloc)
        return decode_noalloc_launch(q, k, v, o, o_dtype == BRASA_OUT_F16, (int)s.hq, (int)s.hkv,
                                     (int)lk, s.kv, as_stream(stream));
    return decode_launch(q, k, v, partials, o, o_dtype == BRASA_OUT_F16, (int)s.hq, (int)s.hkv,
                         (int)lk, s.kv, per_head, as_stream(stream));
}

int brasa_decode_attention_lanes(const float* q, const void* k, const void* v, float* partials,
                                 size_t partials_len, void* o, int o_dtype,
                                 brasa_attn_shape shape, void* stream) {
    return decode_common(q, k, v, partials, partials_len, o, o_dtype, shape, stream, false);
}

int brasa_decode_attention_lanes_noalloc(const float* q, const void* k, const void* v, void* o,
                                         int o_dtype, brasa_attn_shape shape, void* stream) {
    return decode_common(q, k, v, nullptr, 0, o, o_dtype, shape, stream, false, true);
}

int brasa_decode_attention(const float* q, const void* k, const void* v, float* partials,
                           size_t partials_len, void* o, int o_dtype, brasa_attn_shape shape,
                           void* stream) {
    return decode_common(q, k, v, partials, partials_len, o, o_dtype, shape, stream, true);
}

size_t brasa_decode_batch_partials_len(size_t hq, const size_t* lk, size_t n) {
    size_t f = 0;
    for (size_t i = 0; i < n; ++i) f += brasa_decode_partials_len(hq, lk[i]);
    return f;
}

int brasa_decode_attention_batch(const float* q, const void* const* k, const void* const* v,
                                 const size_t* lk, size_t n, float* partials,
                                 size_t partials_len, void* o, int o_dtype, size_t hq,
                                 size_t hkv, size_t dim, int kv, void* stream) {
    g_err[0] = 0;
    if (!valid_kv(kv)) return set_error(BRASA_ERR_ARG, "decode batch: invalid kv type %d", kv);
    if (o_dtype != BRASA_OUT_F32 && o_dtype != BRASA_OUT_F16)
        return set_error(BRASA_ERR_ARG, "decode batch: invalid output dtype %d", o_dtype);
    if (dim != (size_t)kDim)
        return set_error(BRASA_ERR_SHAPE, "decode_attention requires head_dim 128");
    if (hkv == 0 || hq % hkv != 0) return set_error(BRASA_ERR_SHAPE, "hq must be a multiple of hkv");
    if (!brasa_gqa_supported(hq, hkv))
        return set_error(BRASA_ERR_UNSUPPORTED, "decode batch: GQA group %zu not compiled", hq / hkv);
    if (hq > kMaxHeads || n > ((size_t)1 << 20))
        return set_error(BRASA_ERR_SHAPE, "decode batch: shape too large");
    if (n == 0) return BRASA_OK;
    if (!lk || !k || !v) return set_error(BRASA_ERR_ARG, "decode batch: null array");
    std::vector<int> lki(n);
    for (size_t i = 0; i < n; ++i) {
        if (lk[i] == 0) return set_error(BRASA_ERR_SHAPE, "decode batch: sequence %zu has no keys", i);
        if (lk[i] > kMaxPositions) return set_error(BRASA_ERR_SHAPE, "decode batch: shape too large");
        if (!k[i] || !v[i]) return set_error(BRASA_ERR_ARG, "decode batch: null cache pointer %zu", i);
        lki[i] = (int)lk[i];
    }
    const size_t need = brasa_decode_batch_partials_len(hq, lk, n);
    if (partials_len < need)
        return set_error(BRASA_ERR_SCRATCH, "decode scratch too small (%zu < %zu floats)",
                         partials_len, need);
    if (!q || !partials || !o) return set_error(BRASA_ERR_ARG, "decode batch: null pointer");
    return decode_batch_launch(q, k, v, lki.data(), (int)n, partials, o, o_dtype == BRASA_OUT_F16,
                               (int)hq, (int)hkv, kv, false, as_stream(stream));
}

// Shape checks of the prefill entry points (lib.rs:1203-1204, 1227-1231).
static int prefill_check(brasa_attn_shape s, int precision) {
    if (!valid_kv(s.kv)) return set_error(BRASA_ERR_ARG, "flash_attention: invalid kv %d", s.kv);
    if (precision != BRASA_PREFILL_F16 && precision != BRASA_PREFILL_F32 &&
        precision != BRASA_PREFILL_F16_PF32)
        return set_error(BRASA_ERR_ARG, "flash_attention: invalid precision %d", precision);
    // lib.rs:1203-1204
    if (s.dim != (size_t)kDim)
        return set_error(BRASA_ERR_SHAPE, "flash_attention requires head_dim 128");
    if (s.hkv == 0 || s.hq % s.hkv != 0)
        return set_error(BRASA_ERR_SHAPE, "hq must be a multiple of hkv");
    if (s.hq > kMaxHeads || s.pos0 + s.tokens + BRASA_KV_ALIGN > kMaxPositions)
        return set_error(BRASA_ERR_SHAPE, "flash_attention: shape too large");
    // lib.rs:1227-1231: outside the compiled GQA groups only the f32 kernel exists
    if (!brasa_gqa_supported(s.hq, s.hkv) && precision != BRASA_PREFILL_F32)
        return set_error(BRASA_ERR_UNSUPPORTED,
                         "flash_attention: without a compiled GQA group (%zu) attention is f32 only",
                         s.hq / s.hkv);
    return BRASA_OK;
}

int brasa_flash_attention_with(const float* q, const void* k, const void* v, void* o,
                               brasa_attn_shape s, int precision, void* stream) {
    g_err[0] = 0;
    const int st = prefill_check(s, precision);
    if (st != BRASA_OK) return st;
    if (s.tokens == 0) return BRASA_OK;
    if (!q || !k || !v || !o) return set_error(BRASA_ERR_ARG, "flash_attention: null pointer");
    return prefill_launch(q, k, v, o, (int)s.tokens, (int)s.hq, (int)s.hkv, (int)s.pos0, s.kv,
                          precision, false, nullptr, 0, as_stream(stream));
}

size_t brasa_flash_attention_workspace_len(brasa_attn_shape s, int precision) {
    g_err[0] = 0;
    if (prefill_check(s, precision) != BRASA_OK || s.tokens == 0) return 0;
    return prefill_workspace_len((int)s.tokens, (int)s.hq, (int)s.hkv, (int)s.pos0, s.kv,
                                 precision, nullptr);
}

int brasa_flash_attention_ws(const float* q, const void* k, const void* v, void* o,
                             brasa_attn_shape s, int precision, void* workspace,
                             size_t workspace_len, void* stream) {
    g_err[0] = 0;
    const int st = prefill_check(s, precision);
    if (st != BRASA_OK) return st;
    if (s.tokens == 0) return BRASA_OK;
    if (!q || !k || !v || !o) return set_error(BRASA_ERR_ARG, "flash_attention: null pointer");
    // (a split that only makes the call faster is left out of a smaller workspace)
    size_t need = 0;
    prefill_workspace_len((int)s.tokens, (int)s.hq, (int)s.hkv, (int)s.pos0, s.kv, precision, &need);
    if (workspace_len < need || (need > 0 && !workspace))
        return set_error(BRASA_ERR_SCRATCH, "flash_attention workspace too small (%zu < %zu bytes)",
                         workspace_len, need);
    return prefill_launch(q, k, v, o, (int)s.tokens, (int)s.hq, (int)s.hkv, (int)s.pos0, s.kv,
                          precision, true, workspace, workspace_len, as_stream(stream));
}

int brasa_flash_attention(const float* q, const void* k, const void* v, void* o,
                          brasa_attn_shape shape, void* stream) {
    return brasa_flash_attention_with(q, k, v, o, shape, BRASA_PREFILL_F16, stream);
}

int brasa_flash_attention_packed(const float* q, const void* k, const void* v, void* o,
                                 const int32_t* cu, size_t n, brasa_attn_shape s, int precision,
                                 void* stream) {
    g_err[0] = 0;
    const char* what = "flash_attention_packed";
    if (!valid_kv(s.kv)) return set_error(BRASA_ERR_ARG, "%s: invalid kv %d", what, s.kv);
    if (precision != BRASA_PREFILL_F16 && precision != BRASA_PREFILL_F32 &&
        precision != BRASA_PREFILL_F16_PF32)
        return set_error(BRASA_ERR_ARG, "%s: invalid precision %d", what, precision);
    if (s.kv == BRASA_KV_Q8_0)
        return set_error(BRASA_ERR_UNSUPPORTED, "%s: K and V rows are f32 or f16", what);
    if (s.dim != (size_t)kDim) return set_error(BRASA_ERR_SHAPE, "%s requires head_dim 128", what);
    if (s.hq == 0 || s.hkv == 0 || s.hq % s.hkv != 0)
        return set_error(BRASA_ERR_SHAPE, "hq must be a multiple of hkv");
    if (s.pos0 != 0) return set_error(BRASA_ERR_SHAPE, "%s: whole prompts only (pos0 = %zu)", what, s.pos0);
    if (s.hq > kMaxHeads || s.tokens > kMaxPositions / s.hq || n > kMaxSeqs)
        return set_error(BRASA_ERR_SHAPE, "%s: shape too large", what);
    if (s.tokens == 0 || n == 0) return BRASA_OK;
    if (!q || !k || !v || !o || !cu) return set_error(BRASA_ERR_ARG, "%s: null pointer", what);
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) % 16)
        return set_error(BRASA_ERR_ARG, "%s: q, k, v and o must be 16-byte aligned", what);
    return packed_launch(q, k, v, o, cu, (int)n, (int)s.tokens, (int)s.hq, (int)s.hkv, s.kv, precision,
                         as_stream(stream));
}

// The checks every call on a pool makes; `out` is the pool from `layer` on.
static int pool_check(const char* what, brasa_kv_pool p, size_t layer, PoolArgs* out) {
    if (p.dim != (size_t)kDim) return set_error(BRASA_ERR_SHAPE, "%s requires head_dim 128", what);
    if (p.hkv == 0 || p.hkv > kMaxHeads) return set_error(BRASA_ERR_SHAPE, "%s: %zu KV heads", what, p.hkv);
    if (p.pages == 0 || p.pages > kMaxPages || p.layers == 0 ||
        p.layers > ((size_t)1 << 31) / (p.pages * p.hkv))
        return set_error(BRASA_ERR_SHAPE, "%s: a pool of %zu layers of %zu pages", what, p.layers, p.pages);
    if (layer >= p.layers) return set_error(BRASA_ERR_SHAPE, "%s: layer %zu of %zu", what, layer, p.layers);
    if (!p.k || !p.v || !p.k_exp || !p.v_exp) return set_error(BRASA_ERR_ARG, "%s: null pool pointer", what);
    if (((uintptr_t)p.k | (uintptr_t)p.v) % 16)
        return set_error(BRASA_ERR_ARG, "%s: the codes must be 16-byte aligned", what);
    const size_t at = layer * p.pages * p.hkv;
    const size_t tile = (size_t)BRASA_KV_PAGE * kDim;
    *out = PoolArgs{(uint8_t*)p.k + at * tile, (uint8_t*)p.v + at * tile, (uint8_t*)p.k_exp + at,
                    (uint8_t*)p.v_exp + at, (int)(p.layers - layer), (int)p.pages, (int)p.hkv};
    return BRASA_OK;
}
// n rows of `width` table entries
static int table_check(const char* what, size_t n, size_t width) {
    if (n > kMaxSeqs || width > kMaxPages || (n && width > ((size_t)1 << 30) / n))
        return set_error(BRASA_ERR_SHAPE, "%s: a table of %zu x %zu pages is too large", what, n, width);
    return BRASA_OK;
}

size_t brasa_kv_pool_bytes(size_t layers, size_t pages, size_t hkv, size_t dim) {
    return layers * pages * hkv * BRASA_KV_PAGE * dim;
}

int brasa_store_kv_paged(brasa_kv_pool pool, size_t layer, const float* k, const float* v,
                         const int32_t* cu, const int32_t* pos, const int32_t* table, size_t n,
                         size_t width, size_t tokens, void* stream) {
    g_err[0] = 0;
    const char* what = "store_kv_paged";
    PoolArgs p;
    int st = pool_check(what, pool, layer, &p);
    if (st == BRASA_OK) st = table_check(what, n, width);
    if (st != BRASA_OK) return st;
    if (tokens > kMaxPositions / pool.hkv) return set_error(BRASA_ERR_SHAPE, "%s: shape too large", what);
    if (n == 0 || tokens == 0 || width == 0) return BRASA_OK;
    if (!k || !v || !cu || !pos || !table) return set_error(BRASA_ERR_ARG, "%s: null pointer", what);
    if (((uintptr_t)k | (uintptr_t)v) % 16)
        return set_error(BRASA_ERR_ARG, "%s: the rows must be 16-byte aligned", what);
    return store_paged_launch(p, k, v, cu, pos, table, (int)n, (int)width, (int)tokens, as_stream(stream));
}

size_t brasa_decode_paged_workspace_len(size_t hq, size_t hkv) {
    if (hkv == 0 || hq == 0 || hq % hkv != 0 || hq > kMaxHeads) return 0;
    return decode_paged_workspace_len((int)hq, (int)hkv);
}

int brasa_decode_attention_paged(const float* q, brasa_kv_pool pool, size_t layer,
                                 const int32_t* table, size_t width, const int32_t* lk, size_t n,
                                 void* workspace, size_t workspace_len, void* o, int o_dtype,
                                 size_t hq, void* stream) {
    g_err[0] = 0;
    const char* what = "decode_attention_paged";
    if (o_dtype != BRASA_OUT_F32 && o_dtype != BRASA_OUT_F16)
        return set_error(BRASA_ERR_ARG, "%s: invalid output dtype %d", what, o_dtype);
    PoolArgs p;
    int st = pool_check(what, pool, layer, &p);
    if (st == BRASA_OK) st = table_check(what, n, width);
    if (st != BRASA_OK) return st;
    if (hq == 0 || hq > kMaxHeads || hq % pool.hkv != 0)
        return set_error(BRASA_ERR_SHAPE, "hq must be a multiple of hkv, at most %zu", kMaxHeads);
    const size_t need = brasa_decode_paged_workspace_len(hq, pool.hkv);
    if (workspace_len < need)
        return set_error(BRASA_ERR_SCRATCH, "%s: workspace too small (%zu < %zu bytes)", what, workspace_len, need);
    if (n == 0) return BRASA_OK;
    if (!q || (!table && width) || !lk || !workspace || !o)
        return set_error(BRASA_ERR_ARG, "%s: null pointer", what);
    if ((uintptr_t)workspace % 256 || ((uintptr_t)q | (uintptr_t)o) % 16)
        return set_error(BRASA_ERR_ARG, "%s: q and o must be 16-byte, the workspace 256-byte aligned", what);
    return decode_paged_launch(q, p, table, (int)width, lk, (int)n, workspace, o,
                               o_dtype == BRASA_OUT_F16, (int)hq, as_stream(stream));
}

int brasa_kv_pages_fork(const int32_t* parent, const int32_t* table, const int32_t* len,
                        const int32_t* ref, int32_t* table_out, int32_t* len_out,
                        int32_t* ref_out, size_t n, size_t width, size_t pages, void* stream) {
    g_err[0] = 0;
    const char* what = "kv_pages_fork";
    const int st = table_check(what, n, width);
    if (st != BRASA_OK) return st;
    if (pages == 0 || pages > kMaxPages) return set_error(BRASA_ERR_SHAPE, "%s: %zu pages", what, pages);
    if (n == 0 || width == 0) {
        if (n == 0 && ref == ref_out) return BRASA_OK;
        if (width == 0) return set_error(BRASA_ERR_SHAPE, "%s: a table without columns", what);
    }
    if (!parent || !table || !len || !ref || !table_out || !len_out || !ref_out)
        return set_error(BRASA_ERR_ARG, "%s: null pointer", what);
    if (table_out == table || len_out == len)
        return set_error(BRASA_ERR_ARG, "%s: table_out and len_out must be arrays of their own", what);
    return kv_pages_fork_launch(parent, table, len, ref, table_out, len_out, ref_out, (int)n, (int)width,
                                (int)pages, as_stream(stream));
}

size_t brasa_kv_pages_workspace_len(size_t pages, size_t n, size_t width) {
    if (pages > kMaxPages || n > kMaxSeqs || width > kMaxPages || (n && width > ((size_t)1 << 30) / n)) return 0;
    return kv_pages_workspace_len((int)pages, (int)n, (int)width);
}

// What reserve and compact check alike.
static int pages_check(const char* what, brasa_kv_pool pool, size_t n, size_t width, const void* workspace,
                       size_t workspace_len, PoolArgs* p) {
    int st = pool_check(what, pool, 0, p);
    if (st == BRASA_OK) st = table_check(what, n, width);
    if (st != BRASA_OK) return st;
    const size_t need = brasa_kv_pages_workspace_len(pool.pages, n, width);
    if (workspace_len < need)
        return set_error(BRASA_ERR_SCRATCH, "%s: workspace too small (%zu < %zu bytes)", what, workspace_len, need);
    if (!workspace) return set_error(BRASA_ERR_ARG, "%s: null workspace", what);
    if ((uintptr_t)workspace % 256) return set_error(BRASA_ERR_ARG, "%s: the workspace must be 256-byte aligned", what);
    return BRASA_OK;
}

int brasa_kv_pages_reserve(brasa_kv_pool pool, const int32_t* add, const int32_t* table,
                           const int32_t* len, const int32_t* ref, int32_t* table_out,
                           int32_t* ref_out, int32_t* status, size_t n, size_t width,
                           void* workspace, size_t workspace_len, void* stream) {
    g_err[0] = 0;
    PoolArgs p;
    const int st = pages_check("kv_pages_reserve", pool, n, width, workspace, workspace_len, &p);
    if (st != BRASA_OK) return st;
    if (!ref || !ref_out || !status || (n && (!add || !len)) || (n && width && (!table || !table_out)))
        return set_error(BRASA_ERR_ARG, "kv_pages_reserve: null pointer");
    return kv_pages_reserve_launch(p, add, table, len, ref, table_out, ref_out, status, (int)n, (int)width,
                                   workspace, as_stream(stream));
}

int brasa_kv_pages_compact(brasa_kv_pool pool, const int32_t* table, const int32_t* ref,
                           int32_t* table_out, int32_t* ref_out, int32_t* live, size_t n,
                           size_t width, void* workspace, size_t workspace_len, void* stream) {
    g_err[0] = 0;
    PoolArgs p;
    const int st = pages_check("kv_pages_compact", pool, n, width, workspace, workspace_len, &p);
    if (st != BRASA_OK) return st;
    if (!ref || !ref_out || !live || (n && width && (!table || !table_out)))
        return set_error(BRASA_ERR_ARG, "kv_pages_compact: null pointer");
    return kv_pages_compact_launch(p, table, ref, table_out, ref_out, live, (int)n, (int)width, workspace,
                                   as_stream(stream));
}

int brasa_rope_table(double theta, size_t dim, size_t max_pos, float* cos_out, float* sin_out) {
    g_err[0] = 0;
    if (dim == 0 || dim % 2 != 0) return set_error(BRASA_ERR_SHAPE, "rope_table: dim must be even");
    if (max_pos > 0 && (!cos_out || !sin_out))
        return set_error(BRASA_ERR_ARG, "rope_table: null pointer");
    rope_table_host(theta, dim, max_pos, cos_out, sin_out);
    return BRASA_OK;
}

int brasa_rms_norm(const float* x, const float* w, float* out, size_t rows, size_t n, float eps,
                   void* stream) {
    g_err[0] = 0;
    if (rows == 0) return BRASA_OK;
    if (n == 0 || n > ((size_t)1 << 24) || rows > ((size_t)1 << 30))
        return set_error(BRASA_ERR_SHAPE, "rms_norm: bad row length %zu", n);
    if (!x || !w || !out) return set_error(BRASA_ERR_ARG, "rms_norm: null pointer");
    return rms_norm_launch(x, w, out, rows, n, eps, as_stream(stream));
}

int brasa_rope_neox(float* x, brasa_rope_table_view table, size_t tokens, size_t heads,
                    size_t dim, size_t pos0, void* stream) {
    g_err[0] = 0;
    // lib.rs:579-583
    if (dim != table.dim) return set_error(BRASA_ERR_SHAPE, "RoPE table dimension");
    if (pos0 + tokens > table.max_pos) return set_error(BRASA_ERR_SHAPE, "position outside the RoPE table");
    if (dim == 0 || dim % 2 != 0 || heads > kMaxHeads)
        return set_error(BRASA_ERR_SHAPE, "rope_neox: bad shape");
    if (tokens == 0 || heads == 0) return BRASA_OK;
    if (!x || !table.cos || !table.sin) return set_error(BRASA_ERR_ARG, "rope_neox: null pointer");
    return rope_neox_launch(x, table.cos, table.sin, tokens, heads, dim, pos0, as_stream(stream));
}

int brasa_qk_norm_rope_store(int kv, float* q, float* k, const float* v, const float* q_norm,
                             const float* k_norm, float eps, brasa_rope_table_view table,
                             void* k_dst, void* v_dst, brasa_attn_shape s, void* stream) {
    g_err[0] = 0;
    if (!valid_kv(kv)) return set_error(BRASA_ERR_ARG, "qk_norm_rope_store: invalid kv type %d", kv);
    // lib.rs:996-1001
    if (s.dim != (size_t)kDim)
        return set_error(BRASA_ERR_SHAPE, "qk_norm_rope_store requires head_dim 128");
    if (s.dim != table.dim) return set_error(BRASA_ERR_SHAPE, "RoPE table dimension");
    if (s.pos0 + s.tokens > table.max_pos)
        return set_error(BRASA_ERR_SHAPE, "position outside the RoPE table");
    if (s.hq > kMaxHeads || s.hkv > kMaxHeads || s.tokens * (s.hq + 2 * s.hkv) > ((size_t)1 << 30))
        return set_error(BRASA_ERR_SHAPE, "qk_norm_rope_store: shape too large");
    if (s.tokens == 0) return BRASA_OK;
    if (!q || !k || !v || !q_norm || !k_norm || !table.cos || !table.sin || !k_dst || !v_dst)
        return set_error(BRASA_ERR_ARG, "qk_norm_rope_store: null pointer");
    return qk_norm_rope_store_launch(kv, q, k, v, q_norm, k_norm, eps, table.cos, table.sin,
                                     k_dst, v_dst, s.tokens, s.hq, s.hkv, s.pos0,
                                     as_stream(stream));
}

int brasa_release_workspaces(void) {
    g_err[0] = 0;
    prefill_release_workspaces();
    release_stream_slots();
    return BRASA_OK;
}

int brasa_test_flash_attention_layout(const float* q, const void* k, const void* v, void* o,
                                      brasa_attn_shape s, int precision, int variant, int pair,
                                      int parts, void* stream) {
    g_err[0] = 0;
    if (variant != 0 && variant != 1 && variant != 2 && variant != 4)
        return set_error(BRASA_ERR_ARG, "prefill layout: variant %d (0, 1, 2 or 4)", variant);
    if (parts < 1 || parts > 8)
        return set_error(BRASA_ERR_ARG, "prefill layout: %d key parts (1 .. 8)", parts);
    const int st = prefill_check(s, precision);
    if (st != BRASA_OK) return st;
    if (s.tokens == 0) return BRASA_OK;
    if (!q || !k || !v || !o) return set_error(BRASA_ERR_ARG, "flash_attention: null pointer");
    const int layout[3] = {variant, pair ? 1 : 0, parts};
    return prefill_launch(q, k, v, o, (int)s.tokens, (int)s.hq, (int)s.hkv, (int)s.pos0, s.kv,
                          precision, false, nullptr, 0, as_stream(stream), layout);
}

const char* brasa_last_error(void) { return g_err; }

const char* brasa_version(void) { return "brasa_attn 0.1.0 (gfx950)"; }

// ---- device plumbing (brasa_hip_rt.h) -----------------------------------------------------

int brasa_rt_device_count(int* count) { return hip_ok(hipGetDeviceCount(count), "hipGetDeviceCount"); }
int brasa_rt_set_device(int device) { return hip_ok(hipSetDevice(device), "hipSetDevice"); }
int brasa_rt_device_name(char* buf, size_t len) {
    hipDeviceProp_t p;
    int dev = 0;
    int st = hip_ok(hipGetDevice(&dev), "hipGetDevice");
    if (st) return st;
    st = hip_ok(hipGetDeviceProperties(&p, dev), "hipGetDeviceProperties");
    if (st) return st;
    snprintf(buf, len, "%s (%s, %d CUs)", p.name, p.gcnArchName, p.multiProcessorCount);
    return BRASA_OK;
}
int brasa_rt_malloc(void** ptr, size_t bytes) { return hip_ok(hipMalloc(ptr, bytes), "hipMalloc"); }
int brasa_rt_free(void* ptr) { return hip_ok(hipFree(ptr), "hipFree"); }
int brasa_rt_memcpy_htod(void* dst, const void* src, size_t bytes) {
    return hip_ok(hipMemcpy(dst, src, bytes, hipMemcpyHostToDevice), "hipMemcpy H2D");
}
int brasa_rt_memcpy_dtoh(void* dst, const void* src, size_t bytes) {
    return hip_ok(hipMemcpy(dst, src, bytes, hipMemcpyDeviceToHost), "hipMemcpy D2H");
}
int brasa_rt_memcpy_dtod(void* dst, const void* src, size_t bytes, void* stream) {
    return hip_ok(hipMemcpyAsync(dst, src, bytes, hipMemcpyDeviceToDevice, as_stream(stream)),
                  "hipMemcpyAsync D2D");
}
int brasa_rt_fill_u8(void* dst, uint8_t value, size_t bytes, void* stream) {
    return fill_u8_launch(dst, value, bytes, as_stream(stream));
}
int brasa_rt_device_synchronize(void) {
    return hip_ok(hipDeviceSynchronize(), "hipDeviceSynchronize");
}
int brasa_rt_stream_create(void** stream) {
    hipStream_t s = nullptr;
    int st = hip_ok(hipStreamCreateWithFlags(&s, hipStreamNonBlocking), "hipStreamCreate");
    *stream = s;
    return st;
}
int brasa_rt_stream_destroy(void* stream) {
    return hip_ok(hipStreamDestroy(as_stream(stream)), "hipStreamDestroy");
}
int brasa_rt_stream_synchronize(void* stream) {
    return hip_ok(hipStreamSynchronize(as_stream(stream)), "hipStreamSynchronize");
}
int brasa_rt_event_create(void** event) {
    hipEvent_t e = nullptr;
    int st = hip_ok(hipEventCreate(&e), "hipEventCreate");
    *event = e;
    return st;
}
int brasa_rt_event_destroy(void* event) {
    return hip_ok(hipEventDestroy(static_cast<hipEvent_t>(event)), "hipEventDestroy");
}
int brasa_rt_event_record(void* event, void* stream) {
    return hip_ok(hipEventRecord(static_cast<hipEvent_t>(event), as_stream(stream)),
                  "hipEventRecord");
}
int brasa_rt_event_elapsed_ms(float* ms, void* start, void* stop) {
    return hip_ok(hipEventElapsedTime(ms, static_cast<hipEvent_t>(start),
                                      static_cast<hipEvent_t>(stop)),
                  "hipEventElapsedTime");
}
int brasa_rt_event_synchronize(void* event) {
    return hip_ok(hipEventSynchronize(static_cast<hipEvent_t>(event)), "hipEventSynchronize");
}
int brasa_rt_stream_begin_capture(void* stream) {
    return hip_ok(hipStreamBeginCapture(as_stream(stream), hipStreamCaptureModeThreadLocal),
                  "hipStreamBeginCapture");
}
int brasa_rt_stream_end_capture(void* stream, void** graph_exec) {
    *graph_exec = nullptr;
    hipGraph_t g = nullptr;
    int st = hip_ok(hipStreamEndCapture(as_stream(stream), &g), "hipStreamEndCapture");
    if (st) return st;
    hipGraphExec_t e = nullptr;
    st = hip_ok(hipGraphInstantiate(&e, g, nullptr, nullptr, 0), "hipGraphInstantiate");
    const int st2 = hip_ok(hipGraphDestroy(g), "hipGraphDestroy");
    if (st) return st;
    *graph_exec = e;
    return st2;
}
int brasa_rt_graph_launch(void* graph_exec, void* stream) {
    return hip_ok(hipGraphLaunch(static_cast<hipGraphExec_t>(graph_exec), as_stream(stream)),
                  "hipGraphLaunch");
}
int brasa_rt_graph_destroy(void* graph_exec) {
    return hip_ok(hipGraphExecDestroy(static_cast<hipGraphExec_t>(graph_exec)),
                  "hipGraphExecDestroy");
}
int brasa_rt_mem_info(size_t* free_bytes, size_t* total_bytes) {
    return hip_ok(hipMemGetInfo(free_bytes, total_bytes), "hipMemGetInfo");
}
int brasa_rt_fill_normal_f32(float* out, size_t n, uint64_t seed, float scale, void* stream) {
    return fill_normal_launch(out, n, seed, scale, as_stream(stream));
}

}  // extern "C"
