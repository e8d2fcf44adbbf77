// Rotary positions read on the device, with one to four axes: alone on rows of any even head_dim, and
// fused with the per-head norms of q and k and the paged 8-bit cache's writer.
//
// Pair i of a row, (x_i, x_{i + dim / 2}), belongs to axis a(i) and turns by the angle of that axis'
// position p = pos[a(i)][t]: y_i = x_i c - x_{i + dim / 2} s, y_{i + dim / 2} = x_{i + dim / 2} c + x_i s,
// with c and s the table's entries (p, i). One axis is rope_neox, bit for bit.
//
// Bound: HBM, 8 bytes a value in and out. 16000 rows of 32 heads of 128 take 100 us (524 MB, 5.2 TB/s; 85 just
// behind another pass over them), 1027 rows of 16 heads of 72 4.4 to 4.9 (the chain positions -> angles -> rows).
#include "paged.hpp"

namespace brasa {
namespace {

// Two bits for each pair: its axis.
struct AxisMap {
    uint32_t w[8];
    int axes;
};

struct RopeArgs {
    float* x;
    const float* cos_t;
    const float* sin_t;
    const int* pos;  // [axes][tokens]
    AxisMap map;
    int tokens, heads, half, max_pos;  // tokens: of the whole call
    int count;         // tokens of the launch
    int units, spans;  // V-pair units of a row; kSpan-head spans of a token
};

// A row is left as it is where a position is negative, and becomes NaN where one is past the table.
enum RowKind { kTurn, kLeave, kNone };
__device__ __forceinline__ RowKind row_kind(const int* pos, int axes, int tokens, int t, int max_pos) {
    bool leave = false, none = false;
    for (int a = 0; a < axes; ++a) {
        const int p = pos[(size_t)a * tokens + t];
        leave |= p < 0;
        none |= p >= max_pos;
    }
    return leave ? kLeave : none ? kNone : kTurn;
}

// A thread turns V neighbouring pairs of up to kSpan heads of a token, whose angles it loads once. (The rows are
// asked for behind the angles: before them, large calls take 97 us in place of 85.)
constexpr int kSpan = 4;
constexpr int kRopeThreads = 256;
template <int V>
__global__ void __launch_bounds__(kRopeThreads)
rope_axes_kernel(RopeArgs a) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const uint32_t idx = blockIdx.x * kRopeThreads + threadIdx.x;  // (a launch has at most 2^31 of them)
    const uint32_t ts = idx / (uint32_t)a.units;
    const int t = (int)(ts / (uint32_t)a.spans), h0 = (int)(ts % (uint32_t)a.spans) * kSpan;
    if (t >= a.count) return;
    const int i0 = (int)(idx % (uint32_t)a.units) * V;
    const RowKind kind = row_kind(a.pos, a.map.axes, a.tokens, t, a.max_pos);
    if (kind == kLeave) return;
    float c[V], s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = i0 + v, axis = a.map.w[i >> 4] >> 2 * (i & 15) & 3;
        const size_t at = (size_t)(kind == kTurn ? a.pos[(size_t)axis * a.tokens + t] : 0) * a.half + i;
        c[v] = kind == kTurn ? a.cos_t[at] : NAN;
        s[v] = kind == kTurn ? a.sin_t[at] : NAN;
    }
    float* x = a.x + ((size_t)t * a.heads + h0) * (2 * a.half) + i0;
    const int heads = min(a.heads - h0, kSpan);
    vec p[kSpan], q[kSpan];
#pragma unroll
    for (int j = 0; j < kSpan; ++j)
        if (j < heads) {
            p[j] = *reinterpret_cast<const vec*>(x + (size_t)j * 2 * a.half);
            q[j] = *reinterpret_cast<const vec*>(x + (size_t)j * 2 * a.half + a.half);
        }
#pragma unroll
    for (int j = 0; j < kSpan; ++j)
        if (j < heads) {
            vec y, z;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                y[v] = p[j][v] * c[v] - q[j][v] * s[v];
                z[v] = q[j][v] * c[v] + p[j][v] * s[v];
            }
            *reinterpret_cast<vec*>(x + (size_t)j * 2 * a.half) = y;
            *reinterpret_cast<vec*>(x + (size_t)j * 2 * a.half + a.half) = z;
        }
}

// ---- norm, rotation and the paged writer --------------------------------------------------------
//
// A workgroup takes the new rows of one (block, KV head) of K or V, a row per wave and instruction, all
// of them in registers (lane l holds values l and l + 64, a rotary pair and rms_norm's order of sums, so
// q's bits are those of rms_norm and rope_axes in sequence); the workgroups behind them take rows of q.
// Bound: HBM for prompts (5548 rows of 32 + 8 + 8 heads: 242 MB in 51.9 us, 4.7 TB/s; with one row of q a wave in
// place of eight half as long again), the chain lengths -> page -> scale -> codes for a step (64 rows 8.6 us).
constexpr int kWriteWaves = 4;
constexpr int kWriteThreads = 64 * kWriteWaves;
constexpr int kTileRows = kPage / kWriteWaves;  // rows of a block that a wave takes

struct WriteArgs {
    PoolArgs p;  // of one layer
    float* q;
    float* k;
    const float* v;
    const float* qn;
    const float* kn;
    const float* cos_t;
    const float* sin_t;
    const int* rope_pos;  // [axes][tokens]
    AxisMap map;
    NewRows rows;
    float eps;
    int hq, max_pos;
    long long item0;    // first block of the launch
    int t0, spans;      // first token of q; workgroups of a token
    unsigned tiles;     // workgroups that write the cache
};

__device__ __forceinline__ float wave_sum(float p) {
    p = row16_sum(p);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(p), __float_as_int(p), false, false);
    p = __int_as_float(a[0]) + __int_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(p), __float_as_int(p), false, false);
    return __int_as_float(b[0]) + __int_as_float(b[1]);
}

// Rows pass the caches by: 5548 of them in HBM 51.9 us in place of 59.6. (What reads q next finds less of it there: a copy
// of it right behind takes 6 us longer, so 2 are left.)
__device__ __forceinline__ float read_once(const float* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ void write_once(float* p, float x) { __builtin_nontemporal_store(x, p); }

// This lane's angle for row t (NaN where a position is outside the table).
__device__ __forceinline__ void angle_of(const WriteArgs& a, int t, int lane, int axis, float& c, float& s) {
    bool there = true;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < BRASA_ROPE_AXES; ++i)
        if (i < a.map.axes) {
            const int p = scalar(a.rope_pos)[(size_t)i * a.rows.tokens + t];
            there &= p >= 0 && p < a.max_pos;
            mine = i == axis ? p : mine;
        }
    const size_t at = (size_t)(there ? mine : 0) * (kDim / 2) + lane;
    c = a.cos_t[at];
    s = a.sin_t[at];
    if (!there) c = s = NAN;
}
__device__ __forceinline__ void norm_turn(float& x0, float& x1, float w0, float w1, float c, float s, float eps) {
    float p = 0.0f;
    p += x0 * x0;
    p += x1 * x1;
    const float scale = 1.0f / sqrtf(wave_sum(p) / (float)kDim + eps);
    const float a0 = (x0 * scale) * w0, b0 = (x1 * scale) * w1;
    x0 = a0 * c - b0 * s;
    x1 = b0 * c + a0 * s;
}

// A row of k, in 64 bits and rounded once. Its values become codes, and in 32 bits a few of a prompt's (one of 6M, at
// times) came out on the other side of a border between two codes, half a step of the code away. (It takes 1.8 us of 50.)
template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double p) {
    p += dpp64<0x140>(p);
    p += dpp64<0x141>(p);
    p += dpp64<0x1B>(p);
    p += dpp64<0xB1>(p);
    p += __shfl_xor(p, 16);
    p += __shfl_xor(p, 32);
    return p;
}
__device__ __forceinline__ void norm_turn64(float& x0, float& x1, float w0, float w1, float c, float s, float eps) {
    const double m = wave_sum64((double)x0 * x0 + (double)x1 * x1) / kDim + eps;
    double r = __builtin_amdgcn_rsq(m);
    if (r > 0.0 && r < INFINITY) r = fma(r, 0.5 * fma(-m * r, r, 1.0), r);  // (a Newton step: the instruction has 2^-26)
    const double a0 = x0 * r * w0, b0 = x1 * r * w1;
    x0 = (float)(a0 * c - b0 * s);
    x1 = (float)(b0 * c + a0 * s);
}

constexpr int kRows = 8;  // of q for each wave, of one token, whose loads travel together
__global__ void __launch_bounds__(kWriteThreads, 5)
norm_rope_paged_kernel(WriteArgs a) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int axis = a.map.w[lane >> 4] >> 2 * (lane & 15) & 3;
    if (blockIdx.x >= a.tiles) {
        // ---- q: heads h0 .. of token t --------------------------------------------------------------
        const int first = min(max(scalar(a.rows.cu)[0], 0), a.rows.tokens);
        const int last = min(max(scalar(a.rows.cu)[a.rows.n], first), a.rows.tokens);
        const unsigned unit = blockIdx.x - a.tiles;
        const int t = a.t0 + (int)(unit / a.spans), h0 = ((int)(unit % a.spans) * kWriteWaves + wave) * kRows;
        if (t < first || t >= last || h0 >= a.hq) return;
        float* q = a.q + ((size_t)t * a.hq + h0) * kDim + lane;
        float x0[kRows], x1[kRows], c, s;
        const int rows = min(a.hq - h0, kRows);
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int r = min(j, rows - 1);
            x0[j] = read_once(q + r * kDim);
            x1[j] = read_once(q + r * kDim + 64);
        }
        angle_of(a, t, lane, axis, c, s);
        const float w0 = a.qn[lane], w1 = a.qn[lane + 64];
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            if (j >= rows) break;
            norm_turn(x0[j], x1[j], w0, w1, c, s, a.eps);
            write_once(q + j * kDim, x0[j]);
            write_once(q + j * kDim + 64, x1[j]);
        }
        return;
    }
    // ---- a block of K or V --------------------------------------------------------------------------
    const int kh = blockIdx.x / 2 % a.p.hkv;
    const bool is_v = blockIdx.x & 1;
    TouchedBlock t;
    if (!touched_block<true>(a.rows, (int)(a.item0 + blockIdx.x / 2 / a.p.hkv), a.p.pages, t)) return;
    const int s0 = t.s0, s1 = t.s1;
    const size_t tile = (size_t)t.page * a.p.hkv + kh;
    uint8_t* codes = (is_v ? a.p.v : a.p.k) + tile * kTileBytes8;
    uint8_t* scale = (is_v ? a.p.vx : a.p.kx) + tile;
    const int old = s0 > 0 ? *scale : 0;
    // this block's rows (slot 0's may lie before the first): 32-bit offsets from there
    const ptrdiff_t row0 = ((ptrdiff_t)t.row0 * a.p.hkv + kh) * kDim;
    const float* src = (is_v ? a.v : a.k) + row0;
    float* dst = a.k + row0;
    auto row_at = [&](int s) { return s * a.p.hkv * kDim + lane; };
    float x0[kTileRows], x1[kTileRows];
    float amax = 0.0f;
    auto take = [&](float y0, float y1) {  // NaN and inf take no part in the scale
        const float m0 = fabsf(y0), m1 = fabsf(y1);
        amax = fmaxf(amax, fmaxf(m0 < INFINITY ? m0 : 0.0f, m1 < INFINITY ? m1 : 0.0f));
    };
#pragma unroll
    for (int j = 0; j < kTileRows; ++j) {
        const int s = kWriteWaves * j + wave;
        x0[j] = x1[j] = 0.0f;
        if (s >= s0 && s < s1) {
            x0[j] = read_once(src + row_at(s));
            x1[j] = read_once(src + row_at(s) + 64);
        }
    }
    if (!is_v) {
        const float w0 = a.kn[lane], w1 = a.kn[lane + 64];
        constexpr int kAhead = 4;  // rows whose angles are on their way together
#pragma unroll
        for (int j0 = 0; j0 < kTileRows; j0 += kAhead) {
            if (kWriteWaves * (j0 + kAhead) <= s0 || kWriteWaves * j0 >= s1) continue;
            float c[kAhead], sn[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int s = min(max(kWriteWaves * (j0 + j) + wave, s0), s1 - 1);
                angle_of(a, t.row0 + s, lane, axis, c[j], sn[j]);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int s = kWriteWaves * (j0 + j) + wave;
                if (s < s0 || s >= s1) continue;
                norm_turn64(x0[j0 + j], x1[j0 + j], w0, w1, c[j], sn[j], a.eps);
                write_once(dst + row_at(s), x0[j0 + j]);
                write_once(dst + row_at(s) + 64, x1[j0 + j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kTileRows; ++j) take(x0[j], x1[j]);
    __shared__ float s_max[kWriteWaves];
    __shared__ __attribute__((aligned(16))) uint8_t s_codes[kTileBytes8];
#pragma unroll
    for (int d = 32; d; d /= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
    if (lane == 0) s_max[wave] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWriteWaves; ++w) amax = fmaxf(amax, s_max[w]);
    const int ex = max(e4m3_scale(amax), old);
    if (s0 > 0 && ex > old) rescale_rows<kWriteThreads>(codes, s0, old - ex);
    // through LDS, so that the codes leave as whole pieces of 16 bytes
#pragma unroll
    for (int j = 0; j < kTileRows; j += 2) {
        const int s = kWriteWaves * j + wave;
        if (s + kWriteWaves < s0 || s >= s1) continue;
        const float y[4] = {x0[j], x1[j], x0[j + 1], x1[j + 1]};
        const uint32_t w = e4m3_quad(y, 127 - ex);
        uint8_t* to = s_codes + s * kDim + lane;
        to[0] = (uint8_t)w;
        to[64] = (uint8_t)(w >> 8);
        to[kWriteWaves * kDim] = (uint8_t)(w >> 16);
        to[kWriteWaves * kDim + 64] = (uint8_t)(w >> 24);
    }
    __syncthreads();
    for (int i = s0 * (kDim / 16) + (int)threadIdx.x; i < s1 * (kDim / 16); i += kWriteThreads)
        reinterpret_cast<u32x4*>(codes)[i] = reinterpret_cast<const u32x4*>(s_codes)[i];
    // (every thread that needed the old scale has read it before the barriers above)
    if (threadIdx.x == 0) *scale = (uint8_t)ex;
}

AxisMap pack_axes(const brasa_rope_axes_map& m, int half) {
    AxisMap out = {};
    out.axes = (int)m.axes;
    for (int i = 0; i < half; ++i) out.w[i >> 4] |= (uint32_t)m.of[i] << 2 * (i & 15);
    return out;
}

template <int V>
int launch_rope(RopeArgs a, hipStream_t stream) {
    a.units = a.half / V;
    a.spans = (a.heads + kSpan - 1) / kSpan;
    // A launch of 2^32 threads or more runs fewer, without an error: whole tokens of at most 2^31 in each.
    const long long per_token = (long long)a.units * a.spans;
    const int most = (int)std::min((1LL << 31) / per_token - 1, (long long)a.tokens);
    const int tokens = a.tokens;
    for (int t0 = 0; t0 < tokens; t0 += most) {
        RopeArgs b = a;
        const int count = std::min(tokens - t0, most);
        b.x = a.x + (size_t)t0 * a.heads * 2 * a.half;
        b.pos = a.pos + t0;
        b.count = count;
        const long long threads = per_token * count;
        hipLaunchKernelGGL(rope_axes_kernel<V>, dim3((unsigned)((threads + kRopeThreads - 1) / kRopeThreads)),
                           dim3(kRopeThreads), 0, stream, b);
        const int st = check_launch("rope_axes_kernel");
        if (st != BRASA_OK) return st;
    }
    return BRASA_OK;
}

}  // namespace

int rope_axes_launch(float* x, const float* cos_t, const float* sin_t, int max_pos,
                     const brasa_rope_axes_map& map, const int* pos, int tokens, int heads, int dim,
                     hipStream_t stream) {
    RopeArgs a = {};
    a.x = x;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.pos = pos;
    a.map = pack_axes(map, dim / 2);
    a.tokens = tokens;
    a.heads = heads;
    a.half = dim / 2;
    a.max_pos = max_pos;
    // Four pairs a thread, 16 bytes an access, for large calls: 67M values that HBM holds in 100 us, a pair a thread 110; 16.8M
    // 30.6 and 31.3, 10.2M 21.3 and 22.4. Small ones want the threads: 8.4M 19.1 and 18.4, 4.1M 10.7 and 9.8. (Two
    // times the same rows, which the caches then hold: 67M 87 and 110, 16.8M 26.0 and 26.8, 8.4M 12.2 and 14.5, 4.1M 7.8 and 7.6.)
    if (a.half % 4 == 0 && (uintptr_t)x % 16 == 0 && (long long)tokens * heads * dim > (1LL << 23))
        return launch_rope<4>(a, stream);
    return launch_rope<1>(a, stream);
}

int norm_rope_paged_launch(const PoolArgs& pool, float* q, float* k, const float* v, const float* qn,
                           const float* kn, float eps, const float* cos_t, const float* sin_t, int max_pos,
                           const brasa_rope_axes_map& map, const int* rope_pos, const int* cu, const int* pos,
                           const int* table, int n, int width, int tokens, int hq, hipStream_t stream) {
    WriteArgs a = {};
    a.p = pool;
    a.q = q;
    a.k = k;
    a.v = v;
    a.qn = qn;
    a.kn = kn;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.rope_pos = rope_pos;
    a.map = pack_axes(map, kDim / 2);
    a.rows = {cu, pos, table, n, width, tokens};
    a.eps = eps;
    a.hq = hq;
    a.max_pos = max_pos;
    const long long items = width ? most_blocks(n, tokens) : 0;
    a.spans = (hq + kWriteWaves * kRows - 1) / (kWriteWaves * kRows);
    // A launch of 2^32 threads or more runs fewer, without an error: at most 2^30 of each kind in each.
    const long long most = (1LL << 30) / kWriteThreads / (2 * pool.hkv);
    const long long most_q = a.spans ? (1LL << 30) / kWriteThreads / a.spans : tokens;
    for (long long i = 0, t = 0; i < items || t < tokens; i += most, t += most_q) {
        a.item0 = i;
        a.t0 = (int)t;
        a.tiles = (unsigned)(std::min(std::max(items - i, 0LL), most) * 2 * pool.hkv);
        const unsigned more = (unsigned)(std::min(std::max(tokens - t, 0LL), most_q) * a.spans);
        if (a.tiles + more == 0) break;
        hipLaunchKernelGGL(norm_rope_paged_kernel, dim3(a.tiles + more), dim3(kWriteThreads), 0, stream, a);
        const int st = check_launch("norm_rope_paged_kernel");
        if (st != BRASA_OK) return st;
    }
    return BRASA_OK;
}

}  // namespace brasa
