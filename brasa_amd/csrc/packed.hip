// Causal attention over packed prompts.
#include "paged.hpp"

namespace brasa {
namespace {

struct PackedArgs {
    const float* q;
    const uint8_t* k;
    const uint8_t* v;
    void* o;
    const int* cu;
    int n, tokens, hq, hkv, group;
    float scale;
};

template <int KV>
__device__ __forceinline__ f32x2 packed_pair(const uint8_t* rows, size_t row, int d) {
    if constexpr (KV == BRASA_KV_F32) return *reinterpret_cast<const f32x2*>(rows + row * 512 + 4 * d);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(rows + row * 256 + 2 * d);
    return f32x2{h2f(w & 0xffff), h2f(w >> 16)};
}

// One wave per query row and head, one key per step.
template <int KV, bool F16>
__global__ void __launch_bounds__(256)
packed_simple_kernel(PackedArgs a) {
    const int lane = threadIdx.x & 63;
    const int rw = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = rw / a.hq, h = rw % a.hq;
    if (t >= a.tokens) return;
    int start = -1;
    for (int i0 = 0; i0 < a.n; i0 += 64) {
        const int i = i0 + lane;
        const bool in = i < a.n && a.cu[i] <= t && t < a.cu[i + 1];
        const unsigned long long b = __builtin_amdgcn_ballot_w64(in);
        if (b) {
            start = max(a.cu[i0 + __builtin_ctzll(b)], 0);
            break;
        }
    }
    if (start < 0) return;
    const int kh = h / a.group;
    f32x2 q = reinterpret_cast<const f32x2*>(a.q + (size_t)rw * kDim)[lane];
    q.x = as_f32(q.x * a.scale);
    q.y = as_f32(q.y * a.scale);
    if (F16) q = f32x2{h2f(f2h(q.x)), h2f(f2h(q.y))};
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j = start; j <= t; ++j) {
        const f32x2 k = packed_pair<KV>(a.k, (size_t)j * a.hkv + kh, 2 * lane);
        float s = fmaf(q.x, k.x, q.y * k.y);
#pragma unroll
        for (int d = 32; d; d /= 2) s += __shfl_xor(s, d);
        const float mn = fmaxf(m, s);
        const float f = expf(m - mn), p = expf(s - mn);
        const f32x2 v = packed_pair<KV>(a.v, (size_t)j * a.hkv + kh, 2 * lane);
        l = fmaf(l, f, p);
        o0 = fmaf(o0, f, p * v.x);
        o1 = fmaf(o1, f, p * v.y);
        m = mn;
    }
    o0 /= l;
    o1 /= l;
    if (F16) reinterpret_cast<uint32_t*>(a.o)[(size_t)rw * 64 + lane] = f2h(o0) | (uint32_t)f2h(o1) << 16;
    else reinterpret_cast<f32x2*>(a.o)[(size_t)rw * 64 + lane] = f32x2{o0, o1};
}

}  // namespace

int packed_launch(const float* q, const void* k, const void* v, void* o, const int* cu, int n, int tokens,
                  int hq, int hkv, int kv, int precision, hipStream_t stream) {
    PackedArgs a{q, static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), o, cu, n, tokens, hq, hkv,
                 hq / hkv, 1.0f / sqrtf((float)kDim)};
    const dim3 grid((unsigned)(((long long)tokens * hq + 3) / 4));
    const bool f16 = precision != BRASA_PREFILL_F32;
    if (kv == BRASA_KV_F16 && f16)
        hipLaunchKernelGGL((packed_simple_kernel<BRASA_KV_F16, true>), grid, dim3(256), 0, stream, a);
    else if (kv == BRASA_KV_F16)
        hipLaunchKernelGGL((packed_simple_kernel<BRASA_KV_F16, false>), grid, dim3(256), 0, stream, a);
    else if (f16)
        hipLaunchKernelGGL((packed_simple_kernel<BRASA_KV_F32, true>), grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((packed_simple_kernel<BRASA_KV_F32, false>), grid, dim3(256), 0, stream, a);
    return check_launch("packed_simple_kernel");
}

}  // namespace brasa
