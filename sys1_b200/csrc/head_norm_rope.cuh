// Per-head RMSNorm followed by the partial rotate-half rotation, on one head row held by LPR lanes (8 bf16 values each):
// the arithmetic that s1_head_norm_rope applies in place and s1_cache_write applies on the way into the cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace s1 {

__device__ __forceinline__ void unpack8(const uint4& raw, float* f) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 t = __bfloat1622float2(h[e]);
        f[2 * e] = t.x;
        f[2 * e + 1] = t.y;
    }
}

__device__ __forceinline__ uint4 pack8(const float* f) {
    uint4 raw;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
    return raw;
}

__device__ __forceinline__ float bf16r(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// The cosines and sines of lane `sub` of a head (its 8 columns of the rotated span, `rot / 16` lanes to each half).
__device__ __forceinline__ void load_rotation(const float* cos_t, const float* sin_t, int pos, int rot, int sub, float (&c)[8], float (&sn)[8]) {
    const long long tb = static_cast<long long>(pos) * (rot / 2) + (sub & (rot / 16 - 1)) * 8;  // rot / 16 is a power of two
    *reinterpret_cast<float4*>(c) = __ldg(reinterpret_cast<const float4*>(cos_t + tb));
    *reinterpret_cast<float4*>(c + 4) = __ldg(reinterpret_cast<const float4*>(cos_t + tb) + 1);
    *reinterpret_cast<float4*>(sn) = __ldg(reinterpret_cast<const float4*>(sin_t + tb));
    *reinterpret_cast<float4*>(sn + 4) = __ldg(reinterpret_cast<const float4*>(sin_t + tb) + 1);
}

// bf16(x / sqrt(mean(x^2) + eps) * (1 + w)) over the 8 * LPR columns of the head, then the rotation of its first `16 * halfc`
// columns where `rotate`. bf16_ops = 1: each product and the sum are bf16 values (src/archs/qwen35_text.rs:302); 0: products and
// sum in f32, rounded once. Every lane of the warp takes part in the exchanges, also those without a live row.
template <int LPR>
__device__ __forceinline__ uint4 head_norm_rope(const uint4& raw, const __nv_bfloat16* w, float eps, const float (&c)[8], const float (&sn)[8],
                                                bool rotate, int sub, int halfc, int bf16_ops) {
    float f[8];
    unpack8(raw, f);
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sq += f[e] * f[e];
    const float rstd = 1.f / sqrtf(group_sum<LPR>(sq) * (1.f / static_cast<float>(8 * LPR)) + eps);
    float g[8];
    unpack8(__ldg(reinterpret_cast<const uint4*>(w + sub * 8)), g);
    uint4 normed;
    {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = f[e] * rstd * (g[e] + 1.f);
        normed = pack8(y);
        unpack8(normed, f);  // the bf16 values the rotation starts from
    }
    // the partner half of the rotated span sits rot / 16 lanes away
    uint4 other_raw;
    other_raw.x = __shfl_xor_sync(0xffffffffu, normed.x, halfc);
    other_raw.y = __shfl_xor_sync(0xffffffffu, normed.y, halfc);
    other_raw.z = __shfl_xor_sync(0xffffffffu, normed.z, halfc);
    other_raw.w = __shfl_xor_sync(0xffffffffu, normed.w, halfc);
    if (rotate) {
        float o[8];
        unpack8(other_raw, o);
        const bool is_lo = sub < halfc;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float own_c = __fmul_rn(f[e], c[e]);
            const float oth_s = __fmul_rn(is_lo ? -o[e] : o[e], sn[e]);  // rotate_half = [-second, first]
            if (bf16_ops) f[e] = __fadd_rn(bf16r(own_c), bf16r(oth_s));
            else f[e] = is_lo ? __fsub_rn(own_c, __fmul_rn(o[e], sn[e])) : __fadd_rn(__fmul_rn(o[e], sn[e]), own_c);
        }
        normed = pack8(f);
    }
    return normed;
}

}  // namespace s1
