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

// Weights and tables: by the read-only path where the kernel is launched after its operands are complete (FIXED), by plain loads where it
// may be resident before (the read-only path says that the data does not change in the kernel's life, so that the compiler may move such a
// load ahead of the wait for the kernel before).
template <bool FIXED, typename T>
__device__ __forceinline__ T operand(const T* p) {
    return FIXED ? __ldg(p) : *p;
}

// The cosines and sines of lane `sub` of a head (its 8 columns of the rotated span, `rot / 16` lanes to each half).
template <bool FIXED>
__device__ __forceinline__ void load_rotation(const float* cos_t, const float* sin_t, int pos, int rot, int sub, float (&c)[8], float (&sn)[8]) {
    const long long tb = static_cast<long long>(pos) * (rot / 2) + (sub & (rot / 16 - 1)) * 8;  // rot / 16 is a power of two
    *reinterpret_cast<float4*>(c) = operand<FIXED>(reinterpret_cast<const float4*>(cos_t + tb));
    *reinterpret_cast<float4*>(c + 4) = operand<FIXED>(reinterpret_cast<const float4*>(cos_t + tb) + 1);
    *reinterpret_cast<float4*>(sn) = operand<FIXED>(reinterpret_cast<const float4*>(sin_t + tb));
    *reinterpret_cast<float4*>(sn + 4) = operand<FIXED>(reinterpret_cast<const float4*>(sin_t + tb) + 1);
}

// The steps of bf16(x / sqrt(mean(x^2) + eps) * (1 + w)) and of the rotation, on 8 columns.
__device__ __forceinline__ float sum_squares8(const uint4& raw) {
    float f[8], sq = 0.f;
    unpack8(raw, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) sq += f[e] * f[e];
    return sq;
}
__device__ __forceinline__ uint4 norm8(const uint4& raw, float rstd, const uint4& w) {
    float f[8], g[8], y[8];
    unpack8(raw, f);
    unpack8(w, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = f[e] * rstd * (g[e] + 1.f);
    return pack8(y);
}
// `normed` (the bf16 values the rotation starts from) and the same columns of the other half of the rotated span
__device__ __forceinline__ uint4 rotate8(const uint4& normed, const uint4& other, const float (&c)[8], const float (&sn)[8], bool is_lo, int bf16_ops) {
    float f[8], o[8];
    unpack8(normed, f);
    unpack8(other, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float own_c = __fmul_rn(f[e], c[e]);
        const float oth_s = __fmul_rn(o[e], is_lo ? -sn[e] : sn[e]);  // rotate_half = [-second, first]
        f[e] = bf16_ops ? __fadd_rn(bf16r(own_c), bf16r(oth_s)) : __fadd_rn(own_c, oth_s);
    }
    return pack8(f);
}
__device__ __forceinline__ uint4 shfl_xor4(const uint4& v, int mask) {
    return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, mask), __shfl_xor_sync(0xffffffffu, v.y, mask), __shfl_xor_sync(0xffffffffu, v.z, mask),
                      __shfl_xor_sync(0xffffffffu, v.w, mask));
}

// bf16(x / sqrt(mean(x^2) + eps) * (1 + w)) over the 8 * LPR columns of the head, then the rotation of its first `16 * halfc`
// columns where `rotate`. The rotation starts from the norm rounded to bf16, as the norm's own output is in the reference and in
// s1_norm followed by s1_rope, whose bits these are (2^-8 of a value more than one rounding in all). bf16_ops = 1: each product and the sum are bf16 values (src/archs/qwen35_text.rs:302); 0: products and
// sum in f32, rounded once. Every lane of the warp takes part in the exchanges, also those without a live row.
template <int LPR>
__device__ __forceinline__ uint4 head_norm_rope(const uint4& raw, const __nv_bfloat16* w, float eps, const float (&c)[8], const float (&sn)[8],
                                                bool rotate, int sub, int halfc, int bf16_ops) {
    const float rstd = 1.f / sqrtf(group_sum<LPR>(sum_squares8(raw)) * (1.f / static_cast<float>(8 * LPR)) + eps);
    const uint4 normed = norm8(raw, rstd, operand<true>(reinterpret_cast<const uint4*>(w + sub * 8)));
    const uint4 other = shfl_xor4(normed, halfc);  // the partner half of the rotated span sits rot / 16 lanes away
    return rotate ? rotate8(normed, other, c, sn, sub < halfc, bf16_ops) : normed;
}

// The same for a lane that holds columns 8 sub .. and 8 (sub + LPR) .. of a head of 16 LPR columns: the sum over the head adds up in the
// same order (the two pieces first), so the results are the same bits, for half the exchanges and square roots.
template <int LPR>
__device__ __forceinline__ void head_norm_rope(uint4 (&x)[2], const __nv_bfloat16* w, float eps, const float (&c)[8], const float (&sn)[8], bool rotate,
                                               int sub, int halfc, int bf16_ops) {
    const float rstd = 1.f / sqrtf(group_sum<LPR>(sum_squares8(x[0]) + sum_squares8(x[1])) * (1.f / static_cast<float>(16 * LPR)) + eps);
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = norm8(x[i], rstd, operand<false>(reinterpret_cast<const uint4*>(w + (sub + i * LPR) * 8)));
    if (halfc == LPR) {  // the whole head is rotated: a lane's pieces are each other's partners
        const uint4 lo = x[0], hi = x[1];
        if (rotate) x[0] = rotate8(lo, hi, c, sn, true, bf16_ops), x[1] = rotate8(hi, lo, c, sn, false, bf16_ops);
    } else {             // the rotated span ends inside the first pieces
        const uint4 other = shfl_xor4(x[0], halfc);
        if (rotate) x[0] = rotate8(x[0], other, c, sn, sub < halfc, bf16_ops);
    }
}

}  // namespace s1
