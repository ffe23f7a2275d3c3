// The gated delta rule one token further, on a state that is carried from call to call: everything between a linear-attention
// layer's input projections and its output projection (src/archs/qwen35_text.rs:491-626) for one new token of each row, as one kernel:
//     u    = silu(sum_{back < 4} w[c, 3 - back] x_{t - back}[c])                 causal depthwise conv over the new row and a ring of past ones
//     q, k = l2norm of u's query and key heads (q / sqrt(128)),  v = u's value heads,  beta = sigmoid(b),  g = softplus(a + dt_bias) * neg_exp_a
//     S <- e^g S;  d = beta (v - S^T k);  S <- S + k d^T;  o = S^T q;  y = o / sqrt(mean(o^2) + eps) * w * silu(z)
// What bounds it: S, 128 x 128 f32 per row and value head, is read once and written once (128 KB a row and head, against 7 flops an
// element) - HBM. A block holds one S in registers, thread (warp w, lane l) columns 4 l .. 4 l + 3 of the key rows w, w + 16, ...: all
// of it is requested before the conv and the norms are formed, so these run while it is on its way. With
//     S^T k and S^T q taken over the old S,   o = e^g (S^T q) + d (k . q),
// both sums over the key rows come from the same pass and one exchange between the warps, and S leaves as it is updated.
// Sums, norms and state are f32 throughout (the prompt form rounds the conv tap by tap to bf16, as the reference's kernel does; a
// step keeps it in f32). The conv's history is a ring of four rows by position mod 4: the new row's place is one that no conv of
// this step reads, so the blocks of a row need not wait for one another.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "context.h"
#include "device_guard.h"

namespace {

constexpr int kDim = 128;
constexpr int kTaps = 4;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kRows = kDim / kWarps;  // key rows a thread holds

struct StepParams {
    const __nv_bfloat16* mixed;
    long long ldm;
    const __nv_bfloat16* conv_w;  // [C, 4]
    const int32_t* positions;
    const __nv_bfloat16* b;
    const __nv_bfloat16* a;
    long long ldba;
    const float* dt_bias;
    const float* neg_exp_a;
    const __nv_bfloat16* z;
    long long ldz;
    const __nv_bfloat16* norm_w;
    float eps;
    const int32_t* index;
    int num_states, num_seqs;
    __nv_bfloat16* conv_state;  // [num_states, 4, C]
    float* state;               // [num_states, value_heads, 128 (key), 128 (value)]
    int key_heads, value_heads;
    __nv_bfloat16* y;
    long long ldy;
    int* status;
};

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__global__ void __launch_bounds__(kThreads, 2) s1_delta_step_kernel(const StepParams p) {
    __shared__ float u[3][kDim];                 // conv outputs of the head: q, k, v
    __shared__ float part_k[kWarps][kDim], part_q[kWarps][kDim];
    __shared__ float norms[3][4];
    const int row = blockIdx.x / p.value_heads, head = blockIdx.x % p.value_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int slot = p.index ? __ldg(p.index + row) : row;
    __nv_bfloat16* y = p.y + row * p.ldy + head * kDim;
    // an idle row, or a slot that does not exist or that a row before this one has: no state is touched, the output is zero
    bool bad = slot >= p.num_states;
    if (p.index && slot >= 0 && !bad)
        for (int j = tid; j < row; j += kThreads) bad = bad || __ldg(p.index + j) == slot;
    const int pos = slot >= 0 ? __ldg(p.positions + row) : 0;
    bad = bad || pos < 0;
    bad = __syncthreads_or(bad);
    if (slot < 0 || bad) {
        if (tid < kDim) y[tid] = __float2bfloat16_rn(0.f);
        if (bad && tid == 0 && atomicCAS(p.status, 0, pos < 0 ? 120 : 119) == 0) {
            p.status[1] = static_cast<int>(blockIdx.x);
            p.status[2] = row;
            p.status[3] = pos < 0 ? pos : slot;
        }
        return;
    }
    // ---- the state is on its way first
    float* state = p.state + (static_cast<long long>(slot) * p.value_heads + head) * (kDim * kDim) + 4 * lane;
    float4 S[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)  // a sequence's first token starts from zero, whatever the slot held before
        S[i] = pos > 0 ? *reinterpret_cast<const float4*>(state + (warp + kWarps * i) * kDim) : make_float4(0.f, 0.f, 0.f, 0.f);
    // ---- conv + SiLU of this head's 384 channels
    const int share = p.value_heads / p.key_heads, kh = head / share;
    if (tid < 3 * kDim) {
        const int which = tid / kDim, c = which * p.key_heads * kDim + (which == 2 ? head : kh) * kDim + tid % kDim;
        const long long C = static_cast<long long>(2 * p.key_heads + p.value_heads) * kDim;
        const __nv_bfloat16 x = p.mixed[row * p.ldm + c];
        __nv_bfloat16* ring = p.conv_state + slot * kTaps * C + c;
        const uint2 wraw = __ldg(reinterpret_cast<const uint2*>(p.conv_w + static_cast<long long>(c) * kTaps));
        const __nv_bfloat162 w01 = *reinterpret_cast<const __nv_bfloat162*>(&wraw.x), w23 = *reinterpret_cast<const __nv_bfloat162*>(&wraw.y);
        float past[kTaps - 1];
#pragma unroll
        for (int back = 1; back < kTaps; ++back) past[back - 1] = back <= pos ? __bfloat162float(ring[((pos - back) & 3) * C]) : 0.f;
        float s = __bfloat162float(x) * __high2float(w23);
        s = fmaf(past[0], __low2float(w23), s);
        s = fmaf(past[1], __high2float(w01), s);
        s = fmaf(past[2], __low2float(w01), s);
        s *= sigmoid(s);
        u[which][tid % kDim] = s;
        const float sq = warp_sum(s * s);
        if (lane == 0) norms[which][warp & 3] = sq;
        if (which == 2 || head % share == 0) ring[(pos & 3) * C] = x;  // the query and key channels once for the heads that share them
    }
    __syncthreads();
    const float rq = 0.08838834764831845f / sqrtf(norms[0][0] + norms[0][1] + norms[0][2] + norms[0][3] + 1e-6f);  // 128^-1/2 / |q|
    const float rk = 1.f / sqrtf(norms[1][0] + norms[1][1] + norms[1][2] + norms[1][3] + 1e-6f);
    const float beta = sigmoid(__bfloat162float(p.b[row * p.ldba + head]));
    const float f = __bfloat162float(p.a[row * p.ldba + head]) + p.dt_bias[head];
    const float keep = expf((fmaxf(f, 0.f) + log1pf(expf(-fabsf(f)))) * p.neg_exp_a[head]);
    const float kq = warp_sum(u[0][lane] * u[1][lane] + u[0][lane + 32] * u[1][lane + 32] + u[0][lane + 64] * u[1][lane + 64] +
                              u[0][lane + 96] * u[1][lane + 96]) * rq * rk;
    // ---- S^T k and S^T q over this thread's key rows, then over the warps
    float4 sk = make_float4(0.f, 0.f, 0.f, 0.f), sq = sk;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const float kk = u[1][warp + kWarps * i] * rk, qq = u[0][warp + kWarps * i] * rq;
        sk.x = fmaf(S[i].x, kk, sk.x), sk.y = fmaf(S[i].y, kk, sk.y), sk.z = fmaf(S[i].z, kk, sk.z), sk.w = fmaf(S[i].w, kk, sk.w);
        sq.x = fmaf(S[i].x, qq, sq.x), sq.y = fmaf(S[i].y, qq, sq.y), sq.z = fmaf(S[i].z, qq, sq.z), sq.w = fmaf(S[i].w, qq, sq.w);
    }
    *reinterpret_cast<float4*>(&part_k[warp][4 * lane]) = sk;
    *reinterpret_cast<float4*>(&part_q[warp][4 * lane]) = sq;
    __syncthreads();
    sk = sq = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&part_k[w][4 * lane]), v = *reinterpret_cast<const float4*>(&part_q[w][4 * lane]);
        sk.x += x.x, sk.y += x.y, sk.z += x.z, sk.w += x.w;
        sq.x += v.x, sq.y += v.y, sq.z += v.z, sq.w += v.w;
    }
    const float4 v = *reinterpret_cast<const float4*>(&u[2][4 * lane]);
    const float4 d = make_float4(beta * (v.x - keep * sk.x), beta * (v.y - keep * sk.y), beta * (v.z - keep * sk.z), beta * (v.w - keep * sk.w));
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const float kk = u[1][warp + kWarps * i] * rk;
        *reinterpret_cast<float4*>(state + (warp + kWarps * i) * kDim) =
            make_float4(fmaf(kk, d.x, keep * S[i].x), fmaf(kk, d.y, keep * S[i].y), fmaf(kk, d.z, keep * S[i].z), fmaf(kk, d.w, keep * S[i].w));
    }
    if (warp == 0) {
        const float o[4] = {fmaf(d.x, kq, keep * sq.x), fmaf(d.y, kq, keep * sq.y), fmaf(d.z, kq, keep * sq.z), fmaf(d.w, kq, keep * sq.w)};
        const float r = 1.f / sqrtf(warp_sum(o[0] * o[0] + o[1] * o[1] + o[2] * o[2] + o[3] * o[3]) * (1.f / kDim) + p.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float zz = __bfloat162float(p.z[row * p.ldz + head * kDim + 4 * lane + e]);
            y[4 * lane + e] = __float2bfloat16_rn(o[e] * r * __bfloat162float(p.norm_w[4 * lane + e]) * zz * sigmoid(zz));
        }
    }
}

// The last rows before the conv of every sequence of a prompt batch into the ring that the step kernel reads.
__global__ void __launch_bounds__(256) s1_conv_state_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, const int32_t* __restrict__ cu,
                                                            const int32_t* __restrict__ index, int num_states, int C, __nv_bfloat16* __restrict__ ring) {
    const int s = blockIdx.x, back = blockIdx.y;  // the token `back` before the sequence's last
    const int slot = index[s], a = cu[s], len = cu[s + 1] - a;
    // a slot that does not exist, or that a sequence before this one has, is left alone, like the state (delta_chunked.cu reports it)
    bool bad = slot >= num_states;
    for (int j = threadIdx.x; slot >= 0 && j < s; j += 256) bad = bad || (index[j] == slot && cu[j + 1] > cu[j]);
    bad = __syncthreads_or(bad);
    if (slot < 0 || bad || back >= len) return;
    const int pos = len - 1 - back;
    const uint4* src = reinterpret_cast<const uint4*>(x + (a + pos) * ldx);
    uint4* dst = reinterpret_cast<uint4*>(ring + (static_cast<long long>(slot) * kTaps + (pos & 3)) * C);
    for (int i = threadIdx.x; i < C / 8; i += 256) dst[i] = __ldg(src + i);
}

inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

int s1_conv_state_launch(s1_ctx* ctx, const void* mixed, long long ldm, const int32_t* cu_seqlens, int num_seqs, const int32_t* index, int num_states,
                         int channels, void* conv_state) {
    s1_conv_state_kernel<<<dim3(num_seqs, kTaps), 256, 0, ctx->stream>>>(static_cast<const __nv_bfloat16*>(mixed), ldm, cu_seqlens, index, num_states,
                                                                         channels, static_cast<__nv_bfloat16*>(conv_state));
    S1_CUDA_OK(ctx, cudaGetLastError());
    ctx->launches += 1;
    return S1_OK;
}

extern "C" int s1_gated_delta_rule_step(s1_ctx* ctx, const void* mixed, long long ldm, const void* conv_weight, const int32_t* positions,
                                        const void* b_proj, const void* a_proj, long long ldba, const float* dt_bias, const float* neg_exp_a,
                                        const void* z, long long ldz, const void* norm_weight, float eps, const int32_t* state_index, int num_states,
                                        void* conv_state, float* state, int num_seqs, int key_heads, int value_heads, void* y, long long ldy) {
    if (!ctx) return S1_EINVAL;
    const char* who = "s1_gated_delta_rule_step";
    if (!mixed || !conv_weight || !positions || !b_proj || !a_proj || !dt_bias || !neg_exp_a || !z || !norm_weight || !conv_state || !state || !y)
        return s1_fail(ctx, S1_EINVAL, "%s: null pointer", who);
    if (key_heads < 1 || value_heads < key_heads || value_heads % key_heads)
        return s1_fail(ctx, S1_EINVAL, "%s: value_heads must be a multiple of key_heads", who);
    if (num_seqs < 0 || num_states < 1 || (!state_index && num_states < num_seqs))
        return s1_fail(ctx, S1_EINVAL, "%s: %d rows, %d states", who, num_seqs, num_states);
    const long long width = (2LL * key_heads + value_heads) * kDim, out = static_cast<long long>(value_heads) * kDim;
    if (ldm < width || ldba < value_heads || ldz < out || ldy < out)
        return s1_fail(ctx, S1_EINVAL, "%s: mixed needs %lld columns per row, z and y %lld", who, width, out);
    if (!aligned(conv_weight, 8) || !aligned(conv_state, 16) || !aligned(state, 16))
        return s1_fail(ctx, S1_EINVAL, "%s: the states must be 16-byte aligned, the conv weight 8-byte", who);
    const long long blocks = static_cast<long long>(num_seqs) * value_heads;
    if (blocks > 2147483647LL) return s1_fail(ctx, S1_EINVAL, "%s: too many rows", who);
    if (num_seqs == 0) return S1_OK;
    S1DeviceGuard guard(ctx->device);
    if (!guard.ok) return s1_fail(ctx, S1_ECUDA, "%s: cudaSetDevice(%d) failed", who, ctx->device);
    StepParams p{static_cast<const __nv_bfloat16*>(mixed), ldm, static_cast<const __nv_bfloat16*>(conv_weight), positions,
                 static_cast<const __nv_bfloat16*>(b_proj), static_cast<const __nv_bfloat16*>(a_proj), ldba, dt_bias, neg_exp_a,
                 static_cast<const __nv_bfloat16*>(z), ldz, static_cast<const __nv_bfloat16*>(norm_weight), eps, state_index, num_states, num_seqs,
                 static_cast<__nv_bfloat16*>(conv_state), state, key_heads, value_heads, static_cast<__nv_bfloat16*>(y), ldy, ctx->status_dev};
    s1_delta_step_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, ctx->stream>>>(p);
    S1_CUDA_OK(ctx, cudaGetLastError());
    ctx->launches += 1;
    return S1_OK;
}
