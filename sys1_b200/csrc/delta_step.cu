// The gated delta rule one token further, on a state that is carried from call to call: everything between a linear-attention
// layer's input projections and its output projection (src/archs/qwen35_text.rs:491-626) for one new token of each row, as one kernel:
//     u    = silu(sum_{back < 4} w[c, 3 - back] x_{t - back}[c])                 causal depthwise conv over the new row and a ring of past ones
//     q, k = l2norm of u's query and key heads (q / sqrt(128)),  v = u's value heads,  beta = sigmoid(b),  g = softplus(a + dt_bias) * neg_exp_a
//     S <- e^g S;  d = beta (v - S^T k);  S <- S + k d^T;  o = S^T q;  y = o / sqrt(mean(o^2) + eps) * w * silu(z)
// What bounds it: S, 128 x 128 f32 per row and value head, is read once and written once (128 KB a row and head, against 7 flops an
// element) - HBM. Two blocks per SM walk over the (row, head) pairs. Thread (warp w, lane l) owns columns 4 l .. 4 l + 3 of the key rows
// w, w + 8, ... of every S: it holds them in registers while its pieces of the next pair's S come into its own corner of shared memory
// (cp.async, 128 KB an SM on the way) and the next pair's conv inputs into registers, and the other block's loads run under this one's
// arithmetic. With
//     S^T k and S^T q taken over the old S,   o = e^g (S^T q) + d (k . q),
// both sums over the key rows come from the same pass and one exchange between the warps, and S leaves as it is updated. Measured: 64
// rows x 48 heads 71 us = 5.7 TB/s (one block of 512 threads a pair 115 us, one such block an SM with three S in its ring 93), one
// row x 16 heads 5 us.
// Sums, norms and state are f32 throughout (the prompt form rounds the conv tap by tap to bf16, as the reference's kernel does; a
// step keeps it in f32). The conv's history is a ring of four rows by position mod 4: the new row's place is one that no conv of
// this step reads, so the blocks of a row need not wait for one another.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "context.h"
#include "device_guard.h"
#include "ptx.cuh"

namespace {

constexpr int kDim = 128;
constexpr int kTaps = 4;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRows = kDim / kWarps;  // key rows a thread holds
constexpr int kPart = kDim + 16;      // a warp's row of partial sums: the two lanes that read a column stay on different banks

struct StepSmem {
    float4 ring[kRows][kThreads];     // every thread's own pieces of the next S
    float part_k[kWarps][kPart], part_q[kWarps][kPart];
    float u[2][3][kDim];              // conv outputs of the head: q, k, v
    float norms[2][3][2];
    float gates[2][2];                // e^g, beta
    float d[kDim], sq[kDim];          // d scaled for the update, S^T q
};

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

__device__ __forceinline__ void cp16(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src), "r"(bytes) : "memory");
}

// What a thread needs to know of a (row, head) pair ahead of its turn.
struct Pair {
    int row, head, slot, pos;  // slot -1: idle
};
// The conv's inputs of this thread's two channels (threads below 192), or the gates' (thread 192).
struct Inputs {
    uint32_t x, past[kTaps - 1];
    uint4 w;
    float dt, decay;
};

__device__ __forceinline__ float lo_of(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_of(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

__global__ void __launch_bounds__(kThreads, 2) s1_delta_step_kernel(const StepParams p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    StepSmem& sm = *reinterpret_cast<StepSmem*>(smem_raw);
    constexpr int kConv = 3 * kDim / 2;  // threads of the conv
    s1::griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pairs = p.num_seqs * p.value_heads, step = gridDim.x;
    const int share = p.value_heads / p.key_heads;
    const long long C = static_cast<long long>(2 * p.key_heads + p.value_heads) * kDim;

    auto look = [&](int t) {
        Pair r{0, 0, -1, 0};
        if (t < pairs) {
            r.row = t / p.value_heads, r.head = t - r.row * p.value_heads;
            r.slot = p.index ? p.index[r.row] : r.row;
            r.pos = p.positions[r.row];
        }
        return r;
    };
    auto there = [&](const Pair& r) { return r.slot >= 0 && r.slot < p.num_states && r.pos >= 0; };
    auto state_of = [&](const Pair& r) {
        return p.state + (static_cast<long long>(r.slot) * p.value_heads + r.head) * (kDim * kDim) + warp * kDim + 4 * lane;
    };
    auto request = [&](const Pair& r) {  // this thread's pieces of S; a sequence's first token starts from zero, whatever the slot held
        if (there(r)) {
            const float* s = state_of(r);
#pragma unroll
            for (int i = 0; i < kRows; ++i) cp16(&sm.ring[i][tid], s + i * (kWarps * kDim), r.pos > 0 ? 16u : 0u);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto channel = [&](const Pair& r) {
        const int which = tid / (kDim / 2);
        return which * p.key_heads * kDim + (which == 2 ? r.head : r.head / share) * kDim + 2 * (tid % (kDim / 2));
    };
    auto fetch = [&](const Pair& r) {
        Inputs in = {};
        if (!there(r)) return in;
        if (tid < kConv) {
            const int c = channel(r);
            in.x = *reinterpret_cast<const uint32_t*>(p.mixed + r.row * p.ldm + c);
            const __nv_bfloat16* ring = p.conv_state + r.slot * kTaps * C + c;
#pragma unroll
            for (int back = 1; back < kTaps; ++back) in.past[back - 1] = back <= r.pos ? *reinterpret_cast<const uint32_t*>(ring + ((r.pos - back) & 3) * C) : 0u;
            in.w = *reinterpret_cast<const uint4*>(p.conv_w + static_cast<long long>(c) * kTaps);
        } else if (tid == kConv) {
            in.x = __bfloat16_as_ushort(p.b[r.row * p.ldba + r.head]);
            in.past[0] = __bfloat16_as_ushort(p.a[r.row * p.ldba + r.head]);
            in.dt = p.dt_bias[r.head], in.decay = p.neg_exp_a[r.head];
        }
        return in;
    };

    const int mine = p.index && tid < p.num_seqs ? p.index[tid] : -1;  // the state of row `tid`
    Pair now = look(blockIdx.x), next = look(blockIdx.x + step);
    request(now);
    Inputs in = fetch(now);
    int parity = 0, turn = 0;
    for (int t = blockIdx.x; t < pairs; t += step) {
        const Pair after = look(t + 2 * step);
        const Inputs in_next = fetch(next);
        const bool last_warp = warp == turn;  // writes this pair's output
        turn = turn + 1 == kWarps ? 0 : turn + 1;
        uint2 zr = make_uint2(0, 0), wr = zr;
        if (last_warp && there(now)) {
            zr = *reinterpret_cast<const uint2*>(p.z + now.row * p.ldz + now.head * kDim + 4 * lane);
            wr = *reinterpret_cast<const uint2*>(p.norm_w + 4 * lane);
        }
        // ---- conv + SiLU of this head's 384 channels, the gates
        bool bad = now.slot >= p.num_states || (now.slot >= 0 && now.pos < 0);
        if (p.index && now.slot >= 0) {  // a state that a row before this one has
            bad = bad || (tid < now.row && mine == now.slot);
            for (int j = tid + kThreads; j < now.row; j += kThreads) bad = bad || p.index[j] == now.slot;
        }
        float* u = &sm.u[parity][0][0];
        if (tid < kConv) {
            float a = lo_of(in.x) * hi_of(in.w.y), b = hi_of(in.x) * hi_of(in.w.w);
            a = fmaf(lo_of(in.past[0]), lo_of(in.w.y), a), b = fmaf(hi_of(in.past[0]), lo_of(in.w.w), b);
            a = fmaf(lo_of(in.past[1]), hi_of(in.w.x), a), b = fmaf(hi_of(in.past[1]), hi_of(in.w.z), b);
            a = fmaf(lo_of(in.past[2]), lo_of(in.w.x), a), b = fmaf(hi_of(in.past[2]), lo_of(in.w.z), b);
            a *= sigmoid(a), b *= sigmoid(b);
            *reinterpret_cast<float2*>(u + 2 * tid) = make_float2(a, b);
            const float sq = warp_sum(a * a + b * b);
            if (lane == 0) sm.norms[parity][warp >> 1][warp & 1] = sq;
        } else if (tid == kConv) {
            const float f = lo_of(in.past[0]) + in.dt;
            sm.gates[parity][0] = expf((fmaxf(f, 0.f) + log1pf(expf(-fabsf(f)))) * in.decay);
            sm.gates[parity][1] = sigmoid(lo_of(in.x));
        }
        bad = __syncthreads_or(bad);
        const bool live = !bad && now.slot >= 0;
        asm volatile("cp.async.wait_group 0;" ::: "memory");  // this pair's pieces, each thread its own
        float4 S[kRows];
        if (live) {
            // ---- S^T k and S^T q over this thread's key rows, then over the warps (k, q without their norms)
            float4 sk = make_float4(0.f, 0.f, 0.f, 0.f), sq = sk;
#pragma unroll
            for (int i = 0; i < kRows; ++i) S[i] = sm.ring[i][tid];
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const float kk = u[kDim + warp + kWarps * i], qq = u[warp + kWarps * i];
                sk.x = fmaf(S[i].x, kk, sk.x), sk.y = fmaf(S[i].y, kk, sk.y), sk.z = fmaf(S[i].z, kk, sk.z), sk.w = fmaf(S[i].w, kk, sk.w);
                sq.x = fmaf(S[i].x, qq, sq.x), sq.y = fmaf(S[i].y, qq, sq.y), sq.z = fmaf(S[i].z, qq, sq.z), sq.w = fmaf(S[i].w, qq, sq.w);
            }
            *reinterpret_cast<float4*>(&sm.part_k[warp][4 * lane]) = sk;
            *reinterpret_cast<float4*>(&sm.part_q[warp][4 * lane]) = sq;
        }
        request(next);  // into the corner that has just been read
        if (live && tid < kConv && (tid >= kDim || now.head % share == 0))  // the query and key channels once for the heads that share them
            *reinterpret_cast<uint32_t*>(p.conv_state + now.slot * kTaps * C + (now.pos & 3) * C + channel(now)) = in.x;
        __syncthreads();
        const float keep = sm.gates[parity][0], beta = sm.gates[parity][1];
        if (live) {  // a warp sums 16 columns, two lanes to a column
            const int c = 16 * warp + (lane & 15), g = lane >> 4;
            float a = sm.part_k[g][c] + sm.part_k[g + 2][c] + sm.part_k[g + 4][c] + sm.part_k[g + 6][c];
            float b = sm.part_q[g][c] + sm.part_q[g + 2][c] + sm.part_q[g + 4][c] + sm.part_q[g + 6][c];
            a += __shfl_xor_sync(0xffffffffu, a, 16), b += __shfl_xor_sync(0xffffffffu, b, 16);
            const float rk = 1.f / sqrtf(sm.norms[parity][1][0] + sm.norms[parity][1][1] + 1e-6f);
            if (g == 0) {
                sm.d[c] = beta * (u[2 * kDim + c] - keep * (a * rk)) * rk;
                sm.sq[c] = b;
            }
        }
        __syncthreads();
        if (live) {
            const float4 d = *reinterpret_cast<const float4*>(&sm.d[4 * lane]);
            float* state = state_of(now);
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const float kk = u[kDim + warp + kWarps * i];
                *reinterpret_cast<float4*>(state + i * (kWarps * kDim)) =
                    make_float4(fmaf(kk, d.x, keep * S[i].x), fmaf(kk, d.y, keep * S[i].y), fmaf(kk, d.z, keep * S[i].z), fmaf(kk, d.w, keep * S[i].w));
            }
        }
        if (last_warp) {
            float o[4] = {0.f, 0.f, 0.f, 0.f};
            if (live) {
                const float rq = 0.08838834764831845f / sqrtf(sm.norms[parity][0][0] + sm.norms[parity][0][1] + 1e-6f);  // 128^-1/2 / |q|
                const float kq = warp_sum(u[lane] * u[kDim + lane] + u[lane + 32] * u[kDim + lane + 32] + u[lane + 64] * u[kDim + lane + 64] +
                                          u[lane + 96] * u[kDim + lane + 96]);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = rq * fmaf(sm.d[4 * lane + e], kq, keep * sm.sq[4 * lane + e]);
                const float r = 1.f / sqrtf(warp_sum(o[0] * o[0] + o[1] * o[1] + o[2] * o[2] + o[3] * o[3]) * (1.f / kDim) + p.eps);
                const float z[4] = {lo_of(zr.x), hi_of(zr.x), lo_of(zr.y), hi_of(zr.y)}, w[4] = {lo_of(wr.x), hi_of(wr.x), lo_of(wr.y), hi_of(wr.y)};
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] *= r * w[e] * z[e] * sigmoid(z[e]);
            } else if (bad && lane == 0 && atomicCAS(p.status, 0, now.pos < 0 ? 120 : 119) == 0) {
                p.status[1] = static_cast<int>(blockIdx.x);
                p.status[2] = now.row;
                p.status[3] = now.pos < 0 ? now.pos : now.slot;
            }
            // an idle row's output, or a refused one's, is zero
            const __nv_bfloat162 y01 = __floats2bfloat162_rn(o[0], o[1]), y23 = __floats2bfloat162_rn(o[2], o[3]);
            *reinterpret_cast<uint2*>(p.y + now.row * p.ldy + now.head * kDim + 4 * lane) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&y01), *reinterpret_cast<const uint32_t*>(&y23));
        }
        now = next, next = after;
        in = in_next;
        parity ^= 1;
    }
    // (not earlier: the next kernel's blocks would be placed two to an SM on what this grid leaves free - 37 rows of 6 heads 7.6 us
    // instead of 6.9 in a row of steps, when this was tried)
    s1::griddep_launch_dependents();
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The last rows before the conv of every sequence of a prompt batch into the ring that the step kernel reads.
__global__ void __launch_bounds__(256) s1_conv_state_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, const int32_t* __restrict__ cu,
                                                            const int32_t* __restrict__ index, int num_states, int total_tokens, int C, __nv_bfloat16* __restrict__ ring) {
    const int s = blockIdx.x, back = blockIdx.y;  // the token `back` before the sequence's last
    const int slot = index[s], a = cu[s], end = cu[s + 1], len = a >= 0 && end <= total_tokens ? end - a : 0;
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

int s1_conv_state_launch(s1_ctx* ctx, const void* mixed, long long ldm, const int32_t* cu_seqlens, int num_seqs, int total_tokens, const int32_t* index,
                         int num_states, int channels, void* conv_state) {
    if (num_seqs == 0) return S1_OK;
    s1_conv_state_kernel<<<dim3(num_seqs, kTaps), 256, 0, ctx->stream>>>(static_cast<const __nv_bfloat16*>(mixed), ldm, cu_seqlens, index, num_states,
                                                                         total_tokens, channels, static_cast<__nv_bfloat16*>(conv_state));
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
    if (!aligned(conv_weight, 16) || !aligned(conv_state, 16) || !aligned(state, 16) || !aligned(mixed, 4) || (ldm % 2))
        return s1_fail(ctx, S1_EINVAL, "%s: the states and the conv weight must be 16-byte aligned, the rows of mixed 4-byte", who);
    if (!aligned(z, 8) || !aligned(y, 8) || !aligned(norm_weight, 8) || (ldz % 4) || (ldy % 4))
        return s1_fail(ctx, S1_EINVAL, "%s: the rows of z and y and the norm weight must be 8-byte aligned", who);
    const long long blocks = static_cast<long long>(num_seqs) * value_heads;
    if (blocks > (1LL << 30)) return s1_fail(ctx, S1_EINVAL, "%s: too many rows", who);
    if (num_seqs == 0) return S1_OK;
    S1DeviceGuard guard(ctx->device);
    if (!guard.ok) return s1_fail(ctx, S1_ECUDA, "%s: cudaSetDevice(%d) failed", who, ctx->device);
    StepParams p{static_cast<const __nv_bfloat16*>(mixed), ldm, static_cast<const __nv_bfloat16*>(conv_weight), positions,
                 static_cast<const __nv_bfloat16*>(b_proj), static_cast<const __nv_bfloat16*>(a_proj), ldba, dt_bias, neg_exp_a,
                 static_cast<const __nv_bfloat16*>(z), ldz, static_cast<const __nv_bfloat16*>(norm_weight), eps, state_index, num_states, num_seqs,
                 static_cast<__nv_bfloat16*>(conv_state), state, key_heads, value_heads, static_cast<__nv_bfloat16*>(y), ldy, ctx->status_dev};
    static std::atomic<unsigned long long> told{0};  // one bit per device
    if (!(told.load(std::memory_order_relaxed) >> (ctx->device & 63) & 1)) {
        S1_CUDA_OK(ctx, cudaFuncSetAttribute(s1_delta_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(StepSmem))));
        told.fetch_or(1ull << (ctx->device & 63), std::memory_order_relaxed);
    }
    const unsigned grid = static_cast<unsigned>(std::min<long long>(blocks, 2 * ctx->sm_count));
    S1_CUDA_OK(ctx, s1_launch_waiting(ctx, s1_delta_step_kernel, grid, 1u, kThreads, sizeof(StepSmem), p));
    ctx->launches += 1;
    return S1_OK;
}
