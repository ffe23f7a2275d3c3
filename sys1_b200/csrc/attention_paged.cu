// Attention of one new token per request over a paged key-value cache (grouped query heads, head dim 64, 128 or 256):
//     a[b, h] = sum_{j < len_b} softmax_j(scale * q[b, h] . k_j) v_j,   k_j, v_j of KV head h / (heads / kv_heads)
// and, with a gate, a * sigmoid(gate). It is the step form of the causal attention of src/archs/qwen35_text.rs:312-411, whose
// keys and values here come from the cache instead of from the same prompt.
//
// What bounds it: every key and value is read once for the query heads that share it, 4 * group flops per 4 bytes - HBM, whatever
// the group size. So the kernel is built around the loads:
//  * work is cut into units of kUnit keys of one (row, KV head, 8 or 16 of its query heads) - a "span" is all units of one such triple -
//    and the units of the whole batch, in order, are dealt out in contiguous ranges of equal cost, one to each CTA of the grid; a
//    span's beginning is counted too, as so many units (kStart; without it 32 contexts of 128 tokens beside 30 of 8192 take 254 us,
//    with it 161). The CTAs find their ranges from the lengths in device memory, so that nothing of a step depends on the host and
//    the balance holds for one long context and for many ragged ones alike. A span that crosses from one CTA to the next leaves
//    partial results (maximum, sum, unnormalised output in f32) in the workspace, at most two per CTA; and a second
//    kernel joins them, in the order of the units: results do not depend on timing. (Joined by the CTA that finds all pieces of a
//    span there, without the second kernel, the pieces were one CTA's work: an earlier form of this kernel, 21 us for 32 contexts up to
//    2048, took 27 that way.)
//  * inside a CTA the warps take tiles of 16 keys in turn, each through a ring of its own in shared memory (cp.async, 192 KB an SM in
//    flight or in use): no warp waits for another until its span is done. The next span's first keys are fetched into
//    L2 and its queries into registers while the warps' results are put together.
//  * the products run on mma.sync m16n8k16 with the operands turned round - S^T = K Q^T, O^T = V^T P^T - so that the 16 rows are
//    keys and head dimensions, which there are enough of, and the 8 columns the query heads of the group. tcgen05 would want 64 or
//    128 rows of queries where there are 1 to 16; at the rate that HBM delivers keys, the tensor pipe is 15 % busy.
// Measured: 62 contexts of 100 .. 8192 tokens, 24 query and 4 KV heads of 256: 169 us = 6.2 TB/s; one of 131071 tokens, 8 and 2 heads:
// 50 us = 5.4 TB/s; 31 of 1 .. 2048 tokens: 19.6 us; one of 17: 6.5 us.
// Scores, maxima, sums and outputs are f32. For the second product a weight is split into two bf16 values, its first eight bits and
// what they leave (rounded: an error of 2^-15 of the weight, where one bf16 value would be 2^-8 off); their sum over the keys is that of
// the f32 weights. The product with the rest costs 1 % at the first size above and at the third, up to 5 % elsewhere (16 heads to a KV head
// of 64, 450 contexts of 900 tokens: 35.7 -> 37.6 us).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "context.h"
#include "device_guard.h"
#include "ptx.cuh"

using namespace s1;

namespace {

constexpr int kTile = 16;               // keys of one warp step
constexpr int kCols = 8;                // query heads of one MMA (its columns); a span has NT times as many
constexpr int kRings = 192 * 1024;      // bytes of an SM's warps' rings

// What a span costs beyond its units (its queries, the first keys' way, the warps' results put together), in units of its head dim.
template <int D>
constexpr int kStart = 256 / D;

// CTAs of the first kernel at most: two, three or four per SM of any sm_100 part
constexpr int max_ctas(int head_dim) { return head_dim == 256 ? 320 : head_dim == 128 ? 480 : 640; }

struct PagedParams {
    const __nv_bfloat16* q;
    long long ldq, q_head_stride;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    long long page_stride, token_stride, head_stride;
    int num_pages, shift;
    const int32_t* tables;
    long long ldt;
    int table_width;
    const int32_t* lengths;
    int num_seqs, heads, kv_heads, group, spans_per_row, blocks_per_group;  // blocks: of 8 NT heads
    float scale_log2;
    const __nv_bfloat16* gate;
    long long ldg, gate_head_stride;
    __nv_bfloat16* out;
    long long ldo;
    float* parts;   // [2 * grid][heads of a span][D]: unnormalised outputs of the cut spans' pieces
    float2* marks;  // [2 * grid][heads of a span]: maximum (in units of log2) and sum of the same pieces
    int4* records;  // row, span of the row, last (-1: not cut) and first CTA of a span: by_span one for each span, else one for each CTA, of the
    bool by_span;   // span that begins in it and is cut
    int* status;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
// What a weight's first eight bits leave, and never quite nothing: the weight's two parts both take an infinite value to the same infinity.
__device__ __forceinline__ float rest_of(uint32_t weight) {
    const float w = __uint_as_float(weight);
    return fmaxf(w - __uint_as_float(weight & 0xffff0000u), w * 0x1p-24f);
}
__device__ __forceinline__ void report(int* status, int code, int where, int value) {
    if (atomicCAS(status, 0, code) == 0) {
        status[1] = static_cast<int>(blockIdx.x);
        status[2] = where;
        status[3] = value;
    }
}
// (Everything a call is given is read with plain loads: the kernel may be resident while the one before still writes it, which the
// read-only path does not allow for.)
// Keys that a row attends to; a length beyond its block table is reported and the row treated as empty.
__device__ __forceinline__ int row_length(const PagedParams& p, int b, bool tell) {
    const int len = max(p.lengths[b], 0);
    if (len > (static_cast<long long>(p.table_width) << p.shift)) {
        if (tell) report(p.status, 117, b, len);
        return 0;
    }
    return len;
}
__device__ __forceinline__ float rcp_fast(float x) {  // relative error 2^-23, before a rounding to bf16
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_fast(1.f + exp2_fast(-1.4426950408889634f * x)); }
// The sum of a part of a span's weights (maximum, sum) in terms of the whole span's maximum. A part without a finite score counts only
// where the whole has none: 0 if it had no key, else no number.
__device__ __forceinline__ float weighed(float2 mark, float top) {
    return mark.x != -INFINITY ? mark.y * exp2_fast(mark.x - top) : top == -INFINITY ? mark.y : 0.f;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory"); }

// One warp's pass over its tiles of a span: keys first, first + 16 W, ..., 16 to a tile, below `end`. NT = 1: up to 8 query heads, held in registers;
// NT = 2: up to 16, read from shared memory step by step, so that a group of more than 8 does not read its keys twice (32 x 8192
// tokens, 16 heads to a KV head of 256: 166 us as two spans of 8, 98 as one of 16).
template <int D, int NT, int W, int P>
struct WarpPass {
    static constexpr int kUnit = W * kTile;                 // keys of one unit: a tile for each of the CTA's W warps
    static constexpr int kSlotBytes = kTile * D * 2;
    static constexpr int kSlots = kRings / (W * P * kSlotBytes);
    static constexpr int kRingBytes = kSlots * kSlotBytes;
    static constexpr int kChunks = D / 8;                   // 16-byte pieces of a key
    static constexpr int kRowsPerCopy = 32 / kChunks;
    static constexpr int kSteps = D / 16;
    static constexpr int kChains = D == 256 && NT == 1 ? 4 : 2;  // independent accumulators of S^T
    static constexpr int kQueryRow = D + 8;                 // values of a row of queries in shared memory: no bank conflicts by columns

    const PagedParams& p;
    const int lane;
    const uint32_t ring;            // shared address of this warp's ring
    volatile uint32_t* masks;       // [kSlots] which of the 16 keys a slot holds
    float O[NT][kSteps][4];         // O^T: dims 16 s + lane/4 (+ 8), heads 8 t + 2 (lane % 4) (+ 1)
    float m[NT][2], l[NT][2];
    const bool one_page;            // pages of 16 tokens and more: a tile never leaves its page
    long long off;                  // where the tile whose keys were requested last begins (one_page), or lane j's key of it
    uint32_t mask;                  // which of its keys there are

    __device__ __forceinline__ WarpPass(const PagedParams& p_, int lane_, uint32_t ring_, uint32_t* masks_)
        : p(p_), lane(lane_), ring(ring_), masks(masks_), one_page(p_.shift >= 4) {}

    // the keys (or, with `values`, the values) of the tile that begins at key j0, into slot `slot`
    __device__ __forceinline__ void request(bool values, int slot, int b, int kvh, int j0, int end) {
        if (!values) {
            if (one_page) {
                const int page = p.tables[b * p.ldt + (j0 >> p.shift)];
                const bool ok = page >= 0 && page < p.num_pages;
                if (!ok && lane == 0) report(p.status, 118, b, page);
                off = page * p.page_stride + (j0 & ((1 << p.shift) - 1)) * p.token_stride + kvh * p.head_stride;
                mask = ok ? (1u << min(kTile, end - j0)) - 1u : 0u;
            } else {
                const int j = j0 + lane;
                const bool want = lane < kTile && j < end;
                const int page = want ? p.tables[b * p.ldt + (j >> p.shift)] : 0;
                const bool ok = want && page >= 0 && page < p.num_pages;
                if (want && !ok) report(p.status, 118, b, page);
                off = ok ? page * p.page_stride + (j & ((1 << p.shift) - 1)) * p.token_stride + kvh * p.head_stride : 0;
                mask = __ballot_sync(0xffffffffu, ok);
            }
            if (lane == 0) masks[slot] = mask;
        }
        const __nv_bfloat16* base = values ? p.v : p.k;
        const uint32_t dst = ring + slot * kSlotBytes;
        const int row0 = lane / kChunks, ch = lane % kChunks;
        // keys past the end (and those of a bad page) are zeros: what lies in the rest of a page is never multiplied
        if (one_page && mask == (1u << kTile) - 1u) {
            const __nv_bfloat16* src = base + off + row0 * p.token_stride + ch * 8;
#pragma unroll
            for (int i = 0; i < kTile / kRowsPerCopy; ++i, src += kRowsPerCopy * p.token_stride)
                cp16(dst + (i * kRowsPerCopy + row0) * (D * 2) + ((ch ^ ((i * kRowsPerCopy + row0) & 7)) << 4), src, 16u);
        } else {
#pragma unroll 1
            for (int i = 0; i < kTile / kRowsPerCopy; ++i) {
                const int row = i * kRowsPerCopy + row0;
                const bool there = mask >> row & 1u;
                const long long o = one_page ? off + row * p.token_stride : __shfl_sync(0xffffffffu, off, row);
                cp16(dst + row * (D * 2) + ((ch ^ (row & 7)) << 4), base + (there ? o : 0) + ch * 8, there ? 16u : 0u);
            }
        }
    }

    int b, kvh, first, end, requests, wslot;

    // requests of a span's first tiles
    __device__ __forceinline__ void start(int b_, int kvh_, int first_, int end_) {
        b = b_, kvh = kvh_, first = first_, end = end_;
        requests = first < end ? 2 * ((end - first + kUnit - 1) / kUnit) : 0;
        wslot = 0;
#pragma unroll 1
        for (int n = 0; n < kSlots - 1; ++n) {
            if (n < requests) load(n);
            asm volatile("cp.async.commit_group;" ::: "memory");
            ++wslot;
        }
    }
    __device__ __forceinline__ void load(int n) { request(n & 1, wslot, b, kvh, first + (n >> 1) * kUnit, end); }  // request number n

    // `queries`: 8 NT rows of kQueryRow values in shared memory
    __device__ __forceinline__ void run(const __nv_bfloat16* queries) {
        uint32_t qf[NT == 1 ? kSteps : 1][2];
        uint32_t qat = 0;
        if constexpr (NT == 1) {
            const __nv_bfloat16* q = queries + (lane >> 2) * kQueryRow + 2 * (lane & 3);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                qf[s][0] = *reinterpret_cast<const uint32_t*>(q + 16 * s);
                qf[s][1] = *reinterpret_cast<const uint32_t*>(q + 16 * s + 8);
            }
        } else {  // an ldmatrix for each step: heads 0 .. 7 of its two halves, then heads 8 .. 15
            qat = smem_u32(queries + ((lane >> 4) * kCols + (lane & 7)) * kQueryRow + (lane >> 3 & 1) * 8);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) O[t][s][0] = O[t][s][1] = O[t][s][2] = O[t][s][3] = 0.f;
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
        }
        int rslot = 0;
        uint32_t seen = 0;  // whether any key was there
        // this lane's rows of the ldmatrix tiles: the 16-byte pieces 2 s + h of row r lie at r * 2 D + ((2 s + h) ^ (r & 7)) * 16, which is
        // one of four places and a multiple of 128 bytes
        uint32_t kat[4], vat[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            kat[i] = ((lane >> 3 & 1) * 8 + (lane & 7)) * (D * 2) + (((2 * i + (lane >> 4)) ^ (lane & 7)) << 4);
            vat[i] = ((lane >> 4) * 8 + (lane & 7)) * (D * 2) + (((2 * i + (lane >> 3 & 1)) ^ (lane & 7)) << 4);
        }
#pragma unroll 1
        for (int n = 0; n < requests; n += 2) {
            uint32_t high[NT][2], rest[NT][2];  // the weights as two bf16 values each
            // ---- keys: S^T = K Q^T
            asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 2) : "memory");
            __syncwarp();  // the slot has landed for every lane, and every lane is done with the one refilled next
            if (n + kSlots - 1 < requests) load(n + kSlots - 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            wslot = wslot + 1 == kSlots ? 0 : wslot + 1;
            {
                const uint32_t live = masks[rslot], slot = ring + rslot * kSlotBytes;
                seen |= live;
                float c[NT][kChains][4];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < kChains; ++i) c[t][i][0] = c[t][i][1] = c[t][i][2] = c[t][i][3] = 0.f;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    uint32_t a[4];
                    ldsm4(a, slot + kat[s & 3] + (s >> 2) * 128);
                    if constexpr (NT == 1) {
                        mma16816(c[0][s % kChains], a, qf[s][0], qf[s][1]);
                    } else {
                        uint32_t q[4];
                        ldsm4(q, qat + 32 * s);
                        mma16816(c[0][s % kChains], a, q[0], q[1]);
                        mma16816(c[1][s % kChains], a, q[2], q[3]);
                    }
                }
                const bool in0 = live >> (lane >> 2) & 1u, in1 = live >> ((lane >> 2) + 8) & 1u;
                float s[NT][4], top[NT][2];
                bool grows = false;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 1; i < kChains; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[t][0][e] += c[t][i][e];
                    s[t][0] = in0 ? c[t][0][0] * p.scale_log2 : -INFINITY;
                    s[t][1] = in0 ? c[t][0][1] * p.scale_log2 : -INFINITY;
                    s[t][2] = in1 ? c[t][0][2] * p.scale_log2 : -INFINITY;
                    s[t][3] = in1 ? c[t][0][3] * p.scale_log2 : -INFINITY;
                    top[t][0] = fmaxf(s[t][0], s[t][2]), top[t][1] = fmaxf(s[t][1], s[t][3]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        top[t][0] = fmaxf(top[t][0], __shfl_xor_sync(0xffffffffu, top[t][0], o));
                        top[t][1] = fmaxf(top[t][1], __shfl_xor_sync(0xffffffffu, top[t][1], o));
                    }
                    grows = grows || top[t][0] > m[t][0] || top[t][1] > m[t][1];
                }
                if (n == 0) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) m[t][0] = top[t][0], m[t][1] = top[t][1];
                } else if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float scale[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float now = fmaxf(m[t][e], top[t][e]);
                            scale[e] = now == -INFINITY ? 1.f : exp2_fast(m[t][e] - now);
                            m[t][e] = now;
                            l[t][e] *= scale[e];
                        }
#pragma unroll
                        for (int i = 0; i < kSteps; ++i)
                            O[t][i][0] *= scale[0], O[t][i][1] *= scale[1], O[t][i][2] *= scale[0], O[t][i][3] *= scale[1];
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float ref0 = m[t][0] == -INFINITY ? 0.f : m[t][0], ref1 = m[t][1] == -INFINITY ? 0.f : m[t][1];  // no key seen yet: all weights are 0
                    s[t][0] = exp2_fast(s[t][0] - ref0), s[t][1] = exp2_fast(s[t][1] - ref1);
                    s[t][2] = exp2_fast(s[t][2] - ref0), s[t][3] = exp2_fast(s[t][3] - ref1);
                    l[t][0] += s[t][0] + s[t][2];
                    l[t][1] += s[t][1] + s[t][3];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t x = __float_as_uint(s[t][2 * i]), y = __float_as_uint(s[t][2 * i + 1]);
                        high[t][i] = transpose8(__byte_perm(x, y, 0x7632));
                        rest[t][i] = transpose8(pack2(rest_of(x), rest_of(y)));
                    }
                }
            }
            rslot = rslot + 1 == kSlots ? 0 : rslot + 1;
            // ---- values: O^T += V^T P^T
            asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 2) : "memory");
            __syncwarp();
            if (n + kSlots < requests) load(n + kSlots);
            asm volatile("cp.async.commit_group;" ::: "memory");
            wslot = wslot + 1 == kSlots ? 0 : wslot + 1;
            {
                const uint32_t slot = ring + rslot * kSlotBytes;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    uint32_t a[4];
                    ldsm4_t(a, slot + vat[i & 3] + (i >> 2) * 128);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma16816(O[t][i], a, high[t][0], high[t][1]);
                        mma16816(O[t][i], a, rest[t][0], rest[t][1]);
                    }
                }
            }
            rslot = rslot + 1 == kSlots ? 0 : rslot + 1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                l[t][0] += __shfl_xor_sync(0xffffffffu, l[t][0], o);
                l[t][1] += __shfl_xor_sync(0xffffffffu, l[t][1], o);
            }
        if (seen)  // keys whose scores are all -inf: the sum of their weights is no number, unless others have a finite score
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) l[t][e] = m[t][e] == -INFINITY ? __int_as_float(0x7fffffff) : l[t][e];
    }
};

struct Walk {        // a run over a range of the batch's costs
    int at, last;
    int b, kvh, hb;  // row, KV head, which eight query heads of its group
    int inside;      // cost inside that span
};
struct Segment {     // the part of one span that lies in the range
    int b, kvh, hb;      // row, KV head, which eight query heads of its group
    int u0, n, units;    // units u0 .. u0 + n - 1 of `units`
    int end;             // keys u0 * kUnit .. end - 1
};

// P CTAs of W warps per SM (both sides of each pair measured with weights of one part). W = 8 and as many CTAs as the registers allow, one at a head dim of 256 and two below (head dim 128, 28 contexts
// of up to 61259 tokens, 4 heads on 2: 161 us, with one 163; head dim 64, 4 of 66164, 64 on 4: 37 and 44) but one at head dim 128 with NT
// = 2, which would spill (94 of 3443, 64 on 4: 92 us, with two 114). Where there are many spans, W = 4: one's keys come while another puts
// its results together (head dim 256: 512 contexts of 100 tokens 40 us with W = 8, 35 with 4; with few and long ones the larger units
// stream a little faster, 64 contexts up to 8192 tokens 168 and 172 us), and with NT = 1 three CTAs at head dim 128 (512 of 100 tokens 20 us,
// with two 23) and four at 64 (700 of up to 900 tokens 37 us, with two 45; long contexts lose, 128 of 2000 tokens 83 us and 75).
template <int D, int NT, int W, int P>
__global__ void __launch_bounds__(W * 32, P) s1_attention_paged_kernel(const PagedParams p) {
    using Pass = WarpPass<D, NT, W, P>;
    constexpr int kHeads = NT * kCols, kWarps = W, kThreads = W * 32, kUnit = Pass::kUnit;
    extern __shared__ __align__(128) uint8_t ring_smem[];
    float* stage = reinterpret_cast<float*>(ring_smem);  // [warp][head][D + 4], after the rings have been read
    constexpr int kStage = D + 4;                        // keeps the four head columns of a store on different banks
    __shared__ uint32_t masks[kWarps][Pass::kSlots];
    __shared__ float2 marks[kWarps][kHeads];             // maximum and sum of every warp
    __shared__ float2 marks_all[kHeads];
    __shared__ __align__(16) __nv_bfloat16 queries[kHeads][Pass::kQueryRow];
    __shared__ int warp_costs[kWarps];
    __shared__ Walk begin_sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cta = blockIdx.x, ctas = gridDim.x;

    griddep_wait();
    griddep_launch_dependents();  // the join's blocks may take the SMs that run out of work first (they wait for the whole grid)

    // ---- rows without a key: zeros
    for (int b = cta * kWarps + warp; b < p.num_seqs; b += ctas * kWarps)
        if (row_length(p, b, lane == 0) == 0) {
            if (p.by_span)
                for (int i = lane; i < p.spans_per_row; i += 32) p.records[b * p.spans_per_row + i] = make_int4(0, 0, -1, 0);
            for (int i = lane * 8; i < p.heads * D; i += 256) *reinterpret_cast<uint4*>(p.out + b * p.ldo + i) = make_uint4(0, 0, 0, 0);
        }

    // ---- this CTA's range (the host has seen to it that all costs together fit 31 bits)
    auto cost_of = [&](int b) {
        const int units = (row_length(p, b, false) + kUnit - 1) / kUnit;
        return units ? (units + kStart<D>) * p.spans_per_row : 0;
    };
    const int per = (p.num_seqs + kThreads - 1) / kThreads;
    const int rb = min(tid * per, p.num_seqs), re = min(rb + per, p.num_seqs);
    int mine = 0;
    for (int b = rb; b < re; ++b) mine += cost_of(b);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    if (lane == 31) warp_costs[warp] = upto;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += warp_costs[w];
        total += warp_costs[w];
    }
    const int workers = min(ctas, total);
    if (cta >= workers) {
        if (tid == 0 && !p.by_span) p.records[cta] = make_int4(0, 0, -1, 0);
        return;
    }
    const int share = total / workers, longer = total - share * workers;  // the first `longer` CTAs have one more
    {
        const int first = share * cta + min(cta, longer), at = before + upto - mine;
        if (first >= at && first < at + mine) {
            int u = at, b = rb;
            for (int n; b + 1 < re && u + (n = cost_of(b)) <= first; ++b) u += n;
            const int cost = (row_length(p, b, false) + kUnit - 1) / kUnit + kStart<D>;
            const int span = (first - u) / cost, kvh = span / p.blocks_per_group;
            begin_sh = Walk{first, first + share + (cta < longer ? 1 : 0), b, kvh, span - kvh * p.blocks_per_group, first - u - span * cost};
        }
    }
    __syncthreads();
    Walk walk = begin_sh;
    auto advance = [&](Segment& s) {
        while (walk.at < walk.last && walk.b < p.num_seqs) {
            const int len = row_length(p, walk.b, false), units = (len + kUnit - 1) / kUnit, cost = units + kStart<D>;
            if (units == 0) {
                ++walk.b;
                continue;
            }
            const int at = walk.inside, step = min(cost - at, walk.last - walk.at);
            s.b = walk.b, s.kvh = walk.kvh, s.hb = walk.hb, s.units = units;
            s.u0 = max(0, at - kStart<D>), s.n = max(0, at + step - kStart<D>) - s.u0;
            s.end = min(len, (s.u0 + s.n) * kUnit);
            walk.at += step, walk.inside += step;
            if (walk.inside == cost) {  // on to the next span
                walk.inside = 0;
                if (++walk.hb == p.blocks_per_group) walk.hb = 0, ++walk.kvh;
                if (walk.kvh == p.kv_heads) walk.kvh = 0, ++walk.b;
            }
            if (s.n) return true;
        }
        return false;
    };
    int4 record = make_int4(0, 0, -1, 0);
    Pass pass(p, lane, smem_u32(ring_smem) + warp * Pass::kRingBytes, masks[warp]);

    // the queries of a span: 16 bytes a thread and turn, fetched a span ahead (rows past the group's last head repeat it and are not
    // written out)
    constexpr int kQueryThreads = kHeads * D / 8, kTurns = (kQueryThreads + kThreads - 1) / kThreads;
    struct Queries {
        uint4 q[kTurns];
    };
    auto fetch_q = [&](const Segment& s) {
        Queries r;
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int at = tid + i * kThreads, h = s.kvh * p.group + min(s.hb * kHeads + at / (D / 8), p.group - 1);
            r.q[i] = at < kQueryThreads ? *reinterpret_cast<const uint4*>(p.q + s.b * p.ldq + h * p.q_head_stride + at % (D / 8) * 8) : make_uint4(0, 0, 0, 0);
        }
        return r;
    };
    auto hand_q = [&](const Queries& r) {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int at = tid + i * kThreads;
            if (at < kQueryThreads) *reinterpret_cast<uint4*>(&queries[at / (D / 8)][at % (D / 8) * 8]) = r.q[i];
        }
    };

    Segment now = {}, next = {};
    bool more = advance(now);
    if (more) {
        const Queries q = fetch_q(now);
        pass.start(now.b, now.kvh, now.u0 * kUnit + warp * kTile, now.end);
        hand_q(q);
    }
    __syncthreads();
    while (more) {
        const int h0 = now.kvh * p.group + now.hb * kHeads, nh = min(kHeads, p.group - now.hb * kHeads);
        const bool whole = now.u0 == 0 && now.n == now.units;
        const int stop = walk.at;  // where this segment ends
        more = advance(next);
        // where the next span's keys begin for this warp: looked up now, wanted when this span is done
        const int next_j = next.u0 * kUnit + warp * kTile + lane;
        const int next_page = more && lane < kTile && next_j < next.end ? p.tables[next.b * p.ldt + (next_j >> p.shift)] : -1;
        pass.run(&queries[0][0]);
        // ---- the next span's first tile is fetched into L2, its queries and this one's gates into registers, while the warps' results
        //      are put together
        {
            const bool there = next_page >= 0 && next_page < p.num_pages;
            const long long o = there ? next_page * p.page_stride + (next_j & ((1 << p.shift) - 1)) * p.token_stride + next.kvh * p.head_stride : -1;
            constexpr int kLines = D / 64;  // 128-byte lines of a key (one prefetch a lane: the bulk form is issued lane by lane, 2000 cycles here)
#pragma unroll
            for (int i = 0; i < kTile * kLines / 32; ++i) {
                const int at = lane + 32 * i;
                const long long row = __shfl_sync(0xffffffffu, o, at / kLines);
                if (row >= 0) prefetch_l2(p.k + row + at % kLines * 64), prefetch_l2(p.v + row + at % kLines * 64);
            }
            if (kTile * kLines < 32) {  // head dim 64: one line a key
                const long long row = __shfl_sync(0xffffffffu, o, lane % kTile);
                if (row >= 0) prefetch_l2((lane < kTile ? p.k : p.v) + row);
            }
        }
        const Queries next_q = fetch_q(more ? next : now);
        constexpr int kPairs = kHeads * D / 2 / kThreads;  // pairs of outputs of a thread
        uint32_t gates[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const int h = (tid + i * kThreads) / (D / 2), d = 2 * ((tid + i * kThreads) % (D / 2));
            gates[i] = whole && p.gate && h < nh ? *reinterpret_cast<const uint32_t*>(p.gate + now.b * p.ldg + (h0 + h) * p.gate_head_stride + d) : 0u;
        }
        if (lane < 4)
#pragma unroll
            for (int t = 0; t < NT; ++t)
                marks[warp][kCols * t + 2 * lane] = make_float2(pass.m[t][0], pass.l[t][0]), marks[warp][kCols * t + 2 * lane + 1] = make_float2(pass.m[t][1], pass.l[t][1]);
        __syncthreads();  // every ring has been read
        const int parts = min(kWarps, (now.end - now.u0 * kUnit + kTile - 1) / kTile);  // warps that had a tile
        if (warp < parts) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int col = kCols * t + 2 * (lane & 3);
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top[0] = fmaxf(top[0], marks[w][col].x), top[1] = fmaxf(top[1], marks[w][col + 1].x);
                const float f0 = pass.m[t][0] == -INFINITY ? 0.f : exp2_fast(pass.m[t][0] - top[0]);
                const float f1 = pass.m[t][1] == -INFINITY ? 0.f : exp2_fast(pass.m[t][1] - top[1]);
                float* st = stage + (warp * kHeads + col) * kStage + (lane >> 2);
#pragma unroll
                for (int s = 0; s < Pass::kSteps; ++s) {
                    st[16 * s] = pass.O[t][s][0] * f0;
                    st[kStage + 16 * s] = pass.O[t][s][1] * f1;
                    st[16 * s + 8] = pass.O[t][s][2] * f0;
                    st[kStage + 16 * s + 8] = pass.O[t][s][3] * f1;
                }
            }
            if (tid < kHeads) {
                float high = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) high = fmaxf(high, marks[w][tid].x);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) sum += weighed(marks[w][tid], high);
                marks_all[tid] = make_float2(high, sum);
            }
        }
        __syncthreads();
        const int piece = 2 * cta + (now.u0 == 0 ? 1 : 0);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const int h = (tid + i * kThreads) / (D / 2), d = 2 * ((tid + i * kThreads) % (D / 2));
            if (h >= nh) break;
            float2 x = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 y = *reinterpret_cast<const float2*>(&stage[(w * kHeads + h) * kStage + d]);
                x.x += w < parts ? y.x : 0.f, x.y += w < parts ? y.y : 0.f;
            }
            if (whole) {
                const float inv = marks_all[h].y == 0.f ? 0.f : rcp_fast(marks_all[h].y);
                x.x *= inv, x.y *= inv;
                if (p.gate) x.x *= sigmoid_fast(__uint_as_float(gates[i] << 16)), x.y *= sigmoid_fast(__uint_as_float(gates[i] & 0xffff0000u));
                *reinterpret_cast<uint32_t*>(p.out + now.b * p.ldo + (h0 + h) * D + d) = pack2(x.x, x.y);
            } else {
                *reinterpret_cast<float2*>(p.parts + (static_cast<long long>(piece) * kHeads + h) * D + d) = x;
            }
        }
        if (!whole) {
            if (tid < nh) p.marks[piece * kHeads + tid] = marks_all[tid];
            if (now.u0 == 0) {  // a span that begins here and is cut at the end of this CTA's range: the CTA that has its last unit
                const int end = stop - now.n + now.units - 1, border = longer * (share + 1);
                record = make_int4(now.b, now.kvh * p.blocks_per_group + now.hb, end < border ? end / (share + 1) : longer + (end - border) / share, cta);
            }
        }
        if (p.by_span && now.u0 == 0 && tid == 0) p.records[now.b * p.spans_per_row + now.kvh * p.blocks_per_group + now.hb] = record;
        hand_q(next_q);
        __syncthreads();  // the stage is a ring again
        now = next;
        if (more) pass.start(now.b, now.kvh, now.u0 * kUnit + warp * kTile, now.end);
    }
    if (tid == 0 && !p.by_span) p.records[cta] = record;
}

// Joins the pieces of a span (that of record blockIdx.x) that began in one CTA of the first kernel and went on in the CTAs after it, for
// one of its heads (blockIdx.y). There may be over a hundred pieces when one context is alone: a thread looks at a mark, and the warps
// share the pieces, so that the block waits for the record, the marks and the pieces once each. THREADS: 512 where a span has more than
// four pieces (one context of 131071 tokens 49 us, with 256 threads 53), else as many as the head has dimensions (128 at least), since the
// blocks themselves are the cost (300 contexts, 32 heads on 2 of 64: 30 us, with 640 threads 41), and the next kernel's blocks are let in
// when the pieces have come (128 contexts of 2000 tokens, 32 heads on 8 of 128: 121 us, let in at once 143).
template <int D, int NT, int THREADS>
__global__ void __launch_bounds__(THREADS) s1_attention_paged_join_kernel(const PagedParams p) {
    constexpr int kHeads = NT * kCols, kVec = D / 32, kJoinWarps = THREADS / 32;
    __shared__ float sums[kJoinWarps][D];
    __shared__ float weights[max_ctas(D)];
    __shared__ float tops[kJoinWarps], totals[kJoinWarps];
    griddep_wait();
    if (THREADS == 512) griddep_launch_dependents();
    const int4 rec = p.records[blockIdx.x];
    if (rec.z < 0) return;
    const int h = blockIdx.y, kvh = rec.y / p.blocks_per_group, hb = rec.y % p.blocks_per_group;
    if (h >= min(kHeads, p.group - hb * kHeads)) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int head = kvh * p.group + hb * kHeads + h;
    float gate = 0.f;
    if (p.gate && tid < D) gate = __bfloat162float(p.gate[rec.x * p.ldg + head * p.gate_head_stride + tid]);
    const int first = rec.w, pieces = rec.z - first + 1;  // piece i: of CTA first + i, its second (i = 0) or its first
    auto place = [&](int i) { return (2 * (first + i) + (i == 0 ? 1 : 0)) * kHeads + h; };
    const float2 mark = tid < pieces ? p.marks[place(tid)] : make_float2(-INFINITY, 0.f);
    float top = mark.x;
    for (int i = tid + THREADS; i < pieces; i += THREADS) top = fmaxf(top, p.marks[place(i)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, tops[w]);
    float sum = 0.f;
    auto weigh = [&](int i, const float2& m) {
        weights[i] = m.x == -INFINITY ? 0.f : exp2_fast(m.x - top);
        sum += weighed(m, top);
    };
    if (tid < pieces) weigh(tid, mark);
    for (int i = tid + THREADS; i < pieces; i += THREADS) weigh(i, p.marks[place(i)]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) totals[warp] = sum;
    __syncthreads();
    float x[kVec] = {};
#pragma unroll 4
    for (int i = warp; i < pieces; i += kJoinWarps) {
        const float f = weights[i];
        const float* part = p.parts + static_cast<long long>(place(i)) * D + lane;
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] = fmaf(f, __ldcg(part + 32 * e), x[e]);
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) sums[warp][lane + 32 * e] = x[e];
    if (THREADS != 512) griddep_launch_dependents();
    __syncthreads();
    if (tid < D) {
        float y = 0.f, total = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) y += sums[w][tid], total += totals[w];
        y = total == 0.f ? 0.f : y * rcp_fast(total);
        if (p.gate) y *= sigmoid_fast(gate);
        p.out[rec.x * p.ldo + head * D + tid] = __float2bfloat16_rn(y);
    }
}


size_t workspace_bytes_of(int head_dim) {
    return sizeof(int4) * max_ctas(head_dim) + 2 * max_ctas(head_dim) * 2 * kCols * (sizeof(float2) + sizeof(float) * static_cast<size_t>(head_dim));
}

template <int D, int NT, int W, int P>
int launch(s1_ctx* ctx, PagedParams p, int units) {
    constexpr int smem = W * WarpPass<D, NT, W, P>::kRingBytes;
    static std::atomic<unsigned long long> told{0};  // one bit per device
    if (!(told.load(std::memory_order_relaxed) >> (ctx->device & 63) & 1)) {
        S1_CUDA_OK(ctx, cudaFuncSetAttribute(s1_attention_paged_kernel<D, NT, W, P>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        told.fetch_or(1ull << (ctx->device & 63), std::memory_order_relaxed);
    }
    const int ctas = std::min({P * ctx->sm_count, max_ctas(D), units});  // no more than the block tables could make units of
    const long long spans = static_cast<long long>(p.num_seqs) * p.spans_per_row;
    // sixteen blocks of the join to every record: fewer records where there are fewer spans than CTAs (4 contexts of 66164 tokens, 64 heads on 4
    // of 64: 44 us, by CTA 46; with up to 8 heads the few blocks would crowd on a few SMs, one of 131071 51 us and 49)
    p.by_span = NT == 2 && spans <= ctas;
    S1_CUDA_OK(ctx, s1_launch_waiting(ctx, s1_attention_paged_kernel<D, NT, W, P>, static_cast<unsigned>(ctas), 1u, W * 32u, smem, p));
    ctx->launches += 1;
    // a span of one unit is never cut: block tables that hold no more than a unit leave nothing to join (one context of 17 tokens in a
    // table of 32: 7.3 us with the second kernel, 6.3 without). Callers that cut their tables to what is used have this; those of a
    // `PagedCache` are as wide as its longest row may get.
    if (static_cast<long long>(p.table_width) << p.shift <= WarpPass<D, NT, W, P>::kUnit) return S1_OK;
    constexpr int kThreads = D == 256 ? 256 : 128;
    const bool many = 4 * spans >= ctas;  // four pieces to a span at most, were all spans alike
    S1_CUDA_OK(ctx, s1_launch_waiting(ctx, many ? s1_attention_paged_join_kernel<D, NT, kThreads> : s1_attention_paged_join_kernel<D, NT, 512>,
                                      static_cast<unsigned>(p.by_span ? spans : ctas), static_cast<unsigned>(std::min(NT * kCols, p.group)),
                                      many ? kThreads : 512u, 0, p));
    ctx->launches += 1;
    return S1_OK;
}

template <int D>
int launch(s1_ctx* ctx, const PagedParams& p, int units) {
    const bool wide = p.group > kCols, many = static_cast<long long>(p.num_seqs) * p.spans_per_row >= 3ll * ctx->sm_count;
    if (wide) return many ? launch<D, 2, 4, 2>(ctx, p, units) : launch<D, 2, 8, D == 64 ? 2 : 1>(ctx, p, units);
    return many ? launch<D, 1, 4, D == 256 ? 2 : D == 128 ? 3 : 4>(ctx, p, units) : launch<D, 1, 8, D == 256 ? 1 : 2>(ctx, p, units);
}

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

extern "C" size_t s1_attention_paged_workspace(int head_dim) {
    return head_dim == 64 || head_dim == 128 || head_dim == 256 ? workspace_bytes_of(head_dim) : 0;
}

extern "C" int s1_attention_paged(s1_ctx* ctx, const void* q, long long ldq, long long q_head_stride, const void* k_cache, const void* v_cache,
                                  int num_pages, int page_size, long long page_stride, long long token_stride, long long head_stride,
                                  const int32_t* tables, long long ldt, int table_width, const int32_t* lengths, int num_seqs, int heads, int kv_heads,
                                  int head_dim, float scale, const void* gate, long long ldg, long long gate_head_stride, void* out, long long ldo,
                                  void* workspace, size_t workspace_bytes) {
    if (!ctx) return S1_EINVAL;
    const char* who = "s1_attention_paged";
    if (!q || !k_cache || !v_cache || !tables || !lengths || !out || !workspace) return s1_fail(ctx, S1_EINVAL, "%s: null pointer", who);
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return s1_fail(ctx, S1_EINVAL, "%s: head_dim must be 64, 128 or 256 (got %d)", who, head_dim);
    if (num_seqs < 0 || kv_heads < 1 || heads < kv_heads || heads % kv_heads) return s1_fail(ctx, S1_EINVAL, "%s: heads must be a multiple of kv_heads", who);
    // (scores are kept in units of log 2: the scale times log2(e) has to be finite too)
    if (!(scale > 0.f) || !(scale < 2.35e38f)) return s1_fail(ctx, S1_EINVAL, "%s: scale must be positive and below 2.35e38", who);
    if (num_pages < 1 || page_size < 1 || page_size > 65536 || (page_size & (page_size - 1)))
        return s1_fail(ctx, S1_EINVAL, "%s: page_size must be a power of two up to 65536 (got %d)", who, page_size);
    if (static_cast<long long>(table_width) * page_size > (1ll << 30)) return s1_fail(ctx, S1_EINVAL, "%s: block tables of over 2^30 tokens a row", who);
    if (table_width < 1 || ldt < table_width) return s1_fail(ctx, S1_EINVAL, "%s: bad block tables", who);
    if (!al16(q) || !al16(k_cache) || !al16(v_cache) || !al16(out) || !al16(workspace) || ((ldq | q_head_stride | page_stride | token_stride | head_stride | ldo) % 8))
        return s1_fail(ctx, S1_EINVAL, "%s: head rows and the workspace must be 16-byte aligned", who);
    if (q_head_stride < head_dim || ldq < (heads - 1) * q_head_stride + head_dim || ldo < static_cast<long long>(heads) * head_dim)
        return s1_fail(ctx, S1_EINVAL, "%s: heads must lie inside a row", who);
    if (page_stride < head_dim || token_stride < head_dim || head_stride < head_dim) return s1_fail(ctx, S1_EINVAL, "%s: bad cache strides", who);
    if (gate && ((reinterpret_cast<uintptr_t>(gate) & 3u) || ((ldg | gate_head_stride) % 2))) return s1_fail(ctx, S1_EINVAL, "%s: gate rows must be 4-byte aligned", who);
    if (gate && (gate_head_stride < head_dim || ldg < (heads - 1) * gate_head_stride + head_dim))
        return s1_fail(ctx, S1_EINVAL, "%s: gate heads must lie inside a row", who);
    if (workspace_bytes < workspace_bytes_of(head_dim))
        return s1_fail(ctx, S1_EINVAL, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, workspace_bytes_of(head_dim));
    if (num_seqs == 0) return S1_OK;
    S1DeviceGuard guard(ctx->device);
    if (!guard.ok) return s1_fail(ctx, S1_ECUDA, "%s: cudaSetDevice(%d) failed", who, ctx->device);
    const int group = heads / kv_heads, columns = group > kCols ? 2 * kCols : kCols, blocks = (group + columns - 1) / columns;
    // the costs of all spans, with the smaller units, have to fit 31 bits
    const long long spans = static_cast<long long>(num_seqs) * kv_heads * blocks, cost = static_cast<long long>(table_width) * page_size / (4 * kTile) + 5;
    if (spans > (1ll << 31) / cost - 1) return s1_fail(ctx, S1_EINVAL, "%s: rows x KV heads x (tokens of a block table) / 64 must be below 2^31", who);
    float2* marks = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + sizeof(int4) * max_ctas(head_dim));
    PagedParams p{static_cast<const __nv_bfloat16*>(q), ldq, q_head_stride, static_cast<const __nv_bfloat16*>(k_cache),
                  static_cast<const __nv_bfloat16*>(v_cache), page_stride, token_stride, head_stride, num_pages, __builtin_ctz(page_size), tables, ldt,
                  table_width, lengths, num_seqs, heads, kv_heads, group, kv_heads * blocks, blocks, scale * 1.4426950408889634f,
                  static_cast<const __nv_bfloat16*>(gate), ldg, gate_head_stride, static_cast<__nv_bfloat16*>(out), ldo,
                  reinterpret_cast<float*>(marks + 2 * max_ctas(head_dim) * 2 * kCols), marks, static_cast<int4*>(workspace), false, ctx->status_dev};
    const int units = static_cast<int>(std::min(spans * cost, 1ll << 30));
    return head_dim == 64 ? launch<64>(ctx, p, units) : head_dim == 128 ? launch<128>(ctx, p, units) : launch<256>(ctx, p, units);
}
