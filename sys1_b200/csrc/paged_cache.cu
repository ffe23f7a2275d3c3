// The bookkeeping and the writer of a paged key-value cache. The cache of a layer is two tensors of `num_pages` pages, a page
// holding `page_size` tokens (a power of two) of every KV head; a request's tokens lie in the pages its block table row names,
// and a token's slot is page * page_size + (position mod page_size).
//   s1_block_tables    takes pages for the tokens that a step adds, from a stack of free page ids, and writes the block tables,
//                      the new lengths and every token's position and slot
//   s1_release_blocks  puts the pages of requests that have ended back on the stack
//   s1_cache_write     copies keys and values into their slots; the keys may be normed and rotated on the way
// The reference keeps no cache (its decoder runs whole prompts, src/archs/qwen35_text.rs:982-1005): these have no counterpart there.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "context.h"
#include "device_guard.h"
#include "head_norm_rope.cuh"
#include "ptx.cuh"

using namespace s1;
namespace cg = cooperative_groups;

namespace {

constexpr int kTableThreads = 1024;
constexpr unsigned kFull = 1u << 30;  // sums of tokens and pages stop here: beyond every limit, and two of them still fit 32 bits

__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) { return min(a + b, kFull); }

// Inclusive prefix sum over the block's threads; `warp_sums` holds 33 words, the last of them the block's total afterwards.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = add_sat(v, t);
    }
    __syncthreads();  // the sums of the scan before this one have been read
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        unsigned s = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned t = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s = add_sat(s, t);
        }
        const unsigned before = __shfl_up_sync(0xffffffffu, s, 1);
        warp_sums[lane] = lane ? before : 0u;
        if (lane == 31) warp_sums[32] = s;
    }
    __syncthreads();
    return add_sat(v, warp_sums[warp]);
}

__device__ __forceinline__ void report(int* status, int code, int where, int value) {
    if (atomicCAS(status, 0, code) == 0) {
        status[1] = static_cast<int>(blockIdx.x);
        status[2] = where;
        status[3] = value;
    }
}

struct TableParams {
    const int32_t* cached;
    const int32_t* added;  // null: one token each
    int num_seqs, shift;   // page_size = 1 << shift
    const int32_t* free_pages;
    int free_capacity;
    const int32_t* free_count;
    int32_t* free_count_out;
    int32_t* tables;
    long long ldt;
    int table_width;
    int32_t* lengths;
    int32_t* cu_seqlens;
    int32_t* positions;
    int32_t* slots;
    int max_tokens;
    int* status;
};

// Latency is all there is here: a few kilobytes in and out, and the prefix sums over the rows in between. Every block of the
// (one) cluster forms the sums for itself, which costs less than handing them round, and then takes its share of the tokens.
// The cluster's barrier between the last read of an input and the first write lets `lengths` be `cached` and
// `free_count_out` be `free_count`: a step captured into a graph then advances the same buffers at every replay. Measured: 8 rows of one token 2.9 us, 1024 rows 3.6, 31
// prompts of 16399 tokens 6.2.
__global__ void __launch_bounds__(kTableThreads) s1_block_tables_kernel(const TableParams p) {
    extern __shared__ int32_t rows_smem[];
    int32_t* cu = rows_smem;                      // [num_seqs + 1] first token of every row
    int32_t* off = cu + p.num_seqs + 1;           // [num_seqs] first page taken, -1: the row was refused
    int32_t* old = off + p.num_seqs;              // [num_seqs] tokens before this call, negative: idle
    __shared__ unsigned warp_sums[33];
    __shared__ unsigned taken_sh;
    griddep_wait();
    griddep_launch_dependents();
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), blocks = static_cast<int>(cluster.num_blocks());
    const int tid = threadIdx.x;
    const unsigned have_pages = static_cast<unsigned>(min(max(*p.free_count, 0), p.free_capacity));
    if (tid == 0) taken_sh = 0u, cu[0] = 0;
    unsigned tokens = 0, pages = 0;
    for (int b0 = 0; b0 < p.num_seqs; b0 += kTableThreads) {
        const int b = b0 + tid;
        const bool row = b < p.num_seqs;
        const int was = row ? p.cached[b] : -1;
        const bool idle = was < 0;
        const unsigned add = idle ? 0u : p.added ? static_cast<unsigned>(max(p.added[b], 0)) : 1u;
        // in the one-token form token b belongs to row b, idle or not; in the packed form idle rows have no tokens
        const unsigned takes = !row ? 0u : p.added ? min(add, kFull) : 1u;
        const unsigned end = add_sat(tokens, block_scan(takes, warp_sums));
        tokens = add_sat(tokens, warp_sums[32]);
        const long long now = static_cast<long long>(max(was, 0)) + add;
        const long long mask = (1ll << p.shift) - 1;
        const long long had = (max(was, 0) + mask) >> p.shift, want = (now + mask) >> p.shift;
        const bool holds = want <= p.table_width && now <= 2147483647ll;  // lengths and positions are 32 bits, whatever the table could hold
        const bool fits = holds && end <= static_cast<unsigned>(p.max_tokens);
        const unsigned need = (row && fits) ? static_cast<unsigned>(want - had) : 0u;
        const unsigned upto = add_sat(pages, block_scan(need, warp_sums));
        pages = add_sat(pages, warp_sums[32]);
        if (row) {
            const bool served = fits && (need == 0 || upto <= have_pages);
            cu[b + 1] = static_cast<int>(end);
            off[b] = served ? static_cast<int>(upto - need) : -1;
            old[b] = was;
            if (served && need) atomicMax(&taken_sh, upto);
            if (!served && rank == 0) report(p.status, !holds ? 110 : !fits ? 112 : 111, b, static_cast<int>(min(now, 2147483647ll)));
        }
    }
    __syncthreads();
    // what the tokens read: the block tables' pages that are partly filled (never written here) and the free pages (never written)
    cluster.sync();  // every block has read every row's length and the count
    const unsigned taken = taken_sh;
    for (int b = rank * kTableThreads + tid; b < p.num_seqs; b += blocks * kTableThreads) {
        const int was = old[b];
        const int add = was < 0 ? 0 : p.added ? max(p.added[b], 0) : 1;
        p.lengths[b] = off[b] < 0 ? was : was + add;
        if (p.cu_seqlens) p.cu_seqlens[b + 1] = cu[b + 1];
    }
    if (rank == 0 && tid == 0) {
        if (p.cu_seqlens) p.cu_seqlens[0] = 0;
        *p.free_count_out = static_cast<int>(have_pages - taken);
    }
    const int total = cu[p.num_seqs];
    for (int t = rank * kTableThreads + tid; t < p.max_tokens; t += blocks * kTableThreads) {
        int slot = -1, pos = 0;
        if (t < total) {
            int b = t;
            if (p.added) {  // the last row that starts at or before t (rows without tokens start where the next one does)
                int lo = 0, hi = p.num_seqs;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (cu[mid] <= t) lo = mid;
                    else hi = mid;
                }
                b = lo;
            }
            const int was = old[b];
            if (was >= 0 && off[b] >= 0) {
                pos = was + (t - cu[b]);
                const int pg = pos >> p.shift, in = pos & ((1 << p.shift) - 1);
                const int had = static_cast<int>((static_cast<long long>(was) + (1ll << p.shift) - 1) >> p.shift);
                int32_t* entry = p.tables + b * p.ldt + pg;
                int page;
                if (pg < had) {
                    page = *entry;
                } else {
                    page = p.free_pages[have_pages - 1 - static_cast<unsigned>(off[b] + pg - had)];
                    if (in == 0) *entry = page;  // a new page is always entered at its first token
                }
                const long long s = (static_cast<long long>(page) << p.shift) + in;
                if (page < 0 || s > 2147483647ll) report(p.status, 113, b, page);
                else slot = static_cast<int>(s);
            }
        }
        p.positions[t] = pos;
        p.slots[t] = slot;
    }
}

struct ReleaseParams {
    const int32_t* ended;
    int num_seqs, shift;
    int32_t* lengths;
    const int32_t* tables;
    long long ldt;
    int table_width;
    int32_t* free_pages;
    int free_capacity;
    int32_t* free_count;
    int* status;
};

__global__ void __launch_bounds__(kTableThreads) s1_release_blocks_kernel(const ReleaseParams p) {
    extern __shared__ int32_t rows_smem[];
    int32_t* off = rows_smem;           // [num_seqs] first entry of the row's pages on the stack
    int32_t* num = off + p.num_seqs;    // [num_seqs] pages to put back
    __shared__ unsigned warp_sums[33];
    __shared__ unsigned put_sh;
    const int tid = threadIdx.x;
    griddep_wait();
    griddep_launch_dependents();
    const unsigned held = static_cast<unsigned>(min(max(*p.free_count, 0), p.free_capacity));
    if (tid == 0) put_sh = 0u;
    unsigned pages = 0;
    for (int b0 = 0; b0 < p.num_seqs; b0 += kTableThreads) {
        const int b = b0 + tid;
        const bool ends = b < p.num_seqs && p.ended[b] != 0;
        const int len = ends ? max(p.lengths[b], 0) : 0;
        const long long n = (static_cast<long long>(len) + (1ll << p.shift) - 1) >> p.shift;
        const bool fits = n <= p.table_width;
        const unsigned give = fits ? static_cast<unsigned>(n) : 0u;
        const unsigned upto = add_sat(pages, block_scan(give, warp_sums));
        pages = add_sat(pages, warp_sums[32]);
        if (b < p.num_seqs) {
            const bool room = held + upto <= static_cast<unsigned>(p.free_capacity);
            off[b] = static_cast<int>(held + upto - give);
            num[b] = room ? static_cast<int>(give) : 0;
            if (ends) {
                if (fits && (room || give == 0)) {
                    p.lengths[b] = -1;
                    if (give) atomicMax(&put_sh, upto);
                } else {
                    report(p.status, fits ? 115 : 114, b, len);
                }
            }
        }
    }
    __syncthreads();
    const int warp = tid >> 5, lane = tid & 31;
    for (int b = warp; b < p.num_seqs; b += kTableThreads / 32)
        for (int i = lane; i < num[b]; i += 32) p.free_pages[off[b] + i] = p.tables[b * p.ldt + i];
    if (tid == 0) *p.free_count = static_cast<int>(held + put_sh);
}

// ------------------------------------------------------------------------------------------------------ cache write
struct WriteParams {
    const __nv_bfloat16* k;
    long long ldk, k_head_stride;
    const __nv_bfloat16* v;
    long long ldv, v_head_stride;
    const int32_t* slots;
    int T, kv_heads;
    unsigned heads_mul;  // row / kv_heads = row * heads_mul >> heads_shift for row < 2^30
    int heads_shift;
    const __nv_bfloat16* norm_w;
    float eps;
    const float* cos_t;
    const float* sin_t;
    const int32_t* positions;
    int max_pos, rot, bf16_ops;
    __nv_bfloat16* k_cache;
    __nv_bfloat16* v_cache;
    long long num_slots;
    int shift;
    long long page_stride, token_stride, head_stride;
    int* status;
};

constexpr int kWriteThreads = 128, kWriteWarps = kWriteThreads / 32;

// LPR lanes hold one head row, two pieces of 16 bytes each, the halves of the row. Streaming: every value is read and written once.
// Where keys are only copied, a warp takes keys or values (every other warp): short, with two loads a lane on the way (16384 tokens x 4
// heads of 256: 21.2 us = 6.3 TB/s, 1918 x 8 4.6; with 46 registers instead of 32 a thread 21.5 and 5.0, with keys and values of a row in
// one lane 21.4 and 4.8, with one piece a lane and 32 lanes a row 27 and 5.5). With the norm, which costs 250 instructions a row and warp,
// a lane takes a row's key and value: the value's way and the indices come free under the arithmetic (7799 tokens x 4 heads of 256, 32
// rotated: 12.0 us = 5.1 TB/s; keys and values in warps of their own 15.4, and 22.6 with 32 lanes a row, whose exchanges and square roots
// serve half as many columns).
template <int LPR, bool NORM>
__global__ void __launch_bounds__(kWriteThreads, NORM ? 9 : 16) s1_cache_write_kernel(const WriteParams p) {
    constexpr int RPW = 32 / LPR;
    const int lane = threadIdx.x & 31, sub = lane % LPR;
    griddep_wait();
    griddep_launch_dependents();
    unsigned warp = blockIdx.x * kWriteWarps + (threadIdx.x >> 5);  // (warps are counted: threads may pass 32 bits)
    const bool keys = NORM || (warp & 1u) == 0, values = NORM || !keys;
    if (!NORM) warp >>= 1;
    const unsigned row = warp * RPW + lane / LPR;
    bool live = row < static_cast<unsigned>(p.T) * static_cast<unsigned>(p.kv_heads);
    const int t = live ? static_cast<int>(static_cast<unsigned long long>(row) * p.heads_mul >> p.heads_shift) : 0, h = live ? static_cast<int>(row) - t * p.kv_heads : 0;
    const long long slot = live ? p.slots[t] : -1;
    const int pos = NORM && live ? p.positions[t] : 0;
    uint4 k[2] = {}, v[2] = {};
    if (live && keys) {  // (plain loads: see s1_launch_waiting)
        const uint4* src = reinterpret_cast<const uint4*>(p.k + t * p.ldk + h * p.k_head_stride + sub * 8);
        k[0] = src[0], k[1] = src[LPR];
    }
    if (live && values) {
        const uint4* src = reinterpret_cast<const uint4*>(p.v + t * p.ldv + h * p.v_head_stride + sub * 8);
        v[0] = src[0], v[1] = src[LPR];
    }
    live = live && slot >= 0;  // tokens without a slot are left out
    if (live && slot >= p.num_slots) {
        report(p.status, 116, t, static_cast<int>(slot));
        live = false;
    }
    const long long at = (slot >> p.shift) * p.page_stride + (slot & ((1ll << p.shift) - 1)) * p.token_stride + h * p.head_stride + sub * 8;
    if (live && values) {
        uint4* dst = reinterpret_cast<uint4*>(p.v_cache + at);
        dst[0] = v[0], dst[LPR] = v[1];
    }
    if (NORM) {
        const int halfc = p.rot / 16;
        const bool rotates = live && sub < 2 * halfc, pos_ok = pos >= 0 && pos < p.max_pos;
        float c[8], sn[8];
        load_rotation<false>(p.cos_t, p.sin_t, pos_ok ? pos : 0, p.rot, sub, c, sn);  // (whatever the slot says, which may still be on its way)
        head_norm_rope<LPR>(k, p.norm_w, p.eps, c, sn, rotates && pos_ok, sub, halfc, p.bf16_ops);
        if (rotates && !pos_ok) report(p.status, 102, t, pos);
    }
    if (live && keys) {
        uint4* dst = reinterpret_cast<uint4*>(p.k_cache + at);
        dst[0] = k[0], dst[LPR] = k[1];
    }
}

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

constexpr int kMaxTableRows = 8192;

extern "C" int s1_block_tables(s1_ctx* ctx, const int32_t* cached, const int32_t* added, int num_seqs, int page_size, const int32_t* free_pages,
                               int free_capacity, const int32_t* free_count, int32_t* free_count_out, int32_t* tables, long long ldt, int table_width,
                               int32_t* lengths, int32_t* cu_seqlens, int32_t* positions, int32_t* slots, int max_tokens) {
    if (!ctx) return S1_EINVAL;
    const char* who = "s1_block_tables";
    if (!cached || !free_count || !free_count_out || !lengths) return s1_fail(ctx, S1_EINVAL, "%s: null pointer", who);
    if (num_seqs < 1 || num_seqs > kMaxTableRows) return s1_fail(ctx, S1_EINVAL, "%s: 1 to %d rows (got %d)", who, kMaxTableRows, num_seqs);
    if (page_size < 1 || page_size > 65536 || (page_size & (page_size - 1)))
        return s1_fail(ctx, S1_EINVAL, "%s: page_size must be a power of two up to 65536 (got %d)", who, page_size);
    if (free_capacity < 0 || free_capacity >= (1 << 30) || (free_capacity > 0 && !free_pages)) return s1_fail(ctx, S1_EINVAL, "%s: bad stack of free pages", who);
    if (table_width < 1 || ldt < table_width || !tables) return s1_fail(ctx, S1_EINVAL, "%s: bad block tables", who);
    if (max_tokens < 0 || max_tokens >= (1 << 30) || (max_tokens > 0 && (!positions || !slots))) return s1_fail(ctx, S1_EINVAL, "%s: bad token count", who);
    if (!added && max_tokens != num_seqs)
        return s1_fail(ctx, S1_EINVAL, "%s: without `added` every row has one token (max_tokens %d, rows %d)", who, max_tokens, num_seqs);
    S1DeviceGuard guard(ctx->device);
    if (!guard.ok) return s1_fail(ctx, S1_ECUDA, "%s: cudaSetDevice(%d) failed", who, ctx->device);
    TableParams p{cached, added, num_seqs, __builtin_ctz(page_size), free_pages, free_capacity, free_count, free_count_out, tables, ldt, table_width,
                  lengths, cu_seqlens, positions, slots, max_tokens, ctx->status_dev};
    const int smem = static_cast<int>(sizeof(int32_t)) * (3 * num_seqs + 1);
    static std::atomic<unsigned long long> told{0};  // one bit per device
    if (!(told.load(std::memory_order_relaxed) >> (ctx->device & 63) & 1)) {
        S1_CUDA_OK(ctx, cudaFuncSetAttribute(s1_block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * (3 * kMaxTableRows + 1)));
        told.fetch_or(1ull << (ctx->device & 63), std::memory_order_relaxed);
    }
    // one block up to four tokens a thread, then more blocks, up to the eight of a portable cluster
    const unsigned blocks = max_tokens <= 4 * kTableThreads ? 1u : max_tokens <= 8 * kTableThreads ? 2u : max_tokens <= 16 * kTableThreads ? 4u : 8u;
    S1_CUDA_OK(ctx, s1_launch_waiting(ctx, s1_block_tables_kernel, blocks, 1u, kTableThreads, smem, p, blocks));
    ctx->launches += 1;
    return S1_OK;
}

extern "C" int s1_release_blocks(s1_ctx* ctx, const int32_t* ended, int num_seqs, int page_size, int32_t* lengths, const int32_t* tables, long long ldt,
                                 int table_width, int32_t* free_pages, int free_capacity, int32_t* free_count) {
    if (!ctx) return S1_EINVAL;
    const char* who = "s1_release_blocks";
    if (!ended || !lengths || !tables || !free_pages || !free_count) return s1_fail(ctx, S1_EINVAL, "%s: null pointer", who);
    if (num_seqs < 1 || num_seqs > kMaxTableRows) return s1_fail(ctx, S1_EINVAL, "%s: 1 to %d rows (got %d)", who, kMaxTableRows, num_seqs);
    if (page_size < 1 || page_size > 65536 || (page_size & (page_size - 1)))
        return s1_fail(ctx, S1_EINVAL, "%s: page_size must be a power of two up to 65536 (got %d)", who, page_size);
    if (table_width < 1 || ldt < table_width) return s1_fail(ctx, S1_EINVAL, "%s: bad block tables", who);
    if (free_capacity < 0 || free_capacity >= (1 << 30)) return s1_fail(ctx, S1_EINVAL, "%s: bad stack of free pages", who);
    S1DeviceGuard guard(ctx->device);
    if (!guard.ok) return s1_fail(ctx, S1_ECUDA, "%s: cudaSetDevice(%d) failed", who, ctx->device);
    ReleaseParams p{ended, num_seqs, __builtin_ctz(page_size), lengths, tables, ldt, table_width, free_pages, free_capacity, free_count, ctx->status_dev};
    const int smem = static_cast<int>(sizeof(int32_t)) * 2 * num_seqs;
    S1_CUDA_OK(ctx, cudaFuncSetAttribute(s1_release_blocks_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * 2 * kMaxTableRows));
    S1_CUDA_OK(ctx, s1_launch_waiting(ctx, s1_release_blocks_kernel, 1u, 1u, kTableThreads, smem, p));
    ctx->launches += 1;
    return S1_OK;
}

extern "C" int s1_cache_write(s1_ctx* ctx, const void* k, long long ldk, long long k_head_stride, const void* v, long long ldv, long long v_head_stride,
                              const int32_t* slots, int total_tokens, int kv_heads, int head_dim, const void* norm_weight, float eps,
                              const float* cos_table, const float* sin_table, const int32_t* positions, int max_positions, int rotary_dim, int bf16_ops,
                              void* k_cache, void* v_cache, int num_pages, int page_size, long long page_stride, long long token_stride,
                              long long head_stride) {
    if (!ctx) return S1_EINVAL;
    const char* who = "s1_cache_write";
    if (!k || !v || !slots || !k_cache || !v_cache) return s1_fail(ctx, S1_EINVAL, "%s: null pointer", who);
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return s1_fail(ctx, S1_EINVAL, "%s: head_dim must be 64, 128 or 256 (got %d)", who, head_dim);
    if (total_tokens < 0 || kv_heads < 1 || num_pages < 1) return s1_fail(ctx, S1_EINVAL, "%s: bad sizes", who);
    if (page_size < 1 || page_size > 65536 || (page_size & (page_size - 1)))
        return s1_fail(ctx, S1_EINVAL, "%s: page_size must be a power of two up to 65536 (got %d)", who, page_size);
    if (!al16(k) || !al16(v) || !al16(k_cache) || !al16(v_cache) ||
        ((ldk | k_head_stride | ldv | v_head_stride | page_stride | token_stride | head_stride) % 8))
        return s1_fail(ctx, S1_EINVAL, "%s: head rows must be 16-byte aligned", who);
    if (k_head_stride < head_dim || v_head_stride < head_dim || ldk < (kv_heads - 1) * k_head_stride + head_dim || ldv < (kv_heads - 1) * v_head_stride + head_dim)
        return s1_fail(ctx, S1_EINVAL, "%s: heads must lie inside a token's row", who);
    if (page_stride < head_dim || token_stride < head_dim || head_stride < head_dim) return s1_fail(ctx, S1_EINVAL, "%s: bad cache strides", who);
    if (norm_weight) {
        if (!cos_table || !sin_table || !positions) return s1_fail(ctx, S1_EINVAL, "%s: null pointer", who);
        if (rotary_dim != 16 && rotary_dim != 32 && rotary_dim != 64 && rotary_dim != 128 && rotary_dim != 256)
            return s1_fail(ctx, S1_EINVAL, "%s: rotary_dim must be 16, 32, 64, 128 or 256 (got %d)", who, rotary_dim);
        if (rotary_dim > head_dim || max_positions < 1) return s1_fail(ctx, S1_EINVAL, "%s: rotary_dim exceeds head_dim, or no positions", who);
        if (!al16(norm_weight) || !al16(cos_table) || !al16(sin_table)) return s1_fail(ctx, S1_EINVAL, "%s: weight and tables must be 16-byte aligned", who);
    }
    if (total_tokens == 0) return S1_OK;
    const int lpr = head_dim / 16;
    const long long rows = 1LL * total_tokens * kv_heads, warps = (rows * lpr + 31) / 32 * (norm_weight ? 1 : 2), blocks = (warps + kWriteWarps - 1) / kWriteWarps;
    if (rows > (1LL << 29)) return s1_fail(ctx, S1_EINVAL, "%s: too many rows", who);
    int shift = 30;  // 2^(shift - 30) >= kv_heads: then the product is off by less than a row's worth for every row below 2^30
    while (1LL << (shift - 30) < kv_heads) ++shift;
    const unsigned mul = static_cast<unsigned>(((1ULL << shift) + kv_heads - 1) / kv_heads);
    S1DeviceGuard guard(ctx->device);
    if (!guard.ok) return s1_fail(ctx, S1_ECUDA, "%s: cudaSetDevice(%d) failed", who, ctx->device);
    WriteParams p{static_cast<const __nv_bfloat16*>(k), ldk, k_head_stride, static_cast<const __nv_bfloat16*>(v), ldv, v_head_stride, slots, total_tokens,
                  kv_heads, mul, shift, static_cast<const __nv_bfloat16*>(norm_weight), eps, cos_table, sin_table, positions, max_positions, rotary_dim, bf16_ops,
                  static_cast<__nv_bfloat16*>(k_cache), static_cast<__nv_bfloat16*>(v_cache), static_cast<long long>(num_pages) * page_size,
                  __builtin_ctz(page_size), page_stride, token_stride, head_stride, ctx->status_dev};
    auto launch = [&](void (*kernel)(WriteParams)) { return s1_launch_waiting(ctx, kernel, static_cast<unsigned>(blocks), 1u, static_cast<unsigned>(kWriteThreads), 0, p); };
#define S1_WRITE(LPR_) launch(norm_weight ? s1_cache_write_kernel<LPR_, true> : s1_cache_write_kernel<LPR_, false>)
    S1_CUDA_OK(ctx, lpr == 4 ? S1_WRITE(4) : lpr == 8 ? S1_WRITE(8) : S1_WRITE(16));
#undef S1_WRITE
    ctx->launches += 1;
    return S1_OK;
}
