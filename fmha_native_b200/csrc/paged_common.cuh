// paged_common.cuh -- what the kernels over the paged K/V cache share: their
// arguments, the addressing of query rows, bounded waits and the folding of
// partial softmax results.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "host_context.h"
#include "sm100_ptx.cuh"

namespace fmha_paged {

using namespace fmha_sm100;

constexpr int kHeadDim = 64;
constexpr float kLn2 = 0.69314718055994531f;
constexpr int kMostKeys = 0x7fffffff - 4096;  // of a sequence: places are counted in 32 bits, tiles past them too

// Rows.  The new tokens of a call are numbered f = 0 .. tokens-1 (dense:
// batch * seqlen_q + index; packed: the packed index).  For one K/V head the
// rows of a sequence are (token, query head of the group), group fastest:
// row r is token r / group, query head kvh * group + r % group, so all rows
// that read the same keys sit in one tile.
enum : int { kPlanNone, kPlanHere, kPlanList };
struct TileItem;

struct Args {
    CUtensorMap tm_k;
    CUtensorMap tm_v;
    const uint16_t* q;
    uint16_t* o;
    float* lse;                 // or null
    const int32_t* page_table;
    const int32_t* seqlens_k;   // null: every sequence has fixed_len keys
    const int32_t* seqstart_q;  // null: dense
    long long table_stride;
    long long stride_q, nhead_stride_q, batch_stride_q;
    long long stride_o, nhead_stride_o, batch_stride_o;
    int batch, seqlen_q, tokens;
    int nhead_q, nhead_k, group;
    int page_shift, num_pages, max_pages;
    int fixed_len;
    int causal;
    int row_div;                // tokens per batch entry of q/o (packed: INT_MAX)
    int lse_len;                // seqlen_q or total_q
    float scale;                // softmax scale * log2(e)
    // Sequences whose rows per K/V head lie in [min_rows, max_rows] take part.
    int min_rows, max_rows;
    int row_cap;                // rows per K/V head that a sequence of the rows kernel may have
    // Partial results of other launches that the final rows fold in: part_n
    // of them, [part][token * nhead_q + head], normalised O and its LSE in
    // log2 units (-inf: nothing, O unwritten).
    const float* part_o;
    const float* part_lse;
    int part_n;
    // Where a launch that makes such partial results puts its own (a prefix's
    // split s into slot s); null: it writes final rows.
    float* out_o;
    float* out_lse;
    int plan;                   // tile kernel: where its blocks' work comes from
    int splits;                 // kPlanNone: key ranges per row tile
    TileItem* items;            // kPlanList: the list, its length, and scratch to make it
    int* item_count;
    int* tile_first;
    int max_tiles;              // row tiles that the host made room for
    float* slots;               // scratch of the jobs that blocks share
    int max_slots;
    float* pieces;              // rows kernel: scratch between its blocks
    int group_blocks;           // rows kernel: blocks of each group, the groups share out the K/V heads
    int group_heads;
    int2* seq_parts;            // rows kernel under a prefix: per sequence its first block (of each
                                // group) and, if it crosses blocks, how many share it
    int end_merge;              // blocks of the call's last kernel that merge the rows kernel's pieces
    int* err_word;
    unsigned long long wait_limit_ns;
};

__device__ __forceinline__ void flag_index_error(int* err_word) {
    atomicCAS(err_word, 0, fmha_host::kErrIndex);
}

// A sequence as the kernels see it; index data out of range is flagged and
// cut to what memory holds.
struct Sequence {
    int first;   // number of its first new token
    int count;   // new tokens
    int keys;    // keys in the cache
};

__device__ __forceinline__ Sequence load_sequence(const Args& a, int b) {
    Sequence s;
    int past = 0;  // tokens beyond what the call said: only the ones before them are worked on
    if (a.seqstart_q != nullptr) {
        s.first = a.seqstart_q[b];
        s.count = a.seqstart_q[b + 1] - s.first;
        if (s.first < 0 || s.count < 0 || s.first > a.tokens - s.count) {
            flag_index_error(a.err_word);
            s.first = s.count = 0;
        }
        if (s.count > a.seqlen_q) {
            flag_index_error(a.err_word);
            past = s.count - a.seqlen_q;
            s.count = a.seqlen_q;
        }
    } else {
        s.first = b * a.seqlen_q;
        s.count = a.seqlen_q;
    }
    if (a.seqlens_k != nullptr) {
        s.keys = max(a.seqlens_k[b], 0);
        const long long cap = min((long long)a.max_pages << a.page_shift, (long long)kMostKeys);
        if (s.keys > cap) {
            flag_index_error(a.err_word);
            s.keys = (int)cap;
        }
        s.keys = max(s.keys - past, 0);
    } else {
        s.keys = a.fixed_len;
    }
    return s;
}

// Keys visible to new token t of a sequence: [0, limit).
__device__ __forceinline__ int key_limit(const Args& a, const Sequence& s, int t) {
    return a.causal ? min(s.keys, s.keys - s.count + t + 1) : s.keys;
}

__device__ __forceinline__ const uint16_t* q_row(const Args& a, int token, int head) {
    const int b = token / a.row_div;
    return a.q + b * a.batch_stride_q + (long long)(token - b * a.row_div) * a.stride_q +
           head * a.nhead_stride_q;
}
__device__ __forceinline__ uint16_t* o_row(const Args& a, int token, int head) {
    const int b = token / a.row_div;
    return a.o + b * a.batch_stride_o + (long long)(token - b * a.row_div) * a.stride_o +
           head * a.nhead_stride_o;
}
__device__ __forceinline__ float* lse_at(const Args& a, int token, int head) {
    const int b = token / a.row_div;
    return a.lse + ((long long)b * a.nhead_q + head) * a.lse_len + (token - b * a.row_div);
}
__device__ __forceinline__ long long flat_row(const Args& a, int token, int head) {
    return (long long)token * a.nhead_q + head;
}

// Running state of a softmax over disjoint sets of keys: reference maximum m
// (log2 units), weight sum l, and O un-normalised, all fp32.  No key seen: m is
// -inf and l is 0.  A NaN among the scores (or +inf, whose softmax has none but
// inf - inf) makes l NaN, and so whatever it is folded into.
// fold_scales: factors for the state (m, l) and for a newcomer (m2, l2).
struct Fold {
    float keep, take;
};
__device__ __forceinline__ Fold fold_scales(float& m, float m2) {
    const float mn = fmaxf(m, m2);
    Fold f;
    f.keep = m == -INFINITY ? 0.0f : ex2_approx(m - mn);
    f.take = m2 == -INFINITY ? 0.0f : ex2_approx(m2 - mn);
    m = mn;
    return f;
}

__device__ __forceinline__ void fold4(float& m, float& l, float4& o, float m2, float l2, float4 o2) {
    const Fold f = fold_scales(m, m2);
    l = l * f.keep + l2 * f.take;
    o.x = o.x * f.keep + o2.x * f.take;
    o.y = o.y * f.keep + o2.y * f.take;
    o.z = o.z * f.keep + o2.z * f.take;
    o.w = o.w * f.keep + o2.w * f.take;
}

// The final row's four columns [c, c+4) of O and, once per row (`first`), the
// LSE.  O is rounded once, to nearest even.
__device__ __forceinline__ void write_row4(const Args& a, int token, int head, int c, float m, float l, float4 o,
                                           bool first) {
    const float inv = 1.0f / l;
    const uint2 y = make_uint2(pack_bf16_rne(o.x * inv, o.y * inv), pack_bf16_rne(o.z * inv, o.w * inv));
    *reinterpret_cast<uint2*>(o_row(a, token, head) + c) = l == 0.0f ? make_uint2(0, 0) : y;
    if (first && a.lse != nullptr) *lse_at(a, token, head) = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// The same after folding in the part_n partial results of other launches.
__device__ __forceinline__ void finish_row4(const Args& a, int token, int head, int c, float m, float l, float4 o,
                                            bool first) {
    const long long row = flat_row(a, token, head);
    const long long rows = (long long)a.tokens * a.nhead_q;
    constexpr int kBatch = 4;  // partial results in flight
    for (int s0 = 0; s0 < a.part_n; s0 += kBatch) {
        float m2[kBatch];
        float4 x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            m2[u] = -INFINITY;
            x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (s0 + u < a.part_n) {
                m2[u] = a.part_lse[(s0 + u) * rows + row];
                x[u] = *reinterpret_cast<const float4*>(a.part_o + ((s0 + u) * rows + row) * kHeadDim + c);
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (m2[u] != -INFINITY) fold4(m, l, o, m2[u], 1.0f, x[u]);  // else O was not written
    }
    write_row4(a, token, head, c, m, l, o, first);
}

// Bounded wait on an mbarrier phase; false once the block's abort flag is up
// or the time limit ran out (which raises the flag and the error word).
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                           const Args& a) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 0) {
            if (*abort_flag) return false;
            if (globaltimer_ns() - t0 > a.wait_limit_ns) {
                *abort_flag = 1;
                atomicCAS(a.err_word, 0, fmha_host::kErrTimeoutPaged);
                return false;
            }
        }
    }
}
// While tearing down: lets copies in flight land, silently, within the limit.
__device__ __forceinline__ void drain_phase(uint32_t bar, uint32_t parity, const Args& a) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity))
        if (globaltimer_ns() - t0 > a.wait_limit_ns) return;
}

// The tensor maps read zeros for a page id outside the cache.  But they have one
// page at least, also where the cache has none: then every head is outside.
__device__ __forceinline__ int no_page_head(const Args& a) { return a.num_pages == 0 ? a.nhead_k : 0; }

// Values that are not finite.  A matrix product hands 0 * inf = NaN to rows that
// give a key no weight because they do not see it, so where rows differ in what
// they see, such values are taken out of shared memory and added by themselves,
// a weight above 0 times an infinity being the infinity.
// probe: stays 0 while the bf16 pairs are finite (x * 0 + 0), NaN from then on.
__device__ __forceinline__ uint32_t probe_bf16(uint32_t pair, uint32_t probe) {
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(probe) : "r"(pair), "r"(0u));
    return probe;
}
__device__ __forceinline__ uint32_t probe_bf16(uint4 x, uint32_t probe) {
    return probe_bf16(x.w, probe_bf16(x.z, probe_bf16(x.y, probe_bf16(x.x, probe))));
}
__device__ __forceinline__ bool is_finite_bf16(uint32_t bits) { return (bits & 0x7f80u) != 0x7f80u; }
// The pair with 0 for what is not finite.
__device__ __forceinline__ uint32_t finite_bf16(uint32_t pair) {
    return (is_finite_bf16(pair) ? pair & 0xffffu : 0u) | (is_finite_bf16(pair >> 16) ? pair & 0xffff0000u : 0u);
}
__device__ __forceinline__ uint4 finite_bf16(uint4 x) {
    return make_uint4(finite_bf16(x.x), finite_bf16(x.y), finite_bf16(x.z), finite_bf16(x.w));
}

// One box of a page: 64 values x box rows, tensor coordinates (0, token in
// page, head, page).
__device__ __forceinline__ void load_page_box(uint32_t dst, const CUtensorMap* tm, uint32_t bar,
                                              int token, int head, int page, uint64_t policy) {
    tma_load_4d(dst, tm, bar, 0, token, head, page, policy);
}

}  // namespace fmha_paged
