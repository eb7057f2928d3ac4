// fmha_rope.cu -- rotary positions with up to four axes, and appending K/V to
// a paged cache with the rotation on the way (include/fmha_paged.h).
//
// A head's 64 values hold n pairs (a, b); pair j turns by the angle whose
// cosine and sine stand in row positions[axis_of[j]] of the table:
//   a' = a cos - b sin,  b' = a sin + b cos
// and the inverse (the gradient of the rotation, which is orthogonal) negates
// the sine.  Values are rotated in fp32 and rounded once to bf16.
//
// Both entries only move bytes: each row of 128 bytes is read and written
// once.  Four threads share a row; each owns 8 pairs, that is two 16-byte
// vectors, and the 8 cosines and sines that go with them.  A thread takes
// kHeads rows of one token, so that one reading of the angles serves them all
// and their loads are in flight together; its heads lie `groups` apart, so that
// the rows of neighbouring threads lie side by side in memory.
//
// What bounds them is memory; the step to a copy's rate is the angles, gathered
// per token, and for the append the scattered pages.  Measured (in a graph):
// 30011 tokens of 16 + 16 heads with three axes, there and back, 95 us for 497 MB
// (5.2 TB/s, 81 % of a copy's rate); 32k prompt tokens of 16 + 4 + 4 heads into
// pages of 64, 45 us for 199 MB (4.4 TB/s); 16 tokens of 8 + 2 heads 2.5 us,
// which is a launch.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "../../include/fmha_paged.h"
#include "host_context.h"
#include "sm100_ptx.cuh"

namespace {

using namespace fmha_sm100;

constexpr int kThreads = 128;
constexpr int kRowThreads = 4;  // threads per 64-value row

struct RopeArgs {
    FmhaRopeParams p;
    unsigned tokens;
    unsigned groups; // threads' shares of a token's heads
    uint8_t axes4[8];  // axes of pairs 4i .. 4i+3, two bits each
    int page_shift;
    int* err_word;
};

__device__ __forceinline__ void flag_index_error(int* err_word) {
    atomicCAS(err_word, 0, fmha_host::kErrIndex);
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// Sequence of packed token t: the last b with seqstart[b] <= t.
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ seqstart, int batch, int t) {
    int lo = 0, hi = batch;  // seqstart[lo] <= t < seqstart[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (seqstart[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Heads of a token in order: nhead_q of Q, nhead_k of K, and (append) nhead_k
// of V.
template <bool kAppend, int kHeads>
__global__ void __launch_bounds__(kThreads)
fmha_rope_d64_kernel(const __grid_constant__ RopeArgs a) {
    const FmhaRopeParams& p = a.p;
    const unsigned slot = (blockIdx.x * (unsigned)kThreads + threadIdx.x) / kRowThreads;
    const int part = threadIdx.x & (kRowThreads - 1);
    const unsigned tok_u = slot / a.groups;
    if (tok_u >= a.tokens) return;
    const int tok = (int)tok_u;
    const int head0 = (int)(slot - tok_u * a.groups);
    const int heads_q = p.q != nullptr ? p.nhead_q : 0;
    const int heads_k = p.k != nullptr ? p.nhead_k : 0;
    const int heads = heads_q + heads_k * (kAppend ? 2 : 1);

    // Token -> (batch, index); dense tokens are batch-major.
    int b, i;
    const bool packed = p.seqstart_q != nullptr;
    if (packed) {
        b = 0;
        i = tok;
    } else {
        b = tok / p.seqlen_q;
        i = tok - b * p.seqlen_q;
    }

    // Vectors of this thread: pairs 8*part .. 8*part+7, or two vectors past
    // the rotated part.
    const int n = p.n_pairs;
    const bool turns = part * 8 < n;
    int va, vb;
    if (p.interleaved || !turns) {
        va = 2 * part;
        vb = va + 1;
    } else {
        va = part;
        vb = part + n / 8;
    }

    const uint16_t* src[kHeads];
    uint4 xa[kHeads], xb[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
        const int h = head0 + u * (int)a.groups;
        if (h >= heads) break;
        if (h < heads_q)
            src[u] = p.q + b * p.batch_stride_q + i * p.stride_q + h * p.nhead_stride_q;
        else if (h < heads_q + heads_k)
            src[u] = p.k + b * p.batch_stride_k + i * p.stride_k + (h - heads_q) * p.nhead_stride_k;
        else
            src[u] = p.v + b * p.batch_stride_v + i * p.stride_v +
                     (h - heads_q - heads_k) * p.nhead_stride_v;
        xa[u] = __ldcs(reinterpret_cast<const uint4*>(src[u]) + va);
        xb[u] = __ldcs(reinterpret_cast<const uint4*>(src[u]) + vb);
    }

    // Where the token goes (append): place = length - new tokens + index.
    int place = 0;
    bool stored = true, in_cache = true;
    int page = 0;
    if constexpr (kAppend) {
        int seq = b, idx = i, count = p.seqlen_q;
        if (packed) {
            seq = find_sequence(p.seqstart_q, p.batch, tok);
            const int s0 = p.seqstart_q[seq];
            count = p.seqstart_q[seq + 1] - s0;
            idx = tok - s0;
        }
        place = p.seqlens_k[seq] - count + idx;
        const bool inside = idx >= 0 && idx < count;  // else the prefix sums miss the token
        stored = place >= 0 && inside;
        in_cache = stored && (place >> a.page_shift) < p.max_pages;
        if (in_cache) {
            page = p.page_table[seq * p.table_stride + (place >> a.page_shift)];
            in_cache = page >= 0 && page < p.num_pages;
        }
        if (!inside || (stored && !in_cache)) flag_index_error(a.err_word);
        stored = stored && in_cache;
    }

    float cs[8], sn[8];
    bool angle = true;
    if (turns && p.cos_sin != nullptr) {
        const float sign = p.inverse ? -1.0f : 1.0f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int j0 = part * 8 + half * 4;
            const unsigned axes = a.axes4[part * 2 + half];
            const bool given = !kAppend || p.positions != nullptr;
            // At most two axes turn the four pairs, unless axes alternate pair by
            // pair: those of the first and of the last.
            const unsigned ax0 = axes & 3, ax3 = axes >> 6, ax1 = (axes >> 2) & 3, ax2 = (axes >> 4) & 3;
            const bool two = (ax1 == ax0 || ax1 == ax3) && (ax2 == ax0 || ax2 == ax3);
            const int pos0 = given ? p.positions[ax0 * p.axis_stride + tok] : place;
            int pos3 = pos0;
            if (given && ax3 != ax0) pos3 = p.positions[ax3 * p.axis_stride + tok];
            angle = angle && (unsigned)pos0 < (unsigned)p.max_pos && (unsigned)pos3 < (unsigned)p.max_pos;
            float4 c, s;
            if (angle) {
                const float* row = p.cos_sin + (long long)pos0 * (2 * n) + j0;
                c = *reinterpret_cast<const float4*>(row);
                s = *reinterpret_cast<const float4*>(row + n);
            }
            if (given && axes != ax0 * 0x55u) {
                if (angle) {
                    const float* row = p.cos_sin + (long long)pos3 * (2 * n) + j0;
                    const float4 c3 = *reinterpret_cast<const float4*>(row);
                    const float4 s3 = *reinterpret_cast<const float4*>(row + n);
                    if (ax1 != ax0) c.y = c3.y, s.y = s3.y;
                    if (ax2 != ax0) c.z = c3.z, s.z = s3.z;
                    c.w = ax3 != ax0 ? c3.w : c.w, s.w = ax3 != ax0 ? s3.w : s.w;
                }
                if (!two) {  // a third axis in the middle
                    const int pos1 = p.positions[ax1 * p.axis_stride + tok], pos2 = p.positions[ax2 * p.axis_stride + tok];
                    angle = angle && (unsigned)pos1 < (unsigned)p.max_pos && (unsigned)pos2 < (unsigned)p.max_pos;
                    if (angle) {
                        const float* row1 = p.cos_sin + (long long)pos1 * (2 * n) + j0 + 1;
                        const float* row2 = p.cos_sin + (long long)pos2 * (2 * n) + j0 + 2;
                        c.y = row1[0], s.y = row1[n];
                        c.z = row2[0], s.z = row2[n];
                    }
                }
            }
            cs[half * 4 + 0] = c.x, cs[half * 4 + 1] = c.y, cs[half * 4 + 2] = c.z, cs[half * 4 + 3] = c.w;
            sn[half * 4 + 0] = s.x * sign, sn[half * 4 + 1] = s.y * sign;
            sn[half * 4 + 2] = s.z * sign, sn[half * 4 + 3] = s.w * sign;
        }
    }
    // A row whose four threads do not all have their angles is not written in
    // part: the quad agrees.
    const unsigned quad = 0xfu << (threadIdx.x & 28);
    angle = __all_sync(quad, angle);
    // An empty slot of a batch has no position either: only a token that is
    // stored (or rotated without a cache) can miss the table.
    if (!angle && stored) flag_index_error(a.err_word);
    const bool zero_q = !angle || !stored;

#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
        const int h = head0 + u * (int)a.groups;
        if (h >= heads) break;
        const bool is_q = h < heads_q;
        const bool is_v = h >= heads_q + heads_k;
        uint4 ya = xa[u], yb = xb[u];
        if (turns && p.cos_sin != nullptr && !is_v && angle) {
            uint32_t* wa = reinterpret_cast<uint32_t*>(&ya);
            uint32_t* wb = reinterpret_cast<uint32_t*>(&yb);
            if (p.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = unpack_bf16(wa[e]);
                    const float2 g = unpack_bf16(wb[e]);
                    wa[e] = pack_bf16_rne(f.x * cs[e] - f.y * sn[e], f.x * sn[e] + f.y * cs[e]);
                    wb[e] = pack_bf16_rne(g.x * cs[e + 4] - g.y * sn[e + 4],
                                          g.x * sn[e + 4] + g.y * cs[e + 4]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = unpack_bf16(wa[e]);
                    const float2 g = unpack_bf16(wb[e]);
                    const float c0 = cs[2 * e], c1 = cs[2 * e + 1], s0 = sn[2 * e], s1 = sn[2 * e + 1];
                    wa[e] = pack_bf16_rne(f.x * c0 - g.x * s0, f.y * c1 - g.y * s1);
                    wb[e] = pack_bf16_rne(f.x * s0 + g.x * c0, f.y * s1 + g.y * c1);
                }
            }
        }
        uint16_t* dst;
        if (is_q) {
            dst = p.q_out + b * p.batch_stride_qo + i * p.stride_qo + h * p.nhead_stride_qo;
            if (zero_q) ya = yb = make_uint4(0, 0, 0, 0);
        } else if constexpr (kAppend) {
            if (!stored || !angle) continue;
            const int in_page = place & ((1 << a.page_shift) - 1);
            dst = is_v ? p.v_out + page * p.batch_stride_vo + in_page * p.stride_vo +
                             (h - heads_q - heads_k) * p.nhead_stride_vo
                       : p.k_out + page * p.batch_stride_ko + in_page * p.stride_ko +
                             (h - heads_q) * p.nhead_stride_ko;
        } else {
            dst = p.k_out + b * p.batch_stride_ko + i * p.stride_ko + (h - heads_q) * p.nhead_stride_ko;
            if (zero_q) ya = yb = make_uint4(0, 0, 0, 0);
        }
        if (kHeads == 1) {
            reinterpret_cast<uint4*>(dst)[va] = ya;
            reinterpret_cast<uint4*>(dst)[vb] = yb;
        } else {  // more than the caches hold on to (append of 32k tokens: 48 us with plain stores, 44 with these)
            __stcs(reinterpret_cast<uint4*>(dst) + va, ya);
            __stcs(reinterpret_cast<uint4*>(dst) + vb, yb);
        }
    }
}

// ====================================================================== host

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A stride of a dimension of one element is never used.
bool stride_ok(long long s, long long extent, bool out) {
    if (extent <= 1) return true;
    return (out ? s > 0 : s >= 0) && s % 8 == 0 && s < (1ll << 39);
}

int log2_exact(int v) {
    for (int s = 0; s < 31; ++s)
        if ((1 << s) == v) return s;
    return -1;
}

int check(const FmhaRopeParams* p, bool append, RopeArgs& a) {
    if (p == nullptr) return FMHA_ERR_ARG;
    const bool packed = p->seqstart_q != nullptr;
    if (p->batch < 0 || p->seqlen_q < 0 || p->total_q < 0 || p->nhead_q < 0 || p->nhead_k < 0)
        return FMHA_ERR_ARG;
    const long long rows = packed ? p->total_q : p->seqlen_q;
    const long long batch = packed ? 1 : p->batch;
    const long long tokens = rows * batch;
    if (tokens > 0x7fffffffll) return FMHA_ERR_ARG;
    for (const void* i : {(const void*)p->positions, (const void*)p->seqstart_q, (const void*)p->page_table,
                          (const void*)p->seqlens_k})
        if ((reinterpret_cast<uintptr_t>(i) & 3u) != 0) return FMHA_ERR_ARG;
    if (p->q != nullptr) {
        if (p->nhead_q <= 0 || p->q_out == nullptr || !aligned16(p->q) || !aligned16(p->q_out) ||
            !stride_ok(p->stride_q, rows, false) || !stride_ok(p->nhead_stride_q, p->nhead_q, false) ||
            !stride_ok(p->batch_stride_q, batch, false) || !stride_ok(p->stride_qo, rows, true) ||
            !stride_ok(p->nhead_stride_qo, p->nhead_q, true) ||
            !stride_ok(p->batch_stride_qo, batch, true))
            return FMHA_ERR_ARG;
    }
    if (p->k != nullptr) {
        if (p->nhead_k <= 0 || p->k_out == nullptr || !aligned16(p->k) || !aligned16(p->k_out) ||
            !stride_ok(p->stride_k, rows, false) || !stride_ok(p->nhead_stride_k, p->nhead_k, false) ||
            !stride_ok(p->batch_stride_k, batch, false))
            return FMHA_ERR_ARG;
    }
    if (p->cos_sin != nullptr) {
        if (!aligned16(p->cos_sin) || p->max_pos <= 0) return FMHA_ERR_ARG;
        if (p->n_pairs != 8 && p->n_pairs != 16 && p->n_pairs != 24 && p->n_pairs != 32)
            return FMHA_ERR_ARG;
        for (int j = 0; j < p->n_pairs; ++j)
            if (p->axis_of[j] > 3) return FMHA_ERR_ARG;
        if (p->positions != nullptr && p->axis_stride < 0) return FMHA_ERR_ARG;
    }
    if (append) {
        if (p->k == nullptr || p->v == nullptr || p->v_out == nullptr || p->page_table == nullptr ||
            p->seqlens_k == nullptr || p->batch <= 0 || p->inverse != 0)
            return FMHA_ERR_ARG;
        if (!aligned16(p->v) || !aligned16(p->v_out) || !stride_ok(p->stride_v, rows, false) ||
            !stride_ok(p->nhead_stride_v, p->nhead_k, false) ||
            !stride_ok(p->batch_stride_v, batch, false))
            return FMHA_ERR_ARG;
        const int shift = log2_exact(p->page_size);
        if (shift < 3 || shift > 12 || p->num_pages < 0 || p->max_pages < 0 || p->table_stride < 0)
            return FMHA_ERR_ARG;
        a.page_shift = shift;
        if (!stride_ok(p->stride_ko, p->page_size, true) || !stride_ok(p->stride_vo, p->page_size, true) ||
            !stride_ok(p->nhead_stride_ko, p->nhead_k, true) ||
            !stride_ok(p->nhead_stride_vo, p->nhead_k, true) ||
            !stride_ok(p->batch_stride_ko, p->num_pages, true) ||
            !stride_ok(p->batch_stride_vo, p->num_pages, true))
            return FMHA_ERR_ARG;
    } else {
        if ((p->q == nullptr && p->k == nullptr) || p->v != nullptr || p->cos_sin == nullptr ||
            p->positions == nullptr)
            return FMHA_ERR_ARG;
        if (p->k != nullptr && (!stride_ok(p->stride_ko, rows, true) ||
                                !stride_ok(p->nhead_stride_ko, p->nhead_k, true) ||
                                !stride_ok(p->batch_stride_ko, batch, true)))
            return FMHA_ERR_ARG;
    }
    a.p = *p;
    if (p->cos_sin == nullptr) a.p.n_pairs = 32;  // unused, but divides the row as usual
    for (int j = 0; j < 32; ++j) a.axes4[j / 4] |= (uint8_t)((a.p.axis_of[j] & 3) << (2 * (j & 3)));
    a.tokens = (unsigned)tokens;
    return FMHA_OK;
}

template <bool kAppend>
int launch(const FmhaRopeParams* p, cudaStream_t stream) {
    RopeArgs a;
    memset(&a, 0, sizeof(a));
    int st = check(p, kAppend, a);
    if (st != FMHA_OK) return st;
    fmha_host::Context ctx;
    if ((st = fmha_host::acquire(&ctx)) != FMHA_OK) return st;
    if (a.tokens == 0) return FMHA_OK;
    a.err_word = ctx.err_word;
    const int heads = (p->q ? p->nhead_q : 0) + (p->k ? p->nhead_k : 0) * (kAppend ? 2 : 1);
    // One row per thread while all rows fit the device at once, so that nothing
    // waits for another row; four beyond (16 tokens x 10 heads: 2.5 against
    // 3.1 us; 30011 x 32: 142 against 97 us).
    const bool few = (long long)a.tokens * heads * kRowThreads <= 148ll * 1024;
    const int per = few ? 1 : 4;
    a.groups = (unsigned)((heads + per - 1) / per);
    const long long slots = (long long)a.tokens * a.groups;
    // (More rows than that would not fit any memory.)
    if (slots * kRowThreads > 0xffffffffll - kThreads) return FMHA_ERR_ARG;
    const unsigned blocks = (unsigned)((slots * kRowThreads + kThreads - 1) / kThreads);
    if (few) fmha_rope_d64_kernel<kAppend, 1><<<blocks, kThreads, 0, stream>>>(a);
    else fmha_rope_d64_kernel<kAppend, 4><<<blocks, kThreads, 0, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int fmha_rope_d64_bf16(const FmhaRopeParams* params, CUstream_st* stream) try {
    return launch<false>(params, stream);
} catch (...) {
    return FMHA_ERR_LAUNCH;
}

int fmha_paged_append_d64_bf16(const FmhaRopeParams* params, CUstream_st* stream) try {
    return launch<true>(params, stream);
} catch (...) {
    return FMHA_ERR_LAUNCH;
}

}  // extern "C"
