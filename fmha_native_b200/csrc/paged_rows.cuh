// paged_rows.cuh -- attention of few query rows per K/V head over the paged
// cache: single tokens, a few drafted tokens, grouped query heads.
//
// What it computes per (sequence, K/V head): O = softmax(scale Q K^T) V for up
// to kMostRows rows that share the keys, as one pass over the keys with a running
// maximum m, weight sum l and un-normalised O per row (fp32).
//
// What bounds it: the cache is read once (256 bytes per key and K/V head) and
// the arithmetic per byte is small, so it should run at memory speed.  Hence:
//
//   work split   The keys of all sequences are laid end to end in units of 32,
//                and the blocks take equal contiguous ranges of that line, with
//                several K/V heads (group_heads): heads lie side by side in a
//                token, so a block's warps read neighbouring lines of memory at
//                the same time.
//                Inside a block the line (sequence, head, unit) of its range is
//                cut into equal shares for the 8 warps.  Lengths may differ as
//                they like: every warp streams the same number of bytes.
//                Pieces (m, l, O) of a head whose units went to several warps
//                are folded through shared memory, those of a sequence that
//                crosses blocks by fmha_paged_end.  The shares follow
//                from the lengths alone, so results do not depend on timing.
//   streaming    Each warp has its own ring of kRowStages units in shared memory,
//                filled by TMA (one box per page) several units ahead, across
//                heads and sequences; no block-wide step until the share ends.
//   arithmetic   mma.sync m16n8k16 with the rows as M: the tile of a decode
//                step is far too thin for a 128-row tensor-memory tile, and
//                the reads leave the tensor pipe idle anyway.  P enters the
//                second product as a sum of two bf16 (value and remainder, to
//                2^-16 of it), so O is rounded once, at its end.  Both are above
//                0 where P is, so that an infinite V gives an infinite O.
//
// Measured (in a graph): 4 sequences of 60 000 to 130 000 keys, 16 K/V heads,
// 250 us for 1.62 GB (6.5 TB/s, a copy's rate; 254 in a long loop, under the power
// limit); 64 sequences of 100 to 4095 keys, 32 heads over 8, 41 us for 172 MB (4.2
// TB/s: start, first loads and fold are about 12 us of it); one sequence of 776
// keys 9.1 us, which is two launches in line.  The tile kernel, which could take
// these rows too, took 12, 44 and 24 % longer.  (A tensor map that promotes its
// reads to 256 bytes in L2 made it fetch twice what it used.)
//
// Below, where a choice was measured, each pair of figures is of one state of the
// code: what counts is their ratio.
//
// Keys past a row's limit get weight 0 by selection, and value rows past the
// tile's last visible key are zeroed in shared memory before use, so whatever
// the page holds there (NaN included) stays out of O.  In units that some rows
// see in part, values that are not finite are taken out of the product and added
// to the rows that see them.
#pragma once
#include <algorithm>

#include "paged_common.cuh"

namespace fmha_paged {

constexpr int kUnit = 32;             // keys per unit
constexpr int kRowWarps = 8;
constexpr int kRowThreadsTotal = 32 * kRowWarps;
constexpr int kUnitBytes = kUnit * kHeadDim * 2;  // 4 KB of K, as much of V
constexpr int kMaxRowBlocks = 148;    // one block per SM

// Rows of a K/V head that a warp holds: two halves of the matrix instruction's M.
// With 9 to 16 rows this kernel is still ahead of the tile kernel where the keys
// are many (64 sequences of 1365 to 4096 keys, 8 heads of 16 rows: 83 against 95
// us, 32 heads of one with 16384: 32 against 37), and even where they are few (64
// of 100 to 300 keys, 8 heads: 23 and 23).
constexpr int kMostRows = 16;
constexpr int kRowStages = 3;
// A sequence's start and end in a block cost about as much time as this many
// units (its first loads, Q, the results), and the shares count them: 64 sequences
// of 100 to 4095 keys take 5 % longer without, 111 of none or one under a prefix of
// 335 a third longer.
constexpr int kSeqCost = 5;

// Groups of blocks that share out the K/V heads: each group works on all keys.
// More heads a block keep more neighbouring memory together, more groups make
// longer ranges, and so fewer pieces to fold; what the pieces weigh depends on
// the rows.  Per group about 8 heads for 1 or 2 rows (4 sequences of 60 000 to
// 130 000 keys, 16 heads: 7 % longer with one group, 5 % with 4 heads), 4 for up
// to 8 (64 sequences of 100 to 4095 keys, 8 heads of 4 rows: 3 % longer with one
// group), 2 beyond (one sequence of 16384 keys, 32 heads of 16 rows: 32 us, 87 with
// one group, 36 with 8 heads).
constexpr int kMostGroups = 16;
inline int head_groups(int nhead_k, int rows) {
    const int least = rows <= 2 ? 8 : rows <= 8 ? 4 : 2;
    int g = std::min(kMostGroups, (nhead_k + least - 1) / least);
    while (nhead_k % g != 0) --g;
    return g;
}

// A sequence as this kernel takes it.
struct RowSeq {
    int first, count, keys;
    int kv_end;      // keys that any of its rows sees
    int units;       // 0: not ours; a sequence that sees no key counts one (empty) unit
};
// A (sequence, head) result of a block: where it goes.
struct Target {
    int first, rows;  // the sequence's first token; its rows per K/V head
    int h;            // K/V head
    int slot;         // piece slot of the block's scratch, or -1: the final rows
};

struct alignas(1024) RowsShared {
    uint8_t ring[kRowWarps][kRowStages][2][kUnitBytes];
    // A warp's piece of a head that an earlier warp began.  A piece that a later
    // warp goes on with comes last and takes the warp's (then idle) ring.
    float first_o[kRowWarps][kMostRows * kHeadDim];
    float first_ml[kRowWarps][kMostRows * 2];
    uint64_t bar[kRowWarps][kRowStages];
    Target piece_to[kRowWarps][2];
    int piece_job[kRowWarps][2];      // segment of the block * heads + head, -1: none
    int2 scan[kRowWarps];
    unsigned present[kRowWarps];      // bit per thread: its sequences have units
    int run[2 * kRowWarps + 1];
    RowSeq start_seq;                 // of the block's first segment
    int start_b, start_x;
    int abort_flag;
};

// Scratch between blocks: per block two slots (0: a sequence that an earlier
// block began, 1: one that a later block goes on with) of nhead_k x row_cap
// rows of O, then as many (m, l), then a header per block.
struct RowsHeader {
    int first, rows;  // a sequence that begins in this block and goes on: its first token, rows
    int parts;        // blocks that share it; 0: none
    int h0, heads;    // the block's K/V heads
    int pad[3];
};
__host__ __device__ constexpr size_t rows_scratch_bytes(long long rows) {
    return kMaxRowBlocks * (2 * (size_t)rows * (kHeadDim + 2) * sizeof(float) + sizeof(RowsHeader));
}
__device__ __forceinline__ long long piece_row(const Args& a, int slot, int h, int r) {
    return ((long long)slot * a.nhead_k + h) * a.row_cap + r;
}
__device__ __forceinline__ float* piece_o(const Args& a, long long row) { return a.pieces + row * kHeadDim; }
__device__ __forceinline__ float* piece_ml(const Args& a, long long row) {
    return a.pieces + 2ll * kMaxRowBlocks * a.nhead_k * a.row_cap * kHeadDim + row * 2;
}
__device__ __forceinline__ RowsHeader* piece_headers(const Args& a) {
    return reinterpret_cast<RowsHeader*>(a.pieces + 2ll * kMaxRowBlocks * a.nhead_k * a.row_cap * (kHeadDim + 2));
}

__device__ __forceinline__ RowSeq load_row_seq(const Args& a, int b) {
    const Sequence s = load_sequence(a, b);
    RowSeq x{s.first, s.count, s.keys, 0, 0};
    const int rows = s.count * a.group;  // at most row_cap from here on
    if (rows < a.min_rows || rows > a.max_rows) return x;
    x.kv_end = max(0, key_limit(a, Sequence{x.first, x.count, x.keys}, x.count - 1));
    x.units = max(1, (x.kv_end + kUnit - 1) / kUnit);
    return x;
}

__device__ __forceinline__ void prefetch_l1(const void* p) {
    asm volatile("prefetch.global.L1 [%0];" ::"l"(p));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The largest bf16 below x, for x > 0; 0 for 0 (and NaN for NaN).
__device__ __forceinline__ float below_bf16(float x) {
    return __uint_as_float((uint32_t)max((int)__float_as_uint(x) - 1, 0) & 0xffff0000u);
}
__device__ __forceinline__ void fence_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Takes the values that are not finite out of the V of a unit of `keys` keys, and
// notes them in the bits of the o[n][q] (m16n8 fragments of the lane's rows, which
// see seen0 and seen1 of the keys) that they belong to.  One warp, which fences.
__device__ __forceinline__ void note_odd_values(uint4* v, int keys, int seen0, int seen1, uint32_t (&odd)[3]) {
    const int lane = threadIdx.x & 31;
    uint32_t probe = 0;
#pragma unroll 1
    for (int i = lane; i < keys * 8; i += 32) probe = probe_bf16(v[i], probe);
    if (!__any_sync(0xffffffffu, probe != 0)) return;
#pragma unroll 1
    for (int x = 0; x < keys * 8; ++x) {
        const int key = x >> 3, n = x & 7;
        const uint32_t pair = reinterpret_cast<const uint32_t*>(v + key * 8 + (n ^ (key & 7)))[lane & 3];
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
            const uint32_t bits = q & 1 ? pair >> 16 : pair & 0xffffu;
            if (is_finite_bf16(bits) || key >= (q < 2 ? seen0 : seen1)) continue;
            const uint32_t bit = 1u << (4 * n + q);
            if ((bits & 0x7fu) != 0) odd[0] |= bit;
            else if ((bits & 0x8000u) == 0) odd[1] |= bit;
            else odd[2] |= bit;
        }
    }
    __syncwarp();
#pragma unroll 1
    for (int i = lane; i < keys * 8; i += 32) v[i] = finite_bf16(v[i]);
}

// Row rt of a result, columns [4 c4, 4 c4 + 4): into the final rows or the
// block's scratch.
__device__ __forceinline__ void emit_row4(const Args& a, const Target& to, int rt, int c4, float m, float l,
                                          float4 o) {
    const int t = rt / a.group, token = to.first + t, head = to.h * a.group + rt - t * a.group;
    if (to.slot < 0 && a.out_o == nullptr) {
        write_row4(a, token, head, c4 * 4, m, l, o, c4 == 0);
    } else if (to.slot < 0) {
        // Under a prefix: one more partial result of the row.
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const long long row = flat_row(a, token, head);
        *reinterpret_cast<float4*>(a.out_o + row * kHeadDim + c4 * 4) =
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        if (c4 == 0) a.out_lse[row] = l == 0.0f ? -INFINITY : m + __log2f(l);
    } else {
        const long long row = piece_row(a, to.slot, to.h, rt);
        *reinterpret_cast<float4*>(piece_o(a, row) + c4 * 4) = o;
        if (c4 == 0) *reinterpret_cast<float2*>(piece_ml(a, row)) = make_float2(m, l);
    }
}

// Equal contiguous ranges of `total` units: range c of n begins at
// c * base + min(c, rem).
struct Ranges {
    unsigned base, rem;
    __device__ Ranges(unsigned total, unsigned n) : base(total / n), rem(total % n) {}
    __device__ unsigned begin(unsigned c) const { return c * base + min(c, rem); }
    __device__ unsigned owner(unsigned x) const {
        const unsigned wide = rem * (base + 1);
        return x < wide ? x / (base + 1) : rem + (x - wide) / base;
    }
};

__global__ void __launch_bounds__(kRowThreadsTotal, 1)
fmha_paged_rows_kernel(const __grid_constant__ Args a) {
    extern __shared__ uint8_t smem_raw[];
    RowsShared& sm = *reinterpret_cast<RowsShared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                            ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    volatile int* abort_flag = &sm.abort_flag;

    griddep_launch_dependents();
    if (lane == 0) {
        tma_prefetch_desc(&a.tm_k);
        tma_prefetch_desc(&a.tm_v);
        for (int s = 0; s < kRowStages; ++s) mbar_init(smem_u32(&sm.bar[warp][s]), 1);
        sm.piece_job[warp][0] = sm.piece_job[warp][1] = -1;
        if (warp == 0) sm.abort_flag = 0;
        fence_barrier_init();
    }

    // ------------------------------------------------- the block's range
    const int per = (a.batch + kRowThreadsTotal - 1) / kRowThreadsTotal;
    const int b0 = min(a.batch, (int)threadIdx.x * per), b1 = min(a.batch, b0 + per);
    int mine = 0, mine_n = 0;  // units; sequences
    for (int b = b0; b < b1; ++b) {
        const int n = load_row_seq(a, b).units;
        mine += n;
        mine_n += n > 0;
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
    }
    const unsigned present = __ballot_sync(0xffffffffu, mine_n > 0);
    int incl_n;
    if (per == 1) {
        incl_n = __popc(present & (0xffffffffu >> (31 - lane)));
    } else {
        incl_n = mine_n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl_n, d);
            if (lane >= d) incl_n += v;
        }
    }
    if (lane == 31) sm.scan[warp] = make_int2(incl, incl_n), sm.present[warp] = present;
    __syncthreads();
    unsigned before = incl - mine, before_n = incl_n - mine_n, total = 0, total_n = 0;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
        const int2 v = sm.scan[w];
        if (w < warp) before += v.x, before_n += v.y;
        total += v.x;
        total_n += v.y;
    }
    const bool some_absent = total_n < a.batch;
    auto cost_of = [&](int n) { return n > 0 ? n + kSeqCost : 0; };
    // Groups of blocks share out the heads.
    const int group_blocks = a.group_blocks, heads = a.group_heads;
    const int group = (int)blockIdx.x / group_blocks, index = (int)blockIdx.x - group * group_blocks;
    const int head0 = group * heads;
    const int map_head0 = head0 + no_page_head(a);
    const unsigned cost_mine = mine + mine_n * kSeqCost;
    before += before_n * kSeqCost;
    total += total_n * kSeqCost;
    // As many blocks as give every warp a unit of some head.
    const unsigned want = (unsigned)min(((unsigned long long)total * heads + kRowWarps - 1) / kRowWarps,
                                        (unsigned long long)total);
    const unsigned blocks = min((unsigned)group_blocks, want);
    if (head0 >= a.nhead_k || index >= blocks) {
        griddep_wait();  // the grid ends after the launch before it
        if (threadIdx.x == 0) piece_headers(a)[blockIdx.x].parts = 0;
        return;
    }
    const Ranges ranges(total, blocks);
    const unsigned beg = ranges.begin(index), end = ranges.begin(index + 1);
    if (beg >= before && beg < before + cost_mine) {
        unsigned p = before;
        for (int b = b0; b < b1; ++b) {
            const RowSeq x = load_row_seq(a, b);
            const unsigned n = cost_of(x.units);
            if (beg < p + n) {
                sm.start_b = b;
                sm.start_x = (int)(beg - p);
                sm.start_seq = x;
                // The first page ids that the block will want.
                const int page0 = (max(0, (int)(beg - p) - kSeqCost) * kUnit) >> a.page_shift;
                const int32_t* ids = a.page_table + b * a.table_stride + page0;
                if (page0 < a.max_pages) prefetch_l1(ids);
                if (page0 + 32 < a.max_pages) prefetch_l1(ids + 32);
                break;
            }
            p += n;
        }
    }
    __syncthreads();

    // ------------------------------------------------------- the share
    // A place on the block's line: segment (a sequence's units [unit0, unit0 +
    // n) in this block), head (of the block's), unit.  Two cursors: `p` issues loads, `c` computes.
    struct Cursor {
        RowSeq x;
        int b, seg;
        int left, cost;  // cost of the block from this segment on, and of the segment
        int unit0, n, h, u;
    };
    // Sets the segment of sequence k.b that starts `off` into the sequence's cost.
    auto set_segment = [&](Cursor& k, int off) {
        k.cost = min(cost_of(k.x.units) - off, k.left);
        k.unit0 = max(0, off - kSeqCost);
        k.n = max(0, off + k.cost - kSeqCost) - k.unit0;
    };
    // The first sequence from b on that may have units: those of the tile kernel are
    // passed over (53 sequences, 44 of them such: 68 us with a look at each one, 60
    // without).  Where none is absent the search itself would cost up to a fifth.
    auto next_present = [&](int b) {
        if (b % per != 0 || b >= a.batch) return b;
        int t = b / per;
        unsigned bits = sm.present[t >> 5] >> (t & 31);
        while (bits == 0) {
            t = (t | 31) + 1;
            if (t >= kRowThreadsTotal) return a.batch;
            bits = sm.present[t >> 5];
        }
        return (t + __ffs(bits) - 1) * per;
    };
    auto next_segment = [&](Cursor& k) {
        do {
            k.left -= k.cost;
            k.cost = k.n = 0;
            if (k.left <= 0) return false;
            do {
                ++k.b;
                if (some_absent) k.b = next_present(k.b);
                if (k.b >= a.batch) return false;
                k.x = load_row_seq(a, k.b);
            } while (k.x.units == 0);
            ++k.seg;
            set_segment(k, 0);
        } while (k.n == 0);
        return true;
    };
    auto advance = [&](Cursor& k) {
        if (++k.u < k.n) return;
        k.u = 0;
        if (++k.h < heads) return;
        k.h = 0;
        next_segment(k);
    };
    Cursor c;
    c.b = sm.start_b;
    c.x = sm.start_seq;
    c.seg = 0;
    c.left = (int)(end - beg);
    c.h = c.u = 0;
    set_segment(c, sm.start_x);
    bool any = c.n > 0 || next_segment(c);
    const Cursor c0 = c;
    unsigned long long tiles = 0;  // of the block: units x heads
    {
        Cursor k = c;
        for (bool more = any; more; more = next_segment(k)) tiles += (unsigned long long)k.n * heads;
    }
    const unsigned long long from = tiles * warp / kRowWarps;
    const long long count = (long long)(tiles * (warp + 1) / kRowWarps - from);
    if (count > 0) {
        unsigned long long x = from;
        while (x >= (unsigned long long)c.n * heads) {
            x -= (unsigned long long)c.n * heads;
            if (!next_segment(c)) break;
        }
        if (c.n > 0) {
            c.h = x >> 32 ? (int)(x / (unsigned)c.n) : (int)((unsigned)x / (unsigned)c.n);
            c.u = (int)(x - (unsigned long long)c.h * c.n);
        }
        Cursor p = c;
        long long to_issue = count;
        int issued = 0, done = 0;

        // Page ids: lane i holds entry win + i of sequence win_b's table row.
        const int box_shift = min(a.page_shift, 5);  // keys of a box, at most a unit's 32
        const int page_mask = (1 << a.page_shift) - 1;
        int win_b = -1, win = 0, ids = 0, ids_next = 0;
        auto load_ids = [&](int first, int pages) {
            const int i = first + lane;
            return i < pages ? __ldg(a.page_table + win_b * a.table_stride + i) : 0;
        };
        const uint64_t policy = l2_policy_evict_first();
        const uint32_t ring0 = smem_u32(sm.ring[warp]), bar0 = smem_u32(sm.bar[warp]);
        int fill = 0;  // slot of the next load
        auto produce = [&]() {
            while (to_issue > 0 && issued - done < kRowStages) {
                if (p.x.kv_end > 0) {
                    const int key0 = (p.unit0 + p.u) * kUnit;
                    const int page0 = key0 >> a.page_shift;
                    if (win_b != p.b || (unsigned)(page0 - win) >= 32u) {
                        const int pages = (p.x.keys + page_mask) >> a.page_shift;
                        if (win_b == p.b && page0 - win >= 32 && page0 - win < 64) {
                            win += 32;
                            ids = ids_next;
                        } else {
                            win_b = p.b;
                            win = page0 & ~3;
                            ids = load_ids(win, pages);
                        }
                        ids_next = load_ids(win + 32, pages);
                    }
                    const int nbox = (min(kUnit, p.x.kv_end - key0) + (1 << box_shift) - 1) >> box_shift;
                    const uint32_t bar = bar0 + fill * 8;
                    const int id = __shfl_sync(0xffffffffu, ids, (page0 + lane - win) & 31);
                    if (lane == 0) mbar_arrive_expect_tx(bar, (2 * nbox) << (box_shift + 7));
                    __syncwarp();
                    if (lane < nbox) {
                        const uint32_t dst = ring0 + fill * (2 * kUnitBytes) + (lane << (box_shift + 7));
                        if ((unsigned)id >= (unsigned)a.num_pages) flag_index_error(a.err_word);
                        load_page_box(dst, &a.tm_k, bar, key0 & page_mask, map_head0 + p.h, id, policy);
                        load_page_box(dst + kUnitBytes, &a.tm_v, bar, key0 & page_mask, map_head0 + p.h, id, policy);
                    }
                    ++issued;
                    fill = fill == kRowStages - 1 ? 0 : fill + 1;
                }
                advance(p);
                --to_issue;
                if (p.u == 0 && to_issue > 0) {
                    // A new head: its query rows, and at a new sequence the next
                    // one's page ids, will be wanted without delay.
                    if (lane < p.x.count * a.group) {
                        const int t = lane / a.group;
                        prefetch_l1(q_row(a, p.x.first + t, (head0 + p.h) * a.group + lane - t * a.group));
                    }
                    if (p.h == 0 && lane == 31 && p.b + 1 < a.batch)
                        prefetch_l1(a.page_table + (p.b + 1) * a.table_stride);
                }
            }
        };
        produce();

        const int g = lane >> 2, t4 = lane & 3;
        uint32_t qf[4][4];
        float o[8][4], m[2], l[2];
        int lim[2];
        int u0 = 0;
        uint32_t odd[3];  // bit 4 n + q: NaN, +inf or -inf among the values that belong to o[n][q]
        bool ok = true;
        for (long long it = 0; it < count; ++it) {
            const int rows = c.x.count * a.group;
            if (it == 0 || c.u == 0) {
                u0 = c.u;
                odd[0] = odd[1] = odd[2] = 0;
#pragma unroll
                for (int hr = 0; hr < 2; ++hr) {
                    const int r = hr * 8 + g;
                    m[hr] = -INFINITY;
                    l[hr] = 0.0f;
                    lim[hr] = 0;
                    const uint32_t* src = nullptr;
                    if (r < rows) {
                        const int t = r / a.group;
                        lim[hr] = key_limit(a, Sequence{c.x.first, c.x.count, c.x.keys}, t);
                        src = reinterpret_cast<const uint32_t*>(
                            q_row(a, c.x.first + t, (head0 + c.h) * a.group + r - t * a.group));
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        qf[kk][hr] = src ? __ldg(src + kk * 8 + t4) : 0u;
                        qf[kk][hr + 2] = src ? __ldg(src + kk * 8 + 4 + t4) : 0u;
                    }
                }
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int q = 0; q < 4; ++q) o[n][q] = 0.0f;
            }
            if (c.x.kv_end > 0) {
                const int slot = done % kRowStages;
                const bool got =
                    wait_phase(smem_u32(&sm.bar[warp][slot]), (done / kRowStages) & 1, abort_flag, a);
                if (!__all_sync(0xffffffffu, got)) {
                    ok = false;
                    break;
                }
                const uint32_t ks = smem_u32(sm.ring[warp][slot][0]);
                const uint32_t vs = smem_u32(sm.ring[warp][slot][1]);
                const int key0 = (c.unit0 + c.u) * kUnit;
                const int valid = c.x.kv_end - key0;
                // (The first token sees the fewest keys.)
                const int all_see = key_limit(a, Sequence{c.x.first, c.x.count, c.x.keys}, 0) - key0;
                if (all_see < kUnit) {  // some rows see only a part of the unit
                    uint4* v = reinterpret_cast<uint4*>(sm.ring[warp][slot][1]);
                    for (int i = valid * 8 + lane; i < kUnit * 8; i += 32) v[i] = make_uint4(0, 0, 0, 0);
                    if (all_see < min(valid, kUnit)) note_odd_values(v, min(valid, kUnit), lim[0] - key0, lim[1] - key0, odd);
                    fence_async_smem();  // ordered before the slot's next TMA write
                    __syncwarp();
                }
                // S = Q K^T
                float s[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int q = 0; q < 4; ++q) s[n][q] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int row = 16 * j + (lane >> 4) * 8 + (lane & 7);
                        const int chunk = (2 * kk + ((lane >> 3) & 1)) ^ (row & 7);
                        uint32_t kb[4];
                        ldsm4(ks + row * 128 + chunk * 16, kb);
                        mma_16816(s[2 * j], qf[kk], kb[0], kb[1]);
                        mma_16816(s[2 * j + 1], qf[kk], kb[2], kb[3]);
                    }
                // Running maximum, weights, and their two bf16 parts.
                uint32_t ph[2][4], pl[2][4];
#pragma unroll
                for (int hr = 0; hr < 2; ++hr) {
                    if (hr == 1 && rows <= 8) {  // no such rows
#pragma unroll
                        for (int n = 0; n < 4; ++n)
                            ph[n >> 1][1 + 2 * (n & 1)] = pl[n >> 1][1 + 2 * (n & 1)] = 0;
                        break;
                    }
                    if (key0 + kUnit > lim[hr]) {
#pragma unroll
                        for (int n = 0; n < 4; ++n)
#pragma unroll
                            for (int q = 0; q < 2; ++q)
                                if (key0 + n * 8 + 2 * t4 + q >= lim[hr]) s[n][2 * hr + q] = -INFINITY;
                    }
                    float mx = -INFINITY;
#pragma unroll
                    for (int n = 0; n < 4; ++n) mx = fmax3(mx, s[n][2 * hr], s[n][2 * hr + 1]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float mn = fmaxf(m[hr], mx * a.scale);
                    const float mu = mn == -INFINITY ? 0.0f : mn;
                    const float keep = ex2_approx(m[hr] - mu);
                    m[hr] = mn;
                    float sum = 0.0f;
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float p0 = ex2_approx(fmaf(s[n][2 * hr], a.scale, -mu));
                        const float p1 = ex2_approx(fmaf(s[n][2 * hr + 1], a.scale, -mu));
                        sum += p0 + p1;
                        const float h0 = below_bf16(p0), h1 = below_bf16(p1);
                        ph[n >> 1][hr + 2 * (n & 1)] = pack_bf16_trunc(h0, h1);
                        pl[n >> 1][hr + 2 * (n & 1)] = pack_bf16_rne(p0 - h0, p1 - h1);
                    }
                    l[hr] = l[hr] * keep + sum;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        o[n][2 * hr] *= keep;
                        o[n][2 * hr + 1] *= keep;
                    }
                }
                // O += P V
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int dp = 0; dp < 4; ++dp) {
                        const int row = 16 * st + ((lane >> 3) & 1) * 8 + (lane & 7);
                        const int chunk = (2 * dp + (lane >> 4)) ^ (row & 7);
                        uint32_t vb[4];
                        ldsm4_t(vs + row * 128 + chunk * 16, vb);
                        mma_16816(o[2 * dp], ph[st], vb[0], vb[1]);
                        mma_16816(o[2 * dp], pl[st], vb[0], vb[1]);
                        mma_16816(o[2 * dp + 1], ph[st], vb[2], vb[3]);
                        mma_16816(o[2 * dp + 1], pl[st], vb[2], vb[3]);
                    }
                ++done;
                __syncwarp();
            }
            const bool last = it + 1 == count;
            if (last || c.u + 1 == c.n) {
                // All of the head's units in this block: out with it, laid out by
                // rows in the ring slot just read.  A part of them: a piece, kept
                // for the block's fold.
                const bool all = u0 == 0 && c.u + 1 == c.n;
                const bool empty = c.x.kv_end == 0;  // no slot was read, and O is zero
                float* po = all ? reinterpret_cast<float*>(sm.ring[warp][(done + kRowStages - 1) % kRowStages])
                          : last ? reinterpret_cast<float*>(sm.ring[warp]) : sm.first_o[warp];
                float* pml = all || last ? po + kMostRows * kHeadDim : sm.first_ml[warp];
                const Target to{c.x.first, rows, head0 + c.h,
                                c.unit0 == 0 && c.n == c.x.units ? -1 : 2 * (int)blockIdx.x + (c.unit0 == 0)};
                if (!empty) {
#pragma unroll
                    for (int hr = 0; hr < 2; ++hr) {
                        float lt = l[hr];
                        lt += __shfl_xor_sync(0xffffffffu, lt, 1);
                        lt += __shfl_xor_sync(0xffffffffu, lt, 2);
                        const int rt = hr * 8 + g;
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                            *reinterpret_cast<float2*>(po + rt * kHeadDim + n * 8 + 2 * t4) =
                                make_float2(o[n][2 * hr], o[n][2 * hr + 1]);
                        if (t4 == 0) *reinterpret_cast<float2*>(pml + rt * 2) = make_float2(m[hr], lt);
                    }
                    for (uint32_t left = odd[0] | odd[1] | odd[2]; left != 0; left &= left - 1) {
                        const int i = __ffs(left) - 1;
                        float* x = po + ((i >> 1 & 1) * 8 + g) * kHeadDim + (i >> 2) * 8 + 2 * t4 + (i & 1);
                        if (odd[0] >> i & 1) *x = NAN;
                        if (odd[1] >> i & 1) *x += INFINITY;
                        if (odd[2] >> i & 1) *x -= INFINITY;
                    }
                    __syncwarp();
                }
                if (all) {
                    for (int rt = lane >> 4; rt < rows; rt += 2) {
                        float mr = -INFINITY, lr = 0.0f;
                        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (!empty) {
                            mr = pml[rt * 2];
                            lr = pml[rt * 2 + 1];
                            y = *reinterpret_cast<const float4*>(po + rt * kHeadDim + (lane & 15) * 4);
                        }
                        emit_row4(a, to, rt, lane & 15, mr, lr, y);
                    }
                    fence_async_smem();  // ordered before the slot's next TMA write
                    __syncwarp();
                } else if (lane == 0) {
                    sm.piece_to[warp][last] = to;
                    sm.piece_job[warp][last] = c.seg * heads + c.h;
                }
            }
            produce();
            advance(c);
        }
        if (!ok)
            for (int i = done; i < issued; ++i)
                drain_phase(smem_u32(&sm.bar[warp][i % kRowStages]), (i / kRowStages) & 1, a);
    }

    // What the block has to say of the sequences that begin in it.
    RowsHeader header{0, 0, 0, head0, heads, {0, 0, 0}};
    if (threadIdx.x == 0) {
        Cursor k = c0;
        for (bool more = any; more; more = next_segment(k)) {
            if (k.unit0 != 0) continue;
            int parts = 0;
            if (k.n < k.x.units) {
                // Only a last segment goes on; its cost ends that far past the block's.
                parts = (int)ranges.owner(end + (k.x.units - k.n) - 1) - index + 1;
                header.first = k.x.first;
                header.rows = k.x.count * a.group;
                header.parts = parts;
            }
            if (a.seq_parts != nullptr && group == 0) a.seq_parts[k.b] = make_int2(index, parts);
        }
    }

    // --------------------------------------------- the block's fold of pieces
    griddep_wait();  // the grid ends after the launch before it
    if (threadIdx.x == 0) piece_headers(a)[blockIdx.x] = header;
    __syncthreads();
    if (*abort_flag) return;
    // Runs of pieces of one head, in line order: run k is the pieces from the
    // k-th marked one to the next (every warp finds the same).
    const int my_job = lane < 2 * kRowWarps ? sm.piece_job[lane >> 1][lane & 1] : -1;
    const unsigned have = __ballot_sync(0xffffffffu, my_job >= 0);
    const unsigned below = have & ((1u << lane) - 1);
    const int job_before = __shfl_sync(0xffffffffu, my_job, below ? 31 - __clz(below) : 0);
    const bool begins = my_job >= 0 && (below == 0 || job_before != my_job);
    const unsigned runs = __ballot_sync(0xffffffffu, begins);
    if (begins) sm.run[__popc(runs & ((1u << lane) - 1))] = lane;  // the same from every warp
    if (lane == 0) sm.run[__popc(runs)] = 2 * kRowWarps;
    __syncwarp();
    // 16 threads per (run, row).
    const int c4 = threadIdx.x & 15;
    for (int x = threadIdx.x >> 4; x < __popc(runs) * a.row_cap; x += kRowThreadsTotal / 16) {
        const int k = x / a.row_cap, rt = x - k * a.row_cap;
        const int i = sm.run[k], next = sm.run[k + 1];
        const Target to = sm.piece_to[i >> 1][i & 1];
        if (rt >= to.rows) continue;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int j = i; j < next; ++j) {
            if (!((have >> j) & 1)) continue;
            const float* po = (j & 1) ? reinterpret_cast<const float*>(sm.ring[j >> 1]) : sm.first_o[j >> 1];
            const float* pml = (j & 1) ? po + kMostRows * kHeadDim : sm.first_ml[j >> 1];
            fold4(m, l, o, pml[rt * 2], pml[rt * 2 + 1],
                  *reinterpret_cast<const float4*>(po + rt * kHeadDim + c4 * 4));
        }
        emit_row4(a, to, rt, c4, m, l, o);
    }
}

// Folds the pieces of the sequence that begins in block `block` and goes on in
// the blocks after it, four rows at a time (256 threads, the part-th of parts_y
// blocks that share the rows).  64 threads per row: 16 cover the
// columns, the four sixteens take every fourth piece, kBatch of them in flight.
// kMergeBlocks per block of the rows kernel at most: a block without work costs
// a nanosecond, and most have none.
constexpr int kMergeBlocks = 16;
__device__ __forceinline__ void merge_pieces(const Args& a, int block, int part, int parts_y) {
    constexpr int kBatch = 8;
    __shared__ float4 other_o[4][16];
    __shared__ float2 other_ml[4][16];
    const RowsHeader hd = piece_headers(a)[block];
    if (hd.parts == 0) return;
    const int rows = hd.rows;
    for (int y0 = part * 4; y0 < rows * hd.heads; y0 += parts_y * 4) {
        const int y = y0 + (int)(threadIdx.x >> 6);
        const bool has_row = y < rows * hd.heads;
        const int h = has_row ? hd.h0 + y / rows : 0, rt = has_row ? y - y / rows * rows : 0;
        const int lane = threadIdx.x & 31, c4 = lane & 15;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (has_row)
            for (int k0 = (threadIdx.x >> 4) & 3; k0 < hd.parts; k0 += 4 * kBatch) {
                float2 ml[kBatch];
                float4 z[kBatch];
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const int k = k0 + 4 * u;
                    ml[u] = make_float2(-INFINITY, 0.0f);
                    z[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (k < hd.parts) {
                        const long long row = piece_row(a, 2 * (block + k) + (k == 0), h, rt);
                        ml[u] = *reinterpret_cast<const float2*>(piece_ml(a, row));
                        z[u] = *reinterpret_cast<const float4*>(piece_o(a, row) + c4 * 4);
                    }
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) fold4(m, l, o, ml[u].x, ml[u].y, z[u]);
            }
        // Within the warp, then the row's second warp.
        fold4(m, l, o, __shfl_xor_sync(0xffffffffu, m, 16), __shfl_xor_sync(0xffffffffu, l, 16),
              make_float4(__shfl_xor_sync(0xffffffffu, o.x, 16), __shfl_xor_sync(0xffffffffu, o.y, 16),
                          __shfl_xor_sync(0xffffffffu, o.z, 16), __shfl_xor_sync(0xffffffffu, o.w, 16)));
        const int slot = threadIdx.x >> 6;
        if ((threadIdx.x & 32) && lane < 16) {
            other_o[slot][c4] = o;
            other_ml[slot][c4] = make_float2(m, l);
        }
        __syncthreads();
        if (has_row && !(threadIdx.x & 32) && lane < 16) {
            fold4(m, l, o, other_ml[slot][c4].x, other_ml[slot][c4].y, other_o[slot][c4]);
            emit_row4(a, Target{hd.first, rows, h, -1}, rt, c4, m, l, o);
        }
        __syncthreads();
    }
}

// The end of a prefix call: every row's partial results of the prefix and of
// its own keys (one, or the pieces of a sequence that crossed blocks), folded
// into the final row.  16 threads per row, four columns each, kBatch loads in
// flight.  Bound by the partial results' bytes (192 tokens of 32 heads under
// 24577 keys: 12 us; with 16 in flight it was slower).
__global__ void __launch_bounds__(256)
fmha_prefix_finish(const __grid_constant__ Args a) {
    constexpr int kBatch = 8;
    const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4;
    const long long all_rows = (long long)a.tokens * a.nhead_q;
    const int c4 = threadIdx.x & 15;
    bool mine = row < all_rows;
    const int token = mine ? (int)(row / a.nhead_q) : 0, head = mine ? (int)(row - (long long)token * a.nhead_q) : 0;
    int b = token / a.row_div;
    if (a.seqstart_q != nullptr) {
        b = 0;
        for (int hi = a.batch; hi - b > 1;) {
            const int mid = (b + hi) >> 1;
            if (a.seqstart_q[mid] <= token) b = mid;
            else hi = mid;
        }
    }
    const Sequence s = load_sequence(a, b);
    const int rows = s.count * a.group;
    const int h = head / a.group, rt = (token - s.first) * a.group + head - h * a.group;
    mine = mine && token >= s.first && token < s.first + s.count && rows >= a.min_rows && rows <= a.max_rows;
    griddep_wait();  // every thread: the grid ends after the launches before it
    if (!mine) return;
    int2 parts = a.seq_parts[b];  // its first block (of each group of heads), and how many share it
    parts.x += h / a.group_heads * a.group_blocks;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // The prefix's parts and the sequence's own, if one (what is read there
    // otherwise stays out).
    for (int k0 = 0; k0 <= a.part_n; k0 += kBatch) {
        float m2[kBatch];
        float4 x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            m2[u] = -INFINITY;
            x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k0 + u > a.part_n) continue;
            m2[u] = a.part_lse[(k0 + u) * all_rows + row];
            x[u] = *reinterpret_cast<const float4*>(a.part_o + ((k0 + u) * all_rows + row) * kHeadDim + c4 * 4);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (m2[u] != -INFINITY && k0 + u < a.part_n + (parts.y == 0))  // -inf: O may be unwritten
                fold4(m, l, o, m2[u], 1.0f, x[u]);
    }
    for (int k0 = 0; k0 < parts.y; k0 += kBatch) {
        float2 ml[kBatch];
        float4 x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            ml[u] = make_float2(-INFINITY, 0.0f);
            x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k0 + u >= parts.y) continue;
            const long long at = piece_row(a, 2 * (parts.x + k0 + u) + (k0 + u == 0), h, rt);
            ml[u] = *reinterpret_cast<const float2*>(piece_ml(a, at));
            x[u] = *reinterpret_cast<const float4*>(piece_o(a, at) + c4 * 4);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) fold4(m, l, o, ml[u].x, ml[u].y, x[u]);
    }
    write_row4(a, token, head, c4 * 4, m, l, o, c4 == 0);
}

}  // namespace fmha_paged
