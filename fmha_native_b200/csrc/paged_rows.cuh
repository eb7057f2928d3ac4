// paged_rows.cuh -- attention of few query rows per K/V head over the paged
// cache: single tokens, a few drafted tokens, grouped query heads.
//
// What it computes per (sequence, K/V head): O = softmax(scale Q K^T) V for up
// to kRows rows that share the keys, as one pass over the keys with a running
// maximum m, weight sum l and un-normalised O per row (fp32).
//
// What bounds it: the cache is read once (256 bytes per key and K/V head) and
// the arithmetic per byte is small, so it should run at memory speed.  Hence:
//
//   work split   The keys of all (sequence, head) jobs are laid end to end in
//                units of 32 keys; the blocks, and inside a block its 8 warps,
//                take equal contiguous shares of that line.  Lengths may differ
//                as they like: every warp streams the same number of bytes.
//                A job that crosses shares leaves pieces (m, l, O), folded
//                inside the block through shared memory, and between blocks by
//                fmha_paged_rows_merge.  The shares follow from the lengths
//                alone, so results do not depend on timing.
//   streaming    Each warp has its own ring of kStages units in shared memory,
//                filled by TMA (one box per page) several units ahead, across
//                job boundaries too; no block-wide step until the share ends.
//   arithmetic   mma.sync m16n8k16 with the rows as M: the tile of a decode
//                step is far too thin for a 128-row tensor-memory tile, and
//                the reads leave the tensor pipe idle anyway.  P enters the
//                second product as a sum of two bf16 (value and remainder), so
//                O keeps fp32 accuracy until its one rounding at the end.
//
// Keys past a row's limit get weight 0 by selection, and value rows past the
// tile's last visible key are zeroed in shared memory before use, so whatever
// the page holds there (NaN included) stays out of O.
#pragma once
#include "paged_common.cuh"

namespace fmha_paged {

constexpr int kUnit = 32;             // keys per unit
constexpr int kRowWarps = 8;
constexpr int kRowThreadsTotal = 32 * kRowWarps;
constexpr int kUnitBytes = kUnit * kHeadDim * 2;  // 4 KB of K, as much of V
constexpr int kMaxRowBlocks = 148;    // one block per SM

constexpr int row_stages(int mt) { return mt == 1 ? 3 : 2; }

template <int MT>
struct alignas(1024) RowsShared {
    static constexpr int kRows = 16 * MT;
    static constexpr int kStages = row_stages(MT);
    uint8_t ring[kRowWarps][kStages][2][kUnitBytes];
    // A piece whose job ended inside the warp's share; a piece at the share's
    // end reuses the warp's (then idle) ring.
    float first_o[kRowWarps][kRows * kHeadDim];
    float first_ml[kRowWarps][kRows * 2];
    uint64_t bar[kRowWarps][kStages];
    long long scan[kRowWarps];
    long long piece_job[kRowWarps][2];
    int piece_flags[kRowWarps][2];    // -1: none; bit 0: job begins, bit 1: job ends here
    int piece_left[kRowWarps][2];     // units of the job after this piece
    int start_entry[kRowWarps];
    int start_off[kRowWarps];
    int abort_flag;
};

// Scratch between blocks: two piece slots per block, then one header each.
struct RowsHeader {
    long long job;
    int parts;   // blocks that share the job beginning in this block; 0: none
    int pad;
};
__host__ __device__ constexpr size_t rows_piece_floats(int rows) { return (size_t)rows * (kHeadDim + 2); }
__host__ __device__ constexpr size_t rows_scratch_bytes(int rows) {
    return kMaxRowBlocks * (2 * rows_piece_floats(rows) * sizeof(float) + sizeof(RowsHeader));
}
__device__ __forceinline__ float* piece_o(const Args& a, int rows, int slot) {
    return a.pieces + (size_t)slot * rows * kHeadDim;
}
__device__ __forceinline__ float* piece_ml(const Args& a, int rows, int slot) {
    return a.pieces + (size_t)2 * kMaxRowBlocks * rows * kHeadDim + (size_t)slot * rows * 2;
}
__device__ __forceinline__ RowsHeader* piece_headers(const Args& a, int rows) {
    return reinterpret_cast<RowsHeader*>(a.pieces + 2 * kMaxRowBlocks * rows_piece_floats(rows));
}

// One row tile of one sequence; its job exists once per K/V head.
struct Entry {
    Sequence s;
    int b;
    int row0, rows;  // first row of the tile; rows of the sequence
    int kv_end;      // keys that any row of the tile sees
    int units;       // 0: nothing to do; a tile that sees no key counts one (empty) unit
};
template <int kRows>
__device__ __forceinline__ Entry load_entry(const Args& a, int e) {
    Entry x;
    x.b = e / a.m_tiles;
    x.row0 = (e - x.b * a.m_tiles) * kRows;
    x.s = load_sequence(a, x.b);
    x.rows = x.s.count * a.group;
    x.units = 0;
    x.kv_end = 0;
    if (x.rows < a.min_rows || x.rows > a.max_rows) x.rows = 0;
    if (x.rows > a.m_tiles * kRows) flag_index_error(a.err_word);  // more tokens than the call said
    if (x.row0 >= x.rows) return x;
    const int t_last = (min(x.rows, x.row0 + kRows) - 1) / a.group;
    x.kv_end = max(0, key_limit(a, x.s, t_last));
    x.units = max(1, (x.kv_end + kUnit - 1) / kUnit);
    return x;
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
__device__ __forceinline__ void fence_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Equal contiguous shares of `total` units: share c of n starts at
// c * base + min(c, rem).
struct Shares {
    long long base, rem;
    int n;
    __device__ Shares(long long total, int n_) : base(total / n_), rem(total % n_), n(n_) {}
    __device__ long long begin(int c) const { return c * base + min((long long)c, rem); }
    __device__ int owner(long long x) const {
        const long long wide = rem * (base + 1);
        return x < wide ? (int)(x / (base + 1)) : (int)(rem + (x - wide) / base);
    }
};

template <int MT>
__global__ void __launch_bounds__(kRowThreadsTotal, 1)
fmha_paged_rows_kernel(const __grid_constant__ Args a) {
    using Shared = RowsShared<MT>;
    constexpr int kRows = Shared::kRows;
    constexpr int kStages = Shared::kStages;
    extern __shared__ uint8_t smem_raw[];
    Shared& sm = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                            ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    volatile int* abort_flag = &sm.abort_flag;
    RowsHeader* headers = piece_headers(a, kRows);

    griddep_launch_dependents();
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&sm.bar[warp][s]), 1);
        sm.piece_flags[warp][0] = sm.piece_flags[warp][1] = -1;
        if (warp == 0) sm.abort_flag = 0;
        fence_barrier_init();
    }

    // ------------------------------------------------- shares of the line
    const int entries = a.batch * a.m_tiles;
    const int per = (entries + kRowThreadsTotal - 1) / kRowThreadsTotal;
    const int e0 = min(entries, (int)threadIdx.x * per), e1 = min(entries, e0 + per);
    long long mine = 0;
    for (int e = e0; e < e1; ++e) mine += (long long)load_entry<kRows>(a, e).units * a.nhead_k;
    long long incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 31) sm.scan[warp] = incl;
    __syncthreads();
    long long before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
        if (w < warp) before += sm.scan[w];
        total += sm.scan[w];
    }
    const long long want = (total + kRowWarps - 1) / kRowWarps;
    const int blocks = (int)min((long long)gridDim.x, want);
    if ((int)blockIdx.x >= blocks) {
        griddep_wait();  // the grid ends after the launch before it
        if (threadIdx.x == 0) headers[blockIdx.x].parts = 0;
        return;
    }
    const Shares shares(total, blocks);
    const long long beg = shares.begin(blockIdx.x), end = shares.begin(blockIdx.x + 1);
    const long long len = end - beg;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
        const long long x = beg + len * w / kRowWarps;
        if (x >= before && x < before + mine) {
            long long p = before;
            for (int e = e0; e < e1; ++e) {
                const long long c = (long long)load_entry<kRows>(a, e).units * a.nhead_k;
                if (x < p + c) {
                    sm.start_entry[w] = e;
                    sm.start_off[w] = (int)(x - p);
                    break;
                }
                p += c;
            }
        }
    }
    __syncthreads();
    const int count = (int)(len * (warp + 1) / kRowWarps - len * warp / kRowWarps);

    // ------------------------------------------------------- the share
    // Two cursors over the line: `p` issues loads, `c` computes.
    struct Cursor {
        Entry x;
        int e, h, u;
    };
    auto advance = [&](Cursor& k) {
        if (++k.u < k.x.units) return;
        k.u = 0;
        if (++k.h < a.nhead_k) return;
        k.h = 0;
        do {
            if (++k.e >= entries) return;
            k.x = load_entry<kRows>(a, k.e);
        } while (k.x.units == 0);
    };
    if (count > 0) {
        Cursor c;
        c.e = sm.start_entry[warp];
        c.x = load_entry<kRows>(a, c.e);
        c.h = sm.start_off[warp] / c.x.units;
        c.u = sm.start_off[warp] - c.h * c.x.units;
        Cursor p = c;
        int to_issue = count, issued = 0, done = 0;

        // Page ids: lane i holds entry win + i of sequence win_b's table row.
        const int box_rows = min(1 << a.page_shift, kUnit);
        const int boxes = kUnit / box_rows;
        int win_b = -1, win = 0, ids = 0, ids_next = 0;
        auto load_ids = [&](int b, int first, int pages) {
            const int i = first + lane;
            return i < pages ? __ldg(a.page_table + b * a.table_stride + i) : 0;
        };
        const uint64_t policy = l2_policy_evict_first();
        if (lane == 0) {
            tma_prefetch_desc(&a.tm_k);
            tma_prefetch_desc(&a.tm_v);
        }
        auto produce = [&]() {
            while (to_issue > 0 && issued - done < kStages) {
                if (p.x.kv_end > 0) {
                    const int key0 = p.u * kUnit;
                    const int pages = (p.x.s.keys + (1 << a.page_shift) - 1) >> a.page_shift;
                    const int page0 = key0 >> a.page_shift;
                    if (win_b != p.x.b || page0 < win || page0 >= win + 64) {
                        win_b = p.x.b;
                        win = page0 & ~3;
                        ids = load_ids(win_b, win, pages);
                        ids_next = load_ids(win_b, win + 32, pages);
                    } else if (page0 >= win + 32) {
                        win += 32;
                        ids = ids_next;
                        ids_next = load_ids(win_b, win + 32, pages);
                    }
                    const int nbox = min(boxes, (p.x.kv_end - key0 + box_rows - 1) / box_rows);
                    const int slot = issued % kStages;
                    const uint32_t bar = smem_u32(&sm.bar[warp][slot]);
                    if (lane == 0) mbar_arrive_expect_tx(bar, 2 * nbox * box_rows * kHeadDim * 2);
                    __syncwarp();
                    // Lanes 0..nbox-1 load K boxes, the next nbox V boxes.
                    const int box = lane < nbox ? lane : lane - nbox;
                    const int id = __shfl_sync(0xffffffffu, ids, (page0 + box - win) & 31);
                    if (lane < 2 * nbox) {
                        if (id < 0 || id >= a.num_pages) flag_index_error(a.err_word);
                        const bool is_v = lane >= nbox;
                        load_page_box(smem_u32(&sm.ring[warp][slot][is_v][box * box_rows * kHeadDim * 2]),
                                      is_v ? &a.tm_v : &a.tm_k, bar, key0 & ((1 << a.page_shift) - 1), p.h,
                                      id, policy);
                    }
                    ++issued;
                }
                advance(p);
                --to_issue;
            }
        };
        produce();

        const int g = lane >> 2, t4 = lane & 3;
        uint32_t qf[MT][4][4];
        float o[MT][8][4], m[MT][2], l[MT][2];
        int lim[MT][2];
        int seg_begin = 0;
        bool ok = true;
        for (int it = 0; it < count; ++it) {
            if (it == 0 || c.u == 0) {
                seg_begin = c.u;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
#pragma unroll
                    for (int hr = 0; hr < 2; ++hr) {
                        const int r = c.x.row0 + i * 16 + hr * 8 + g;
                        m[i][hr] = -INFINITY;
                        l[i][hr] = 0.0f;
                        lim[i][hr] = 0;
                        const uint32_t* src = nullptr;
                        if (r < c.x.rows) {
                            const int t = r / a.group;
                            lim[i][hr] = key_limit(a, c.x.s, t);
                            src = reinterpret_cast<const uint32_t*>(
                                q_row(a, c.x.s.first + t, c.h * a.group + r - t * a.group));
                        }
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            qf[i][kk][hr] = src ? __ldg(src + kk * 8 + t4) : 0u;
                            qf[i][kk][hr + 2] = src ? __ldg(src + kk * 8 + 4 + t4) : 0u;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int q = 0; q < 4; ++q) o[i][n][q] = 0.0f;
                }
            }
            if (c.x.kv_end > 0) {
                const int slot = done % kStages;
                const bool got =
                    wait_phase(smem_u32(&sm.bar[warp][slot]), (done / kStages) & 1, abort_flag, a);
                if (!__all_sync(0xffffffffu, got)) {
                    ok = false;
                    break;
                }
                const uint32_t ks = smem_u32(sm.ring[warp][slot][0]);
                const uint32_t vs = smem_u32(sm.ring[warp][slot][1]);
                const int key0 = c.u * kUnit;
                const int valid = c.x.kv_end - key0;
                if (valid < kUnit) {
                    uint4* v = reinterpret_cast<uint4*>(sm.ring[warp][slot][1]);
                    for (int i = valid * 8 + lane; i < kUnit * 8; i += 32) v[i] = make_uint4(0, 0, 0, 0);
                    fence_async_smem();  // ordered before the slot's next TMA write
                    __syncwarp();
                }
                // S = Q K^T
                float s[MT][4][4];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int q = 0; q < 4; ++q) s[i][n][q] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int row = 16 * j + (lane >> 4) * 8 + (lane & 7);
                        const int chunk = (2 * kk + ((lane >> 3) & 1)) ^ (row & 7);
                        uint32_t kb[4];
                        ldsm4(ks + row * 128 + chunk * 16, kb);
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            mma_16816(s[i][2 * j], qf[i][kk], kb[0], kb[1]);
                            mma_16816(s[i][2 * j + 1], qf[i][kk], kb[2], kb[3]);
                        }
                    }
                // Running maximum, weights, and their two bf16 parts.
                uint32_t ph[MT][2][4], pl[MT][2][4];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int hr = 0; hr < 2; ++hr) {
                        if (key0 + kUnit > lim[i][hr]) {
#pragma unroll
                            for (int n = 0; n < 4; ++n)
#pragma unroll
                                for (int q = 0; q < 2; ++q)
                                    if (key0 + n * 8 + 2 * t4 + q >= lim[i][hr]) s[i][n][2 * hr + q] = -INFINITY;
                        }
                        float mx = -INFINITY;
#pragma unroll
                        for (int n = 0; n < 4; ++n) mx = fmax3(mx, s[i][n][2 * hr], s[i][n][2 * hr + 1]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const float mn = fmaxf(m[i][hr], mx * a.scale);
                        const float mu = mn == -INFINITY ? 0.0f : mn;
                        const float keep = ex2_approx(m[i][hr] - mu);
                        m[i][hr] = mn;
                        float sum = 0.0f;
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const float p0 = ex2_approx(fmaf(s[i][n][2 * hr], a.scale, -mu));
                            const float p1 = ex2_approx(fmaf(s[i][n][2 * hr + 1], a.scale, -mu));
                            sum += p0 + p1;
                            const uint32_t hi = pack_bf16_rne(p0, p1);
                            ph[i][n >> 1][hr + 2 * (n & 1)] = hi;
                            pl[i][n >> 1][hr + 2 * (n & 1)] =
                                pack_bf16_rne(p0 - __uint_as_float(hi << 16),
                                              p1 - __uint_as_float(hi & 0xffff0000u));
                        }
                        l[i][hr] = l[i][hr] * keep + sum;
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            o[i][n][2 * hr] *= keep;
                            o[i][n][2 * hr + 1] *= keep;
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
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            mma_16816(o[i][2 * dp], ph[i][st], vb[0], vb[1]);
                            mma_16816(o[i][2 * dp], pl[i][st], vb[0], vb[1]);
                            mma_16816(o[i][2 * dp + 1], ph[i][st], vb[2], vb[3]);
                            mma_16816(o[i][2 * dp + 1], pl[i][st], vb[2], vb[3]);
                        }
                    }
                ++done;
                __syncwarp();
            }
            produce();

            const bool last = it + 1 == count;
            if (last || c.u + 1 == c.x.units) {
                const bool begins = seg_begin == 0, ends = c.u + 1 == c.x.units;
                const bool whole = begins && ends;
                griddep_wait();  // a launch before this one may hold partial results of the row
                float* po = last ? reinterpret_cast<float*>(sm.ring[warp]) : sm.first_o[warp];
                float* pml = last ? po + kRows * kHeadDim : sm.first_ml[warp];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int hr = 0; hr < 2; ++hr) {
                        float lt = l[i][hr];
                        lt += __shfl_xor_sync(0xffffffffu, lt, 1);
                        lt += __shfl_xor_sync(0xffffffffu, lt, 2);
                        const int rt = i * 16 + hr * 8 + g;
                        const int r = c.x.row0 + rt;
                        if (r >= c.x.rows) continue;
                        if (!whole) {
#pragma unroll
                            for (int n = 0; n < 8; ++n)
                                *reinterpret_cast<float2*>(po + rt * kHeadDim + n * 8 + 2 * t4) =
                                    make_float2(o[i][n][2 * hr], o[i][n][2 * hr + 1]);
                            if (t4 == 0) {
                                pml[rt * 2] = m[i][hr];
                                pml[rt * 2 + 1] = lt;
                            }
                            continue;
                        }
                        const int t = r / a.group;
                        const int token = c.x.s.first + t, head = c.h * a.group + r - t * a.group;
                        const long long row = flat_row(a, token, head);
                        const long long rows = (long long)a.tokens * a.nhead_q;
                        float mm = m[i][hr];
                        for (int s = 0; s < a.part_n; ++s) {
                            const float m2 = a.part_lse[s * rows + row];
                            if (m2 == -INFINITY) continue;
                            const Fold f = fold_scales(mm, m2);
                            lt = lt * f.keep + f.take;
                            const float* x = a.part_o + (s * rows + row) * kHeadDim + 2 * t4;
#pragma unroll
                            for (int n = 0; n < 8; ++n) {
                                const float2 y = *reinterpret_cast<const float2*>(x + n * 8);
                                o[i][n][2 * hr] = o[i][n][2 * hr] * f.keep + y.x * f.take;
                                o[i][n][2 * hr + 1] = o[i][n][2 * hr + 1] * f.keep + y.y * f.take;
                            }
                        }
                        const float inv = lt > 0.0f ? 1.0f / lt : 0.0f;
                        const float lse2 = lt > 0.0f ? mm + __log2f(lt) : -INFINITY;
                        uint32_t* dst = reinterpret_cast<uint32_t*>(o_row(a, token, head));
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                            dst[n * 4 + t4] = pack_bf16_rne(o[i][n][2 * hr] * inv, o[i][n][2 * hr + 1] * inv);
                        if (t4 == 0 && a.lse != nullptr) *lse_at(a, token, head) = lse2 * kLn2;
                    }
                if (!whole && lane == 0) {
                    sm.piece_job[warp][last] = (long long)c.e * a.nhead_k + c.h;
                    sm.piece_left[warp][last] = c.x.units - 1 - c.u;
                    sm.piece_flags[warp][last] = (begins ? 1 : 0) | (ends ? 2 : 0);
                }
            }
            advance(c);
        }
        if (!ok)
            for (int i = done; i < issued; ++i)
                drain_phase(smem_u32(&sm.bar[warp][i % kStages]), (i / kStages) & 1, a);
    }

    // ------------------------------------- pieces: inside the block, then out
    griddep_wait();
    __syncthreads();
    RowsHeader header{0, 0, 0};
    if (!*abort_flag) {
        const int c4 = threadIdx.x & 15;
        for (int i = 0; i < 2 * kRowWarps;) {
            const int flags = sm.piece_flags[i >> 1][i & 1];
            if (flags < 0) {
                ++i;
                continue;
            }
            const long long job = sm.piece_job[i >> 1][i & 1];
            int last = i, next = i + 1;
            for (; next < 2 * kRowWarps; ++next) {
                if (sm.piece_flags[next >> 1][next & 1] < 0) continue;
                if (sm.piece_job[next >> 1][next & 1] != job) break;
                last = next;
            }
            const bool begins = flags & 1, ends = sm.piece_flags[last >> 1][last & 1] & 2;
            const int slot = 2 * (int)blockIdx.x + (begins ? 1 : 0);
            const Entry x = load_entry<kRows>(a, (int)(job / a.nhead_k));
            const int h = (int)(job % a.nhead_k);
#pragma unroll
            for (int pass = 0; pass < MT; ++pass) {
                const int rt = pass * 16 + (int)(threadIdx.x >> 4);
                const int r = x.row0 + rt;
                if (r >= x.rows) continue;
                float m = -INFINITY, l = 0.0f;
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int k = i; k <= last; ++k) {
                    if (sm.piece_flags[k >> 1][k & 1] < 0) continue;
                    const float* po = (k & 1) ? reinterpret_cast<const float*>(sm.ring[k >> 1])
                                              : sm.first_o[k >> 1];
                    const float* pml = (k & 1) ? po + kRows * kHeadDim : sm.first_ml[k >> 1];
                    const Fold f = fold_scales(m, pml[rt * 2]);
                    l = l * f.keep + pml[rt * 2 + 1] * f.take;
                    const float4 y = *reinterpret_cast<const float4*>(po + rt * kHeadDim + c4 * 4);
                    o.x = o.x * f.keep + y.x * f.take;
                    o.y = o.y * f.keep + y.y * f.take;
                    o.z = o.z * f.keep + y.z * f.take;
                    o.w = o.w * f.keep + y.w * f.take;
                }
                if (begins && ends) {
                    const int t = r / a.group;
                    finish_row4(a, x.s.first + t, h * a.group + r - t * a.group, c4 * 4, m, l, o, c4 == 0);
                } else {
                    *reinterpret_cast<float4*>(piece_o(a, kRows, slot) + rt * kHeadDim + c4 * 4) = o;
                    if (c4 == 0)
                        *reinterpret_cast<float2*>(piece_ml(a, kRows, slot) + rt * 2) = make_float2(m, l);
                }
            }
            if (begins && !ends) {
                const long long job_end = end + sm.piece_left[last >> 1][last & 1];
                header.job = job;
                header.parts = shares.owner(job_end - 1) - (int)blockIdx.x + 1;
            }
            i = next;
        }
    }
    if (threadIdx.x == 0) headers[blockIdx.x] = header;
}

// Folds the pieces of the job that begins in block blockIdx.x and goes on in
// the blocks after it.  One warp per row: 16 lanes cover the columns, the two
// halves take alternate pieces.
template <int MT>
__global__ void __launch_bounds__(256)
fmha_paged_rows_merge(const __grid_constant__ Args a) {
    constexpr int kRows = 16 * MT;
    griddep_wait();
    const RowsHeader hd = piece_headers(a, kRows)[blockIdx.x];
    if (hd.parts == 0) return;
    const Entry x = load_entry<kRows>(a, (int)(hd.job / a.nhead_k));
    const int h = (int)(hd.job % a.nhead_k);
    const int rt = blockIdx.y * 8 + (int)(threadIdx.x >> 5);
    const int r = x.row0 + rt;
    if (r >= x.rows) return;
    const int lane = threadIdx.x & 31, c4 = lane & 15;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int kBatch = 4;  // pieces in flight per half
    for (int k0 = lane >> 4; k0 < hd.parts; k0 += 2 * kBatch) {
        float2 ml[kBatch];
        float4 y[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int k = k0 + 2 * u;
            ml[u] = make_float2(-INFINITY, 0.0f);
            y[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k < hd.parts) {
                const int slot = 2 * ((int)blockIdx.x + k) + (k == 0 ? 1 : 0);
                ml[u] = *reinterpret_cast<const float2*>(piece_ml(a, kRows, slot) + rt * 2);
                y[u] = *reinterpret_cast<const float4*>(piece_o(a, kRows, slot) + rt * kHeadDim + c4 * 4);
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const Fold f = fold_scales(m, ml[u].x);
            l = l * f.keep + ml[u].y * f.take;
            o.x = o.x * f.keep + y[u].x * f.take;
            o.y = o.y * f.keep + y[u].y * f.take;
            o.z = o.z * f.keep + y[u].z * f.take;
            o.w = o.w * f.keep + y[u].w * f.take;
        }
    }
    // The other half's state (every lane of the warp is here: r is per warp).
    const float m2 = __shfl_xor_sync(0xffffffffu, m, 16);
    const float l2 = __shfl_xor_sync(0xffffffffu, l, 16);
    const float4 y = make_float4(
        __shfl_xor_sync(0xffffffffu, o.x, 16), __shfl_xor_sync(0xffffffffu, o.y, 16),
        __shfl_xor_sync(0xffffffffu, o.z, 16), __shfl_xor_sync(0xffffffffu, o.w, 16));
    const Fold f = fold_scales(m, m2);
    l = l * f.keep + l2 * f.take;
    o.x = o.x * f.keep + y.x * f.take;
    o.y = o.y * f.keep + y.y * f.take;
    o.z = o.z * f.keep + y.z * f.take;
    o.w = o.w * f.keep + y.w * f.take;
    if (lane < 16) {
        const int t = r / a.group;
        finish_row4(a, x.s.first + t, h * a.group + r - t * a.group, c4 * 4, m, l, o, c4 == 0);
    }
}

}  // namespace fmha_paged
