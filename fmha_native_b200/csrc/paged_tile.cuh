// paged_tile.cuh -- attention of many query rows per K/V head over the paged
// cache: prompt chunks, and a whole batch's rows against a shared prefix.
//
// One block owns a tile of 128 rows (tokens x query heads of one K/V head's
// group, so a tile's rows share their keys) and walks the keys in tiles of
// 128; two blocks share an SM, each with its own pipeline, so one block's
// softmax runs under the other's matrix products:
//
//   warps 0-3  softmax   one row per thread (tensor-memory lane = row); they
//                        also stage Q and write O
//   warp  4    loads     K and V tiles by TMA, one box per page (or per 128
//                        keys of a larger page), into a ring of kStages slots
//   warp  5    products  one elected lane issues every tcgen05.mma; before the
//                        last one the warp zeroes the value rows past the last
//                        visible key, so what a page holds there (NaN included)
//                        stays out of O
//   warps 6-7  idle      complete the warpgroup for setmaxnreg
//
// Tensor memory of a block (256 of 512 columns): S [0,128), O [128,192), P as
// bf16 pairs [192,256).
//
// Softmax: running maximum per row in log2 units with lazy rescaling (O is
// rescaled only when the maximum grew by more than 2^8; P stays below that).
// P is rounded to nearest bf16 for the second product, which is what the
// tensor pipe takes; the row sum adds the unrounded fp32 values.
//
// What bounds it: per key tile a block runs 16384 exponentials against 2 x
// 128 x 128 x 64 multiply-adds, so the special-function unit (16 per clock)
// would need twice the tensor pipe's time; a quarter of the exponentials
// therefore runs as a polynomial on the FMA pipe.
//
// Few row tiles: each tile's keys are cut into `splits` equal ranges, a block
// each, whose normalised results are folded by fmha_paged_combine (or by the
// rows kernel that ends a prefix call).
#pragma once
#include <type_traits>

#include "paged_common.cuh"

namespace fmha_paged {

constexpr int kTileM = 128;
constexpr int kTileN = 128;
constexpr int kTileStages = 4;
constexpr int kTileBytes = 128 * kHeadDim * 2;  // 16 KB: Q, K or V tile
constexpr int kTileThreads = 256;
constexpr int kTileBlocks = 2 * 148;            // resident blocks of the device
constexpr uint32_t kTileTmemCols = 256;
constexpr uint32_t kColS = 0, kColO = 128, kColP = 192;
// setmaxnreg split of the launch's 256 x 128 registers.
constexpr int kTileRegsSoftmax = 192, kTileRegsControl = 64;
static_assert(128 * (kTileRegsSoftmax + kTileRegsControl) <= kTileThreads * 128, "register split");
constexpr float kLazyLog2 = 8.0f;
constexpr int kPolyOf16 = 4;  // pairs of every 16 whose exponential runs on the FMA pipe

struct alignas(1024) TileShared {
    uint8_t q[kTileBytes];
    uint8_t kv[kTileStages][kTileBytes];
    uint64_t bar_q;                   // Q staged (128 arrivals)
    uint64_t bar_full[kTileStages];
    uint64_t bar_empty[kTileStages];
    uint64_t bar_s;                   // S written (commit)
    uint64_t bar_sfree;               // S in registers (a thread's arrival per row)
    uint64_t bar_p;                   // P written, O rescaled (likewise)
    uint64_t bar_pv;                  // O += P V done (commit)
    uint64_t bar_drain;
    uint32_t tmem_base;
    int abort_flag;
    int warp_tiles[8];
    int found_b, found_m, found_total;
};

// 2^x for a pair on the FMA and integer pipes: x = n + f, n = round(x), and a
// degree-4 minimax polynomial for 2^f on [-1/2, 1/2] (relative error 3e-6,
// csrc/fit_exp2_poly.py with deg = 4), scaled by 2^n in the exponent field.
// x is finite and clamped from below.
__device__ __forceinline__ float2 exp2_poly4(float2 x) {
    constexpr float kRound = 12582912.0f;  // 1.5 * 2^23
    x.x = fmaxf(x.x, -120.0f);
    x.y = fmaxf(x.y, -120.0f);
    const float2 t = fadd2(x, make_float2(kRound, kRound));
    const float2 n = fadd2(t, make_float2(-kRound, -kRound));
    const float2 f = ffma2(n, make_float2(-1.0f, -1.0f), x);
    float2 p = ffma2(make_float2(9.570101276e-03f, 9.570101276e-03f), f, make_float2(5.591786280e-02f, 5.591786280e-02f));
    p = ffma2(p, f, make_float2(2.402474433e-01f, 2.402474433e-01f));
    p = ffma2(p, f, make_float2(6.931217909e-01f, 6.931217909e-01f));
    p = ffma2(p, f, make_float2(9.999992847e-01f, 9.999992847e-01f));
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                       __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

// Row tile `slot` of the grid -> (sequence, tile), tiles of later tokens (the
// ones with more keys) first.  All threads; false: past the last tile.
__device__ __forceinline__ bool find_tile(const Args& a, TileShared& sm, int slot, int& b, int& m) {
    if (a.seqstart_q == nullptr) {
        const int tiles = (a.seqlen_q * a.group + kTileM - 1) / kTileM;
        m = tiles - 1 - slot / a.batch;
        b = slot % a.batch;
        return m >= 0;
    }
    auto tiles_of = [&](int i) {
        const int rows = load_sequence(a, i).count * a.group;
        return rows < a.min_rows || rows > a.max_rows ? 0 : (rows + kTileM - 1) / kTileM;
    };
    const int per = (a.batch + kTileThreads - 1) / kTileThreads;
    const int b0 = min(a.batch, (int)threadIdx.x * per), b1 = min(a.batch, b0 + per);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int mine = 0;
    for (int i = b0; i < b1; ++i) mine += tiles_of(i);
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 31) sm.warp_tiles[warp] = incl;
    __syncthreads();
    int before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        if (w < warp) before += sm.warp_tiles[w];
        total += sm.warp_tiles[w];
    }
    if (slot >= total) return false;
    const int x = total - 1 - slot;
    if (x >= before && x < before + mine) {
        for (int i = b0, p = before; i < b1; ++i) {
            const int n = tiles_of(i);
            if (x < p + n) {
                sm.found_b = i;
                sm.found_m = x - p;
                break;
            }
            p += n;
        }
    }
    __syncthreads();
    b = sm.found_b;
    m = sm.found_m;
    return true;
}

__global__ void __launch_bounds__(kTileThreads, 2)
fmha_paged_tile_kernel(const __grid_constant__ Args a) {
    extern __shared__ uint8_t smem_raw[];
    TileShared& sm = *reinterpret_cast<TileShared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                    ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &sm.abort_flag;

    // What follows on the stream may be scheduled as soon as this grid's last
    // blocks run; it waits for their results where it needs them.
    griddep_launch_dependents();

    // Blocks in order: row tile, K/V head, key range.
    const int split = blockIdx.x % a.splits;
    const int head_slot = blockIdx.x / a.splits;
    const int kvh = head_slot % a.nhead_k;
    int b, mt;
    if (!find_tile(a, sm, head_slot / a.nhead_k, b, mt)) return;
    const Sequence seq = load_sequence(a, b);
    const int rows = seq.count * a.group;
    const int row0 = mt * kTileM;
    if (rows < a.min_rows || rows > a.max_rows || row0 >= rows) return;
    const int row_end = min(rows, row0 + kTileM);
    const int kv_end = max(0, key_limit(a, seq, (row_end - 1) / a.group));
    const int all = (kv_end + kTileN - 1) / kTileN;
    const int chunk = (all + a.splits - 1) / a.splits;
    const int j0 = split * chunk;
    const int n = max(0, min(all, j0 + chunk) - j0);
    const int tail = kv_end - (j0 + n - 1) * kTileN;  // visible keys of the range's last tile
    const bool has_tail = n > 0 && tail < kTileN;
    const int active = (row_end - row0 + 31) / 32;    // softmax warps with rows

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&sm.bar_q), 128);
        for (int s = 0; s < kTileStages; ++s) {
            mbar_init(smem_u32(&sm.bar_full[s]), 1);
            mbar_init(smem_u32(&sm.bar_empty[s]), 1);
        }
        mbar_init(smem_u32(&sm.bar_s), 1);
        mbar_init(smem_u32(&sm.bar_sfree), 32 * active);
        mbar_init(smem_u32(&sm.bar_p), 32 * active);
        mbar_init(smem_u32(&sm.bar_pv), 1);
        mbar_init(smem_u32(&sm.bar_drain), 1);
        sm.abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 5) {
        tmem_alloc(smem_u32(&sm.tmem_base), kTileTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    // K_j is load 2j, V_j load 2j + 1 of the ring.
    auto slot_of = [](int i) { return i % kTileStages; };
    auto phase_of = [](int i) { return (uint32_t)((i / kTileStages) & 1); };

    if (warp >= 4) {
        regs_dec<kTileRegsControl>();
        if (warp == 4 && n > 0) {
            // ---------------------------------------------------- loads
            if (lane == 0) {
                tma_prefetch_desc(&a.tm_k);
                tma_prefetch_desc(&a.tm_v);
            }
            const uint64_t policy = l2_policy_evict_last();
            const int box_rows = min(1 << a.page_shift, kTileN);
            const int32_t* table = a.page_table + b * a.table_stride;
            // Lane i loads box i of a tile: box_rows keys of one page.
            auto page_of = [&](int j) {
                const int key = (j0 + j) * kTileN + lane * box_rows;
                return lane * box_rows < kTileN && key < kv_end ? __ldg(table + (key >> a.page_shift)) : 0;
            };
            int page = page_of(0);
            bool ok = true;
            int issued = 0;
            for (int j = 0; j < n && ok; ++j) {
                const int next = j + 1 < n ? page_of(j + 1) : 0;
                const int key0 = (j0 + j) * kTileN;
                const int boxes = (min(kTileN, kv_end - key0) + box_rows - 1) / box_rows;
                if (lane < boxes && (page < 0 || page >= a.num_pages)) flag_index_error(a.err_word);
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int i = 2 * j + v, slot = slot_of(i);
                    ok = wait_phase(smem_u32(&sm.bar_empty[slot]), phase_of(i) ^ 1, abort_flag, a);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint32_t bar = smem_u32(&sm.bar_full[slot]);
                    if (lane == 0) mbar_arrive_expect_tx(bar, boxes * box_rows * kHeadDim * 2);
                    __syncwarp();
                    if (lane < boxes)
                        load_page_box(smem_u32(sm.kv[slot]) + lane * box_rows * kHeadDim * 2,
                                      v ? &a.tm_v : &a.tm_k, bar, (key0 + lane * box_rows) & ((1 << a.page_shift) - 1),
                                      kvh, page, policy);
                    issued = i + 1;
                }
                page = next;
            }
            if (!ok || *abort_flag)
                for (int i = max(0, issued - kTileStages); i < issued; ++i)
                    drain_phase(smem_u32(&sm.bar_full[slot_of(i)]), phase_of(i), a);
            __syncwarp();
        } else if (warp == 5 && n > 0) {
            // ---------------------------------------------------- products
            const bool leader = elect_one();
            constexpr uint32_t idesc_qk = idesc_bf16_f32(kTileM, kTileN, 0, 0);
            constexpr uint32_t idesc_pv = idesc_bf16_f32(kTileM, kHeadDim, 0, 1);
            const uint64_t dq = smem_desc_sw128(smem_u32(sm.q), 16, 1024);
            const uint64_t dk = smem_desc_sw128(smem_u32(sm.kv[0]), 16, 1024);
            const uint64_t dv = smem_desc_sw128(smem_u32(sm.kv[0]), 0, 1024);
            auto wait_all = [&](uint64_t* bar, uint32_t parity) {
                return (bool)__all_sync(0xffffffffu, wait_phase(smem_u32(bar), parity, abort_flag, a));
            };
            auto commit = [&](uint64_t* bar) {
                if (leader) mma_commit(smem_u32(bar));
            };
            // S = Q K^T, four K16 steps 32 bytes apart in the swizzled rows.
            auto issue_s = [&](int slot) {
                const uint64_t db = dk + (uint64_t)(slot * (kTileBytes >> 4));
                if (leader) {
                    mma_ss(tmem + kColS, dq, db, idesc_qk, 0u);
                    mma_ss(tmem + kColS, dq + 2, db + 2, idesc_qk, 1u);
                    mma_ss(tmem + kColS, dq + 4, db + 4, idesc_qk, 1u);
                    mma_ss(tmem + kColS, dq + 6, db + 6, idesc_qk, 1u);
                }
            };
            // O += P V: V is MN-major, 16 keys = two 8-row atoms = 2048 bytes a step.
            auto issue_pv = [&](int slot, bool accumulate) {
                const uint64_t db = dv + (uint64_t)(slot * (kTileBytes >> 4));
                if (leader) {
                    mma_ts(tmem + kColO, tmem + kColP, db, idesc_pv, accumulate ? 1u : 0u);
#pragma unroll
                    for (int kk = 1; kk < kTileN / 16; ++kk)
                        mma_ts(tmem + kColO, tmem + kColP + kk * 8, db + (uint64_t)(kk * 128), idesc_pv, 1u);
                }
            };
            bool ok = wait_all(&sm.bar_q, 0) && wait_all(&sm.bar_full[0], 0);
            if (ok) {
                tc_fence_after();
                issue_s(0);
                commit(&sm.bar_s);
                commit(&sm.bar_empty[0]);
            }
            for (int j = 0; j < n && ok; ++j) {
                const int iv = 2 * j + 1, ik = 2 * j + 2;
                if (j + 1 < n) {
                    // S(j+1) as soon as the softmax holds S(j) in registers.
                    ok = wait_all(&sm.bar_full[slot_of(ik)], phase_of(ik)) && wait_all(&sm.bar_sfree, j & 1);
                    if (!ok) break;
                    tc_fence_after();
                    issue_s(slot_of(ik));
                    commit(&sm.bar_s);
                    commit(&sm.bar_empty[slot_of(ik)]);
                }
                ok = wait_all(&sm.bar_full[slot_of(iv)], phase_of(iv));
                if (ok && j == n - 1 && has_tail) {
                    // Value rows past the last visible key: zero, whatever is there.
                    uint4* v = reinterpret_cast<uint4*>(sm.kv[slot_of(iv)]);
                    for (int x = tail * 8 + lane; x < kTileN * 8; x += 32) v[x] = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                ok = ok && wait_all(&sm.bar_p, j & 1);
                if (!ok) break;
                tc_fence_after();
                issue_pv(slot_of(iv), j > 0);
                commit(&sm.bar_pv);
                commit(&sm.bar_empty[slot_of(iv)]);
            }
            // Every product must have finished before tensor memory is freed.
            commit(&sm.bar_drain);
            drain_phase(smem_u32(&sm.bar_drain), 0, a);
            __syncwarp();
        }
    } else {
        regs_inc<kTileRegsSoftmax>();
        // -------------------------------------------------------- softmax
        const int t = threadIdx.x;
        const int row = row0 + t;
        const bool has_row = row < row_end;
        const int tok = has_row ? row / a.group : 0;
        const int token = seq.first + tok, head = kvh * a.group + (has_row ? row - tok * a.group : 0);
        if (n > 0) {
            // Stage Q: the thread's row, 16-byte chunks swizzled by row mod 8.
            uint4 x[8];
            const uint4* src = has_row ? reinterpret_cast<const uint4*>(q_row(a, token, head)) : nullptr;
#pragma unroll
            for (int c = 0; c < 8; ++c) x[c] = src ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
            uint4* dst = reinterpret_cast<uint4*>(sm.q) + t * 8;
#pragma unroll
            for (int c = 0; c < 8; ++c) dst[c ^ (t & 7)] = x[c];
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(smem_u32(&sm.bar_q));
        }
        if (warp < active) {
            const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
            const uint32_t tS = tmem + lane_base + kColS, tO = tmem + lane_base + kColO,
                           tP = tmem + lane_base + kColP;
            const float scale = a.scale;
            const int lim = has_row ? key_limit(a, seq, tok) : kv_end;
            const int lim_min = key_limit(a, seq, row0 / a.group);  // of the tile's first token
            float m_run = -INFINITY, l_run = 0.0f;
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                bool got = wait_phase(smem_u32(&sm.bar_s), j & 1, abort_flag, a);
                if (!__all_sync(0xffffffffu, got)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t r[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, r[c]);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; ++c) reg_fence(r[c]);
                tc_fence_before();
                mbar_arrive(smem_u32(&sm.bar_sfree));

                const int k0 = (j0 + j) * kTileN;
                const bool masked = k0 + kTileN > lim_min;
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (k0 + c * 32 + e >= lim) r[c][e] = __float_as_uint(-INFINITY);
                }
                float mx[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const uint32_t* rr = &r[q >> 1][(q & 1) * 16];
                    mx[q] = __uint_as_float(rr[0]);
#pragma unroll
                    for (int e = 1; e < 15; e += 2)
                        mx[q] = fmax3(mx[q], __uint_as_float(rr[e]), __uint_as_float(rr[e + 1]));
                    mx[q] = fmaxf(mx[q], __uint_as_float(rr[15]));
                }
                const float row_max = fmax3(fmax3(mx[0], mx[1], mx[2]), fmax3(mx[3], mx[4], mx[5]),
                                            fmaxf(mx[6], mx[7]));
                const float m_new = fmaxf(m_run, row_max);
                const bool upd = (m_new - m_run) * scale > kLazyLog2;
                float alpha = 1.0f;
                if (upd) {
                    alpha = ex2_approx((m_run - m_new) * scale);
                    m_run = m_new;
                }
                const float neg = m_run == -INFINITY ? 0.0f : -m_run * scale;
                const float2 scale2 = make_float2(scale, scale), neg2 = make_float2(neg, neg);
                float2 sum[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[q] = make_float2(0.0f, 0.0f);
                uint32_t p[2][32];
                auto exp_tile = [&](auto poly_tag) {
                    constexpr bool kPoly = decltype(poly_tag)::value;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const int pr = e >> 1;
                            const float2 x = ffma2(
                                make_float2(__uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1])), scale2, neg2);
                            float2 pp;
                            if (kPoly && (pr + 1) * kPolyOf16 / 16 > pr * kPolyOf16 / 16)
                                pp = exp2_poly4(x);
                            else
                                pp = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                            sum[pr & 3] = fadd2(sum[pr & 3], pp);
                            p[c >> 1][(c & 1) * 16 + pr] = pack_bf16_rne(pp.x, pp.y);
                        }
                };
                if (masked) exp_tile(std::false_type{});  // may hold -inf
                else exp_tile(std::true_type{});
                const float2 s01 = fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3]));
                l_run = fmaf(l_run, alpha, s01.x + s01.y);
                if (j > 0) {
                    // P(j-1) consumed, O settled.
                    got = wait_phase(smem_u32(&sm.bar_pv), (j - 1) & 1, abort_flag, a);
                    if (!__all_sync(0xffffffffu, got)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                }
                tmem_st32(tP, p[0]);
                tmem_st32(tP + 32, p[1]);
                if (j > 0 && __any_sync(0xffffffffu, upd)) {
                    const float2 a2 = make_float2(alpha, alpha);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tO + c * 32, o);
                        tmem_wait_ld();
                        reg_fence(o);
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 y = fmul2(make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), a2);
                            o[e] = __float_as_uint(y.x);
                            o[e + 1] = __float_as_uint(y.y);
                        }
                        tmem_st32(tO + c * 32, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(smem_u32(&sm.bar_p));
            }
            // ---------------------------------------------------- results
            if (ok && n > 0) {
                const bool got = wait_phase(smem_u32(&sm.bar_pv), (n - 1) & 1, abort_flag, a);
                ok = __all_sync(0xffffffffu, got);
            }
            if (ok) {
                uint32_t o[2][32];
                if (n > 0) {
                    tc_fence_after();
                    tmem_ld32(tO, o[0]);
                    tmem_ld32(tO + 32, o[1]);
                    tmem_wait_ld();
                    reg_fence(o[0]);
                    reg_fence(o[1]);
                }
                const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;
                const float lse2 = l_run > 0.0f ? fmaf(m_run, scale, __log2f(l_run)) : -INFINITY;
                auto val = [&](int col) {
                    return n > 0 ? __uint_as_float(o[col >> 5][col & 31]) * inv : 0.0f;
                };
                if (has_row && a.out_o != nullptr) {
                    const long long at = (long long)split * a.tokens * a.nhead_q + flat_row(a, token, head);
                    a.out_lse[at] = lse2;
                    if (l_run > 0.0f) {
                        float4* dst = reinterpret_cast<float4*>(a.out_o + at * kHeadDim);
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            dst[c] = make_float4(val(4 * c), val(4 * c + 1), val(4 * c + 2), val(4 * c + 3));
                    }
                } else if (has_row) {
                    uint4* dst = reinterpret_cast<uint4*>(o_row(a, token, head));
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint32_t pk[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) pk[e] = pack_bf16_rne(val(8 * c + 2 * e), val(8 * c + 2 * e + 1));
                        dst[c] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                    }
                    if (a.lse != nullptr) *lse_at(a, token, head) = lse2 * kLn2;
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc(tmem, kTileTmemCols);
    }
}

// Final rows from part_n partial results: 16 threads per row, one float4 of
// columns each.  Rows of sequences outside [min_rows, max_rows] belong to
// another launch.
__global__ void __launch_bounds__(256)
fmha_paged_combine(const __grid_constant__ Args a) {
    griddep_wait();
    const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4;
    if (row >= (long long)a.tokens * a.nhead_q) return;
    const int c4 = threadIdx.x & 15;
    const int token = (int)(row / a.nhead_q), head = (int)(row - (long long)token * a.nhead_q);
    if (a.seqstart_q != nullptr) {
        int lo = 0, hi = a.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.seqstart_q[mid] <= token) lo = mid;
            else hi = mid;
        }
        const Sequence s = load_sequence(a, lo);
        const int rows = s.count * a.group;
        if (token < s.first || token >= s.first + s.count || rows < a.min_rows || rows > a.max_rows) return;
    }
    finish_row4(a, token, head, c4 * 4, -INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f), c4 == 0);
}

}  // namespace fmha_paged
