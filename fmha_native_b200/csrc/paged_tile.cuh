// paged_tile.cuh -- attention of many query rows per K/V head over the paged
// cache: prompt chunks, and a whole batch's rows against a shared prefix.
//
// One block owns a tile of 128 rows (tokens x query heads of one K/V head's
// group, so a tile's rows share their keys) and walks the keys in tiles of
// 128; two blocks share an SM, each with its own pipeline, so one block's
// softmax runs under the other's matrix products:
//
//   warps 0-7    softmax   two threads per row (tensor-memory lane = row), 64 of
//                          the tile's columns each; they also stage Q and write O
//   warp  8      loads     K and V tiles by TMA, one box per page (or per 128
//                          keys of a larger page), into a ring of kTileStages
//                          slots; a lane per box
//   warp  9      products  one elected lane issues every tcgen05.mma; before the
//                          last one the warp zeroes the value rows past the last
//                          visible key, so what a page holds there (NaN included)
//                          stays out of O; in tiles that some tokens see in part
//                          it also sets values that are not finite aside, which
//                          the softmax threads add to the rows that see them
//   warps 10-11  idle      complete the warpgroup for setmaxnreg
//
// Tensor memory of a block (256 of 512 columns): S [0,128), O [128,192), P as
// bf16 pairs [192,256).
//
// Softmax: running maximum per row in log2 units with lazy rescaling (O is
// rescaled only when the maximum grew by more than 2^8; P stays below that), on
// which the two threads of a row agree over a named barrier of their two warps.
// P is rounded to nearest bf16 for the second product, which is what the
// tensor pipe takes; the row sum adds the unrounded fp32 values.
//
// What bounds it: per key tile a block runs 16384 exponentials against 2 x
// 128 x 128 x 64 multiply-adds, so the special-function unit (16 per clock)
// would need twice the tensor pipe's time; three of sixteen exponentials
// therefore run as a polynomial on the FMA pipe.  What remains is the chain
// S -> registers -> P -> tensor memory of each tile, which the SM's other block
// hides in part.  Measured: 4 sequences of 2048 tokens, 16 heads over 4 K/V
// heads, no mask, 579 TF/s from pages of 64 keys, 522 of 16 and 434 of 8 (the
// dense kernel: 702); 6 prompt chunks of 513 to 2048 tokens over up to 8191
// keys, 200 us (118 GFLOP); the kernel alone, with cold caches, 205: tensor pipe
// 30 % busy, special functions 52 %, issue slots 52 %.  There one thread per row
// took 3 % longer than two, blocks of 64 keys a tile (three to an SM) 30 to 47 %,
// an arrival per warp instead of per thread at the barriers of S and P 4 to 6 %.
//
// Work split.  A shared prefix has one length, so the host cuts every row
// tile's keys into `splits` equal ranges, a block each, and whatever ends the
// call folds their results (kPlanNone).  Sequences' own keys differ as they
// like, and their lengths are on the device: with fewer (row tile, head) jobs
// than resident blocks, every block works out for itself the ranges that keep
// all of them busy (kPlanHere: 24 sequences of 5 tokens, 24 heads over 4, 200 to
// 3001 keys 17 us, with a list 26); with more, a first kernel writes the list of
// whole tiles, cutting only what is far longer than the rest (kPlanList: the
// prompt chunks take 4 % longer with every block planning for itself).  Jobs of one
// range go to the output, the others through scratch slots that fmha_paged_end
// folds.
#pragma once
#include <climits>
#include <type_traits>

#include "paged_common.cuh"

namespace fmha_paged {

constexpr int kTileM = 128;
constexpr int kTileN = 128;
constexpr int kTileStages = 4;
constexpr int kTileBytes = 128 * kHeadDim * 2;  // 16 KB: Q, K or V tile
constexpr int kTileThreads = 384;
constexpr int kTileWarps = kTileThreads / 32;
constexpr int kSoftmaxWarps = 8, kWarpLoad = 8, kWarpMma = 9;
constexpr int kTileBlocks = 2 * 148;            // resident blocks of the device
constexpr uint32_t kTileTmemCols = 256;
constexpr uint32_t kColS = 0, kColO = 128, kColP = 192;
// setmaxnreg split of the launch's 384 x 80 registers.
constexpr int kTileRegsSoftmax = 96, kTileRegsControl = 48;
static_assert(256 * kTileRegsSoftmax + 128 * kTileRegsControl <= kTileThreads * 80, "register split");
constexpr float kLazyLog2 = 8.0f;
// Key tiles up to which a job is not worth cutting where jobs abound (prompt chunks
// take 11 % longer with no job cut, however long; as long with 8).
constexpr int kLongRange = 16;
constexpr int kMostParts = 64;  // ranges of a job (their fold is one block's work per 16 rows)
// Pairs of every 16 whose exponential runs on the FMA pipe, by a polynomial as
// exact as the function unit (degree 5), since the row sums and the LSE take it
// in fp32.  Prompt chunks: 200 us; 5 % longer with 0, 1 % with 2, 4 % with 4 (a
// polynomial of degree 3, whose 7.5e-5 show in the LSE: 1 % shorter with 4).
constexpr int kPolyOf16 = 3;

// A block's work (for one K/V head): range k of the keys of a row tile.
struct alignas(16) TileItem {
    int b, first, count, keys;    // the sequence
    int row0, row_end;            // the tile's rows
    int kv_end, j0, n;            // keys that any of them sees; the range's key tiles
    int k, parts;                 // which range of how many
    int slot;                     // scratch slot of the job's first range (parts > 1), for head 0; -1: none
};
__device__ __forceinline__ TileItem make_item(const Args& a, int b, const Sequence& s, int m, int k, int parts,
                                              int slot) {
    TileItem it;
    it.b = b, it.first = s.first, it.count = s.count, it.keys = s.keys;
    it.row0 = m * kTileM;
    it.row_end = min(s.count * a.group, it.row0 + kTileM);
    it.kv_end = max(0, key_limit(a, s, (it.row_end - 1) / a.group));
    const int all = (it.kv_end + kTileN - 1) / kTileN;
    const int each = all / parts, more = all - each * parts;
    it.j0 = k * each + min(k, more);
    it.n = each + (k < more);
    it.k = k, it.parts = parts;
    it.slot = slot;
    return it;
}

struct alignas(1024) TileShared {
    uint8_t q[kTileBytes];
    uint8_t kv[kTileStages][kTileBytes];
    uint64_t bar_full[kTileStages];
    uint64_t bar_empty[kTileStages];
    uint64_t bar_s;                   // S written (commit)
    uint64_t bar_sfree;               // S in registers (a thread's arrival per row)
    uint64_t bar_p;                   // P written, O rescaled (likewise)
    uint64_t bar_pv;                  // O += P V done (commit; an arrival for what the warp wrote itself)
    uint64_t bar_drain;
    uint32_t tmem_base;
    int abort_flag;
    // Keys of the range from all_see on are seen by some of the tile's tokens only
    // (`partly`: there are such).  Of their values that are not finite: per column
    // the first key with NaN, +inf and -inf (INT_MAX: none), and whether there is any.
    int all_see;
    bool partly, any_odd;
    int first_odd[3][kHeadDim];
    int scan[kTileWarps];
    long long scan64[kTileWarps];
    TileItem item;
    int2 tile_of[kTileThreads];
    float half_max[2][kTileM], half_sum[2][kTileM];  // between the two threads of a row
    int half_ok[kSoftmaxWarps];
};

// Scratch of the jobs that several blocks share.
constexpr int kMaxTileSlots = 4 * kTileBlocks;
struct TileHeader {
    int first;         // the job: its sequence's first token, the tile's rows
    int row0, rows, h; // row0 .. row0 + rows - 1 of K/V head h
    int parts;         // its ranges, in the slots from this one on, nhead_k apart; 0: no job begins here
    int pad[3];
};
__host__ __device__ constexpr size_t tile_slot_floats() { return (size_t)kTileM * (kHeadDim + 1); }
__device__ __forceinline__ float* tile_slot_o(const Args& a, int slot) {
    return a.slots + (size_t)slot * kTileM * kHeadDim;
}
__device__ __forceinline__ float* tile_slot_lse(const Args& a, int slot) {
    return a.slots + (size_t)a.max_slots * kTileM * kHeadDim + (size_t)slot * kTileM;
}
__device__ __forceinline__ TileHeader* tile_headers(const Args& a) {
    return reinterpret_cast<TileHeader*>(a.slots + (size_t)a.max_slots * tile_slot_floats());
}

// Named barriers of `threads` threads: plain, and with an OR over a predicate.
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("barrier.cta.sync.aligned %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool bar_or(int id, int threads, bool p) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\t"
        "barrier.cta.red.or.aligned.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"(id), "r"(threads), "r"((uint32_t)p) : "memory");
    return r != 0;
}

// Exclusive scan of `mine` over a block of kWarps warps; `total` = the sum.
template <int kWarps, typename T>
__device__ __forceinline__ T block_scan(T mine, T (&warp_sums)[kWarps], T& total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    T incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const T v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    T before = incl - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const T v = warp_sums[w];
        if (w < warp) before += v;
        total += v;
    }
    __syncthreads();  // warp_sums may be used again
    return before;
}

__device__ __forceinline__ int tile_count(const Args& a, const Sequence& s) {
    const int rows = s.count * a.group;
    return rows < a.min_rows || rows > a.max_rows ? 0 : (rows + kTileM - 1) / kTileM;
}
// Key tiles of row tile m, at least one.
__device__ __forceinline__ int key_tiles(const Args& a, const Sequence& s, int m) {
    const int row_end = min(s.count * a.group, (m + 1) * kTileM);
    return max(1, (key_limit(a, s, (row_end - 1) / a.group) + kTileN - 1) / kTileN);
}
__device__ __forceinline__ int parts_of(int n, long long len) {
    return n <= len ? 1 : min((n + (int)len - 1) / (int)len, kMostParts);
}

// No job begins in the slots from `i` on (to be called by `n` threads).
__device__ __forceinline__ void clear_headers(const Args& a, int i, int n) {
    for (; i < a.max_slots; i += n) tile_headers(a)[i].parts = 0;
}

// The plan for fewer jobs (row tile, head) than resident blocks, by every block
// for itself: the shortest range length whose ranges all fit the device at
// once.  All threads; false: no item for this block.  Prefix sums that decrease
// let sequences overlap, and so have more row tiles than the host made room for
// (max_tiles, below kTileBlocks): they are reported, and none is worked on.
static_assert(kTileBlocks <= kTileThreads, "a row tile per thread");
__device__ __forceinline__ bool plan_here(const Args& a, TileShared& sm, int y, TileItem& it) {
    const int tid = threadIdx.x;
    const int me = (int)blockIdx.x * kTileThreads + tid, everyone = (int)gridDim.x * kTileThreads;
    // Row tiles in order, one per thread.
    int tiles, b = 0, m = 0;
    if (a.seqstart_q != nullptr) {
        const int per = (a.batch + kTileThreads - 1) / kTileThreads;
        const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
        long long mine = 0, sum;
        for (int i = b0; i < b1; ++i) mine += tile_count(a, load_sequence(a, i));
        long long at = block_scan(mine, sm.scan64, sum);
        if (sum > a.max_tiles) {
            flag_index_error(a.err_word);
            clear_headers(a, me, everyone);
            return false;
        }
        tiles = (int)sum;
        for (int i = b0; i < b1 && mine > 0; ++i) {
            const int c = tile_count(a, load_sequence(a, i));
            for (int k = 0; k < c; ++k, ++at) sm.tile_of[at] = make_int2(i, k);
        }
        __syncthreads();
        if (tid < tiles) b = sm.tile_of[tid].x, m = sm.tile_of[tid].y;
    } else {
        const int per_seq = (a.seqlen_q * a.group + kTileM - 1) / kTileM;
        tiles = a.batch * per_seq;
        b = tid / per_seq;
        m = tid - b * per_seq;
    }
    Sequence s{0, 0, 0};
    int n = 0;
    if (tid < tiles) {
        s = load_sequence(a, b);
        n = key_tiles(a, s, m);
    }
    long long total;
    block_scan((long long)n, sm.scan64, total);
    // The shortest length that may do, or else (jobs round up) one that surely does:
    // all / len + jobs <= kTileBlocks ranges.
    const long long all = total * a.nhead_k;
    const int jobs = tiles * a.nhead_k;
    long long len = (all + kTileBlocks - 1) / kTileBlocks;
    int parts, before, sum;
    for (bool again = false;; again = true) {
        parts = tid < tiles ? parts_of(n, len) : 0;
        // Items in the upper half, those of split jobs in the lower.
        before = block_scan(parts << 16 | (parts > 1 ? parts : 0), sm.scan, sum);
        if (again || (sum >> 16) * a.nhead_k <= kTileBlocks) break;
        len = (all + kTileBlocks - jobs - 1) / (kTileBlocks - jobs);
    }
    // The slots that stay unused (a range has one at most, and kTileBlocks < max_slots).
    clear_headers(a, (sum & 0xffff) * a.nhead_k + me, everyone);
    const int x = (sum >> 16) - 1 - y;  // tiles of later tokens (the ones with more keys) first
    if (x < 0) return false;
    const int k = x - (before >> 16);
    if (k >= 0 && k < parts) sm.item = make_item(a, b, s, m, k, parts, parts > 1 ? (before & 0xffff) * a.nhead_k : -1);
    __syncthreads();
    it = sm.item;
    return true;
}

// The plan for more jobs than that, once for all blocks: writes the list of
// items and their number, tiles of later tokens first.  Whole tiles, except
// that what is longer than half a resident block's share is cut into such
// lengths.  One block; a.tile_first is scratch for batch + 1 integers.
constexpr int kPlanThreads = 256;
__global__ void __launch_bounds__(kPlanThreads, 1)
fmha_paged_plan(const __grid_constant__ Args a) {
    __shared__ long long scan64[kPlanThreads / 32];
    griddep_launch_dependents();
    const int tid = threadIdx.x;
    const bool packed = a.seqstart_q != nullptr;
    const int per_seq = packed ? 1 : (a.seqlen_q * a.group + kTileM - 1) / kTileM;
    int* first = a.tile_first;
    int tiles = a.batch * per_seq;
    if (packed) {
        const int per = (a.batch + kPlanThreads - 1) / kPlanThreads;
        const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
        long long mine = 0, sum;
        for (int b = b0; b < b1; ++b) mine += tile_count(a, load_sequence(a, b));
        long long at = block_scan(mine, scan64, sum);
        const bool fits = sum <= a.max_tiles;  // else sequences overlap, see plan_here
        if (!fits) flag_index_error(a.err_word);
        tiles = fits ? (int)sum : 0;
        for (int b = b0; b < b1; ++b) {
            first[b] = fits ? (int)at : 0;
            at += tile_count(a, load_sequence(a, b));
        }
        if (tid == 0) first[a.batch] = tiles;
        __syncthreads();
    }
    const int per = (tiles + kPlanThreads - 1) / kPlanThreads;
    const int t0 = min(tiles, tid * per), t1 = min(tiles, t0 + per);
    int b_first = 0, m_first = 0;
    if (packed) {
        int lo = 0, hi = a.batch;  // the last sequence with first <= t0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= t0) lo = mid;
            else hi = mid;
        }
        b_first = lo;
        m_first = t0 - first[lo];
    } else {
        b_first = t0 / per_seq;
        m_first = t0 - b_first * per_seq;
    }
    // f(b, sequence, m) for the thread's row tiles.
    auto each_tile = [&](auto f) {
        int b = b_first, m = m_first, have = -1;
        Sequence s{0, 0, 0};
        for (int t = t0; t < t1; ++t) {
            if (b != have) s = load_sequence(a, have = b);
            f(b, s, m);
            ++m;
            if (packed)
                while (b + 1 < a.batch && first[b + 1] <= t + 1) ++b, m = 0;
            else if (m == per_seq)
                ++b, m = 0;
        }
    };
    long long mine = 0, total;
    each_tile([&](int, const Sequence& s, int m) { mine += key_tiles(a, s, m); });
    block_scan(mine, scan64, total);
    const long long len = max((long long)kLongRange, (total * a.nhead_k + 2 * kTileBlocks - 1) / (2 * kTileBlocks));
    long long both = 0, sum;  // items in the upper half, those of split jobs in the lower
    each_tile([&](int, const Sequence& s, int m) {
        const int p = parts_of(key_tiles(a, s, m), len);
        both += (long long)p << 32 | (p > 1 ? p : 0);
    });
    const long long before = block_scan(both, scan64, sum);
    const int items = (int)(sum >> 32), split = (int)sum;
    int at = (int)(before >> 32), slot = (int)before;
    each_tile([&](int b, const Sequence& s, int m) {
        const int p = parts_of(key_tiles(a, s, m), len);
        for (int k = 0; k < p; ++k, ++at) {
            a.items[items - 1 - at] = make_item(a, b, s, m, k, p, p > 1 ? slot * a.nhead_k : -1);
        }
        if (p > 1) slot += p;
    });
    // A job longer than len has less than 2 n / len ranges, all of them less than
    // 4 * kTileBlocks = max_slots over the heads; and the items are the tiles and
    // less than total / len <= 2 * kTileBlocks / heads more, as the list has room for.
    if (tid == 0) *a.item_count = items;
    clear_headers(a, split * a.nhead_k + tid, kPlanThreads);
}

// Takes the values that are not finite out of rows [lo, hi) of a V tile whose
// first key is k0, and notes the first key with each kind of them (one warp).
// (Loops kept small: unrolled they took registers from the softmax, 3 % of the
// prompt chunks' time.)
__device__ __forceinline__ void set_aside_odd_values(TileShared& sm, int slot, int k0, int lo, int hi) {
    const int lane = threadIdx.x & 31;
    uint4* v = reinterpret_cast<uint4*>(sm.kv[slot]);
    uint32_t probe = 0;
#pragma unroll 1
    for (int x = lo * 8 + lane; x < hi * 8; x += 32) probe = probe_bf16(v[x], probe);
    if (!__any_sync(0xffffffffu, probe != 0)) return;
#pragma unroll 1
    for (int x = lo * 8 + lane; x < hi * 8; x += 32) {
        const int key = x >> 3, col0 = ((x & 7) ^ (key & 7)) * 8;
        const uint16_t* bits = reinterpret_cast<const uint16_t*>(v + x);
#pragma unroll 1
        for (int e = 0; e < 8; ++e)
            if (!is_finite_bf16(bits[e]))
                atomicMin(&sm.first_odd[(bits[e] & 0x7f) != 0 ? 0 : bits[e] >> 15 ? 2 : 1][col0 + e], k0 + key);
        v[x] = finite_bf16(v[x]);
    }
    if (lane == 0) sm.any_odd = true;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

// Adds them to the 32 columns from col0 on, at tensor memory address `at`, of the
// threads' rows, which see the keys before `end`.
__device__ __forceinline__ void add_odd_values(const TileShared& sm, uint32_t at, int col0, int end) {
#pragma unroll 1
    for (int e = 0; e < kHeadDim / 2; ++e) {
        uint32_t r = tmem_ld1(at + e);
        tmem_wait_ld();
        asm volatile("" : "+r"(r));  // used after the wait
        float o = __uint_as_float(r);
        if (sm.first_odd[0][col0 + e] < end) o = NAN;
        if (sm.first_odd[1][col0 + e] < end) o += INFINITY;
        if (sm.first_odd[2][col0 + e] < end) o -= INFINITY;
        tmem_st1(at + e, __float_as_uint(o));
    }
    tmem_wait_st();
}

__global__ void __launch_bounds__(kTileThreads, 2)
fmha_paged_tile_kernel(const __grid_constant__ Args a) {
    extern __shared__ uint8_t smem_raw[];
    TileShared& sm = *reinterpret_cast<TileShared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                    ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &sm.abort_flag;

    // Tensor memory first: the SM's second block does not start before the first
    // has given the permit to allocate back (2-3 us later, if that waits for the
    // block's work to be known).
    if (warp == kWarpMma) {
        tmem_alloc(smem_u32(&sm.tmem_base), kTileTmemCols);
        tmem_relinquish();
    }
    auto leave = [&]() {  // a block without work
        griddep_wait();   // (the grid ends after the launch before it)
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (warp == kWarpMma) tmem_dealloc(sm.tmem_base, kTileTmemCols);
    };
    // Neighbouring blocks take the heads of one key range: they read
    // neighbouring lines of memory at the same time.
    const int kvh = blockIdx.x % a.nhead_k, y = blockIdx.x / a.nhead_k;
    TileItem it;
    if (a.plan == kPlanNone) {
        // One sequence, every tile cut as the host said.
        const int m = y / a.splits;
        it = make_item(a, 0, load_sequence(a, 0), m, y - m * a.splits, a.splits, -1);
    } else if (a.plan == kPlanHere) {
        if (!plan_here(a, sm, y, it)) return leave();
    } else {
        griddep_wait();  // for the list
        if (y >= *a.item_count) return leave();
        it = a.items[y];
    }
    // What follows on the stream may be scheduled as soon as this grid's last
    // blocks run; it waits for their results where it needs them.
    griddep_launch_dependents();

    const Sequence seq{it.first, it.count, it.keys};
    const int row0 = it.row0, row_end = it.row_end, kv_end = it.kv_end, j0 = it.j0, n = it.n;
    const bool shared_job = it.slot >= 0;  // through scratch slots
    const int slot_job = it.slot + it.k * a.nhead_k + kvh;
    if (shared_job && threadIdx.x == 0) {
        if (it.k == 0) tile_headers(a)[slot_job] = TileHeader{seq.first, row0, row_end - row0, kvh, it.parts, {0, 0, 0}};
        else tile_headers(a)[slot_job].parts = 0;
    }
    const int tail = kv_end - (j0 + n - 1) * kTileN;  // visible keys of the range's last tile
    const bool has_tail = n > 0 && tail < kTileN;
    const int active = (row_end - row0 + 31) / 32;    // softmax warps with rows

    // K_j is load 2j, V_j load 2j + 1 of the ring.
    auto slot_of = [](int i) { return i % kTileStages; };
    auto phase_of = [](int i) { return (uint32_t)((i / kTileStages) & 1); };

    // Softmax warps: the thread's row and its half of the columns.
    const int t = threadIdx.x & (kTileM - 1), half = (int)threadIdx.x >> 7;
    const int row = row0 + t;
    const bool has_row = row < row_end;
    const int tok = has_row ? row / a.group : 0;
    const int token = seq.first + tok, head = kvh * a.group + (has_row ? row - tok * a.group : 0);

    // Load warp: box_rows keys of one page per box, lane i loads box i of a tile.
    const uint64_t policy = l2_policy_evict_last();
    const int box_rows = min(1 << a.page_shift, kTileN);
    auto page_of = [&](int j) {
        const int key = (j0 + j) * kTileN + lane * box_rows;
        return lane * box_rows < kTileN && key < kv_end
                   ? __ldg(a.page_table + it.b * a.table_stride + (key >> a.page_shift)) : 0;
    };
    auto issue_load = [&](int i, int page) {
        const int key0 = (j0 + (i >> 1)) * kTileN, slot = slot_of(i);
        const int boxes = (min(kTileN, kv_end - key0) + box_rows - 1) / box_rows;
        const uint32_t bar = smem_u32(&sm.bar_full[slot]);
        if (lane == 0) mbar_arrive_expect_tx(bar, boxes * box_rows * kHeadDim * 2);
        __syncwarp();
        if (lane < boxes) {
            if (page < 0 || page >= a.num_pages) flag_index_error(a.err_word);
            load_page_box(smem_u32(sm.kv[slot]) + lane * box_rows * kHeadDim * 2, (i & 1) ? &a.tm_v : &a.tm_k, bar,
                          (key0 + lane * box_rows) & ((1 << a.page_shift) - 1), kvh + no_page_head(a), page, policy);
        }
    };
    constexpr int kAhead = kTileStages / 2;  // tiles loaded before the block starts
    int page = 0;

    // Start, the roles side by side: barriers and the first copies, and Q (its
    // 16-byte chunks swizzled by row mod 8).
    if (warp == kWarpLoad) {
        page = page_of(0);
        if (lane == 0) {
            for (int s = 0; s < kTileStages; ++s) {
                mbar_init(smem_u32(&sm.bar_full[s]), 1);
                mbar_init(smem_u32(&sm.bar_empty[s]), 1);
            }
            mbar_init(smem_u32(&sm.bar_s), 1);
            mbar_init(smem_u32(&sm.bar_sfree), 64 * active);
            mbar_init(smem_u32(&sm.bar_p), 64 * active);
            mbar_init(smem_u32(&sm.bar_pv), 2);
            mbar_init(smem_u32(&sm.bar_drain), 1);
            sm.abort_flag = 0;
            fence_barrier_init();
        }
        __syncwarp();
        for (int j = 0; j < min(n, kAhead); ++j) {
            const int next = j + 1 < n ? page_of(j + 1) : 0;
            issue_load(2 * j, page);
            issue_load(2 * j + 1, page);
            page = next;
        }
    } else if (warp == kWarpMma) {
        for (int i = lane; i < 3 * kHeadDim; i += 32) sm.first_odd[0][i] = INT_MAX;
        if (lane == 0) {
            sm.any_odd = false;
            sm.all_see = max(0, key_limit(a, seq, row0 / a.group));
            sm.partly = n > 0 && sm.all_see < min(kv_end, (j0 + n) * kTileN);
        }
    } else if (warp < kSoftmaxWarps && n > 0) {
        uint4 x[4];
        const uint4* src = has_row ? reinterpret_cast<const uint4*>(q_row(a, token, head)) + half * 4 : nullptr;
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = src ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
        uint4* dst = reinterpret_cast<uint4*>(sm.q) + t * 8;
#pragma unroll
        for (int c = 0; c < 4; ++c) dst[(half * 4 + c) ^ (t & 7)] = x[c];
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    if (warp >= kSoftmaxWarps) {
        regs_dec<kTileRegsControl>();
        if (warp == kWarpLoad && n > 0) {
            // ---------------------------------------------------- loads
            bool ok = true;
            int issued = 2 * min(n, kAhead);
            for (int j = kAhead; j < n && ok; ++j) {
                const int next = j + 1 < n ? page_of(j + 1) : 0;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int i = 2 * j + v;
                    ok = wait_phase(smem_u32(&sm.bar_empty[slot_of(i)]), phase_of(i) ^ 1, abort_flag, a);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    issue_load(i, page);
                    issued = i + 1;
                }
                page = next;
            }
            if (!ok || *abort_flag)
                for (int i = max(0, issued - kTileStages); i < issued; ++i)
                    drain_phase(smem_u32(&sm.bar_full[slot_of(i)]), phase_of(i), a);
            __syncwarp();
        } else if (warp == kWarpMma && n > 0) {
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
            bool ok = wait_all(&sm.bar_full[0], 0);
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
                if (ok && sm.partly) {
                    const int k0 = (j0 + j) * kTileN;
                    set_aside_odd_values(sm, slot_of(iv), k0, max(0, sm.all_see - k0), min(kTileN, kv_end - k0));
                }
                ok = ok && wait_all(&sm.bar_p, j & 1);
                if (!ok) break;
                tc_fence_after();
                issue_pv(slot_of(iv), j > 0);
                if (leader) mbar_arrive(smem_u32(&sm.bar_pv));
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
        if ((warp & 3) < active) {
            const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t tS = tmem + lane_base + kColS + half * 64, tO = tmem + lane_base + kColO + half * 32,
                           tP = tmem + lane_base + kColP + half * 32;
            const int pair_bar = 1 + (warp & 3);  // named barrier of the warps w and w + 4
            const float scale = a.scale;
            const int lim = (has_row ? key_limit(a, seq, tok) : kv_end) - half * 64;
            const int lim_min = key_limit(a, seq, row0 / a.group);  // of the tile's first token
            float m_run = -INFINITY, l_run = 0.0f;
            bool finite = false;  // every m_run of the warp is
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                bool got = wait_phase(smem_u32(&sm.bar_s), j & 1, abort_flag, a);
                got = __all_sync(0xffffffffu, got);
                if (!got) ok = false;
                tc_fence_after();
                uint32_t r[2][32];
                tmem_ld32(tS, r[0]);
                tmem_ld32(tS + 32, r[1]);
                tmem_wait_ld();
                reg_fence(r[0]);
                reg_fence(r[1]);
                tc_fence_before();
                mbar_arrive(smem_u32(&sm.bar_sfree));

                const int k0 = (j0 + j) * kTileN;
                const bool masked = k0 + kTileN > lim_min;
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (k0 + c * 32 + e >= lim) r[c][e] = __float_as_uint(-INFINITY);
                }
                float mx[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t* rr = &r[q >> 1][(q & 1) * 16];
                    mx[q] = __uint_as_float(rr[0]);
#pragma unroll
                    for (int e = 1; e < 15; e += 2)
                        mx[q] = fmax3_nan(mx[q], __uint_as_float(rr[e]), __uint_as_float(rr[e + 1]));
                    mx[q] = fmax_nan(mx[q], __uint_as_float(rr[15]));
                }
                const float half_max = fmax3_nan(mx[0], mx[1], fmax_nan(mx[2], mx[3]));
                // Does either half of any of the 32 rows outgrow the reference (or
                // did either warp give up)?  Seldom after the first tile.  NaN does
                // (and, to no effect, a row that has seen no key yet).
                const bool grew = !((half_max - m_run) * scale <= kLazyLog2);
                float alpha = 1.0f;
                bool any = bar_or(pair_bar, 64, grew || !ok);
                if (any) {
                    sm.half_max[half][t] = half_max;
                    if (lane == 0) sm.half_ok[warp] = ok;
                    bar_sync(pair_bar, 64);
                    const float other = sm.half_max[half ^ 1][t];
                    ok = sm.half_ok[warp] && sm.half_ok[warp ^ 4];  // the same for both warps
                    if (!ok) break;
                    const float m_new = fmax_nan(half_max, other);
                    if (m_new != -INFINITY && !((m_new - m_run) * scale <= kLazyLog2)) {
                        alpha = ex2_approx((m_run - m_new) * scale);
                        m_run = m_new;
                    }
                    finite = __all_sync(0xffffffffu, fabsf(m_run) < INFINITY);
                }
                const float neg = m_run == -INFINITY ? 0.0f : -m_run * scale;
                const float2 scale2 = make_float2(scale, scale), neg2 = make_float2(neg, neg);
                float2 sum[2];
                sum[0] = sum[1] = make_float2(0.0f, 0.0f);
                uint32_t p[32];
                auto exp_tile = [&](auto poly_tag) {
                    constexpr bool kPoly = decltype(poly_tag)::value;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const int pr = e >> 1;
                            const float2 x = ffma2(
                                make_float2(__uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1])), scale2, neg2);
                            float2 pp;
                            if (kPoly && (pr + 1) * kPolyOf16 / 16 > pr * kPolyOf16 / 16)
                                pp = exp2_poly2<5>(x);
                            else
                                pp = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                            sum[pr & 1] = fadd2(sum[pr & 1], pp);
                            p[c * 16 + pr] = pack_bf16_rne(pp.x, pp.y);
                        }
                };
                // The polynomial takes no NaN, and -inf as 2^-120: not under a mask, and
                // not where a row's maximum is NaN or infinite.
                if (masked || !finite) exp_tile(std::false_type{});
                else exp_tile(std::true_type{});
                const float2 s01 = fadd2(sum[0], sum[1]);
                l_run = fmaf(l_run, alpha, s01.x + s01.y);
                if (j > 0) {
                    // P(j-1) consumed, O settled.  (Giving up waits for the next
                    // tile's agreement with the row's other warp.)
                    got = wait_phase(smem_u32(&sm.bar_pv), (j - 1) & 1, abort_flag, a);
                    if (!__all_sync(0xffffffffu, got)) ok = false;
                    tc_fence_after();
                }
                tmem_st32(tP, p);
                if (j > 0 && any && __any_sync(0xffffffffu, alpha != 1.0f)) {
                    const float2 a2 = make_float2(alpha, alpha);
                    uint32_t o[32];
                    tmem_ld32(tO, o);
                    tmem_wait_ld();
                    reg_fence(o);
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 y = fmul2(make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), a2);
                        o[e] = __float_as_uint(y.x);
                        o[e + 1] = __float_as_uint(y.y);
                    }
                    tmem_st32(tO, o);
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
            griddep_wait();  // a prefix's results may come from the launch before
            // The row's sum, from both halves.
            sm.half_sum[half][t] = l_run;
            if (bar_or(pair_bar, 64, !ok)) ok = false;
            l_run += sm.half_sum[half ^ 1][t];
            if (ok) {
                uint32_t o[32];
                if (n > 0) {
                    tc_fence_after();
                    if (sm.any_odd) add_odd_values(sm, tO, half * 32, lim + half * 64);
                    tmem_ld32(tO, o);
                    tmem_wait_ld();
                    reg_fence(o);
                }
                const bool none = l_run == 0.0f;  // the row sees no key of the range
                const float inv = 1.0f / l_run;
                const float lse2 = none ? -INFINITY : fmaf(m_run, scale, __log2f(l_run));
                auto val = [&](int col) {
                    return none ? 0.0f : __uint_as_float(o[col]) * inv;
                };
                float* part_o = nullptr;
                float* part_lse = nullptr;
                if (shared_job) {
                    part_o = tile_slot_o(a, slot_job) + t * kHeadDim;
                    part_lse = tile_slot_lse(a, slot_job) + t;
                } else if (a.out_o != nullptr) {
                    const long long at = (long long)it.k * a.tokens * a.nhead_q + flat_row(a, token, head);
                    part_o = a.out_o + at * kHeadDim;
                    part_lse = a.out_lse + at;
                }
                if (has_row && part_o != nullptr) {
                    if (half == 0) *part_lse = lse2;
                    if (!none) {
                        float4* dst = reinterpret_cast<float4*>(part_o) + half * 8;
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            dst[c] = make_float4(val(4 * c), val(4 * c + 1), val(4 * c + 2), val(4 * c + 3));
                    }
                } else if (has_row && a.part_n > 0) {
                    // Under a prefix: its results belong to the row, too.
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        finish_row4(a, token, head, half * 32 + c * 4, lse2, none ? 0.0f : 1.0f,
                                    make_float4(val(4 * c), val(4 * c + 1), val(4 * c + 2), val(4 * c + 3)),
                                    half == 0 && c == 0);
                } else if (has_row) {
                    uint4* dst = reinterpret_cast<uint4*>(o_row(a, token, head)) + half * 4;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t pk[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) pk[e] = pack_bf16_rne(val(8 * c + 2 * e), val(8 * c + 2 * e + 1));
                        dst[c] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                    }
                    if (half == 0 && a.lse != nullptr) *lse_at(a, token, head) = lse2 * kLn2;
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kWarpMma) {
        tc_fence_after();
        tmem_dealloc(tmem, kTileTmemCols);
    }
}

// Folds the ranges of the jobs that several blocks shared into final rows: 16
// rows from row0 on of the jobs that begin in the slots first + i * kCombineBlocks;
// 16 threads per row, four columns each, kBatch ranges in flight.
constexpr int kCombineBlocks = 148;
constexpr int kCombineRows = 16;
__device__ __forceinline__ void combine_ranges(const Args& a, int first, int row0) {
    constexpr int kEach = (kMaxTileSlots + kCombineBlocks - 1) / kCombineBlocks;
    constexpr int kBatch = 8;
    TileHeader head[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int slot = first + i * kCombineBlocks;
        head[i].parts = 0;
        if (slot < a.max_slots) head[i] = tile_headers(a)[slot];
    }
    const int c4 = threadIdx.x & 15, rt = row0 + (int)(threadIdx.x >> 4);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (rt >= head[i].rows || head[i].parts == 0) continue;
        const int slot0 = first + i * kCombineBlocks;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k0 = 0; k0 < head[i].parts; k0 += kBatch) {
            float m2[kBatch];
            float4 x[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                m2[u] = -INFINITY;
                x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (k0 + u < head[i].parts) {
                    const int slot = slot0 + (k0 + u) * a.nhead_k;
                    m2[u] = tile_slot_lse(a, slot)[rt];
                    x[u] = *reinterpret_cast<const float4*>(tile_slot_o(a, slot) + rt * kHeadDim + c4 * 4);
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (m2[u] != -INFINITY) fold4(m, l, o, m2[u], 1.0f, x[u]);  // else O was not written
        }
        const int row = head[i].row0 + rt, t = row / a.group;
        finish_row4(a, head[i].first + t, head[i].h * a.group + row - t * a.group, c4 * 4, m, l, o, c4 == 0);
    }
}

}  // namespace fmha_paged
