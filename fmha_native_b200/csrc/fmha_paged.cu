// fmha_paged.cu -- launchers of the attention over the paged K/V cache and of
// the shared-prefix attention declared in include/fmha_paged.h.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>
#include <cstring>

#include "../../include/fmha_paged.h"
#include "host_context.h"
#include "paged_common.cuh"
#include "paged_rows.cuh"
#include "paged_tile.cuh"

using namespace fmha_paged;

// The end of a call: the merge of the sequences that cross the rows kernel's
// blocks, by the first end_merge blocks, and the fold of the key ranges that
// the tile kernel's blocks shared, by the others.  One kernel for both saves a
// launch (50 sequences of 3 to 12 tokens: 20.2 -> 19.5 us); where there is only
// the merge, the fold's registers would cost more (64 sequences of 100 to 4095
// keys: 3 % longer with it).
constexpr int kEndThreads = 256;
template <bool kMerge, bool kCombine>
__global__ void __launch_bounds__(kEndThreads)
fmha_paged_end(const __grid_constant__ Args a) {
    griddep_wait();
    const int x = blockIdx.x;
    if (kMerge && (!kCombine || x < a.end_merge)) {
        merge_pieces(a, x % kMaxRowBlocks, x / kMaxRowBlocks, a.end_merge / kMaxRowBlocks);
    } else if (kCombine) {
        const int y = x - (kMerge ? a.end_merge : 0);
        combine_ranges(a, y % kCombineBlocks, y / kCombineBlocks * kCombineRows);
    }
}

namespace {

static_assert(sizeof(RowsShared) + 1024 <= 227 * 1024, "shared memory of a block");
static_assert(2 * (sizeof(TileShared) + 2048) <= 228 * 1024, "two tile blocks per SM");

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// A stride of a dimension of one element is never used.
bool stride_ok(long long s, long long extent) {
    if (extent <= 1) return true;
    return s > 0 && s % 8 == 0 && s < (1ll << 39);
}
bool in_stride_ok(long long s, long long extent) { return s == 0 || stride_ok(s, extent); }

int log2_exact(int v) {
    for (int s = 0; s < 31; ++s)
        if ((1 << s) == v) return s;
    return -1;
}

// Sequences with at most kMostRows rows per K/V head (tokens x group) go to the
// rows kernel, the others to the tile kernel.  The launches of a call and its
// scratch, from sizes that the host has.
struct Plan {
    long long tokens;
    int group;
    int max_rows;             // rows per K/V head that one sequence may have
    bool rows, tile;          // which kernels serve the sequences' own keys
    int row_cap;              // max_rows for the rows kernel's sequences
    long long tiles;          // row tiles of the tile kernel (at most)
    int plan;                 // how its key ranges are found
    long long ranges;         // and how many they are at most
    long long prefix_tiles;   // row tiles against the prefix, and their key ranges
    int prefix_splits;
    // Bytes: the two kernels' scratch, the list of work; under a prefix, what the
    // rows kernel says of the sequences, and one partial result of all rows.
    size_t pieces, slots, list, info, part;
    int parts;                // partial results: the prefix's, then the rows kernel's
    size_t total;
};

// Key ranges per row tile where the number of key tiles is known, by the time
// (in 0.05 us, as measured) of the waves of blocks and of the final fold: a
// block starts and ends in 5.5 us, takes 0.9 us per key tile alone on its SM and
// 1.45 beside another one, and every range adds 0.35 us to the fold.
int pick_splits(long long jobs, long long tiles) {
    const long long most = std::min({(long long)16, tiles, std::max(1ll, 4ll * kTileBlocks / jobs)});
    int best = 1;
    long long cost = LLONG_MAX;
    for (int s = 1; s <= most; ++s) {
        const long long waves = (jobs * s + kTileBlocks - 1) / kTileBlocks;
        const long long per_tile = jobs * s <= kTileBlocks / 2 ? 18 : 29;
        const long long c = waves * ((tiles + s - 1) / s * per_tile + 110) + 7 * s;
        if (c < cost) cost = c, best = s;
    }
    return best;
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

bool make_plan(int batch, int seqlen_q, int total_q, bool packed, int nhead_q, int nhead_k, int prefix_len,
               Plan& z) {
    memset(&z, 0, sizeof(z));
    if (batch <= 0 || seqlen_q < 0 || total_q < 0 || nhead_q <= 0 || nhead_k <= 0 ||
        nhead_q % nhead_k != 0 || prefix_len < 0)
        return false;
    z.tokens = packed ? total_q : (long long)batch * seqlen_q;
    z.group = nhead_q / nhead_k;
    const long long max_rows = (long long)(packed ? std::min(seqlen_q, total_q) : seqlen_q) * z.group;
    if (z.tokens * nhead_q > INT_MAX || nhead_q > 8192 || prefix_len > kMostKeys || (z.tokens > 0 && max_rows == 0)) return false;
    z.max_rows = (int)max_rows;
    z.tile = max_rows > kMostRows;
    z.rows = packed || !z.tile;
    if (z.rows) {
        z.row_cap = (int)std::min<long long>(max_rows, kMostRows);
        z.pieces = round16(rows_scratch_bytes((long long)z.row_cap * nhead_k));
    }
    if (z.tile) {
        const long long all = z.tokens * z.group;
        z.tiles = packed ? all / kTileM + std::min<long long>(batch, all / (kMostRows + 1))
                         : (max_rows + kTileM - 1) / kTileM * batch;
        if ((z.tiles + 2 * kTileBlocks) * nhead_k > INT_MAX) return false;
        // A range per resident block, or per row tile and two per resident block.
        const long long resident = (kTileBlocks + nhead_k - 1) / nhead_k;
        z.plan = z.tiles * nhead_k < kTileBlocks ? kPlanHere : kPlanList;
        z.ranges = z.plan == kPlanHere ? resident : z.tiles + 2 * resident;
        z.slots = round16(kMaxTileSlots * (tile_slot_floats() * sizeof(float) + sizeof(TileHeader)));
        if (z.plan == kPlanList) z.list = round16(z.ranges * sizeof(TileItem) + (batch + 2) * sizeof(int));
    }
    if (prefix_len > 0) {
        z.prefix_tiles = (z.tokens * z.group + kTileM - 1) / kTileM;
        z.prefix_splits = pick_splits(std::max(1ll, z.prefix_tiles * nhead_k), (prefix_len + kTileN - 1) / kTileN);
        z.part = (size_t)z.tokens * nhead_q * (kHeadDim + 1) * sizeof(float);
        z.parts = z.prefix_splits + (z.rows ? 1 : 0);
        z.info = round16((long long)batch * sizeof(int2));
    }
    z.total = z.pieces + z.slots + z.list + z.info + z.part * z.parts;
    return true;
}

// Tensor map over a cache seen as (64, token in page, head, page).
int cache_map(const fmha_host::Context& ctx, CUtensorMap* tm, const uint16_t* base, const FmhaPagedParams* p,
              long long token, long long head, long long page, int box_rows) {
    cuuint64_t dims[4] = {(cuuint64_t)kHeadDim, (cuuint64_t)p->page_size, (cuuint64_t)p->nhead_k,
                          (cuuint64_t)std::max(1, p->num_pages)};
    if (p->nhead_k == 1) head = 8;
    if (p->num_pages <= 1) page = 8;
    cuuint64_t strides[3] = {(cuuint64_t)token * 2, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
    cuuint32_t box[4] = {(cuuint32_t)kHeadDim, (cuuint32_t)box_rows, 1, 1};
    cuuint32_t one[4] = {1, 1, 1, 1};
    const CUresult r = ctx.encode(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<uint16_t*>(base), dims,
                                  strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FMHA_OK : FMHA_ERR_ARG;
}

int cache_maps(const fmha_host::Context& ctx, Args& a, const FmhaPagedParams* p, int box_rows) {
    const int box = std::min(p->page_size, box_rows);
    const int st = cache_map(ctx, &a.tm_k, p->k_cache, p, p->stride_k, p->nhead_stride_k, p->page_stride_k, box);
    if (st != FMHA_OK) return st;
    return cache_map(ctx, &a.tm_v, p->v_cache, p, p->stride_v, p->nhead_stride_v, p->page_stride_v, box);
}

int check(const FmhaPagedParams* p, bool prefix, Plan& z) {
    if (p == nullptr) return FMHA_ERR_ARG;
    const bool packed = p->seqstart_q != nullptr;
    if (!p->q || !p->k_cache || !p->v_cache || !p->o || !p->page_table || !p->seqlens_k) return FMHA_ERR_ARG;
    if (prefix ? (p->prefix_len <= 0 || !p->prefix_pages) : false) return FMHA_ERR_ARG;
    if (!make_plan(p->batch, p->seqlen_q, p->total_q, packed, p->nhead_q, p->nhead_k,
                  prefix ? p->prefix_len : 0, z))
        return FMHA_ERR_ARG;
    if (!aligned16(p->q) || !aligned16(p->k_cache) || !aligned16(p->v_cache) || !aligned16(p->o))
        return FMHA_ERR_ARG;
    if (!aligned4(p->lse) || !aligned4(p->page_table) || !aligned4(p->seqlens_k) || !aligned4(p->seqstart_q) ||
        !aligned4(p->prefix_pages))
        return FMHA_ERR_ARG;
    const int shift = log2_exact(p->page_size);
    if (shift < 3 || shift > 12 || p->num_pages < 0 || p->max_pages < 0 || p->table_stride < 0)
        return FMHA_ERR_ARG;
    const long long rows = packed ? p->total_q : p->seqlen_q, batch = packed ? 1 : p->batch;
    if (!in_stride_ok(p->stride_q, rows) || !in_stride_ok(p->nhead_stride_q, p->nhead_q) ||
        !in_stride_ok(p->batch_stride_q, batch) || !stride_ok(p->stride_o, rows) ||
        !stride_ok(p->nhead_stride_o, p->nhead_q) || !stride_ok(p->batch_stride_o, batch))
        return FMHA_ERR_ARG;
    if (!stride_ok(p->stride_k, p->page_size) || !stride_ok(p->nhead_stride_k, p->nhead_k) ||
        !stride_ok(p->page_stride_k, p->num_pages) || !stride_ok(p->stride_v, p->page_size) ||
        !stride_ok(p->nhead_stride_v, p->nhead_k) || !stride_ok(p->page_stride_v, p->num_pages))
        return FMHA_ERR_ARG;
    // Units of 32 keys over the whole batch are counted in 31 bits.
    if ((long long)p->batch * (((long long)p->max_pages << shift) / kUnit + 1 + kSeqCost) > INT_MAX) return FMHA_ERR_ARG;
    if (!(p->scale > 0.0f) || p->scale > 1e30f) return FMHA_ERR_ARG;
    if (z.tokens > 0 && (p->workspace == nullptr || !aligned16(p->workspace) ||
                         p->workspace_bytes < (long long)z.total))
        return FMHA_ERR_ARG;
    return FMHA_OK;
}

Args base_args(const FmhaPagedParams* p, const Plan& z, const fmha_host::Context& ctx) {
    Args a;
    memset(&a, 0, sizeof(a));
    const bool packed = p->seqstart_q != nullptr;
    a.q = p->q;
    a.o = p->o;
    a.lse = p->lse;
    a.page_table = p->page_table;
    a.seqlens_k = p->seqlens_k;
    a.seqstart_q = p->seqstart_q;
    a.table_stride = p->table_stride;
    a.stride_q = p->stride_q, a.nhead_stride_q = p->nhead_stride_q, a.batch_stride_q = p->batch_stride_q;
    a.stride_o = p->stride_o, a.nhead_stride_o = p->nhead_stride_o, a.batch_stride_o = p->batch_stride_o;
    a.batch = p->batch;
    a.seqlen_q = p->seqlen_q;
    a.tokens = (int)z.tokens;
    a.nhead_q = p->nhead_q, a.nhead_k = p->nhead_k, a.group = z.group;
    a.page_shift = log2_exact(p->page_size);
    a.num_pages = p->num_pages, a.max_pages = p->max_pages;
    a.causal = p->causal != 0;
    a.row_div = packed ? INT_MAX : std::max(1, p->seqlen_q);
    a.lse_len = packed ? p->total_q : p->seqlen_q;
    a.scale = p->scale;
    a.min_rows = 1, a.max_rows = INT_MAX;
    a.err_word = ctx.err_word;
    a.wait_limit_ns = ctx.wait_limit_ns;
    return a;
}

// Once per kernel and device (bit `device` of `ready`): its shared memory.
bool allow_smem(std::atomic<unsigned long long>& ready, int device, const void* kernel, size_t bytes) {
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (bit & ready.load(std::memory_order_acquire)) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
        return false;
    ready.fetch_or(bit, std::memory_order_release);
    return true;
}

// A launch that may start while the one before it on the stream still runs.
template <typename Kernel>
int launch_dependent(Kernel kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}

// after: it follows another kernel of the call.
int launch_rows(const Args& a, bool after, int device, cudaStream_t stream) {
    constexpr size_t smem = sizeof(RowsShared) + 1024;
    static std::atomic<unsigned long long> ready{0};
    if (!allow_smem(ready, device, reinterpret_cast<const void*>(fmha_paged_rows_kernel), smem))
        return FMHA_ERR_LAUNCH;
    if (after) return launch_dependent(fmha_paged_rows_kernel, dim3(kMaxRowBlocks), kRowThreadsTotal, smem, stream, a);
    fmha_paged_rows_kernel<<<kMaxRowBlocks, kRowThreadsTotal, smem, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}

// `ranges`: key ranges of row tiles; after: it follows another kernel of the call.
int launch_tile(const Args& a, long long ranges, bool after, int device, cudaStream_t stream) {
    constexpr size_t smem = sizeof(TileShared) + 1024;
    static std::atomic<unsigned long long> ready{0};
    if (!allow_smem(ready, device, reinterpret_cast<const void*>(fmha_paged_tile_kernel), smem))
        return FMHA_ERR_LAUNCH;
    const dim3 grid((unsigned)(ranges * a.nhead_k));
    if (after) return launch_dependent(fmha_paged_tile_kernel, grid, kTileThreads, smem, stream, a);
    fmha_paged_tile_kernel<<<grid, kTileThreads, smem, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}

int run(const FmhaPagedParams* p, bool prefix, cudaStream_t stream) {
    Plan z;
    int st = check(p, prefix, z);
    if (st != FMHA_OK) return st;
    fmha_host::Context ctx;
    if ((st = fmha_host::acquire(&ctx)) != FMHA_OK) return st;
    if (z.tokens == 0) return FMHA_OK;
    Args a = base_args(p, z, ctx);
    uint8_t* scratch = static_cast<uint8_t*>(p->workspace);
    a.pieces = reinterpret_cast<float*>(scratch);
    a.slots = reinterpret_cast<float*>(scratch + z.pieces);
    const size_t part_rows = (size_t)z.tokens * p->nhead_q;
    uint8_t* list = scratch + z.pieces + z.slots;
    int2* info = reinterpret_cast<int2*>(list + z.list);
    float* part_o = reinterpret_cast<float*>(list + z.list + z.info);
    float* part_lse = part_o + part_rows * kHeadDim * z.parts;
    if (z.tile || prefix) {
        Args t = a;
        if ((st = cache_maps(ctx, t, p, kTileN)) != FMHA_OK) return st;
        t.min_rows = kMostRows + 1;
        t.max_slots = kMaxTileSlots;
        t.max_tiles = (int)z.tiles;
        if (z.tile && z.plan == kPlanList) {
            t.items = reinterpret_cast<TileItem*>(list);
            t.item_count = reinterpret_cast<int*>(t.items + z.ranges);
            t.tile_first = t.item_count + 1;
            fmha_paged_plan<<<1, kPlanThreads, 0, stream>>>(t);
            if (cudaGetLastError() != cudaSuccess) return FMHA_ERR_LAUNCH;
        }
        if (prefix) {
            // Every token's rows against the prefix, as one sequence without mask.
            Args b = t;
            b.seqstart_q = nullptr;
            b.seqlens_k = nullptr;
            b.fixed_len = p->prefix_len;
            b.page_table = p->prefix_pages;
            b.batch = 1;
            b.seqlen_q = a.tokens;
            b.causal = 0;
            b.min_rows = 1;
            b.splits = z.prefix_splits;
            b.out_o = part_o;
            b.out_lse = part_lse;
            st = launch_tile(b, z.prefix_tiles * z.prefix_splits, false, ctx.device, stream);
            if (st != FMHA_OK) return st;
            a.part_o = t.part_o = part_o;
            a.part_lse = t.part_lse = part_lse;
            t.part_n = z.prefix_splits;
        }
        if (z.tile) {
            t.plan = z.plan;
            st = launch_tile(t, z.ranges, z.plan == kPlanList || prefix, ctx.device, stream);
            if (st != FMHA_OK) return st;
        }
    }
    if (z.rows) {
        a.row_cap = z.row_cap;
        const int groups = head_groups(p->nhead_k, z.row_cap);
        a.group_blocks = kMaxRowBlocks / groups;
        a.group_heads = p->nhead_k / groups;
        Args r = a;
        if (z.tile) r.max_rows = kMostRows;
        if ((st = cache_maps(ctx, r, p, kUnit)) != FMHA_OK) return st;
        if (prefix) {
            r.part_n = z.prefix_splits;
            r.seq_parts = info;
            r.out_o = part_o + part_rows * kHeadDim * z.prefix_splits;
            r.out_lse = part_lse + part_rows * z.prefix_splits;
        }
        if ((st = launch_rows(r, z.tile || prefix, ctx.device, stream)) != FMHA_OK) return st;
        if (prefix) {
            const long long threads = part_rows * 16;
            st = launch_dependent(fmha_prefix_finish, dim3((unsigned)((threads + 255) / 256)), 256, 0, stream, r);
            if (st != FMHA_OK) return st;
        }
    }
    unsigned blocks = 0;
    if (z.rows && !prefix) {
        a.end_merge = kMaxRowBlocks * std::min(kMergeBlocks, (a.group_heads * z.row_cap + 3) / 4);
        blocks += a.end_merge;
    }
    if (z.tile) {
        a.max_slots = kMaxTileSlots;
        a.part_n = z.prefix_splits;
        blocks += kCombineBlocks * ((std::min(z.max_rows, kTileM) + kCombineRows - 1) / kCombineRows);
    }
    if (blocks > 0) {
        const auto end = !z.tile ? fmha_paged_end<true, false>
                         : a.end_merge ? fmha_paged_end<true, true> : fmha_paged_end<false, true>;
        st = launch_dependent(end, dim3(blocks), kEndThreads, 0, stream, a);
    }
    return st;
}

}  // namespace

extern "C" {

size_t fmha_paged_workspace_bytes(int batch, int seqlen_q, int total_q, int nhead_q, int nhead_k,
                                  int prefix_len) {
    Plan z;
    if (!make_plan(batch, seqlen_q, total_q, total_q > 0, nhead_q, nhead_k, prefix_len, z)) return 0;
    return z.total;
}

int fmha_paged_fwd_d64_bf16(const FmhaPagedParams* params, CUstream_st* stream) try {
    return run(params, false, stream);
} catch (...) {
    return FMHA_ERR_LAUNCH;
}

int fmha_prefix_fwd_d64_bf16(const FmhaPagedParams* params, CUstream_st* stream) try {
    return run(params, true, stream);
} catch (...) {
    return FMHA_ERR_LAUNCH;
}

}  // extern "C"
