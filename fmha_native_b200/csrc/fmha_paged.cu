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

using namespace fmha_paged;

namespace {

static_assert(sizeof(RowsShared<1>) + 1024 <= 227 * 1024, "shared memory of a block");
static_assert(sizeof(RowsShared<2>) + 1024 <= 227 * 1024, "shared memory of a block");

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

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

// Rows per K/V head that one sequence may have, and the scratch of a call.
struct Sizes {
    long long tokens;
    int group;
    long long max_rows;
    size_t pieces;    // bytes of the rows kernel's scratch
    size_t partials;  // bytes of partial results between launches
    size_t total;
};

bool sizes_of(int batch, int seqlen_q, int total_q, bool packed, int nhead_q, int nhead_k, int prefix_len,
              Sizes& z) {
    if (batch <= 0 || seqlen_q < 0 || total_q < 0 || nhead_q <= 0 || nhead_k <= 0 ||
        nhead_q % nhead_k != 0 || prefix_len < 0)
        return false;
    z.tokens = packed ? total_q : (long long)batch * seqlen_q;
    z.group = nhead_q / nhead_k;
    z.max_rows = (long long)(packed ? std::min(seqlen_q, total_q) : seqlen_q) * z.group;
    if (z.tokens * nhead_q > INT_MAX || z.max_rows > INT_MAX) return false;
    z.pieces = rows_scratch_bytes(32);
    z.partials = prefix_len > 0 ? (size_t)z.tokens * nhead_q * (kHeadDim + 1) * sizeof(float) : 0;
    z.total = z.pieces + z.partials;
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
                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FMHA_OK : FMHA_ERR_ARG;
}

int cache_maps(const fmha_host::Context& ctx, Args& a, const FmhaPagedParams* p, int box_rows) {
    const int box = std::min(p->page_size, box_rows);
    const int st = cache_map(ctx, &a.tm_k, p->k_cache, p, p->stride_k, p->nhead_stride_k, p->page_stride_k, box);
    if (st != FMHA_OK) return st;
    return cache_map(ctx, &a.tm_v, p->v_cache, p, p->stride_v, p->nhead_stride_v, p->page_stride_v, box);
}

int check(const FmhaPagedParams* p, bool prefix, Sizes& z) {
    if (p == nullptr) return FMHA_ERR_ARG;
    const bool packed = p->seqstart_q != nullptr;
    if (!p->q || !p->k_cache || !p->v_cache || !p->o || !p->page_table || !p->seqlens_k) return FMHA_ERR_ARG;
    if (prefix ? (p->prefix_len <= 0 || !p->prefix_pages) : false) return FMHA_ERR_ARG;
    if (!sizes_of(p->batch, p->seqlen_q, p->total_q, packed, p->nhead_q, p->nhead_k,
                  prefix ? p->prefix_len : 0, z))
        return FMHA_ERR_ARG;
    if (!aligned16(p->q) || !aligned16(p->k_cache) || !aligned16(p->v_cache) || !aligned16(p->o))
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
    if (!(p->scale > 0.0f) || p->scale > 1e30f) return FMHA_ERR_ARG;
    if (z.tokens > 0 && (p->workspace == nullptr || !aligned16(p->workspace) ||
                         p->workspace_bytes < (long long)z.total))
        return FMHA_ERR_ARG;
    return FMHA_OK;
}

Args base_args(const FmhaPagedParams* p, const Sizes& z, const fmha_host::Context& ctx) {
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
    a.pieces = static_cast<float*>(p->workspace);
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

// The rows kernel and, as its programmatic dependent, the merge of the jobs
// that cross blocks.
template <int MT>
int launch_rows_mt(Args& a, int max_rows, int device, cudaStream_t stream) {
    constexpr int kRows = 16 * MT;
    constexpr size_t smem = sizeof(RowsShared<MT>) + 1024;
    static std::atomic<unsigned long long> ready{0};
    if (!allow_smem(ready, device, reinterpret_cast<const void*>(fmha_paged_rows_kernel<MT>), smem))
        return FMHA_ERR_LAUNCH;
    a.m_tiles = std::max(1, (max_rows + kRows - 1) / kRows);
    if ((long long)a.batch * a.m_tiles > INT_MAX) return FMHA_ERR_ARG;
    fmha_paged_rows_kernel<MT><<<kMaxRowBlocks, kRowThreadsTotal, smem, stream>>>(a);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kMaxRowBlocks, kRows / 8);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, fmha_paged_rows_merge<MT>, a) != cudaSuccess) return FMHA_ERR_LAUNCH;
    return cudaGetLastError() == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}
int launch_rows(Args& a, int max_rows, int device, cudaStream_t stream) {
    return max_rows <= 16 ? launch_rows_mt<1>(a, max_rows, device, stream)
                          : launch_rows_mt<2>(a, max_rows, device, stream);
}

int run(const FmhaPagedParams* p, bool prefix, cudaStream_t stream) {
    Sizes z;
    int st = check(p, prefix, z);
    if (st != FMHA_OK) return st;
    fmha_host::Context ctx;
    if ((st = fmha_host::acquire(&ctx)) != FMHA_OK) return st;
    if (z.tokens == 0) return FMHA_OK;
    Args a = base_args(p, z, ctx);
    if ((st = cache_maps(ctx, a, p, kUnit)) != FMHA_OK) return st;
    if (prefix) {
        // Every token's rows against the prefix, as one sequence without mask.
        Args b = a;
        b.seqstart_q = nullptr;
        b.seqlens_k = nullptr;
        b.fixed_len = p->prefix_len;
        b.page_table = p->prefix_pages;
        b.table_stride = 0;
        b.max_pages = (p->prefix_len + p->page_size - 1) / p->page_size;
        b.batch = 1;
        b.seqlen_q = a.tokens;
        b.causal = 0;
        b.out_o = reinterpret_cast<float*>(static_cast<uint8_t*>(p->workspace) + z.pieces);
        b.out_lse = b.out_o + (size_t)a.tokens * a.nhead_q * kHeadDim;
        const long long rows = (long long)a.tokens * a.group;
        if (rows > INT_MAX) return FMHA_ERR_ARG;
        if ((st = launch_rows(b, (int)rows, ctx.device, stream)) != FMHA_OK) return st;
        a.part_o = b.out_o;
        a.part_lse = b.out_lse;
        a.part_n = 1;
    }
    return launch_rows(a, (int)z.max_rows, ctx.device, stream);
}

}  // namespace

extern "C" {

size_t fmha_paged_workspace_bytes(int batch, int seqlen_q, int total_q, int nhead_q, int nhead_k,
                                  int prefix_len) {
    Sizes z;
    if (!sizes_of(batch, seqlen_q, total_q, total_q > 0, nhead_q, nhead_k, prefix_len, z)) return 0;
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
