// Keys and values of a paged cache by TMA: a tensor map over the pool (head_dim, then heads and rows of a page in the order of
// their strides, then pages), whose boxes are 64 columns of one head of a page's rows; 128-byte swizzle.
#pragma once
#include <algorithm>
#include <numeric>

#include "paged.cuh"
#include "tc_common.cuh"

namespace sanic {
namespace paged {

#ifdef __CUDACC__
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
#endif

// Row-major view of rank 3 or 4, 128-byte swizzle, zero fill out of bounds; strides in elements of 2 bytes, dims innermost first.
static inline int32_t encode_map(sanic_ctx* ctx, CUtensorMap* map, bool bf16, const void* ptr, int rank, const cuuint64_t* dims, const int64_t* strides,
               const cuuint32_t* box) {
    if (!ctx->encode_tiled) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
        if (e != cudaSuccess || !fn) return sanic_fail(ctx, SANIC_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
        ctx->encode_tiled = fn;
    }
    cuuint64_t st[3];
    for (int i = 0; i + 1 < rank; ++i) st[i] = (cuuint64_t)strides[i] * 2;
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUresult r = ((tc::encode_tiled_fn)ctx->encode_tiled)(
        map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(ptr), dims, st, box, ones,
        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return sanic_fail(ctx, SANIC_ERR_CUDA, "attn_paged: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return SANIC_OK;
}

// Strides of a pool as the tensor map wants them: (heads, rows) ordered by stride, every stride a multiple of the one before.
struct Pool { int64_t inner, outer; bool heads_inner; };
static inline bool pool_of(int64_t page, int64_t row, int64_t head, int n_pages, int page_size, int heads, int d, Pool* out) {
    if (heads == 1) head = d;              // a single head's stride is never used
    if (page_size == 1) row = d;
    const bool hi = head <= row;
    const int64_t in = hi ? head : row, o = hi ? row : head;
    if (n_pages == 1) page = o * (hi ? page_size : heads);
    *out = Pool{in, o, hi};
    return in >= d && o % in == 0 && page % o == 0 && page >= o && page < (1ll << 38);
}


// The map of the key pool (kv = 0) or the value pool (1); heads_inner: which of its middle coordinates is the head.
static inline int32_t encode_pool(sanic_ctx* ctx, CUtensorMap* map, bool bf16, const Params& p, int kv, int d, int box_rows, bool* heads_inner) {
    Pool pool;
    const int64_t page = kv ? p.v_page_stride : p.k_page_stride;
    pool_of(page, kv ? p.v_row_stride : p.k_row_stride, kv ? p.v_head_stride : p.k_head_stride, p.n_pages, p.page_size, p.kv_heads, d, &pool);
    const cuuint64_t hd = p.kv_heads, rd = p.page_size;
    const cuuint64_t dims[4] = {(cuuint64_t)d, pool.heads_inner ? hd : rd, pool.heads_inner ? rd : hd, (cuuint64_t)p.n_pages};
    const int64_t strides[3] = {pool.inner, pool.outer, p.n_pages == 1 ? pool.outer * (int64_t)dims[2] : page};
    const cuuint32_t br = box_rows;
    const cuuint32_t box[4] = {64, pool.heads_inner ? 1u : br, pool.heads_inner ? br : 1u, 1};
    *heads_inner = pool.heads_inner;
    return encode_map(ctx, map, bf16, kv ? p.v : p.k, 4, dims, strides, box);
}

// Rows of a box: what divides both the page and the tile, so that a tile is made of whole boxes and none crosses a page's end.
static inline int box_rows_of(int page_size, int tile) { return std::gcd(page_size, tile); }

// Whether the pool can be read in tiles of `tile` keys (64 or 128): pages of a multiple of 8 rows (the swizzle's period, so that every box
// starts on one); strides that nest.
// 2048 tokens over 30,000 keys of 128: 970 us in pages of 16, 96 or 128 rows, 1030 of 48, 1410 of 24 and 1330 of 8 (boxes of 8 rows are
// 1 KB each: their number bounds it), 4410 in pages of 20 (the rows form by 16-byte copies). 64 decodes of 8000 keys in pages of 16,
// 48, 24, 8 and 20: 348, 355, 443, 417, 451 us.
static inline bool pool_supported(const sanic_attn_paged_params* p, int tile) {
    const int ps = p->page_size;
    if (box_rows_of(ps, tile) < 8) return false;
    Pool pool;
    return pool_of(p->k_page_stride, p->k_row_stride, p->k_head_stride, p->n_pages, ps, p->kv_heads, p->head_dim, &pool) &&
           pool_of(p->v_page_stride, p->v_row_stride, p->v_head_stride, p->n_pages, ps, p->kv_heads, p->head_dim, &pool);
}

}  // namespace paged
}  // namespace sanic
