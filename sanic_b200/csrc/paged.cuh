// Attention of ragged chunks over a paged cache: what its two kernels (paged_attn.cu, paged_attn_tc.cu) share. The lengths
// live on the device: every CTA finds its own range of the work (paged_sched.h) from them.
#pragma once
#include "common.cuh"
#include "paged_sched.h"

namespace sanic {
namespace paged {

constexpr int STATUS_POOL = 53;     // page_table_append: free list, table row or token rows exhausted, or a negative length
constexpr int STATUS_ATTN = 54;     // attn_paged: a page or a length out of range
constexpr int STATUS_VERIFY = 55;   // draft_verify: a token, draft length or target row out of range
constexpr int STATUS_WRITE = 56;    // paged_cache_write: a slot or position out of range
constexpr int MAX_REQUESTS = 8000;  // prefix sums over the requests are held in shared memory

// What both kernels need of sanic_attn_paged_params, plus the split of the rows and of the workspace.
struct Params : Shape {
    const void* q; void* out; float* lse; const void* k; const void* v;
    const int32_t* table; const int32_t* query_start; const int32_t* kv_lens;
    int64_t q_token_stride, q_head_stride, k_page_stride, k_row_stride, k_head_stride, v_page_stride, v_row_stride, v_head_stride,
        table_stride;
    int n_tokens, q_heads, group, page_size, page_shift, n_pages, max_pages;
    float scale;
    int rows;              // rows of a partial slot (at least block_tokens * group)
    int rows_above, rows_upto;   // requests of this launch: those whose chunk has more and at most this many query rows
    int beside;            // 1: this launch may start before the one before it (the other class of requests) has ended, and waits for it at
                           // its end. Each needs most of an SM (196 KB of shared memory for the rows form's CTAs, 226 for the other's), so
                           // the two follow one another on every SM; what is saved is the gap between launches.
    // workspace: float [2 * ctas][rows][head_dim], float2 (max in log2 units, sum) [2 * ctas][rows], one int4 per CTA: the item
    // that starts in its range and is shared with the next CTAs (first token row, tokens, kv head, CTAs that hold a part; 0: none)
    float* ws_o; float2* ws_ml; int4* ws_merge;
};

#ifdef __CUDACC__
// Lengths come from the device and are never trusted beyond what the host vouched for: token rows inside [0, n_tokens],
// keys inside the table's row.
struct LoadReq {
    const Params* p;
    int* err;              // null: do not report
    __device__ __forceinline__ Req operator()(int b) const {
        const int s = __ldcg(p->query_start + b), e = __ldcg(p->query_start + b + 1), kv = __ldcg(p->kv_lens + b);
        Req r;
        r.q0 = min(max(s, 0), p->n_tokens);
        r.qn = min(max(e, r.q0), p->n_tokens) - r.q0;
        r.kv = (int)min((long long)max(kv, 0), (long long)p->max_pages * p->page_size);
        const long long rows = (long long)r.qn * p->group;
        if ((r.q0 != s || r.q0 + r.qn != e || r.kv != kv) && err) atomicCAS(err, 0, STATUS_ATTN);
        if (rows <= p->rows_above || rows > p->rows_upto) r.qn = 0;
        return r;
    }
};
template <int KT> using DeviceWalk = Walk<KT, LoadReq>;

// Prefix sums of the requests' costs into cum[0 .. n] (shared memory), by `nt` threads that meet at `sync`.
template <int KT, class Sync>
__device__ __forceinline__ void scan_costs(const Params& p, long long* cum, int* err, int tid, int nt, Sync sync) {
    __shared__ long long warp_sums[32];
    const int lane = tid & 31, warp = tid >> 5;
    const LoadReq load{&p, blockIdx.x == 0 ? err : nullptr};
    long long carry = 0;
    if (tid == 0) cum[0] = 0;
    for (int b0 = 0; b0 < p.n_requests; b0 += nt) {
        const int b = b0 + tid;
        long long c = b < p.n_requests ? request_cost<KT>(p, load(b)) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, c, o); if (lane >= o) c += x; }
        if (lane == 31) warp_sums[warp] = c;
        sync();
        long long before = carry, all = 0;
        for (int w = 0; w < nt / 32; ++w) { const long long x = warp_sums[w]; if (w < warp) before += x; all += x; }
        if (b < p.n_requests) cum[b + 1] = before + c;
        carry += all;
        sync();
    }
    sync();
}

template <int KT>
__device__ __forceinline__ void scan_costs(const Params& p, long long* cum, int* err) {
    scan_costs<KT>(p, cum, err, threadIdx.x, blockDim.x, [] { __syncthreads(); });
}

// The page and row of a key, and whether the page is one of the pool's. A table entry outside the pool reads as zeros and is
// reported; nothing is ever read through it.
__device__ __forceinline__ bool locate(const Params& p, const int32_t* row, int key, int& page, int& in_page, int* err) {
    const int idx = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
    in_page = key - idx * p.page_size;
    page = __ldcg(row + idx);
    if ((unsigned)page < (unsigned)p.n_pages) return true;
    if (err) atomicCAS(err, 0, STATUS_ATTN);
    return false;
}

// A key that only some rows of an item see has weight 0 in the others' product with the values, and 0 times an infinity or a NaN is NaN.
// Rows that came out NaN for it are folded again (paged_attn.cu), one row over the keys [k0, k1) that it sees by a warp: a key per lane
// for the scores, then four columns per lane for the values. Some 0.5 ms for 30,000 keys, and only where values are not finite. Leaves the row's maximum (log2 units), its sum of weights 2^(s - m + shift) and this lane's columns col .. col + 3;
// false, and no sum, where every column is NaN before the end: so they stay.
template <bool BF16> __device__ __forceinline__ void widen2(uint32_t w, float& lo, float& hi) {
    if (BF16) { lo = bf16lo(w); hi = bf16hi(w); }
    else asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(lo), "=f"(hi) : "r"(w));
}
template <int D, bool BF16>
__device__ __forceinline__ bool fold_row(const Params& p, int b, int hk, const uint16_t* q, int k0, int k1, float shift, int col, float& m, float& l, float (&acc)[4]) {
    const int lane = threadIdx.x & 31;
    const float sl2 = p.scale * LOG2E;
    m = -INFINITY; l = 0.0f;
    acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
    for (int at = k0; at < k1; at += 32) {
        const int key = at + lane;
        float s = -INFINITY;
        long long off = -1;                          // of the key's value row; none for a bad page: key and value are zeros
        if (key < k1) {
            int page, in_page;
            s = 0.0f;
            if (locate(p, p.table + (int64_t)b * p.table_stride, key, page, in_page, nullptr)) {
                off = page * p.v_page_stride + in_page * p.v_row_stride + hk * p.v_head_stride;
                const uint16_t* k = (const uint16_t*)p.k + page * p.k_page_stride + in_page * p.k_row_stride + hk * p.k_head_stride;
#pragma unroll 2
                for (int c = 0; c < D; c += 8) {
                    const uint4 x = *(const uint4*)(k + c), y = *(const uint4*)(q + c);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x0, x1, y0, y1;
                        widen2<BF16>(xs[i], x0, x1); widen2<BF16>(ys[i], y0, y1);
                        s = fmaf(x0, y0, s); s = fmaf(x1, y1, s);
                    }
                }
            }
            s *= sl2;
        }
        float mx = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m, mx), scale = m > -INFINITY ? exp2f(m - mn) : 1.0f;
        const float w = key < k1 ? exp2f(s - (mn > -INFINITY ? mn : 0.0f) + shift) : 0.0f;
        m = mn;
        float sum = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = l * scale + sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= scale;
        const int n = min(32, k1 - at);
        for (int i = 0; i < n; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            const long long o = __shfl_sync(0xffffffffu, off, i);
            if (o < 0) continue;
            const uint2 x = *(const uint2*)((const uint16_t*)p.v + o + col);
            float v[4];
            widen2<BF16>(x.x, v[0], v[1]); widen2<BF16>(x.y, v[2], v[3]);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = fmaf(wi, v[c], acc[c]);
        }
        if (__all_sync(0xffffffffu, acc[0] != acc[0] && acc[1] != acc[1] && acc[2] != acc[2] && acc[3] != acc[3])) return false;
    }
    return true;
}

#endif

// paged_attn_tc.cu: the form for many rows. Whether its loads suit this layout; its launch (`q` complete).
bool tc_supported(const sanic_attn_paged_params* p);
int32_t tc_launch(sanic_ctx* ctx, const Params& q, int head_dim, int dtype, int ctas, void* stream);
constexpr int TC_ROWS = 256;

}  // namespace paged
}  // namespace sanic
