// Causal attention of ragged chunks of new tokens over a paged key/value cache: the online-softmax fold (m, l, o) of
// out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j at or before token i's own position (and inside a sliding
// window), keys and values found through a page table.
//
// This file: the form for few query rows per (request, kv head) (decode, drafted tokens), the merge of items that several
// CTAs share, and the entry point. paged_attn_tc.cu: the form for many rows.
//
// With R = tokens * (query heads per kv head) rows the fold does 4 R flop per key element and reads it once (2 bytes for
// each of k and v), so up to some tens of rows HBM bounds it: what matters is bytes in flight and equal ranges. Four warps fold
// 64-key tiles out of a ring of 3 (head_dim 128) or 4 (64) stages that a fifth fills. (128-key tiles at head_dim 64, two CTAs
// per SM instead of three: 77 instead of 67 us for 64 decodes of 2000 keys.) The rows of an item are 16 MT rows of m16n8k16
// MMAs: with MT = 1 each warp takes 16 of the tile's keys, with MT = 2 a warp takes 16 rows and half of the keys, with MT = 4 a
// warp takes 16 rows and all keys. Carriers stay in registers; the warps that share rows merge once per segment. P goes to the tensor core rounded
// to the storage type (off by at most 2^-8 of a weight in bf16, 2^-11 in f16, there after a shift by 2^8, which keeps the weights of a long flat
// softmax out of f16's subnormals), sums and maxima are f32.
// The work is spread over an exactly resident grid as one contiguous range of (item, key tile) per CTA (paged_sched.h).
// 64 decodes of 8000 keys on average, 32 + 8 heads of 128, bf16 (2.14 GB): 340 us = 6.3 TB/s, 0.96 of the measured copy rate.
#include <type_traits>

#include "paged_tma.cuh"

namespace {
using namespace sanic;
using namespace sanic::paged;

constexpr int KT = 64;
// Chunks of more query rows than this (tokens * heads of a group) go to the tensor-memory form where its loads suit the layout.
// Groups of 4 heads of 128 over 4000 keys, rows form against tensor-memory form: 20 rows of 32 requests 104 / 125 us, 32 rows
// 107 / 126 us, 64 rows of 16 requests 92 / 80 us, of 2 requests 53 / 28 us. That is the border where no request may have more (by
// max_query_len, or by n_tokens where it is left out). Where one may, two launches share the requests and the border is what a
// single token of the group needs, 16 rows for groups up to 16 (make_plan): a rows form of 32 rows would fold single tokens, the most
// of such a batch, in items of twice the rows. Drafts beside a prompt, or without max_query_len, are served slower for it.
constexpr int TC_ABOVE_ROWS = 32;

template <int D> struct Cfg {
    static constexpr int STAGES = (D == 128) ? 3 : 4;
    static constexpr int TILE_BYTES = KT * D * 2;
    static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
    static constexpr int RING = STAGES * STAGE_BYTES;
    static constexpr int PREFIX_MAX = RING;            // the prefix sums over the requests share the ring's memory
    static_assert((MAX_REQUESTS + 1) * 8 <= PREFIX_MAX, "prefix sums fit the ring");
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF16> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool BF16> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16> constexpr float p_shift() { return BF16 ? 0.0f : 8.0f; }

// One K tile and one V tile into a stage: [D/64 halves][64 keys][128 B], chunk index xor (key & 7). `off` holds the tile's
// element offsets of k and v per key, -1 where nothing is to be read (beyond the keys the item sees, or a bad page): zeros
// then, so that whatever a page holds there never meets a zero weight.
template <int D>
__device__ __forceinline__ void load_tile(const uint16_t* k, const uint16_t* v, const longlong2* off, uint32_t stage, int tid) {
    constexpr int CPR = D / 8;
#pragma unroll
    for (int i = 0; i < (KT * CPR) / 128; ++i) {
        const int id = i * 128 + tid, key = id / CPR, c = id % CPR;
        const longlong2 o = off[key];
        const uint32_t dst = stage + (c >> 3) * (KT * 128) + key * 128 + (((c & 7) ^ (key & 7)) << 4);
        cp_async16(dst, k + (o.x >= 0 ? o.x + c * 8 : 0), o.x >= 0 ? 16 : 0);
        cp_async16(dst + Cfg<D>::TILE_BYTES, v + (o.x >= 0 ? o.y + c * 8 : 0), o.x >= 0 ? 16 : 0);
    }
}

// The fold of one item's rows by one warp: 16 MT rows of the item over the four warps of a CTA, warp (wr, wk) taking rows
// 16 wr .. and the wk-th part of a tile's keys.
template <int D, int MT, bool BF16> struct Fold {
    static constexpr int R = 16 * MT, WK = 4 / MT, KW = KT / WK, NC = KW / 16;    // rows, warps along keys, keys and 16-key chunks per warp
    static constexpr int KS = D / 16, NT = D / 8;
    int wr, wk, g, t, lane;
    uint32_t qf[KS][4];
    float o[NT][4], m0, m1, l0, l1;      // of rows ra and ra + 8; maxima in log2 units
    int lo_a, lo_c;                      // keys a row sees: [lo, lo + cnt)
    unsigned cnt_a, cnt_c;
    int inner_lo, inner_hi;              // every row of the item sees the whole of a tile between these
    bool nan_met;                        // a result held a NaN in a segment that hides keys from some of its rows (see repair)

    __device__ __forceinline__ void place(int warp, int lane_) { wr = warp % MT; wk = warp / MT; lane = lane_; g = lane >> 2; t = lane & 3; nan_met = false; }
    __device__ __forceinline__ int ra() const { return wr * 16 + g; }

    // row r of the item is head r % group of token r / group
    __device__ __forceinline__ void begin(const Params& p, const Seg& s, int block0, int n_tok) {
        const int r0 = ra(), r1 = r0 + 8, ta = r0 / p.group, tc = r1 / p.group;
        const uint16_t* Q = (const uint16_t*)p.q + (int64_t)(s.r.q0 + block0) * p.q_token_stride + (int64_t)s.hk * p.group * p.q_head_stride;
        const uint16_t* qa = Q + ta * p.q_token_stride + (r0 - ta * p.group) * p.q_head_stride + 2 * t;
        const uint16_t* qc = Q + tc * p.q_token_stride + (r1 - tc * p.group) * p.q_head_stride + 2 * t;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qf[ks][0] = ta < n_tok ? *(const uint32_t*)(qa + ks * 16) : 0u;
            qf[ks][1] = tc < n_tok ? *(const uint32_t*)(qc + ks * 16) : 0u;
            qf[ks][2] = ta < n_tok ? *(const uint32_t*)(qa + ks * 16 + 8) : 0u;
            qf[ks][3] = tc < n_tok ? *(const uint32_t*)(qc + ks * 16 + 8) : 0u;
        }
        const int pos0 = s.r.kv - s.r.qn + block0, pos_a = pos0 + ta, pos_c = pos0 + tc;
        lo_a = p.window > 0 ? max(0, pos_a - p.window + 1) : 0;
        lo_c = p.window > 0 ? max(0, pos_c - p.window + 1) : 0;
        cnt_a = ta < n_tok ? max(0, pos_a + 1 - lo_a) : 0;
        cnt_c = tc < n_tok ? max(0, pos_c + 1 - lo_c) : 0;
        inner_hi = pos0 + 1;
        inner_lo = p.window > 0 ? pos0 + n_tok - p.window : 0;
#pragma unroll
        for (int i = 0; i < NT; ++i) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f; }
        m0 = m1 = -INFINITY; l0 = l1 = 0.0f;
    }

    // One tile: [D/64 halves][64 keys][128 B] of K and of V, chunk index xor (key & 7).
    __device__ __forceinline__ void tile(uint32_t ks_addr, uint32_t vs_addr, int tile_key, float sl2) {
        float sc[NC][2][4];
        const int mi = lane >> 3, r = lane & 7;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[c][0][i] = sc[c][1][i] = 0.0f;
            const int krow = wk * KW + c * 16 + (mi >> 1) * 8 + r;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int ch = 2 * ks + (mi & 1);
                uint32_t r0, r1, r2, r3;
                ldmatrix_x4(ks_addr + (ch >> 3) * (KT * 128) + krow * 128 + (((ch & 7) ^ (krow & 7)) << 4), r0, r1, r2, r3);
                mma16816<BF16>(sc[c][0], qf[ks], r0, r1);
                mma16816<BF16>(sc[c][1], qf[ks], r2, r3);
            }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
        const int key0 = tile_key + wk * KW + 2 * t;
        const bool edge = tile_key + KT > inner_hi || tile_key < inner_lo;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (edge) {
                        const int key = key0 + c * 16 + h * 8 + i;
                        if (!((unsigned)(key - lo_a) < cnt_a)) sc[c][h][i] = -INFINITY;
                        if (!((unsigned)(key - lo_c) < cnt_c)) sc[c][h][2 + i] = -INFINITY;
                    }
                    mx0 = fmaxf(mx0, sc[c][h][i]); mx1 = fmaxf(mx1, sc[c][h][2 + i]);
                }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float mn0 = fmaxf(m0, mx0 * sl2), mn1 = fmaxf(m1, mx1 * sl2);      // the scale is positive
        // (a maximum that is still -inf has nothing to scale; 1 keeps such rows from asking for it)
        const float a0 = m0 > -INFINITY ? ex2(m0 - mn0) : 1.0f, a1 = m1 > -INFINITY ? ex2(m1 - mn1) : 1.0f;
        const float sub0 = (mn0 > -INFINITY ? mn0 : 0.0f) - p_shift<BF16>(), sub1 = (mn1 > -INFINITY ? mn1 : 0.0f) - p_shift<BF16>();
        m0 = mn0; m1 = mn1;
        float t0 = 0.0f, t1 = 0.0f;
        uint32_t pf[NC][4];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float e[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                e[h][0] = ex2(fmaf(sc[c][h][0], sl2, -sub0)); e[h][1] = ex2(fmaf(sc[c][h][1], sl2, -sub0));
                e[h][2] = ex2(fmaf(sc[c][h][2], sl2, -sub1)); e[h][3] = ex2(fmaf(sc[c][h][3], sl2, -sub1));
                t0 += e[h][0] + e[h][1]; t1 += e[h][2] + e[h][3];
            }
            pf[c][0] = pack2<BF16>(e[0][0], e[0][1]); pf[c][1] = pack2<BF16>(e[0][2], e[0][3]);
            pf[c][2] = pack2<BF16>(e[1][0], e[1][1]); pf[c][3] = pack2<BF16>(e[1][2], e[1][3]);
        }
        l0 = l0 * a0 + t0; l1 = l1 * a1 + t1;
        if (__any_sync(0xffffffffu, a0 != 1.0f || a1 != 1.0f)) {
#pragma unroll
            for (int i = 0; i < NT; ++i) { o[i][0] *= a0; o[i][1] *= a0; o[i][2] *= a1; o[i][3] *= a1; }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int krow = wk * KW + c * 16 + (mi & 1) * 8 + r;
#pragma unroll
            for (int dp = 0; dp < D / 16; ++dp) {
                const int ch = 2 * dp + (mi >> 1);
                uint32_t r0, r1, r2, r3;
                ldmatrix_x4_trans(vs_addr + (ch >> 3) * (KT * 128) + krow * 128 + (((ch & 7) ^ (krow & 7)) << 4), r0, r1, r2, r3);
                mma16816<BF16>(o[2 * dp], pf[c], r0, r1);
                mma16816<BF16>(o[2 * dp + 1], pf[c], r2, r3);
            }
        }
    }

    // The end of a segment: the carriers of the warps that share rows meet in shared memory (`os`, [WK][R][D] floats with the column
    // xor 8 (row & 3) against bank conflicts; `ml`, [WK][R]) and the rows leave, to out or to the segment's partial. `meet` is
    // a barrier of the 128 threads; all of them are done with what `os` held when this begins.
    template <class Meet>
    __device__ __forceinline__ void finish(const Params& p, const Seg& s, int block0, int n_tok, float* os, float2* ml, int tid, Meet meet) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        const int r0 = ra(), r1 = r0 + 8;
        if (t == 0) { ml[wk * R + r0] = make_float2(m0, l0); ml[wk * R + r1] = make_float2(m1, l1); }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int c = (8 * i + 2 * t) ^ ((g & 3) << 3);
            *(float2*)(os + (wk * R + r0) * D + c) = make_float2(o[i][0], o[i][1]);
            *(float2*)(os + (wk * R + r1) * D + c) = make_float2(o[i][2], o[i][3]);
        }
        meet();
        const bool whole = s.starts && s.finishes;
        const size_t slot = partial_slot(s, blockIdx.x);
        const int rows = n_tok * p.group;
        const bool hides = min(s.hi, s.je * KT) > inner_hi || max(s.lo, s.jb * KT) < inner_lo;
        for (int idx = tid; idx < rows * (D / 4); idx += 128) {
            const int r = idx / (D / 4), d = (idx % (D / 4)) * 4, c = d ^ ((r & 3) << 3);
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int w = 0; w < WK; ++w) m = fmaxf(m, ml[w * R + r].x);
            float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                const float2 x = ml[w * R + r];
                const float f = x.x > -INFINITY ? ex2(x.x - m) : 0.0f;       // a side that saw nothing has weight 0
                const float4 v4 = *(const float4*)(os + (w * R + r) * D + c);
                l += f * x.y;
                acc.x += f * v4.x; acc.y += f * v4.y; acc.z += f * v4.z; acc.w += f * v4.w;
            }
            const float all4 = (acc.x + acc.y) + (acc.z + acc.w);
            nan_met |= hides && all4 != all4;
            if (whole) {
                const int tok = r / p.group, head = s.hk * p.group + r - tok * p.group;
                const int64_t at = (int64_t)(s.r.q0 + block0 + tok) * p.q_heads + head;
                const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;      // no visible key: zeros, and -inf for the log-sum-exp
                *(uint2*)((uint16_t*)p.out + at * D + d) =
                    make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
                if (p.lse && d == 0) p.lse[at] = (m + log2f(l) - p_shift<BF16>()) * LN2;
            } else {
                *(float4*)(p.ws_o + (slot * p.rows + r) * D + d) = acc;
                if (d == 0) p.ws_ml[slot * p.rows + r] = make_float2(m, l);
            }
        }
    }
};

// Writes a row that was folded again: four columns per lane of the first D / 4 lanes.
template <bool BF16> __device__ __forceinline__ void store4(const Params& p, int64_t at, const float (&acc)[4], float inv) {
    *(uint2*)((uint16_t*)p.out + at) = make_uint2(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv));
}
template <bool BF16> __device__ __forceinline__ bool holds_nan(const Params& p, int64_t at) {      // the same four columns of the result
    const uint2 x = __ldcg((const uint2*)((const uint16_t*)p.out + at));
    float v[4];
    widen2<BF16>(x.x, v[0], v[1]); widen2<BF16>(x.y, v[2], v[3]);
    return v[0] != v[0] || v[1] != v[1] || v[2] != v[2] || v[3] != v[3];
}

// Where the rows form is alone, its CTAs that met a NaN while some key of a segment was hidden from some of its rows go over their
// segments once more at their end (128 threads that meet at `sync`; `cum`, shared memory, is free again): such rows that hold a
// NaN are folded again over the keys of the segment that they see (fold_row), a warp per row. 24 drafted chunks 0.5-1.5 us slower for it.
template <int D, bool BF16, class Sync>
__device__ __noinline__ void repair(const Params& p, long long* cum, int tid, Sync sync) {
    const int warp = tid >> 5, lane = tid & 31, col = (lane % (D / 4)) * 4;
    scan_costs<KT>(p, cum, nullptr, tid, 128, sync);
    DeviceWalk<KT> walk{LoadReq{&p, nullptr}};
    walk.init(p, cum, blockIdx.x, gridDim.x);
    Seg s;
    while (walk.next(p, s)) {
        const int block0 = s.rb * p.block_tokens, n_tok = min(p.block_tokens, s.r.qn - block0), pos0 = s.r.kv - s.r.qn + block0;
        const int first_key = max(s.lo, s.jb * KT), end_key = min(s.hi, s.je * KT);
        const bool whole = s.starts && s.finishes;
        for (int r = warp; r < n_tok * p.group; r += 4) {
            const int tok = r / p.group, head = s.hk * p.group + r - tok * p.group, pos = pos0 + tok;
            const int k0 = max(first_key, p.window > 0 ? max(0, pos - p.window + 1) : 0), k1 = min(end_key, max(0, pos + 1));
            if (k0 == first_key && k1 == end_key) continue;
            const int64_t at = ((int64_t)(s.r.q0 + block0 + tok) * p.q_heads + head) * D + col;
            const size_t slot_row = (size_t)partial_slot(s, blockIdx.x) * p.rows + r;
            float4* part = (float4*)(p.ws_o + slot_row * D + col);
            bool lost;
            if (whole) lost = holds_nan<BF16>(p, at);
            else { const float4 x = __ldcg(part); lost = x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w; }
            if (!__any_sync(0xffffffffu, lost)) continue;
            const uint16_t* q = (const uint16_t*)p.q + (int64_t)(s.r.q0 + block0 + tok) * p.q_token_stride + (int64_t)head * p.q_head_stride;
            float m, l, acc[4];
            const bool summed = fold_row<D, BF16>(p, s.b, s.hk, q, k0, k1, p_shift<BF16>(), col, m, l, acc);
            if (lane >= D / 4) continue;
            if (whole) store4<BF16>(p, at, acc, summed && l > 0.0f ? 1.0f / l : 0.0f);
            else {
                *part = make_float4(acc[0], acc[1], acc[2], acc[3]);
                if (lane == 0 && summed) p.ws_ml[slot_row] = make_float2(m, l);
            }
        }
    }
}

// Any layout: the four warps copy the tiles themselves, 16 bytes a time (cp.async). ALONE: no tensor-memory form beside (its merge looks at
// both forms' results, and a longer kernel in front of it costs 3-5 us).
template <int D, int MT, bool BF16, bool ALONE>
__global__ void __launch_bounds__(128) paged_rows_kernel(const __grid_constant__ Params p, int* err) {
    constexpr int STAGES = Cfg<D>::STAGES;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ longlong2 s_off[STAGES][KT];
    __shared__ float2 s_ml[64];
    const int tid = threadIdx.x;
    const uint32_t base = smem_u32(smem);
    Fold<D, MT, BF16> f;
    f.place(tid >> 5, tid & 31);

    griddep_wait();        // q, the pages, the table and the lengths come from earlier kernels of the step
    griddep_launch();
    scan_costs<KT>(p, (long long*)smem, err);
    DeviceWalk<KT> walk{LoadReq{&p, nullptr}};
    walk.init(p, (long long*)smem, blockIdx.x, gridDim.x);
    __syncthreads();       // the prefix sums' memory becomes the tile ring

    int4 merge = make_int4(0, 0, 0, 0);
    const float sl2 = p.scale * LOG2E;
    Seg s;
    while (walk.next(p, s)) {
        const int n_tiles = s.je - s.jb;
        const int32_t* row = p.table + (int64_t)s.b * p.table_stride;
        const uint16_t* K = (const uint16_t*)p.k + s.hk * p.k_head_stride;
        const uint16_t* V = (const uint16_t*)p.v + s.hk * p.v_head_stride;
        const int block0 = s.rb * p.block_tokens;                              // first token of the item in its chunk
        const int n_tok = min(p.block_tokens, s.r.qn - block0);

        // Page and offsets of a tile's keys, by threads 0..63; the table entry is loaded two tiles ahead of the copies that need it.
        auto page_of = [&](int tile, int key_in_tile) {
            const int key = (s.jb + tile) * KT + key_in_tile;
            int page = -1, in_page;
            if (tile < n_tiles && key >= s.lo && key < s.hi && !locate(p, row, key, page, in_page, err)) page = -1;
            return page;
        };
        auto offsets = [&](int page, int tile, int key_in_tile) {
            const int key = (s.jb + tile) * KT + key_in_tile;
            const int in_page = p.page_shift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
            return page < 0 ? make_longlong2(-1, -1)
                            : make_longlong2(page * p.k_page_stride + in_page * p.k_row_stride, page * p.v_page_stride + in_page * p.v_row_stride);
        };
        for (int i = tid; i < STAGES * KT; i += 128)
            if (i / KT < n_tiles) s_off[i / KT][i % KT] = offsets(page_of(i / KT, i % KT), i / KT, i % KT);
        int page = tid < KT ? page_of(STAGES, tid) : -1;       // of tile it + STAGES
        __syncthreads();
#pragma unroll
        for (int st = 0; st < STAGES - 1; ++st) {
            if (st < n_tiles) load_tile<D>(K, V, s_off[st], base + st * Cfg<D>::STAGE_BYTES, tid);
            cp_async_commit();
        }
        f.begin(p, s, block0, n_tok);
        for (int it = 0; it < n_tiles; ++it) {
            cp_async_wait<STAGES - 2>();
            __syncthreads();
            const int nx = it + STAGES - 1;
            if (nx < n_tiles) load_tile<D>(K, V, s_off[nx % STAGES], base + (nx % STAGES) * Cfg<D>::STAGE_BYTES, tid);
            cp_async_commit();
            const int ahead = tid < KT ? page_of(nx + 2, tid) : -1;
            const uint32_t ks_addr = base + (it % STAGES) * Cfg<D>::STAGE_BYTES;
            f.tile(ks_addr, ks_addr + Cfg<D>::TILE_BYTES, (s.jb + it) * KT, sl2);
            if (tid < KT) s_off[(nx + 1) % STAGES][tid] = offsets(page, nx + 1, tid);
            page = ahead;
        }
        cp_async_wait<0>();
        __syncthreads();      // every warp is done with the ring: it takes the warps' carriers
        f.finish(p, s, block0, n_tok, (float*)smem, s_ml, tid, [] { __syncthreads(); });
        if (s.parts > 1) merge = make_int4(s.r.q0 + block0, n_tok, s.hk, s.parts);
        __syncthreads();
    }
    if (tid == 0) p.ws_merge[blockIdx.x] = merge;
    if (ALONE && __syncthreads_or(f.nan_met)) repair<D, BF16>(p, (long long*)smem, tid, [] { __syncthreads(); });
}

// Pools that TMA can read (paged_tma.cuh): a fifth warp produces. It walks the same segments ahead of the others, through the ends
// of items, so that bytes stay in flight while they merge and store; it looks up a tile's pages one tile ahead and issues one
// copy per lane (a box of a page's rows, 64 columns, of K or of V). The four warps wait for a tile, fold it and hand the stage
// back, each for itself: no barrier between tiles. (With the copies issued by the folding warps: 434 us by cp.async, 363 us
// by TMA from warp 0, for 64 requests of 8000 keys on average.)
struct RowsArgs { int box_rows, k_heads_inner, v_heads_inner; };
// Registers: at head_dim 128 two CTAs per SM leave a thread 168; 32, 56 and 132 bytes spill for 16, 32 and 64 rows.
constexpr int TMA_THREADS = 160;
template <int D, int MT> constexpr int tma_ctas_per_sm() { return D == 128 ? 2 : (MT == 1 ? 3 : 2); }

template <int D, int MT, bool BF16, bool ALONE>
__global__ void __launch_bounds__(TMA_THREADS, (tma_ctas_per_sm<D, MT>()))
paged_rows_tma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Params p, const RowsArgs a, int* err) {
    using F = Fold<D, MT, BF16>;
    constexpr int STAGES = Cfg<D>::STAGES;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);      // the swizzle counts from 1024-byte lines
    __shared__ uint64_t s_full[STAGES], s_empty[STAGES];
    __shared__ float2 s_ml[64];
    __shared__ volatile int s_abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(smem);
    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) { tc::mbar_init(&s_full[i], 1); tc::mbar_init(&s_empty[i], 4); }
        s_abort = 0;
        tc::mbar_init_fence();
    }
    griddep_wait();
    griddep_launch();
    scan_costs<KT>(p, (long long*)smem, err);
    DeviceWalk<KT> walk{LoadReq{&p, nullptr}};
    walk.init(p, (long long*)smem, blockIdx.x, gridDim.x);
    tc::fence_async_smem();
    __syncthreads();       // the prefix sums' memory becomes the tile ring
    Seg s;
    uint32_t u = 0;        // tiles so far: position in the ring

    if (warp == 4) {
        constexpr int COPIES = 2 * (D / 64);
        const int box = lane / COPIES, slab = (lane % COPIES) >> 1, of_v = lane & 1;
        const bool inner = of_v ? a.v_heads_inner : a.k_heads_inner;
        const CUtensorMap* map = of_v ? &map_v : &map_k;
        const int in_tile = box * a.box_rows;
        const uint32_t to = base + of_v * Cfg<D>::TILE_BYTES + slab * (KT * 128) + in_tile * 128;
        while (walk.next(p, s)) {
            const int32_t* row = p.table + (int64_t)s.b * p.table_stride;
            // -1 where no visible key lies in the box, n_pages (read as zeros) for a bad entry
            auto page_of = [&](int j) {
                const int key = j * KT + in_tile;
                if (j >= s.je || in_tile >= KT || key >= s.hi || key + a.box_rows <= s.lo) return -1;
                int page, in_page;
                return locate(p, row, key, page, in_page, err) ? page : p.n_pages;
            };
            int page = page_of(s.jb), next = page_of(s.jb + 1);
            for (int j = s.jb; j < s.je; ++j, ++u) {
                const int after = page_of(j + 2);
                const int st = u % STAGES;
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&s_empty[st], ((u / STAGES) & 1) ^ 1, &s_abort, err, 26))) return;
                const int key = j * KT + in_tile, in_page = p.page_shift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, page >= 0)) * a.box_rows * 128;
                if (lane == 0) tc::mbar_expect_tx(&s_full[st], bytes);
                __syncwarp();
                if (page >= 0) tma_load_4d(to + st * Cfg<D>::STAGE_BYTES, map, &s_full[st], slab * 64, inner ? s.hk : in_page, inner ? in_page : s.hk, page);
                page = next; next = after;
            }
        }
        return;
    }

    F f;
    f.place(warp, lane);
    auto meet = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    int4 merge = make_int4(0, 0, 0, 0);
    const float sl2 = p.scale * LOG2E;
    bool ok = true;        // a wait that ran out is not repeated; the barriers below are still met by every warp
    while (walk.next(p, s)) {
        const int block0 = s.rb * p.block_tokens;
        const int n_tok = min(p.block_tokens, s.r.qn - block0);
        f.begin(p, s, block0, n_tok);
        uint32_t ks_addr = base;
        for (int j = s.jb; j < s.je; ++j, ++u) {
            const int st = u % STAGES;
            if (ok) ok = tc::mbar_wait(&s_full[st], (u / STAGES) & 1, &s_abort, err, 27);
            __syncwarp();
            ks_addr = base + st * Cfg<D>::STAGE_BYTES;
            const uint32_t vs_addr = ks_addr + Cfg<D>::TILE_BYTES;
            const int tile_key = j * KT, first = tile_key + f.wk * F::KW;
            if (first < s.lo || first + F::KW > s.hi) {
                // rows of V outside the keys the item sees hold whatever the page does: zeros, where this warp reads
                for (int i = lane; i < F::KW * (D / 8); i += 32) {
                    const int r = i / (D / 8), c = i % (D / 8), rr = f.wk * F::KW + r;
                    if (tile_key + rr < s.lo || tile_key + rr >= s.hi)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(vs_addr + (c >> 3) * (KT * 128) + rr * 128 + (c & 7) * 16), "r"(0) : "memory");
                }
                tc::fence_async_smem();        // before a later copy into the stage
                __syncwarp();
            }
            f.tile(ks_addr, vs_addr, tile_key, sl2);
            __syncwarp();
            if (lane == 0 && j + 1 < s.je) tc::mbar_arrive(&s_empty[st]);
        }
        // the last tile's stage takes the warps' carriers, then it goes back too
        meet();
        if (s.je > s.jb) {
            f.finish(p, s, block0, n_tok, (float*)(smem + (ks_addr - base)), s_ml, tid, meet);
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s_empty[(u - 1) % STAGES]);
        } else {                               // no key is visible: zeros, and -inf for the log-sum-exp
            for (int i = tid; i < n_tok * p.group * (D / 4); i += 128) {
                const int r = i / (D / 4), d = (i % (D / 4)) * 4, tok = r / p.group;
                const int64_t at = (int64_t)(s.r.q0 + block0 + tok) * p.q_heads + s.hk * p.group + r - tok * p.group;
                *(uint2*)((uint16_t*)p.out + at * D + d) = make_uint2(0, 0);
                if (p.lse && d == 0) p.lse[at] = -INFINITY;
            }
        }
        if (s.parts > 1) merge = make_int4(s.r.q0 + block0, n_tok, s.hk, s.parts);
    }
    if (tid == 0) p.ws_merge[blockIdx.x] = merge;
    if (ALONE) {
        int nan_met;
        asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %1, 0;\n\tbarrier.cta.red.or.pred b, 1, 128, a;\n\tselp.s32 %0, 1, 0, b;\n\t}"
                     : "=r"(nan_met) : "r"((int)(f.nan_met && ok)) : "memory");
        if (nan_met) repair<D, BF16>(p, (long long*)smem, tid, meet);
    }
}

struct Merge { const float* ws_o; const float2* ws_ml; const int4* ws_merge; int rows, ctas; };      // one fold's partials

// With the tensor-memory form, whose kernel is left as it is (a look at its sums costs it 2-5 %, one at its tiles 8-16), a few blocks of
// the merge's launch look at some of the results instead: a value that is hidden from some rows of an item is seen by its last
// token, or with a window by its first (by some token, where the window is shorter than the item), and a row that sees a value
// that is not finite is not finite itself (zeros, where each of its few weights was 0). Where they find such a row they go over its item: rows
// that hold a NaN are folded again over all keys that they see. Items that several CTAs share are written by the merging blocks,
// which do the same for theirs. A warp's unit is CHECKS such rows of a request and kv head, every `split`-th.
constexpr int CHECKS = 8;
struct Look { int blocks, split; long long units; int few, tokens_few, tokens_many; };      // tokens of an item: of requests of up to `few` query rows, of others
struct Items { int n, r0, r1; int4 item[16 * CHECKS]; };      // to go over: request, first token in its chunk, kv head, first token row; a merging block's one: rows [r0, r1)

template <int D, bool BF16>
__device__ __forceinline__ void go_over(const Params& p, const int4& it, int r0, int r1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = (lane % (D / 4)) * 4;
    const Req r = LoadReq{&p, nullptr}(it.x);
    if (r.qn < 2) return;                          // a token alone: nothing is hidden from it
    for (int k = r0 + warp; k < r1; k += 16) {
        const int i = it.y + k / p.group, head = it.z * p.group + k % p.group, pos = r.kv - r.qn + i, t = r.q0 + i;
        const int64_t at = ((int64_t)t * p.q_heads + head) * D + col;
        if (i >= r.qn || pos < 0 || !__any_sync(0xffffffffu, holds_nan<BF16>(p, at))) continue;
        float m, l, acc[4];
        const bool summed = fold_row<D, BF16>(p, it.x, it.z, (const uint16_t*)p.q + (int64_t)t * p.q_token_stride + (int64_t)head * p.q_head_stride,
                                              p.window > 0 ? max(0, pos - p.window + 1) : 0, pos + 1, 0.0f, col, m, l, acc);
        if (lane < D / 4) store4<BF16>(p, at, acc, summed && l > 0.0f ? 1.0f / l : 0.0f);
    }
}

template <int D, bool BF16>
__device__ __forceinline__ void look_at_results(const Params& p, const Merge& first, const Merge& second, const Look& look, Items& items) {
    constexpr int LANES = D / 8, ROWS = 32 / LANES;      // lanes of a row, rows of a load
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    long long u = (long long)blockIdx.x * 16 + warp;
    int c0 = -1;                                   // the unit's next rows; -1: its first
    if (threadIdx.x == 0) items.n = 0;
    // The first turn is taken twice: while the folds still run, for the instructions and lengths that it fetches (their latencies are
    // most of it), and for its result once they have ended.
    bool ahead = true;
    while (__syncthreads_or(u < look.units)) {     // (the block's turns end together: what one finds is gone over by all of its warps)
        if (u < look.units) {
            const long long v = u / look.split;
            const int hk = (int)(v % p.kv_heads), b = (int)(v / p.kv_heads);
            const Req r = LoadReq{&p, nullptr}(b);
            const int bt = (long long)r.qn * p.group <= look.few ? look.tokens_few : look.tokens_many;
            const int edges = p.window == 0 ? 1 : p.window >= bt ? 2 : bt;      // rows looked at per item
            if (c0 < 0) c0 = (int)(u - v * look.split) * CHECKS;
            const int c = c0 + lane % CHECKS, block0 = c / edges * bt, n_tok = min(bt, r.qn - block0);
            const int i = block0 + (edges == bt ? c % edges : c % edges ? 0 : n_tok - 1);
            long long off = -1;
            if (n_tok > 1 && i < block0 + n_tok && r.kv - r.qn + i >= 0) off = ((long long)(r.q0 + i) * p.q_heads + hk * p.group) * D;
            unsigned odd = 0u, full = 0u;          // not finite; not all zeros
#pragma unroll
            for (int k = 0; k < CHECKS; k += ROWS) {
                const long long o = __shfl_sync(0xffffffffu, off, k + lane / LANES);
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (o >= 0) x = __ldcg((const uint4*)((const uint16_t*)p.out + o + (lane % LANES) * 8));
                constexpr uint32_t one = BF16 ? 0x00800080u : 0x04000400u;      // exponents all ones, in either half of a word
                const uint32_t y = ((x.x & 0x7fff7fffu) + one) | ((x.y & 0x7fff7fffu) + one) | ((x.z & 0x7fff7fffu) + one) | ((x.w & 0x7fff7fffu) + one);
                if (y & 0x80008000u) odd |= 1u << (k + lane / LANES);
                if ((x.x | x.y | x.z | x.w) & 0x7fff7fffu) full |= 1u << (k + lane / LANES);
            }
            odd = __reduce_or_sync(0xffffffffu, odd);
            full = __reduce_or_sync(0xffffffffu, full);
            if (edges == bt) odd |= __ballot_sync(0xffffffffu, off >= 0 && lane < CHECKS) & ~full;
            if (ahead) odd = 0u;
            if (((odd >> lane) & 1u) && (__match_any_sync(odd, block0) & ((1u << lane) - 1u)) == 0u)      // one lane per item
                items.item[atomicAdd(&items.n, 1)] = make_int4(b, block0, hk, r.q0 + block0);
            if (!ahead) {
                c0 += look.split * CHECKS;
                if (c0 >= (r.qn + bt - 1) / bt * edges) { u += (long long)look.blocks * 16; c0 = -1; }
            }
        }
        if (ahead) { griddep_wait(); ahead = false; }
        __syncthreads();
        for (int x = 0; x < items.n; ++x) {
            const int4 it = items.item[x];
            bool shared = false;                   // those are the merging blocks'
            for (int c = lane; c < first.ctas + second.ctas; c += 32) {
                const int4 m = c < first.ctas ? first.ws_merge[c] : second.ws_merge[c - first.ctas];
                shared |= m.w > 1 && m.x == it.w && m.z == it.z;
            }
            if (!__any_sync(0xffffffffu, shared)) go_over<D, BF16>(p, it, 0, look.tokens_many * p.group);      // (a chunk of the other form is one item, and smaller)
        }
        __syncthreads();
        if (threadIdx.x == 0) items.n = 0;
    }
}

// Merge of the items that several CTAs share, for one fold or for two that ran side by side. The item that starts in one CTA's
// range is served by a block per 16 rows of the rows form's items (24 drafted chunks of 3-6 tokens: 97.5 us with one block per item,
// 95.7 so, 99 with a block per 8 rows), by four blocks of the tensor-memory form's (all resident at once: 16 drafted chunks of 16 tokens 78.3
// us, 81.2 with eight, 87.8 with 16; two or four rows of a warp at once: 79.5-85). A row's partials are split over 16 / rows warps
// (at least one) and joined through shared memory in a fixed order. Bound by latency: its start, an item's record, the partials (39 MB
// at most of the tensor-memory form and 20 MB of the rows form, in L2), the join; 148 shared items of 256 rows 16-18 us.
constexpr int TC_MERGE_SPLIT = 4;      // blocks per item of the tensor-memory form
// One block's part of a shared item; true (NOTE) where one of its rows came out NaN, noted in `items`.
template <int D, bool BF16, bool NOTE>
__device__ __forceinline__ bool merge_item(const Params& p, const Merge& first, const Merge& second, int index, int n_first, int split_first, float2 (&s_ml)[16], float (&s_o)[16][D], Items* items) {
    const bool one = index < n_first;
    const int n_parts = one ? split_first : TC_MERGE_SPLIT, block = one ? index : index - n_first;
    const int cta = block / n_parts, part = block - cta * n_parts;
    // field by field: a reference to one of two parameters would be read through memory at every use
    const float* ws_o = one ? first.ws_o : second.ws_o;
    const float2* ws_ml = one ? first.ws_ml : second.ws_ml;
    const int slot_rows = one ? first.rows : second.rows;
    const int4 it = (one ? first.ws_merge : second.ws_merge)[cta];
    if (it.w <= 1) return false;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int V = D / 32;                      // floats per lane
    const int rows = it.y * p.group, r0 = rows * part / n_parts, r1 = rows * (part + 1) / n_parts;
    int wpr = 16;                                  // warps per row
    while (wpr > 1 && (r1 - r0) * wpr > 16) wpr >>= 1;
    const int rpp = 16 / wpr, sub = warp % wpr;    // rows at a time, this warp's share of the parts
    bool met = false;                              // a row that came out NaN
    for (int rr = r0; rr < r1; rr += rpp) {
        const int r = rr + warp / wpr;
        float m = -INFINITY, l = 0.0f, o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.0f;
        if (r < r1) {
            for (int q0 = sub; q0 < it.w; q0 += wpr * 4) {
                float2 x[4]; float a[4][V];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int q = q0 + u * wpr;
                    x[u] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                    for (int i = 0; i < V; ++i) a[u][i] = 0.0f;
                    if (q < it.w) {
                        const size_t at = ((size_t)(cta + q) * 2 + (q == 0 ? 1 : 0)) * slot_rows + r;
                        x[u] = __ldcg(ws_ml + at);
                        const float* po = ws_o + at * D + lane * V;
                        if (V == 4) { const float4 f = __ldcg((const float4*)po); a[u][0] = f.x; a[u][1] = f.y; a[u][V - 2] = f.z; a[u][V - 1] = f.w; }
                        else { const float2 f = __ldcg((const float2*)po); a[u][0] = f.x; a[u][1] = f.y; }
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float mn = fmaxf(m, x[u].x);
                    const float fa = m > -INFINITY ? ex2(m - mn) : 0.0f, fb = x[u].x > -INFINITY ? ex2(x[u].x - mn) : 0.0f;
                    l = l * fa + x[u].y * fb;
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = o[i] * fa + a[u][i] * fb;
                    m = mn;
                }
            }
        }
        if (wpr > 1) {
            if (lane == 0) s_ml[warp] = make_float2(m, l);
#pragma unroll
            for (int i = 0; i < V; ++i) s_o[warp][lane * V + i] = o[i];
            __syncthreads();
            if (sub == 0) {
                for (int w = 1; w < wpr; ++w) {
                    const float2 x = s_ml[warp + w];
                    const float mn = fmaxf(m, x.x);
                    const float fa = m > -INFINITY ? ex2(m - mn) : 0.0f, fb = x.x > -INFINITY ? ex2(x.x - mn) : 0.0f;
                    l = l * fa + x.y * fb;
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = o[i] * fa + s_o[warp + w][lane * V + i] * fb;
                    m = mn;
                }
            }
            __syncthreads();
        }
        if (r < r1 && sub == 0) {
            const int tok = r / p.group, head = it.z * p.group + r - tok * p.group;
            const int64_t at = (int64_t)(it.x + tok) * p.q_heads + head;
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            uint16_t* dst = (uint16_t*)p.out + at * D + lane * V;
            *(uint32_t*)dst = pack2<BF16>(o[0] * inv, o[1] * inv);
            if (V == 4) *(uint32_t*)(dst + 2) = pack2<BF16>(o[V - 2] * inv, o[V - 1] * inv);
            if (p.lse && lane == 0) p.lse[at] = (m + log2f(l) - p_shift<BF16>()) * LN2;
            if (NOTE) {
                float all = o[0] + o[1];
                if (V == 4) all += o[V - 2] + o[V - 1];
                met |= all != all;
            }
        }
    }
    if (!NOTE || !__syncthreads_or(met)) return false;
    if (threadIdx.x == 0) {                        // the request: the last that starts at or before the item
        int b = 0, hi = p.n_requests - 1;
        while (b < hi) { const int mid = (b + hi + 1) >> 1; if (__ldcg(p.query_start + mid) <= it.x) b = mid; else hi = mid - 1; }
        items->r0 = r0; items->r1 = r1;
        items->item[0] = make_int4(b, it.x - LoadReq{&p, nullptr}(b).q0, it.z, it.x);
    }
    __syncthreads();
    return true;
}

// LOOK: with the blocks that look at results in front. p: of all requests, whichever form served them.
template <int D, bool BF16, bool LOOK>
__global__ void __launch_bounds__(512) paged_merge_kernel(const __grid_constant__ Params p, const Merge first, const Merge second, const Look look, const int n_first, const int split_first) {
    if (!LOOK || blockIdx.x >= look.blocks) griddep_wait();
    griddep_launch();
    struct Rows { float2 ml[16]; float o[16][D]; };
    struct Nothing {};
    __shared__ union { Rows rows; std::conditional_t<LOOK, Items, Nothing> items; } sh;
    Items* items = (Items*)&sh;
    if (LOOK && blockIdx.x < look.blocks) look_at_results<D, BF16>(p, first, second, look, *items);
    else if (merge_item<D, BF16, LOOK>(p, first, second, blockIdx.x - look.blocks, n_first, split_first, sh.rows.ml, sh.rows.o, items)) go_over<D, BF16>(p, items->item[0], items->r0, items->r1);
}

template <int D, int MT, bool BF16, bool ALONE>
int32_t launch_rows(sanic_ctx* ctx, const Params& p, bool tma, int ctas, cudaStream_t st) {
    constexpr int smem = Cfg<D>::RING;
    static_assert(4 * 16 * D * 4 <= Cfg<D>::STAGE_BYTES, "the warps' carriers fit a stage");
    static thread_local int ready_on = -1;       // the attribute is per device
    if (ready_on != ctx->device) {
        SANIC_CUDA_CHECK(ctx, cudaFuncSetAttribute(paged_rows_kernel<D, MT, BF16, ALONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        SANIC_CUDA_CHECK(ctx, cudaFuncSetAttribute(paged_rows_tma_kernel<D, MT, BF16, ALONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem + 1024));
        ready_on = ctx->device;
    }
    if (!tma) {
        SANIC_CUDA_CHECK(ctx, launch_pdl(paged_rows_kernel<D, MT, BF16, ALONE>, dim3(ctas), dim3(128), smem, st, p, ctx->status_dev));
        return SANIC_OK;
    }
    CUtensorMap mk, mv;
    RowsArgs a{};
    a.box_rows = box_rows_of(p.page_size, KT);
    bool ki, vi;
    int32_t rc = encode_pool(ctx, &mk, BF16, p, 0, D, a.box_rows, &ki);
    if (rc == SANIC_OK) rc = encode_pool(ctx, &mv, BF16, p, 1, D, a.box_rows, &vi);
    if (rc != SANIC_OK) return rc;
    a.k_heads_inner = ki; a.v_heads_inner = vi;
    SANIC_CUDA_CHECK(ctx, launch_pdl(paged_rows_tma_kernel<D, MT, BF16, ALONE>, dim3(ctas), dim3(TMA_THREADS), smem + 1024, st, mk, mv, p, a, ctx->status_dev));
    return SANIC_OK;
}
template <int MT, bool ALONE>
int32_t launch_rows_any(sanic_ctx* ctx, const Params& p, int D, int dtype, bool tma, int ctas, cudaStream_t st) {
    if (D == 128) return dtype == SANIC_BF16 ? launch_rows<128, MT, true, ALONE>(ctx, p, tma, ctas, st) : launch_rows<128, MT, false, ALONE>(ctx, p, tma, ctas, st);
    return dtype == SANIC_BF16 ? launch_rows<64, MT, true, ALONE>(ctx, p, tma, ctas, st) : launch_rows<64, MT, false, ALONE>(ctx, p, tma, ctas, st);
}

// Resident CTAs of the rows form: what its shared memory (96 or 64 KB) and registers leave.
int rows_ctas(const sanic_ctx* ctx, int D, int rows) { return ctx->sm_count * (D == 128 ? tma_ctas_per_sm<128, 1>() : rows == 16 ? tma_ctas_per_sm<64, 1>() : tma_ctas_per_sm<64, 2>()); }

// Which forms serve a call: the rows form (`rows` query rows per item; 0: not launched) and the tensor-memory form (`tc`).
struct Plan { int rows, rows_ctas; bool tc; int tc_ctas; };
int pow2_rows(long long want) { int r = 16; while (r < 64 && r < want) r *= 2; return r; }
Plan make_plan(const sanic_ctx* ctx, const sanic_attn_paged_params* p) {
    const int group = p->q_heads / p->kv_heads;
    const long long want = (long long)(p->max_query_len > 0 ? p->max_query_len : p->n_tokens) * group;
    Plan pl{};
    pl.tc = want > TC_ABOVE_ROWS && tc_supported(p);
    if (pl.tc) {
        // A batch may hold single tokens beside its chunks: those are the rows form's, in a launch of their own (28 decodes beside
        // four chunks of 300-600 tokens: 145 us in one launch of the tensor-memory form). Not where the single tokens of a large
        // group are all there is: one launch (64 requests of one token, 64 heads of 128 to a kv head, 4000 keys: 45 us; in the
        // rows form 56, in both 58; head_dim 64: 37, 38, 41)
        pl.tc_ctas = ctx->sm_count;
        pl.rows = p->n_requests > 1 && want > pow2_rows(group) ? pow2_rows(group) : 0;
    } else {
        pl.rows = pow2_rows(want);
    }
    pl.rows_ctas = rows_ctas(ctx, p->head_dim, pl.rows);
    return pl;
}

size_t slots_bytes(int ctas, int rows, int D) { return 2 * (size_t)ctas * rows * (D * 4 + 8) + (size_t)ctas * 16; }
size_t workspace_bytes(const Plan& pl, int D) {
    return (pl.rows ? slots_bytes(pl.rows_ctas, pl.rows, D) : 0) + (pl.tc ? slots_bytes(pl.tc_ctas, TC_ROWS, D) : 0);
}
// Lays one launch's partials out in the workspace; returns what follows them.
unsigned char* place(Params& q, unsigned char* ws, int ctas, int rows, int D) {
    const size_t slots = 2 * (size_t)ctas * rows;
    q.rows = rows;
    q.ws_o = (float*)ws;
    q.ws_ml = (float2*)(q.ws_o + slots * D);
    q.ws_merge = (int4*)(q.ws_ml + slots);
    return ws + slots_bytes(ctas, rows, D);
}

int32_t validate(sanic_ctx* ctx, const sanic_attn_paged_params* p) {
    SANIC_REQUIRE(ctx, p->n_requests >= 0 && p->n_tokens >= 0 && p->max_query_len >= 0, "attn_paged: negative count");
    // an empty call has tensors without elements
    SANIC_REQUIRE(ctx, p->n_requests == 0 || p->n_tokens == 0 || (p->q && p->out && p->k_pages && p->v_pages && p->block_table && p->query_start && p->kv_lens),
                  "attn_paged: null tensor");
    SANIC_REQUIRE(ctx, p->dtype == SANIC_BF16 || p->dtype == SANIC_F16, "attn_paged: q, the pages and out are bf16 or f16");
    if (p->head_dim != 64 && p->head_dim != 128) return sanic_fail(ctx, SANIC_ERR_UNSUPPORTED, "attn_paged: head_dim must be 64 or 128");
    SANIC_REQUIRE(ctx, p->kv_heads > 0 && p->q_heads > 0 && p->q_heads % p->kv_heads == 0, "attn_paged: query heads must be a multiple of key/value heads");
    if (p->q_heads / p->kv_heads > 64) return sanic_fail(ctx, SANIC_ERR_UNSUPPORTED, "attn_paged: at most 64 query heads per key/value head");
    SANIC_REQUIRE(ctx, p->n_requests <= MAX_REQUESTS, "attn_paged: at most 8000 requests per call");
    SANIC_REQUIRE(ctx, p->page_size > 0 && p->n_pages > 0 && p->max_pages > 0, "attn_paged: empty page pool or table");
    SANIC_REQUIRE(ctx, (long long)p->n_tokens * p->q_heads < (1ll << 31), "attn_paged: too many rows");
    // positions run from -n_tokens (more tokens than keys) to the row's last key, and a window's start below them: all in 32 bits
    SANIC_REQUIRE(ctx, (long long)p->max_pages * p->page_size + p->n_tokens < (1ll << 31) - 256, "attn_paged: a table row spans 2^31 keys or more");
    SANIC_REQUIRE(ctx, p->window >= 0, "attn_paged: negative window");
    SANIC_REQUIRE(ctx, p->scale > 0.0f && p->scale < INFINITY, "attn_paged: scale must be positive and finite");
    SANIC_REQUIRE(ctx, p->q_token_stride % 8 == 0 && p->q_head_stride % 8 == 0 && p->k_page_stride % 8 == 0 && p->k_row_stride % 8 == 0 &&
                  p->k_head_stride % 8 == 0 && p->v_page_stride % 8 == 0 && p->v_row_stride % 8 == 0 && p->v_head_stride % 8 == 0 &&
                  ((uintptr_t)p->q % 16) == 0 && ((uintptr_t)p->k_pages % 16) == 0 && ((uintptr_t)p->v_pages % 16) == 0 && ((uintptr_t)p->out % 16) == 0,
                  "attn_paged: rows of q, k, v and out must be 16-byte aligned");
    SANIC_REQUIRE(ctx, p->q_token_stride >= 0 && p->q_head_stride >= 0 && p->k_page_stride >= 0 && p->k_row_stride >= 0 && p->k_head_stride >= 0 &&
                  p->v_page_stride >= 0 && p->v_row_stride >= 0 && p->v_head_stride >= 0, "attn_paged: negative stride");
    SANIC_REQUIRE(ctx, p->n_requests <= 1 || p->table_stride >= p->max_pages, "attn_paged: table rows overlap");
    return SANIC_OK;
}
}  // namespace

namespace {
// a: the rows form's launch with n_a CTAs, b: the tensor-memory form's; 0 CTAs: not launched
cudaError_t launch_merge(int sm_count, const Params& a, int n_a, const Params& b, int n_b, int max_query_len, int D, int dtype, cudaStream_t st) {
    const int split = std::max(1, a.rows / 16), n_first = n_a * split;
    Look look{};
    if (n_b && b.n_tokens > 1) {       // (a token alone hides nothing)
        const int longest = std::min(max_query_len ? max_query_len : INT32_MAX, b.n_tokens), items = (longest + b.block_tokens - 1) / b.block_tokens;
        look.split = std::max(1, (b.window == 0 ? items : b.window >= b.block_tokens ? 2 * items : longest) / CHECKS);
        look.units = (long long)b.n_requests * b.kv_heads * look.split;
        look.blocks = (int)std::min<long long>((look.units + 15) / 16, 2 * sm_count);
        look.few = n_a ? a.rows_upto : 0; look.tokens_few = n_a ? a.block_tokens : 1; look.tokens_many = b.block_tokens;
    }
    Params p = b;
    p.rows_above = 0; p.rows_upto = INT32_MAX;
    const dim3 grid(look.blocks + n_first + n_b * TC_MERGE_SPLIT), block(512);
    const Merge x{a.ws_o, a.ws_ml, a.ws_merge, a.rows, n_a}, y{b.ws_o, b.ws_ml, b.ws_merge, b.rows, n_b};
    auto go = [&](auto kernel) { return launch_pdl(kernel, grid, block, 0, st, p, x, y, look, n_first, split); };
    auto of = [&](auto d, auto bf16) { return look.blocks ? go(paged_merge_kernel<d.value, bf16.value, true>) : go(paged_merge_kernel<d.value, bf16.value, false>); };
    using std::integral_constant;
    if (D == 128) return dtype == SANIC_BF16 ? of(integral_constant<int, 128>{}, std::true_type{}) : of(integral_constant<int, 128>{}, std::false_type{});
    return dtype == SANIC_BF16 ? of(integral_constant<int, 64>{}, std::true_type{}) : of(integral_constant<int, 64>{}, std::false_type{});
}
}  // namespace

extern "C" {

size_t sanic_attn_paged_workspace_bytes(sanic_ctx* ctx, const sanic_attn_paged_params* p) {
    if (!ctx || !p || validate(ctx, p) != SANIC_OK) return 0;
    return workspace_bytes(make_plan(ctx, p), p->head_dim);
}

int32_t sanic_attn_paged(sanic_ctx* ctx, const sanic_attn_paged_params* p, void* stream) {
    if (!ctx || !p) return SANIC_ERR_INVALID;
    int32_t rc = validate(ctx, p);
    if (rc != SANIC_OK) return rc;
    if (p->n_requests == 0 || p->n_tokens == 0) return SANIC_OK;
    const Plan pl = make_plan(ctx, p);
    SANIC_REQUIRE(ctx, p->workspace && ((uintptr_t)p->workspace % 16) == 0 && p->workspace_bytes >= workspace_bytes(pl, p->head_dim),
                  "attn_paged: the workspace must be 16-byte aligned and of sanic_attn_paged_workspace_bytes()");
    sanic_set_device(ctx);
    Params q{};
    q.q = p->q; q.out = p->out; q.lse = p->lse; q.k = p->k_pages; q.v = p->v_pages;
    q.table = p->block_table; q.query_start = p->query_start; q.kv_lens = p->kv_lens;
    q.q_token_stride = p->q_token_stride; q.q_head_stride = p->q_head_stride;
    q.k_page_stride = p->k_page_stride; q.k_row_stride = p->k_row_stride; q.k_head_stride = p->k_head_stride;
    q.v_page_stride = p->v_page_stride; q.v_row_stride = p->v_row_stride; q.v_head_stride = p->v_head_stride;
    q.table_stride = p->table_stride;
    q.n_requests = p->n_requests; q.n_tokens = p->n_tokens; q.q_heads = p->q_heads; q.kv_heads = p->kv_heads; q.group = p->q_heads / p->kv_heads;
    q.page_size = p->page_size; q.n_pages = p->n_pages; q.max_pages = p->max_pages; q.scale = p->scale;
    q.window = p->window < (long long)p->max_pages * p->page_size ? p->window : 0;      // wider than a table row: it hides nothing
    q.page_shift = -1;
    for (int i = 0; i < 31; ++i) if ((1 << i) == p->page_size) q.page_shift = i;
    q.rows_upto = INT32_MAX;
    Params t = q;             // the tensor-memory form's launch
    unsigned char* ws = (unsigned char*)p->workspace;
    cudaStream_t st = (cudaStream_t)stream;
    if (pl.rows) {
        ws = place(q, ws, pl.rows_ctas, pl.rows, p->head_dim);
        q.block_tokens = pl.rows / q.group;
        if (pl.tc) { q.rows_upto = t.rows_above = pl.rows; t.beside = 1; }
        const bool tma = pool_supported(p, KT);
        auto launch = [&](auto mt) {
            return pl.tc ? launch_rows_any<mt.value, false>(ctx, q, p->head_dim, p->dtype, tma, pl.rows_ctas, st)
                         : launch_rows_any<mt.value, true>(ctx, q, p->head_dim, p->dtype, tma, pl.rows_ctas, st);
        };
        rc = pl.rows == 16   ? launch(std::integral_constant<int, 1>{})
             : pl.rows == 32 ? launch(std::integral_constant<int, 2>{})
                             : launch(std::integral_constant<int, 4>{});
        if (rc != SANIC_OK) return rc;
    }
    if (pl.tc) {
        place(t, ws, pl.tc_ctas, TC_ROWS, p->head_dim);
        t.block_tokens = 2 * (128 / t.group);
        rc = tc_launch(ctx, t, p->head_dim, p->dtype, pl.tc_ctas, st);
        if (rc != SANIC_OK) return rc;
    }
    SANIC_CUDA_CHECK(ctx, launch_merge(ctx->sm_count, q, pl.rows ? pl.rows_ctas : 0, t, pl.tc ? pl.tc_ctas : 0, p->max_query_len, p->head_dim, p->dtype, st));
    return SANIC_OK;
}

}  // extern "C"
