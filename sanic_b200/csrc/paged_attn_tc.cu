// Attention of ragged chunks over a paged cache, the form for many query rows per (request, kv head): S = Q K^T and O += P V are
// tcgen05 MMAs with accumulators in tensor memory; Q, K and V arrive by TMA, keys and values one page at a time.
//
// An item (paged_sched.h) is up to 256 query rows of one (request, kv head): the heads of a group are packed next to their
// token (row = token * group + head), so a chunk of 64 tokens of a 4-head group fills both 128-row tiles and reads its keys
// once. The two tiles ping-pong on the tensor core: while one tile's softmax warpgroup turns S into P, the other tile's MMAs run.
//   warp 0       producer: page ids of a 128-key tile one tile ahead (a lane per page), then one TMA box per page and 64
//                columns; K and V tiles share one ring
//   warp 1       MMA issuer (head_dim 64: of tile 0, warp 3 of tile 1)
//   warp 2       tensor-memory allocator, then the walk over the CTA's segments: it hands them to the other warps through a ring of
//                four in shared memory, so that none of them spends registers or global loads on it
//   warps 4-7    softmax, correction and epilogue of tile 0, one thread per row;   warps 8-11 the same for tile 1
// Tensor memory, 512 columns. head_dim 64: S0 S1 | P0 P1 | O0 O1 with P in columns of its own, so the next S is computed while
// the exponentials of this one run. head_dim 128: S0 S1 | O0 O1, P over the S it came from: S(j+1) follows PV(j) in the
// tensor core's own order, and the other tile's products fill the time in between.
// Rows of V outside the keys the item sees (the tail of the last page, pages before the window) are zeroed in shared memory
// before the product, since 0 times what a page holds there may be NaN; scores of such keys are replaced, not added to.
// The rescale of O waits until a row's maximum has moved by more than 2^8 (f16: 2^4, since its weights are shifted up by 2^8
// against subnormals and must stay below 65504); after the first tile of a segment the maximum is taken inside the first
// half of the exponentials, which are redone in the rare case that it moved.
//
// Bound: 4 rows keys head_dim flop on the tensor pipe (8192 per clock and SM) against one exponential per score on the SFU (16
// per clock and SM): equal at head_dim 128, SFU-bound at 64. Measured, 32 + 8 heads, bf16, replayed from a graph: 2048 tokens over
// 30,000 keys of 128 950-960 us = 1090 TFLOP/s, 0.65 of the measured matrix-product rate (at the power cap, back to back for seconds,
// 1140); 8 prompts of 4096 of 128 1185 us = 928 TFLOP/s, of 64 1002 us = 549 TFLOP/s. A 256 x 128 block of scores takes 3840 clocks
// where either pipe needs 2048: a tile's exponentials (2000) and its products with four barrier hops (1800) follow one another, and only
// the other tile's lie over them. (Tile 0 leaving out a last key tile that only tile 1 sees: 4 % slower at head_dim 128 even so, since
// the tiles fall out of the order below; descriptors and ring places computed ahead of the issuer's waits: the same 4 %.)
#include <algorithm>

#include "paged_tma.cuh"

namespace {
using namespace sanic;
using namespace sanic::tc;
using namespace sanic::paged;

constexpr int BM = 128, BN = 128, NTHREADS = 384;

template <int D> struct Tc {
    static constexpr bool ALIAS = D == 128;            // P shares S's columns
    static constexpr int SLABS = D / 64, SLAB = BN * 128;      // 64-column slabs of 128-byte rows
    static constexpr int TILE = BN * D * 2;
    static constexpr int QBUF = D == 64 ? 2 : 1;       // query buffers across items
    static constexpr int NS = D == 64 ? 10 : 5;        // ring slots, one K or V tile each
    static constexpr int TM_S = 0, TM_P = ALIAS ? 0 : 256, P_STEP = ALIAS ? 128 : 64, TM_O = ALIAS ? 256 : 384;
    static constexpr int ISSUERS = ALIAS ? 1 : 2;      // MMA-issuing warps
    static constexpr int DATA = (2 * QBUF + NS) * TILE;
};
// A segment as the roles read it.
struct __align__(16) Work {
    int row0, n_tok;       // first token row of the item's block, tokens of it
    int b, hk, lo, hi;     // keys the item's tokens see
    int jb, je;            // the segment's key tiles
    int pos0;              // position of the block's first token
    int parts;
    int whole, slot;       // the item's only segment; else the partial slot
};
constexpr int END = -1;    // n_tok of the entry behind the last segment
// Waits for a segment last as long as the segments before it, not as one tile, and so may a wait for scores: tile 1 passes over
// segments without rows for it that tile 0 still folds, whatever their length. A limit of their own, then: 16 times that of the
// other waits (in probes, so no exact time: a sleep asked for 32 ns takes anything from none to 64). Those are for one tile
// each, and end these too when they run out.
constexpr uint32_t SEGMENT_SPINS = 1u << 28;

template <int D> struct Shared {
    uint64_t q_full[2], q_empty[2], full[Tc<D>::NS], empty[Tc<D>::NS];
    uint64_t s_full[2], s_free[2], p_half[2], p_full[2], pv_done[2], o_free[2];      // per query tile
    uint64_t seg_full[4], seg_empty[4];
    Work seg[4];
    uint32_t tmem_base;
    volatile int abort_flag;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ffma2(float& d0, float& d1, float a0, float a1, float b, float c) {
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %4};\n\tmov.b64 rc, {%5, %5};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void fadd2(float& d0, float& d1, float a0, float a1) {   // d += a
    asm("{\n\t.reg .b64 ra, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rd, {%0, %1};\n\tadd.rn.f32x2 rd, rd, ra;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "+f"(d0), "+f"(d1) : "f"(a0), "f"(a1));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
template <bool BF16> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 32 bytes to a 16-byte boundary; `wide`: to a 32-byte one
__device__ __forceinline__ void store8(void* dst, const uint32_t (&w)[8], bool wide) {
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                     "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
    } else {
        ((uint4*)dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        ((uint4*)dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
    return pred != 0;
}
// Bounded wait of a role that is ahead of the others: asks and sleeps, and leaves the issue slots of its sub-partition to the
// softmax warps (a suspended try_wait wakes and asks again often enough to cost them a tenth of their rate).
__device__ __forceinline__ bool mbar_wait_idle(uint64_t* bar, uint32_t parity, uint32_t ns, volatile int* abort_flag, int* err, int code,
                                               uint32_t limit = SPIN_LIMIT >> 2) {
    for (uint32_t it = 0; it < limit; ++it) {
        if (mbar_test(bar, parity)) return true;
        __nanosleep(ns);
        if ((it & 255u) == 255u && *abort_flag) return false;
    }
    *abort_flag = 1;
    atomicCAS(err, 0, code);
    return false;
}
__host__ __device__ constexpr uint32_t idesc_of(int M, int N, bool b_mn_major, bool bf16) {     // f16 operands: format fields 0
    return make_idesc(M, N, b_mn_major) & (bf16 ? ~0u : ~((1u << 7) | (1u << 10)));
}

struct TcArgs { int tile_tokens, box_rows, k_heads_inner, v_heads_inner; };

template <int D, bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ Params p, const TcArgs a, int* err) {
    using C = Tc<D>;
    constexpr float P_SHIFT = BF16 ? 0.0f : 8.0f, SLACK = BF16 ? 8.0f : 4.0f;
    extern __shared__ unsigned char smem_dyn[];
    const uint32_t raw = smem_u32(smem_dyn);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* aligned = smem_dyn + (base - raw);
    const uint32_t q_addr = base, ring_addr = base + 2 * C::QBUF * C::TILE;
    Shared<D>* sh = (Shared<D>*)(aligned + C::DATA);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) { mbar_init(&sh->q_full[i], 1); mbar_init(&sh->q_empty[i], C::ISSUERS); }
        for (int s = 0; s < C::NS; ++s) { mbar_init(&sh->full[s], 1); mbar_init(&sh->empty[s], C::ISSUERS); }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sh->s_full[t], 1); mbar_init(&sh->s_free[t], 4); mbar_init(&sh->p_half[t], 4); mbar_init(&sh->p_full[t], 4);
            mbar_init(&sh->pv_done[t], 1); mbar_init(&sh->o_free[t], 4);
        }
        for (int i = 0; i < 4; ++i) { mbar_init(&sh->seg_full[i], 1); mbar_init(&sh->seg_empty[i], 9 + C::ISSUERS); }      // producer, issuers, softmax
        sh->abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 2) tmem_alloc(&sh->tmem_base, 512);
    // Lengths, table, q and pages come from earlier kernels of the step. Beside a rows launch there is nothing to wait for here:
    // that one started this one behind its own wait. It is waited for at the end, so that what follows this kernel follows both.
    if (!p.beside) griddep_wait();
    griddep_launch();
    long long* cum = (long long*)(aligned + 2 * C::QBUF * C::TILE);      // the prefix sums share the ring's memory
    scan_costs<BN>(p, cum, err);
    DeviceWalk<BN> walk{LoadReq{&p, nullptr}};
    if (warp == 2) walk.init(p, cum, blockIdx.x, gridDim.x);
    fence_async_smem();      // generic accesses to the ring end before TMA writes it
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh->tmem_base;
    volatile int* abortp = &sh->abort_flag;
    const int tile_rows = a.tile_tokens * p.group;
    // The next segment of a role: every reading warp takes every entry.
    uint32_t n_seg = 0;
    auto next = [&](Work& w) {
        const int i = n_seg & 3;
        bool there = mbar_test(&sh->seg_full[i], (n_seg >> 2) & 1);
        if (!there) there = mbar_wait_idle(&sh->seg_full[i], (n_seg >> 2) & 1, 32, abortp, err, 15, SEGMENT_SPINS);
        if (!__all_sync(0xffffffffu, there)) return false;
        w = sh->seg[i];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->seg_empty[i]);
        ++n_seg;
        return w.n_tok != END;
    };
    Work s;

    // The first warpgroup gives registers to the softmax warpgroups: 128 x 72 + 256 x 216 =
    // the 64,512 the launch was given.
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
        int slot = 0; uint32_t phase = 1;
        bool ok = true;
        int n = 0;
        const int boxes = BN / a.box_rows;
        while (ok && next(s)) {
            if (s.je <= s.jb) continue;
            const int32_t* row = p.table + (int64_t)s.b * p.table_stride;
            const int tiles = s.n_tok > a.tile_tokens ? 2 : 1;
            // a lane's page of key tile j: -1 where no visible key lies in its box, n_pages (read as zeros) for a bad entry
            auto page_of = [&](int j) {
                const int key = j * BN + lane * a.box_rows;
                if (lane >= boxes || key >= s.hi || key + a.box_rows <= s.lo) return -1;
                int page, in_page;
                return locate(p, row, key, page, in_page, err) ? page : p.n_pages;
            };
            int page = page_of(s.jb);
            for (int j = s.jb; j < s.je && ok; ++j) {
                const int ahead = j + 1 < s.je ? page_of(j + 1) : -1;
                const int key = j * BN + lane * a.box_rows;
                const int in_page = p.page_shift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, page >= 0)) * a.box_rows * 128 * C::SLABS;
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    ok = __all_sync(0xffffffffu, mbar_wait_idle(&sh->empty[slot], phase, 64, abortp, err, 11));
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&sh->full[slot], bytes);
                    __syncwarp();
                    if (page >= 0) {
                        const uint32_t dst = ring_addr + slot * C::TILE + lane * a.box_rows * 128;
                        const bool inner = kv ? a.v_heads_inner : a.k_heads_inner;
                        const int y = inner ? s.hk : in_page, z = inner ? in_page : s.hk;
#pragma unroll
                        for (int c = 0; c < C::SLABS; ++c)
                            tma_load_4d(dst + c * C::SLAB, kv ? &map_v : &map_k, &sh->full[slot], c * 64, y, z, page);
                    }
                    if (++slot == C::NS) { slot = 0; phase ^= 1; }
                }
                if (ok && j == s.jb) {       // the query tiles, behind the first keys: those need not wait for the last item's last product
                    const int qb = C::QBUF == 2 ? n & 1 : 0;
                    ok = __all_sync(0xffffffffu, mbar_wait_idle(&sh->q_empty[qb], ((C::QBUF == 2 ? n >> 1 : n) & 1) ^ 1, 64, abortp, err, 10));
                    if (!ok) break;
                    if (lane == 0) {
                        mbar_expect_tx(&sh->q_full[qb], tiles * tile_rows * 128 * C::SLABS);
                        for (int t = 0; t < tiles; ++t)
                            for (int c = 0; c < C::SLABS; ++c)
                                tma_load_3d(q_addr + (qb * 2 + t) * C::TILE + c * C::SLAB, &map_q, &sh->q_full[qb], c * 64, s.hk * p.group,
                                            s.row0 + t * a.tile_tokens);
                    }
                    __syncwarp();
                }
                page = ahead;
            }
            ++n;
        }
    } else if (warp == 1 || (C::ISSUERS == 2 && warp == 3)) {
        // head_dim 128: one warp issues for both tiles, in the order PV0 QK0 PV1 QK1. Two issuers interleave on the tensor core,
        // both tiles' scores then arrive at the same moment and the tiles fall into step (softmax together, products
        // together: 4200 clocks per key tile); in one order tile 0's scores arrive while tile 1's products run, and the tiles
        // stay half a period apart. head_dim 64: the scores run one key tile ahead of the weights and the exponentials set
        // the pace, so a warp per tile waits for its own tile only (one for both: 1330 against 1000 us).
        const int t_first = __shfl_sync(0xffffffffu, warp == 3 ? 1 : 0, 0);
        const bool leader = elect_one();
        constexpr uint32_t idesc_qk = idesc_of(BM, BN, false, BF16), idesc_pv = idesc_of(BM, D, true, BF16);
        bool ok = true;
        int n = 0;
        uint32_t u_base = 0;                 // ring position of the segment's first key tile
        uint32_t n_qk[2] = {0, 0}, n_pv[2] = {0, 0};      // products issued so far
        uint32_t n_act[2] = {0, 0};          // earlier segments in which the tile had rows
        while (ok && next(s)) {
            if (s.je <= s.jb) continue;
            const bool both = s.n_tok > a.tile_tokens;
            const int last_t = both && C::ISSUERS == 1 ? 1 : t_first;      // the tile behind which this issuer hands K, V and Q back
            const int qb = C::QBUF == 2 ? n & 1 : 0;
            const uint32_t q_phase = (C::QBUF == 2 ? n >> 1 : n) & 1;
            ++n;
            auto wait_on = [&](uint64_t* bar, uint32_t parity, int code) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abortp, err, code));
            };
            auto ring_wait = [&](uint32_t u) { wait_on(&sh->full[u % C::NS], (u / C::NS) & 1, 13); };
            auto qk = [&](int t, int j) {          // K's tile has arrived
                if (!C::ALIAS && n_qk[t] > 0) wait_on(&sh->s_free[t], (n_qk[t] - 1) & 1, 17);
                if (!ok) return;
                const int slot = (u_base + 2 * (uint32_t)(j - s.jb)) % C::NS;
                const uint64_t ad = make_desc(q_addr + (qb * 2 + t) * C::TILE, 16, 1024), bd = make_desc(ring_addr + slot * C::TILE, 16, 1024);
                fence_after();
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t o = (kk >> 2) * (C::SLAB >> 4) + (kk & 3) * 2;
                        umma_f16(tmem + C::TM_S + t * BN, ad + o, bd + o, idesc_qk, kk > 0 ? 1u : 0u);
                    }
                    umma_commit(&sh->s_full[t]);
                    if (t == last_t) {
                        umma_commit(&sh->empty[slot]);
                        if (j + 1 == s.je) umma_commit(&sh->q_empty[qb]);
                    }
                }
                __syncwarp();
                ++n_qk[t];
            };
            auto pv = [&](int t, int j) {          // V's tile has arrived
                const int slot = (u_base + 2 * (uint32_t)(j - s.jb) + 1) % C::NS;
                const bool first = j == s.jb;
                const uint64_t vd = make_desc(ring_addr + slot * C::TILE, C::SLAB, 1024);
                // the first PV of a segment overwrites O: the epilogue of the tile's previous segment must have read it
                if (first && n_act[t] > 0) wait_on(&sh->o_free[t], (n_act[t] - 1) & 1, 18);
                // A = P from tensor memory: 16 keys = 8 columns per step. head_dim 128: the first 64 keys while the others' weights are
                // computed. (head_dim 64, where the exponentials set the pace, in one go: 8 sequences of 4096 keys 975 us, 999 in two.)
                if (C::ALIAS) {
                    wait_on(&sh->p_half[t], n_pv[t] & 1, 20);
                    if (!ok) return;
                    fence_after();
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < BN / 32; ++kk)
                            umma_f16_ts(tmem + C::TM_O + t * D, tmem + C::TM_P + t * C::P_STEP + 8 * kk, vd + 128 * kk, idesc_pv, (!first || kk > 0) ? 1u : 0u);
                    }
                    __syncwarp();
                }
                wait_on(&sh->p_full[t], n_pv[t] & 1, 19);
                if (!ok) return;
                fence_after();
                if (leader) {
#pragma unroll
                    for (int kk = C::ALIAS ? BN / 32 : 0; kk < BN / 16; ++kk)
                        umma_f16_ts(tmem + C::TM_O + t * D, tmem + C::TM_P + t * C::P_STEP + 8 * kk, vd + 128 * kk, idesc_pv, (!first || kk > 0) ? 1u : 0u);
                    if (!C::ALIAS || j + 1 == s.je) umma_commit(&sh->pv_done[t]);
                    if (t == last_t) umma_commit(&sh->empty[slot]);
                }
                __syncwarp();
                ++n_pv[t];
            };
            auto values = [&](int j) {             // V's tile, with nothing in its rows [0, za) and [zb, 128) but zeros
                const uint32_t u = u_base + 2 * (uint32_t)(j - s.jb) + 1;
                ring_wait(u);
                const int za = max(0, s.lo - j * BN), zb = min(BN, s.hi - j * BN);
                if (ok && (za > 0 || zb < BN)) {
                    const int n_rows = za + BN - zb;
                    for (int i = lane; i < n_rows * 8 * C::SLABS; i += 32) {
                        const int r = i / (8 * C::SLABS), c = i % (8 * C::SLABS);
                        const int rr = r < za ? r : zb + r - za;
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(ring_addr + (u % C::NS) * C::TILE + (c >> 3) * C::SLAB + rr * 128 + (c & 7) * 16), "r"(0) : "memory");
                    }
                    fence_async_smem();
                    __syncwarp();
                }
            };
            wait_on(&sh->q_full[qb], q_phase, 12);
            if (C::ISSUERS == 2 && t_first == 1 && !both) {
                // No rows for this tile: everything goes back untouched, but in step with the producer, so that no barrier is
                // ever asked for a phase more than one ahead of its own.
                if (ok && leader) mbar_arrive(&sh->q_empty[qb]);
                for (int i = 0; i < 2 * (s.je - s.jb) && ok; ++i, ++u_base) {
                    ring_wait(u_base);
                    if (ok && leader) mbar_arrive(&sh->empty[u_base % C::NS]);
                }
                continue;
            }
            ring_wait(u_base);
            if (C::ALIAS) {
                qk(0, s.jb);
                if (both) qk(1, s.jb);
                for (int j = s.jb; j < s.je && ok; ++j) {
                    const bool more = j + 1 < s.je;
                    values(j);
                    if (more) ring_wait(u_base + 2 * (uint32_t)(j + 1 - s.jb));
                    pv(0, j);
                    if (more) qk(0, j + 1);
                    if (both) {
                        pv(1, j);
                        if (more) qk(1, j + 1);
                    }
                }
            } else {
                qk(t_first, s.jb);
                for (int j = s.jb; j < s.je && ok; ++j) {
                    if (j + 1 < s.je) {
                        ring_wait(u_base + 2 * (uint32_t)(j + 1 - s.jb));
                        qk(t_first, j + 1);
                    }
                    values(j);
                    pv(t_first, j);
                }
            }
            u_base += 2 * (uint32_t)(s.je - s.jb);
            if (t_first == 0) ++n_act[0];
            if (t_first == 1 || (C::ISSUERS == 1 && both)) ++n_act[1];
        }
    } else if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int t = (warp - 4) >> 2, q4 = warp & 3, row = q4 * 32 + lane;
        const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
        const uint32_t s_tmem = tmem + lane_base + C::TM_S + t * BN;
        const uint32_t p_tmem = tmem + lane_base + C::TM_P + t * C::P_STEP;
        const uint32_t o_tmem = tmem + lane_base + C::TM_O + t * D;
        const float sl2 = p.scale * LOG2E;
        const int row_tok = row / p.group, row_head = row - row_tok * p.group;
        uint32_t n_it = 0, n_act = 0;        // key tiles folded, segments served by this tile so far
        bool ok = true, scores_ready = false;
        while (ok && next(s)) {
            const int n_tok = s.n_tok;
            const int tok = t * a.tile_tokens + row_tok;
            const bool valid = row < tile_rows && tok < n_tok;
            if (t == 1 && n_tok <= a.tile_tokens) continue;
            const bool empty = s.je <= s.jb;
            const int64_t at = (int64_t)(s.row0 + tok) * p.q_heads + s.hk * p.group + row_head;
            float m = -INFINITY, l = 0.0f;
            const int pos = s.pos0 + tok;
            const int khi = valid ? max(0, pos + 1) : 0, klo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
            // key tiles from inner_lo to inner_hi are seen whole by every row of the tile
            const int tile_pos = s.pos0 + t * a.tile_tokens;
            const int inner_hi = tile_pos + 1;
            const int inner_lo = p.window > 0 ? tile_pos + a.tile_tokens - p.window : 0;
            const bool busy = __any_sync(0xffffffffu, valid);      // a warp without rows only keeps the barriers' count
            for (int j = s.jb; j < s.je && ok; ++j, ++n_it) {
                const bool first = j == s.jb;
                if (!scores_ready) ok = mbar_wait(&sh->s_full[t], n_it & 1, abortp, err, 21, SEGMENT_SPINS);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                scores_ready = false;
                fence_after();
                if (!busy) {
                    fence_before();
                    __syncwarp();
                    if (!C::ALIAS) {
                        if (lane == 0) mbar_arrive(&sh->s_free[t]);
                        // P(j)'s arrival may not count for P(j - 1), which the other warps may still be writing: in step with them
                        ok = __all_sync(0xffffffffu, n_it == 0 || mbar_wait(&sh->pv_done[t], (n_it - 1) & 1, abortp, err, 24));
                        if (!ok) break;
                    }
                    if (lane == 0) {
                        if (C::ALIAS) mbar_arrive(&sh->p_half[t]);
                        mbar_arrive(&sh->p_full[t]);
                    }
                    continue;
                }
                const int k0 = j * BN;
                const bool edge = k0 + BN > inner_hi || k0 < inner_lo;
                uint32_t r[BN];
#pragma unroll
                for (int c = 0; c < BN / 32; ++c) tmem_ld32_nowait(s_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]));
                tmem_ld_wait();
                if (!C::ALIAS) {
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->s_free[t]);        // S is in registers
                }
                if (edge) {        // 32 columns at a time, where an edge of some row's is
                    const int hi = khi - k0, lo = klo - k0;
#pragma unroll
                    for (int c = 0; c < BN; c += 32) {
                        if (k0 + c + 32 <= inner_hi && k0 + c >= inner_lo) continue;
                        if (p.window > 0) {
#pragma unroll
                            for (int i = c; i < c + 32; ++i) if (!(i >= lo && i < hi)) r[i] = 0xFF800000u;      // -inf
                        } else {
#pragma unroll
                            for (int i = c; i < c + 32; ++i) if (!(i < hi)) r[i] = 0xFF800000u;
                        }
                    }
                }
                const bool spec = !first;
                float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                float alpha = 1.0f;
                bool need = false;
                auto new_reference = [&]() {
                    const float mx = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3]));
                    const float m_cand = fmaxf(m, mx * sl2);
                    need = valid && ((m_cand - m > SLACK) || (!(m > -INFINITY) && m_cand > -INFINITY));
                    if (need) { alpha = (m > -INFINITY) ? ex2(m - m_cand) : 0.0f; m = m_cand; }
                };
                if (!spec) {
#pragma unroll
                    for (int i = 0; i < BN; i += 8) {
                        mxs[0] = max3(mxs[0], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                        mxs[1] = max3(mxs[1], __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
                        mxs[2] = max3(mxs[2], __uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
                        mxs[3] = max3(mxs[3], __uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
                    }
                    new_reference();
                }
                float msub = ((m > -INFINITY) ? m : 0.0f) - P_SHIFT;
                const bool pv_ready = !C::ALIAS && n_it > 0 && mbar_test(&sh->pv_done[t], (n_it - 1) & 1);
                float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                uint32_t pk[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    if (spec) {     // the row maximum of all 128 scores, four per step
                        mxs[0] = max3(mxs[0], __uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]));
                        mxs[1] = max3(mxs[1], __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
                    }
                    float x0, x1;
                    ffma2(x0, x1, __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), sl2, -msub);
                    const float p0 = ex2(x0), p1 = ex2(x1);
                    fadd2(sums[(2 * i) & 7], sums[(2 * i + 1) & 7], p0, p1);
                    pk[i] = pack2<BF16>(p0, p1);
                }
                if (spec) {
                    new_reference();
                    if (__any_sync(0xffffffffu, need)) {       // some row's reference moved: the half is taken again
                        msub = ((m > -INFINITY) ? m : 0.0f) - P_SHIFT;
#pragma unroll
                        for (int i = 0; i < 8; ++i) sums[i] = 0.0f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            float x0, x1;
                            ffma2(x0, x1, __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), sl2, -msub);
                            const float p0 = ex2(x0), p1 = ex2(x1);
                            fadd2(sums[(2 * i) & 7], sums[(2 * i + 1) & 7], p0, p1);
                            pk[i] = pack2<BF16>(p0, p1);
                        }
                    }
                }
                // Before P or O is written the previous PV of this tile must be done. With P over S it is: S(j) was computed
                // behind it, and its commit covered both.
                if (!C::ALIAS && n_it > 0) {
                    if (!pv_ready) ok = mbar_wait_spin(&sh->pv_done[t], (n_it - 1) & 1, abortp, err, 22);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    fence_after();
                }
                if (!first && __any_sync(0xffffffffu, need)) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(o_tmem + c * 32, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st32(o_tmem + c * 32, o);
                    }
                }
                tmem_st32(p_tmem, pk);
                if (!C::ALIAS) scores_ready = (j + 1 < s.je) && mbar_test(&sh->s_full[t], (n_it + 1) & 1);
#pragma unroll
                for (int i = 32; i < 64; ++i) {
                    float x0, x1;
                    ffma2(x0, x1, __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), sl2, -msub);
                    const float p0 = ex2(x0), p1 = ex2(x1);
                    fadd2(sums[(2 * i) & 7], sums[(2 * i + 1) & 7], p0, p1);
                    r[i] = pack2<BF16>(p0, p1);
                    if (C::ALIAS && i == 36) {        // by now the first half has landed: its product may start
                        tmem_st_wait();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh->p_half[t]);
                    }
                }
                tmem_st32(p_tmem + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
                l = l * alpha + (((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7])));
                tmem_st_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->p_full[t]);
            }
            if (!ok) break;
            uint32_t o[D];
            if (!empty) {
                ok = __all_sync(0xffffffffu, mbar_wait_spin(&sh->pv_done[t], ((C::ALIAS ? n_act : n_it - 1)) & 1, abortp, err, 23));
                if (!ok) break;
                ++n_act;
                fence_after();
#pragma unroll
                for (int c = 0; c < D / 32; ++c) tmem_ld32_nowait(o_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&o[c * 32]));
                tmem_ld_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->o_free[t]);
            } else {
#pragma unroll
                for (int i = 0; i < D; ++i) o[i] = 0u;
            }
            if (!valid) continue;
            if (s.whole) {
                const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;      // no visible key: zeros, and -inf for the log-sum-exp
                uint16_t* dst = (uint16_t*)p.out + at * D;
                const bool wide = ((uintptr_t)p.out & 31) == 0;
                if (!(l != 0.0f)) {
#pragma unroll
                    for (int i = 0; i < D; ++i) o[i] = 0u;                   // every weight of the row was 0: V's zero rows and NaN alike
                }
#pragma unroll
                for (int q = 0; q < D / 16; ++q) {
                    uint32_t wv[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        wv[j] = pack2<BF16>(__uint_as_float(o[16 * q + 2 * j]) * inv, __uint_as_float(o[16 * q + 2 * j + 1]) * inv);
                    store8(dst + q * 16, wv, wide);
                }
                if (p.lse) p.lse[at] = (m + log2f(l) - P_SHIFT) * LN2;
            } else {
                const size_t r = (size_t)s.slot * p.rows + t * tile_rows + row;
                float* dst = p.ws_o + r * D;
                const bool wide = ((uintptr_t)p.ws_o & 31) == 0;
#pragma unroll
                for (int q = 0; q < D / 8; ++q) store8(dst + q * 8, *reinterpret_cast<uint32_t(*)[8]>(&o[8 * q]), wide);
                p.ws_ml[r] = make_float2(m, l);
            }
        }
    } else if (warp == 2) {
        int4 merge = make_int4(0, 0, 0, 0);
        Seg g;
        for (bool more = true; more; ++n_seg) {
            more = walk.next(p, g);
            const int i = n_seg & 3;
            if (!__all_sync(0xffffffffu, mbar_wait_idle(&sh->seg_empty[i], ((n_seg >> 2) & 1) ^ 1, 256, abortp, err, 16, SEGMENT_SPINS))) break;
            if (lane == 0) {
                Work w{};
                w.n_tok = END;
                if (more) {
                    const int block0 = g.rb * p.block_tokens;
                    w.row0 = g.r.q0 + block0; w.n_tok = min(p.block_tokens, g.r.qn - block0);
                    w.b = g.b; w.hk = g.hk; w.lo = g.lo; w.hi = g.hi; w.jb = g.jb; w.je = g.je;
                    w.pos0 = g.r.kv - g.r.qn + block0; w.parts = g.parts;
                    w.whole = g.starts && g.finishes; w.slot = (int)partial_slot(g, blockIdx.x);
                    if (g.parts > 1) merge = make_int4(w.row0, w.n_tok, g.hk, g.parts);
                }
                sh->seg[i] = w;
                mbar_arrive(&sh->seg_full[i]);
            }
            __syncwarp();
        }
        if (lane == 0) p.ws_merge[blockIdx.x] = merge;
    }
    fence_before();
    __syncthreads();
    if (warp == 2) { fence_after(); tmem_dealloc(tmem, 512); }
    if (p.beside) griddep_wait();
}

template <int D, bool BF16>
int32_t launch(sanic_ctx* ctx, const Params& p, int ctas, cudaStream_t st) {
    using C = Tc<D>;
    TcArgs a{};
    a.tile_tokens = p.block_tokens / 2;
    a.box_rows = box_rows_of(p.page_size, BN);
    CUtensorMap mq, mk, mv;
    {
        const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.q_heads, (cuuint64_t)p.n_tokens};
        const int64_t strides[2] = {p.q_heads == 1 ? D : p.q_head_stride, p.q_token_stride};
        const cuuint32_t box[3] = {64, (cuuint32_t)p.group, (cuuint32_t)a.tile_tokens};
        const int32_t rc = encode_map(ctx, &mq, BF16, p.q, 3, dims, strides, box);
        if (rc != SANIC_OK) return rc;
    }
    for (int kv = 0; kv < 2; ++kv) {
        bool inner;
        const int32_t rc = encode_pool(ctx, kv ? &mv : &mk, BF16, p, kv, D, a.box_rows, &inner);
        if (rc != SANIC_OK) return rc;
        (kv ? a.v_heads_inner : a.k_heads_inner) = inner;
    }
    const int smem = C::DATA + (int)sizeof(Shared<D>) + 1024;
    static_assert(C::NS * C::TILE >= (MAX_REQUESTS + 1) * 8, "prefix sums fit the ring");
    static thread_local int ready_on = -1;
    if (ready_on != ctx->device) {
        SANIC_CUDA_CHECK(ctx, cudaFuncSetAttribute(paged_tc_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        ready_on = ctx->device;
    }
    SANIC_CUDA_CHECK(ctx, launch_pdl(paged_tc_kernel<D, BF16>, dim3(ctas), dim3(NTHREADS), smem, st, mq, mk, mv, p, a, ctx->status_dev));
    return SANIC_OK;
}
}  // namespace

namespace sanic {
namespace paged {
// The page pool as TMA needs it, and the heads of a group side by side within a token. Other layouts are served by the rows form.
bool tc_supported(const sanic_attn_paged_params* p) {
    if (!pool_supported(p, BN)) return false;
    const int64_t hs = p->q_heads == 1 ? p->head_dim : p->q_head_stride;
    return hs >= p->head_dim && (p->n_tokens == 1 || (p->q_token_stride % hs == 0 && p->q_token_stride >= hs)) && p->q_token_stride < (1ll << 38) && p->q_token_stride > 0;
}
int32_t tc_launch(sanic_ctx* ctx, const Params& p, int head_dim, int dtype, int ctas, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    if (head_dim == 128) return dtype == SANIC_BF16 ? launch<128, true>(ctx, p, ctas, st) : launch<128, false>(ctx, p, ctas, st);
    return dtype == SANIC_BF16 ? launch<64, true>(ctx, p, ctas, st) : launch<64, false>(ctx, p, ctas, st);
}
}  // namespace paged
}  // namespace sanic
