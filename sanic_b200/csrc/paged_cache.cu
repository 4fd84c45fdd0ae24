// The two bookkeeping operators of a paged cache: page tables and slots from request lengths, and the write of a step's keys
// and values (with RoPE of q and k) into their slots.
#include <algorithm>

#include "paged.cuh"

namespace {
using namespace sanic;
using namespace sanic::paged;

// ── page_table_append ──
// Two running sums over the requests (pages taken, tokens) place everything: page j of request b's taken ones is
// free[F - 1 - (taken before b) - j], token i of b is row (tokens before b) + i. Up to 8000 requests fit one block's shared
// memory, so every block takes the sums itself and then fills its own slice of the token rows, the table entries and the
// per-request outputs: one launch, no hand-over between blocks, and the time of a decode step is the latency of two
// dependent loads and a scan. Bytes only start to matter for the slots and positions of whole prompts (12 per token).
// From a graph: 256 requests of one token 6.3 us, 48 prompts of 124,750 tokens together 8.3 us.
constexpr int AT = 512;      // threads of a block
constexpr int append_smem(int n_requests) { return (2 * n_requests + 2) * 4; }

struct AppendShared { int warp_pages[AT / 32], warp_tokens[AT / 32]; };

// Pages that a row holds, inside the row; `bad` is set where the count given was not.
__device__ __forceinline__ int held_of(const sanic_page_append_params& p, int b, int seq, bool& bad) {
    const int h = p.held_pages ? p.held_pages[b] : (int)(((long long)seq + p.page_size - 1) / p.page_size);
    const int inside = min(max(h, 0), p.max_pages);
    bad |= inside != h;
    return inside;
}
__device__ __forceinline__ int held_of(const sanic_page_append_params& p, int b, int seq) {
    bool reported = false;
    return held_of(p, b, seq, reported);
}

__global__ void __launch_bounds__(AT) page_append_kernel(const sanic_page_append_params p, int* err) {
    extern __shared__ int s_dyn[];
    int* s_tok = s_dyn;                          // [n + 1] token rows before request b, clamped to n_tokens
    int* s_pg = s_dyn + p.n_requests + 1;        // [n + 1] pages taken before request b
    __shared__ AppendShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.n_requests;
    griddep_wait();
    griddep_launch();
    const int free_given = *p.free_count, free_n = min(max(free_given, 0), p.free_capacity);
    long long tok_carry = 0, pg_carry = 0;
    bool bad = free_n != free_given;
    if (tid == 0) { s_tok[0] = 0; s_pg[0] = 0; }
    for (int b0 = 0; b0 < n; b0 += AT) {
        const int b = b0 + tid;
        int tok = 0, pg = 0;
        if (b < n) {
            const int seq = p.seq_lens[b], add = p.new_lens[b];
            bad |= seq < 0 || add < 0;
            tok = min(max(add, 0), p.n_tokens + 1);      // more than the token rows there are: reported below, and the sums stay small
            const long long need = ((long long)max(seq, 0) + max(add, 0) + p.page_size - 1) / p.page_size;
            bad |= need > p.max_pages;
            pg = max(0, (int)min(need, (long long)p.max_pages) - held_of(p, b, max(seq, 0), bad));
        }
        int ct = tok, cp = pg;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, ct, o), y = __shfl_up_sync(0xffffffffu, cp, o);
            if (lane >= o) { ct = (int)min((long long)ct + x, 1ll << 30); cp = (int)min((long long)cp + y, 1ll << 30); }
        }
        if (lane == 31) { sh.warp_tokens[warp] = ct; sh.warp_pages[warp] = cp; }
        __syncthreads();
        long long bt = tok_carry, bp = pg_carry, at = 0, ap = 0;
        for (int w = 0; w < AT / 32; ++w) {
            if (w < warp) { bt += sh.warp_tokens[w]; bp += sh.warp_pages[w]; }
            at += sh.warp_tokens[w]; ap += sh.warp_pages[w];
        }
        if (b < n) {
            s_tok[b + 1] = (int)min(bt + ct, (long long)p.n_tokens);
            s_pg[b + 1] = (int)min(bp + cp, 1ll << 30);      // a free list holds no more: what is beyond gets no pages
            bad |= bt + ct > p.n_tokens || bp + cp > free_n;
        }
        tok_carry += at; pg_carry += ap;
        __syncthreads();
    }
    __syncthreads();

    const int stride = gridDim.x * AT, first = blockIdx.x * AT + tid;
    for (int b = first; b < n; b += stride) {
        const int seq = max(p.seq_lens[b], 0), add = max(p.new_lens[b], 0), held = held_of(p, b, seq);
        const int got = min(max(free_n - s_pg[b], 0), s_pg[b + 1] - s_pg[b]);
        p.query_start[b + 1] = s_tok[b + 1];
        p.kv_lens[b] = (int)min((long long)seq + add, (long long)INT32_MAX);
        p.pages_out[b] = held + got;
    }
    if (first == 0) {
        p.query_start[0] = 0;
        *p.free_count_out = (int)max(0ll, (long long)free_n - pg_carry);
    }
    bad &= blockIdx.x == 0;                      // every block found the same so far
    // the r-th page taken; -1 where the list ends before it or holds no page there
    auto taken_page = [&](int r) { return r < free_n ? max(p.free_pages[free_n - 1 - r], -1) : -1; };
    // table entries: the taken pages of all requests, in order
    const int taken = s_pg[n];
    for (int r = first; r < taken; r += stride) {
        int lo = 0, hi = n - 1;                  // the last request with s_pg[b] <= r
        while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (s_pg[mid] <= r) lo = mid; else hi = mid - 1; }
        const int col = held_of(p, lo, max(p.seq_lens[lo], 0)) + r - s_pg[lo];
        const int page = taken_page(r);
        bad |= page < 0;
        p.block_table[(int64_t)lo * p.table_stride + col] = page;
    }
    // token rows
    const int used = s_tok[n];
    for (int t = first; t < p.n_tokens; t += stride) {
        long long pos = 0, slot = -1;            // 64 bits: a length near 2^31 must not wrap into a page index
        if (t < used) {
            int lo = 0, hi = n - 1;              // the last request with s_tok[b] <= t
            while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (s_tok[mid] <= t) lo = mid; else hi = mid - 1; }
            const int seq = max(p.seq_lens[lo], 0), held = held_of(p, lo, seq);
            pos = (long long)seq + t - s_tok[lo];
            const long long idx = pos / p.page_size;
            int page = -1;
            if (idx < held) page = p.block_table[(int64_t)lo * p.table_stride + idx];      // entries of earlier steps: nobody writes them here
            else if (idx < p.max_pages) page = taken_page(s_pg[lo] + (int)idx - held);
            bad |= page < 0;
            if (page >= 0) slot = (long long)page * p.page_size + pos - idx * p.page_size;
        }
        p.positions[t] = (int)min(pos, (long long)INT32_MAX);
        p.slots[t] = slot;
    }
    if (bad && err) atomicCAS(err, 0, STATUS_POOL);
}

// ── paged_cache_write ──
// Bytes: every source element read once, every rotated or copied one written once. A thread takes 8 neighbouring elements of
// the first half of a head's row and their 8 partners of the second half (16-byte accesses on both sides), for HP heads of its
// token: the eight (cos, sin) pairs stay in registers and 2 HP loads are in flight. The heads of q, k and v lie side by side
// in the order of threads.
struct Bf16 {};
struct F16 {};
__device__ __forceinline__ uint4 ldg16(const void* p) { return __ldcs((const uint4*)p); }      // read once
__device__ __forceinline__ float f16_to_f32(uint16_t h) { float f; asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"(h)); return f; }
// eight neighbouring elements as loaded, and widened
template <typename T> struct Raw {
    uint4 w;
    __device__ __forceinline__ void load(const void* base, int64_t at) { w = ldg16((const uint16_t*)base + at); }
    __device__ __forceinline__ void widen(float (&x)[8]) const {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (__is_same(T, Bf16)) { x[2 * i] = bf16lo(v[i]); x[2 * i + 1] = bf16hi(v[i]); }
            else { x[2 * i] = f16_to_f32((uint16_t)(v[i] & 0xffffu)); x[2 * i + 1] = f16_to_f32((uint16_t)(v[i] >> 16)); }
        }
    }
};
template <> struct Raw<float> {
    uint4 w, z;
    __device__ __forceinline__ void load(const void* base, int64_t at) { w = ldg16((const float*)base + at); z = ldg16((const float*)base + at + 4); }
    __device__ __forceinline__ void widen(float (&x)[8]) const {
        x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
        x[4] = __uint_as_float(z.x); x[5] = __uint_as_float(z.y); x[6] = __uint_as_float(z.z); x[7] = __uint_as_float(z.w);
    }
};
template <bool BF16> __device__ __forceinline__ void store8(void* base, int64_t at, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (BF16) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    }
    *(uint4*)((uint16_t*)base + at) = make_uint4(w[0], w[1], w[2], w[3]);
}

// A resident grid walks the tokens: the slot and position of a thread's next token are asked for under the rows of this one, so a
// token costs one latency after the other only for its rows and rotation, which are asked for together.
// HP heads per thread, WT threads per block. 8191 tokens of 32 + 2 * 8 heads of 128, f16 (206 MB): 36.9 us = 5.6 TB/s, 0.85 of the
// measured copy rate; 41.7 us with a block per token (its slot, position, rotation in turn), 39.0 us with blocks of 256, 41.0 us with
// four heads and four blocks per SM, 38.8 us with four times the resident blocks. From f32 (302 MB, 122 registers, four blocks per SM): 51.6
// us = 5.9 TB/s, 0.91. (Stores marked as streaming: 35.8 us; not taken, since attention
// reads q and the new keys next.)
constexpr int HP = 3, WT = 128;
template <typename S> constexpr int write_blocks() { return sizeof(Raw<S>) == 16 ? 5 : 4; }      // resident per SM

template <typename S, bool BF16>
__global__ void __launch_bounds__(WT, write_blocks<S>()) paged_write_kernel(const __grid_constant__ sanic_paged_write_params p, const int tokens_per_block, const int page_shift, int* err) {
    const int per_head = p.head_dim / 16, nq = p.q ? p.q_heads : 0, heads = nq + 2 * p.kv_heads, half = p.head_dim / 2;
    const int groups = (heads + HP - 1) / HP, per_token = groups * per_head;      // threads of a token
    const int passes = (tokens_per_block * per_token + WT - 1) / WT;              // of a block over its tokens: more than one where one has many heads
    const int64_t n_work = (int64_t)((p.n_tokens + tokens_per_block - 1) / tokens_per_block) * passes;
    griddep_wait();
    griddep_launch();
    // this thread's token and part of it in pass w, and what the row's address and rotation depend on
    auto token = [&](int64_t w, int& rem) -> int64_t {
        const int64_t g = passes == 1 ? w : w / passes;
        const int i = threadIdx.x + (passes == 1 ? 0 : (int)(w - g * passes) * WT), tl = i / per_token;
        rem = i - tl * per_token;
        const int64_t t = g * tokens_per_block + tl;
        return w < n_work && tl < tokens_per_block && t < p.n_tokens ? t : -1;
    };
    int64_t w = blockIdx.x;
    int rem;
    int64_t t = token(w, rem);
    int64_t slot = t >= 0 ? p.slots[t] : -1;
    int pos = t >= 0 && p.table ? p.positions[t] : 0;
    for (; w < n_work; w += gridDim.x) {
        const int hg = rem / per_head, c = (rem - hg * per_head) * 8;
        Raw<S> a_raw[HP], b_raw[HP];
        bool ok = slot >= 0;
        if (ok && (slot >= (int64_t)p.n_pages * p.page_size || (p.table && (unsigned)pos >= (unsigned)p.n_positions))) {
            if (rem == 0 && err) atomicCAS(err, 0, STATUS_WRITE);
            ok = false;
        }
        if (ok) {
#pragma unroll
            for (int u = 0; u < HP; ++u) {
                const int hh = hg + u * groups;
                if (hh >= heads) continue;
                const bool is_q = hh < nq, is_k = !is_q && hh < nq + p.kv_heads;
                const void* src = is_q ? p.q : is_k ? p.k : p.v;
                const int64_t at = t * (is_q ? p.q_stride : is_k ? p.k_stride : p.v_stride) + (int64_t)(hh - (is_q ? 0 : is_k ? nq : nq + p.kv_heads)) * p.head_dim + c;
                a_raw[u].load(src, at); b_raw[u].load(src, at + half);
            }
        }
        float cs[16];
        if (ok && p.table) {
            const float4* x = (const float4*)(p.table + ((int64_t)pos * half + c) * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) { const float4 y = __ldg(x + i); cs[4 * i] = y.x; cs[4 * i + 1] = y.y; cs[4 * i + 2] = y.z; cs[4 * i + 3] = y.w; }
        }
        // the next token's, under this one's rows
        const int64_t t_now = t, slot_now = slot;
        int rem_next;
        t = token(w + gridDim.x, rem_next);
        slot = t >= 0 ? p.slots[t] : -1;
        pos = t >= 0 && p.table ? p.positions[t] : 0;
        rem = rem_next;
        if (!ok) continue;
        const int64_t page = page_shift >= 0 ? slot_now >> page_shift : (slot_now >> 32) == 0 ? (int64_t)((uint32_t)slot_now / (uint32_t)p.page_size) : slot_now / p.page_size;
        const int64_t row = slot_now - page * p.page_size;
#pragma unroll
        for (int u = 0; u < HP; ++u) {
            const int hh = hg + u * groups;
            if (hh >= heads) continue;
            const bool is_q = hh < nq, is_k = !is_q && hh < nq + p.kv_heads;
            float a[8], b[8];
            a_raw[u].widen(a); b_raw[u].widen(b);
            if (p.table && (is_q || is_k)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = a[i], y = b[i];
                    a[i] = x * cs[2 * i] - y * cs[2 * i + 1]; b[i] = y * cs[2 * i] + x * cs[2 * i + 1];
                }
            }
            void* dst = is_q ? p.q_out : is_k ? p.k_pages : p.v_pages;
            const int64_t at = is_q ? t_now * p.q_out_stride + (int64_t)hh * p.head_dim + c
                             : is_k ? page * p.k_page_stride + row * p.k_row_stride + (int64_t)(hh - nq) * p.k_head_stride + c
                                    : page * p.v_page_stride + row * p.v_row_stride + (int64_t)(hh - nq - p.kv_heads) * p.v_head_stride + c;
            store8<BF16>(dst, at, a); store8<BF16>(dst, at + half, b);
        }
    }
}

bool overlaps(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && x < y + nb && y < x + na;
}
}  // namespace

extern "C" {

int32_t sanic_page_table_append(sanic_ctx* ctx, const sanic_page_append_params* p, void* stream) {
    if (!ctx || !p) return SANIC_ERR_INVALID;
    SANIC_REQUIRE(ctx, p->n_requests >= 0 && p->n_tokens >= 0 && p->free_capacity >= 0, "page_table_append: negative count");
    SANIC_REQUIRE(ctx, p->n_requests <= MAX_REQUESTS, "page_table_append: at most 8000 requests per call");
    SANIC_REQUIRE(ctx, p->n_tokens < (1 << 30), "page_table_append: too many token rows");
    SANIC_REQUIRE(ctx, p->page_size > 0 && p->max_pages > 0, "page_table_append: empty pages or table rows");
    SANIC_REQUIRE(ctx, p->max_pages <= (1 << 30) && p->free_capacity <= (1 << 30), "page_table_append: too many pages");
    SANIC_REQUIRE(ctx, p->free_count && p->query_start && p->free_count_out, "page_table_append: null scalar or query_start");
    SANIC_REQUIRE(ctx, p->n_requests == 0 || (p->seq_lens && p->new_lens && p->block_table && p->kv_lens && p->pages_out),
                  "page_table_append: null tensor");
    SANIC_REQUIRE(ctx, p->n_tokens == 0 || (p->positions && p->slots), "page_table_append: null token rows");
    SANIC_REQUIRE(ctx, p->free_capacity == 0 || p->free_pages, "page_table_append: null free list");
    SANIC_REQUIRE(ctx, p->n_requests <= 1 || p->table_stride >= p->max_pages, "page_table_append: table rows overlap");
    // every block reads the inputs while others write the outputs
    const size_t nb = (size_t)p->n_requests * 4;
    const struct { const void* ptr; size_t n; } in[] = {{p->seq_lens, nb}, {p->new_lens, nb}, {p->held_pages, nb}, {p->free_pages, (size_t)p->free_capacity * 4},
                                                        {p->free_count, 4}, {p->block_table, p->n_requests ? ((size_t)(p->n_requests - 1) * p->table_stride + p->max_pages) * 4 : 0}},
                   out[] = {{p->query_start, nb + 4}, {p->kv_lens, nb}, {p->pages_out, nb}, {p->free_count_out, 4}, {p->positions, (size_t)p->n_tokens * 4},
                            {p->slots, (size_t)p->n_tokens * 8}};
    for (const auto& o : out)
        for (const auto& i : in) SANIC_REQUIRE(ctx, !overlaps(o.ptr, o.n, i.ptr, i.n), "page_table_append: an output overlaps an input");
    for (int i = 0; i < 5; ++i)
        SANIC_REQUIRE(ctx, !overlaps(in[5].ptr, in[5].n, in[i].ptr, in[i].n), "page_table_append: the table overlaps an input");
    sanic_set_device(ctx);
    // The limit is the largest batch's for every call: it is one value per function and device, so a call that set it to its own size
    // could lower it between another thread's set and launch; and static shared memory counts towards the 48 KB that need none.
    static thread_local int ready_on = -1;
    if (ready_on != ctx->device) {
        SANIC_CUDA_CHECK(ctx, cudaFuncSetAttribute(page_append_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, append_smem(MAX_REQUESTS)));
        ready_on = ctx->device;
    }
    const int smem = append_smem(p->n_requests);
    // a block's slice: about four token rows or requests per thread, at most two blocks per SM
    const long long rows = std::max<long long>(p->n_tokens, p->n_requests);
    const int blocks = (int)std::min<long long>(std::max<long long>(1, (rows + 4 * AT - 1) / (4 * AT)), 2 * ctx->sm_count);
    SANIC_CUDA_CHECK(ctx, launch_pdl(page_append_kernel, dim3(blocks), dim3(AT), smem, (cudaStream_t)stream, *p, ctx->status_dev));
    return SANIC_OK;
}

int32_t sanic_paged_cache_write(sanic_ctx* ctx, const sanic_paged_write_params* p, void* stream) {
    if (!ctx || !p) return SANIC_ERR_INVALID;
    SANIC_REQUIRE(ctx, p->n_tokens >= 0 && p->kv_heads > 0 && p->q_heads >= 0, "paged_cache_write: bad counts");
    if (p->head_dim <= 0 || p->head_dim % 16 || p->head_dim > 256)
        return sanic_fail(ctx, SANIC_ERR_UNSUPPORTED, "paged_cache_write: head_dim must be a multiple of 16, at most 256");
    SANIC_REQUIRE(ctx, p->cache_dtype == SANIC_BF16 || p->cache_dtype == SANIC_F16, "paged_cache_write: the pages are bf16 or f16");
    SANIC_REQUIRE(ctx, p->src_dtype == SANIC_F32 || p->src_dtype == p->cache_dtype, "paged_cache_write: the source is f32 or of the pages' type");
    SANIC_REQUIRE(ctx, p->page_size > 0 && p->n_pages > 0, "paged_cache_write: empty page pool");
    if (p->n_tokens == 0) return SANIC_OK;
    SANIC_REQUIRE(ctx, p->k && p->v && p->k_pages && p->v_pages && p->slots, "paged_cache_write: null tensor");
    SANIC_REQUIRE(ctx, !p->q == !p->q_out && (!p->q || p->q_heads > 0), "paged_cache_write: q and q_out go together");
    SANIC_REQUIRE(ctx, !p->table || (p->positions && p->n_positions > 0), "paged_cache_write: a table needs positions");
    const int src = p->src_dtype == SANIC_F32 ? 4 : 2;
    // 16-byte accesses on every side
    auto aligned = [](const void* ptr, int64_t stride, int bytes) { return ((uintptr_t)ptr % 16) == 0 && (stride * bytes) % 16 == 0 && stride >= 0; };
    SANIC_REQUIRE(ctx, aligned(p->q, p->q ? p->q_stride : 0, src) && aligned(p->k, p->k_stride, src) && aligned(p->v, p->v_stride, src) &&
                  aligned(p->q_out, p->q ? p->q_out_stride : 0, 2) && aligned(p->table, 0, 4) &&
                  aligned(p->k_pages, p->k_page_stride, 2) && aligned(p->v_pages, p->v_page_stride, 2) &&
                  p->k_row_stride % 8 == 0 && p->k_head_stride % 8 == 0 && p->v_row_stride % 8 == 0 && p->v_head_stride % 8 == 0 &&
                  p->k_row_stride >= 0 && p->k_head_stride >= 0 && p->v_row_stride >= 0 && p->v_head_stride >= 0,
                  "paged_cache_write: rows must be 16-byte aligned");
    SANIC_REQUIRE(ctx, !p->q || p->q_out_stride >= (int64_t)p->q_heads * p->head_dim || p->n_tokens == 1, "paged_cache_write: q_out rows overlap");
    SANIC_REQUIRE(ctx, p->q != p->q_out || !p->q || (src == 2 && p->q_stride == p->q_out_stride), "paged_cache_write: in place needs one type and one stride");
    sanic_set_device(ctx);
    const int heads = (p->q ? p->q_heads : 0) + 2 * p->kv_heads, per_token = (heads + HP - 1) / HP * (p->head_dim / 16);
    const int tpb = std::max(1, WT / per_token);
    const long long work = (long long)((p->n_tokens + tpb - 1) / tpb) * ((tpb * per_token + WT - 1) / WT);
    const dim3 grid((unsigned)std::min<long long>(work, (long long)(src == 4 ? write_blocks<float>() : write_blocks<Bf16>()) * ctx->sm_count)), block(WT);
    int shift = -1;
    for (int i = 0; i < 31; ++i) if ((1 << i) == p->page_size) shift = i;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (p->cache_dtype == SANIC_BF16)
        e = src == 4 ? launch_pdl(paged_write_kernel<float, true>, grid, block, 0, st, *p, tpb, shift, ctx->status_dev)
                     : launch_pdl(paged_write_kernel<Bf16, true>, grid, block, 0, st, *p, tpb, shift, ctx->status_dev);
    else
        e = src == 4 ? launch_pdl(paged_write_kernel<float, false>, grid, block, 0, st, *p, tpb, shift, ctx->status_dev)
                     : launch_pdl(paged_write_kernel<F16, false>, grid, block, 0, st, *p, tpb, shift, ctx->status_dev);
    SANIC_CUDA_CHECK(ctx, e);
    return SANIC_OK;
}

}  // extern "C"
