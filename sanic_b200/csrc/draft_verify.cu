// Verification of drafted tokens by rejection sampling, from given uniform numbers, so that the tokens kept are distributed as
// the target's: draft x_i is kept while u_i q_i(x_i) < p_i(x_i) (an exact product of two f32 in f64); the token behind the kept
// ones is drawn from max(p - q, 0) after a rejection, else from the next row's p, as the first index whose running sum exceeds
// u times the total.
//
// Only one row of p (and of q after a rejection) is read per request: which one is known after at most max_draft gathered
// pairs, which one warp takes at once. HBM bounds a batch (4 or 8 bytes per vocabulary entry); a single request is a chain of
// latencies: lengths and tokens, their probabilities, the row, the join. One cluster of CTAs serves a request: each CTA sums
// its slice of the row in groups of 1024 entries, the slices' totals are exchanged through distributed shared memory, and the
// CTA that holds the drawn token finds its group from the sums that it kept, so that only one group is read twice. No
// workspace, no atomics: the sums have a fixed order for a given cluster size. They are f64 (a running sum in f32 would put
// the border of about one entry in a thousand on its other side at a vocabulary of 1e5), with one reduction over the lanes per
// group: a 64-bit butterfly costs as much as reading 512 entries. (Four blocks per SM leave a thread 64 registers, of which 28 bytes
// spill. 64 requests 20.7 us where their bytes take 7.3: the chain in front of the first row byte, which every block pays at the same
// time, and the join behind the last; the 12 M conversions to 64 bits are
// 3 us at 16 per clock and SM.)
#include <cooperative_groups.h>

#include "paged.cuh"

namespace {
using namespace sanic;
namespace cg = cooperative_groups;

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int CHUNK = 128, PER_GROUP = 8, GROUP = CHUNK * PER_GROUP;      // entries of a warp's load, loads of a group
constexpr int MAX_GROUPS = 512;                   // of a CTA: 2^19 entries
constexpr int MAX_CLUSTER = 16;

enum { FROM_TARGET = 0, FROM_DIFFERENCE = 1, WITHOUT_TOKEN = 2 };

struct Row { const float* p; const float* q; int mode, token; bool vec; };

// The weight of entry j. NaN, infinities and weights that are not positive count as 0: p - q > 0 exactly where p > q.
__device__ __forceinline__ double weight(float p, float q, const Row& r, int j) {
    const bool counts = p > q && p <= 3.402823466e38f && q >= -3.402823466e38f && !(r.mode == WITHOUT_TOKEN && j == r.token);
    return counts ? (double)p - (double)q : 0.0;
}
// A lane's four entries of the chunk at c: neighbours where the rows start on 16-byte boundaries, else 32 apart.
__device__ __forceinline__ int entry(const Row& r, int c, int lane, int i) { return r.vec ? c + lane * 4 + i : c + i * 32 + lane; }
__device__ __forceinline__ void load4(const Row& r, int c, int end, int lane, float (&p)[4], float (&q)[4]) {
    if (r.vec && c + CHUNK <= end) {
        const float4 a = __ldcs((const float4*)(r.p + c + lane * 4));
        p[0] = a.x; p[1] = a.y; p[2] = a.z; p[3] = a.w;
        if (r.mode == FROM_DIFFERENCE) {
            const float4 b = __ldcs((const float4*)(r.q + c + lane * 4));
            q[0] = b.x; q[1] = b.y; q[2] = b.z; q[3] = b.w;
        } else q[0] = q[1] = q[2] = q[3] = 0.0f;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = entry(r, c, lane, i);
        p[i] = j < end ? __ldcs(r.p + j) : 0.0f;
        q[i] = j < end && r.mode == FROM_DIFFERENCE ? __ldcs(r.q + j) : 0.0f;
    }
}
__device__ __forceinline__ double group_sum(const Row& r, int g, int end, int lane) {      // this lane's part
    double s = 0.0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {                 // four loads of p and of q in flight
        float p[PER_GROUP / 2][4], q[PER_GROUP / 2][4];
#pragma unroll
        for (int k = 0; k < PER_GROUP / 2; ++k) load4(r, g * GROUP + (h * PER_GROUP / 2 + k) * CHUNK, end, lane, p[k], q[k]);
#pragma unroll
        for (int k = 0; k < PER_GROUP / 2; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) s += weight(p[k][i], q[k][i], r, entry(r, g * GROUP + (h * PER_GROUP / 2 + k) * CHUNK, lane, i));
    }
    return s;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double warp_scan64(double v, int lane) {     // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const double x = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += x; }
    return v;
}

__global__ void __launch_bounds__(THREADS, 4) draft_verify_kernel(const sanic_draft_verify_params p, int* err) {
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int b = blockIdx.x / cs;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __shared__ double s_sum[MAX_GROUPS];              // per group: its sum, then the sum of all groups of this CTA up to it
    __shared__ double s_total;
    __shared__ int s_count, s_len, s_start, s_token;
    __shared__ float s_u;
    griddep_wait();
    griddep_launch();

    if (warp == 0) {
        const int K = p.max_draft;
        // everything that no other load decides is asked for together
        int len = p.draft_lens ? p.draft_lens[b] : K;
        const int start = p.target_start ? p.target_start[b] : b * (K + 1);
        int tok = lane < K ? p.draft_tokens[(int64_t)b * K + lane] : -1;
        const float u = lane < K ? p.u_accept[(int64_t)b * K + lane] : 0.0f;
        if (lane == 0) s_u = p.u_sample[b];
        bool bad = len < 0 || len > K;
        len = min(max(len, 0), K);
        const bool no_rows = start < 0 || (long long)start + len >= p.target_rows;
        bad |= no_rows;
        bool ok = false;
        if (lane >= len) tok = -1;
        if (lane < len && !no_rows) {
            if ((unsigned)tok < (unsigned)p.vocab) {
                const float pt = p.target_probs[(int64_t)(start + lane) * p.target_stride + tok];
                const float qt = p.draft_probs ? p.draft_probs[(int64_t)b * p.draft_request_stride + (int64_t)lane * p.draft_stride + tok] : 1.0f;
                ok = (double)u * (double)qt < (double)pt;
            } else bad = true;
        }
        const unsigned failed = ~__ballot_sync(0xffffffffu, ok);      // lanes past the drafts are among them
        const int count = failed ? __ffs(failed) - 1 : 32;
        const int rejected = __shfl_sync(0xffffffffu, tok, min(count, 31));
        if (rank == 0) {
            int32_t* out = p.tokens_out + (int64_t)b * (K + 1);
            for (int i = lane; i <= K; i += 32) if (i != count || no_rows) out[i] = -1;      // the drawn token's place is written below
            __syncwarp();
            if (lane < count) out[lane] = tok;
            if (lane == 0) p.accepted[b] = count;
            if (__any_sync(0xffffffffu, bad) && lane == 0 && err) atomicCAS(err, 0, paged::STATUS_VERIFY);
        }
        if (lane == 0) { s_count = count; s_len = len; s_start = no_rows ? -1 : start; s_token = rejected; }
    }
    __syncthreads();
    if (s_start < 0) return;                          // every CTA of the cluster alike
    const int count = s_count;
    const bool rejected = count < s_len;
    Row row;
    row.p = p.target_probs + (int64_t)(s_start + count) * p.target_stride;
    row.q = p.draft_probs ? p.draft_probs + (int64_t)b * p.draft_request_stride + (int64_t)min(count, max(p.max_draft - 1, 0)) * p.draft_stride : nullptr;
    row.token = s_token;
    row.mode = !rejected ? FROM_TARGET : (p.draft_probs ? FROM_DIFFERENCE : WITHOUT_TOKEN);

    // this CTA's slice: whole groups
    const int groups_all = (p.vocab + GROUP - 1) / GROUP;
    const int g0 = (int)((long long)groups_all * rank / cs), g1 = (int)((long long)groups_all * (rank + 1) / cs);
    const int n_groups = g1 - g0;
    double total = 0.0, upto = 0.0;
    while (true) {
        row.vec = ((uintptr_t)row.p % 16) == 0 && (row.mode != FROM_DIFFERENCE || ((uintptr_t)row.q % 16) == 0);
        for (int g = g0 + warp; g < g1; g += WARPS) {
            const double v = warp_sum64(group_sum(row, g, p.vocab, lane));
            if (lane == 0) s_sum[g - g0] = v;
        }
        __syncthreads();
        if (warp == 0) {                              // running sums over the groups
            double carry = 0.0;
            for (int i = 0; i < n_groups; i += 32) {
                double v = warp_scan64(i + lane < n_groups ? s_sum[i + lane] : 0.0, lane) + carry;
                if (i + lane < n_groups) s_sum[i + lane] = v;
                carry = __shfl_sync(0xffffffffu, v, 31);
            }
            if (lane == 0) s_total = carry;
        }
        cluster.sync();
        // every warp takes the slices' running sums: a lane per CTA of the cluster
        upto = warp_scan64(lane < cs ? *cluster.map_shared_rank(&s_total, lane) : 0.0, lane);
        total = __shfl_sync(0xffffffffu, upto, 31);
        const bool again = !(total > 0.0) && row.mode != FROM_TARGET;
        if (!again) break;
        row.mode = FROM_TARGET;                       // nothing left of p - q: p itself
        cluster.sync();                               // the totals are read before they are written again
    }
    const double x = (double)s_u * total;
    // the owner: the first CTA whose running sum exceeds x; the last one with any weight if rounding left none
    const double before_me = __shfl_up_sync(0xffffffffu, upto, 1);
    const unsigned over = __ballot_sync(0xffffffffu, lane < cs && upto > x);
    const unsigned any = __ballot_sync(0xffffffffu, lane < cs && upto > (lane > 0 ? before_me : 0.0));
    const int owner = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : -1;
    const double base = rank > 0 ? __shfl_sync(0xffffffffu, upto, max(rank - 1, 0)) : 0.0;
    int32_t* drawn = p.tokens_out + (int64_t)b * (p.max_draft + 1) + count;
    if (owner < 0) { if (rank == 0 && tid == 0) *drawn = -1; }
    else if (rank == owner && warp == 0) {
        int group = -1, final_group = 0;
        for (int i = 0; i < n_groups && group < 0; i += 32) {
            const bool in = i + lane < n_groups;
            const double v = in ? s_sum[i + lane] : 0.0, before = in && i + lane > 0 ? s_sum[i + lane - 1] : 0.0;
            const unsigned over = __ballot_sync(0xffffffffu, in && base + v > x), some = __ballot_sync(0xffffffffu, in && v > before);
            if (over) group = i + __ffs(over) - 1;
            if (some) final_group = i + 31 - __clz(some);
        }
        if (group < 0) group = final_group;
        // the group's chunks: their sums first, then the entries of the one that crosses x
        const int c0 = (g0 + group) * GROUP;
        row.vec = true;                               // a lane's entries are neighbours here, whatever the alignment
        double acc = base + (group > 0 ? s_sum[group - 1] : 0.0);
        int hit = -1, positive = -1;
        unsigned hits = 0;
        for (int half = 0; half < 2; ++half) {
            float w_p[PER_GROUP / 2][4], w_q[PER_GROUP / 2][4];
            const int ch = c0 + half * (GROUP / 2);
#pragma unroll
            for (int k = 0; k < PER_GROUP / 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = ch + k * CHUNK + lane * 4 + i;
                    w_p[k][i] = j < p.vocab ? row.p[j] : 0.0f;
                    w_q[k][i] = j < p.vocab && row.mode == FROM_DIFFERENCE ? row.q[j] : 0.0f;
                }
#pragma unroll
            for (int k = 0; k < PER_GROUP / 2; ++k) {
                double w[4], own = 0.0;
#pragma unroll
                for (int i = 0; i < 4; ++i) { w[i] = weight(w_p[k][i], w_q[k][i], row, ch + k * CHUNK + lane * 4 + i); own += w[i]; }
                const double scan = warp_scan64(own, lane);
                double at = acc + (scan - own);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    at += w[i];
                    if (w[i] > 0.0 && !hits) { positive = ch + k * CHUNK + lane * 4 + i; if (hit < 0 && at > x) hit = positive; }
                }
                if (!hits) hits = __ballot_sync(0xffffffffu, hit >= 0);      // the first chunk with a crossing; in it, the first lane
                acc += __shfl_sync(0xffffffffu, scan, 31);
            }
        }
        if (!hits) {                                  // rounding left no crossing: the last entry with a weight
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) positive = max(positive, __shfl_xor_sync(0xffffffffu, positive, o));
            hit = positive; hits = 1;
        }
        const int token = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
        if (lane == 0) *drawn = token;
    }
    cluster.sync();                                   // no CTA leaves while another may read its total
}
}  // namespace

extern "C" int32_t sanic_draft_verify(sanic_ctx* ctx, const sanic_draft_verify_params* p, void* stream) {
    if (!ctx || !p) return SANIC_ERR_INVALID;
    SANIC_REQUIRE(ctx, p->n_requests >= 0 && p->max_draft >= 0 && p->vocab > 0, "draft_verify: bad counts");
    if (p->max_draft > 32) return sanic_fail(ctx, SANIC_ERR_UNSUPPORTED, "draft_verify: at most 32 drafted tokens per request");
    if (p->vocab > (1 << 19)) return sanic_fail(ctx, SANIC_ERR_UNSUPPORTED, "draft_verify: at most 524288 vocabulary entries");
    if (p->n_requests == 0) return SANIC_OK;
    SANIC_REQUIRE(ctx, p->target_probs && p->u_sample && p->tokens_out && p->accepted && p->target_rows > 0, "draft_verify: null tensor");
    SANIC_REQUIRE(ctx, p->max_draft == 0 || (p->draft_tokens && p->u_accept), "draft_verify: drafts need tokens and u_accept");
    SANIC_REQUIRE(ctx, (long long)p->n_requests * (p->max_draft + 1) < (1ll << 31), "draft_verify: too many rows");
    SANIC_REQUIRE(ctx, p->target_stride >= p->vocab || p->target_rows == 1, "draft_verify: target rows overlap");
    SANIC_REQUIRE(ctx, !p->draft_probs || ((p->draft_stride >= p->vocab || p->max_draft == 1) && p->draft_stride >= 0 && p->draft_request_stride >= 0),
                  "draft_verify: draft rows overlap");
    sanic_set_device(ctx);
    // CTAs per request: enough that the batch covers four blocks per SM, at most 16 (a cluster's limit) and never less than a
    // group each (64 requests of 128256 entries: 8 each 21 us, 16 each 34 us, 4 each 23 us; one request: 16 10.6 us, 8 13.1 us)
    const int groups = (p->vocab + GROUP - 1) / GROUP;
    int cs = 1;
    while (cs < MAX_CLUSTER && 2 * cs * (long long)p->n_requests <= 4ll * ctx->sm_count && 2 * cs <= groups) cs *= 2;
    static thread_local int ready_on = -1;
    if (ready_on != ctx->device) {
        SANIC_CUDA_CHECK(ctx, cudaFuncSetAttribute(draft_verify_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        ready_on = ctx->device;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p->n_requests * cs); cfg.blockDim = dim3(THREADS); cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    static const bool pdl = getenv("SANIC_NO_PDL") == nullptr;
    cfg.attrs = attr; cfg.numAttrs = pdl ? 2 : 1;
    SANIC_CUDA_CHECK(ctx, cudaLaunchKernelEx(&cfg, draft_verify_kernel, *p, ctx->status_dev));
    return SANIC_OK;
}
