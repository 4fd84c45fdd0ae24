// How attention over a paged cache is cut into work: plain index arithmetic, the same on the device (paged.cuh) and on the
// host (where a test walks it for every CTA and checks that each key tile of each item is folded exactly once).
//
// An item is (request, kv head, block of query tokens) and folds the tiles of keys its tokens see. The items' tiles, laid end
// to end in the order request, kv head, block, are one axis, cut into one equal range per CTA of an exactly resident grid
// (a stream-K split): ragged lengths cost no last wave, and a single long request uses the whole device.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define SANIC_HD __host__ __device__ __forceinline__
#else
#define SANIC_HD inline
#endif

namespace sanic {
namespace paged {

struct Shape {
    int n_requests, kv_heads, window;
    int block_tokens;      // query tokens of an item
};

struct Req { int q0, qn, kv; };      // first token row, tokens of the chunk, keys (the chunk's own included)

SANIC_HD int imin(int a, int b) { return a < b ? a : b; }
SANIC_HD int imax(int a, int b) { return a > b ? a : b; }

// Keys [lo, hi) that the tokens of block rb see, taken together: token i of the chunk stands at position kv - qn + i and
// sees the keys up to its own, at most `window` of them.
SANIC_HD void key_range(const Shape& p, const Req& r, int rb, int& lo, int& hi) {
    const int t0 = rb * p.block_tokens, t1 = imin(r.qn, t0 + p.block_tokens) - 1, base = r.kv - r.qn;
    hi = imax(0, base + t1 + 1);
    lo = p.window > 0 ? imax(0, base + t0 - p.window + 1) : 0;
}
template <int KT>
SANIC_HD void tile_range(const Shape& p, const Req& r, int rb, int& lo, int& hi, int& jb, int& je) {
    key_range(p, r, rb, lo, hi);
    jb = lo / KT;
    je = hi > lo ? (hi + KT - 1) / KT : jb;
}

// Cost of an item in key tiles: its tiles (at least one, so that an item without a visible key is still somebody's and its
// rows are written) and OVERHEAD tiles' worth of start and end (five prompts 187 us with 1, 181 with 2, 189 with 4; 64 decodes
// of 8000 keys 339, 337, 338).
constexpr int OVERHEAD = 2;
template <int KT>
SANIC_HD int item_cost(const Shape& p, const Req& r, int rb) {
    int lo, hi, jb, je;
    tile_range<KT>(p, r, rb, lo, hi, jb, je);
    return imax(1, je - jb) + OVERHEAD;
}
SANIC_HD int blocks_of(const Shape& p, const Req& r) { return (r.qn + p.block_tokens - 1) / p.block_tokens; }
template <int KT>
SANIC_HD long long request_cost(const Shape& p, const Req& r) {
    long long c = 0;
    const int blocks = blocks_of(p, r);
    for (int rb = 0; rb < blocks; ++rb) c += item_cost<KT>(p, r, rb);
    return c * p.kv_heads;
}

// A CTA's part of one item: tiles [jb, je) of the item's, the first and the last of them or not.
struct Seg {
    Req r;
    int b, hk, rb;
    int lo, hi;            // keys the item's tokens see
    int jb, je;            // this segment's key tiles; equal when no key is visible
    bool starts, finishes;
    int parts;             // CTAs that share the item, this one the first of them (1 unless starts && !finishes)
};

// Walks the segments of one CTA's range in order; `load(b)` gives request b. All threads that walk hold the same state.
template <int KT, class Load>
struct Walk {
    Load load;
    long long pos, end, total, ctas;
    long long item;        // cost position at which the current item begins
    int b, hk, rb;
    Req r;

    // cum[0 .. n]: exclusive prefix sums of request_cost
    SANIC_HD void init(const Shape& p, const long long* cum, int cta, int grid) {
        total = cum[p.n_requests];
        ctas = total < grid ? total : grid;
        if (cta >= ctas) { pos = end = 0; return; }
        pos = cta * total / ctas;
        end = (cta + 1) * total / ctas;
        int lo = 0, hi = p.n_requests - 1;       // the last request whose items begin at or before pos: its cost is not 0
        while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (cum[mid] <= pos) lo = mid; else hi = mid - 1; }
        b = lo;
        r = load(b);
        const long long per_head = (cum[b + 1] - cum[b]) / p.kv_heads;
        hk = (int)((pos - cum[b]) / per_head);
        item = cum[b] + hk * per_head;
        rb = 0;
        for (int c1; item + (c1 = item_cost<KT>(p, r, rb)) <= pos; ++rb) item += c1;
    }
    SANIC_HD long long cta_of(long long x) const { return ((x + 1) * ctas - 1) / total; }   // whose range holds position x
    // The next segment with work in it; false at the end of the range.
    SANIC_HD bool next(const Shape& p, Seg& s) {
        while (pos < end) {
            int jb, je;
            tile_range<KT>(p, r, rb, s.lo, s.hi, jb, je);
            const long long first = item + OVERHEAD, stop = first + imax(1, je - jb);      // cost positions of the item's tiles
            const long long a = pos > first ? pos : first, z = end < stop ? end : stop;
            const bool work = a < z;
            if (work) {
                s.r = r; s.b = b; s.hk = hk; s.rb = rb;
                s.starts = a == first; s.finishes = z == stop;
                s.jb = jb + (int)(a - first); s.je = je > jb ? jb + (int)(z - first) : s.jb;
                s.parts = (s.starts && !s.finishes) ? (int)(cta_of(stop - 1) - cta_of(first)) + 1 : 1;
            }
            if (end >= stop) {     // on to the next item
                item = stop;
                if (++rb >= blocks_of(p, r)) {
                    rb = 0;
                    if (++hk >= p.kv_heads) {
                        hk = 0;
                        do { if (++b >= p.n_requests) { end = stop; break; } r = load(b); } while (r.qn <= 0);
                    }
                }
            }
            pos = end < stop ? end : stop;
            if (work) return true;
        }
        return false;
    }
};

// Where segment s of CTA `cta` leaves its partial: a CTA has at most one segment that continues an item (slot 0) and one that
// starts an item and leaves the rest to the next CTAs (slot 1).
SANIC_HD long long partial_slot(const Seg& s, int cta) { return (long long)cta * 2 + (s.starts ? 1 : 0); }

}  // namespace paged
}  // namespace sanic
