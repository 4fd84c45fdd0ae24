"""The paged-cache serving operators against plain 64-bit implementations.

Tolerances, from the arithmetic (u = eps / 2 of the storage type, the largest relative error of one rounding):
  * attention: the output is rounded once (u |out|) and every weight once before the product with v (u A with
    A = sum_j w_j |v_j|); scores are f32 sums of D products, |error| <= D 2^-24 sum |q k| scale <= 1e-4 for the inputs here
    (D <= 128, unit-normal k, q of deviation 1.5: sum |q k| scale stays below 14), which moves a weight by at most that share on
    each side of the quotient, 2e-4 A; f32 sums over at most a few hundred steps stay below 3e-5. So
    |got - want| <= u |want| + (u + 2.5e-4) A.
  * log-sum-exp: 1e-4 from the scores, 3e-5 from the sum and 2^-22 from the exponentials: 1.5e-4 absolute.
  * RoPE: three f32 roundings of terms bounded by |a| + |b| (cos, sin <= 1), then one to storage: u |want| + 2^-22 (|a| + |b|),
    plus the smallest subnormal step of f16 (2^-25).
  * page tables, slots, positions, counts and tokens: exact.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    from sanic_b200 import CudaDevice
    return CudaDevice(0)


def ints(dev, xs, dtype=torch.int32):
    return torch.tensor(xs, dtype=dtype, device=dev.torch_device)


def gen(dev, seed):
    g = torch.Generator(device=dev.torch_device)
    g.manual_seed(seed)
    return g


# ───────────────────────── attention ─────────────────────────
def make_problem(dev, new, ctx, hq, hkv, d, dtype, page, heads_first=False, window=0, seed=0, poison=True, extra_pages=3, table_pad=1):
    """Ragged chunks `new` over caches of `ctx` held tokens. Every pool row that no token may see holds NaN."""
    g = gen(dev, seed)
    td = dev.torch_device
    kv = [c + n for c, n in zip(ctx, new)]
    need = [-(-x // page) for x in kv]
    n_pages = sum(need) + extra_pages
    order = torch.randperm(n_pages, generator=g, device=td)
    shape = (n_pages, hkv, page, d) if heads_first else (n_pages, page, hkv, d)
    pools = []
    for _ in range(2):
        x = torch.full(shape, float("nan") if poison else 3.0, device=td, dtype=DT[dtype])
        pools.append(x.transpose(1, 2) if heads_first else x)
    table = torch.full((len(new), max(need + [1]) + table_pad), n_pages + 77, dtype=torch.int32, device=td)   # entries past the need are never read
    at = 0
    keys, values = [], []
    for b, (n, x) in enumerate(zip(need, kv)):
        pages = order[at:at + n]
        at += n
        table[b, :n] = pages.to(torch.int32)
        first = max(0, ctx[b] - window + 1) if window else 0
        if n == 0:
            keys.append(torch.zeros(0, hkv, d, device=td)); values.append(torch.zeros(0, hkv, d, device=td))
            continue
        k = torch.randn(x, hkv, d, generator=g, device=td).to(DT[dtype])
        v = torch.randn(x, hkv, d, generator=g, device=td).to(DT[dtype])
        keys.append(k); values.append(v)
        if new[b]:
            pos = torch.arange(first, x, device=td)
            pools[0][pages[pos // page], pos % page] = k[first:]
            pools[1][pages[pos // page], pos % page] = v[first:]
    starts = np.concatenate([[0], np.cumsum(new)]).tolist()
    q = (1.5 * torch.randn(starts[-1], hq, d, generator=g, device=td)).to(DT[dtype])
    return dict(q=q, k_pages=pools[0], v_pages=pools[1], block_table=table, query_start=ints(dev, starts), kv_lens=ints(dev, kv)), keys, values


def plain_attention(q, keys, values, new, kv, window, scale):
    """f64; also A = sum_j w_j |v_j|."""
    hq, d = q.shape[1:]
    outs, bounds, lses = [], [], []
    at = 0
    for b, n in enumerate(new):
        k, v = keys[b].double(), values[b].double()
        group = hq // k.shape[1]
        qb = q[at:at + n].double()
        at += n
        out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
        amp = torch.zeros_like(out)
        lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=q.device)
        for i in range(n):
            pos = kv[b] - n + i
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                continue
            kk, vv = (x[lo:pos + 1].repeat_interleave(group, 1) for x in (k, v))
            s = torch.einsum("hd,jhd->hj", qb[i], kk) * scale
            lse[i] = torch.logsumexp(s, 1)
            w = torch.exp(s - lse[i][:, None])
            out[i] = torch.einsum("hj,jhd->hd", w, vv)
            amp[i] = torch.einsum("hj,jhd->hd", w, vv.abs())
        outs.append(out); bounds.append(amp); lses.append(lse)
    return torch.cat(outs), torch.cat(bounds), torch.cat(lses)


def check_attention(got, lse, want, amp, want_lse):
    u = torch.finfo(got.dtype).eps / 2
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    over = err - (u * want.abs() + (u + 2.5e-4) * amp)
    assert (over <= 0).all(), f"worst excess {over.max().item():.3e} at {np.unravel_index(int(over.argmax()), over.shape)}; err {err.max().item():.3e}"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all()
    assert ((lse.double() - want_lse)[~empty].abs() <= 1.5e-4).all(), (lse.double() - want_lse)[~empty].abs().max()


def run_case(dev, new, ctx, hq, hkv, d, dtype, page, heads_first=False, window=0, seed=0, max_query_len=None, scale=None):
    args, keys, values = make_problem(dev, new, ctx, hq, hkv, d, dtype, page, heads_first, window, seed)
    got, lse = dev.attn_paged(**args, max_query_len=max(new) if max_query_len is None else max_query_len, window=window, scale=scale, return_lse=True)
    dev.sync()
    kv = [c + n for c, n in zip(ctx, new)]
    check_attention(got, lse, *plain_attention(args["q"], keys, values, new, kv, window, scale if scale is not None else 1.0 / math.sqrt(d)))


HEADS = [(4, 1), (8, 2), (3, 3), (7, 1), (10, 2), (16, 1)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page", [1, 16, 24, 64, 256])
def test_attn_single_tokens(dev, d, dtype, page):
    ctx = [0, 1, 14, 15, 16, 63, 64, 65, 127, 128, 200, 700]
    hq, hkv = HEADS[(page + d) % len(HEADS)]
    run_case(dev, [1] * len(ctx), ctx, hq, hkv, d, dtype, page, heads_first=page == 64, seed=page)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (32, 8), (5, 1), (33, 1), (64, 1), (12, 4)])
@pytest.mark.parametrize("window", [0, 1, 70])
def test_attn_heads_and_windows(dev, hq, hkv, window):
    run_case(dev, [1, 3, 2, 1], [90, 300, 0, 517], hq, hkv, 64, "bf16", 16, window=window, seed=hq + window)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("new,ctx", [([5, 3, 6, 1], [33, 250, 0, 100]), ([0, 4, 0, 0, 2, 0], [10, 70, 0, 5, 64, 9]), ([13], [129]), ([40, 1, 17], [3, 400, 0])])
@pytest.mark.parametrize("window", [0, 37])
def test_attn_short_chunks(dev, d, dtype, new, ctx, window):
    run_case(dev, new, ctx, 8, 2, d, dtype, 16, window=window, seed=len(new))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page,heads_first", [(8, False), (16, True), (24, False), (32, False), (128, True), (256, False)])
def test_attn_long_chunks(dev, d, dtype, page, heads_first):
    run_case(dev, [129, 1, 300, 65], [0, 500, 77, 640], 8, 2, d, dtype, page, heads_first=heads_first, seed=page)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("maxq", [1, 200])
@pytest.mark.parametrize("page,heads_first", [(8, True), (12, False), (20, True), (40, True), (48, False), (72, True), (96, False), (136, False), (1000, True)])
def test_attn_odd_page_sizes(dev, d, maxq, page, heads_first):
    # what the page and a tile have in common decides how much one copy takes: 8 rows up to a tile, or 16 bytes at a time
    run_case(dev, [1, 75, 200, 3], [700, 513, 0, 1100], 6, 2, d, "bf16", page, heads_first=heads_first, window=333 if page == 72 else 0, seed=page, max_query_len=maxq)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (7, 1), (12, 4), (64, 1), (33, 1)])
@pytest.mark.parametrize("window", [0, 1, 100, 300])
def test_attn_long_chunks_heads_and_windows(dev, d, hq, hkv, window):
    run_case(dev, [257, 70, 1, 0, 128], [5, 600, 900, 40, 0], hq, hkv, d, "bf16", 16, window=window, seed=hq + window)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("maxq", [1, 5, 200])
@pytest.mark.parametrize("window", [0, 40])
def test_attn_hidden_keys_and_values_of_any_kind(dev, d, dtype, page, maxq, window):
    """Keys and values of the chunk's own tokens that are infinite or NaN: tokens that see them have what the formula gives, tokens
    that do not (before them, or past the window) their finite result. Long caches, whose items several CTAs share, among them."""
    new, ctx, hq, hkv = [70, 9, 1, 3, 300], [300, 20000, 64, 0, 1100], 8, 2
    args, keys, values = make_problem(dev, new, ctx, hq, hkv, d, dtype, page, window=window, seed=page + maxq)
    inf, nan = math.inf, math.nan

    def put(pool, mine, b, pos, col, x):       # into a request's row and the page that holds it
        mine[b][pos, :, col] = x
        args[pool][args["block_table"][b, pos // page].long(), pos % page, :, col] = x

    for pos, col, x in ((305, slice(None), nan), (310, 3, inf), (311, 5, -inf), (330, 3, -inf), (369, slice(0, 8), nan)):
        put("v_pages", values, 0, pos, col, x)
    for pos, col, x in ((20004, slice(1, 60, 2), inf), (20007, slice(None), nan)):
        put("v_pages", values, 1, pos, col, x)
    put("k_pages", keys, 1, 20006, 9, nan)
    put("v_pages", values, 3, 2, slice(None), -inf)
    if window:
        put("v_pages", values, 4, 1075, slice(0, 32), nan)        # the first 15 tokens see it, the others no longer
    put("v_pages", values, 4, 1290, slice(16, None), nan)
    put("k_pages", keys, 4, 1340, slice(None), nan)
    kv = [c + n for c, n in zip(ctx, new)]
    got, lse = dev.attn_paged(**args, max_query_len=maxq, window=window, return_lse=True)
    dev.sync()
    want, amp, wl = plain_attention(args["q"], keys, values, new, kv, window, d ** -0.5)
    fine = torch.isfinite(want)
    assert fine.sum() > want.numel() // 2 and not fine.all()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (torch.isnan(got) != torch.isnan(want)).nonzero()[:4].tolist()
    assert torch.equal(got.double()[torch.isinf(want)], want[torch.isinf(want)])
    u = torch.finfo(got.dtype).eps / 2
    assert ((got.double() - want).abs()[fine] <= (u * want.abs() + (u + 2.5e-4) * amp)[fine]).all()
    fine = torch.isfinite(wl)
    assert torch.equal(torch.isfinite(lse), fine) and ((lse.double() - wl).abs()[fine] <= 1.5e-4).all()


@pytest.mark.parametrize("hq,hkv", [(2, 2), (7, 1), (40, 1), (64, 1)])
@pytest.mark.parametrize("window", [1, 3, 64, 100, 300])
@pytest.mark.parametrize("maxq", [1, 300])
def test_attn_values_that_leave_the_window_and_a_replay_over_others(dev, hq, hkv, window, maxq):
    """Values that are not finite below and inside the window's edges, in blocks of every size a form makes of a chunk; then the
    same graph over finite values."""
    new, ctx, d, page = [300, 40, 2], [700, 5, 130], 64, 16
    args, keys, values = make_problem(dev, new, ctx, hq, hkv, d, "bf16", page, window=window, seed=window + hq)
    dev.attn_paged(**args, max_query_len=maxq, window=window)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got, lse = dev.attn_paged(**args, max_query_len=maxq, window=window, return_lse=True)
    spots = [(b, p, c, x) for b, p, c, x in ((0, 700 - window + 1, 3, math.nan), (0, 700 - window // 2, 60, -math.inf), (0, 801, 7, math.inf),
                                             (0, 999, slice(None), math.nan), (1, 6, 1, math.nan), (1, 44, 2, math.inf), (2, 131, 5, math.nan)) if p >= 0]
    kv = [c + n for c, n in zip(ctx, new)]
    for poisoned in (True, False):
        for b, pos, col, x in spots:
            if not poisoned:
                x = 0.25
            values[b][pos, :, col] = x
            args["v_pages"][args["block_table"][b, pos // page].long(), pos % page, :, col] = x
        graph.replay()
        dev.sync()
        want, amp, wl = plain_attention(args["q"], keys, values, new, kv, window, d ** -0.5)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), (torch.isnan(got) != torch.isnan(want)).nonzero()[:4].tolist()
        assert torch.equal(got.double()[torch.isinf(want)], want[torch.isinf(want)])
        fine = torch.isfinite(want)
        assert fine.all() != poisoned
        assert ((got.double() - want).abs()[fine] <= (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.5e-4) * amp)[fine]).all()
        assert ((lse.double() - wl).abs() <= 1.5e-4).all()


@pytest.mark.parametrize("maxq", [33, 100])
def test_attn_hidden_values_in_more_blocks_than_are_noted(dev, maxq):
    # 100 tokens of 400 requests over 32 kv heads: a NaN value in both blocks of every one of them, at tokens 40 and 90
    n, t, hkv, group, d, page, td = 400, 100, 32, 4, 64, 16, dev.torch_device
    g = gen(dev, 41)
    per = -(-t // page)
    k, v = (torch.randn(n * per, page, hkv, d, generator=g, device=td).to(torch.bfloat16) for _ in range(2))
    table = torch.randperm(n * per, generator=g, device=td).to(torch.int32).view(n, per)
    for i, cols in ((40, slice(3, 20)), (90, slice(17, 40))):
        v[table[:, i // page].long(), i % page, :, cols] = math.nan
    q = torch.randn(n * t, hkv * group, d, generator=g, device=td).to(torch.bfloat16)
    got = dev.attn_paged(q, k, v, table, ints(dev, list(range(0, n * t + 1, t))), ints(dev, [t] * n), max_query_len=maxq)
    dev.sync()
    hidden = torch.ones(t, t, dtype=torch.bool, device=td).triu(1)
    for b in range(0, n, 20):
        rows = table[b:b + 20].long()
        kk, vv = (x[rows].flatten(1, 2)[:, :t].double().transpose(1, 2).repeat_interleave(group, 1) for x in (k, v))
        s = q[b * t:(b + 20) * t].view(20, t, hkv * group, d).double().transpose(1, 2) @ kk.transpose(2, 3) * 0.125
        w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        want, amp = w @ torch.nan_to_num(vv), w @ torch.nan_to_num(vv).abs()
        want[:, :, 40:, 3:20] = math.nan
        want[:, :, 90:, 17:40] = math.nan
        have = got[b * t:(b + 20) * t].view(20, t, hkv * group, d).double().transpose(1, 2)
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(have), nan)
        assert ((have - want).abs()[~nan] <= (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.5e-4) * amp)[~nan]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_attn_blocks_of_one_tile_before_blocks_of_two(dev, d):
    # every head's items are a block of two tiles and one of a single row; an uneven number of them per CTA, so that the second
    # tile's warps pass over long segments that the first tile still folds and wait for their own behind those
    run_case(dev, [257], [3000], 222, 222, d, "bf16", 64, seed=d)
    run_case(dev, [257, 129, 2], [700, 1500, 900], 96, 96, d, "f16", 16, seed=d + 1)


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (128, "f16")])
def test_attn_splits_a_long_cache(dev, d, dtype):
    # few items over a long key axis: every CTA of the device holds a part, and the parts are merged
    run_case(dev, [1], [40000], 8, 1, d, dtype, 64, seed=3)
    run_case(dev, [2, 1], [20011, 9], 4, 2, d, dtype, 32, seed=4)
    run_case(dev, [60], [12000], 8, 1, d, dtype, 64, seed=5)


@pytest.mark.parametrize("maxq", [1, 300])
def test_attn_chunk_longer_than_the_hint_and_more_tokens_than_keys(dev, maxq):
    # the hint only selects a kernel; tokens before key 0 (a chunk longer than its keys) see nothing: zeros and -inf
    args, keys, values = make_problem(dev, [90, 30, 7], [20, 0, 0], 8, 2, 64, "bf16", 16, seed=9)
    args["kv_lens"] = ints(dev, [110, 12, 0])
    got, lse = dev.attn_paged(**args, max_query_len=maxq, return_lse=True)
    dev.sync()
    check_attention(got, lse, *plain_attention(args["q"], [keys[0], keys[1][:12], keys[2][:0]], [values[0], values[1][:12], values[2][:0]],
                                               [90, 30, 7], [110, 12, 0], 0, 0.125))
    assert (got[90:108] == 0).all() and (got[120:] == 0).all() and torch.isinf(lse[120:]).all()


@pytest.mark.parametrize("maxq", [4, 200])
def test_attn_leaves_rows_outside_the_chunks_alone(dev, maxq):
    args, keys, values = make_problem(dev, [3, 2], [40, 7], 4, 2, 64, "f16", 16, seed=2)
    q = torch.full((11, 4, 64), float("nan"), dtype=torch.float16, device=dev.torch_device)
    q[4:9] = args["q"]
    args.update(q=q, query_start=args["query_start"] + 4)
    out = torch.full((11, 4, 64), 5.0, dtype=torch.float16, device=dev.torch_device)
    dev.attn_paged(**args, max_query_len=maxq, out=out)
    dev.sync()
    assert (out[:4] == 5.0).all() and (out[9:] == 5.0).all()
    want, amp, _ = plain_attention(q[4:9], keys, values, [3, 2], [43, 9], 0, 0.125)
    assert ((out[4:9].double() - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.5e-4) * amp).all()


@pytest.mark.parametrize("maxq", [2, 100])
def test_attn_strided_queries_and_a_view_of_the_pool(dev, maxq):
    # q cut from a fused projection; pages that are every other page of a larger pool, keys and values interleaved in one tensor
    args, keys, values = make_problem(dev, [2, 70], [100, 30], 8, 2, 128, "bf16", 16, seed=6)
    T = args["q"].shape[0]
    rows = torch.randn(T, 20, 128, device=dev.torch_device).to(torch.bfloat16)
    rows[:, 3:11] = args["q"]
    n = args["k_pages"].shape[0]
    pool = torch.full((2 * n, 16, 2, 2, 128), float("nan"), dtype=torch.bfloat16, device=dev.torch_device)
    pool[::2, :, 0], pool[::2, :, 1] = args["k_pages"], args["v_pages"]
    args.update(q=rows[:, 3:11], k_pages=pool[::2, :, 0], v_pages=pool[::2, :, 1])
    got, lse = dev.attn_paged(**args, max_query_len=maxq, return_lse=True)
    dev.sync()
    check_attention(got, lse, *plain_attention(args["q"], keys, values, [2, 70], [102, 100], 0, 128 ** -0.5))


@pytest.mark.parametrize("maxq", [1, 64])
def test_attn_pool_past_32_bit_offsets(dev, maxq):
    # more than 2^31 elements of keys: the pages used are the last ones
    page, hkv, d = 128, 8, 128
    n_pages = (1 << 31) // (page * hkv * d) + 40
    small, keys, values = make_problem(dev, [1, 33], [700, 100], 8, 8, d, "bf16", page, seed=8)
    used = small["k_pages"].shape[0]
    k = torch.zeros(n_pages, page, hkv, d, dtype=torch.bfloat16, device=dev.torch_device)
    v = torch.zeros_like(k)
    k[-used:], v[-used:] = small["k_pages"], small["v_pages"]
    table = torch.where(small["block_table"] < used, small["block_table"] + (n_pages - used), n_pages + 5).to(torch.int32)
    got, lse = dev.attn_paged(small["q"], k, v, table, small["query_start"], small["kv_lens"], max_query_len=maxq, return_lse=True)
    dev.sync()
    check_attention(got, lse, *plain_attention(small["q"], keys, values, [1, 33], [701, 133], 0, d ** -0.5))


def test_attn_large_scores(dev):
    # scores of some hundreds: the running maximum moves by more than any slack, weights underflow
    args, keys, values = make_problem(dev, [1, 200], [300, 50], 4, 1, 64, "bf16", 16, seed=11)
    for maxq in (1, 200):
        got, lse = dev.attn_paged(**args, max_query_len=maxq, scale=20.0, return_lse=True)
        dev.sync()
        want, amp, wl = plain_attention(args["q"], keys, values, [1, 200], [301, 250], 0, 20.0)
        # the f32 scores are now up to 160 times larger: |error| <= 1e-4 * 160 on each
        err = (got.double() - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 3.3e-2) * amp).all()
        assert ((lse.double() - wl).abs() <= 2e-2).all()


@pytest.mark.parametrize("maxq", [1, 200])
def test_attn_many_requests_and_a_table_cut_from_a_wider_one(dev, maxq):
    # more requests than threads of a block; rows of the table further apart than its width
    r = np.random.default_rng(3)
    new = r.integers(0, 3, 1500)
    if maxq > 1:
        new[700] = 150
    ctx = r.integers(0, 90, 1500)
    args, keys, values = make_problem(dev, new.tolist(), ctx.tolist(), 4, 2, 64, "bf16", 16, seed=14)
    wide = torch.full((1500, args["block_table"].shape[1] + 37), 1 << 29, dtype=torch.int32, device=dev.torch_device)
    wide[:, 5:5 + args["block_table"].shape[1]] = args["block_table"]
    args["block_table"] = wide[:, 5:5 + args["block_table"].shape[1]]
    got, lse = dev.attn_paged(**args, max_query_len=maxq, return_lse=True)
    dev.sync()
    check_attention(got, lse, *plain_attention(args["q"], keys, values, new.tolist(), (ctx + new).tolist(), 0, 0.125))


@pytest.mark.parametrize("page", [192, 384, 2048])
@pytest.mark.parametrize("maxq", [1, 200])
def test_attn_large_and_odd_pages(dev, page, maxq):
    # pages that are a multiple of a tile but no power of two; a pool of one page
    new, ctx = ([1, 140, 3], [500, 300, 0]) if page < 2048 else ([150], [1000])
    args, keys, values = make_problem(dev, new, ctx, 8, 2, 128, "bf16", page, seed=15, extra_pages=0 if page == 2048 else 2)
    assert page < 2048 or args["k_pages"].shape[0] == 1
    got, lse = dev.attn_paged(**args, max_query_len=maxq, return_lse=True)
    dev.sync()
    check_attention(got, lse, *plain_attention(args["q"], keys, values, new, [n + c for n, c in zip(new, ctx)], 0, 128 ** -0.5))


@pytest.mark.parametrize("maxq", [1, 100])
def test_attn_shared_prefix_pages(dev, maxq):
    # two requests whose tables name the same pages for their common prefix
    args, keys, values = make_problem(dev, [1, 40, 1], [64, 100, 64], 4, 2, 64, "f16", 16, seed=16)
    table = args["block_table"]
    table[2, :4] = table[0, :4]
    keys[2] = torch.cat([keys[0][:64], keys[2][64:]]); values[2] = torch.cat([values[0][:64], values[2][64:]])
    got, lse = dev.attn_paged(**args, max_query_len=maxq, return_lse=True)
    dev.sync()
    check_attention(got, lse, *plain_attention(args["q"], keys, values, [1, 40, 1], [65, 140, 65], 0, 0.125))


@pytest.mark.parametrize("maxq", [1, 100])
def test_attn_and_append_at_the_largest_batch(dev, maxq):
    # 8000 requests of 5 held tokens and one new one, through the page tables
    from sanic_b200 import RunError
    n, page, td = 8000, 4, dev.torch_device
    g = gen(dev, 17)
    seq, one = torch.full((n,), 5, dtype=torch.int32, device=td), torch.ones(n, dtype=torch.int32, device=td)
    table = torch.full((n, 2), -1, dtype=torch.int32, device=td)
    free = torch.randperm(2 * n, generator=g, device=td).to(torch.int32)
    first = dev.page_table_append(torch.zeros_like(seq), seq, table, free, ints(dev, [2 * n]), page, 5 * n)
    step = dev.page_table_append(seq, one, table, free, first.free_count, page, n, held_pages=first.held_pages)
    dev.sync()
    assert step.free_count.item() == 0 and sorted(table.flatten().tolist()) == list(range(2 * n)) and (step.positions == 5).all()
    k, v = (torch.randn(n, 6, 1, 64, generator=g, device=td).to(torch.bfloat16) for _ in range(2))
    kp, vp = (torch.full((2 * n, page, 1, 64), float("nan"), dtype=torch.bfloat16, device=td) for _ in range(2))
    dev.paged_cache_write(k[:, :5].reshape(-1, 1, 64), v[:, :5].reshape(-1, 1, 64), kp, vp, first.slots)
    dev.paged_cache_write(k[:, 5], v[:, 5], kp, vp, step.slots)
    q = torch.randn(n, 4, 64, generator=g, device=td).to(torch.bfloat16)
    got, lse = dev.attn_paged(q, kp, vp, table, step.query_start, step.kv_lens, max_query_len=maxq, return_lse=True)
    dev.sync()
    s = torch.einsum("nhd,nkd->nhk", q.double(), k[:, :, 0].double()) * 0.125
    w = torch.softmax(s, -1)
    check_attention(got, lse, torch.einsum("nhk,nkd->nhd", w, v[:, :, 0].double()), torch.einsum("nhk,nkd->nhd", w, v[:, :, 0].double().abs()),
                    torch.logsumexp(s, -1))
    with pytest.raises(RunError, match="8000"):
        dev.attn_paged(q, kp, vp, torch.zeros(8001, 2, dtype=torch.int32, device=td), torch.zeros(8002, dtype=torch.int32, device=td),
                       torch.zeros(8001, dtype=torch.int32, device=td))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("maxq", [1, 200])
def test_attn_outputs_and_workspaces_on_16_byte_boundaries(dev, d, maxq):
    from sanic_b200 import abi
    new, ctx, hq, hkv = [1, 140, 3], [500, 300, 0], 4, 2
    args, keys, values = make_problem(dev, new, ctx, hq, hkv, d, "bf16", 16, seed=18)
    T, td, n = sum(new), dev.torch_device, 3
    want = plain_attention(args["q"], keys, values, new, [a + b for a, b in zip(new, ctx)], 0, d ** -0.5)
    flat = torch.full((T * hq * d + 16,), 3.0, dtype=torch.bfloat16, device=td)
    out = flat[8:8 + T * hq * d].view(T, hq, d)
    assert out.data_ptr() % 32 == 16
    got, lse = dev.attn_paged(**args, max_query_len=maxq, return_lse=True, out=out)
    dev.sync()
    check_attention(got, lse, *want)
    assert (flat[:8] == 3.0).all() and (flat[-8:] == 3.0).all()
    # the same with a workspace on a 16-byte boundary, its bytes of any value, and nothing written past its end
    q, kp, vp, bt = args["q"], args["k_pages"], args["v_pages"], args["block_table"]
    out.fill_(3.0); lse = torch.empty(T, hq, device=td)
    p = abi.AttnPagedParams(q.data_ptr(), out.data_ptr(), lse.data_ptr(), kp.data_ptr(), vp.data_ptr(), bt.data_ptr(), args["query_start"].data_ptr(),
                            args["kv_lens"].data_ptr(), None, 0, q.stride(0), q.stride(1), kp.stride(0), kp.stride(1), kp.stride(2), vp.stride(0),
                            vp.stride(1), vp.stride(2), bt.stride(0), abi.BF16, n, T, maxq, hq, hkv, d, 16, kp.shape[0], bt.shape[1], 0, d ** -0.5)
    nbytes = dev.lib.sanic_attn_paged_workspace_bytes(dev.h, C.byref(p))
    ws = torch.full((nbytes // 4 + 8,), -1, dtype=torch.int32, device=td)
    p.workspace, p.workspace_bytes = ws.data_ptr() + 16, nbytes
    dev._check(dev.lib.sanic_attn_paged(dev.h, C.byref(p), dev.stream()), "attn_paged")
    dev.sync()
    check_attention(out, lse, *want)
    assert (ws[:4] == -1).all() and (ws[4 + nbytes // 4:] == -1).all() and (flat[:8] == 3.0).all() and (flat[-8:] == 3.0).all()
    p.workspace = ws.data_ptr() + 8
    from sanic_b200 import RunError
    with pytest.raises(RunError, match="workspace"):
        dev._check(dev.lib.sanic_attn_paged(dev.h, C.byref(p), dev.stream()), "attn_paged")


@pytest.mark.parametrize("hq,hkv", [(64, 1), (40, 1), (66, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_attn_single_tokens_of_large_groups_are_one_launch(dev, hq, hkv, d):
    # every token's rows fit one form: a batch of them has the workspace of that form alone, as a single request has
    from sanic_b200 import abi
    x = torch.zeros(16, dtype=torch.int32, device=dev.torch_device).data_ptr()

    def size(n, maxq):      # nothing is launched: the addresses are only looked at
        p = abi.AttnPagedParams(x, x, None, x, x, x, x, x, None, 0, hq * d, d, 16 * hkv * d, hkv * d, d, 16 * hkv * d, hkv * d, d, 4, abi.BF16, n, n * maxq,
                                maxq, hq, hkv, d, 16, 4 * n, 4, 0, 1.0)
        return dev.lib.sanic_attn_paged_workspace_bytes(dev.h, C.byref(p))

    assert size(1, 1) == size(2, 1) == size(1000, 1) > 0
    assert size(2, 2) > size(1, 2)                        # single tokens beside chunks of two: two launches
    ctx = [0, 700, 31, 32, 5, 2000]
    run_case(dev, [1] * 6, ctx, hq, hkv, d, "bf16", 16, seed=hq)
    run_case(dev, [1, 1, 3, 1, 0, 1], ctx, hq, hkv, d, "f16", 16, seed=hq, max_query_len=1)        # the hint is too small


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 400, 2 ** 63 - 1])
@pytest.mark.parametrize("maxq", [1, 300])
def test_attn_windows_wider_than_the_table(dev, window, maxq):
    # and more tokens than keys, so that the first positions are negative
    from sanic_b200 import RunError
    args, keys, values = make_problem(dev, [40, 9], [0, 30], 4, 2, 64, "bf16", 16, seed=19)
    args["kv_lens"] = ints(dev, [25, 39])
    got, lse = dev.attn_paged(**args, max_query_len=maxq, window=window, return_lse=True)
    dev.sync()
    check_attention(got, lse, *plain_attention(args["q"], [keys[0][:25], keys[1]], [values[0][:25], values[1]], [40, 9], [25, 39], 0, 0.125))
    wide = torch.zeros(1, (2 ** 31 - 300) // 16, dtype=torch.int32, device=dev.torch_device)       # positions would pass 32 bits
    with pytest.raises(RunError, match="2\\^31 keys"):
        dev.attn_paged(args["q"], args["k_pages"], args["v_pages"], wide, ints(dev, [0, 49]), ints(dev, [49]))


FIRST_IN_CAPTURE = r'''
import torch
from sanic_b200 import CudaDevice
dev = CudaDevice(0)
z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
kp, vp, table, free = z(8, 16, 2, 64), z(8, 16, 2, 64), i32([[0, 0], [0, 0]]), i32([7, 6, 5, 4, 3, 2, 1, 0])
seq, new, count = i32([0, 0]), i32([20, 3]), i32([8])
k, q = torch.randn(23, 2, 64, device="cuda").bfloat16(), torch.randn(23, 4, 64, device="cuda").bfloat16()
probs, drafts, ua, us = torch.full((4, 50), 0.02, device="cuda"), i32([[1], [2]]), z(2, 1, t=torch.float32), z(2, t=torch.float32)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    step = dev.page_table_append(seq, new, table, free, count, 16, 23)
    qr = dev.paged_cache_write(k, k, kp, vp, step.slots, q=q)
    a = dev.attn_paged(qr, kp, vp, table, step.query_start, step.kv_lens, max_query_len=20)
    b = dev.attn_paged(qr, kp, vp, table, step.query_start, step.kv_lens, max_query_len=1)
    t, n = dev.draft_verify(probs, drafts, ua, us)
for _ in range(3):
    g.replay()
torch.cuda.synchronize()
dev.sync()
assert torch.equal(a[0], b[0]) and torch.isfinite(a.float()).all() and (a.float() - b.float()).abs().max() < 0.05
assert n.tolist() == [1, 1] and table.tolist() == [[0, 1], [2, 0]], (n, table)
print("captured")
'''


def test_first_calls_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE], cwd=root, capture_output=True, text=True, timeout=180)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("code,what", [(53, "page_table_append"), (54, "attn_paged"), (55, "draft_verify"), (56, "paged_cache_write")])
def test_status_codes_name_their_operator(dev, code, what):
    from sanic_b200 import RunError
    assert dev.lib.sanic_status_inject(dev.h, code) == 0
    with pytest.raises(RunError, match=what):
        dev.sync()
    dev.sync()


@pytest.mark.parametrize("maxq", [1, 64])
def test_attn_bad_pages_and_lengths_are_reported(dev, maxq):
    from sanic_b200 import RunError
    args, keys, values = make_problem(dev, [1, 40], [100, 30], 4, 2, 64, "bf16", 16, seed=12)
    good = dev.attn_paged(**args, max_query_len=maxq)
    dev.sync()
    for entry in (-1, args["k_pages"].shape[0], 1 << 30):
        bad = args["block_table"].clone()
        bad[0, 2] = entry
        got = dev.attn_paged(**dict(args, block_table=bad), max_query_len=maxq)
        with pytest.raises(RunError, match="code 54"):
            dev.sync()
        assert torch.equal(got[1:], good[1:]) and torch.isfinite(got[0]).all()       # the other request is untouched; zeros are read instead
    for name, val in (("kv_lens", [101, 1 << 30]), ("kv_lens", [-5, 70]), ("query_start", [0, 1, 500]), ("query_start", [-3, 1, 41])):
        dev.attn_paged(**dict(args, **{name: ints(dev, val)}), max_query_len=maxq)
        with pytest.raises(RunError, match="code 54"):
            dev.sync()
    assert torch.equal(dev.attn_paged(**args, max_query_len=maxq), good)
    dev.sync()


def test_attn_refusals(dev):
    from sanic_b200 import CompileError, RunError
    args, _, _ = make_problem(dev, [2], [20], 4, 2, 64, "bf16", 16)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev.torch_device)
    with pytest.raises(CompileError, match="head_dim"):
        dev.attn_paged(z(2, 4, 96), z(3, 16, 2, 96), z(3, 16, 2, 96), args["block_table"], args["query_start"], args["kv_lens"])
    with pytest.raises(RunError, match="multiple"):
        dev.attn_paged(z(2, 3, 64), args["k_pages"], args["v_pages"], args["block_table"], args["query_start"], args["kv_lens"])
    with pytest.raises(CompileError, match="64 query heads"):
        dev.attn_paged(z(2, 130, 64), args["k_pages"], args["v_pages"], args["block_table"], args["query_start"], args["kv_lens"])
    with pytest.raises(RunError, match="scale"):
        dev.attn_paged(**args, scale=0.0)
    with pytest.raises(RunError, match="window"):
        dev.attn_paged(**args, window=-1)
    with pytest.raises(RunError, match="16-byte"):
        dev.attn_paged(**dict(args, q=z(2 * 4 * 64 + 1)[1:].view(2, 4, 64)))
    with pytest.raises(RunError, match="not a tensor on"):
        dev.attn_paged(**dict(args, q=args["q"].cpu()))
    from sanic_b200 import abi
    p = abi.AttnPagedParams()
    assert dev.lib.sanic_attn_paged_workspace_bytes(dev.h, C.byref(p)) == 0


def test_attn_nothing_to_do(dev):
    args, _, _ = make_problem(dev, [0, 0], [20, 0], 4, 2, 64, "bf16", 16)
    assert dev.attn_paged(**args).shape == (0, 4, 64)
    args["q"] = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=dev.torch_device)
    out = torch.full((3, 4, 64), 2.0, dtype=torch.bfloat16, device=dev.torch_device)
    dev.attn_paged(**args, out=out)
    dev.sync()
    assert (out == 2.0).all()


@pytest.mark.parametrize("maxq", [1, 200])
def test_attn_is_deterministic_and_runs_on_other_streams(dev, maxq):
    args, _, _ = make_problem(dev, [1, 200, 3], [3000, 10, 40], 8, 2, 128, "bf16", 16, seed=13)
    first = dev.attn_paged(**args, max_query_len=maxq, return_lse=True)
    dev.sync()
    side = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for i in range(12):
        with torch.cuda.stream(side[i % 3]):
            results.append(dev.attn_paged(**args, max_query_len=maxq, return_lse=True))
    torch.cuda.synchronize()
    for r in results:
        assert torch.equal(r[0], first[0]) and torch.equal(r[1], first[1])


@pytest.mark.parametrize("maxq", [1, 40])
def test_attn_captured_twice_replays_side_by_side_over_new_lengths(dev, maxq):
    sets = [make_problem(dev, [1, 40, 1], [900, 5, 60], 8, 2, 64, "f16", 16, seed=20 + i) for i in range(2)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for args, _, _ in sets:
        dev.attn_paged(**args, max_query_len=maxq)
    torch.cuda.synchronize()
    for i, (args, _, _) in enumerate(sets):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(dev.attn_paged(**args, max_query_len=maxq, return_lse=True))
        graphs.append(g)
    for kv in ([901, 45, 61], [350, 45, 17], [1, 45, 61]):
        for args, _, _ in sets:
            args["kv_lens"].copy_(ints(dev, kv))
        torch.cuda.synchronize()
        for _ in range(4):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for (args, keys, values), (got, lse) in zip(sets, outs):
            check_attention(got, lse, *plain_attention(args["q"], [k[:n] for k, n in zip(keys, kv)], [v[:n] for v, n in zip(values, kv)],
                                                       [1, 40, 1], kv, 0, 0.125))


# ───────────────────────── page tables ─────────────────────────
def plain_append(seq, new, held, table, free, count, page, n_tokens):
    table = table.copy()
    max_pages = table.shape[1]
    start, kv, pages, pos, slots, bad = [0], [], [], [], [], False
    left = count
    for b, (s, n) in enumerate(zip(seq, new)):
        s, n, h = max(s, 0), max(n, 0), held[b]
        need = -(-(s + n) // page)
        bad |= need > max_pages or seq[b] < 0 or new[b] < 0
        got = h
        for col in range(h, min(need, max_pages)):
            if left > 0:
                left -= 1
                table[b, col] = free[left]
                got += 1
            else:
                table[b, col] = -1
                bad = True
        pages.append(got)
        kv.append(min(s + n, (1 << 31) - 1))
        for i in range(n):
            if len(pos) >= n_tokens:
                bad = True
                break
            p = s + i
            e = table[b, p // page] if p // page < max_pages else -1
            pos.append(min(p, (1 << 31) - 1))
            slots.append(-1 if e < 0 else int(e) * page + p % page)
        start.append(len(pos))
    rest = n_tokens - len(pos)
    return table, start, kv, pages, left, pos + [0] * rest, slots + [-1] * rest, bad


def check_append(dev, seq, new, page, max_pages, count, n_tokens, held=None, capacity=None, seed=0):
    from sanic_b200 import RunError
    r = np.random.default_rng(seed)
    h = held if held is not None else [min(-(-max(s, 0) // page), max_pages) for s in seq]
    ids = r.permutation(sum(h) + (capacity or count) + 5).astype(np.int32)
    table = np.full((len(seq), max_pages), -7, np.int32)
    at = 0
    for b, n in enumerate(h):
        table[b, :n] = ids[at:at + n]
        at += n
    free = ids[at:at + (capacity or count)]
    want = plain_append(seq, new, h, table, free, count, page, n_tokens)
    t = ints(dev, table.tolist()) if len(seq) else torch.zeros(0, max_pages, dtype=torch.int32, device=dev.torch_device)
    got = dev.page_table_append(ints(dev, seq), ints(dev, new), t, ints(dev, free.tolist()), ints(dev, [count]), page, n_tokens,
                                held_pages=None if held is None else ints(dev, held))
    if want[-1]:
        with pytest.raises(RunError, match="code 53"):
            dev.sync()
    else:
        dev.sync()
    assert t.cpu().numpy().tolist() == want[0].tolist()
    for g, w in zip(got, (want[1], want[2], want[3], [want[4]], want[5], want[6])):
        assert g.tolist() == list(w)
    return t, got


@pytest.mark.parametrize("page", [1, 16, 24, 256])
@pytest.mark.parametrize("n", [1, 3, 300, 1100])
def test_append_random(dev, page, n):
    r = np.random.default_rng(page * 1000 + n)
    seq = r.integers(0, 5 * page + 20, n)
    new = r.integers(0, 3 * page + 3, n) * (r.random(n) < 0.7)
    seq[r.random(n) < 0.2] = 0
    need = sum(-(-int(s + x) // page) - -(-int(s) // page) for s, x in zip(seq, new))
    check_append(dev, seq.tolist(), new.tolist(), page, 9 + 24 // page + (20 if page == 1 else 0), need + 5, int(new.sum()) + 13, seed=n)


def test_append_edges(dev):
    check_append(dev, [], [], 16, 4, 3, 0)                                       # no requests at all
    check_append(dev, [], [], 16, 4, 3, 5)
    check_append(dev, [0, 0, 0], [0, 0, 0], 16, 4, 0, 4, capacity=0 or 2)         # nothing appended: every row is padding
    check_append(dev, [15, 16, 17], [1, 1, 1], 16, 4, 1, 3)                       # the last row of a page, the first of a new one, inside one
    check_append(dev, [31, 5], [1, 4], 16, 6, 4, 5, held=[4, 3])                  # more pages held than the tokens need: a rolled-back draft keeps them
    check_append(dev, [20], [60], 16, 5, 3, 60, held=[2])
    check_append(dev, [8000 * 16 - 3], [5], 16, 8001, 4, 5)


def test_append_shortages_are_reported(dev):
    check_append(dev, [16, 30, 0], [40, 10, 33], 16, 6, 4, 83)                    # the free list ends inside the last request
    check_append(dev, [16, 30], [40, 10], 16, 6, 0, 50, capacity=3)               # an empty one
    check_append(dev, [60, 10], [30, 3], 16, 4, 8, 33)                            # a table row too short
    check_append(dev, [3, 3, 3], [10, 10, 10], 16, 4, 8, 17)                      # more new tokens than token rows
    check_append(dev, [-4, 9], [3, -2], 16, 4, 8, 6)                              # negative lengths read as 0
    check_append(dev, [(1 << 31) - 5, 3], [9, 4], 16, 4, 8, 13, held=[1, 1])      # a length that nearly wraps: no page, no slot
    check_append(dev, [(1 << 31) - 5, 3], [9, 4], 1, 4, 8, 13, held=[1, 1])       # the same where a position is a page
    check_append(dev, [5], [2], 16, 4, 8, 2)                                      # and the next call is clean again


@pytest.mark.parametrize("n", [2, 700])
def test_append_counts_and_entries_out_of_range_are_reported(dev, n):
    # the last two requests are looked at, behind none or more than a block's worth of others that append nothing
    from sanic_b200 import RunError
    td = dev.torch_device

    def step(held=(1, 1), count=4, free=(40, 41, 42, 43), entry=7, report=True, seq=(15, 16), new=(3, 2)):
        pad = n - 2
        table = torch.full((n, 4), -7, dtype=torch.int32, device=td)
        table[pad, 0], table[pad + 1, 0] = entry, 9
        got = dev.page_table_append(ints(dev, [0] * pad + list(seq)), ints(dev, [0] * pad + list(new)), table, ints(dev, list(free)), ints(dev, [count]),
                                    16, sum(new), held_pages=ints(dev, [0] * pad + list(held)))
        if report:
            with pytest.raises(RunError, match="code 53"):
                dev.sync()
        dev.sync()
        assert got.query_start.tolist()[pad:] == [0, new[0], new[0] + new[1]]
        return table[pad:].tolist(), got.held_pages.tolist()[pad:], got.free_count.item(), got.slots.tolist()

    good = [[7, 43, -7, -7], [9, 42, -7, -7]], [2, 2], 2, [7 * 16 + 15, 43 * 16, 43 * 16 + 1, 42 * 16, 42 * 16 + 1]
    assert step(report=False) == good
    # a count of free pages outside the list: nothing is read behind it, none taken in front of it
    assert step(count=9) == good
    assert step(count=-1) == ([[7, -1, -7, -7], [9, -1, -7, -7]], [1, 1], 0, [7 * 16 + 15, -1, -1, -1, -1])
    # counts of held pages outside a table row: the nearest count inside it
    assert step(held=(-2, 1)) == ([[43, 42, -7, -7], [9, 41, -7, -7]], [2, 2], 1, [43 * 16 + 15, 42 * 16, 42 * 16 + 1, 41 * 16, 41 * 16 + 1])
    assert step(held=(1, 5))[:3] == ([[7, 43, -7, -7], [9, -7, -7, -7]], [2, 4], 3)
    # a negative page that a new token would use: no slot; one that no new token uses is not looked at
    assert step(entry=-1) == ([[-1, 43, -7, -7], [9, 42, -7, -7]], [2, 2], 2, [-1, 43 * 16, 43 * 16 + 1, 42 * 16, 42 * 16 + 1])
    assert step(entry=-1, seq=(16, 16), new=(2, 2), report=False)[3] == [43 * 16, 43 * 16 + 1, 42 * 16, 42 * 16 + 1]
    # a negative page on the free list: a missing one
    assert step(free=(40, 41, 42, -3)) == ([[7, -1, -7, -7], [9, 42, -7, -7]], [2, 2], 2, [7 * 16 + 15, -1, -1, 42 * 16, 42 * 16 + 1])
    assert step(report=False) == good


def test_append_with_an_empty_free_list(dev):
    # a list without any memory: enough where no request needs a page
    from sanic_b200 import RunError
    none = torch.zeros(0, dtype=torch.int32, device=dev.torch_device)
    for new, want, held in (([1, 0], [7 * 16 + 15], [1, 2]), ([2, 0], [7 * 16 + 15, -1], [1, 2])):
        table = ints(dev, [[7, -7], [8, 9]])
        got = dev.page_table_append(ints(dev, [15, 20]), ints(dev, new), table, none, ints(dev, [0]), 16, sum(new))
        if -1 in want:
            with pytest.raises(RunError, match="code 53"):
                dev.sync()
        dev.sync()
        assert got.slots.tolist() == want and got.held_pages.tolist() == held and got.free_count.item() == 0
        assert table.tolist() == [[7, -1 if -1 in want else -7], [8, 9]]


def test_append_refusals(dev):
    from sanic_b200 import RunError
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev.torch_device)
    args = dict(seq_lens=z(2), new_lens=z(2), block_table=z(2, 4), free_pages=z(5), free_count=z(1), page_size=16, n_tokens=4)
    with pytest.raises(RunError, match="empty pages"):
        dev.page_table_append(**dict(args, page_size=0))
    with pytest.raises(RunError, match="8000"):
        dev.page_table_append(**dict(args, seq_lens=z(8001), new_lens=z(8001), block_table=z(8001, 4)))
    t = z(12)
    with pytest.raises(RunError, match="overlaps"):
        dev.page_table_append(**dict(args, block_table=t[:8].view(2, 4), seq_lens=t[6:8]))
    from sanic_b200 import abi
    x = t.data_ptr()
    for max_pages, capacity in (((1 << 30) + 1, 4), (4, (1 << 30) + 1)):          # refused, nothing is read
        p = abi.PageAppendParams(x, x, None, x, x, x, max_pages, x, x, x, x, x, x, 2, 4, 16, max_pages, capacity)
        with pytest.raises(RunError, match="too many pages"):
            dev._check(dev.lib.sanic_page_table_append(dev.h, C.byref(p), dev.stream()), "page_table_append")


APPEND_COUNTS = r'''
import threading
import torch
from sanic_b200 import CudaDevice

def step(dev, n, stream=None):
    """n requests of one new token each, a page each off the end of the free list."""
    i32 = dict(dtype=torch.int32, device="cuda")
    seq, new, table = torch.zeros(n, **i32), torch.ones(n, **i32), torch.full((n, 2), -1, **i32)
    free = torch.arange(n, **i32)
    got = dev.page_table_append(seq, new, table, free, torch.full((1,), n, **i32), 16, n)
    dev.sync()
    assert table[:, 0].tolist() == list(range(n - 1, -1, -1)) and (table[:, 1] == -1).all()
    assert got.query_start.tolist() == list(range(n + 1)) and got.free_count.item() == 0
    assert got.slots.tolist() == [16 * (n - 1 - b) for b in range(n)]

dev = CudaDevice(0)
for n in COUNTS:
    step(dev, n)
failed = []
def many(counts):
    try:
        mine = CudaDevice(0)
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(15):
                for n in counts:
                    step(mine, n)
    except BaseException as e:
        failed.append(e)
threads = [threading.Thread(target=many, args=(c,)) for c in ((6200, 7000), (8000, 6500), (7999, 6144))]
for t in threads: t.start()
for t in threads: t.join()
assert not failed, failed
print("appended")
'''


@pytest.mark.parametrize("counts", [(6127, 6128), (6135,), (6143, 6144), (8000, 6140)])
def test_append_counts_around_the_default_shared_memory(counts):
    # the first calls of a process: no larger call has raised the kernel's limit before; then threads with counts of their own
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", APPEND_COUNTS.replace("COUNTS", repr(counts))], cwd=root, capture_output=True, text=True, timeout=180)
    assert r.returncode == 0 and "appended" in r.stdout, r.stderr[-2000:]


# ───────────────────────── cache writes ─────────────────────────
def check_write(dev, t, hq, hkv, d, src, cache, page, heads_first=False, fused=False, rope=True, with_q=True, in_place=False, seed=0):
    g = gen(dev, seed)
    td = dev.torch_device
    S = torch.float32 if src == "f32" else DT[src]
    n_pages = -(-t // page) + 2
    rows = torch.randn(t, hq + 2 * hkv, d, generator=g, device=td).to(S)
    q, k, v = rows.split([hq, hkv, hkv], 1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    shape = (n_pages, hkv, page, d) if heads_first else (n_pages, page, hkv, d)
    kp, vp = (torch.randn(shape, generator=g, device=td).to(DT[cache]) for _ in range(2))
    if heads_first:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    kp0, vp0 = kp.clone(), vp.clone()
    slots = torch.randperm(n_pages * page, generator=g, device=td)[:t]
    skip = torch.rand(t, generator=g, device=td) < 0.2
    slots[skip] = -1
    table = dev.rope_table([500000.0 ** (-i / (d // 2)) for i in range(d // 2)], 97)
    pos = torch.randint(0, 97, (t,), generator=g, device=td, dtype=torch.int32)
    out = q if in_place else torch.full((t, hq, d), 9.0, dtype=DT[cache], device=td)
    got = dev.paged_cache_write(k, v, kp, vp, slots, q=q if with_q else None, positions=pos if rope else None,
                                rope_table=table if rope else None, q_out=out if with_q else None)
    dev.sync()
    cs = table.double()[pos.long()][:, None]
    u, tiny = torch.finfo(DT[cache]).eps / 2, 2.0 ** -25

    def want(x):
        a, b = x.double().chunk(2, -1)
        if not rope:
            return x.double(), torch.zeros_like(x, dtype=torch.float64)
        w = torch.cat([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], -1)
        return w, (a.abs() + b.abs()).repeat(1, 1, 2)

    def close(x, w, size):
        return ((x.double() - w).abs() <= u * w.abs() + 2.0 ** -22 * size + tiny).all()

    keep = ~skip
    pg, row = slots // page, slots % page
    wk, sk = want(k0)
    assert close(kp[pg[keep], row[keep]], wk[keep], sk[keep])
    assert torch.equal(vp[pg[keep], row[keep]], v0[keep].to(DT[cache]))
    touched = torch.zeros(n_pages * page, dtype=torch.bool, device=td)
    touched[slots[keep]] = True
    left = ~touched.view(n_pages, page)
    assert torch.equal(kp[left], kp0[left]) and torch.equal(vp[left], vp0[left])
    if with_q:
        assert got.data_ptr() == out.data_ptr()
        wq, sq = want(q0)
        assert close(got[keep], wq[keep], sq[keep])
        assert torch.equal(got[skip], q0[skip] if in_place else torch.full_like(got[skip], 9.0))
    else:
        assert got is None


@pytest.mark.parametrize("d", [16, 64, 128, 256])
@pytest.mark.parametrize("src,cache", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("t", [1, 7, 300])
def test_write(dev, d, src, cache, t):
    check_write(dev, t, 5, 2, d, src, cache, 16, heads_first=t == 7, fused=d == 64, seed=t + d)


def test_write_forms(dev):
    check_write(dev, 33, 4, 4, 64, "bf16", "bf16", 1)
    check_write(dev, 33, 4, 1, 128, "f16", "f16", 24, rope=False)
    check_write(dev, 33, 4, 2, 128, "f32", "f16", 64, with_q=False)
    check_write(dev, 33, 4, 2, 128, "bf16", "bf16", 64, in_place=True)
    check_write(dev, 33, 4, 2, 64, "bf16", "bf16", 16, in_place=True, fused=True)
    check_write(dev, 2500, 32, 8, 64, "bf16", "bf16", 16)


@pytest.mark.parametrize("src,cache", [("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("t,hq,hkv,d", [(5003, 32, 8, 128), (401, 64, 40, 256), (40001, 1, 1, 16), (9001, 5, 3, 48)])
def test_write_more_tokens_than_resident_blocks(dev, src, cache, t, hq, hkv, d):
    check_write(dev, t, hq, hkv, d, src, cache, 16, fused=src == "bf16", in_place=src == "bf16", seed=t)


def test_write_out_of_range_is_reported_and_skipped(dev):
    from sanic_b200 import RunError
    td = dev.torch_device
    k = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=td)
    kp, vp = (torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=td) for _ in range(2))
    table = dev.rope_table([1.0] * 32, 10)
    for slots, pos in (([0, 64, 1], [0, 1, 2]), ([0, 1 << 40, 1], [0, 1, 2]), ([0, 5, 1], [0, 10, 2]), ([0, 5, 1], [0, -1, 2])):
        kp.zero_(); vp.zero_()
        dev.paged_cache_write(k, k, kp, vp, ints(dev, slots, torch.int64), positions=ints(dev, pos), rope_table=table)
        with pytest.raises(RunError, match="code 56"):
            dev.sync()
        assert (vp.flatten(0, 1)[[0, 1]] == 1).all() and vp.sum() == 2 * 128


def test_write_refusals(dev):
    from sanic_b200 import CompileError, RunError
    td = dev.torch_device
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=td)
    slots = z(2, t=torch.int64)
    with pytest.raises(CompileError, match="head_dim"):
        dev.paged_cache_write(z(2, 1, 24), z(2, 1, 24), z(3, 16, 1, 24), z(3, 16, 1, 24), slots)
    with pytest.raises(RunError, match="16-byte"):
        dev.paged_cache_write(z(2 * 64 + 4)[4:].view(2, 1, 64), z(2, 1, 64), z(3, 16, 1, 64), z(3, 16, 1, 64), slots)
    dev.paged_cache_write(z(0, 1, 64), z(0, 1, 64), z(3, 16, 1, 64), z(3, 16, 1, 64), z(0, t=torch.int64))


# ───────────────────────── draft verification ─────────────────────────
def plain_verify(target, tokens, ua, us, draft, lens, start):
    n, k = tokens.shape
    out, counts, margin = [], [], math.inf
    for b in range(n):
        row, c = [], 0
        while c < lens[b]:
            x = int(tokens[b, c])
            p = float(target[start[b] + c, x])
            q = 1.0 if draft is None else float(draft[b, c, x])
            if not float(ua[b, c]) * q < p:
                break
            row.append(x)
            c += 1
        valid = lambda w: np.where(np.isfinite(w) & (w > 0), w, 0.0)      # NaN, infinite and non-positive weights count as 0
        w = target[start[b] + c].astype(np.float64)
        if c < lens[b]:
            r = w.copy()
            if draft is None:
                r[int(tokens[b, c])] = 0.0
            else:
                r = w - draft[b, c].astype(np.float64)
            if valid(r).any():
                w = r
        w = valid(w)
        cum = np.cumsum(w)
        if cum[-1] > 0:
            x = float(us[b]) * cum[-1]
            j = min(int(np.searchsorted(cum, x, side="right")), int(np.flatnonzero(w)[-1]))
            margin = min(margin, np.min(np.abs(cum - x)) / cum[-1])
            row.append(j)
        else:
            row.append(-1)
        out.append(row + [-1] * (k + 1 - len(row)))
        counts.append(c)
    return out, counts, margin


def check_verify(dev, n, k, vocab, probs=True, ragged=False, packed=False, seed=0, tweak=None):
    r = np.random.default_rng(seed)
    soft = lambda x: (np.exp(x) / np.exp(x).sum(-1, keepdims=True)).astype(np.float32)
    lens = r.integers(0, k + 1, n).tolist() if ragged else [k] * n
    if packed:
        start = np.concatenate([[0], np.cumsum([x + 1 for x in lens])])
        start, rows = start[:-1].tolist(), int(start[-1])
    else:
        start, rows = [b * (k + 1) for b in range(n)], n * (k + 1)
    logits = r.normal(size=(rows, vocab)) * 2
    target = soft(logits)
    draft = np.zeros((n, k, vocab), np.float32)
    tokens = np.zeros((n, k), np.int32)
    for b in range(n):
        for i in range(k):
            draft[b, i] = soft(logits[min(start[b] + i, rows - 1)] + 0.8 * r.normal(size=vocab))
            tokens[b, i] = r.choice(vocab, p=draft[b, i].astype(np.float64) / draft[b, i].astype(np.float64).sum())
    ua, us = r.random((n, k)).astype(np.float32), r.random(n).astype(np.float32)
    ua, us = np.minimum(ua, np.float32(1 - 2 ** -24)), np.minimum(us, np.float32(1 - 2 ** -24))
    if tweak:
        tweak(target, draft, tokens, ua, us)
    want, counts, margin = plain_verify(target, tokens, ua, us, draft if probs else None, lens, start)
    up = lambda a: torch.tensor(a, device=dev.torch_device)
    got, acc = dev.draft_verify(up(target), up(tokens), up(ua), up(us), draft_probs=up(draft) if probs else None,
                                draft_lens=ints(dev, lens) if ragged else None, target_start=ints(dev, start) if packed else None)
    dev.sync()
    assert acc.tolist() == counts
    assert got.tolist() == want, (got.tolist(), want, margin)
    return got, acc


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("n,k,vocab", [(1, 4, 1), (1, 4, 2), (3, 1, 127), (5, 3, 129), (2, 8, 2048), (2, 5, 2049), (7, 2, 10007), (1, 6, 128256),
                                       (40, 3, 5000), (300, 2, 333), (3, 0, 500), (2, 32, 700)])
def test_verify(dev, n, k, vocab, probs):
    check_verify(dev, n, k, vocab, probs, seed=n + k)
    check_verify(dev, n, k, vocab, probs, ragged=True, packed=True, seed=n + k + 1)


def test_verify_takes_every_branch_and_the_exact_borders(dev):
    # dyadic probabilities: products and sums are exact, so borders are hit on the nose
    def tweak(target, draft, tokens, ua, us):
        target[:] = 0.0
        target[:, 1], target[:, 3], target[:, 6] = 0.25, 0.5, 0.25
        draft[:] = 0.0
        draft[:, :, 3], draft[:, :, 5] = 0.5, 0.5
        tokens[:] = 3
        ua[:] = 0.5
        us[:] = [0.0, 0.25, 0.75, np.float32(1 - 2 ** -24)] * 2
        tokens[4:, 1] = 5                    # p = 0: rejected; left over: 1 and 6 at 0.25 each
        tokens[7, 0], ua[7, 0] = 1, 0.0      # q = 0, u = 0: 0 < 0.25 holds
    got, acc = check_verify(dev, 8, 2, 8, tweak=tweak)
    assert acc.tolist() == [2, 2, 2, 2, 1, 1, 1, 1]
    assert [row[c] for row, c in zip(got.tolist(), acc.tolist())] == [1, 3, 6, 6, 1, 1, 6, 6]

    def equal(target, draft, tokens, ua, us):          # u q = p is a rejection; p - q leaves nothing: p itself is drawn from
        target[:] = 1.0 / 8
        draft[:] = 1.0 / 4
        ua[:] = 0.5
    check_verify(dev, 3, 2, 8, tweak=equal)


def test_verify_odd_weights(dev):
    def tweak(target, draft, tokens, ua, us):
        target[:, 5] = np.nan
        target[:, 7] = np.inf
        target[:, 9] = -1.0
        target[-1] = 0.0                               # nothing to draw from: -1
        tokens[0, 0], tokens[1, 0] = 5, 9              # NaN and negative: rejected
    got, acc = check_verify(dev, 4, 2, 600, probs=False, tweak=tweak)
    assert acc.tolist()[:2] == [0, 0]
    check_verify(dev, 4, 2, 600, tweak=tweak)


def test_verify_unaligned_rows(dev):
    r = np.random.default_rng(5)
    flat = torch.rand(4 * 1003 + 1, device=dev.torch_device)
    target = flat[1:].view(4, 1003)
    tokens = ints(dev, r.integers(0, 1003, (1, 3)).tolist())
    ua, us = torch.zeros(1, 3, device=dev.torch_device), torch.full((1,), 0.37, device=dev.torch_device)
    got, acc = dev.draft_verify(target, tokens, ua, us)
    dev.sync()
    want, counts, _ = plain_verify(target.cpu().numpy(), tokens.cpu().numpy(), ua.cpu().numpy(), us.cpu().numpy(), None, [3], [0])
    assert got.tolist() == want and acc.tolist() == counts


def test_verify_one_draft_whatever_its_stride(dev):
    # one drafted token: the stride between a request's drafts is never used; requests may share one row of probabilities
    n, vocab, td = 3, 700, dev.torch_device
    g = gen(dev, 31)
    target = torch.softmax(torch.randn(2 * n, vocab, generator=g, device=td), -1)
    rows = torch.softmax(torch.randn(n, vocab, generator=g, device=td), -1)
    tokens = ints(dev, [[5], [699], [0]])
    ua, us = torch.full((n, 1), 0.999, device=td), torch.full((n,), 0.6, device=td)
    for probs in (rows.as_strided((n, 1, vocab), (vocab, 1, 1)), rows[:1].as_strided((n, 1, vocab), (0, 0, 1))):
        got, acc = dev.draft_verify(target, tokens, ua, us, draft_probs=probs)
        dev.sync()
        want, counts, _ = plain_verify(target.cpu().numpy(), tokens.cpu().numpy(), ua.cpu().numpy(), us.cpu().numpy(),
                                       probs.cpu().contiguous().numpy(), [1] * n, [2 * b for b in range(n)])
        assert got.tolist() == want and acc.tolist() == counts


def test_verify_out_of_range_is_reported(dev):
    from sanic_b200 import CompileError, RunError
    td = dev.torch_device
    target = torch.full((6, 40), 1 / 40, device=td)
    ua, us = torch.zeros(2, 2, device=td), torch.full((2,), 0.5, device=td)
    ok = ints(dev, [[1, 2], [3, 4]])
    for tokens in ([[1, 40], [3, 4]], [[1, -1], [3, 4]]):
        got, acc = dev.draft_verify(target, ints(dev, tokens), ua, us)
        with pytest.raises(RunError, match="code 55"):
            dev.sync()
        assert acc.tolist() == [1, 2] and got[0].tolist() == [1, 20, -1] and got[1, :2].tolist() == [3, 4]
    got, acc = dev.draft_verify(target, ok, ua, us, draft_lens=ints(dev, [7, -2]))
    with pytest.raises(RunError, match="code 55"):
        dev.sync()
    assert acc.tolist() == [2, 0]
    for start in ([0, 4], [-1, 3]):
        got, acc = dev.draft_verify(target, ok, ua, us, target_start=ints(dev, start))
        with pytest.raises(RunError, match="code 55"):
            dev.sync()
        bad = 1 if start[0] == 0 else 0
        assert acc[bad] == 0 and got[bad].tolist() == [-1, -1, -1] and acc[1 - bad] == 2
    with pytest.raises(CompileError, match="32 drafted"):
        dev.draft_verify(torch.zeros(34, 8, device=td), torch.zeros(1, 33, dtype=torch.int32, device=td), torch.zeros(1, 33, device=td), us[:1])
    from sanic_b200 import abi
    x = target.data_ptr()
    p = abi.DraftVerifyParams(x, 40, 6, None, None, 0, 0, x, None, x, x, x, x, 1 << 26, 31, 40)      # 2^31 rows: refused, nothing is read
    with pytest.raises(RunError, match="too many rows"):
        dev._check(dev.lib.sanic_draft_verify(dev.h, C.byref(p), dev.stream()), "draft_verify")
    got, acc = dev.draft_verify(target, ok, ua, us)
    dev.sync()
    assert acc.tolist() == [2, 2]


# ───────────────────────── the operators together ─────────────────────────
@pytest.mark.parametrize("captured", [False, True])
def test_a_speculative_serving_loop(dev, captured):
    """Admission of prompts, then steps of up to three drafted tokens per request with rejections, over one page pool: lengths
    go from verification straight into the next step's page tables, on the device. Checked each step against plain attention
    over caches kept contiguously on the side, and the table against every other request's pages."""
    td = dev.torch_device
    n, hq, hkv, d, page, vocab, K = 5, 8, 2, 64, 16, 200, 3
    g = gen(dev, 77)
    dt = torch.bfloat16
    emb = {x: torch.randn(vocab, h, d, generator=g, device=td).to(dt) for x, h in (("q", hq), ("k", hkv), ("v", hkv))}
    head = torch.randn(hq * d, vocab, generator=g, device=td) * 0.3
    n_pages = 60
    kp, vp = (torch.full((n_pages, page, hkv, d), float("nan"), dtype=dt, device=td) for _ in range(2))
    table = torch.full((n, 12), -1, dtype=torch.int32, device=td)
    free = torch.randperm(n_pages, generator=g, device=td).to(torch.int32)
    rope = dev.rope_table([10000.0 ** (-i / (d // 2)) for i in range(d // 2)], 12 * page)
    state = dict(seq=torch.zeros(n, dtype=torch.int32, device=td), held=torch.zeros(n, dtype=torch.int32, device=td), count=ints(dev, [n_pages]))
    caches = [[torch.zeros(0, hkv, d, device=td) for _ in range(2)] for _ in range(n)]

    def forward(tokens, new, n_tokens, maxq):
        step = dev.page_table_append(state["seq"], new, table, free, state["count"], page, n_tokens, held_pages=state["held"])
        q = dev.paged_cache_write(emb["k"][tokens], emb["v"][tokens], kp, vp, step.slots, q=emb["q"][tokens], positions=step.positions, rope_table=rope)
        return step, q, *dev.attn_paged(q, kp, vp, table, step.query_start, step.kv_lens, max_query_len=maxq, return_lse=True)

    def check(step, tokens, new, seq, q, out, lse):
        starts = step.query_start.tolist()
        for b in range(n):
            t = tokens[starts[b]:starts[b + 1]]
            cs = rope.double()[step.positions[starts[b]:starts[b + 1]].long()][:, None]
            a, c = emb["k"][t].double().chunk(2, -1)
            turned = torch.cat([a * cs[..., 0] - c * cs[..., 1], c * cs[..., 0] + a * cs[..., 1]], -1)
            # the written keys are within one rounding of these; the kernel's own values go on
            mine = kp[step.slots[starts[b]:starts[b + 1]] // page, step.slots[starts[b]:starts[b + 1]] % page]
            assert ((mine.double() - turned).abs() <= 2.0 ** -8 * turned.abs() + 2.0 ** -19).all()
            caches[b][0] = torch.cat([caches[b][0][:seq[b]], mine.float()])
            caches[b][1] = torch.cat([caches[b][1][:seq[b]], emb["v"][t].float()])
        total = starts[-1]
        want, amp, wl = plain_attention(q[:total], [c[0] for c in caches], [c[1] for c in caches], new, step.kv_lens.tolist(), 0, d ** -0.5)
        check_attention(out[:total], lse[:total], want, amp, wl)
        owned = [table[b, :h].tolist() for b, h in enumerate(step.held_pages.tolist())]
        flat = sum(owned, []) + free[:int(step.free_count)].tolist()
        assert sorted(flat) == list(range(n_pages))          # every page in one place

    prompt = [30, 1, 16, 47, 5]
    tokens = torch.randint(0, vocab, (sum(prompt),), generator=g, device=td)
    step, q, out, lse = forward(tokens, ints(dev, prompt), sum(prompt), max(prompt))
    dev.sync()
    check(step, tokens, prompt, [0] * n, q, out, lse)
    state = dict(seq=step.kv_lens.clone(), held=step.held_pages.clone(), count=step.free_count.clone())
    last = torch.randint(0, vocab, (n,), generator=g, device=td)

    # every step: the last kept token and up to K drafts of each request (request 3 stops drafting, request 1 pauses)
    buf = dict(tokens=torch.zeros(n * (K + 1), dtype=torch.int64, device=td), new=torch.zeros(n, dtype=torch.int32, device=td),
               draft=torch.zeros(n, K, dtype=torch.int32, device=td), lens=torch.zeros(n, dtype=torch.int32, device=td),
               ua=torch.zeros(n, K, device=td), us=torch.zeros(n, device=td), dp=torch.full((n, K, vocab), 1.0 / vocab, device=td))

    def whole():
        step, q, out, lse = forward(buf["tokens"], buf["new"], n * (K + 1), K + 1)
        probs = torch.softmax(torch.where(torch.isfinite(out), out, 0).float().flatten(1) @ head, -1)
        kept, acc = dev.draft_verify(probs, buf["draft"], buf["ua"], buf["us"], draft_probs=buf["dp"], draft_lens=buf["lens"],
                                     target_start=step.query_start[:n].contiguous())
        return step, q, out, lse, probs, kept, acc

    graph = None
    accepted = 0
    for it in range(12):
        lens = [int(x) for x in torch.randint(0, K + 1, (n,), generator=g, device=td)]
        lens[3] = 0
        new = [x + 1 for x in lens]
        drafts = torch.randint(0, vocab, (n, K), generator=g, device=td)
        flat = torch.cat([torch.cat([last[b:b + 1], drafts[b, :lens[b]]]) for b in range(n)])
        buf["tokens"].zero_(); buf["tokens"][:len(flat)] = flat
        buf["new"].copy_(ints(dev, new)); buf["draft"].copy_(drafts); buf["lens"].copy_(ints(dev, lens))
        buf["ua"].copy_(torch.rand(n, K, generator=g, device=td) * (0.02 if it % 2 else 1.0)); buf["us"].copy_(torch.rand(n, generator=g, device=td))
        seq = state["seq"].tolist()
        if captured:
            if graph is None:
                keep = {k: v.clone() for k, v in state.items()}
                t0, k0, v0 = table.clone(), kp.clone(), vp.clone()
                whole(); torch.cuda.synchronize()
                table.copy_(t0); kp.copy_(k0); vp.copy_(v0)
                for k in state: state[k].copy_(keep[k])
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    result = whole()
            graph.replay()
        else:
            result = whole()
        step, q, out, lse, probs, kept, acc = result
        dev.sync()
        check(step, buf["tokens"][:sum(new)], new, seq, q, out, lse)
        want, counts, _ = plain_verify(probs.cpu().numpy(), buf["draft"].cpu().numpy(), buf["ua"].cpu().numpy(), buf["us"].cpu().numpy(),
                                       buf["dp"].cpu().numpy(), lens, step.query_start.tolist()[:n])
        assert acc.tolist() == counts and kept.tolist() == want
        accepted += sum(counts)
        # the next step's lengths: what was kept; pages taken for rejected drafts stay with their rows
        state["seq"].copy_(state["seq"] + acc + 1)
        state["held"].copy_(step.held_pages)
        state["count"].copy_(step.free_count)
        last = kept.gather(1, acc[:, None].long())[:, 0].long()
    assert accepted > 0
