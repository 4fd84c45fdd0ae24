"""The paged-cache serving operators as workloads: their plain forms in elementary torch operations, the calls a
program makes of sanic_b200, the inputs, the work each pass cannot do without, and a 64-bit evaluation.

Four operators of one serving step, in the order a step uses them:

  append   page tables, slots and positions of a step's new tokens, built on the device from the request lengths
  write    rotate-half RoPE of q and k and the write of k and v into their page slots
  attn     causal attention of every request's new tokens over its pages (one token, a drafted chunk, a prompt)
  verify   acceptance of drafted tokens against the target's probabilities, and the token that follows them
"""
import math
import random

import numpy as np
import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_dev = None


def _device():
    """The framework's device handle; a program opens it once."""
    global _dev
    if _dev is None:
        import sanic_b200
        _dev = sanic_b200.CudaDevice(0)
    return _dev


# ── cases ──
def listed():
    return [
        # one generated token for each of 256 running requests: a latency
        dict(name="append_step", op="append", requests=256, new_lo=1, new_hi=1, ctx_lo=100, ctx_hi=8000, page=16, lens=1),
        # the prompts of 48 requests admitted at once: bytes of slots and positions
        dict(name="append_prompts", op="append", requests=48, new_lo=400, new_hi=4100, ctx_lo=0, ctx_hi=0, page=64, lens=2),
        # the keys and values of one token of 16 requests, the 1B decode configuration's heads
        dict(name="write_step", op="write", tokens=16, q_heads=32, kv_heads=8, head_dim=64, dtype="bf16", src="bf16", page=16,
             fused=False, heads_first=False),
        # a prefill chunk's rows, cut from the fused projection's output
        dict(name="write_chunk", op="write", tokens=8191, q_heads=32, kv_heads=8, head_dim=128, dtype="f16", src="f16", page=64,
             fused=True, heads_first=False),
        # a single chat: one token over a short cache
        dict(name="attn_one", op="attn", requests=1, ones=1, new_lo=1, new_hi=1, ctx_lo=1022, ctx_hi=1022,
             q_heads=32, kv_heads=8, head_dim=64, dtype="bf16", page=16, window=0, heads_first=False, lens=3),
        # the decode step of a busy server: ragged lengths, one token each
        dict(name="attn_step", op="attn", requests=64, ones=64, new_lo=1, new_hi=1, ctx_lo=500, ctx_hi=16000,
             q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=32, window=0, heads_first=False, lens=4),
        # the target model's pass over drafted tokens
        dict(name="attn_draft", op="attn", requests=24, ones=0, new_lo=3, new_hi=6, ctx_lo=1000, ctx_hi=9000,
             q_heads=32, kv_heads=8, head_dim=128, dtype="f16", page=16, window=0, heads_first=True, lens=5),
        # one chunk of a long document's prefill
        dict(name="attn_chunk", op="attn", requests=1, ones=0, new_lo=2048, new_hi=2048, ctx_lo=30000, ctx_hi=30000,
             q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=128, window=0, heads_first=False, lens=6),
        # prefill chunks and decodes in one batch, with a sliding window
        dict(name="attn_mixed", op="attn", requests=32, ones=28, new_lo=300, new_hi=600, ctx_lo=200, ctx_hi=6000,
             q_heads=32, kv_heads=8, head_dim=64, dtype="f16", page=32, window=2000, heads_first=False, lens=7),
        # whole prompts, as many key/value heads as query heads
        dict(name="attn_prompts", op="attn", requests=5, ones=0, new_lo=900, new_hi=4100, ctx_lo=0, ctx_hi=0,
             q_heads=16, kv_heads=16, head_dim=128, dtype="bf16", page=16, window=0, heads_first=False, lens=8),
        # a single chat with four drafted tokens
        dict(name="verify_one", op="verify", requests=1, draft=4, vocab=128256, ragged=False, has_draft_probs=True, lens=9),
        # a batch of ragged drafts
        dict(name="verify_batch", op="verify", requests=64, draft=5, vocab=128256, ragged=True, has_draft_probs=True, lens=10),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_largest = {}


def _fits(case):
    if not _largest:
        for c in listed():
            w = work(c)
            best = _largest.setdefault(c["op"], {"bytes": 0, "flops": 0})
            for k in best:
                best[k] = max(best[k], w[k])
    w, top = work(case), _largest[case["op"]]
    return w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]


def draw(rng):
    """A case of the same ranges: the operator first, then its sizes; one that costs more than the largest listed one of its
    operator is drawn again with fewer requests or tokens."""
    op = rng.choice(["append", "write", "attn", "attn", "attn", "verify"])
    if op == "append":
        prompts = rng.random() < 0.5
        case = dict(op=op, requests=_log(rng, 1, 1500), new_lo=int(prompts),
                    new_hi=_log(rng, 2, 4000) if prompts else rng.choice([1, 2, 6]), ctx_lo=0, ctx_hi=0 if prompts else _log(rng, 20, 16000), page=rng.choice([1, 16, 24, 32, 64, 128, 256]),
                    lens=rng.randrange(1 << 30))
    elif op == "write":
        heads = rng.choice([(32, 8), (8, 8), (16, 2), (24, 8), (7, 1)])
        dtype = rng.choice(["bf16", "f16"])
        case = dict(op=op, tokens=_log(rng, 1, 8000), q_heads=heads[0], kv_heads=heads[1], head_dim=rng.choice([64, 128]), dtype=dtype,
                    src=rng.choice([dtype, dtype, "f32"]), page=rng.choice([8, 16, 20, 64, 128]), fused=rng.random() < 0.5,
                    heads_first=rng.random() < 0.5)
    elif op == "attn":
        kind = rng.choice(["step", "draft", "chunk", "mixed", "prompts"])
        heads = rng.choice([(32, 8), (32, 8), (16, 16), (32, 4), (24, 8), (7, 1), (20, 4)])
        n = {"step": _log(rng, 1, 128), "draft": _log(rng, 1, 64), "chunk": rng.randint(1, 3), "mixed": rng.randint(2, 40),
             "prompts": rng.randint(1, 8)}[kind]
        new = {"step": (1, 1), "draft": (2, rng.randint(2, 9)), "chunk": (_log(rng, 16, 2048),) * 2, "mixed": (1, _log(rng, 20, 900)),
               "prompts": (1, _log(rng, 40, 4000))}[kind]
        top = 0 if kind == "prompts" else _log(rng, 16, 30000)
        case = dict(op=op, requests=n, ones=n if kind == "step" else (n - 1 - n // 8 if kind == "mixed" else 0), new_lo=new[0],
                    new_hi=new[1], ctx_lo=top // rng.choice([1, 4, 16, 100]), ctx_hi=top, q_heads=heads[0], kv_heads=heads[1],
                    head_dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "f16"]), page=rng.choice([8, 16, 16, 24, 32, 64, 128, 256]),
                    window=rng.choice([0, 0, 0, _log(rng, 5, 5000)]), heads_first=rng.random() < 0.3, lens=rng.randrange(1 << 30))
    else:
        case = dict(op=op, requests=_log(rng, 1, 64), draft=rng.randint(0, 8), vocab=rng.choice([128256, _log(rng, 50, 160000)]),
                    ragged=rng.random() < 0.5, has_draft_probs=rng.random() < 0.7, lens=rng.randrange(1 << 30))
    while not _fits(case):
        if op == "write":
            case["tokens"] = max(1, case["tokens"] * 3 // 4)
        elif case["requests"] > 1:
            case["requests"] = max(1, case["requests"] * 3 // 4)
            if op == "attn":
                case["ones"] = min(case["ones"], case["requests"])
        elif op == "verify":
            case["vocab"] = case["vocab"] * 3 // 4
        else:
            for key in ("new_lo", "new_hi", "ctx_lo", "ctx_hi"):
                case[key] = max(int(key.startswith("new")), case[key] * 3 // 4)
    return case


def _lens(case):
    """(tokens held, tokens new) of every request: part of the case, not of the seed, so that its work is known."""
    r = random.Random(case["lens"])
    held, new = [], []
    for i in range(case["requests"]):
        held.append(r.randint(case["ctx_lo"], case["ctx_hi"]))
        new.append(1 if i < case.get("ones", 0) else r.randint(case["new_lo"], case["new_hi"]))
    return held, new


def _drafts(case):
    r = random.Random(case["lens"])
    return [r.randint(0, case["draft"]) if case["ragged"] else case["draft"] for _ in range(case["requests"])]


def _pages(tokens, page):
    return -(-tokens // page)


# about this share of the drafted tokens is accepted with the probabilities that `prepare` makes
_ACCEPTED = 0.75


def work(case):
    if case["op"] == "append":
        held, new = _lens(case)
        taken = sum(_pages(h + n, case["page"]) - _pages(h, case["page"]) for h, n in zip(held, new))
        n, t = case["requests"], sum(new)
        # lengths, held pages and free pages in; table entries, starts, lengths, held pages, positions and slots out
        return {"bytes": 4 * (3 * n + taken) + 4 * (taken + 3 * n) + 12 * t, "flops": 2 * n + 4 * t}
    if case["op"] == "write":
        t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        src = 4 if case["src"] == "f32" else 2
        return {"bytes": t * ((hq + 2 * hkv) * d * (src + 2) + 12 + d * 4), "flops": 3 * t * (hq + hkv) * d}
    if case["op"] == "attn":
        held, new = _lens(case)
        hq, hkv, d, w = case["q_heads"], case["kv_heads"], case["head_dim"], case["window"]
        keys = pairs = 0
        for h, n in zip(held, new):
            first = max(0, h - w + 1) if w else 0
            keys += h + n - first if n else 0
            if w:
                pairs += sum(min(h + i + 1, w) for i in range(n))
            else:
                pairs += n * h + n * (n + 1) // 2
        # every visible key and value once; q in, out and the log-sum-exp out
        return {"bytes": keys * hkv * d * 4 + sum(new) * hq * (d * 4 + 4), "flops": 4 * pairs * hq * d}
    n, v = case["requests"], case["vocab"]
    rejected = sum(1.0 - _ACCEPTED ** k for k in _drafts(case)) if case["has_draft_probs"] else 0.0
    # the target's row that the last token is drawn from, and the draft's row where a token was rejected
    return {"bytes": int(4 * v * (n + rejected)), "flops": int(2 * v * (n + rejected))}


# ── inputs ──
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


def _page_pool(case, n_pages, g):
    """k and v pages as [pages, rows, heads, dim] views of either layout, full of a long-running cache's values."""
    hkv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    shape = (n_pages, hkv, page, d) if case["heads_first"] else (n_pages, page, hkv, d)
    out = []
    for _ in range(2):
        t = torch.empty(shape, dtype=_TORCH[case["dtype"]], device="cuda")
        t.normal_(generator=g)
        out.append(t.transpose(1, 2) if case["heads_first"] else t)
    return out


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "append":
        held, new = _lens(case)
        page = case["page"]
        have = [_pages(h, page) for h in held]
        most = max(_pages(h + n, page) for h, n in zip(held, new)) + 3
        total = sum(have) + sum(_pages(h + n, page) for h, n in zip(held, new)) + 64
        order = torch.randperm(total, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        table = torch.full((case["requests"], most), -1, dtype=torch.int32, device="cuda")
        held_pages = _ints(have)
        mask = torch.arange(most, device="cuda")[None, :] < held_pages[:, None]
        table[mask] = order[:sum(have)]
        s.update(seq_lens=_ints(held), new_lens=_ints(new), held_pages=held_pages, table=table, free_pages=order[sum(have):].contiguous(),
                 free_count=_ints([total - sum(have)]), n_tokens=sum(new))
        return s
    if case["op"] == "write":
        t, hq, hkv, d, page = (case[k] for k in ("tokens", "q_heads", "kv_heads", "head_dim", "page"))
        src = _TORCH[case["src"]]
        if case["fused"]:
            rows = torch.randn(t, (hq + 2 * hkv) * d, generator=g, device="cuda").to(src)
            q, k, v = rows.split([hq * d, hkv * d, hkv * d], dim=1)
        else:
            q, k, v = (torch.randn(t, h * d, generator=g, device="cuda").to(src) for h in (hq, hkv, hkv))
        n_pages = _pages(t, page) + 8
        k_pages, v_pages = _page_pool(case, n_pages, g)
        n_pos = 16384
        inv = 500000.0 ** (-torch.arange(d // 2, device="cuda", dtype=torch.float64) / (d // 2))
        ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
        slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:t].sort().values
        first = int(torch.randint(0, n_pos - t + 1, (1,), generator=g, device="cuda"))
        s.update(q=q.unflatten(1, (hq, d)), k=k.unflatten(1, (hkv, d)), v=v.unflatten(1, (hkv, d)), k_pages=k_pages, v_pages=v_pages,
                 slots=slots, positions=torch.arange(first, first + t, device="cuda", dtype=torch.int32),
                 table=torch.stack([ang.cos(), ang.sin()], -1).to(torch.float32).contiguous())
        return s
    if case["op"] == "attn":
        held, new = _lens(case)
        page = case["page"]
        need = [_pages(h + n, page) for h, n in zip(held, new)]
        n_pages = sum(need) + sum(need) // 8 + 2
        k_pages, v_pages = _page_pool(case, n_pages, g)
        order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        table = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
        table[torch.arange(max(need), device="cuda")[None, :] < _ints(need)[:, None]] = order[:sum(need)]
        q = torch.randn(sum(new), case["q_heads"], case["head_dim"], generator=g, device="cuda")
        s.update(q=(1.5 * q).to(_TORCH[case["dtype"]]), k_pages=k_pages, v_pages=v_pages, table=table,
                 query_start=_ints(np.concatenate([[0], np.cumsum(new)]).tolist()), kv_lens=_ints([h + n for h, n in zip(held, new)]),
                 held=held, new=new, max_query_len=max(new))
        return s
    n, k, v = case["requests"], case["draft"], case["vocab"]
    drafts = _drafts(case)
    base = torch.randn(n, k + 1, v, generator=g, device="cuda") * 2.5
    target = torch.softmax(base, -1)
    other = torch.softmax(base[:, :k] + 0.65 * torch.randn(n, k, v, generator=g, device="cuda"), -1)
    if k:
        tokens = torch.multinomial(other.view(n * k, v), 1, generator=g).view(n, k).to(torch.int32)
    else:
        tokens = torch.zeros(n, 0, dtype=torch.int32, device="cuda")
    s.update(target=target.view(n * (k + 1), v), draft_probs=other if case["has_draft_probs"] and k else None, tokens=tokens,
             u_accept=torch.rand(n, k, generator=g, device="cuda"), u_sample=torch.rand(n, generator=g, device="cuda"),
             draft_lens=_ints(drafts) if case["ragged"] else None, target_start=_ints([i * (k + 1) for i in range(n)]))
    return s


# ── one pass ──
def run(state):
    return {"append": _append, "write": _write, "attn": _attn, "verify": _verify}[state["op"]](state)


def _append(s):
    if own:
        r = _device().page_table_append(s["seq_lens"], s["new_lens"], s["table"], s["free_pages"], s["free_count"], s["page"],
                                        s["n_tokens"], held_pages=s["held_pages"])
        return [s["table"], r.query_start, r.kv_lens, r.held_pages, r.free_count, r.positions, r.slots]
    page, t = s["page"], s["n_tokens"]
    held, new, have = s["seq_lens"].long(), s["new_lens"].long(), s["held_pages"].long()
    kv = held + new
    need = (kv + page - 1) // page
    taken = (need - have).clamp(min=0)
    before = taken.cumsum(0) - taken
    cols = torch.arange(s["table"].shape[1], device="cuda")[None, :]
    fresh = (cols >= have[:, None]) & (cols < need[:, None])
    rank = s["free_count"].long() - 1 - (before[:, None] + cols - have[:, None])
    picked = s["free_pages"][rank.clamp(0, s["free_pages"].shape[0] - 1)]
    s["table"].copy_(torch.where(fresh, picked, s["table"]))
    start = torch.zeros(held.shape[0] + 1, dtype=torch.int64, device="cuda")
    start[1:] = new.cumsum(0)
    token = torch.arange(t, device="cuda")
    req = torch.searchsorted(start[1:].contiguous(), token, right=True)
    pos = held[req] + token - start[req]
    slots = s["table"][req, pos // page].long() * page + pos % page
    i32 = torch.int32
    return [s["table"], start.to(i32), kv.to(i32), torch.maximum(need, have).to(i32), s["free_count"] - taken.sum().to(i32),
            pos.to(i32), slots]


def _write(s):
    if own:
        q = _device().paged_cache_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], q=s["q"], positions=s["positions"],
                                        rope_table=s["table"])
        return [q, s["k_pages"], s["v_pages"]]
    cs = s["table"][s["positions"].long()]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]

    def turn(x):
        a, b = x.float().chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    dt = _TORCH[s["dtype"]]
    page, row = s["slots"] // s["page"], s["slots"] % s["page"]
    s["k_pages"][page, row] = turn(s["k"]).to(dt)
    s["v_pages"][page, row] = s["v"].float().to(dt)
    return [turn(s["q"]).to(dt), s["k_pages"], s["v_pages"]]


def _attn(s):
    if own:
        return list(_device().attn_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["query_start"], s["kv_lens"],
                                         max_query_len=s["max_query_len"], window=s["window"], return_lse=True))
    q = s["q"]
    hq, hkv, d, page = s["q_heads"], s["kv_heads"], s["head_dim"], s["page"]
    g = hq // hkv
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[0], hq, dtype=torch.float32, device="cuda")
    at = 0
    for i, (held, new) in enumerate(zip(s["held"], s["new"])):
        kv = held + new
        first = max(0, held - s["window"] + 1) if s["window"] else 0
        pos = torch.arange(first, kv, device="cuda")
        rows = s["table"][i].long()[pos // page]
        step = max(1, (1 << 28) // max(1, kv * hq))       # query rows whose scores are held at once
        k = s["k_pages"][rows, pos % page].float().permute(1, 2, 0)
        v = s["v_pages"][rows, pos % page].float().transpose(0, 1)
        for a in range(0, new, step):
            b = min(new, a + step)
            x = q[at + a:at + b].float().view(b - a, hkv, g, d).transpose(0, 1).reshape(hkv, -1, d) @ k * (1.0 / math.sqrt(d))
            here = torch.arange(held + a, held + b, device="cuda").repeat_interleave(g)[:, None]
            hidden = pos[None, :] > here
            if s["window"]:
                hidden |= pos[None, :] <= here - s["window"]
            x.masked_fill_(hidden, -math.inf)
            m = x.max(-1, keepdim=True).values
            e = (x - m).exp()
            z = e.sum(-1, keepdim=True)
            out[at + a:at + b] = (e @ v / z).view(hkv, b - a, g, d).transpose(0, 1).reshape(b - a, hq, d).to(q.dtype)
            lse[at + a:at + b] = (m + z.log()).view(hkv, b - a, g).transpose(0, 1).reshape(b - a, hq)
        at += new
    return [out, lse]


def _verify(s):
    if own:
        return list(_device().draft_verify(s["target"], s["tokens"], s["u_accept"], s["u_sample"], draft_probs=s["draft_probs"],
                                           draft_lens=s["draft_lens"], target_start=s["target_start"]))
    n, k, v = s["requests"], s["draft"], s["vocab"]
    who = torch.arange(n, device="cuda")
    lens = s["draft_lens"].long() if s["draft_lens"] is not None else torch.full((n,), k, device="cuda")
    col = torch.arange(k, device="cuda")[None, :]
    tok = s["tokens"].long()
    p = s["target"][s["target_start"].long()[:, None] + col, tok].double()
    q = torch.gather(s["draft_probs"], 2, tok[:, :, None])[:, :, 0].double() if s["draft_probs"] is not None else torch.ones_like(p)
    good = (s["u_accept"].double() * q < p) & (col < lens[:, None])
    count = good.long().cumprod(1).sum(1) if k else torch.zeros(n, dtype=torch.int64, device="cuda")
    w = s["target"][s["target_start"].long() + count].double()
    if k:
        at = count.clamp(max=k - 1)
        rejected = (count < lens)[:, None]
        if s["draft_probs"] is not None:
            left = (w - s["draft_probs"][who, at].double()).clamp(min=0.0)
        else:
            left = w.scatter(1, tok[who, at][:, None], 0.0)
        left = torch.where(left.sum(1, keepdim=True) > 0, left, w)
        w = torch.where(rejected, left, w)
    c = w.cumsum(1)
    over = (c > s["u_sample"].double()[:, None] * c[:, -1:]) & (w > 0)
    last = over.to(torch.int8).argmax(1)
    tokens = torch.full((n, k + 1), -1, dtype=torch.int32, device="cuda")
    if k:
        tokens[:, :k] = torch.where(col < count[:, None], s["tokens"], -1)
    tokens[who, count] = last.to(torch.int32)
    return [tokens, count.to(torch.int32)]


# ── the definition in 64 bits ──
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "write":
        return _exact_write(s)
    if case["op"] == "attn":
        return _exact_attn(s) if work(case)["flops"] < 3e12 else None
    return _exact_verify(s)


def _exact_append(s):
    table, free, page = s["table"].cpu().numpy().copy(), s["free_pages"].cpu().numpy(), s["page"]
    left = int(s["free_count"].item())
    start, kv, have, pos, slots = [0], [], [], [], []
    for r, (h, n, got) in enumerate(zip(s["seq_lens"].tolist(), s["new_lens"].tolist(), s["held_pages"].tolist())):
        while got * page < h + n:
            left -= 1
            table[r, got] = free[left]
            got += 1
        have.append(got)
        kv.append(h + n)
        start.append(start[-1] + n)
        p = np.arange(h, h + n)
        pos.append(p)
        slots.append(table[r][p // page].astype(np.int64) * page + p % page)
    i32 = np.int32
    return [table, np.array(start, i32), np.array(kv, i32), np.array(have, i32), np.array([left], i32), np.concatenate(pos).astype(i32),
            np.concatenate(slots)]


def _exact_write(s):
    half = s["head_dim"] // 2
    c = s["table"].double()[s["positions"].long()]
    z = torch.complex(c[..., 0], c[..., 1])[:, None, :]

    def turn(x):
        x = x.double()
        y = torch.complex(x[..., :half], x[..., half:]) * z
        return torch.cat([y.real, y.imag], -1)

    k, v = s["k_pages"].double().contiguous(), s["v_pages"].double().contiguous()
    flat = (-1, s["kv_heads"], s["head_dim"])
    k.view(flat)[s["slots"]] = turn(s["k"])
    v.view(flat)[s["slots"]] = s["v"].double()
    return [turn(s["q"]), k, v]


def _exact_attn(s):
    hq, hkv, d, w = s["q_heads"], s["kv_heads"], s["head_dim"], s["window"]
    g = hq // hkv
    outs, lses = [], []
    for i, (held, new) in enumerate(zip(s["held"], s["new"])):
        kv = held + new
        rows = s["table"][i, :_pages(kv, s["page"])].long()
        out = torch.empty(new, hq, d, dtype=torch.float64, device="cuda")
        lse = torch.empty(new, hq, dtype=torch.float64, device="cuda")
        qi = s["q"][sum(s["new"][:i]):sum(s["new"][:i]) + new]
        key = torch.arange(kv, device="cuda")
        for h in range(hq):
            k = s["k_pages"][rows, :, h // g].reshape(-1, d)[:kv].double()
            v = s["v_pages"][rows, :, h // g].reshape(-1, d)[:kv].double()
            for a in range(0, new, 512):
                x = torch.einsum("qd,kd->qk", qi[a:a + 512, h].double(), k) / math.sqrt(d)
                gap = torch.arange(held + a, held + a + x.shape[0], device="cuda")[:, None] - key
                seen = (gap >= 0) & (gap < w) if w else gap >= 0
                z = torch.logsumexp(torch.where(seen, x, -math.inf), 1)
                out[a:a + 512, h] = torch.where(seen, torch.exp(x - z[:, None]), 0.0) @ v
                lse[a:a + 512, h] = z
        outs.append(out)
        lses.append(lse)
    return [torch.cat(outs), torch.cat(lses)]


def _exact_verify(s):
    n, k = s["requests"], s["draft"]
    tok, ua, us = s["tokens"].tolist(), s["u_accept"].tolist(), s["u_sample"].tolist()
    lens = s["draft_lens"].tolist() if s["draft_lens"] is not None else [k] * n
    start = s["target_start"].tolist()
    tokens, counts = [], []
    for r in range(n):
        count, row = 0, []
        while count < lens[r]:
            x = tok[r][count]
            p = float(s["target"][start[r] + count, x])
            q = float(s["draft_probs"][r, count, x]) if s["draft_probs"] is not None else 1.0
            if not ua[r][count] * q < p:
                break
            row.append(x)
            count += 1
        w = s["target"][start[r] + count].cpu().numpy().astype(np.float64)
        if count < lens[r]:
            left = w.copy()
            if s["draft_probs"] is not None:
                left = np.maximum(left - s["draft_probs"][r, count].cpu().numpy().astype(np.float64), 0.0)
            else:
                left[tok[r][count]] = 0.0
            w = left if left.any() else w
        c = np.cumsum(w)
        row.append(int(np.searchsorted(c, us[r] * c[-1], side="right")))
        tokens.append(row + [-1] * (k + 1 - len(row)))
        counts.append(count)
    return [np.array(tokens, np.int32), np.array(counts, np.int32)]
