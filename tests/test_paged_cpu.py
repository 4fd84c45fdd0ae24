"""CPU-side checks of the paged-cache entry points: parameter layouts against the header, the split of the attention work
over CTAs (the kernels' own index arithmetic, compiled for the host), and the refusals that need no device."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from sanic_b200 import _abi as abi
from sanic_b200 import backend

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_parameter_layouts_match_the_header(tmp_path):
    structs = {"sanic_page_append_params": abi.PageAppendParams, "sanic_paged_write_params": abi.PagedWriteParams,
               "sanic_attn_paged_params": abi.AttnPagedParams, "sanic_draft_verify_params": abi.DraftVerifyParams}
    lines = []
    want = []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "sanic_b200.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "p")], check=True)
    got = [int(t) for t in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


WALK = r'''
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>
#include "paged_sched.h"
using namespace sanic::paged;
struct Load { const std::vector<Req>* reqs; Req operator()(int b) const { return (*reqs)[b]; } };
#define CHECK(c) do { if (!(c)) { printf("line %d: %s (trial %d)\n", __LINE__, #c, trial); return 1; } } while (0)
template <int KT> int run(int trials, unsigned seed) {
    std::mt19937 rng(seed);
    auto u = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    for (int trial = 0; trial < trials; ++trial) {
        Shape p{u(1, 40), u(1, 9), u(0, 2) ? 0 : u(1, 700), u(1, 64)};
        std::vector<Req> reqs;
        std::vector<long long> cum{0};
        int q0 = 0;
        const int big = u(0, 3) ? 40 : 3000;
        for (int b = 0; b < p.n_requests; ++b) {
            Req r{q0, u(0, 4) ? u(0, big) : 1, u(0, 9) ? u(0, 5000) : 0};     // chunks longer than the keys are among them
            q0 += r.qn;
            reqs.push_back(r);
            cum.push_back(cum.back() + request_cost<KT>(p, r));
        }
        const int grid = u(0, 4) ? u(1, 500) : 1;
        std::map<std::tuple<int, int, int>, std::vector<std::tuple<int, int, int, Seg>>> items;    // item -> (jb, je, cta, seg)
        for (int c = 0; c < grid; ++c) {
            Walk<KT, Load> w{Load{&reqs}};
            w.init(p, cum.data(), c, grid);
            Seg s;
            int slots[2] = {0, 0};
            while (w.next(p, s)) {
                items[{s.b, s.hk, s.rb}].push_back({s.jb, s.je, c, s});
                if (!(s.starts && s.finishes)) { CHECK(partial_slot(s, c) / 2 == c); CHECK(slots[partial_slot(s, c) % 2]++ == 0); }
            }
        }
        size_t want = 0;
        for (int b = 0; b < p.n_requests; ++b)
            for (int hk = 0; hk < p.kv_heads; ++hk)
                for (int rb = 0; rb < blocks_of(p, reqs[b]); ++rb, ++want) {
                    auto it = items.find({b, hk, rb});
                    CHECK(it != items.end());
                    int lo, hi, jb, je;
                    tile_range<KT>(p, reqs[b], rb, lo, hi, jb, je);
                    auto& v = it->second;
                    int at = jb;
                    for (size_t i = 0; i < v.size(); ++i) {       // in CTA order: a part each, consecutive CTAs, consecutive tiles
                        auto& [a, z, c, s] = v[i];
                        CHECK(a == at); CHECK(z > a || (je == jb && v.size() == 1)); CHECK(z <= je);
                        CHECK(s.starts == (i == 0)); CHECK(s.finishes == (i + 1 == v.size()));
                        CHECK(i == 0 || c == std::get<2>(v[i - 1]) + 1);
                        CHECK(s.lo == lo && s.hi == hi);
                        at = z;
                    }
                    CHECK(at == je);
                    CHECK(std::get<3>(v[0]).parts == (int)v.size());
                    // the range covers what every token of the block sees, and no key outside it
                    for (int t = rb * p.block_tokens; t < imin(reqs[b].qn, (rb + 1) * p.block_tokens); ++t) {
                        const int pos = reqs[b].kv - reqs[b].qn + t;
                        if (pos < 0) continue;
                        CHECK(pos < hi); CHECK(hi <= reqs[b].kv);
                        CHECK(lo <= (p.window ? imax(0, pos - p.window + 1) : 0));
                    }
                }
        CHECK(want == items.size());
    }
    return 0;
}
int main() { return run<64>(1500, 1) || run<128>(1500, 2); }
'''


def test_every_key_tile_of_every_item_is_folded_once(tmp_path):
    src = tmp_path / "walk.cpp"
    src.write_text(WALK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "sanic_b200", "csrc"), str(src), "-o", str(tmp_path / "walk")], check=True)
    r = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


class HostDevice(backend.CudaDevice):
    """The host mirror's own checks on CPU tensors: no context, nothing is launched."""

    def __init__(self):
        self.lib, self.h, self.ordinal, self.torch_device, self._scratch = abi.load(), None, -1, torch.device("cpu"), {}

    def stream(self):
        return C.c_void_p(0)


def refuses(match, fn, *args, **kw):
    with pytest.raises(backend.RunError, match=match):
        fn(*args, **kw)


def test_host_refusals():
    d = HostDevice()
    i32, bf = torch.int32, torch.bfloat16
    z = lambda *s, t=i32: torch.zeros(*s, dtype=t)
    # page_table_append
    good = dict(seq_lens=z(3), new_lens=z(3), block_table=z(3, 4), free_pages=z(9), free_count=z(1), page_size=16, n_tokens=5)
    ap = lambda **kw: d.page_table_append(**dict(good, **kw))
    refuses("block_table has 2 rows", ap, block_table=z(2, 4))
    refuses("dtype", ap, seq_lens=z(3, t=torch.int64))
    refuses("new_lens", ap, new_lens=z(4))
    refuses("held_pages", ap, held_pages=z(2))
    refuses("free_count", ap, free_count=z(2))
    refuses("not be negative", ap, n_tokens=-1)
    refuses("last axis", ap, block_table=z(4, 3).T)
    # paged_cache_write
    good = dict(k=z(5, 2, 64, t=bf), v=z(5, 2, 64, t=bf), k_pages=z(3, 16, 2, 64, t=bf), v_pages=z(3, 16, 2, 64, t=bf), slots=z(5, t=torch.int64))
    wr = lambda **kw: d.paged_cache_write(**dict(good, **kw))
    refuses("disagree", wr, v_pages=z(3, 16, 2, 128, t=bf))
    refuses("dtype", wr, k=z(5, 2, 64, t=torch.float16))
    refuses("shape", wr, v=z(5, 3, 64, t=bf))
    refuses("side by side", wr, k=z(5, 64, 2, t=bf).transpose(1, 2).contiguous().transpose(0, 1).contiguous().transpose(0, 1))
    refuses("slots", wr, slots=z(4, t=torch.int64))
    refuses("needs positions", wr, rope_table=z(8, 32, 2, t=torch.float32))
    refuses("rope_table", wr, rope_table=z(8, 16, 2, t=torch.float32), positions=z(5))
    refuses("needs q", wr, q_out=z(5, 4, 64, t=bf))
    # attn_paged
    good = dict(q=z(5, 4, 64, t=bf), k_pages=z(3, 16, 2, 64, t=bf), v_pages=z(3, 16, 2, 64, t=bf), block_table=z(2, 3), query_start=z(3), kv_lens=z(2))
    at = lambda **kw: d.attn_paged(**dict(good, **kw))
    refuses("disagree", at, q=z(5, 4, 128, t=bf))
    refuses("disagree", at, q=z(5, 4, 64, t=torch.float16))
    refuses("dtype", at, q=z(5, 4, 64, t=torch.float32))
    refuses("axes", at, q=z(5, 256, t=bf))
    refuses("query_start", at, query_start=z(2))
    refuses("kv_lens", at, kv_lens=z(2, t=torch.int64))
    refuses("`out`", at, out=z(5, 4, 32, t=bf))
    # draft_verify
    f32 = torch.float32
    good = dict(target_probs=z(8, 50, t=f32), draft_tokens=z(2, 3), u_accept=z(2, 3, t=f32), u_sample=z(2, t=f32), draft_probs=z(2, 3, 50, t=f32))
    ve = lambda **kw: d.draft_verify(**dict(good, **kw))
    refuses("draft_probs", ve, draft_probs=z(2, 3, 51, t=f32))
    refuses("dtype", ve, target_probs=z(8, 50, t=bf))
    refuses("u_accept", ve, u_accept=z(2, 4, t=f32))
    refuses("draft_lens", ve, draft_lens=z(3))
    refuses("requests, drafts", ve, draft_tokens=z(6))


def test_host_refuses_numbers_that_would_wrap():
    # the C side counts in 32 bits: 2^32 + 16 would be a page of 16 rows, a window of -2^32 none
    d = HostDevice()
    i32, bf = torch.int32, torch.bfloat16
    z = lambda *s, t=i32: torch.zeros(*s, dtype=t)
    good = dict(seq_lens=z(3), new_lens=z(3), block_table=z(3, 4), free_pages=z(9), free_count=z(1), page_size=16, n_tokens=5)
    ap = lambda **kw: d.page_table_append(**dict(good, **kw))
    refuses("32 bits", ap, page_size=2 ** 32 + 16)
    refuses("32 bits", ap, page_size=16 - 2 ** 32)
    refuses("32 bits", ap, n_tokens=2 ** 32 + 5)
    refuses("32 bits", ap, block_table=torch.zeros(3, 2 ** 32 + 4, dtype=i32, device="meta"))       # (no memory behind them)
    refuses("32 bits", ap, free_pages=torch.zeros(2 ** 32 + 9, dtype=i32, device="meta"))
    good = dict(q=z(5, 4, 64, t=bf), k_pages=z(3, 16, 2, 64, t=bf), v_pages=z(3, 16, 2, 64, t=bf), block_table=z(2, 3), query_start=z(3), kv_lens=z(2))
    at = lambda **kw: d.attn_paged(**dict(good, **kw))
    refuses("window", at, window=-2 ** 32)
    refuses("max_query_len", at, max_query_len=-2 ** 32)


def test_entry_points_refuse_a_null_context():
    lib = abi.load()
    assert lib.sanic_page_table_append(None, C.byref(abi.PageAppendParams()), None) == abi.ERR_INVALID
    assert lib.sanic_paged_cache_write(None, C.byref(abi.PagedWriteParams()), None) == abi.ERR_INVALID
    assert lib.sanic_attn_paged(None, C.byref(abi.AttnPagedParams()), None) == abi.ERR_INVALID
    assert lib.sanic_draft_verify(None, C.byref(abi.DraftVerifyParams()), None) == abi.ERR_INVALID
    assert lib.sanic_attn_paged_workspace_bytes(None, C.byref(abi.AttnPagedParams())) == 0
