"""Servers of different sizes, caches, prompts and random numbers that step on streams of their own at once: each gives what it gives
alone, so nothing that a call of one uses meanwhile belongs to a call of the other."""
import numpy as np
import pytest
import torch

from test_gpu_serving_loop import EPS, TOP, Server
from test_gpu_serving_step import D, _t

pytestmark = pytest.mark.gpu

STEPS = 16


class Run:
    """A server's steps without the linears, whose workspaces are one a device; inputs made from the seed."""

    def __init__(self, seed, B, Hq, Hkv, bits, longest):
        self.make = lambda: Server(seed, B, Hq, Hkv, bits, width=64)   # noqa: E731
        rng = np.random.default_rng(1000 + seed)
        prompt = rng.integers(1, longest, B).astype(np.int32)
        new = [prompt] + [rng.choice([1, 1, 1, 3, 0, -5], B).astype(np.int32) for _ in range(STEPS)]
        rows = [int(np.maximum(n, 0).sum()) + 2 for n in new]
        self.steps = [(_t(rng.standard_normal((r, 256))).half(), _t(n), _t(rng.random(r).astype(np.float32)))
                      for r, n in zip(rows, new)]

    def step(self, s, i):
        (x, new, u), ops, (_, Hq, Hkv) = self.steps[i], s.ops, s.shape
        plan = ops.kv_step_plan(s.table, s.lens, new, s.ring, s.ring_state, x.shape[0])
        heads = x.repeat(1, (Hq + 2 * Hkv + 1) // 2).unflatten(1, (-1, D))
        q, k = ops.qk_norm_rope(heads[:, :Hq].contiguous(), heads[:, Hq:Hq + Hkv].contiguous(), s.qw, s.kw, s.cs, plan.positions, EPS)
        ops.kv_append(k, heads[:, Hq + Hkv:Hq + 2 * Hkv].contiguous(), *s.cache, s.table, s.lens, s.bits, row_start=plan.row_start,
                      counts=plan.counts)
        ops.kv_page_bounds(s.cache[0], s.table, plan.lens_after, s.bits, s.bounds, first=s.lens)
        pages = ops.kv_select_pages(q, s.bounds, s.cache[2], s.table, plan.row_lens, s.bits, TOP, row_seq=plan.row_seq)
        a = ops.kv_sparse_attention(q, *s.cache, s.table, plan.row_lens, s.bits, pages, row_seq=plan.row_seq)
        y, h = ops.add_norm(a.flatten(1)[:, :256], x, s.w, EPS, post_weight=s.post, gate=s.gate)
        tokens, probs = ops.sample_tokens(a.flatten(1), u, 0.8, 30, 0.9, return_probs=True)
        s.lens.copy_(plan.lens_after)
        return [*plan, pages, a, y, h, tokens, probs]


def test_servers_of_their_own_on_two_streams():
    runs = [Run(1, 6, 8, 2, 8, 500), Run(2, 9, 10, 2, 4, 300)]
    want = []
    for r in runs:
        s = r.make()
        want.append(([r.step(s, i) for i in range(STEPS + 1)], s.state()))
    torch.cuda.synchronize()
    assert not torch.equal(want[0][0][1][9][:4, 0], want[1][0][1][9][:4, 0])   # the two have different outputs
    servers = [r.make() for r in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(STEPS + 1):
        for j in (0, 1) if i % 2 else (1, 0):
            with torch.cuda.stream(streams[j]):
                got[j].append(runs[j].step(servers[j], i))
    torch.cuda.synchronize()
    for j in (0, 1):
        for i, (step, expected) in enumerate(zip(got[j], want[j][0])):
            for k, (a, b) in enumerate(zip(step, expected)):
                assert torch.equal(a, b), (j, i, k)
        assert all(torch.equal(a, b) for a, b in zip(servers[j].state(), want[j][1]))
