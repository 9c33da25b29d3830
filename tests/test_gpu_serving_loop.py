"""A serving loop from the operators together, as a server that never asks the GPU for lengths runs it: step plan -> quantised
linear -> head norms with rotation -> cache append -> page bounds -> choice of pages -> sparse attention -> quantised linear ->
residual norm -> quantised linear -> sampling.  Each stage is held to its 64-bit reference on the inputs that the stage before
gave it; then the same loop eagerly, captured into a graph and replayed, and from two streams."""
import numpy as np
import pytest
import torch

import attn_step_ref
import serving_step_ref as ref
from test_gpu_attn_step import _angles
from test_gpu_serving_step import D, PAGE, _check_sparse, _n, _t

pytestmark = pytest.mark.gpu

TOP, EPS = 6, 1e-5


def _linear(rng, k, n):
    """One EXL3 matrix [k, n] whose outputs are of the size of its inputs."""
    return ([_t(rng.integers(-32768, 32768, (k // 16, n // 16, 48), dtype=np.int16))],
            [torch.ones(k, dtype=torch.float16, device="cuda")],
            [torch.full((n,), 0.8 * k ** -0.5, dtype=torch.float16, device="cuda")], 1)


class Server:
    """Sequences with their caches and a small model of one block; all state on the GPU, updated in place."""

    def __init__(self, seed, B, Hq, Hkv, bits, width=40, spare=0):
        from trellis_serve_amd import ops
        self.ops, self.bits, self.shape = ops, bits, (B, Hq, Hkv)
        rng = np.random.default_rng(seed)
        self.V, self.hidden = 1024, 256
        P = B * width + spare
        self.cache = [torch.zeros((P, Hkv, PAGE, 16 * bits), dtype=torch.int8 if bits == 8 else torch.uint8, device="cuda")
                      for _ in range(2)] + [torch.zeros((P, Hkv), dtype=torch.float16, device="cuda") for _ in range(2)]
        self.bounds = torch.zeros((P, Hkv, 2, 16 * bits), dtype=self.cache[0].dtype, device="cuda")
        self.table = torch.zeros((B, width), dtype=torch.int32, device="cuda")
        self.ring, self.ring_state = _t(rng.permutation(P).astype(np.int32)), _t(np.array([0, P], np.int32))
        self.lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.qkv, self.o = _linear(rng, self.hidden, (Hq + 2 * Hkv) * D), _linear(rng, Hq * D, self.hidden)
        self.head = _linear(rng, self.hidden, self.V)
        half = lambda a: _t(a).half()   # noqa: E731
        self.qw, self.kw = half(1 + 0.1 * rng.standard_normal(D)), half(1 + 0.1 * rng.standard_normal(D))
        self.w, self.post = half(1 + 0.1 * rng.standard_normal(self.hidden)), half(1 + 0.1 * rng.standard_normal(self.hidden))
        self.gate = half(rng.standard_normal(self.hidden))
        self.cs = _t(_angles(2048, 128))
        self.embed = half(rng.standard_normal((self.V, self.hidden)))

    def state(self):
        return [*self.cache, self.bounds, self.table, self.ring, self.ring_state, self.lens]

    def step(self, x, new, uniform, keep=None):
        """x fp16 [rows, hidden]; new int32 [B]; returns the tokens drawn for every row."""
        ops, (B, Hq, Hkv), rows = self.ops, self.shape, x.shape[0]
        plan = ops.kv_step_plan(self.table, self.lens, new, self.ring, self.ring_state, rows)
        qkv = ops.linear(x, *self.qkv)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
        q, k = ops.qk_norm_rope(q, k, self.qw, self.kw, self.cs, plan.positions, EPS)
        ops.kv_append(k, v, *self.cache, self.table, self.lens, self.bits, row_start=plan.row_start, counts=plan.counts)
        ops.kv_page_bounds(self.cache[0], self.table, plan.lens_after, self.bits, self.bounds, first=self.lens, max_new=rows)
        pages = ops.kv_select_pages(q, self.bounds, self.cache[2], self.table, plan.row_lens, self.bits, TOP,
                                    row_seq=plan.row_seq)
        a = ops.kv_sparse_attention(q, *self.cache, self.table, plan.row_lens, self.bits, pages, row_seq=plan.row_seq)
        o = ops.linear(a.flatten(1), *self.o)
        y, h = ops.add_norm(o, x, self.w, EPS, post_weight=self.post, gate=self.gate, gate_sigmoid=True)
        logits = ops.linear(y, *self.head)
        tokens, probs = ops.sample_tokens(logits, uniform, 0.9, 200, 0.95, 0.001, return_probs=True)
        if keep is not None:
            keep.update(plan=plan, q=q, k=k, v=v, pages=pages, a=a, o=o, y=y, h=h, logits=logits, probs=probs)
        self.lens.copy_(plan.lens_after)
        return tokens


def _check_step(s, x, new, uniform):
    B, Hq, Hkv = s.shape
    before = [_n(t) for t in s.state()]
    table, ring, ring_state, lens = before[5:]
    keep = {}
    tokens = s.step(x, _t(new.astype(np.int32)), uniform, keep)
    want, table_w, ring_w, state_w = ref.plan(table, lens, new, ring, ring_state, x.shape[0])
    for g, w in zip(keep["plan"], want):
        assert np.array_equal(_n(g), w)
    assert np.array_equal(_n(s.table), table_w) and np.array_equal(_n(s.ring), ring_w)
    assert np.array_equal(_n(s.ring_state), state_w) and np.array_equal(_n(s.lens), want[2])
    starts, counts, after = want[:3]
    rows_of = [[starts[b] + i for i in range(counts[b])] for b in range(B)]
    for i, name in ((0, "k"), (1, "v")):
        got = keep[name].double().cpu().numpy()
        c, sc = attn_step_ref.append(got, before[i], before[2 + i], table_w, lens.tolist(), s.bits, rows_of)
        assert np.array_equal(_n(s.cache[i]), c) and np.array_equal(_n(s.cache[2 + i]), sc)
    edge = before[4].copy()
    for b in range(B):   # (a sequence without new tokens has nothing made anew)
        one = ref.bounds(_n(s.cache[0]), edge, table_w[b:b + 1], [int(after[b])], [int(lens[b])], s.bits)
        edge = one if after[b] > lens[b] else edge
    assert np.array_equal(_n(s.bounds), edge)
    q, row_lens, row_seq = _n(keep["q"]), want[4], want[5]
    chosen = ref.select(q, edge, _n(s.cache[2]), table_w, row_lens, s.bits, TOP, 1, 2, row_seq)
    assert np.array_equal(_n(keep["pages"]), chosen)
    _check_sparse(keep["a"], q, [_n(t) for t in s.cache], table_w, row_lens, s.bits, chosen, row_seq=row_seq)
    y, h, size = ref.add_norm(keep["o"].double().cpu().numpy(), x.double().cpu().numpy(), s.w.double().cpu().numpy(), EPS,
                              s.post.double().cpu().numpy(), s.gate.double().cpu().numpy(), True, 1.0, 0.0)
    for got, exact in ((keep["h"], h), (keep["y"], y)):   # a rounding, and fp32 sums of 256 terms
        d = np.abs(got.double().cpu().numpy() - exact)
        assert (d <= np.abs(exact) * 2.0 ** -11 + 2.0 ** -16 * (1 + size)).all()
    logits, u = keep["logits"].double().cpu().numpy(), uniform.cpu().numpy()
    for r in range(x.shape[0]):
        token, probs = ref.sample(logits[r], float(u[r]), 0.9, 200, 0.95, 0.001)
        assert int(tokens[r]) == token
        d = np.abs(_n(keep["probs"][r]).astype(np.float64) - probs)
        assert (d <= probs * (2.0 ** -24 + 2.0 ** -38)).all()
    return tokens


@pytest.mark.parametrize("bits,Hq,Hkv", [(8, 8, 2), (4, 10, 2)])
def test_loop_against_references(bits, Hq, Hkv):
    """Prompts in ragged chunks, decode steps, a sequence that ends, one that comes, a step that does not fit."""
    rng = np.random.default_rng(bits)
    B = 4
    s = Server(bits, B, Hq, Hkv, bits, spare=-100)   # 60 pages for 4 sequences
    steps = [np.array([200, 17, 0, 64]), np.array([1, 90, 33, 1]), np.array([1, 1, 1, 1]), np.array([130, 1, -40, 600]),
             np.array([-331, 1, 1, 1]), np.array([1, 1, 1, 220]), np.array([1, 1, 1, 1])]
    for new in steps:
        rows = int(np.maximum(new, 0).sum()) + (3 if new[0] == 1 else 0)   # some rows behind the last sequence
        x = _t(rng.standard_normal((rows, s.hidden))).half()
        _check_step(s, x, new, _t(rng.random(rows).astype(np.float32)))


@pytest.mark.parametrize("bits", [8, 4])
def test_loop_captured_and_replayed(bits):
    """Two servers in one state: one steps eagerly, the other by a graph, with eager work between the replays; every state and
    every token is the same."""
    B, rng = 5, np.random.default_rng(3)
    pair = [Server(11, B, 8, 2, bits) for _ in range(2)]
    prompt = np.array([150, 3, 97, 16, 400])
    x = _t(rng.standard_normal((int(prompt.sum()), 256))).half()
    u = _t(rng.random(int(prompt.sum())).astype(np.float32))
    for s in pair:
        s.step(x, _t(prompt.astype(np.int32)), u)
    eager, graphed = pair
    new, x, u = torch.ones(B, dtype=torch.int32, device="cuda"), torch.empty((B, 256), device="cuda").half(), torch.empty(B, device="cuda")
    x.copy_(_t(rng.standard_normal((B, 256))))
    u.copy_(_t(rng.random(B)))
    assert torch.equal(eager.step(x, new, u), graphed.step(x, new, u))   # (workspaces of the linears exist now)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    saved = [t.clone() for t in graphed.state()]
    with torch.cuda.graph(graph):
        tokens = graphed.step(x, new, u)
    for t, old in zip(graphed.state(), saved):
        assert torch.equal(t, old)   # capturing runs nothing
    for step in range(40):
        u.copy_(_t(rng.random(B)))
        if step % 3 == 1:
            new.copy_(_t(np.array([1, 0, 1, 1, -20], np.int32)))   # one waits, one gives tokens back
        else:
            new.fill_(1)
        want = eager.step(x, new, u)
        graph.replay()
        assert torch.equal(tokens, want)
        for a, b in zip(eager.state(), graphed.state()):
            assert torch.equal(a, b)
        x.copy_(eager.embed[want.clamp(min=0).long()])
        torch.cuda.synchronize()


def test_two_servers_on_two_streams():
    rng = np.random.default_rng(9)
    B, steps = 6, 12
    prompt = np.array([90, 31, 500, 7, 64, 222], np.int32)
    x0 = _t(rng.standard_normal((int(prompt.sum()), 256))).half()
    xs = [_t(rng.standard_normal((B, 256))).half() for _ in range(steps)]
    us = [_t(rng.random(B).astype(np.float32)) for _ in range(steps)]
    u0 = _t(rng.random(int(prompt.sum())).astype(np.float32))
    new0, new = _t(prompt), torch.ones(B, dtype=torch.int32, device="cuda")

    def operators(s, x, new, u):
        """The step without the linears, whose workspaces are one a device."""
        ops = s.ops
        plan = ops.kv_step_plan(s.table, s.lens, new, s.ring, s.ring_state, x.shape[0])
        heads = x.repeat(1, 8).unflatten(1, (16, D))
        q, k = ops.qk_norm_rope(heads[:, :8].contiguous(), heads[:, 8:10].contiguous(), s.qw, s.kw, s.cs, plan.positions, EPS)
        ops.kv_append(k, k, *s.cache, s.table, s.lens, s.bits, row_start=plan.row_start, counts=plan.counts)
        ops.kv_page_bounds(s.cache[0], s.table, plan.lens_after, s.bits, s.bounds, first=s.lens)
        pages = ops.kv_select_pages(q, s.bounds, s.cache[2], s.table, plan.row_lens, s.bits, TOP, row_seq=plan.row_seq)
        a = ops.kv_sparse_attention(q, *s.cache, s.table, plan.row_lens, s.bits, pages, row_seq=plan.row_seq)
        y, h = ops.add_norm(a.flatten(1)[:, :256], x, s.w, EPS)
        s.lens.copy_(plan.lens_after)
        return a, y, h, ops.sample_tokens(a.flatten(1), u, 0.8, 30, 0.9)

    want = []
    s = Server(1, B, 8, 2, 8)
    want.append(operators(s, x0, new0, u0))
    for x, u in zip(xs, us):
        want.append(operators(s, x, new, u))
    torch.cuda.synchronize()
    servers = [Server(1, B, 8, 2, 8) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in servers]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(steps + 1):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[j].append(operators(servers[j], x0 if i == 0 else xs[i - 1], new0 if i == 0 else new, u0 if i == 0 else us[i - 1]))
    torch.cuda.synchronize()
    for run in got:
        for step, expected in zip(run, want):
            assert all(torch.equal(a, b) for a, b in zip(step, expected))


def test_sampled_drafts_are_verified():
    """Drafts drawn by sample_tokens with their distributions, verified against sampling_probs of the target: where target and
    draft agree every draft stays; otherwise the accepted run is the reference's."""
    from trellis_serve_amd import ops
    rng = np.random.default_rng(6)
    B, N, V = 7, 5, 3000
    target = _t(3 * rng.standard_normal((B, N, V))).half()
    settings = dict(temperature=0.8, top_k=300, top_p=0.9)
    p = ops.sampling_probs(target, **settings)
    u = _t(rng.random((B, N)).astype(np.float32))
    for noise in (0.0, 0.7):
        draft = (target.float() + noise * _t(rng.standard_normal((B, N, V)))).half()
        drawn, q = ops.sample_tokens(draft, _t(rng.random((B, N)).astype(np.float32)), **settings, return_probs=True)
        tokens = torch.cat([torch.zeros((B, 1), dtype=torch.int32, device="cuda"), drawn[:, :-1]], dim=1)
        accepted, counts, out = ops.verify_drafts(p, tokens, u, draft_probs=q)
        want = attn_step_ref.verify(_n(p), _n(q), _n(tokens), None, _n(u), None)
        assert np.array_equal(_n(accepted), want[0]) and np.array_equal(_n(counts), want[1])
        if noise == 0.0:
            assert (counts == N).all()
            assert torch.equal(out[:, :-1], drawn[:, :-1])
