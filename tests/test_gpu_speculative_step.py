"""The operators around the quantized-KV attention together, as a speculative decoding step uses them: fused q/k/v linear ->
norms with rotation -> attention of the drafted tokens over the cache -> verification -> the accepted nodes' keys and values
into the cache -> decode attention and read-back of what was written.  Each stage is held to its 64-bit reference on the
inputs that the stage before gave it; then the same step eagerly, captured into a graph and replayed, and from two streams."""
import numpy as np
import pytest
import torch

import attn_step_ref as ref
from test_gpu_attn_step import D, PAGE, _angles, _check_tree, _masks, _probs, _random_cache, _t

pytestmark = pytest.mark.gpu


class Step:
    """A batch of sequences with a cache, and the inputs of one step (fixed tensors, as a captured graph needs them)."""

    def __init__(self, seed, B, N, Hq, Hkv, V, bits, longest):
        from trellis_serve_amd import ops
        self.ops, self.bits, self.shape = ops, bits, (B, N, Hq, Hkv, V)
        self.rng = rng = np.random.default_rng(seed)
        self.width = -(-(longest + 8 * N) // PAGE)
        P = B * self.width
        self.cache = [_t(c) for c in _random_cache(rng, P, Hkv, bits)]
        self.table = rng.permutation(P).reshape(B, self.width).astype(np.int32)
        self.table_t = _t(self.table)
        self.lens = _t(rng.integers(0, longest + 1, B).astype(np.int32))
        self.qw, self.kw = (_t(1 + 0.1 * rng.standard_normal(D)).half() for _ in range(2))
        self.cs = _t(_angles(4096, 128))
        ns = [Hq * D, Hkv * D, Hkv * D]
        self.k_in = 256
        self.tr = [_t(rng.integers(-32768, 32768, (self.k_in // 16, n // 16, 48), dtype=np.int16)) for n in ns]
        self.suh = [torch.ones(self.k_in, dtype=torch.float16, device="cuda") for _ in ns]
        self.svh = [torch.full((n,), self.k_in ** -0.5, dtype=torch.float16, device="cuda") for n in ns]
        self.x = torch.empty((B * N, self.k_in), dtype=torch.float16, device="cuda")
        self.p = torch.empty((B, N, V), device="cuda")
        self.u = torch.empty((B, N), device="cuda")
        self.tokens, self.parents = (torch.empty((B, N), dtype=torch.int32, device="cuda") for _ in range(2))
        self.mask = torch.empty((B, N), dtype=torch.int64, device="cuda")
        self.depth = torch.empty((B, N), dtype=torch.int32, device="cuda")
        self.new_inputs()

    def new_inputs(self):
        B, N, Hq, Hkv, V = self.shape
        rng = self.rng
        parents, depth = np.full((B, N), -1), np.zeros((B, N), np.int64)
        seen = np.zeros((B, N, N), bool)
        p = _probs(rng, B, N, V, sharp=4.0)   # peaked: drafts are accepted
        tokens = rng.integers(0, V, (B, N))
        for b in range(B):
            for i in range(N):
                if i:
                    up = parents[b, i] = rng.integers(max(0, i - 3), i)
                    seen[b, i], depth[b, i] = seen[b, up], depth[b, up] + 1
                    tokens[b, i] = np.argsort(-p[b, up])[rng.integers(0, 2)]
                seen[b, i, i] = True
        self.seen = seen
        for dst, src in ((self.x, rng.standard_normal((B * N, self.k_in))), (self.p, p), (self.u, rng.random((B, N))),
                         (self.tokens, tokens), (self.parents, parents), (self.mask, _masks(seen)), (self.depth, depth)):
            dst.copy_(torch.from_numpy(src))

    def run(self):
        B, N, Hq, Hkv, V = self.shape
        ops = self.ops
        qkv = ops.linear(self.x, self.tr, self.suh, self.svh, 1).view(B * N, -1)
        q, k = qkv[:, :Hq * D].unflatten(1, (Hq, D)), qkv[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D))
        v = qkv.view(B, N, -1)[..., (Hq + Hkv) * D:].unflatten(2, (Hkv, D))
        pos = (self.lens[:, None] + self.depth).view(-1)
        q, k = ops.qk_norm_rope(q, k, self.qw, self.kw, self.cs, pos)
        q, k = q.view(B, N, Hq, D), k.view(B, N, Hkv, D)
        o = ops.kv_tree_attention(q, k, v, self.mask, *self.cache, self.table_t, self.lens, self.bits)
        nodes, counts, out = ops.verify_drafts(self.p, self.tokens, self.u, parents=self.parents)
        ops.kv_append(k, v, *self.cache, self.table_t, self.lens, self.bits, select=nodes, counts=counts)
        self.lens.add_(counts)
        dec = ops.kv_decode_attention(q[:, 0].contiguous(), *self.cache, self.table_t, self.lens, self.bits)
        return q, k, v, o, nodes, counts, out, dec


@pytest.mark.parametrize("bits", [8, 4])
def test_speculative_steps_stage_by_stage(bits):
    B, N, Hq, Hkv, V = 3, 7, 8, 2, 1000
    s = Step(50 + bits, B, N, Hq, Hkv, V, bits, 70)
    emitted = 0
    for _ in range(4):
        cache0, lens0 = [c.cpu().numpy() for c in s.cache], s.lens.cpu().numpy()
        q, k, v, o, nodes, counts, out, dec = s.run()
        _check_tree(o, q, k, v, s.seen, cache0, s.table, lens0, bits)
        want = ref.verify(s.p.cpu().numpy(), None, s.tokens.cpu().numpy(), s.parents.cpu().numpy(), s.u.cpu().numpy(), None)
        for g, w in zip((nodes, counts, out), want):
            assert np.array_equal(g.cpu().numpy(), w)
        rows_of = [[b * N + i for i in want[0][b, :want[1][b]]] for b in range(B)]
        for x, c in ((k, 0), (v, 1)):
            wc, ws = ref.append(x.double().cpu().numpy().reshape(B * N, Hkv, D), cache0[c], cache0[2 + c], s.table, lens0,
                                bits, rows_of)
            assert np.array_equal(s.cache[c].cpu().numpy(), wc)
            assert np.array_equal(s.cache[2 + c].cpu().numpy(), ws)
        lens1 = lens0 + want[1]
        assert np.array_equal(s.lens.cpu().numpy(), lens1)
        cache1 = [c.cpu().numpy() for c in s.cache]
        empty = np.zeros((B, 1, 1), bool)
        _check_tree(dec[:, None], q[:, :1], k[:, :1], v[:, :1], empty, cache1, s.table, lens1, bits)
        start = np.concatenate([[0], np.cumsum(lens1)]).astype(np.int32)
        back = s.ops.kv_gather(*s.cache, s.table_t, s.lens, bits, _t(start), int(start[-1]))
        for b in range(B):
            for y, c in zip(back, (0, 1)):
                want_v = ref.values(cache1[c], cache1[2 + c], s.table[b], lens1[b], bits)
                assert np.array_equal(y[start[b]:start[b + 1]].cpu().numpy(), want_v.astype(np.float16))
        emitted += int(want[1].sum())
        s.new_inputs()
    assert emitted > 4 * B   # some drafts were taken


def _state(s):
    return [t.clone() for t in (*s.cache, s.lens)]


def _restore(s, state):
    for t, x in zip((*s.cache, s.lens), state):
        t.copy_(x)


def test_captured_steps_equal_eager_ones():
    """Two graphs, of different shapes, captured one after the other; replayed in turns, four times each with new inputs, with
    eager work and synchronisations between; each replay against the eager step from the same state."""
    steps = [Step(1, 3, 7, 8, 2, 1000, 8, 300), Step(2, 5, 16, 10, 2, 4099, 4, 900)]
    graphs, outs = [], []
    for s in steps:   # the linears' and the decode attention's reservations, as an engine makes them at load
        B, N, Hq, Hkv, _ = s.shape
        s.ops.reserve_linear(s.x.device, B * N, s.k_in, (Hq + 2 * Hkv) * D, 3)
        s.ops.reserve_prefill(s.x.device, B * N, s.k_in, (Hq + 2 * Hkv) * D, 3)
        s.ops.reserve_kv(s.x.device, B, Hq, Hkv, s.width)
    for s in steps:
        state = _state(s)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.run()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
        _restore(s, state)
    for _ in range(4):
        for s, g, o in zip(steps, graphs, outs):
            s.new_inputs()
            state = _state(s)
            want = [t.clone() for t in s.run()]
            after = _state(s)
            _restore(s, state)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(o, want):
                assert torch.equal(a, b)
            for a, b in zip(_state(s), after):
                assert torch.equal(a, b)


def test_steps_on_two_streams_at_once():
    """Two sequences' batches on two streams, with nothing between them: tree attention and verification take workspaces of
    their own."""
    steps = [Step(5, 4, 16, 10, 2, 5000, 8, 2000), Step(6, 4, 16, 10, 2, 5000, 8, 2000)]
    args, want = [], []
    for s in steps:
        q, k, v, *_ = s.run()
        a = (q, k, v, s.mask, *s.cache, s.table_t, s.lens, 8)
        args.append(a)
        want.append((s.ops.kv_tree_attention(*a), *s.ops.verify_drafts(s.p, s.tokens, s.u, parents=s.parents)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(steps):
            with torch.cuda.stream(streams[i]):
                got[i].append((s.ops.kv_tree_attention(*args[i]),
                               *s.ops.verify_drafts(s.p, s.tokens, s.u, parents=s.parents)))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


def test_prompt_chunks_equal_one_append():
    """A prompt written in chunks that end at page borders equals the prompt written at once, and its read-back and the decode
    attention over it agree with the reference."""
    from trellis_serve_amd import ops
    rng = np.random.default_rng(3)
    Hkv, n = 2, 200
    k = torch.from_numpy(rng.standard_normal((n, Hkv, D))).half().cuda()
    for bits in (8, 4):
        caches = [[_t(c) for c in _random_cache(np.random.default_rng(1), 13, Hkv, bits)] for _ in range(2)]
        table = _t(rng.permutation(13).reshape(1, 13).astype(np.int32))
        i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")   # noqa: E731
        ops.kv_append(k, k, *caches[0], table, i32(0), bits, row_start=i32(0, n))
        for a, b in ((0, 48), (48, 64), (64, 192), (192, 200)):
            ops.kv_append(k[a:b], k[a:b], *caches[1], table, i32(a), bits, row_start=i32(0, b - a), max_new=b - a)
        for x, y in zip(*caches):
            assert torch.equal(x, y)
        back, _ = ops.kv_gather(*caches[0], table, i32(n), bits, i32(0, n), n)
        scale = caches[0][2][table[0].long()].float().repeat_interleave(PAGE, 0)[:n, :, None]
        # half a step, and the read-back's rounding to fp16
        assert ((back.float() - k.float()).abs() <= scale / 2 + back.float().abs() * 2.0 ** -11).all()
