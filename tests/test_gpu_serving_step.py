"""GPU parity of the operators around the attention and at the ends of a serving step (step plans, residual norms, page bounds,
choice of pages and attention over them, sampling) against 64-bit references in plain numpy.  The reference project has no such
kernels: parity unpinned against it.  Whole numbers are compared for equality; the tolerances of the floating results count
their roundings and are derived beside their uses."""
import numpy as np
import pytest
import torch

import attn_step_ref
import serving_step_ref as ref

pytestmark = pytest.mark.gpu

D, PAGE = 128, 16
T_OF = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _ops():
    from trellis_serve_amd import ops
    return ops


def _t(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _i(a):
    return _t(np.asarray(a, dtype=np.int32))


def _n(t):
    return t.cpu().numpy()


def _typed(a, dtype):
    """The values of a in a type: the tensor, and the same values in float64."""
    t = torch.from_numpy(np.ascontiguousarray(a)).to(T_OF[dtype])
    return t.cuda(), t.double().numpy()


# ---- step plans --------------------------------------------------------------------------------------------------------

def _check_plan(table, lens, new, ring, state, rows, in_place=False):
    want, table_w, ring_w, state_w = ref.plan(table, lens, new, ring, state, rows)
    table_t, ring_t, state_t = _i(table), _i(ring), _i(state)
    state_out = state_t if in_place else torch.full_like(state_t, 77)
    got = _ops().kv_step_plan(table_t, _i(lens), _i(new), ring_t, state_t, rows, None if in_place else state_out)
    for name, g, w in zip(got._fields, got, want):
        assert g.dtype == (torch.int64 if name == "slots" else torch.int32)
        assert np.array_equal(_n(g), w), (name, np.flatnonzero(_n(g) != w)[:8])
    assert np.array_equal(_n(table_t), table_w)
    assert np.array_equal(_n(ring_t), ring_w)
    assert np.array_equal(_n(state_out), state_w)
    if not in_place:
        assert np.array_equal(_n(state_t), state)
    return want


def _plan_case(seed, B, W, longest, most, extra, shrink=0.2):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, longest + 1, B)
    new = rng.integers(0, most + 1, B)
    new = np.where(rng.random(B) < shrink, -rng.integers(1, longest + 2, B), new)
    used = sum(-(-int(n) // PAGE) for n in lens)
    need = sum(-(-int(n + max(m, 0)) // PAGE) - -(-int(n) // PAGE) for n, m in zip(lens, new))
    P = used + need + max(extra, 0) + 3
    perm = rng.permutation(P)
    table, at = np.full((B, W), -1), 0
    for b, n in enumerate(lens):
        k = -(-int(n) // PAGE)
        table[b, :k] = perm[at:at + k]
        at += k
    live = max(0, need + extra)
    ring, head = np.full(P, 1 << 20), int(rng.integers(0, P))
    ring[(head + np.arange(live)) % P] = perm[at:at + live]
    return table, lens, new, ring, np.array([head, live]), int(np.maximum(new, 0).sum())


@pytest.mark.parametrize("B,W,longest,most,extra", [
    (1, 1, 0, 1, 0), (1, 4, 33, 17, 5), (3, 8, 60, 40, 0), (8, 300, 4096, 1, 2), (64, 20, 200, 33, -4), (65, 64, 700, 8, 9),
    (256, 64, 500, 7, 0), (257, 64, 500, 7, -20), (300, 40, 300, 60, 10), (1024, 30, 256, 40, 0), (1025, 30, 200, 20, -200),
    (2500, 16, 150, 9, 3), (2, 600, 3000, 5000, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_step_plan(B, W, longest, most, extra, in_place):
    table, lens, new, ring, state, rows = _plan_case(B + W, B, W, longest, most, extra)
    _check_plan(table, lens, new, ring, state, rows, in_place)


@pytest.mark.parametrize("B,W,longest,most", [(5, 9, 100, 30), (400, 12, 100, 30), (1100, 40, 600, 10)])
def test_step_plan_of_steps_that_do_not_fit(B, W, longest, most):
    """Too few rows, rows behind the last sequence, table rows that end before their tokens, an empty ring, odd lengths."""
    table, lens, new, ring, state, rows = _plan_case(B, B, W, longest, most, 4)
    for r in (0, rows // 2, rows + 100):
        _check_plan(table, lens, new, ring, state, r)
    _check_plan(table, lens, new, ring, np.array([state[0], 0]), rows)
    new2 = new.copy()
    new2[::3] = W * PAGE
    new2[1::7] = 2 ** 31 - 1
    new2[2::11] = -2 ** 31
    _check_plan(table, lens, new2, ring, state, rows)
    lens2 = lens.copy()
    lens2[::5] = -4
    _check_plan(table, lens2, new, ring, state, rows)
    _check_plan(table, np.full(B, W * PAGE + 9) if (table >= 0).all() else lens, np.zeros(B, int), ring, state, 0)


def test_step_plan_empty():
    plan = _ops().kv_step_plan(torch.empty((0, 4), dtype=torch.int32, device="cuda"), _i([]), _i([]), _i([1]), _i([0, 1]), 0)
    assert [tuple(t.shape) for t in plan] == [(1,), (0,), (0,), (0,), (0,), (0,), (0,)] and plan.row_start.item() == 0


def test_step_plan_pages_circulate():
    """Steps in a row, in place: every page is in the ring or in one table row, whatever is taken and given back."""
    rng = np.random.default_rng(5)
    B, W, P = 9, 20, 60
    table, ring = torch.full((B, W), -1, dtype=torch.int32, device="cuda"), _i(rng.permutation(P))
    state, lens = _i([0, P]), _i(np.zeros(B))
    for step in range(60):
        new = rng.integers(-120, 60, B)
        rows = int(np.maximum(new, 0).sum())
        args = _n(table), _n(lens), new, _n(ring), _n(state), rows
        want, table_w, ring_w, state_w = ref.plan(*args)
        plan = _ops().kv_step_plan(table, lens, _i(new), ring, state, rows)
        assert np.array_equal(_n(table), table_w) and np.array_equal(_n(ring), ring_w) and np.array_equal(_n(state), state_w)
        assert all(np.array_equal(_n(g), w) for g, w in zip(plan, want))
        lens = plan.lens_after.clone()
        held = [int(p) for b, n in enumerate(_n(lens)) for p in _n(table)[b, :-(-int(n) // PAGE)]]
        head, live = _n(state)
        assert sorted(held + [int(_n(ring)[(head + j) % P]) for j in range(live)]) == list(range(P))


# ---- residual norms ----------------------------------------------------------------------------------------------------

def _check_norm(T, dim, dtype="bf16", res="bf16", w="bf16", post=True, gate="none", g="bf16", sigmoid=False, scale=0.5,
                offset=False, pre=True, spread=True, pad=0, eps=1e-5, in_place=False):
    rng = np.random.default_rng(T * 7919 + dim)
    size = rng.uniform(0.01, 30, (T, 1)) if spread else np.ones((T, 1))
    x, x64 = _typed(rng.standard_normal((T, dim + pad)) * size, dtype)
    x, x64 = x[:, :dim], x64[:, :dim]
    r = r64 = None
    if res:
        r, r64 = _typed(rng.standard_normal((T, dim + pad)) * 3, res)
        r, r64 = r[:, :dim], r64[:, :dim]
    one = 0.0 if offset else 1.0
    wt, wt64 = _typed(one + 0.3 * rng.standard_normal(dim), w) if pre else (None, None)
    pw, pw64 = _typed(one + 0.3 * rng.standard_normal(dim), w) if post else (None, None)
    gt = gt64 = None
    if gate != "none":
        shape = {"channel": (dim,), "token": (T, 1), "full": (T, dim + pad)}[gate]
        gt, gt64 = _typed(rng.standard_normal(shape), g)
        if gate == "full":
            gt, gt64 = gt[:, :dim], gt64[:, :dim]
    y64, h64, size = ref.add_norm(x64, r64, wt64, eps, pw64, gt64, sigmoid, scale, 1.0 if offset else 0.0)
    out = None
    if in_place:
        r = r.contiguous()
        out = (None, r) if not pre else (torch.empty((T, dim), dtype=x.dtype, device="cuda"), r)
    y, h = _ops().add_norm(x, r, wt, eps, post_weight=pw, gate=gt, gate_sigmoid=sigmoid, scale=scale, unit_offset=offset,
                           out=out)
    # fp32 inside: a sum of squares of n terms, at most 64 in a row and then pairwise, is off by some 80 roundings, its root by
    # half of that; with the products 64 of 2^-24 for each norm, of the magnitudes of h's terms
    fp32 = 64 * 2.0 ** -24
    half = {t: torch.finfo(T_OF[t]).eps / 2 for t in T_OF}
    tiny = {"fp16": 2.0 ** -25, "bf16": 0.0, "fp32": 0.0}
    assert h.dtype == T_OF[res or dtype] and h.shape == (T, dim) and h.is_contiguous()
    d = np.abs(h.double().cpu().numpy() - h64)
    tol = np.abs(h64) * half[res or dtype] + size * fp32 * (1 + half[res or dtype]) + tiny[res or dtype]
    assert (d <= tol).all(), (d / np.maximum(tol, 1e-300)).max()
    if not pre:
        assert y is None
        return
    assert y.dtype == x.dtype and y.shape == (T, dim) and y.is_contiguous()
    rms = np.sqrt((h64 * h64).mean(-1, keepdims=True) + eps)
    # h's own error reaches y through its value and through the norm (by the mean of |error| |h| / rms^2 <= rms(error) / rms)
    dh = size * fp32
    through = np.abs(wt64 + (1.0 if offset else 0.0)) / rms * dh + np.abs(y64) * np.sqrt((dh * dh).mean(-1, keepdims=True)) / rms
    tol = np.abs(y64) * (half[dtype] + 2 * fp32) + through * (1 + half[dtype]) + tiny[dtype]
    d = np.abs(y.double().cpu().numpy() - y64)
    assert (d <= tol).all(), (d / np.maximum(tol, 1e-300)).max()


@pytest.mark.parametrize("T,dim", [(1, 1), (3, 2), (5, 7), (2, 8), (1, 64), (9, 100), (4, 513), (33, 640), (1, 5120), (130, 4096),
                                   (7, 5121), (3, 8200), (2, 16384), (2, 16387), (1, 32768), (1, 32767), (1100, 8192), (1030, 9000), (1025, 16384), (700, 5120),
                                   (2100, 1280), (1030, 8192), (5000, 72)])
@pytest.mark.parametrize("post,gate,dtype", [(False, "none", "bf16"), (True, "channel", "fp16"), (True, "token", "bf16"),
                                             (False, "full", "fp16")])
def test_add_norm(T, dim, post, gate, dtype):
    if dim == 1 and gate == "full":
        gate = "token"
    _check_norm(T, dim, dtype, dtype, dtype, post, gate, dtype, sigmoid=T % 2 == 0, scale=1.0 if T % 3 else 0.22,
                offset=dim % 3 == 0)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("res", ["fp16", "bf16", "fp32", None])
@pytest.mark.parametrize("w,g", [("fp32", "fp16"), ("bf16", "fp32"), ("fp16", "bf16")])
def test_add_norm_types(dtype, res, w, g):
    for gate, dim, T in (("channel", 264, 5), ("full", 263, 3), ("token", 1024, 18)):
        _check_norm(T, dim, dtype, res, w, True, gate, g, sigmoid=True, pad=8 if dim % 8 == 0 else 3)


@pytest.mark.parametrize("T,dim,pad", [(6, 512, 8), (6, 512, 1), (300, 1280, 40), (4, 100, 5), (1300, 640, 8)])
def test_add_norm_strides_and_in_place(T, dim, pad):
    _check_norm(T, dim, pad=pad, gate="full")
    _check_norm(T, dim, pad=pad, gate="token", in_place=True)
    _check_norm(T, dim, pad=pad, pre=False, in_place=True)
    _check_norm(T, dim, pad=pad, pre=False, post=False, res=None)


def test_add_norm_misaligned():
    """Rows that begin at other places than multiples of 16 bytes."""
    rng = np.random.default_rng(3)
    base = torch.randn(3 * 512 + 1, device="cuda").half()
    x, r = base[1:1 + 3 * 512].view(3, 512), torch.randn(3, 512, device="cuda").half()
    w = torch.randn(513, device="cuda").half()[1:]
    y, h = _ops().add_norm(x, r, w)
    y2, h2 = _ops().add_norm(x.clone(), r, w.clone())
    assert torch.equal(h, h2) and torch.allclose(y.float(), y2.float(), rtol=2.0 ** -9, atol=1e-6)
    del rng


def test_add_norm_zero_rows_and_special_values():
    ops = _ops()
    w = torch.ones(256, device="cuda").half()
    y, h = ops.add_norm(torch.zeros((0, 256), device="cuda").half(), torch.zeros((0, 256), device="cuda").half(), w)
    assert y.shape == h.shape == (0, 256)
    x = torch.zeros((4, 256), device="cuda").half()
    r = torch.zeros((4, 256), device="cuda").half()
    x[1, 5], x[2, 5], r[3, 9] = float("inf"), float("nan"), float("nan")
    y, h = ops.add_norm(x, r, w, post_weight=w)
    assert (y[0] == 0).all() and (h[0] == 0).all()          # eps keeps zeros zeros
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all() and torch.isnan(h[1, 5]) and not torch.isnan(y[0]).any()


# ---- page bounds ---------------------------------------------------------------------------------------------------------

def _random_cache(rng, P, Hkv, bits, spread=1.0):
    qmax = 127 if bits == 8 else 7
    codes = lambda: attn_step_ref.pack(np.clip(np.rint(rng.standard_normal((P, Hkv, PAGE, D)) * qmax / 3   # noqa: E731
                                                       + rng.standard_normal((P, Hkv, 1, D)) * qmax / 4 * spread),
                                               -qmax, qmax).astype(np.int64), bits)
    scale = lambda: (rng.uniform(0.5, 1.5, (P, Hkv)) * 3 / qmax).astype(np.float16)   # noqa: E731
    return [codes(), codes(), scale(), scale()]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens,first,Hkv,max_new", [
    ([1], None, 1, None), ([16], [15], 1, 1), ([17], [15], 2, 2), ([0, 15, 33], [0, 3, 33], 8, 40), ([64, 31], [63, 1], 5, 30),
    ([5] * 70, [4] * 70, 2, 1), ([700, 0, 129, 16], None, 4, None), ([700, 0, 129, 16], [650, -5, 200, 15], 4, 64),
    ([90, 90], [0, 0], 1, 20)])
def test_page_bounds(bits, lens, first, Hkv, max_new):
    rng = np.random.default_rng(sum(lens) + bits)
    width = max(1, -(-max(lens) // PAGE)) + 1
    P = len(lens) * width + 2
    cache = _random_cache(rng, P, Hkv, bits)
    table = rng.permutation(P)[:len(lens) * width].reshape(len(lens), width).astype(np.int32)
    old = rng.integers(0, 100, (P, Hkv, 2, 16 * bits)).astype(cache[0].dtype)
    got = _t(old)
    _ops().kv_page_bounds(_t(cache[0]), _t(table), _i(lens), bits, got, None if first is None else _i(first), max_new)
    want = ref.bounds(cache[0], old, table, lens, first, bits, 1 << 30 if max_new is None else max_new)
    assert np.array_equal(_n(got), want)


@pytest.mark.parametrize("bits", [8, 4])
def test_page_bounds_extremes_and_bad_pages(bits):
    """The type's lowest and highest codes, pages outside the cache, lengths past the table, slots past the last token."""
    rng = np.random.default_rng(bits)
    lo, hi = (-128, 127) if bits == 8 else (-8, 7)
    k = attn_step_ref.pack(rng.choice([lo, hi, 0, -1], (6, 3, PAGE, D)), bits)
    table = np.array([[2, -1, 9, 0], [6, 5, 3, 1]], np.int32)
    old = np.zeros((6, 3, 2, 16 * bits), k.dtype)
    got = _t(old)
    _ops().kv_page_bounds(_t(k), _t(table), _i([1000, 49]), bits, got)
    assert np.array_equal(_n(got), ref.bounds(k, old, table, [1000, 49], None, bits))


# ---- choice of pages -----------------------------------------------------------------------------------------------------

def _rows_case(seed, lens, Hq, Hkv, bits, spare=2, spread=1.0):
    rng = np.random.default_rng(seed)
    B, width = len(lens), max(1, -(-max(lens) // PAGE)) + spare
    P = B * width + 1
    cache = _random_cache(rng, P, Hkv, bits, spread)
    table = rng.permutation(P)[:B * width].reshape(B, width).astype(np.int32)
    edge = ref.bounds(cache[0], np.zeros((P, Hkv, 2, 16 * bits), cache[0].dtype), table, lens, None, bits)
    return rng, cache, table, edge, rng.standard_normal((B, Hq, D)).astype(np.float16)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens,Hq,Hkv,top,first,last", [
    ([1], 1, 1, 1, 0, 1), ([500], 5, 1, 4, 1, 2), ([0, 64, 65, 700], 16, 2, 4, 1, 2), ([1000], 16, 1, 1, 0, 1),
    ([1000, 3], 8, 8, 2, 0, 2), ([2000, 1999], 12, 4, 3, 1, 2), ([9000], 40, 8, 64, 1, 2), ([9000, 8193], 6, 2, 511, 0, 1),
    ([300] * 40, 2, 1, 10, 3, 5), ([40000], 3, 1, 100, 1, 2), ([33000], 1, 1, 2000, 4, 4)])
def test_select_pages(bits, lens, Hq, Hkv, top, first, last):
    rng, cache, table, edge, q = _rows_case(sum(lens) + bits, lens, Hq, Hkv, bits)
    got = _ops().kv_select_pages(_t(q), _t(edge), _t(cache[2]), _t(table), _i(lens), bits, top, first, last)
    want = ref.select(q, edge, cache[2], table, lens, bits, top, first, last)
    assert got.dtype == torch.int32 and np.array_equal(_n(got), want), np.argwhere(_n(got) != want)[:5]


@pytest.mark.parametrize("bits", [8, 4])
def test_select_pages_ties_and_odd_queries(bits):
    """Equal bounds everywhere, equal scales, two worths only; zero queries, infinities and NaN in queries and scales; page ids
    outside the cache; the codes' extremes."""
    lens = [1600, 1500, 800, 333, 1600]
    rng, cache, table, edge, q = _rows_case(9 + bits, lens, 6, 2, bits)
    table[3, :5] = [-7, 10 ** 6, 2, -1, 3]
    scale = cache[2]
    call = lambda q, e, s, top, first, last: (   # noqa: E731
        _n(_ops().kv_select_pages(_t(q), _t(e), _t(s), _t(table), _i(lens), bits, top, first, last)),
        ref.select(q, e, s, table, lens, bits, top, first, last))
    same = np.broadcast_to(edge[:1], edge.shape).copy()
    ones = np.ones_like(scale)
    odd = q.copy()
    odd[0] = 0
    odd[1, :3, ::5], odd[1, 3:, 7], odd[2, 1] = np.inf, -np.inf, np.nan
    odd[3, :, 1:] = np.nan
    odd[4] *= 6e-5
    bad = scale.copy()
    bad[table[0, 3:60:4]], bad[table[1, ::3]], bad[table[2, 5]] = np.nan, np.inf, 0
    wild = attn_step_ref.pack(rng.choice([-128, 127, 0] if bits == 8 else [-8, 7, 0], (*edge.shape[:3], D)), bits).astype(edge.dtype)
    for args in ((q, same, ones), (np.broadcast_to(q[:1], q.shape), same, scale), (odd, edge, scale), (odd, edge, bad),
                 (np.zeros_like(q), edge, scale), (q, wild, ones), (np.full_like(q, 65504), wild, np.full_like(scale, 65504))):
        for top, first, last in ((7, 1, 2), (30, 0, 1), (3, 1, 2), (50, 20, 10)):
            got, want = call(*args, top, first, last)
            assert np.array_equal(got, want), (top, np.argwhere(got != want)[:5])


@pytest.mark.parametrize("bits", [8, 4])
def test_rows_of_shared_sequences(bits):
    """row_seq: several rows a sequence, rows of none, columns of a wider tensor as queries."""
    lens = [900, 17, 2600]
    rng, cache, table, edge, _ = _rows_case(31, lens, 10, 2, bits)
    row_seq, seen = [2, 2, 0, 1, -1, 3, 2, 0, 1], [2600, 2599, 850, 17, 50, 60, 1, 0, 5000]
    wide = torch.randn((9, 10 * D + 64), device="cuda").half()
    q = wide[:, 32:32 + 10 * D].unflatten(1, (10, D))
    pages = _ops().kv_select_pages(q, _t(edge), _t(cache[2]), _t(table), _i(seen), bits, 12, row_seq=_i(row_seq))
    want = ref.select(_n(q), edge, cache[2], table, seen, bits, 12, 1, 2, row_seq)
    assert np.array_equal(_n(pages), want)
    got = _ops().kv_sparse_attention(q, *[_t(c) for c in cache], _t(table), _i(seen), bits, pages, row_seq=_i(row_seq))
    _check_sparse(got, _n(q), cache, table, seen, bits, want, row_seq=row_seq)
    assert (got[4:6] == 0).all() and (got[7] == 0).all()


# ---- attention over chosen pages -------------------------------------------------------------------------------------------

def _check_sparse(got, q, cache, table, seen, bits, pages, sm=D ** -0.5, row_seq=None):
    """The roundings of the tree attention, whose tolerance this is: probabilities in fp16 of the type's whole range, so that
    keys within 2^-25 of the largest p |v| keep half a step, the rest at most 2^-25 of it each."""
    out, mean, slip = ref.sparse_attention(q, cache, table, seen, bits, pages, sm, row_seq)
    vmax = float(np.nanmax(np.abs(cache[3].astype(np.float32)))) * (127 if bits == 8 else 8)
    tol = attn_step_ref.tree_tolerance(out, mean, slip, pages.shape[-1] * PAGE * 2.0 ** -11, vmax)
    got = got.double().cpu().numpy()
    # fp16 rounds magnitudes from 65520 up to infinity
    d = np.where(np.isinf(got) & (np.abs(out) + tol >= 65520) & (np.sign(got) == np.sign(out)), 0, np.abs(got - out))
    assert (d <= tol).all(), ((d / tol).max(), d.max())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens,Hq,Hkv,top", [
    ([1], 1, 1, 1), ([16, 0, 17], 5, 1, 3), ([333], 16, 1, 5), ([700, 64, 5], 40, 8, 64), ([3000] * 20, 8, 2, 33),
    ([9000], 32, 8, 200), ([2000] * 70, 8, 8, 16), ([5000, 40], 6, 2, 129), ([1000], 12, 4, 1), ([700] * 300, 4, 2, 7)])
def test_sparse_attention(bits, lens, Hq, Hkv, top):
    rng, cache, table, edge, q = _rows_case(sum(lens) * 3 + bits, lens, Hq, Hkv, bits)
    pages = np.full((len(lens), Hkv, top), -1, np.int32)
    for r, n in enumerate(lens):
        have = -(-n // PAGE)
        for h in range(Hkv):
            take = rng.permutation(have)[:top]
            pages[r, h, :len(take)] = np.sort(take) if r % 2 else take
    got = _ops().kv_sparse_attention(_t(q), *[_t(c) for c in cache], _t(table), _i(lens), bits, _t(pages))
    _check_sparse(got, q, cache, table, lens, bits, pages)


def test_sparse_attention_lists_of_other_choices():
    """Entries that are no page of what the row sees, anywhere in the list; a list of none; page ids outside the cache."""
    lens = [500, 100, 260]
    rng, cache, table, edge, q = _rows_case(4, lens, 8, 2, 8)
    table[2, 3], table[2, 4] = -5, 10 ** 7
    pages = np.full((3, 2, 9), -1, np.int32)
    pages[0, 0] = [31, -1, 32, 3, -9, 2 ** 30, 0, 31 + 2 ** 20, 7]
    pages[0, 1, 8] = 5
    pages[2] = [16, 3, 4, 0, -1, 17, 1, -2, 2]
    got = _ops().kv_sparse_attention(_t(q), *[_t(c) for c in cache], _t(table), _i(lens), 8, _t(pages))
    _check_sparse(got, q, cache, table, lens, 8, pages)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_sparse_attention_scales(bits):
    """Value scales from fp16's subnormals to its largest, zero scales, sharp and negative softmax scales, stale codes and
    scales in pages that are not read."""
    lens, top = [1500, 1490], 40
    rng, cache, table, edge, q = _rows_case(8, lens, 10, 2, bits)
    pages = np.stack([[np.sort(rng.permutation(93)[:top]) for _ in range(2)] for _ in lens]).astype(np.int32)
    read = np.zeros((len(cache[0]), 2), bool)
    for r in range(2):
        for h in range(2):
            read[table[r, pages[r, h]], h] = True
    for sm, vs in ((D ** -0.5, 2.0 ** -24), (D ** -0.5, 2.0 ** -16), (2.0, 0.01), (-0.3, 300.0), (0.02, 2.0)):
        scales = (rng.uniform(1, 2, cache[3].shape) * vs).astype(np.float16)
        scales[~read] = np.nan
        ks = cache[2].copy()
        ks[~read] = np.inf
        c = [cache[0], cache[1], ks, scales]
        got = _ops().kv_sparse_attention(_t(q), *[_t(x) for x in c], _t(table), _i(lens), bits, _t(pages), sm)
        ks2 = np.where(read, ks, 0).astype(np.float16)
        _check_sparse(got, q, [cache[0], cache[1], ks2, np.where(read, scales, 0).astype(np.float16)], table, lens, bits, pages, sm)
    zero = [cache[0], cache[1], cache[2], np.zeros_like(cache[3])]
    zero[3][table[1, pages[1, 0, 3]], 0] = 0.5
    got = _ops().kv_sparse_attention(_t(q), *[_t(x) for x in zero], _t(table), _i(lens), bits, _t(pages))
    _check_sparse(got, q, zero, table, lens, bits, pages)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_sparse_attention_over_all_pages_is_decode_attention(bits):
    lens = [700, 1, 333, 64]
    rng, cache, table, edge, q = _rows_case(12, lens, 20, 4, bits)
    c = [_t(x) for x in cache]
    pages = _ops().kv_select_pages(_t(q), _t(edge), c[2], _t(table), _i(lens), bits, 46)
    got = _ops().kv_sparse_attention(_t(q), *c, _t(table), _i(lens), bits, pages)
    whole = _ops().kv_decode_attention(_t(q), *c, _t(table), _i(lens), bits)
    want = _n(pages)
    _check_sparse(got, q, cache, table, lens, bits, want)
    _check_sparse(whole, q, cache, table, lens, bits, want)


def test_pages_past_four_gigabytes():
    """Codes, bounds and pages behind 2^32 bytes."""
    P, Hkv, bits = 300000, 8, 8   # 4.9 GB of key codes
    ops = _ops()
    k = torch.zeros((P, Hkv, PAGE, D), dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    rng = np.random.default_rng(0)
    lens, ids = [16 * 30], P - 40 + rng.permutation(32)
    small = _random_cache(rng, 32, Hkv, bits)
    scales = [torch.ones((P, Hkv), dtype=torch.float16, device="cuda") for _ in range(2)]
    for t, s in ((k, small[0]), (v, small[1]), (scales[0], small[2]), (scales[1], small[3])):
        t[P - 40:P - 8] = _t(s)
    table = ids.reshape(1, -1).astype(np.int32)
    edge = torch.zeros((P, Hkv, 2, D), dtype=torch.int8, device="cuda")
    ops.kv_page_bounds(k, _t(table), _i(lens), bits, edge)
    near = ids - (P - 40)
    want = ref.bounds(small[0], np.zeros((32, Hkv, 2, D), np.int8), near.reshape(1, -1), lens, None, bits)
    assert np.array_equal(_n(edge[P - 40:P - 8]), want) and not edge[:P - 40].any()
    q = rng.standard_normal((1, 16, D)).astype(np.float16)
    pages = ops.kv_select_pages(_t(q), edge, scales[0], _t(table), _i(lens), bits, 8)
    chosen = ref.select(q, want, small[2], near.reshape(1, -1), lens, bits, 8, 1, 2)
    assert np.array_equal(_n(pages), chosen)
    got = ops.kv_sparse_attention(_t(q), k, v, *scales, _t(table), _i(lens), bits, pages)
    _check_sparse(got, q, small, near.reshape(1, -1), lens, bits, chosen)


# ---- sampling ------------------------------------------------------------------------------------------------------------

def _check_sample(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    """logits: a tensor [B, V]; settings: numbers, or arrays of one a row."""
    B, V = logits.shape
    one = lambda x, b: float(x[b]) if isinstance(x, np.ndarray) else x   # noqa: E731
    dev = lambda x, d: _t(x.astype(d)) if isinstance(x, np.ndarray) else x   # noqa: E731
    settings = dev(t, np.float32), dev(k, np.int32), dev(p, np.float32), dev(m, np.float32)
    settings64 = [x.astype(d) if isinstance(x, np.ndarray) else x
                  for x, d in zip((t, k, p, m), (np.float32, np.int32, np.float32, np.float32))]
    u = u.astype(np.float32)
    tokens, probs = _ops().sample_tokens(logits, _t(u), *settings, return_probs=True)
    x = logits.double().cpu().numpy()
    got_t, got_p = _n(tokens), _n(probs).astype(np.float64)
    for b in range(B):
        token, want = ref.sample(x[b], float(u[b]), one(settings64[0], b), int(one(settings64[1], b)), one(settings64[2], b),
                                 one(settings64[3], b))
        assert got_t[b] == token, (b, got_t[b], token)
        # one rounding to fp32 (2^-149 where it is subnormal); the 64-bit weights and sums are within 2^-40
        d = np.abs(got_p[b] - want)
        assert (d <= want * (2.0 ** -24 + 2.0 ** -38) + 2.0 ** -149).all(), (b, (d / np.maximum(want, 1e-300)).max())
        assert ((got_p[b] > 0) <= (want > 0)).all()
    assert torch.equal(_ops().sample_tokens(logits, _t(u), *settings), tokens)
    assert torch.equal(_ops().sampling_probs(logits, *settings), probs)


def _logits(rng, B, V, dtype, spread=2.5):
    x = rng.standard_normal((B, V)) * spread
    for b in range(B):
        x[b, rng.integers(0, V, 4)] += rng.uniform(2, 8, 4)
    return _t(x).to(T_OF[dtype])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 63), (4, 64), (9, 1000), (2, 4097), (1, 32003), (3, 50001), (70, 3001),
                                 (2, 131072)])
def test_sample_settings(dtype, B, V):
    rng = np.random.default_rng(B * 1000 + V)
    logits, u = _logits(rng, B, V, dtype), rng.random(B)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 50, 1.0, 0.0), (0.8, 40, 0.95, 0.05), (1.0, 1, 0.5, 0.5),
                       (0.0, 0, 1.0, 0.0), (2.0, 0, 1.0, 0.1), (1.0, V - 1 if V > 1 else 5, 0.3, 0.0), (1.0, 0, 0.0, 0.0),
                       (5.0, 700, 0.99, 0.001), (0.05, 0, 0.999, 1.0)):
        _check_sample(logits, u, t, k, p, m)
    some = lambda a, b: np.where(rng.random(B) < 0.3, a, b)   # noqa: E731
    _check_sample(logits, u, some(0.0, rng.uniform(0.2, 2, B)), some(0, rng.integers(-1, 2 * V, B)),
                  some(1.0, rng.uniform(0, 1.1, B)), some(0.0, rng.uniform(0, 0.3, B)))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_sample_ties(dtype):
    """Few different logits, so that every cut falls among equals; all equal; both zeros."""
    rng = np.random.default_rng(1)
    for V, values in ((5000, [0.0, 1.0, 1.5]), (40000, [-1.0, -0.5]), (3000, [0.0, -0.0]), (9000, [2.0])):
        logits = _t(rng.choice(values, (6, V))).to(T_OF[dtype])
        for t, k, p, m in ((1.0, 7, 1.0, 0.0), (1.0, V - 3, 0.7, 0.0), (0.5, 0, 0.31, 0.0), (1.0, 0, 1.0, 0.5), (0.0, 0, 1.0, 0.0),
                           (1.0, 2000, 0.9, 0.2)):
            _check_sample(logits, rng.random(6), t, k, p, m)


def test_sample_odd_logits():
    """Masks of -inf, of the type's lowest value, of NaN; rows that they leave nothing of; infinite logits; logits far apart
    and temperatures at either end."""
    rng = np.random.default_rng(2)
    V, low = 3000, torch.finfo(torch.float32).min
    x = 2 * rng.standard_normal((14, V)).astype(np.float32)
    x[0, 5:], x[1, ::2], x[2, :-1], x[3] = -np.inf, np.nan, low, -np.inf
    x[4], x[5], x[6, 77], x[7, [3, 9, 2999]] = np.nan, low, np.inf, np.inf
    x[8] = np.where(rng.random(V) < 0.5, low, 3.4e38)
    x[9], x[10] = -np.inf, -np.inf
    x[9, 2999], x[10, [0, 1]] = -1e30, [1e-40, -1e-40]
    x[11] *= 1e30
    x[12] *= 1e-30
    logits, u = _t(x), rng.random(14)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 30, 0.9, 0.0), (1e-30, 0, 0.9, 0.0), (1e30, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.1),
                       (0.0, 0, 1.0, 0.0), (1e-44, 5, 1.0, 0.0), (3e38, 100, 0.99, 0.9), (float("inf"), 0, 0.5, 0.0),
                       (1e300, 0, 0.9, 0.0)):
        _check_sample(logits, u, t, k, p, m)
    tokens, probs = _ops().sample_tokens(logits, _t(u.astype(np.float32)), return_probs=True)
    assert tokens[3] == tokens[4] == -1 and not probs[3].any() and not probs[4].any()
    nan = np.full(14, np.nan)
    _check_sample(logits, u, np.ones(14), np.zeros(14), np.where(np.arange(14) % 2, nan, 2.0), np.where(np.arange(14) % 2, nan, -1.0))
    assert torch.equal(_ops().sample_tokens(logits, _t(u.astype(np.float32)), _t(nan.astype(np.float32))),
                       _ops().sample_tokens(logits, _t(u.astype(np.float32)), 0.0))


def test_sample_covers_its_distribution():
    """Random numbers across [0, 1) give each kept token its share, and no other token."""
    rng = np.random.default_rng(3)
    row = _logits(rng, 1, 50, "fp32", 1.0)
    n = 16384
    u = (np.arange(n) + 0.5) / n
    tokens = _n(_ops().sample_tokens(row.expand(n, 50).contiguous(), _t(u.astype(np.float32)), 0.8, 20, 0.9, 0.01))
    _, want = ref.sample(_n(row)[0], 0.5, 0.8, 20, 0.9, 0.01)
    share = np.bincount(tokens, minlength=50) / n
    assert np.abs(share - want).max() <= 1.01 / n and (share[want == 0] == 0).all()
    ends = _n(_ops().sample_tokens(row.expand(4, 50).contiguous(), _t(np.array([0, 1 - 2.0 ** -24, 1, -1], np.float32)), 0.8, 20))
    kept = np.flatnonzero(ref.sample(_n(row)[0], 0.5, 0.8, 20, 1.0, 0.0)[1])
    assert ends.tolist() == [kept[0], kept[-1], kept[-1], kept[0]]


def test_sample_shapes_and_strides():
    rng = np.random.default_rng(4)
    logits = _logits(rng, 12, 777, "fp16")
    u = _t(rng.random(12).astype(np.float32))
    want = _ops().sample_tokens(logits, u, 0.9, 10)
    wide = torch.full((12, 1000), 9.0, dtype=torch.float16, device="cuda")
    wide[:, 100:877] = logits
    assert torch.equal(_ops().sample_tokens(wide[:, 100:877], u, 0.9, 10), want)
    assert torch.equal(_ops().sample_tokens(wide[:, 101:877], u, 0.0),
                       logits[:, 1:].float().argmax(1).int())
    t3, p3 = _ops().sample_tokens(logits.view(3, 4, 777), u.view(3, 4), torch.full((3, 4), 0.9, device="cuda").double().float(), 10,
                                  return_probs=True)
    assert t3.shape == (3, 4) and p3.shape == (3, 4, 777)
    t1 = _ops().sample_tokens(logits[5], u[5], 0.9, 10)
    assert t1.shape == () and t1.item() == want[5].item()
    assert _ops().sample_tokens(logits[:0], u[:0]).shape == (0,)
    out = torch.empty((12, 777), device="cuda")
    assert _ops().sampling_probs(logits, 0.9, 10, out=out) is out


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_sample_flat_rows(dtype):
    """Rows so flat that a rule's last element may be any of them."""
    rng = np.random.default_rng(5)
    B, V = 3, 60013
    logits = _t(5 + np.array([[0.0], [0.003], [0.05]]) * rng.standard_normal((B, V))).to(T_OF[dtype])
    for t, k, p, m in ((1.0, 0, 0.9, 0.0), (0.7, 30000, 1.0, 0.0), (1.0, 45001, 0.6, 0.97), (2.0, 0, 1.0, 0.99), (1.0, 60012, 0.999, 0.0),
                       (1.0, 0, 1e-6, 0.0), (1.0, 5000, 0.5, 0.0)):
        _check_sample(logits, rng.random(B), t, k, p, m)


def test_sample_many_rows_of_own_settings():
    rng = np.random.default_rng(6)
    B, V = 1030, 70
    some = lambda a, b: np.where(rng.random(B) < 0.3, a, b)   # noqa: E731
    _check_sample(_logits(rng, B, V, "fp32"), rng.random(B), some(0.0, rng.uniform(0.2, 2, B)), some(0, rng.integers(-1, 2 * V, B)),
                  some(1.0, rng.uniform(0, 1.1, B)), some(0.0, rng.uniform(0, 0.3, B)))


def test_sample_largest_vocabulary():
    rng = np.random.default_rng(7)
    B, V = 2, 1 << 20
    logits = _logits(rng, B, V, "fp32")
    u = rng.random(B).astype(np.float32)
    x = _n(logits)
    for t, k, p, m in ((1.0, 0, 0.9, 0.0), (0.8, 1000, 0.97, 0.0), (1.0, 0, 1.0, 0.01), (1.0, 0, 1.0, 0.0)):
        tokens, probs = _ops().sample_tokens(logits, _t(u), t, k, p, m, return_probs=True)
        for b in range(B):
            token, want = ref.sample(x[b], float(u[b]), t, k, p, m)
            assert int(tokens[b]) == token
            # the kept weights, of which the largest is 1, are summed in units of 2^-42: half a unit each, and one rounding to fp32
            d = np.abs(_n(probs[b]).astype(np.float64) - want)
            kept = int((want > 0).sum())
            assert (d <= want * (2.0 ** -24 + kept * 2.0 ** -43 + 2.0 ** -38) + 2.0 ** -149).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("top", [3, 70])   # one part a head, and several
def test_sparse_attention_of_a_query_that_is_no_number(bits, top):
    """NaN in a head's query: NaN in its output, and in no other's."""
    rng = np.random.default_rng(bits)
    L, Hq, Hkv = 1500, 8, 2
    P = (L + PAGE - 1) // PAGE
    cache = [_t(x) for x in _random_cache(rng, P, Hkv, bits)]
    q = _t(rng.standard_normal((1, Hq, D))).half()
    table, seen = _i([list(range(P))]), _i([L])
    pages = _i(np.sort([rng.permutation(P)[:top] for _ in range(Hkv)], 1)[None])
    clean = _ops().kv_sparse_attention(q, *cache, table, seen, bits, pages)
    q[0, 5, 77] = float("nan")
    got = _ops().kv_sparse_attention(q, *cache, table, seen, bits, pages)
    assert got[0, 5].isnan().all()
    others = [h for h in range(Hq) if h != 5]
    assert torch.equal(got[0, others], clean[0, others])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("top,first,last", [(50, 1, 2), (9000, 3, 4), (1, 0, 1)])
def test_choice_among_tens_of_thousands_of_pages(bits, top, first, last):
    """One sequence whose table names few pages again and again, so that thousands of equal worths lie at the border."""
    rng = np.random.default_rng(bits + top)
    L, Hq, Hkv, P = 300001, 6, 2, 300
    cache = _random_cache(rng, P, Hkv, bits)
    pages = (L + PAGE - 1) // PAGE
    edge = ref.bounds(cache[0], np.zeros((P, Hkv, 2, 16 * bits), cache[0].dtype), np.arange(P, dtype=np.int32)[None], [P * PAGE],
                      None, bits)
    q = rng.standard_normal((2, Hq, D)).astype(np.float16)
    for names in (P, 3):
        table = rng.integers(0, names, (1, pages + 5)).astype(np.int32)
        seen, row_seq = [L, L - 40000], [0, 0]
        got = _ops().kv_select_pages(_t(q), _t(edge), _t(cache[2]), _t(table), _i(seen), bits, top, first, last, row_seq=_i(row_seq))
        want = ref.select(q, edge, cache[2], table, seen, bits, top, first, last, row_seq)
        assert np.array_equal(_n(got), want)
    out = _ops().kv_sparse_attention(_t(q), *[_t(c) for c in cache], _t(table), _i(seen), bits, got, row_seq=_i(row_seq))
    _check_sparse(out, q, cache, table, seen, bits, want, row_seq=row_seq)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_sample_rows_flat_in_places(dtype):
    """Flat rows with a few peaks, with masked places, with one value in every sixteen of them, of large values."""
    rng = np.random.default_rng(8)
    V = 40007
    x = 0.03 * rng.standard_normal((6, V))
    x[0, rng.integers(0, V, 5)] += 9
    x[1, ::3] = -np.inf
    x[2, V // 2:] = torch.finfo(torch.float32).min / 2
    x[3, : V // 32 * 31] = 0.5
    x[3, V // 32 * 31 + 16:] -= rng.uniform(0, 30, V - V // 32 * 31 - 16)
    x[4] = x[4] * 1e-4 + 3000
    x[5, ::2] -= 40
    logits = _t(x).to(T_OF[dtype])
    for t, k, p, m in ((1.0, 0, 0.9, 0.0), (1.0, 100, 1.0, 0.0), (0.9, 20000, 0.7, 0.0), (3.0, 0, 1.0, 0.98), (0.02, 0, 0.99, 0.001)):
        _check_sample(logits, rng.random(6), t, k, p, m)
