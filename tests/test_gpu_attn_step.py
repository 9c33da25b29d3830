"""GPU parity of the operators around the quantized-KV attention (norms with rotation, cache writes and read-back, attention
of drafted tokens, verification of drafts) against 64-bit references in plain numpy.  The reference project has no such
kernels: parity unpinned against it.  Cache codes and scales, read-back values and verification are compared for equality;
the tolerances of the two floating results count their roundings and are derived beside their uses."""
import numpy as np
import pytest
import torch

import attn_step_ref as ref

pytestmark = pytest.mark.gpu

D, PAGE = 128, 16
T_OF = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    from trellis_serve_amd import ops
    return ops


def _t(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _half(a, dtype):
    """The values of a in a 16-bit type: the tensor, and the same values in float64."""
    t = torch.from_numpy(np.ascontiguousarray(a)).to(T_OF[dtype])
    return t.cuda(), t.double().numpy()


# ---- norms with rotation ---------------------------------------------------------------------------------------------

def _angles(max_pos, rotary):
    a = np.arange(max_pos)[:, None] * 10000.0 ** (-np.arange(0, rotary, 2) / rotary)
    return np.concatenate([np.cos(a), np.sin(a)], axis=1).astype(np.float32)


@pytest.mark.parametrize("T,Hq,Hkv,rotary,pairs,dtype,out,weights", [
    (1, 40, 8, 128, False, "bf16", "fp16", "x"), (1, 1, 1, 128, True, "fp16", "fp16", "x"),
    (7, 5, 1, 64, False, "fp16", "bf16", "fp32"), (33, 16, 1, 96, True, "bf16", "bf16", "x"),
    (130, 32, 2, 32, False, "fp16", "fp16", "fp32"), (3, 6, 3, 16, True, "fp16", "fp16", None),
    (65, 3, 2, 48, False, "bf16", "fp16", None), (19, 40, 8, 0, False, "fp16", "fp16", "x"),
    (900, 40, 8, 128, False, "bf16", "bf16", "x"), (2000, 17, 4, 112, False, "fp16", "fp16", "x")])
def test_qk_norm_rope(T, Hq, Hkv, rotary, pairs, dtype, out, weights):
    rng = np.random.default_rng(T * 131 + Hq)
    W = (Hq + 2 * Hkv) * D + 24
    x, x64 = _half(rng.standard_normal((T, W)) * rng.uniform(0.01, 30, (T, 1)), dtype)
    q, k = x[:, 8:8 + Hq * D].unflatten(1, (Hq, D)), x[:, 8 + Hq * D:8 + (Hq + Hkv) * D].unflatten(1, (Hkv, D))
    q64, k64 = x64[:, 8:8 + Hq * D].reshape(T, Hq, D), x64[:, 8 + Hq * D:8 + (Hq + Hkv) * D].reshape(T, Hkv, D)
    wq = wk = wq64 = wk64 = None
    if weights:
        w = torch.from_numpy(1 + 0.3 * rng.standard_normal((2, D))).to(torch.float32 if weights == "fp32" else T_OF[dtype])
        (wq, wk), (wq64, wk64) = w.cuda(), w.double().numpy()
    cs = _angles(777, rotary) if rotary else None
    pos = rng.integers(-3, 790, T)   # past both ends: clamped
    pos_t = _t(pos) if T % 2 else _t(pos.astype(np.int32))
    got = _ops().qk_norm_rope(q, k, wq, wk, None if cs is None else _t(cs), pos_t if rotary else None, 1e-5, pairs,
                              out_dtype=T_OF[out])
    for y, x_, w_ in ((got[0], q64, wq64), (got[1], k64, wk64)):
        z, size = ref.norm_rope(x_, w_, cs, pos, 1e-5, pairs)
        # fp32: the sum of squares (11 additions in turn), root, quotient, two products: within 16 roundings of each term;
        # then half a step of the output type (2^-25 where fp16 is subnormal)
        step = torch.finfo(T_OF[out]).eps / 2
        tol = size * 16 * 2.0 ** -24 * (1 + step) + np.abs(z) * step + (2.0 ** -25 if out == "fp16" else 0)
        d = np.abs(y.double().cpu().numpy() - z)
        assert y.dtype == T_OF[out] and y.is_contiguous() and (d <= tol).all(), (d / tol).max()


def test_qk_norm_rope_in_place_and_special_values():
    """Outputs that are the inputs; a head with an infinity or NaN is NaN or 0 by the formula and leaves the others alone; a
    head of zeros stays zero."""
    ops, rng = _ops(), np.random.default_rng(5)
    q, _ = _half(rng.standard_normal((5, 8, D)), "fp16")
    k, _ = _half(rng.standard_normal((5, 2, D)), "fp16")
    w = torch.ones(D, dtype=torch.float16, device="cuda")
    cs, pos = _t(_angles(100, 128)), torch.arange(5, device="cuda")
    want = ops.qk_norm_rope(q, k, w, w, cs, pos)
    a, b = q.clone(), k.clone()
    got = ops.qk_norm_rope(a, b, w, w, cs, pos, out=(a, b))
    assert got[0] is a and torch.equal(a, want[0]) and torch.equal(b, want[1])
    bad = q.clone()
    bad[1, 3, 7], bad[2, 0, 100], bad[3, 5] = float("nan"), float("inf"), 0
    y, _ = ops.qk_norm_rope(bad, k, w, w, cs, pos)
    same = torch.ones((5, 8), dtype=torch.bool, device="cuda")
    same[1, 3] = same[2, 0] = same[3, 5] = False
    assert torch.equal(y[same], want[0][same])
    assert y[1, 3].isnan().all() and y[2, 0].isnan().any() and (y[3, 5] == 0).all()


# ---- cache writes and read-back ----------------------------------------------------------------------------------------

def _random_cache(rng, P, Hkv, bits):
    """K and V codes with every value of the type, scales around those of unit values."""
    top = 127 if bits == 8 else 7
    c = [ref.pack(rng.integers(-top, top + 1, (P, Hkv, PAGE, D)), bits) for _ in range(2)]
    s = [(rng.uniform(0.5, 1.5, (P, Hkv)) * 3 / top).astype(np.float16) for _ in range(2)]
    return c[0], c[1], s[0], s[1]


def _table(rng, B, width, P):
    return rng.permutation(P)[:B * width].reshape(B, width).astype(np.int32)


def _check_append(cache, got, want_k, want_v):
    for g, w in zip(got, (want_k[0], want_v[0], want_k[1], want_v[1])):
        g = g.cpu().numpy()
        assert np.array_equal(g.view(np.uint8), w.view(np.uint8)), np.argwhere(g != w)[:5]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,new,Hkv", [([0], [1], 1), ([0, 15, 16, 31], [1, 1, 1, 1], 8), ([5], [11], 2),
                                          ([17, 3, 0, 40], [15, 64, 33, 0], 3), ([100, 1], [1, 200], 1),
                                          ([9], [7], 8), ([0], [16], 2)])
def test_kv_append_ragged(bits, dtype, lens, new, Hkv):
    """Row ranges over k and v columns of one wider row; every code, scale and untouched byte of the cache."""
    rng = np.random.default_rng(sum(lens) + 7 * sum(new) + bits)
    B, width = len(lens), max(-(-(a + n) // PAGE) for a, n in zip(lens, new)) + 1
    P = B * width + 3
    cache, table = _random_cache(rng, P, Hkv, bits), _table(rng, B, width, P)
    rows = sum(new)
    x, x64 = _half(rng.standard_normal((rows, 2 * Hkv * D + 8)) * np.exp(rng.normal(0, 1, (rows, 1))), dtype)
    k, v = x[:, :Hkv * D].unflatten(1, (Hkv, D)), x[:, Hkv * D:2 * Hkv * D].unflatten(1, (Hkv, D))
    start = np.concatenate([[0], np.cumsum(new)])
    got = [_t(c) for c in cache]
    for max_new in (max(new), None):   # the second call finds its own pages and leaves them as they are
        _ops().kv_append(k, v, *got, _t(table), _t(np.int32(lens)), bits, row_start=_t(start.astype(np.int32)),
                         max_new=max_new)
        rows_of = [list(range(start[b], start[b + 1])) for b in range(B)]
        wk = ref.append(x64[:, :Hkv * D].reshape(rows, Hkv, D), cache[0], cache[2], table, lens, bits, rows_of)
        wv = ref.append(x64[:, Hkv * D:2 * Hkv * D].reshape(rows, Hkv, D), cache[1], cache[3], table, lens, bits, rows_of)
        _check_append(cache, got, wk, wv)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("B,most,Hkv", [(1, 90, 2), (64, 20, 1), (65, 40, 2), (200, 33, 1), (4500, 3, 1)])
def test_kv_append_many_sequences_without_a_bound(bits, B, most, Hkv):
    """Ragged rows, empty sequences among them, and no bound on a sequence's new tokens."""
    rng = np.random.default_rng(B + bits)
    lens, new = rng.integers(0, 40, B), rng.integers(0, most + 1, B) * rng.integers(0, 2, B)
    new[B // 2] = most
    width = int(max(-(-(a + n) // PAGE) for a, n in zip(lens, new))) + 4   # room: places go by rows
    cache, table = _random_cache(rng, B * width + 1, Hkv, bits), _table(rng, B, width, B * width + 1)
    rows = int(new.sum())
    x, x64 = _half(rng.standard_normal((rows, 2 * Hkv * D)), "fp16")
    k, v = x[:, :Hkv * D].unflatten(1, (Hkv, D)), x[:, Hkv * D:].unflatten(1, (Hkv, D))
    start = np.concatenate([[0], np.cumsum(new)])
    got = [_t(c) for c in cache]
    _ops().kv_append(k, v, *got, _t(table), _t(np.int32(lens)), bits, row_start=_t(start.astype(np.int32)))
    rows_of = [list(range(start[b], start[b + 1])) for b in range(B)]
    wk = ref.append(x64[:, :Hkv * D].reshape(rows, Hkv, D), cache[0], cache[2], table, list(lens), bits, rows_of)
    wv = ref.append(x64[:, Hkv * D:].reshape(rows, Hkv, D), cache[1], cache[3], table, list(lens), bits, rows_of)
    _check_append(cache, got, wk, wv)


@pytest.mark.parametrize("bits", [8, 4])
def test_kv_append_to_a_page_of_infinite_scale(bits):
    """The page keeps its scale, and every finite value over it is 0."""
    rng = np.random.default_rng(bits)
    cache, table = _random_cache(rng, 3, 2, bits), np.int32([[1]])
    cache[2][1], cache[3][1] = np.inf, np.inf
    x, x64 = _half(rng.standard_normal((5, 2, D)), "fp16")
    got = [_t(c) for c in cache]
    _ops().kv_append(x, x, *got, _t(table), _t(np.int32([7])), bits, row_start=_t(np.int32([0, 5])))
    assert np.array_equal(got[2].cpu().numpy(), cache[2]) and np.array_equal(got[3].cpu().numpy(), cache[3])
    for g, c in zip(got[:2], cache[:2]):
        want = c.copy()
        want[1, :, 7:12] = 0
        assert np.array_equal(g.cpu().numpy(), want)


@pytest.mark.parametrize("bits", [8, 4])
def test_kv_append_selected_rows(bits):
    """Accepted nodes of a draft tree: counts, -1 padding, a node named twice, nodes outside the sequence's rows."""
    rng = np.random.default_rng(bits)
    B, N, Hkv, width = 4, 6, 2, 4
    P = B * width
    cache, table = _random_cache(rng, P, Hkv, bits), _table(rng, B, width, P)
    k, k64 = _half(rng.standard_normal((B, N, Hkv, D)), "fp16")
    v, v64 = _half(rng.standard_normal((B, N, Hkv, D)), "fp16")
    lens = [14, 0, 33, 63]   # the last has one slot left in its table
    select = np.array([[0, 2, 5, -1, -1, -1], [0, 0, 3, 1, -1, 4], [0, 9, -5, 2, 1, 1], [0, 1, 2, -1, -1, -1]], np.int32)
    counts = np.array([3, 4, 5, 3], np.int32)
    got = [_t(c) for c in cache]
    _ops().kv_append(k, v, *got, _t(table), _t(np.int32(lens)), bits, select=_t(select), counts=_t(counts))
    rows_of = [[b * N + s if 0 <= s < N else -1 for s in select[b, :counts[b]]] for b in range(B)]
    wk = ref.append(k64.reshape(-1, Hkv, D), cache[0], cache[2], table, lens, bits, rows_of)
    wv = ref.append(v64.reshape(-1, Hkv, D), cache[1], cache[3], table, lens, bits, rows_of)
    _check_append(cache, got, wk, wv)


@pytest.mark.parametrize("bits", [8, 4])
def test_kv_append_special_values_and_bad_pages(bits):
    """Infinities, NaN, zeros, subnormal and largest values; page ids outside the cache are not written, nor is anything
    past the table; counts below 0 and past the rows."""
    rng = np.random.default_rng(40 + bits)
    B, n, Hkv, width, P = 7, 5, 2, 2, 14
    cache, table = _random_cache(rng, P, Hkv, bits), _table(rng, B, width, P)
    x = rng.standard_normal((2, B, n, Hkv, D)).astype(np.float32)
    x[:, 0, 1, :, 3], x[:, 0, 2, 0, 9], x[:, 0, 3, 1, 11] = np.inf, np.nan, -np.inf
    x[:, 1] = 0
    x[:, 2] *= 1e-7
    x[:, 3] *= 3e4
    x[:, 4] *= 1e36   # bf16 only: past the scale's range, the codes saturate
    table[5, 0], table[6, 1] = -1, P
    lens = [0, 16, 3, 12, 0, 13, 30]
    (k, k64), (v, v64) = _half(x[0], "bf16"), _half(x[1], "bf16")
    got = [_t(c) for c in cache]
    counts = np.array([5, 5, 99, 5, 5, 5, -1], np.int32)
    _ops().kv_append(k, v, *got, _t(table), _t(np.int32(lens)), bits, counts=_t(counts))
    rows_of = [list(range(b * n, b * n + min(max(counts[b], 0), n))) for b in range(B)]
    wk = ref.append(k64.reshape(-1, Hkv, D), cache[0], cache[2], table, lens, bits, rows_of)
    wv = ref.append(v64.reshape(-1, Hkv, D), cache[1], cache[3], table, lens, bits, rows_of)
    _check_append(cache, got, wk, wv)


@pytest.mark.parametrize("bits", [8, 4])
def test_kv_append_token_by_token_stays_within_its_steps(bits):
    """A page filled one token at a time, each louder than the last: a value is off by half a step when it is written and by
    half a step of each later scale."""
    rng = np.random.default_rng(3)
    cache = [_t(c) for c in _random_cache(rng, 2, 1, bits)]
    table = _t(np.array([[1, 0]], np.int32))
    x = rng.standard_normal((PAGE, 1, 1, D)) * 1.3 ** np.arange(PAGE)[:, None, None, None]
    k, k64 = _half(x, "fp16")
    bound = np.zeros(PAGE)
    last = 0.0
    for t in range(PAGE):
        _ops().kv_append(k[t], k[t], *cache, table, _t(np.int32([t])), bits)
        s = float(cache[2][1, 0])
        assert s >= last
        bound[:t] += s / 2 * (s > last)
        bound[t] = s / 2
        last = s
    back = ref.values(cache[0].cpu().numpy(), cache[2].cpu().numpy(), np.array([1]), PAGE, bits)
    assert (np.abs(back - k64[:, 0]).max(axis=(1, 2)) <= bound * (1 + 1e-12)).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,starts,Hkv", [([1], None, 1), ([16, 0, 5], None, 8), ([70, 33, 16], [64, 0, 16], 3),
                                             ([2100, 1], [7, 0], 8), ([9000], None, 1)])
def test_kv_gather(bits, dtype, lens, starts, Hkv):
    rng = np.random.default_rng(sum(lens) + bits)
    B, width = len(lens), max(1, max(-(-n // PAGE) for n in lens))
    P = B * width + 1
    cache, table = _random_cache(rng, P, Hkv, bits), _table(rng, B, width, P)
    first = starts or [0] * B
    counts = [n - f for n, f in zip(lens, first)]
    start = np.concatenate([[2], 2 + np.cumsum(counts)])   # two rows before and three behind belong to nobody
    rows = int(start[-1]) + 3
    out = tuple(torch.full((rows, Hkv, D), 77.0, dtype=T_OF[dtype], device="cuda") for _ in range(2))
    _ops().kv_gather(*[_t(c) for c in cache], _t(table), _t(np.int32(lens)), bits, _t(start.astype(np.int32)), rows,
                     starts=None if starts is None else _t(np.int32(starts)), out=out)
    for o, codes, scales in ((out[0], cache[0], cache[2]), (out[1], cache[1], cache[3])):
        want = np.full((rows, Hkv, D), 77.0)
        for b in range(B):
            want[start[b]:start[b + 1]] = ref.values(codes, scales, table[b], lens[b], bits)[first[b]:]
        # code * scale has 18 bits: exact in fp32, so one rounding to the output type
        assert torch.equal(o.cpu(), torch.from_numpy(want).to(T_OF[dtype]))


def test_kv_gather_odd_tables():
    """Page ids outside the cache are clamped; rows past a sequence's tokens, tokens past the table and negative starts are
    left alone."""
    rng = np.random.default_rng(9)
    cache = _random_cache(rng, 3, 2, 8)
    table = np.array([[-7, 2], [99, 1], [0, 0]], np.int32)
    out = tuple(torch.full((60, 2, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    lens, starts, start = [20, 40, 5], [0, 0, -3], [0, 25, 60, 60]
    _ops().kv_gather(*[_t(c) for c in cache], _t(table), _t(np.int32(lens)), 8, _t(np.int32(start)), 60,
                     starts=_t(np.int32(starts)), out=out)
    want = np.full((60, 2, D), 7.0)
    want[:20] = ref.values(cache[0], cache[2], table[0], 20, 8)
    want[25:57] = ref.values(cache[0], cache[2], table[1], 32, 8)
    assert torch.equal(out[0].cpu(), torch.from_numpy(want).half())


# ---- attention of drafted tokens ---------------------------------------------------------------------------------------

def _seen(rng, B, N, how):
    if how == "chain":
        return np.tril(np.ones((B, N, N), bool))
    seen = np.zeros((B, N, N), bool)
    for b in range(B):
        for i in range(N):
            if i and how == "tree":
                seen[b, i] = seen[b, rng.integers(max(0, i - 5), i)]
            seen[b, i, i] = True
        if how == "random":
            seen[b] = rng.random((N, N)) < 0.3
            seen[b, N // 2] = False   # a node that sees no node at all
    return seen


def _masks(seen):
    B, N, _ = seen.shape
    bits = np.zeros((B, N), np.uint64)
    for j in range(N):
        bits |= seen[:, :, j].astype(np.uint64) << np.uint64(j)
    return bits.view(np.int64)


def _tree_case(seed, lens, N, Hq, Hkv, bits, how, spare=1, scale=1.0):
    rng = np.random.default_rng(seed)
    B, width = len(lens), max(1, max(-(-n // PAGE) for n in lens)) + spare
    P = B * width + 2
    cache, table = _random_cache(rng, P, Hkv, bits), _table(rng, B, width, P)
    for b, n in enumerate(lens):   # nothing past a sequence's pages is read
        for p in table[b, -(-n // PAGE):]:
            cache[2][p] = cache[3][p] = np.nan
        table[b, -(-n // PAGE):] = -1
    x, _ = _half(rng.standard_normal((B, N, (Hq + 2 * Hkv) * D)) * scale, "fp16")
    q, k, v = torch.split(x, [Hq * D, Hkv * D, Hkv * D], dim=2)
    return (q.unflatten(2, (Hq, D)), k.unflatten(2, (Hkv, D)), v.unflatten(2, (Hkv, D)), _seen(rng, B, N, how), cache,
            table)


def _check_tree(got, q, k, v, seen, cache, table, lens, bits, sm=D ** -0.5, nodes=None, live=None):
    n = lambda t: t.float().cpu().numpy()   # noqa: E731
    out, mean, slip = ref.tree_attention(n(q), n(k), n(v), seen, cache, table, lens, bits, sm)
    top = 127 if bits == 8 else 7
    vmax = max(float(np.abs(n(v)).max()), float(np.nanmax(cache[3].astype(np.float32))) * top)
    keys = max(lens) + q.shape[1]
    tol = ref.tree_tolerance(out, mean, slip, keys, vmax)
    d = np.abs(got.double().cpu().numpy() - out)
    if nodes is not None:
        live = torch.arange(q.shape[1])[None, :] < torch.tensor(nodes)[:, None]
    if live is not None:
        d, tol = d[live.cpu().numpy()], tol[live.cpu().numpy()]
    assert (d <= tol).all(), ((d / tol).max(), d.max())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens,N,Hq,Hkv,how", [
    ([0], 1, 1, 1, "chain"), ([1], 1, 5, 1, "chain"), ([16], 2, 8, 8, "tree"), ([127, 0, 129], 5, 40, 8, "tree"),
    ([17, 300], 16, 8, 2, "tree"), ([128, 1000], 17, 4, 1, "random"), ([33], 33, 5, 1, "chain"),
    ([700, 15, 64], 16, 10, 2, "chain"), ([250], 64, 1, 1, "random"), ([31, 513], 64, 16, 1, "tree"),
    ([40] * 70, 3, 2, 1, "tree"), ([2049, 5], 24, 16, 4, "tree"), ([90, 2], 20, 12, 2, "random")])
def test_kv_tree_attention(bits, lens, N, Hq, Hkv, how):
    q, k, v, seen, cache, table = _tree_case(N * 7 + bits + len(lens), lens, N, Hq, Hkv, bits, how)
    mask = None if how == "chain" else _t(_masks(seen))
    got = _ops().kv_tree_attention(q, k, v, mask, *[_t(c) for c in cache], _t(table), _t(np.int32(lens)), bits)
    assert got.shape == q.shape and got.is_contiguous()
    _check_tree(got, q, k, v, seen, cache, table, lens, bits)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens,copies,N,Hq", [
    ([9001, 1, 8300], 300, 3, 2), ([9001, 130, 8192], 160, 6, 6), ([8999, 0, 9000], 110, 16, 6),
    ([1601, 17, 1024], 200, 25, 4), ([2100, 1025, 0], 120, 32, 8), ([1500, 33, 1111], 150, 64, 5),
    ([1300, 64, 5], 120, 64, 8)])
def test_kv_tree_attention_long_runs(bits, lens, copies, N, Hq):
    """Many sequences over the same pages: each workgroup goes through thousands of tokens of several of them."""
    q, k, v, seen, cache, table = _tree_case(copies + bits, lens, N, Hq, 1, bits, "tree")
    many = torch.arange(len(lens) * copies) % len(lens)
    got = _ops().kv_tree_attention(*(t[many.to(t.device)].contiguous() for t in (q, k, v, _t(_masks(seen)))),
                                   *[_t(c) for c in cache], _t(table)[many.to(q.device)].contiguous(),
                                   _t(np.int32(lens))[many.to(q.device)].contiguous(), bits)
    assert not torch.isnan(got).any()
    got = got.unflatten(0, (copies, len(lens)))
    lo, hi = got.float().amin(0), got.float().amax(0)
    for end in (lo, hi):   # the smallest and largest of a value's copies are within its tolerance, so all are
        _check_tree(end, q, k, v, seen, cache, table, lens, bits)


@pytest.mark.parametrize("lens,N,Hq,Hkv", [([64, 0, 500, 7, 90], 16, 10, 2), ([30, 200, 0], 64, 5, 1), ([100, 100], 1, 4, 4)])
def test_kv_tree_attention_ragged_nodes(lens, N, Hq, Hkv):
    """num_nodes 0, 1, .. N: the rest of a sequence is neither written nor read (its K and V hold NaN)."""
    q, k, v, seen, cache, table = _tree_case(N, lens, N, Hq, Hkv, 8, "tree")
    nodes = [min(N, [N, 0, 1, N // 2 + 1, 2][b]) for b in range(len(lens))]
    k2, v2 = k.clone(), v.clone()
    for b, n in enumerate(nodes):
        k2[b, n:] = float("nan")
        v2[b, n:] = float("nan")
        seen[b, :, n:] = False
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    got = _ops().kv_tree_attention(q.contiguous(), k2, v2, _t(_masks(np.ones_like(seen)) if N == 1 else _masks(seen)),
                                   *[_t(c) for c in cache], _t(table), _t(np.int32(lens)), 8,
                                   num_nodes=_t(np.int32(nodes)), out=out)
    _check_tree(got, q, k, v, seen, cache, table, lens, 8, nodes=nodes)
    for b, n in enumerate(nodes):
        assert (got[b, n:] == 7.0).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_kv_tree_attention_empty_rows_and_odd_nodes(bits):
    """No cached token: a node that sees nothing gives zeros.  Infinities and NaN in a node's K and V reach the nodes that
    see it, and no other."""
    ops = _ops()
    lens, N, Hq, Hkv = [0, 37], 20, 10, 2
    q, k, v, seen, cache, table = _tree_case(77, lens, N, Hq, Hkv, bits, "tree")
    seen[0, 4] = False
    k, v = k.clone(), v.clone()
    clean = v.clone()
    v[0, 17, :, 5], v[1, 3, 0, 100], v[1, 18, 1, 0] = float("nan"), float("inf"), float("-inf")
    k[1, 19] = float("nan")
    clean[0, 17, :, 5], clean[1, 3, 0, 100], clean[1, 18, 1, 0] = 0, 0, 0
    args = [_t(_masks(seen)), *[_t(c) for c in cache], _t(table), _t(np.int32(lens)), bits]
    got = ops.kv_tree_attention(q, k, v, *args)
    assert (got[0, 4] == 0).all()
    G = Hq // Hkv
    for b, j, h, d in ((0, 17, 0, 5), (0, 17, 1, 5), (1, 3, 0, 100), (1, 18, 1, 0)):
        sees = torch.from_numpy(seen[b, :, j]).cuda()
        part = got[b, :, h * G:(h + 1) * G, d]
        assert sees.any() and not part[sees].isfinite().any() and part[~sees].isfinite().all()
    dirty = ~got.isfinite()
    assert got[1, 19].isnan().all()   # its own key: NaN logits
    assert dirty[0].sum() == 2 * G * seen[0, :, 17].sum()
    # elsewhere the values are those of finite nodes, within the operator's bound: such a node's products are taken in fp32,
    # outside the matrix instruction, so neither its probabilities' rounding nor the order of the sums is the same bits
    k0 = torch.where(k.isnan(), 0, k)
    _check_tree(torch.where(dirty, torch.nan, got), q, k0, clean, seen, cache, table, lens, bits, live=~dirty)


def test_kv_tree_attention_scales():
    """Value scales over the fp16 range within one sequence, zero and negative ones, and sharp softmaxes."""
    for bits in (8, 4):
        lens, N, Hq, Hkv = [333, 64], 9, 4, 2
        q, k, v, seen, cache, table = _tree_case(5 + bits, lens, N, Hq, Hkv, bits, "tree", scale=3.0)
        rng = np.random.default_rng(1)
        live = np.isfinite(cache[3])
        cache[3][live] = (10.0 ** rng.uniform(-6, 2, live.sum())).astype(np.float16)
        pages = table[0, :21]
        cache[3][pages[3]], cache[3][pages[5], 0], cache[2][pages[7]] = 0, -0.5, 0
        got = _ops().kv_tree_attention(q, k, v, _t(_masks(seen)), *[_t(c) for c in cache], _t(table), _t(np.int32(lens)),
                                       bits)
        _check_tree(got, q, k, v, seen, cache, table, lens, bits)


def test_kv_tree_attention_equals_decode_attention_on_one_node():
    """One node without keys of its own (an empty mask) is the framework's decode attention: both within the bound."""
    ops = _ops()
    lens = [1, 500, 2000, 16]
    q, k, v, seen, cache, table = _tree_case(8, lens, 1, 40, 8, 8, "tree")
    seen[:] = False
    c = [_t(x) for x in cache]
    got = ops.kv_tree_attention(q, k, v, _t(_masks(seen)), *c, _t(table), _t(np.int32(lens)), 8)
    _check_tree(got, q, k, v, seen, cache, table, lens, 8)
    dec = ops.kv_decode_attention(q[:, 0].contiguous(), *c, _t(table), _t(np.int32(lens)), 8)
    _check_tree(dec[:, None], q, k, v, seen, cache, table, lens, 8)


@pytest.mark.parametrize("bits", [8, 4])
def test_kv_tree_attention_is_deterministic(bits):
    lens, N, Hq, Hkv = [3000, 100, 1500], 16, 20, 4
    q, k, v, seen, cache, table = _tree_case(2, lens, N, Hq, Hkv, bits, "tree")
    args = [q, k, v, _t(_masks(seen)), *[_t(c) for c in cache], _t(table), _t(np.int32(lens)), bits]
    want = _ops().kv_tree_attention(*args)
    for _ in range(3):
        ws = torch.full((_ops().kv_tree_workspace_bytes(3, N, Hq, Hkv, table.shape[1]),), 255, dtype=torch.uint8,
                        device="cuda")
        assert torch.equal(_ops().kv_tree_attention(*args, workspace=ws), want)


@pytest.mark.parametrize("N", [3, 9, 40])
def test_pages_past_four_gigabytes(N):
    """The same pages at the end of a cache of more than 2^32 bytes give the same codes, values and attention."""
    rng = np.random.default_rng(N)
    lens, Hq, Hkv, far = [300, 5, 77], 24, 8, 270000
    q, k, v, seen, cache, table = _tree_case(N, lens, N, Hq, Hkv, 8, "tree", spare=4)
    table[:] = rng.permutation(len(cache[0]))[: table.size].reshape(table.shape)
    for c in cache[2:]:
        c[:] = np.abs(rng.normal(0, 0.02, c.shape)).astype(np.float16)
    near = [_t(c) for c in cache]
    P, first = len(cache[0]), far - len(cache[0])
    wide = [torch.empty((far, *c.shape[1:]), dtype=c.dtype, device="cuda") for c in near]
    for w, c in zip(wide, near):
        w[first:] = c
    start, lt, results = _t(np.cumsum([0] + [n + N for n in lens]).astype(np.int32)), _t(np.int32(lens)), []
    for caches, t in ((near, _t(table)), (wide, _t(table + np.int32(first)))):
        out = _ops().kv_tree_attention(q, k, v, _t(_masks(seen)), *caches, t, lt, 8)
        _ops().kv_append(k, v, *caches, t, lt, 8)
        back = _ops().kv_gather(*caches, t, lt + N, 8, start, int(sum(lens)) + 3 * N)
        results.append([out, *back, *(c[-P:] for c in caches)])
    for x, y in zip(*results):
        assert torch.equal(x, y)


# ---- verification --------------------------------------------------------------------------------------------------------

def _probs(rng, *shape, sharp=2.0):
    x = np.exp(rng.normal(0, sharp, shape))
    return (x / x.sum(-1, keepdims=True)).astype(np.float32)


def _check_verify(p, q, tokens, parents, u, nodes=None, wide=False):
    i = torch.int64 if wide else torch.int32
    got = _ops().verify_drafts(_t(p), _t(tokens, i), _t(u), parents=None if parents is None else _t(parents, i),
                               draft_probs=None if q is None else _t(q), num_nodes=None if nodes is None else _t(nodes))
    want = ref.verify(p, q, tokens, parents, u, nodes)
    for g, w in zip(got, want):
        assert g.dtype == torch.int32 and np.array_equal(g.cpu().numpy(), w), (g, w)
    return want


@pytest.mark.parametrize("B,N,V", [(1, 1, 1), (3, 2, 2), (5, 6, 1001), (2, 64, 4097), (17, 8, 32003), (1, 5, 200001),
                                   (300, 4, 37)])
def test_verify_chain_with_draft_probabilities(B, N, V):
    rng = np.random.default_rng(B * N + V)
    p, q = _probs(rng, B, N, V), _probs(rng, B, N, V)
    q = ((p + 0.3 * q) / 1.3).astype(np.float32)   # near the target: some are accepted
    tokens = np.zeros((B, N), np.int64)
    for b in range(B):
        for i in range(1, N):
            tokens[b, i] = min(V - 1, np.searchsorted(np.cumsum(q[b, i - 1]), rng.random()))
    u = rng.random((B, N), dtype=np.float32)
    nodes = rng.integers(0, N + 1, B).astype(np.int32) if B > 2 else None
    want = _check_verify(p, q, tokens, None, u, nodes, wide=V % 2 == 0)
    if B == 17:
        assert want[1].max() > 2 and (want[1] < N).any()


@pytest.mark.parametrize("B,N,V", [(1, 1, 3), (2, 9, 5), (4, 64, 1000), (16, 16, 32003), (3, 33, 131072), (70, 7, 4096)])
@pytest.mark.parametrize("how", ["tree", "chain"])
def test_verify_candidates(B, N, V, how):
    rng = np.random.default_rng(B * N + V + len(how))
    p = _probs(rng, B, N, V)
    parents = np.full((B, N), -1)
    tokens = np.zeros((B, N), np.int64)
    for b in range(B):
        seen = {}
        for i in range(1, N):
            up = parents[b, i] = int(rng.integers(max(0, i - 6), i)) if how == "tree" else i - 1
            rank = seen[up] = seen.get(up, -1) + 1   # the fourth brother repeats the first one's token
            tokens[b, i] = np.argsort(-p[b, up])[rank % 3 if rng.random() < 0.9 else rng.integers(0, V)]
    u = rng.random((B, N), dtype=np.float32)
    _check_verify(p, None, tokens, None if how == "chain" else parents, u, wide=N % 2 == 0)
    if B > 1:
        _check_verify(p, None, tokens, None if how == "chain" else parents, u, rng.integers(0, N + 1, B).astype(np.int32))


@pytest.mark.parametrize("B,N,V", [(64, 3, 70001), (1, 2, 5000011), (2, 2, 67 * 65536 + 1)])
def test_verify_large_vocabularies(B, N, V):
    """Two parts a wave; more parts than a wave scans at once."""
    rng = np.random.default_rng(V)
    p = rng.random((B, N, V), dtype=np.float32)
    p /= p.sum(-1, keepdims=True, dtype=np.float64).astype(np.float32)
    tokens = rng.integers(0, V, (B, N))
    u = rng.random((B, N), dtype=np.float32)
    _check_verify(p, None, tokens, None, u)
    p[:, :, : V - 3] = 0   # all weight at the end of the last part
    _check_verify(p, None, tokens, None, u)


def test_verify_odd_inputs():
    """Tokens and parents out of range, probabilities of 0, infinity and NaN, numbers at the ends of [0, 1), rows without
    mass, a residual without mass."""
    rng = np.random.default_rng(0)
    B, N, V = 10, 5, 300
    p = _probs(rng, B, N, V)
    tokens = rng.integers(0, V, (B, N))
    parents = np.tile(np.array([-1, 0, 0, 1, 2]), (B, 1))
    u = rng.random((B, N), dtype=np.float32)
    tokens[0, 1], tokens[0, 2] = -1, V
    parents[1] = [-1, 1, -5, 99, 3]
    p[2, 0, :50], p[2, 0, 60], p[2, 0, 61] = np.nan, np.inf, -1
    tokens[2, 1:3] = 3, 61
    p[3, 0] = 0
    u[4], u[5] = 0, np.float32(1) - np.float32(2 ** -24)
    u[6, 0], u[7, 0], u[8, 0] = 1.0, np.nan, -0.5
    p[9, 0] = 0
    p[9, 0, 7] = 1
    tokens[9, 1:3] = 7, 7
    u[9, 1] = 1.0   # refused although certain: nothing is left, the next token comes from the row itself
    _check_verify(p, None, tokens, parents, np.where(np.isnan(u), 0, u).astype(np.float32))
    _check_verify(p, p.copy(), tokens, None, np.where(np.isnan(u), 0, u).astype(np.float32))
    got = _ops().verify_drafts(_t(p), _t(tokens), _t(u), parents=_t(parents))
    assert int(got[1].min()) >= 1


def test_verify_drafts_of_infinite_probability_are_refused():
    rng = np.random.default_rng(5)
    p = _probs(rng, 3, 4, 70)
    tokens, u = rng.integers(0, 70, (3, 4)), rng.random((3, 4), dtype=np.float32)
    for b in range(3):
        p[b, 0, tokens[b, 1]] = (np.inf, np.nan, -np.inf)[b]
    for q in (None, _probs(rng, 3, 4, 70)):
        got = _check_verify(p, q, tokens, None, u)
        assert (got[1] == 1).all()


def test_verify_in_a_given_workspace():
    rng = np.random.default_rng(6)
    B, N, V = 5, 3, 3001
    args = _t(_probs(rng, B, N, V)), _t(rng.integers(0, V, (B, N))), _t(rng.random((B, N), dtype=np.float32))
    ws = torch.full((_ops().verify_workspace_bytes(B, V),), 255, dtype=torch.uint8, device="cuda")
    want = _ops().verify_drafts(*args)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(_ops().verify_drafts(*args, workspace=ws), want))


def test_verify_emits_the_targets_distribution():
    """The tokens after the root, over many uniform numbers, are distributed as the target's row 0: a chain with sampled drafts
    and a tree of fixed candidates.  8192 sequences over 8 tokens: the expected squared distance of the counts is below 1
    per sequence (sum p (1 - p)); 6 times that has a probability far below 1e-6."""
    rng = np.random.default_rng(11)
    B, N, V = 8192, 4, 8
    p, q = np.repeat(_probs(rng, 1, N, V), B, 0), np.repeat(_probs(rng, 1, N, V), B, 0)
    u = rng.random((B, N), dtype=np.float32)
    tokens = np.zeros((B, N), np.int64)
    tokens[:, 1:] = [[np.searchsorted(np.cumsum(q[0, i]), rng.random() * 0.999999) for i in range(N - 1)] for _ in range(B)]
    _, _, out = _ops().verify_drafts(_t(p), _t(tokens), _t(u), draft_probs=_t(q))
    tree = np.tile(np.array([0, 2, 5, 2]), (B, 1))
    _, _, out2 = _ops().verify_drafts(_t(p), _t(tree), _t(u), parents=_t(np.tile(np.array([-1, 0, 0, 0]), (B, 1))))
    for o in (out, out2):
        counts = np.bincount(o[:, 0].cpu().numpy(), minlength=V)
        assert ((counts - B * p[0, 0].astype(np.float64)) ** 2).sum() < 6 * B
