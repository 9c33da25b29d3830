"""The operators around the attention and at the ends of a serving step at batches of every size: workspaces made for the largest,
and sampling in the chunks that large batches have."""
import numpy as np
import pytest
import torch

import serving_step_ref as ref
from test_gpu_serving_step import T_OF, _check_sparse, _i, _logits, _n, _ops, _rows_case, _t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
def test_sparse_attention_with_one_workspace_for_all_batches(bits):
    most, top, Hq, Hkv = 130, 40, 16, 8
    rng = np.random.default_rng(bits)
    lens = rng.integers(1, 900, most).tolist()
    rng, cache, table, edge, q = _rows_case(bits, lens, Hq, Hkv, bits)
    c = [_t(x) for x in cache]
    ops = _ops()
    ws = torch.empty(ops.kv_sparse_workspace_bytes(most, Hq, Hkv, top), dtype=torch.uint8, device="cuda")
    choice_ws = torch.empty(ops.kv_select_workspace_bytes(most, Hkv, table.shape[1]), dtype=torch.uint8, device="cuda")
    for rows in (1, 2, 3, 18, 19, 64, 126, 127, 128, 130):
        args = _t(table[:rows]), _i(lens[:rows]), bits
        pages = ops.kv_select_pages(_t(q[:rows]), _t(edge), c[2], *args, top, workspace=choice_ws)
        got = ops.kv_sparse_attention(_t(q[:rows]), *c, *args, pages, workspace=ws)
        assert torch.equal(got, ops.kv_sparse_attention(_t(q[:rows]), *c, *args, pages))
        _check_sparse(got, q[:rows], cache, table[:rows], lens[:rows], bits, _n(pages))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("Hq,Hkv,top", [(5, 1, 3), (8, 1, 40), (9, 1, 40), (32, 2, 64), (40, 8, 17)])
def test_sparse_attention_keeps_probabilities_past_sixteen_bits(bits, Hq, Hkv, top):
    """Queries of zeros: every key has the same probability, so outputs are means of values of every scale.  A product loses 2^-21,
    fp32 sums some 64 roundings (a wave's pages, the waves, the parts) of 2^-24 of the mean |v|, and the output half a step of fp16
    (2^-25 where it is subnormal); the same probabilities rounded to fp16 would be up to another half a step off."""
    lens = [16 * top, 16 * top - 7, 900, 33, 1]
    rng, cache, table, edge, q = _rows_case(top + bits, lens, Hq, Hkv, bits)
    cache[3] = (rng.uniform(1, 2, cache[3].shape) * 2.0 ** rng.integers(-6, 3, (cache[3].shape[0], 1))).astype(np.float16)
    q[:] = 0
    pages = np.full((len(lens), Hkv, top), -1, np.int32)
    for r, n in enumerate(lens):
        for h in range(Hkv):
            take = rng.permutation(-(-n // 16))[:top]
            pages[r, h, :len(take)] = np.sort(take)
    got = _ops().kv_sparse_attention(_t(q), *[_t(x) for x in cache], _t(table), _i(lens), bits, _t(pages))
    out, mean, _ = ref.sparse_attention(q, cache, table, lens, bits, pages, 128 ** -0.5)
    d = np.abs(got.double().cpu().numpy() - out)
    tol = np.maximum(np.abs(out) * 2.0 ** -11, 2.0 ** -25) + mean * (2.0 ** -21 + 64 * 2.0 ** -24)
    assert (d <= tol).all(), ((d / tol).max(), (d > tol).mean())


# ---- sampling of more than 2^19 logits in all, which are worked on in chunks of 8192 -------------------------------------

def _check_large(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    """Settings: numbers, or arrays of one a row."""
    B, V = logits.shape
    assert B * V > 1 << 19
    kinds = (np.float32, np.int32, np.float32, np.float32)
    typed = [x.astype(d) if isinstance(x, np.ndarray) else x for x, d in zip((t, k, p, m), kinds)]
    settings = [_t(x) if isinstance(x, np.ndarray) else x for x in typed]
    u = u.astype(np.float32)
    tokens, probs = _ops().sample_tokens(logits, _t(u), *settings, return_probs=True)
    assert torch.equal(_ops().sample_tokens(logits, _t(u), *settings), tokens)
    assert torch.equal(_ops().sampling_probs(logits, *settings), probs)
    x, got, tokens = logits.double().cpu().numpy(), _n(probs), _n(tokens)
    unit = 2.0 ** -(62 - (V - 1).bit_length())   # of a row's sums: V weights of at most 1 stay within 2^62 of them
    for b in range(B):
        mine = [s[b].item() if isinstance(s, np.ndarray) else s for s in typed]
        token, want = ref.sample(x[b], float(u[b]), *mine)
        assert tokens[b] == token, (b, mine, tokens[b], token)
        # the largest weight is 1: the sum of the kept is off by half a unit each; a weight's exponent, of up to 2^8, by some 2^-53 of
        # itself on either side; one rounding to fp32
        kept = int((want > 0).sum())
        d = np.abs(got[b].astype(np.float64) - want)
        assert (d <= want * (2.0 ** -24 + kept * unit / 2 + 2.0 ** -42) + 2.0 ** -149).all(), (b, mine)
        assert ((got[b] > 0) <= (want > 0)).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,V", [(6, 100353), (20, 32003), (70, 8191), (65, 8192), (9, 65537)])
def test_sample_in_large_chunks(dtype, B, V):
    """Several chunks, of which the last ends anywhere; settings for all rows and for each, fewer than 256 first ones and more."""
    rng = np.random.default_rng(B)
    logits, u = _logits(rng, B, V, dtype), rng.random(B)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.8, 0, 0.95, 0.0), (1.0, 40, 1.0, 0.0), (1.0, 256, 0.9, 0.0), (1.2, 257, 0.97, 0.01),
                       (1.0, 3000, 1.0, 0.0), (0.9, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (3.0, V - 1, 0.5, 0.0)):
        _check_large(logits, u, t, k, p, m)
    some = lambda a, b: np.where(rng.random(B) < 0.3, a, b)   # noqa: E731
    for _ in range(2):
        _check_large(logits, u, some(0.0, rng.uniform(0.2, 2, B)), some(0, rng.integers(-1, 600, B)),
                     some(1.0, rng.uniform(0, 1.1, B)), some(0.0, rng.uniform(0, 0.3, B)))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_sample_flat_and_masked_rows_in_large_chunks(dtype):
    """Flat rows, rows of one value, rows whose masks leave whole chunks empty, or all but one element, or nothing."""
    rng = np.random.default_rng(11)
    B, V = 12, 50003
    x = rng.standard_normal((B, V)) * np.array([0.0, 1e-3, 0.02, 0.1, 0.4, 1.0, 1.5, 2.0, 2.0, 2.0, 2.0, 2.0])[:, None]
    x[7, :20000], x[8, 9000:], x[9], x[9, 49999], x[10], x[11, ::2] = -np.inf, -np.inf, -np.inf, 3.0, np.nan, np.nan
    logits, u = _t(x).to(T_OF[dtype]), rng.random(B)
    for t, k, p, m in ((1.0, 0, 0.9, 0.0), (1.0, 100, 1.0, 0.0), (0.7, 20000, 0.6, 0.0), (2.0, 0, 1.0, 0.97), (1.0, 0, 1.0, 0.0),
                       (1.0, 0, 0.3, 0.001)):
        _check_large(logits, u, t, k, p, m)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_sample_more_rows_than_a_slice_in_large_chunks(dtype):
    """More than 512 rows of several chunks, of a wider tensor."""
    rng = np.random.default_rng(12)
    B, V = 517, 9001
    wide = torch.full((B, V + 37), 50.0, dtype=T_OF[dtype], device="cuda")
    wide[:, 5:5 + V] = _logits(rng, B, V, dtype)
    some = lambda a, b: np.where(rng.random(B) < 0.3, a, b)   # noqa: E731
    _check_large(wide[:, 5:5 + V], rng.random(B), some(0.0, rng.uniform(0.2, 2, B)), some(0, rng.integers(-1, 600, B)),
                 some(1.0, rng.uniform(0, 1.1, B)), some(0.0, rng.uniform(0, 0.3, B)))


def test_sample_with_one_workspace_for_all_batches():
    rng = np.random.default_rng(13)
    V, most = 20011, 90
    logits, u = _logits(rng, most, V, "bf16"), _t(rng.random(most).astype(np.float32))
    ws = torch.empty(_ops().sample_workspace_bytes(most, V), dtype=torch.uint8, device="cuda")
    for rows in (1, 2, 26, 27, 89, 90):   # (27 rows and more are worked on in large chunks)
        got = _ops().sample_tokens(logits[:rows], u[:rows], 0.8, 50, 0.9, workspace=ws)
        assert torch.equal(got, _ops().sample_tokens(logits[:rows], u[:rows], 0.8, 50, 0.9))
