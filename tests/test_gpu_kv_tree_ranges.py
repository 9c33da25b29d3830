"""Attention of drafted tokens (ops.kv_tree_attention) where its arithmetic and its deal of rows are stretched, in every form
of its kernels: rows whose first keys have logits far below zero, sharp softmaxes, small value scales beside larger ones, and
node counts that differ between sequences.  Against the 64-bit reference; parity unpinned (the reference project has none)."""
import numpy as np
import pytest
import torch

import attn_step_ref as ref
from test_gpu_attn_step import D, PAGE, _check_tree, _masks, _ops, _t, _tree_case

pytestmark = pytest.mark.gpu

# nodes, query and kv heads: 1, 3 and 6 groups of 16 rows, all pages of a wave; 8, 15 and 20 groups, dealt to 8 waves
FORMS = [(3, 4, 1), (11, 8, 2), (24, 4, 1), (31, 4, 1), (60, 8, 2), (64, 5, 1)]


def _aim(rng, case, size, bits, pages, nodes):
    """Queries along a fixed direction, `size` long per value; the keys of the given physical pages, and those of the nodes
    if `nodes`, the other way: their logits are some -22.6 * size, the others' around zero."""
    q, k, v, seen, cache, table = case
    w = np.where(rng.permutation(D) < D // 2, 1, -1)
    top = 127 if bits == 8 else 7
    q = (0.1 * size * q + size * torch.from_numpy(w).cuda()).half()
    code = (100, 28) if bits == 8 else (5, 3)
    cache[0][pages] = ref.pack(rng.integers(-code[1] + 1, code[1], (len(pages), *cache[0].shape[1:3], D)) - code[0] * w, bits)
    cache[2][pages] = np.float16(2.0 / code[0])
    if nodes:
        k = (0.3 * k - 2.0 * torch.from_numpy(w).cuda()).half()
    assert top >= code[0] + code[1] - 1
    return q, k, v, seen, cache, table


def _own_pages(table, lens):
    return np.concatenate([table[b, :-(-n // PAGE)] for b, n in enumerate(lens)])


def _run(case, lens, bits, **kw):
    q, k, v, seen, cache, table = case
    return _ops().kv_tree_attention(q, k, v, _t(_masks(seen)), *[_t(c) for c in cache], _t(table), _t(np.int32(lens)), bits,
                                    **kw)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("N,Hq,Hkv", FORMS)
@pytest.mark.parametrize("where", ["all", "far", "cache", "nodes", "stretch", "zero"])
def test_first_keys_far_below_zero(bits, N, Hq, Hkv, where):
    """Logits around -160 (8 bits; -1000 "far") or -100 (4 bits, and where the pages' value scale is zero): of all keys, of
    the cache's or the nodes' alone, of 32 to 320 tokens from a page's beginning on.  A row's first keys set its reference,
    however low they are.  (Sizes that keep the logits' own error, `slip`, below a tenth, where its bound is linear.)"""
    lens = [700, 0, 65, 33]
    if where == "far" and bits == 4:
        pytest.skip("fp32 sums over 4-bit codes do not resolve logits of 1000")
    size = 45 if where == "far" else 4.5 if where == "zero" or bits == 4 else 7
    rng = np.random.default_rng(N + bits)
    case = _tree_case(N + bits, lens, N, Hq, Hkv, bits, "random" if where in ("all", "far") else "tree")
    pages = _own_pages(case[5], lens)
    if where == "nodes":
        pages = pages[:0]
    elif where == "stretch":
        pages = np.concatenate([case[5][0, :4], case[5][0, 20:40], case[5][2, :2]])
    case = _aim(rng, case, size, bits, pages, where in ("all", "far", "nodes", "zero"))
    if where == "zero":
        case[4][3][pages] = 0
    got = _run(case, lens, bits)
    assert not got.isnan().any()
    _check_tree(got, *case, lens, bits)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("N,Hq,Hkv", FORMS)
def test_sharp_logits_of_both_signs(bits, N, Hq, Hkv):
    """Logits of a standard deviation of some 190 (8 bits) and 13 (4 bits, whose fp32 sums resolve no more): the references
    jump, in both directions at a row's beginning."""
    lens = [700, 0, 65, 1040]
    wide = 10.0 if bits == 8 else 2.4
    case = _tree_case(3 * N + bits, lens, N, Hq, Hkv, bits, "tree", scale=wide)
    case[4][2][np.isfinite(case[4][2])] *= np.float16(wide)
    _check_tree(_run(case, lens, bits), *case, lens, bits)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("N,Hq,Hkv", FORMS)
def test_forms_repeat_bit_for_bit(bits, N, Hq, Hkv):
    lens = [3000, 0, 100, 1500]
    case = _tree_case(2 * N + bits, lens, N, Hq, Hkv, bits, "tree")
    want = _run(case, lens, bits)
    for _ in range(3):
        ws = torch.full((_ops().kv_tree_workspace_bytes(len(lens), N, Hq, Hkv, case[5].shape[1]),), 255, dtype=torch.uint8,
                        device="cuda")
        assert torch.equal(_run(case, lens, bits, workspace=ws), want)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("N,Hq,Hkv,nodes", [
    (64, 5, 1, [4, 20, 33, 44, 64, 26]), (64, 16, 1, [2, 7, 14, 30, 58, 0]), (40, 16, 2, [3, 28, 15, 40, 9, 1]),
    (20, 16, 1, [2, 14, 8, 20, 11, 5]), (33, 4, 1, [1, 33, 17, 5, 25, 29]), (61, 4, 1, [2, 40, 33, 61, 17, 9])])
def test_fewer_live_nodes_than_the_launch_has_room_for(bits, N, Hq, Hkv, nodes):
    """Units whose waves get fewer groups of rows than planned, from none to all but one, split over many workgroups: the
    reference's values, the same bits on every run, and nothing past the live nodes (K and V hold NaN there)."""
    lens = [1500, 700, 2100, 40, 0, 333]
    q, k, v, seen, cache, table = _tree_case(N + Hq + bits, lens, N, Hq, Hkv, bits, "tree", scale=2.0)
    k, v = k.clone(), v.clone()
    for b, n in enumerate(nodes):
        k[b, n:] = v[b, n:] = float("nan")
        seen[b, :, n:] = False
    args = [q, k, v, _t(_masks(seen)), *[_t(c) for c in cache], _t(table), _t(np.int32(lens)), bits]
    first = None
    for fill in (0, 255, 0x3C, 255):
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
        ws = torch.full((_ops().kv_tree_workspace_bytes(len(lens), N, Hq, Hkv, table.shape[1]),), fill, dtype=torch.uint8,
                        device="cuda")
        got = _ops().kv_tree_attention(*args, num_nodes=_t(np.int32(nodes)), out=out, workspace=ws)
        for b, n in enumerate(nodes):
            assert (got[b, n:] == 7.0).all()
        first = got if first is None else first
        assert torch.equal(got, first)
    clean = [torch.where(x.isnan(), 0, x) for x in (k, v)]
    _check_tree(first, q, *clean, seen, cache, table, lens, bits, nodes=nodes)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("N,Hq,Hkv", [(1, 4, 1), (11, 4, 1), (24, 4, 1), (31, 4, 1), (64, 5, 1)])
@pytest.mark.parametrize("scale", [2.0 ** -8, 2.0 ** -14, 2.0 ** -19])
def test_many_keys_far_below_a_node(bits, N, Hq, Hkv, scale):
    """8192 cached keys 12 below each node's own logit hold 5 % of its weight between them, each 2^-17 of the node's, and
    2^-17 times the pages' value scale where that is folded into the probability.  The values of both are of one size.  Many
    copies of the sequence: most of them are one workgroup's whole."""
    lens, copies = [8192], 512
    rng = np.random.default_rng(N + bits)
    q, k, v, seen, cache, table = _tree_case(N, lens, N, Hq, Hkv, bits, "tree", spare=0)
    top, w = (127, 7)[bits == 4], np.where(rng.permutation(D) < D // 2, 1, -1)
    q, k = torch.empty_like(q).copy_(torch.from_numpy(w)), torch.empty_like(k).copy_(torch.from_numpy(w * 12 * D ** -0.5))
    v = (v.clamp(-3, 3) * (scale * top / 3)).contiguous()
    seen[:] = np.eye(N, dtype=bool)
    cache[0][:] = 0
    cache[1][:] = ref.pack(rng.integers(top // 2, top + 1, (len(cache[1]), Hkv, PAGE, D)), bits)
    cache[3][:] = np.float16(scale)
    many = [t.expand(copies, *t.shape[1:]).contiguous() for t in (q, k, v, _t(_masks(seen)))]
    got = _ops().kv_tree_attention(*many, *[_t(c) for c in cache], _t(table).expand(copies, -1).contiguous(),
                                   _t(np.int32(lens * copies)), bits)
    for end in (got.float().amin(0, keepdim=True), got.float().amax(0, keepdim=True)):   # so all copies
        _check_tree(end, q, k, v, seen, cache, table, lens, bits)
