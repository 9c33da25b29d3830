"""What the operators around the attention and at the ends of a serving step refuse, without a GPU: the C-ABI before any launch
(placeholder pointers are never used), and the torch-facing ops before the library is called."""
import pytest
import torch

from trellis_serve_amd import _lib, ops

N = None
BAD, OK = _lib.EXL3_ERR_INVALID, _lib.EXL3_OK
FAR = 1 << 44   # apart: each placeholder has a range of its own


def at(i):
    return i * FAR


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def plan(lib, table=at(1), width=4, lens=at(2), new=at(3), batch=2, page=16, ring=at(4), num=9, state=at(5), state_out=at(6),
         rows=5, outs=None, ws=at(20), ws_bytes=1 << 20, **named):
    o = {name: at(10 + i) for i, name in enumerate(("start", "counts", "after", "pos", "row_lens", "seq", "slots"))} | named
    return lib.exl3_kv_step_plan(table, width, lens, new, batch, page, ring, num, state, state_out, rows, *o.values(), ws,
                                 ws_bytes, N)


def norm(lib, x=at(1), xt=1, ld_x=512, r=at(2), rt=1, ld_r=512, w=at(3), pw=at(4), wt=1, gate=N, gt=1, kind=0, ld_g=0, rows=3,
         dim=512, y=at(6), h=at(7)):
    return lib.exl3_add_norm(x, xt, ld_x, r, rt, ld_r, w, pw, wt, 0, gate, gt, kind, ld_g, 0, 1.0, 1e-6, rows, dim, y, h, N)


def bounds(lib, k=at(1), pages=8, table=at(2), width=4, lens=at(3), first=N, max_new=64, batch=2, hkv=2, dim=128, page=16, bits=8,
           out=at(4)):
    return lib.exl3_kv_page_bounds(k, pages, table, width, lens, first, max_new, batch, hkv, dim, page, bits, out, N)


def select(lib, q=at(1), ld_q=512, ks=at(2), edge=at(3), pages=8, table=at(4), batch=2, width=30, row_seq=N, lens=at(5), rows=2,
           hq=4, hkv=2, dim=128, page=16, bits=8, top=8, first=1, last=2, out=at(6), ws=at(7), ws_bytes=1 << 20):
    return lib.exl3_kv_select_pages(q, ld_q, ks, edge, pages, table, batch, width, row_seq, lens, rows, hq, hkv, dim, page, bits,
                                    top, first, last, out, ws, ws_bytes, N)


def sparse(lib, q=at(1), ld_q=512, k=at(2), v=at(3), ks=at(4), vs=at(5), pages=8, table=at(6), batch=2, width=30, row_seq=N,
           lens=at(7), rows=2, hq=4, hkv=2, dim=128, page=16, bits=8, chosen=at(8), top=8, out=at(9), ws=at(10),
           ws_bytes=1 << 24):
    return lib.exl3_kv_sparse_attention(q, ld_q, k, v, ks, vs, pages, table, batch, width, row_seq, lens, rows, hq, hkv, dim, page,
                                        bits, chosen, top, 0.1, out, ws, ws_bytes, N)


def sample(lib, logits=at(1), type=2, ld=100, rows=3, vocab=100, u=at(2), t=N, k=N, p=N, m=N, tokens=at(3), probs=N, ws=at(4),
           ws_bytes=1 << 30, all_t=1.0):
    return lib.exl3_sample(logits, type, ld, rows, vocab, u, t, all_t, k, 0, p, 1.0, m, 0.0, tokens, probs, ws, ws_bytes, N)


@pytest.mark.parametrize("call,kw,msg", [
    (plan, dict(page=32), "page_size = 32"), (plan, dict(batch=-1), "batch = -1"), (plan, dict(width=0), "max_pages = 0"),
    (plan, dict(num=0), "free pages = 0"), (plan, dict(rows=-1), "rows = -1"), (plan, dict(batch=0), "no sequence"),
    (plan, dict(batch=1 << 20, width=1 << 20), "max_pages = 1048576"), (plan, dict(table=N), "null"), (plan, dict(slots=N), "null"),
    (plan, dict(state_out=N), "null"), (plan, dict(ws=N), "workspace"), (plan, dict(ws_bytes=12), "workspace"),
    (plan, dict(pos=at(1) + 4), "overlaps"), (plan, dict(after=at(2)), "overlaps"), (plan, dict(ring=at(1) + 8), "overlaps"),
    (plan, dict(state_out=at(3) + 4), "overlaps"), (plan, dict(state_out=at(5) + 4), "overlaps"),
    (plan, dict(ws=at(12) + 4), "overlaps"), (plan, dict(slots=at(13) - 8), "overlaps"),
    (norm, dict(dim=0), "dim = 0"), (norm, dict(dim=32769), "dim = 32769"), (norm, dict(rows=-1), "rows = -1"),
    (norm, dict(xt=2), "types 2"), (norm, dict(rt=3), "types"), (norm, dict(wt=-1), "types"), (norm, dict(gt=5), "types"),
    (norm, dict(kind=4), "gate kind 4"), (norm, dict(kind=1), "without a gate"), (norm, dict(gate=at(5)), "gate kind 0 with a gate"),
    (norm, dict(w=N), "a weight and its output"), (norm, dict(y=N), "a weight and its output"),
    (norm, dict(w=N, y=N, h=N), "h alone"), (norm, dict(x=N), "null"), (norm, dict(ld_x=511), "row strides"),
    (norm, dict(ld_r=500), "row strides"), (norm, dict(kind=3, gate=at(5), ld_g=500), "row strides"),
    (norm, dict(kind=2, gate=at(5)), "row strides"), (norm, dict(x=at(1) + 1), "aligned"), (norm, dict(rt=2, h=at(7) + 2), "aligned"),
    (norm, dict(y=at(1)), "overlaps"), (norm, dict(y=at(2) + 1024), "overlaps"), (norm, dict(h=at(1) + 64), "overlaps"),
    (norm, dict(h=at(2) + 1024), "overlaps"), (norm, dict(h=at(2), ld_r=1024), "overlaps"), (norm, dict(h=at(6) + 2), "overlaps"),
    (norm, dict(h=at(3) - 2 * 3 * 512 + 2), "overlaps"), (norm, dict(y=at(4)), "overlaps"),
    (norm, dict(kind=1, gate=at(6)), "overlaps"), (norm, dict(kind=2, gate=at(7) + 64, ld_g=1), "overlaps"),
    (bounds, dict(dim=64), "head_dim = 64"), (bounds, dict(page=32), "page_size = 32"), (bounds, dict(bits=6), "bits = 6"),
    (bounds, dict(pages=0), "pages = 0"), (bounds, dict(hkv=0), "kv heads = 0"), (bounds, dict(max_new=-1), "max_new = -1"),
    (bounds, dict(k=N), "null"), (bounds, dict(out=at(4) + 8), "aligned"), (bounds, dict(table=N), "null"),
    (bounds, dict(out=at(1) + 64), "overlap"), (bounds, dict(out=at(3) - 16), "overlap"), (bounds, dict(first=at(4) + 4), "overlap"),
    (bounds, dict(batch=1 << 20, width=1 << 12, max_new=1 << 20), "sequences"),
    (select, dict(dim=64), "head_dim = 64"), (select, dict(bits=2), "bits = 2"), (select, dict(rows=70000, row_seq=at(8)), "rows = 70000"),
    (select, dict(top=0), "top = 0"), (select, dict(hq=40, hkv=2), "group <= 16"), (select, dict(hq=5), "heads 5"),
    (select, dict(rows=3), "without row_seq"), (select, dict(last=0), "last = 0"), (select, dict(first=7), "first = 7"),
    (select, dict(first=-1), "first = -1"), (select, dict(edge=N), "null"), (select, dict(edge=at(3) + 8), "aligned"),
    (select, dict(q=N), "null"), (select, dict(batch=0, row_seq=at(8)), "no sequence"), (select, dict(ld_q=500), "row stride"),
    (select, dict(q=at(1) + 8), "row stride"), (select, dict(ws=N), "workspace"), (select, dict(ws_bytes=511), "workspace"),
    (select, dict(ws=at(7) + 4), "aligned"), (select, dict(out=at(1) + 8), "overlaps"), (select, dict(ws=at(3) - 16), "overlaps"),
    (select, dict(out=at(7) + 4), "overlaps"), (select, dict(row_seq=at(6) + 4), "overlaps"),
    (sparse, dict(page=8), "page_size = 8"), (sparse, dict(bits=16), "bits = 16"), (sparse, dict(top=(1 << 20) + 1), "top"),
    (sparse, dict(rows=5), "without row_seq"), (sparse, dict(v=N), "null"), (sparse, dict(k=at(2) + 4), "aligned"),
    (sparse, dict(chosen=N), "null"), (sparse, dict(out=at(9) + 8), "row stride"), (sparse, dict(ld_q=516), "row stride"),
    (sparse, dict(ws=N), "workspace"), (sparse, dict(ws_bytes=100), "workspace"), (sparse, dict(out=at(2) + 16), "overlaps"),
    (sparse, dict(out=at(8)), "overlaps"), (sparse, dict(ws=at(9) + 16), "overlaps"), (sparse, dict(ws=at(5) - 16), "overlaps"),
    (sample, dict(rows=-1), "rows = -1"), (sample, dict(vocab=0), "vocab = 0"), (sample, dict(vocab=(1 << 20) + 1, ld=1 << 21), "vocab"),
    (sample, dict(type=3), "type 3"), (sample, dict(tokens=N), "neither"), (sample, dict(u=N), "random numbers"),
    (sample, dict(logits=N), "null"), (sample, dict(ld=99), "stride 99"), (sample, dict(logits=at(1) + 2), "aligned"),
    (sample, dict(ws=N), "workspace"), (sample, dict(ws_bytes=64), "workspace"), (sample, dict(ws=at(4) + 8), "aligned"),
    (sample, dict(probs=at(1) + 400), "overlaps"), (sample, dict(tokens=at(2)), "overlaps"), (sample, dict(ws=at(1) - 16), "overlaps"),
    (sample, dict(t=at(3) + 4), "overlaps"), (sample, dict(k=at(4)), "overlaps"), (sample, dict(probs=at(3) - 8), "overlaps")])
def test_refusals_of_the_c_abi(lib, call, kw, msg):
    assert call(lib, **kw) == BAD
    assert msg in lib.exl3_last_error().decode(), lib.exl3_last_error()


def test_empty_calls_launch_nothing(lib):
    assert plan(lib, batch=0, rows=0, table=N, lens=N) == OK
    assert norm(lib, rows=0, x=N, r=N, y=N, h=N) == OK
    assert bounds(lib, batch=0, table=N, lens=N) == OK and bounds(lib, max_new=0) == OK
    assert select(lib, rows=0, batch=0, q=N, lens=N, out=N, table=N, ws=N, ws_bytes=0) == OK
    assert sparse(lib, rows=0, batch=0, q=N, lens=N, out=N, table=N, chosen=N, ws=N, ws_bytes=0) == OK
    assert sample(lib, rows=0, logits=N, u=N, tokens=N, ws=N, ws_bytes=0) == OK


def test_workspace_sizes(lib):
    for batch in (1, 3, 5000):
        need = lib.exl3_kv_step_plan_workspace_bytes(batch)
        assert plan(lib, batch=batch, ws_bytes=need - 1) == BAD
    for rows, hkv, width in ((1, 1, 30), (7, 8, 9000), (300, 2, 65)):
        need = lib.exl3_kv_select_workspace_bytes(rows, hkv, width)
        kw = dict(rows=rows, batch=rows, hkv=hkv, hq=hkv, ld_q=hkv * 128, width=width)
        assert need > 0 and select(lib, **kw, ws_bytes=need - 1) == BAD
    for rows, hkv, top in ((1, 8, 64), (16, 2, 300), (2, 1, 100000)):
        need = lib.exl3_kv_sparse_workspace_bytes(rows, hkv * 4, hkv, top)
        kw = dict(rows=rows, batch=rows, hkv=hkv, hq=hkv * 4, ld_q=hkv * 512, top=top)
        assert need > 0 and sparse(lib, **kw, ws_bytes=need - 1) == BAD
    assert lib.exl3_kv_sparse_workspace_bytes(2000, 8, 8, 4) == 0   # one part: no states
    for rows, vocab in ((1, 1), (1, 32003), (64, 131072), (5000, 4097), (2, 1 << 20)):
        need = lib.exl3_sample_workspace_bytes(rows, vocab)
        assert need > 0 and sample(lib, rows=rows, vocab=vocab, ld=vocab, ws_bytes=need - 1) == BAD
    # a workspace for the most rows serves fewer
    for vocab in (1000, 32003, 131072, 1 << 20):
        sizes = [lib.exl3_sample_workspace_bytes(rows, vocab) for rows in range(1, 200)]
        assert sizes == sorted(sizes)
    for f, args in ((lib.exl3_kv_step_plan_workspace_bytes, (0,)), (lib.exl3_kv_select_workspace_bytes, (0, 1, 1)),
                    (lib.exl3_kv_sparse_workspace_bytes, (1, 0, 1, 1)), (lib.exl3_sample_workspace_bytes, (3, -1)),
                    (lib.exl3_sample_workspace_bytes, (3, 1 << 21))):
        assert f(*args) == 0


# ---- the torch-facing ops, on host tensors: shapes and types are refused first, then the device ---------------------------

def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def h(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


def _refuses(call, cases):
    for args, kw, msg in cases:
        with pytest.raises(ValueError, match=msg):
            call(*args, **kw)


def test_kv_step_plan_refuses():
    good = [i32(2, 4), i32(2), i32(2), i32(9), i32(2), 5]

    def but(i, x):
        return [*good[:i], x, *good[i + 1:]]

    _refuses(ops.kv_step_plan, [
        (but(0, i32(2, 4).long()), {}, "page_table"), (but(0, i32(8)), {}, "page_table"), (but(0, i32(4, 2).t()), {}, "page_table"),
        (but(1, i32(3)), {}, "seq_lens"), (but(2, i32(2).long()), {}, "new_lens"), (but(3, i32(3, 3)), {}, "free_pages"),
        (but(3, i32(18)[::2]), {}, "free_pages"), (but(4, i32(3)), {}, "free_state"), (good, dict(state_out=i32(1)), "state_out"),
        (but(5, -1), {}, "rows = -1"), (good, {}, "cuda")])


def test_add_norm_refuses():
    x, w = h(3, 64), h(64)
    f = ops.add_norm
    _refuses(f, [
        ((h(64), x, w), {}, "x must be"), ((x.float(), x, w), {}, "x must be one of"), ((x, h(3, 65), w), {}, "residual must be"),
        ((x, x.double(), w), {}, "residual must be one of"), ((x, x, h(63)), {}, "weight must be"),
        ((x, x, w), dict(post_weight=w.float()), "one type"), ((x, x, w.double()), {}, "weight must be"),
        ((x, x, w), dict(gate=h(63)), "gate must be"), ((x, x, w), dict(gate=h(3)), "gate must be"),
        ((x, x, w), dict(gate=h(3, 2)), "gate must be"), ((x, x, w), dict(gate=h(64).double()), "gate must be"),
        ((x, x, w), dict(gate=h(1, 1).expand(3, 1)), "strides"), ((x, x, w), dict(gate=h(64, 3).t()), "contiguous"),
        ((h(64, 3).t(), x, w), {}, "contiguous"), ((x, x, w), dict(out=(None, x.clone())), "comes with a weight"),
        ((x, x, None), dict(out=(x.clone(), None)), "comes with a weight"), ((x, x, w), dict(out=(h(3, 63), None)), "shape"),
        ((x, x.float(), w), dict(out=(x.clone(), x.clone())), "out must be one of"), ((x, x, w), {}, "cuda")])


def test_kv_page_bounds_refuses():
    k, table, lens, out = h(8, 2, 16, 128).to(torch.int8), i32(2, 3), i32(2), h(8, 2, 2, 128).to(torch.int8)
    _refuses(ops.kv_page_bounds, [
        ((k, table, lens, 5, out), {}, "bits"), ((k, table, lens, 4, out), {}, "k_cache must be"),
        ((k.half(), table, lens, 8, out), {}, "k_cache must be"), ((k, table, lens, 8, out[:, :, :1]), {}, "bounds must be"),
        ((k, table, lens, 8, out.half()), {}, "bounds must be"), ((k, table.long(), lens, 8, out), {}, "page_table"),
        ((k, table, i32(3), 8, out), {}, "seq_lens"), ((k, table, lens, 8, out), dict(first=i32(1)), "first"),
        ((k, table, lens, 8, out), dict(max_new=-1), "max_new"), ((k.transpose(0, 1).contiguous().transpose(0, 1), table, lens, 8, out), {}, "contiguous"),
        ((k, table, lens, 8, out), {}, "cuda")])


def test_kv_select_pages_and_sparse_attention_refuse():
    q, edge, ks, table, lens = h(2, 4, 128), h(8, 2, 2, 128).to(torch.int8), h(8, 2), i32(2, 3), i32(2)
    f = ops.kv_select_pages
    _refuses(f, [
        ((q, edge, ks, table, lens, 6, 4), {}, "bits"), ((q, edge, ks, table, lens, 4, 4), {}, "bounds must be"),
        ((q, edge, ks.float(), table, lens, 8, 4), {}, "k_scale"), ((q.bfloat16(), edge, ks, table, lens, 8, 4), {}, "q must be"),
        ((h(2, 5, 128), edge, ks, table, lens, 8, 4), {}, "query heads"), ((h(3, 4, 128), edge, ks, table, i32(3), 8, 4), {}, "row_seq"),
        ((q, edge, ks, table, i32(3), 8, 4), {}, "seq_lens"), ((q, edge, ks, table, lens, 8, 4), dict(row_seq=i32(3)), "row_seq"),
        ((q, edge, ks, table, lens, 8, 2), {}, "top = 2"), ((q, edge, ks, table, lens, 8, 4), dict(last=0), "last = 0"),
        ((q, edge, ks, table, lens, 8, 4), dict(out=i32(2, 2, 5)), "shape"), ((q, edge, ks, table.t(), lens, 8, 4), {}, "page_table"),
        ((q, edge, ks, table, lens, 8, 4), {}, "cuda")])
    c = h(8, 2, 16, 128).to(torch.int8)
    pages = i32(2, 2, 4)
    f = ops.kv_sparse_attention
    _refuses(f, [
        ((q, c, c, ks, ks, table, lens, 4, pages), {}, "k_cache / v_cache"), ((q, c, c[:4], ks, ks, table, lens, 8, pages), {}, "k_cache"),
        ((q, c, c, ks, ks[:4], table, lens, 8, pages), {}, "v_scale"), ((q, c, c, ks, ks, table, lens, 8, pages.long()), {}, "pages must"),
        ((q, c, c, ks, ks, table, lens, 8, i32(2, 1, 4)), {}, "pages must"), ((q, c, c.half(), ks, ks, table, lens, 8, pages), {}, "1-byte"),
        ((q[:, :, :64], c, c, ks, ks, table, lens, 8, pages), {}, "128"), ((q, c, c, ks, ks, table, i32(1), 8, pages), {}, "seq_lens"),
        ((q, c, c, ks, ks, table, lens, 8, pages), dict(out=h(2, 4, 64)), "shape"), ((q, c, c, ks, ks, table, lens, 8, pages), {}, "cuda")])


def test_sampling_refuses():
    x, u = torch.zeros(3, 50), torch.zeros(3)
    _refuses(ops.sample_tokens, [
        ((x.double(), u), {}, "logits must be"), ((x, u.double()), {}, "uniform"), ((x, u[:2]), {}, "uniform"),
        ((x.t().contiguous().t(), u), {}, "contiguous"), ((torch.zeros(3, 2, 50)[:, 0:1], u.view(3, 1)), {}, "contiguous"),
        ((x, u), dict(temperature=-1.0), "temperature = -1"), ((x, u), dict(temperature=float("nan")), "temperature = nan"),
        ((x, u), dict(top_k=-1), "top_k = -1"), ((x, u), dict(top_p=-0.1), "top_p"), ((x, u), dict(min_p=1.5), "min_p"),
        ((x, u), dict(min_p=-0.5), "min_p"), ((x, u), dict(temperature=u.double()), "temperature"),
        ((x, u), dict(top_k=torch.zeros(3)), "top_k"), ((x, u), dict(top_p=u[:1]), "top_p"), ((x, u), dict(min_p=u.half()), "min_p"),
        ((x, u), dict(probs=torch.zeros(3, 49)), "shape"), ((x, u), {}, "cuda")])
    _refuses(ops.sampling_probs, [((x.long(),), {}, "logits"), ((x,), dict(out=x.half()), "out must be"), ((x,), {}, "cuda")])
