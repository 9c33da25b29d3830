"""What the operators around the quantized-KV attention refuse, without a GPU: the C-ABI before any launch (placeholder
pointers are never used), and the torch-facing ops before the library is called."""
import pytest
import torch

from trellis_serve_amd import _lib, ops

P, N = 0x1000, None
BAD = _lib.EXL3_ERR_INVALID


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def norm(lib, q=P, k=P, ld_q=5120, ld_k=1024, tokens=4, hq=40, hkv=8, dim=128, wq=P, wk=P, wt=0, cs=P, max_pos=10,
         rotary=128, pos=P, qo=P, ko=P):
    return lib.exl3_qk_norm_rope(q, k, 0, ld_q, ld_k, tokens, hq, hkv, dim, wq, wk, wt, 1e-6, cs, max_pos, rotary, 0, pos, 0,
                                 qo, ko, 0, N)


def append(lib, k=P, v=P, ld_k=1024, ld_v=1024, rows=4, row_start=N, per=2, select=N, counts=N, max_new=2, kc=P, vc=P,
           ks=P, vs=P, pages=8, table=P, width=4, lens=P, batch=2, hkv=8, dim=128, page=16, bits=8):
    return lib.exl3_kv_append(k, v, 0, ld_k, ld_v, rows, row_start, per, select, counts, max_new, kc, vc, ks, vs, pages,
                              table, width, lens, batch, hkv, dim, page, bits, N)


def gather(lib, kc=P, vs=P, pages=8, table=P, width=4, lens=P, starts=N, row_start=P, batch=2, rows=9, hkv=8, dim=128,
           page=16, bits=8, ko=P, vo=P):
    return lib.exl3_kv_gather(kc, P, P, vs, pages, table, width, lens, starts, row_start, batch, rows, hkv, dim, page, bits,
                              ko, vo, 0, N)


def tree(lib, q=P, ld_q=5120, k=P, v=P, ld_k=1024, ld_v=1024, nodes=5, kc=P, pages=8, table=P, width=4, lens=P, batch=2,
         hq=40, hkv=8, dim=128, page=16, bits=8, out=P, ws=P, ws_bytes=1 << 40):
    return lib.exl3_kv_tree_attention(q, ld_q, k, v, ld_k, ld_v, N, nodes, N, kc, P, P, P, pages, table, width, lens, batch,
                                      hq, hkv, dim, page, bits, 0.1, out, ws, ws_bytes, N)


def verify(lib, p=P, q=N, tokens=P, parents=N, u=P, batch=2, nodes=5, vocab=100, acc=P, counts=P, out=P, ws=P,
           ws_bytes=1 << 30):
    return lib.exl3_verify_drafts(p, q, tokens, parents, u, N, batch, nodes, vocab, acc, counts, out, ws, ws_bytes, N)


@pytest.mark.parametrize("call,kw,msg", [
    (norm, dict(dim=64), "head_dim = 64"), (norm, dict(hq=0), "heads 0"), (norm, dict(tokens=-1), "tokens = -1"),
    (norm, dict(wk=N), "both weights"), (norm, dict(wt=3), "weight type 3"), (norm, dict(wq=N, wk=N, cs=N), "neither"),
    (norm, dict(rotary=24), "rotary_dim = 24"), (norm, dict(rotary=144), "rotary_dim = 144"),
    (norm, dict(max_pos=0), "max_pos = 0"), (norm, dict(pos=N), "null"), (norm, dict(qo=N), "null"),
    (norm, dict(ld_q=5112), "token strides"), (norm, dict(ld_k=1028), "token strides"), (norm, dict(q=P + 2), "aligned"),
    (norm, dict(wk=P + 8), "aligned"),
    (append, dict(dim=64), "head_dim = 64"), (append, dict(page=32), "page_size = 32"), (append, dict(bits=5), "bits = 5"),
    (append, dict(kc=N), "null"), (append, dict(k=N), "null"), (append, dict(lens=N), "null"),
    (append, dict(rows=5), "5 rows are not 2 sequences of 2"), (append, dict(ld_v=1000), "token strides"),
    (append, dict(vc=P + 4), "aligned"), (append, dict(max_new=-1), "max_new = -1"), (append, dict(pages=0), "pages = 0"),
    (append, dict(batch=-1), "batch = -1"), (append, dict(k=P + 8), "aligned"),
    (append, dict(batch=1 << 20, rows=1 << 21, max_new=1 << 20, width=1 << 20), "new tokens"),
    (gather, dict(dim=256), "head_dim = 256"), (gather, dict(bits=2), "bits = 2"), (gather, dict(vs=N), "null"),
    (gather, dict(row_start=N), "null"), (gather, dict(ko=P + 2), "aligned"), (gather, dict(rows=-1), "rows = -1"),
    (gather, dict(width=0), "max_pages = 0"),
    (tree, dict(dim=64), "head_dim = 64"), (tree, dict(page=8), "page_size = 8"), (tree, dict(bits=16), "bits = 16"),
    (tree, dict(nodes=0), "nodes = 0"), (tree, dict(nodes=65), "nodes = 65"), (tree, dict(hq=40, hkv=2), "group <= 16"),
    (tree, dict(hq=41), "heads 41"), (tree, dict(ld_q=5000), "token strides"), (tree, dict(q=N), "null"),
    (tree, dict(out=P + 8), "aligned"), (tree, dict(ws=N), "workspace"), (tree, dict(ws_bytes=64), "workspace"),
    (tree, dict(batch=60000, width=1 << 20), "too large"), (tree, dict(kc=N), "null"),
    (verify, dict(nodes=0), "nodes = 0"), (verify, dict(nodes=65), "nodes = 65"), (verify, dict(vocab=0), "vocab = 0"),
    (verify, dict(q=P, parents=P), "chain"), (verify, dict(p=N), "null"), (verify, dict(counts=N), "null"),
    (verify, dict(ws=N), "workspace"), (verify, dict(ws_bytes=8), "workspace"), (verify, dict(ws=P + 4), "aligned"),
    (verify, dict(batch=70000), "batch = 70000")])
def test_refusals_of_the_c_abi(lib, call, kw, msg):
    assert call(lib, **kw) == BAD
    assert msg in lib.exl3_last_error().decode(), lib.exl3_last_error()


def test_empty_calls_launch_nothing(lib):
    ok = _lib.EXL3_OK
    assert norm(lib, q=N, k=N, tokens=0, pos=N, qo=N, ko=N) == ok
    assert append(lib, k=N, v=N, rows=0, batch=0, table=N, lens=N) == ok
    assert append(lib, k=N, v=N, rows=0, row_start=P, per=0) == ok
    assert gather(lib, rows=0, ko=N, vo=N) == ok and gather(lib, batch=0, table=N, lens=N, row_start=N) == ok
    assert tree(lib, q=N, k=N, v=N, batch=0, table=N, lens=N, out=N, ws=N, ws_bytes=0) == ok
    assert verify(lib, p=N, tokens=N, u=N, batch=0, acc=N, counts=N, out=N, ws=N, ws_bytes=0) == ok


def test_workspace_sizes(lib):
    """0 for shapes that are refused; a call with the reported size gets past the check (with no GPU present it then fails at
    its first launch), one byte less does not."""
    size = lib.exl3_kv_tree_workspace_bytes
    assert size(0, 4, 8, 8, 4) == size(1, 65, 8, 8, 4) == size(1, 4, 9, 8, 4) == size(1, 4, 136, 8, 4) == 0
    assert lib.exl3_verify_workspace_bytes(0, 5) == lib.exl3_verify_workspace_bytes(1, 0) == 0
    for batch, nodes, hq, hkv, width in ((1, 1, 8, 8, 1), (3, 7, 40, 8, 100), (64, 64, 16, 1, 9), (2, 33, 64, 4, 2048)):
        need = size(batch, nodes, hq, hkv, width)
        assert need > 0
        kw = dict(batch=batch, nodes=nodes, hq=hq, hkv=hkv, width=width, ld_q=hq * 128, ld_k=hkv * 128, ld_v=hkv * 128)
        assert tree(lib, **kw, ws_bytes=need - 1) == BAD
        if not torch.cuda.is_available():
            assert tree(lib, **kw, ws_bytes=need) == _lib.EXL3_ERR_HIP
    for batch, vocab in ((1, 1), (5, 4096), (7, 200001), (1, 1 << 28)):
        need = lib.exl3_verify_workspace_bytes(batch, vocab)
        assert need > 0 and verify(lib, batch=batch, vocab=vocab, ws_bytes=need - 1) == BAD
        if not torch.cuda.is_available():
            assert verify(lib, batch=batch, vocab=vocab, ws_bytes=need) == _lib.EXL3_ERR_HIP


# ---- the torch-facing ops, on host tensors: shapes and types are refused first, then the device ---------------------------

def _cache(B=2, width=3, hkv=2, bits=8, pages=8):
    codes = torch.zeros((pages, hkv, 16, 16 * bits), dtype=torch.int8 if bits == 8 else torch.uint8)
    scale = torch.ones((pages, hkv), dtype=torch.float16)
    return [codes, codes.clone(), scale, scale.clone(), torch.zeros((B, width), dtype=torch.int32),
            torch.zeros(B, dtype=torch.int32)]


def _h(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


def test_qk_norm_rope_refuses():
    q, k, w, cs, pos = _h(3, 4, 128), _h(3, 2, 128), _h(128), torch.zeros((9, 64)), torch.zeros(3, dtype=torch.int64)
    f = ops.qk_norm_rope
    for args, msg in (((q.float(), k.float(), w, w, cs, pos), "q must be one of"), ((q[..., :64], k, w, w, cs, pos), "128"),
                      ((q.transpose(0, 1), k, w, w, cs, pos), "contiguous"), ((q, k[:2], w, w, cs, pos), "3 tokens"),
                      ((q, k.bfloat16(), w, w, cs, pos), "3 tokens"), ((q, k, w, None, cs, pos), "both weights"),
                      ((q, k, w, w.float(), cs, pos), "k_weight"), ((q, k, w[:64], w, cs, pos), "q_weight"),
                      ((q, k, w, w, cs.half(), pos), "cos_sin"), ((q, k, w, w, cs, pos[:2]), "positions"),
                      ((q, k, w, w, cs, None), "positions"), ((q, k, w, w, cs[:, :40].contiguous(), pos), "multiple of 16"),
                      ((q, k, w, w, torch.zeros((0, 64)), pos), "cos_sin"), ((q, k, None, None, None, pos), "neither"),
                      ((q, k, w, w, cs, pos), "cuda")):
        with pytest.raises(ValueError, match=msg):
            f(*args)
    with pytest.raises(ValueError, match="out_dtype"):
        f(q, k, w, w, cs, pos, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="shape"):
        f(q, k, w, w, cs, pos, out=(k, k))
    with pytest.raises(ValueError, match="one type"):
        f(q, k, w, w, cs, pos, out=(q.clone(), k.bfloat16()))
    wide = _h(3, 1024)
    with pytest.raises(ValueError, match="may be its input"):
        f(wide[:, :512].unflatten(1, (4, 128)), k, w, w, cs, pos, out=(wide.view(-1)[:1536].view(3, 4, 128), k.clone()))


def test_cache_ops_refuse():
    c = _cache()
    k = _h(2, 5, 2, 128)

    def both(cache, msg, bits=8):
        with pytest.raises(ValueError, match=msg):
            ops.kv_append(k, k, *cache, bits)
        with pytest.raises(ValueError, match=msg):
            ops.kv_gather(*cache, bits, torch.zeros(3, dtype=torch.int32), 4)
        with pytest.raises(ValueError, match=msg):
            ops.kv_tree_attention(_h(2, 5, 4, 128), k, k, None, *cache, bits)

    both(c, "bits must be 4 or 8", bits=6)
    both(c, "at 4 bits", bits=4)
    for i, t, msg in ((0, c[0][:4], "must both be"), (1, c[1].half(), "1-byte"), (2, c[2].float(), "k_scale"),
                      (3, c[3][:, :1], "v_scale"), (4, c[4].long(), "page_table"), (4, c[4][0], "page_table"),
                      (5, c[5].long(), "seq_lens"), (5, c[5][:1], "seq_lens"), (4, c[4].t().contiguous().t(), "contiguous")):
        both([t if j == i else x for j, x in enumerate(c)], msg)
    both(c, "cuda")
    f, start = ops.kv_append, torch.zeros(3, dtype=torch.int32)
    for a, kw, msg in (((k[0, 0], k[0, 0]), {}, "k must be"), ((k, k), dict(row_start=start), "k must be"),
                       ((k, k[:, :4].contiguous()), {}, "alike"), ((k, k.bfloat16()), {}, "alike"), ((k[:, :, :1], k[:, :, :1]), {}, "2 heads"),
                       ((k[:1], k[:1]), {}, "holds 1 sequences"), ((k[0], k[0]), {}, "holds 5 sequences"),
                       ((k[0], k[0]), dict(row_start=start[:2]), "row_start"), ((k, k), dict(counts=start), "counts"),
                       ((k, k), dict(select=start), "select"), ((k, k), dict(select=torch.zeros((2, 3))), "select"),
                       ((k[0], k[0]), dict(row_start=start, max_new=-1), "max_new"),
                       ((k.transpose(0, 1).contiguous().transpose(0, 1),) * 2, {}, "one stride")):
        with pytest.raises(ValueError, match=msg):
            f(*a, *c, 8, **kw)
    g = ops.kv_gather
    for a, kw, msg in (((start.long(), 4), {}, "row_start"), ((start, 4), dict(starts=start), "starts"),
                       ((start, -1), {}, "rows"), ((start, 4), dict(dtype=torch.float32), "dtype"),
                       ((start, 4), dict(out=(_h(4, 2, 128), _h(3, 2, 128))), "shape"),
                       ((start, 4), dict(out=(_h(4, 2, 128), _h(4, 2, 128, dtype=torch.bfloat16))), "must be one of")):
        with pytest.raises(ValueError, match=msg):
            g(*c, 8, *a, **kw)


def test_kv_tree_attention_refuses():
    c, q, k = _cache(), _h(2, 5, 4, 128), _h(2, 5, 2, 128)
    mask, nodes = torch.ones((2, 5), dtype=torch.int64), torch.ones(2, dtype=torch.int32)
    f = ops.kv_tree_attention
    for a, kw, msg in (((q.bfloat16(), k, k, mask), {}, "q must be one of"), ((q, k.float(), k, mask), {}, "k_new"),
                       ((q[:1], k, k, mask), {}, "2 sequences"), ((q, k[:, :4].contiguous(), k, mask), {}, "2 sequences"),
                       ((q, k, k[:, :, :1], mask), {}, "2 kv heads"), ((q[:, :, :3], k, k, mask), {}, "heads 3 / 2"),
                       ((q, k, k, mask.int()), {}, "tree_mask"), ((q, k, k, mask[:, :4]), {}, "tree_mask"),
                       ((q, k, k, mask), dict(num_nodes=nodes.long()), "num_nodes"),
                       ((q, k, k, mask), dict(out=_h(2, 5, 4, 64)), "shape"),
                       ((_h(2, 65, 4, 128), _h(2, 65, 2, 128), _h(2, 65, 2, 128), None), {}, "65 nodes"),
                       ((_h(2, 5, 34, 128), k, k, mask), {}, "heads 34 / 2"), ((q, k, k, mask), {}, "cuda")):
        with pytest.raises(ValueError, match=msg):
            f(*a, *c, 8, **kw)


def test_verify_drafts_refuses():
    p, t, u = torch.zeros((2, 5, 30)), torch.zeros((2, 5), dtype=torch.int64), torch.zeros((2, 5))
    f = ops.verify_drafts
    for a, kw, msg in (((p.half(), t, u), {}, "target_probs"), ((p[0], t, u), {}, "target_probs"),
                       ((p[:, :, ::2], t, u), {}, "target_probs"), ((p, t.float(), u), {}, "tokens"),
                       ((p, t[:, :4], u), {}, "tokens"), ((p, t, u.double()), {}, "uniform"), ((p, t, u[:1]), {}, "uniform"),
                       ((p, t, u), dict(parents=t.short()), "parents"),
                       ((p, t, u), dict(parents=t, draft_probs=p), "chain"),
                       ((p, t, u), dict(draft_probs=p[:, :4]), "draft_probs"),
                       ((p, t, u), dict(num_nodes=torch.zeros(3, dtype=torch.int32)), "num_nodes"),
                       ((torch.zeros((2, 65, 3)), torch.zeros((2, 65), dtype=torch.int32), torch.zeros((2, 65))), {}, "65"),
                       ((torch.zeros((2, 5, 0)), t, u), {}, "0 tokens"), ((p, t, u), {}, "cuda")):
        with pytest.raises(ValueError, match=msg):
            f(*a, **kw)


def test_token_strides_of_views():
    """Columns of a wider row are taken as they lie; sizes of 1 carry no stride."""
    wide = _h(3, 4, 7 * 128 + 8)
    for t, dims, want in ((wide[..., 128:384].unflatten(2, (2, 128)), 4, 904), (wide[0, :, :256].unflatten(1, (2, 128)), 3, 904),
                          (wide[:, :1, :256].unflatten(2, (2, 128)), 4, 4 * 904), (wide[:1, :1, :256].unflatten(2, (2, 128)), 4, 256),
                          (_h(5, 3, 128)[:1], 3, 384)):
        assert ops._token_stride(t, "x", dims) == want
    with pytest.raises(ValueError, match="one stride"):
        ops._token_stride(wide[:, :3, :256].unflatten(2, (2, 128)), "x", 4)


def test_outputs_that_overlap_are_refused():
    x = torch.zeros(4 * 24 * 128, dtype=torch.float16)
    q, k = x[: 4 * 16 * 128].view(4, 16, 128), x[4 * 16 * 128:].view(4, 8, 128)
    cs, pos = torch.zeros(9, 128), torch.zeros(4, dtype=torch.int32)
    shifted = torch.zeros(4 * 16 * 128 + 8, dtype=torch.float16)
    q2 = shifted[: 4 * 16 * 128].view(4, 16, 128)
    for a, b, out in ((q, k, (x[4 * 8 * 128:].view(4, 16, 128), torch.zeros_like(k))),      # q_out over k
                      (q, k, (torch.zeros_like(q), x[: 4 * 8 * 128].view(4, 8, 128))),      # k_out over q
                      (q2, k, (shifted[8:].view(4, 16, 128), torch.zeros_like(k)))):        # q_out 8 values into q
        with pytest.raises(ValueError, match="overlaps"):
            ops.qk_norm_rope(a, b, None, None, cs, pos, out=out)
    y = torch.zeros(2 * 5 * 16 * 128, dtype=torch.float16)
    qt = y.view(2, 5, 16, 128)
    kt = torch.zeros(2, 5, 2, 128, dtype=torch.float16)
    cache = [torch.zeros(8, 2, 16, 128, dtype=torch.int8)] * 2 + [torch.zeros(8, 2, dtype=torch.float16)] * 2
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="overlaps"):
        ops.kv_tree_attention(qt, kt, kt, None, *cache, table, lens, 8, out=qt)
    both = torch.zeros(3, 2, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="overlaps"):
        ops.kv_gather(*cache, table, lens, 8, torch.zeros(3, dtype=torch.int32), 3, out=(both, both))


def test_wide_token_ids_do_not_wrap():
    t = torch.tensor([[5, 2 ** 32 + 5, -2 ** 40, 99, 100, -1]])
    assert ops._narrow(t, 100).tolist() == [[5, 100, -1, 99, 100, -1]] and ops._narrow(t, 100).dtype == torch.int32
