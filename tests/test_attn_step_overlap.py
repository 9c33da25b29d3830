"""Calls around the quantized-KV attention whose outputs, workspaces or caches lie in another tensor of the call are refused,
without a GPU: one workgroup would write what another still reads."""
import pytest
import torch

from trellis_serve_amd import _lib, ops

B, N, HQ, HKV, PAGES, WIDTH = 2, 5, 16, 2, 8, 4


def _half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def _cache():
    codes = lambda: torch.zeros(PAGES, HKV, 16, 128, dtype=torch.int8)   # noqa: E731
    return [codes(), codes(), _half(PAGES, HKV), _half(PAGES, HKV), torch.zeros(B, WIDTH, dtype=torch.int32),
            torch.zeros(B, dtype=torch.int32)]


def _over(t, shape, dtype=torch.float16):
    """A tensor of `shape` whose memory begins with that of t (of its storage, which is made large enough)."""
    n = torch.Size(shape).numel() * torch.empty((), dtype=dtype).element_size()
    store = torch.zeros(max(n, t.numel() * t.element_size()), dtype=torch.uint8)
    return store[:t.numel() * t.element_size()].view(t.dtype).view(t.shape), store[:n].view(dtype).view(shape)


def _refused(call, *args, **kw):
    with pytest.raises(ValueError, match="overlaps"):
        call(*args, **kw)


def test_norm_outputs_over_weights_tables_and_positions():
    q, k = _half(4, HQ, 128), _half(4, HKV, 128)
    rest = [_half(128), _half(128), torch.zeros(9, 128), torch.zeros(4, dtype=torch.int64)]
    for i in range(4):
        for o in range(2):
            r, out = list(rest), [torch.zeros_like(q), torch.zeros_like(k)]
            r[i], out[o] = _over(rest[i], out[o].shape)
            _refused(ops.qk_norm_rope, q, k, *r, out=tuple(out))


def test_read_back_over_the_cache_and_its_tables():
    start, starts = torch.zeros(B + 1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    rest = [*_cache(), start, starts]
    for i in range(len(rest)):
        for o in range(2):
            r, out = list(rest), [_half(3, HKV, 128), _half(3, HKV, 128)]
            r[i], out[o] = _over(rest[i], out[o].shape)
            _refused(ops.kv_gather, *r[:6], 8, r[6], 3, starts=r[7], out=tuple(out))


def test_tree_attention_output_and_workspace():
    rest = [_half(B, N, HQ, 128), _half(B, N, HKV, 128), _half(B, N, HKV, 128), torch.zeros(B, N, dtype=torch.int64), *_cache(),
            torch.zeros(B, dtype=torch.int32)]
    call = lambda r, **kw: _refused(ops.kv_tree_attention, *r[:10], 8, num_nodes=r[10], **kw)   # noqa: E731
    for i in range(len(rest)):
        r = list(rest)
        r[i], out = _over(rest[i], (B, N, HQ, 128))
        call(r, out=out)
        r[i], ws = _over(rest[i], (1 << 20,), torch.uint8)
        call(r, workspace=ws)
    out, ws = _over(_half(B, N, HQ, 128), (1 << 20,), torch.uint8)
    call(rest, out=out, workspace=ws)


def test_verification_workspace():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)   # noqa: E731
    p, t, u, up, q, n = torch.zeros(B, N, 30), i32(B, N), torch.zeros(B, N), i32(B, N), torch.zeros(B, N, 30), i32(B)
    for chain in (True, False):
        rest = [p, t, u, None if chain else up, q if chain else None, n]
        for i, x in enumerate(rest):
            if x is not None:
                r = list(rest)
                r[i], ws = _over(x, (1 << 16,), torch.uint8)
                _refused(ops.verify_drafts, *r, workspace=ws)


@pytest.mark.parametrize("bits", [8, 4])
def test_append_onto_its_own_inputs(bits):
    """Placeholder addresses, never used: caches and scales against each other and against every input, by one byte of overlap
    at either end.  Apart (with no GPU present) the call gets as far as its launch."""
    lib = _lib.load()
    codes, scales, rows = PAGES * HKV * 16 * 16 * bits, PAGES * HKV * 2, B * 3
    size = dict(kc=codes, vc=codes, ks=scales, vs=scales, k=rows * HKV * 128 * 2, v=rows * HKV * 128 * 2, table=B * WIDTH * 4,
                lens=B * 4, start=B * 4 + 4, select=B * 3 * 4, counts=B * 4)
    at = {name: (i + 1) << 20 for i, name in enumerate(size)}

    def append(**kw):
        a = {**at, **kw}
        return lib.exl3_kv_append(a["k"], a["v"], 0, HKV * 128, HKV * 128, rows, a["start"], 0, a["select"], a["counts"], 3,
                                  a["kc"], a["vc"], a["ks"], a["vs"], PAGES, a["table"], WIDTH, a["lens"], B, HKV, 128, 16,
                                  bits, None)

    for name in ("kc", "vc", "ks", "vs"):
        for other in size:
            if other == name:
                continue
            step = 16 if name in ("kc", "vc", "k", "v") or other in ("kc", "vc", "k", "v") else 2
            for where in (at[other] + size[other] - step, at[other] - size[name] + step):
                if name in ("kc", "vc") and where % 16:
                    where += 16 - where % 16 if where < at[other] else -(where % 16)
                assert append(**{name: where}) == _lib.EXL3_ERR_INVALID
                assert "overlap" in lib.exl3_last_error().decode(), (name, other, lib.exl3_last_error())
    if not torch.cuda.is_available():
        assert append() == _lib.EXL3_ERR_HIP
        assert append(vc=at["kc"] + codes) == _lib.EXL3_ERR_HIP
