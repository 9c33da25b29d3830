"""`max_new` of ops.kv_append bounds every form of the call, not the ragged one alone."""
import numpy as np
import pytest
import torch

import attn_step_ref as ref
from trellis_serve_amd import ops


def _cache():
    codes = lambda: torch.zeros(8, 2, 16, 128, dtype=torch.int8)   # noqa: E731
    return [codes(), codes(), *(torch.ones(8, 2, dtype=torch.float16) for _ in range(2)),
            torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)]


def test_a_bound_below_the_selection_is_refused():
    k, select = torch.zeros(2, 5, 2, 128, dtype=torch.float16), torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="max_new = 2"):
        ops.kv_append(k, k, *_cache(), 8, select=select, max_new=2)
    with pytest.raises(ValueError, match="max_new = -1"):
        ops.kv_append(k, k, *_cache(), 8, max_new=-1)
    with pytest.raises(ValueError, match="cuda"):   # past the checks of arguments
        ops.kv_append(k, k, *_cache(), 8, select=select, max_new=3)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("max_new", [0, 1, 3, 20, 21, 99])
def test_a_bound_below_the_rows_of_a_sequence(bits, max_new):
    from test_gpu_attn_step import PAGE, _check_append, _half, _random_cache, _t, _table
    rng = np.random.default_rng(max_new + bits)
    lens, n, Hkv = [0, 13, 30], 21, 2
    width = -(-(max(lens) + n) // PAGE)
    cache, table = _random_cache(rng, 3 * width, Hkv, bits), _table(rng, 3, width, 3 * width)
    k, k64 = _half(rng.standard_normal((3, n, Hkv, 128)), "fp16")
    v, v64 = _half(rng.standard_normal((3, n, Hkv, 128)), "fp16")
    got = [_t(c) for c in cache]
    ops.kv_append(k, v, *got, _t(table), _t(np.int32(lens)), bits, max_new=max_new)
    rows_of = [[b * n + i for i in range(min(n, max_new))] for b in range(3)]
    want = [ref.append(x.reshape(3 * n, Hkv, 128), c, s, table, lens, bits, rows_of)
            for x, c, s in ((k64, cache[0], cache[2]), (v64, cache[1], cache[3]))]
    _check_append(cache, got, *want)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [5, 2 ** 31, 2 ** 32, 2 ** 32 + 2, 2 ** 63 - 1])
def test_a_bound_past_32_bits_is_no_bound(max_new):
    from test_gpu_attn_step import _check_append, _half, _random_cache, _t, _table
    rng = np.random.default_rng(5)
    lens, start = [3, 30], [0, 5, 9]
    cache, table = _random_cache(rng, 8, 2, 8), _table(rng, 2, 4, 8)
    x, x64 = _half(rng.standard_normal((9, 2, 128)), "fp16")
    got = [_t(c) for c in cache]
    ops.kv_append(x, x, *got, _t(table), _t(np.int32(lens)), 8, row_start=_t(np.int32(start)), max_new=max_new)
    rows_of = [list(range(start[b], start[b + 1])) for b in range(2)]
    _check_append(cache, got, *[ref.append(x64, c, s, table, lens, 8, rows_of) for c, s in ((cache[0], cache[2]),
                                                                                         (cache[1], cache[3]))])
