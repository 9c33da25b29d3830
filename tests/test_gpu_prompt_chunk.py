"""A prompt's chunk as the integration notes write it: ragged rows appended, then the whole sequences read back by the lengths
after the append."""
import numpy as np
import pytest
import torch

import attn_step_ref as ref
from test_gpu_attn_step import PAGE, _half, _ops, _random_cache, _t, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
def test_chunk_appended_and_sequences_read_back(bits):
    rng = np.random.default_rng(bits)
    lens, new, Hkv = [0, 35, 7, 16], [20, 0, 64, 1], 3
    width = max(-(-(a + n) // PAGE) for a, n in zip(lens, new)) + 1
    cache, table = _random_cache(rng, 4 * width, Hkv, bits), _table(rng, 4, width, 4 * width)
    (k, k64), (v, v64) = (_half(rng.standard_normal((sum(new), Hkv, 128)), "bf16") for _ in range(2))
    start = np.concatenate([[0], np.cumsum(new)])
    got, page_table, seq_lens, row_start = [_t(c) for c in cache], _t(table), _t(np.int32(lens)), _t(np.int32(start))
    _ops().kv_append(k, v, *got, page_table, seq_lens, bits, row_start=row_start, max_new=max(new))
    after = seq_lens + row_start.diff()
    assert after.dtype == torch.int32
    total = [a + n for a, n in zip(lens, new)]
    back_start, back_rows = _t(np.int32(np.concatenate([[0], np.cumsum(total)]))), sum(total)
    back = _ops().kv_gather(*got, page_table, after, bits, back_start, back_rows)
    rows_of = [list(range(start[b], start[b + 1])) for b in range(4)]
    for x, codes, scales, out in ((k64, cache[0], cache[2], back[0]), (v64, cache[1], cache[3], back[1])):
        codes, scales = ref.append(x, codes, scales, table, lens, bits, rows_of)
        want = np.concatenate([ref.values(codes, scales, table[b], total[b], bits) for b in range(4)])
        assert torch.equal(out.cpu(), torch.from_numpy(want).half())
