"""The operators around the attention and at the ends of a serving step at batches of every size: workspaces made for the largest."""
import numpy as np
import pytest
import torch

from test_gpu_serving_step import _check_sparse, _i, _n, _ops, _rows_case, _t

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
