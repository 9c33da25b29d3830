"""Workspaces of the operators around the attention and at the ends of a serving step: one for the most rows serves fewer."""
import pytest

from trellis_serve_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _parts(rows, hkv, top):
    """List entries of a workgroup's share, four waves a workgroup: (workgroups of a row and kv head)."""
    most = min(64, -(-top // 4))
    parts = max(1, min(most, -(-1024 // (rows * hkv))))
    per = 4 * -(-top // (4 * parts))
    return -(-top // per)


@pytest.mark.parametrize("hq,hkv", [(40, 8), (1, 1), (32, 2), (16, 16), (1500, 1500), (14, 7)])
@pytest.mark.parametrize("top", [1, 4, 5, 64, 256, 300, 100000])
def test_sparse_attention_workspace_for_the_most_rows_serves_fewer(lib, hq, hkv, top):
    rows = [*range(1, 300), 1023, 1024, 5000, 65535]
    sizes = [lib.exl3_kv_sparse_workspace_bytes(r, hq, hkv, top) for r in rows]
    assert sizes == sorted(sizes)
    for r, size in zip(rows, sizes):
        parts = _parts(r, hkv, top)
        used = 0 if parts == 1 else r * hq * parts * 130 * 4   # 128 values, a maximum and a sum of each part
        assert size >= used
        if r == 1:
            assert size <= hq * min(64, -(-top // 4)) * 130 * 4
    largest = max(r * hq * _parts(r, hkv, top) * 130 * 4 for r in rows)
    assert sizes[-1] <= 2 * largest


@pytest.mark.parametrize("hkv,width", [(1, 30), (8, 9000), (2, 65)])
def test_choice_workspace_for_the_most_rows_serves_fewer(lib, hkv, width):
    sizes = [lib.exl3_kv_select_workspace_bytes(r, hkv, width) for r in range(1, 300)]
    assert sizes == sorted(sizes)
