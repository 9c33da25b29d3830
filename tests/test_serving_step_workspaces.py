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


@pytest.mark.parametrize("vocab", [1, 5, 8, 70, 777, 1023, 1024, 1025, 4097, 32003, 131072, 1 << 20])
def test_sampling_workspace_is_one_slice_of_rows(lib, vocab):
    """Rows are worked on 512 at a time: more of them take no more, and a workspace for the most serves fewer."""
    rows = [*range(1, 530), 1030, 16384, 65536, 100000, (1 << 26) - 1]
    sizes = [lib.exl3_sample_workspace_bytes(r, vocab) for r in rows]
    assert sizes == sorted(sizes)
    assert sizes[-1] == sizes[511]
    chunks = -(-vocab // 4096)
    # a row's state (256 bytes at most), its list of 8192 numbers of 8 bytes, and 256 bins of 12 bytes and some sums a chunk
    assert sizes[-1] <= 512 * (256 + 8192 * 8 + chunks * (256 * 12 + 64))
