"""Where the ragged form of ops.kv_append finds the sequence and the page of a place, restated: ascending row starts reach every
page of every sequence once; row starts that do not ascend never lead before a page table's beginning."""
import numpy as np
import pytest
import torch

PAGE = 16


def _place(row_start, batch, at):
    lo, n = 0, batch
    while True:
        step = (n + 63) // 64
        before = sum(1 for lane in range(64) if lane * step < n
                     and row_start[min(lo + lane * step, batch)] // PAGE + 2 * (lo + lane * step) <= at)
        if before == 0:
            return -1
        lo += (before - 1) * step
        if step == 1:
            return lo
        n = min(step, n - (before - 1) * step)


def _pages(row_start, lens, rows):
    """(sequence, logical page) of every place that writes."""
    batch, found = len(lens), []
    for at in range(rows // PAGE + 2 * batch):
        b = _place(row_start, batch, at)
        if b < 0:
            continue
        pg = at - row_start[b] // PAGE - 2 * b
        count = row_start[b + 1] - row_start[b]
        if count <= 0 or pg < 0 or pg > count // PAGE + 1:
            continue
        lp = lens[b] // PAGE + pg
        if lp * PAGE < lens[b] + count:
            found.append((b, lp))
    return found


@pytest.mark.parametrize("batch", [1, 2, 7, 65, 200])
def test_ascending_row_starts_reach_every_page_once(batch):
    rng = np.random.default_rng(batch)
    for _ in range(8):
        new, lens = rng.integers(0, 60, batch), rng.integers(0, 100, batch)
        start = [int(x) for x in np.concatenate([[0], np.cumsum(new)])]
        want = [(b, lp) for b in range(batch) for lp in range(lens[b] // PAGE, -(-(lens[b] + new[b]) // PAGE)) if new[b]]
        assert sorted(_pages(start, [int(n) for n in lens], start[-1])) == want


def test_other_row_starts_stay_inside_the_table():
    rng = np.random.default_rng(0)
    before = 0
    for _ in range(300):
        batch = int(rng.integers(1, 80))
        start = [int(x) for x in rng.integers(0, 400, batch + 1)]
        assert all(lp >= 0 for _, lp in _pages(start, [0] * batch, 400))
        for at in range(400 // PAGE + 2 * batch):
            b = _place(start, batch, at)
            before += b >= 0 and start[b + 1] > start[b] and at - start[b] // PAGE - 2 * b < 0
    assert before > 0   # such places exist: they are the ones left out


@pytest.mark.gpu
def test_row_starts_that_do_not_ascend_write_no_other_page():
    from test_gpu_attn_step import _ops, _random_cache, _t, _table
    rng = np.random.default_rng(1)
    for start in ([100, 200, 0, 50], [300, 310, 20, 90, 80, 250]):
        B, rows, Hkv, width, P = len(start) - 1, 400, 2, 30, 200
        cache, table = _random_cache(rng, P, Hkv, 8), _table(rng, B, width, P)
        lens = rng.integers(0, 40, B)
        got = [_t(c) for c in cache]
        x = _t(rng.standard_normal((rows, Hkv, 128))).half()
        _ops().kv_append(x, x, *got, _t(table), _t(np.int32(lens)), 8, row_start=_t(np.int32(start)))
        torch.cuda.synchronize()
        own = [table[b, lens[b] // PAGE:-(-(lens[b] + max(start[b + 1] - start[b], 0)) // PAGE)] for b in range(B)]
        others = np.setdiff1d(np.arange(P), np.concatenate(own))
        for g, c in zip(got, cache):
            assert np.array_equal(g.cpu().numpy()[others].view(np.uint8), c[others].view(np.uint8))
