"""Step plans whose ring has fewer places than there are pages: what a step gives up goes to places of what it takes."""
import numpy as np
import pytest

import serving_step_ref as ref
from test_gpu_serving_step import PAGE, _check_plan, _i, _n, _ops

pytestmark = pytest.mark.gpu


def test_given_up_pages_take_the_places_of_taken_ones():
    table = np.array([[-1, -1, -1], [20, 21, 22]])
    want = _check_plan(table, np.array([0, 48]), np.array([32, -32]), np.array([10, 11, 12, 13]), np.array([0, 4]), 32)
    assert want[6].tolist() == [160 + i for i in range(16)] + [176 + i for i in range(16)]


def _full_ring(seed, B, longest, most):
    """A ring without a free place; every second sequence grows, the others give up at most as many pages as are taken."""
    rng = np.random.default_rng(seed)
    W = -(-(longest + most) // PAGE) + 1
    lens, new = rng.integers(0, longest + 1, B), rng.integers(1, most + 1, B)
    order = rng.permutation(B)
    pages = lambda n: -(-n // PAGE)   # noqa: E731
    taken = sum(pages(int(lens[b] + new[b])) - pages(int(lens[b])) for b in order[::2])
    left = taken
    for b in order[1::2]:
        keep = max(0, int(lens[b]) - int(new[b]))
        give = pages(int(lens[b])) - pages(keep)
        new[b] = -new[b] if give <= left else 0
        left -= give if give <= left else 0
    P = taken + 3
    ids = rng.permutation(P + sum(pages(int(n)) for n in lens))
    table, at = np.full((B, W), -1), P
    for b, n in enumerate(lens):
        table[b, :pages(int(n))] = ids[at:at + pages(int(n))]
        at += pages(int(n))
    return table, lens, new, ids[:P], np.array([int(rng.integers(0, P)), P]), int(np.maximum(new, 0).sum())


@pytest.mark.parametrize("B,longest,most", [(2, 60, 40), (9, 300, 90), (200, 64, 9), (256, 500, 7), (257, 100, 40), (1030, 64, 30),
                                            (6, 3000, 2000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_full_ring(B, longest, most, in_place):
    table, lens, new, ring, state, rows = _full_ring(B, B, longest, most)
    _check_plan(table, lens, new, ring, state, rows, in_place)


@pytest.mark.parametrize("B,rows_behind", [(8, 0), (300, 0), (8, 3000)])
def test_given_up_pages_without_a_place_are_left_out(B, rows_behind):
    """The first ones, in order of the sequences, find places; the rest of the ring, and its state, stay whole."""
    rng = np.random.default_rng(B)
    W, P = 6, 2 * B
    ids = rng.permutation(P + 5 * B)
    table = np.full((B, W), -1)
    table[:, :5] = ids[P:].reshape(B, 5)
    lens = np.full(B, 80)
    new = np.where(np.arange(B) % 2, -64, 16)   # every second gives four pages up, the others take one
    head, live = int(rng.integers(0, P)), P - 1
    ring = ids[:P]
    rows = 16 * (B // 2) + rows_behind
    want = ref.plan(table, lens, new, ring, np.array([head, live]), rows)
    table_t, ring_t, state_t = _i(table), _i(ring), _i([head, live])
    got = _ops().kv_step_plan(table_t, _i(lens), _i(new), ring_t, state_t, rows)
    for g, w in zip(got, want[0]):
        assert np.array_equal(_n(g), w)
    assert np.array_equal(_n(table_t), want[1])
    taken = B // 2
    back = [p for b in range(1, B, 2) for p in table[b, 1:5]][:P - (live - taken)]
    assert _n(state_t).tolist() == [(head + taken) % P, P]
    at = (head + taken + np.arange(P)) % P
    still = [ring[(head + taken + j) % P] for j in range(live - taken)]
    assert _n(ring_t)[at].tolist() == still + back


def test_pages_circulate_through_a_short_ring():
    """Steps in a row, in place, in a ring that is full after most of them: no page is lost or doubled."""
    rng = np.random.default_rng(7)
    B, W, P = 300, 12, 400
    free = 380
    lens = np.full(B, 150)
    table = np.full((B, W), -1)
    ids = rng.permutation(B * 10 + free)
    table[:, :10] = ids[free:].reshape(B, 10)
    ring = np.full(P, -7)
    ring[:free] = ids[:free]
    table_t, ring_t, state_t, lens_t = _i(table), _i(ring), _i([0, free]), _i(lens)
    for _ in range(40):
        now, live = _n(lens_t), int(_n(state_t)[1])
        new = rng.integers(-60, 34, B)
        grow = np.maximum(new, 0)
        taken = ref.plan(_n(table_t), now, grow, _n(ring_t), _n(state_t), int(grow.sum()))[3]
        spare = P - int(taken[1])
        for b in rng.permutation(B):
            if new[b] < 0:
                give = -(-int(now[b]) // PAGE) - -(-max(0, int(now[b]) + int(new[b])) // PAGE)
                new[b] = 0 if give > spare else new[b]
                spare -= give if new[b] else 0
        rows = int(np.maximum(new, 0).sum())
        want, table_w, ring_w, state_w = ref.plan(_n(table_t), now, new, _n(ring_t), _n(state_t), rows)
        plan = _ops().kv_step_plan(table_t, lens_t, _i(new), ring_t, state_t, rows)
        assert all(np.array_equal(_n(g), w) for g, w in zip(plan, want))
        assert np.array_equal(_n(table_t), table_w) and np.array_equal(_n(ring_t), ring_w) and np.array_equal(_n(state_t), state_w)
        lens_t = plan.lens_after.clone()
        held = [int(p) for b, n in enumerate(_n(lens_t)) for p in _n(table_t)[b, :-(-int(n) // PAGE)]]
        head, live = _n(state_t)
        assert sorted(held + [int(_n(ring_t)[(head + j) % P]) for j in range(live)]) == list(range(B * 10 + free))


def test_an_empty_step_passes_the_state_on():
    state, state_out, ring = _i([3, 2]), _i([99, 98]), _i([5, 6, 7, 8])
    none = _i(np.zeros(0))
    plan = _ops().kv_step_plan(_i(np.zeros((0, 4))), none, none, ring, state, 0, state_out)
    assert _n(state_out).tolist() == _n(state).tolist() == [3, 2] and _n(ring).tolist() == [5, 6, 7, 8]
    assert plan.row_start.tolist() == [0] and plan.counts.numel() == plan.slots.numel() == 0
