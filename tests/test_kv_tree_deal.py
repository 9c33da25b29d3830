"""How the shared form of the draft-tree attention deals a unit's groups of 16 rows to the 8 waves of a workgroup, restated (the
tile's size is read back through the workspace size): every live row belongs to one wave, whatever the node counts are."""
import pytest

from trellis_serve_amd import _lib

WAVES, MOST, SPLIT_GROUPS = 8, 3, 6


def _plan(nodes, per_kv):
    """(rows of a unit, most groups of a wave), None where the split form serves."""
    groups = -(-nodes * per_kv // 16)
    if groups <= SPLIT_GROUPS:
        return None
    tiles = -(-groups // (WAVES * MOST))
    per_tile = -(-groups // tiles)
    return 16 * per_tile, -(-per_tile // WAVES)


def _deal(rg, groups, w):
    """(first group, groups that the code runs) of wave w.  There is code for RG and RG - 1 groups."""
    least = max(rg - 1, 1)
    each, more = divmod(groups, WAVES)
    if each >= least:
        first, mine = w * each + min(w, more), each + (w < more)
    else:
        first = min(w * least, groups)
        mine = min(groups - first, least)
    return first, rg if mine == rg else rg - 1 if rg > 1 and mine > 0 else 0


@pytest.mark.parametrize("per_kv", range(1, 17))
def test_every_live_row_is_stored_by_one_wave(per_kv):
    size = _lib.load().exl3_kv_tree_workspace_bytes
    for nodes in range(1, 65):
        plan = _plan(nodes, per_kv)
        if plan is None:
            continue
        tile, rg = plan
        assert size(1, nodes, per_kv, 1, 1 << 20) == 256 * 2 * tile * (128 + 2) * 4
        assert 1 <= rg <= MOST
        for live in range(nodes + 1):
            owners = [0] * (live * per_kv)
            for first in range(0, live * per_kv, tile):
                rows = min(live * per_kv - first, tile)
                for w in range(WAVES):
                    at, runs = _deal(rg, -(-rows // 16), w)
                    row0 = first + 16 * at
                    for r in range(row0, min(row0 + 16 * runs, live * per_kv)):   # rows past the live ones are not stored
                        owners[r] += 1
            assert owners == [1] * (live * per_kv), (nodes, live)
