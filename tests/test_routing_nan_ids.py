"""The softmax selection on NaN logits, lane by lane: a token all of whose logits are NaN gets an id outside [0, E) from its second
slot on, and one NaN among them can do it, so whoever takes the selection's ids as indices has to check them first (the dispatch and the layer for a few tokens do,
test_gpu_few_nan.py)."""
import math

import pytest

EMPTY = 0x7FFFFFFF


def take(mine, other):
    """argmax_take: the larger value, equal values to the lower index; EMPTY marks no candidate."""
    (bv, be), (ov, oe) = mine, other
    return other if oe != EMPTY and (be == EMPTY or ov > bv or (ov == bv and oe < be)) else mine


def select(logits, k):
    """The ids of a token's k slots: 16 lanes, one expert each, exchange by xor; lane j keeps selection j."""
    E = len(logits)
    taken = [False] * 16
    ids = []
    for slot in range(k):
        lane = [(logits[e], e) if e < E and not taken[e] else (0.0, EMPTY) for e in range(16)]
        for step in (8, 4, 2, 1):
            lane = [take(lane[i], lane[i ^ step]) for i in range(16)]
        for e in range(16):
            taken[e] |= lane[e][1] == e
        ids.append(lane[slot][1])
    return ids


@pytest.mark.parametrize("E,k", [(16, 2), (10, 3), (3, 3), (2, 2)])
def test_nan_token_leaves_slots_without_an_expert(E, k):
    ids = select([math.nan] * E, k)
    assert ids == [0] + [EMPTY] * (k - 1)
    named = [e if 0 <= e < E else -1 for e in ids]  # what may be grouped
    assert named == [0] + [-1] * (k - 1)


@pytest.mark.parametrize("E,k", [(16, 4), (10, 3), (3, 3), (1, 1)])
def test_tokens_without_nan_get_experts(E, k):
    finite = [math.sin(7.0 * e + E) for e in range(E)]
    assert select(finite, k) == sorted(range(E), key=lambda e: (-finite[e], e))[:k]
    assert all(0 <= e < E for e in select([-math.inf] * E, k))


@pytest.mark.parametrize("E,k", [(16, 4), (10, 3), (3, 3), (2, 2)])
def test_one_nan_expert(E, k):
    """The first slot names an expert; a later one does, or is empty (the lane of the NaN takes itself while the others choose)."""
    finite = [math.sin(7.0 * e + E) for e in range(E)]
    every = [select(finite[:bad] + [math.nan] + finite[bad + 1:], k) for bad in range(E)]
    assert all(0 <= ids[0] < E and all(0 <= e < E or e == EMPTY for e in ids) for ids in every)
    if E == k:
        assert any(EMPTY in ids for ids in every)
