"""Drafted tokens on the card (include/maplemoe.h, Part 3), at the ends of what the header allows."""
import numpy as np
import pytest

from draft_ref import tree, tree_plan
from test_gpu_drafts import run_tree_plan

pytestmark = pytest.mark.gpu
LEAST = -2 ** 31


@pytest.mark.parametrize("sizes,words", [([130], 3), ([512, 200, 65], 8), ([256] * 3, 4)])
@pytest.mark.parametrize("none", [LEAST, LEAST + 1, LEAST + 63, LEAST + 64, LEAST + 447, LEAST + 448, -64, -65])
def test_parents_near_the_smallest_number(sizes, words, none):
    """nodes of every word that follow nobody, whatever negative number says so: the first one of a word, one in its middle, the last one"""
    print(f"\n  {sizes} parent={none}", flush=True)
    rng = np.random.default_rng(len(sizes) + words)
    qstart = np.concatenate([[0], np.cumsum(sizes)])
    parent = np.concatenate([tree(rng, n, 9) for n in sizes]).astype(np.int64)
    for t0, n in zip(qstart, sizes):
        for i in (0, 3, 64, 70, 127, 128, 191, 192, 255, 448, 449, 511):
            if i < n:
                parent[t0 + i] = none
    length = np.array(sizes) + rng.integers(0, 1 << 29, len(sizes))
    got, want = run_tree_plan(qstart, length, parent, words, len(parent)), tree_plan(qstart, length, parent, words, len(parent))
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
