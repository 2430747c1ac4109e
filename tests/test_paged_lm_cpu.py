"""The drafted tree's depths and mask words."""
import numpy as np
import pytest

import paged_lm as PL
import paged_model as M


@pytest.mark.parametrize("n", [1, 5, 31, 32, 33, 70])
def test_tree_words(n):
    rng = np.random.default_rng(n)
    parents = [int(rng.integers(-1, j)) for j in range(n)]
    depth, words = PL.tree(parents)
    seen = M.tree_mask(parents)
    assert words.dtype == np.int32 and np.array_equal(words, M.pack_mask(seen, -(-n // 32)))
    assert depth == [int(x) - 1 for x in seen.sum(1)]


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 0, -2]])
def test_tree_refusals(parents):
    with pytest.raises(ValueError):
        PL.tree(parents)
