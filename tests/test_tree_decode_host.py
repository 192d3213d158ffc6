"""Host side of decoding with drafted tokens: the tree of guesses, its masks and the accepted path."""
import numpy as np

from mini_llama_b200.tree_decode import accepted_path, draft_tree, tree_mask


def test_draft_tree_shares_beginnings_and_stays_in_size():
    history = [5, 6, 7, 8, 1, 5, 6, 7, 9, 2, 5, 6]
    tokens, parents = draft_tree(history, 6)
    assert tokens[0] == 6 and parents[0] == -1 and len(tokens) <= 6
    paths = []
    for i in range(len(tokens)):
        p, n = [], i
        while n >= 0:
            p.append(tokens[n])
            n = parents[n]
        paths.append(p[::-1])
    assert [6, 7] in paths and [6, 7, 9] in paths and [6, 7, 8] in paths
    assert sum(p == [6, 7] for p in paths) == 1  # both occurrences share it
    assert all(p < i for i, p in enumerate(parents))
    assert draft_tree([3], 8) == ([3], [-1])
    assert len(draft_tree(list(range(4)) * 30, 64)[0]) <= 64


def test_tree_mask_is_the_ancestors():
    parents = [-1, 0, 0, 1, 3] + [4] * 70
    m = tree_mask(parents)
    assert m.shape == (75, 2) and m.dtype == np.uint64
    for i in range(75):
        want, n = 0, i
        while n >= 0:
            want |= 1 << n
            n = parents[n]
        assert int(m[i, 0]) | (int(m[i, 1]) << 64) == want


def test_accepted_path():
    tokens, parents = [4, 7, 8, 9], [-1, 0, 0, 2]
    assert accepted_path(tokens, parents, [8, 0, 9, 3]) == ([0, 2, 3], 3)
    assert accepted_path(tokens, parents, [5, 0, 0, 0]) == ([0], 5)
