"""Host side of decoding with drafted tokens: the tree of guesses, its masks and the accepted path."""
import numpy as np
import pytest

from mini_llama_b200 import capi
from mini_llama_b200.tree_decode import SPECS, TreeDecoder, accepted_path, draft_tree, tree_mask


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


class HostLib:
    """Stands in for the library: notes the calls' names, hands out addresses."""

    def __init__(self):
        self.names, self.at = [], 1 << 20

    def malloc(self, device, nbytes):
        self.at += nbytes + 256
        return self.at

    def free(self, device, ptr):
        pass

    def call(self, name, *args):
        self.names.append(name)


class HostModel:
    device, spec = 0, SPECS["tiny"]

    def __init__(self):
        self.lib = HostLib()

    def weight(self, layer, kind):
        return 1 << 16, 0


@pytest.mark.parametrize("nodes,parents", [(17, 17), (0, 0), (5, 4)])
def test_a_pass_of_too_many_nodes_is_refused(nodes, parents):
    """The device buffers hold max_rows rows: more are refused before anything is copied or launched."""
    d = TreeDecoder(HostModel(), capi.Q8_0, 16)
    before = len(d.lib.names)
    with pytest.raises(ValueError, match="nodes"):
        d.forward([1] * nodes, list(range(-1, parents - 1)))
    assert len(d.lib.names) == before


def test_a_pass_beyond_the_cache_is_refused():
    d = TreeDecoder(HostModel(), capi.Q8_0, 16)
    d.len = SPECS["tiny"]["max_seq_len"] - 3
    before = len(d.lib.names)
    with pytest.raises(ValueError, match="slots"):
        d.forward([1, 2, 3, 4], [-1, 0, 1, 2])
    assert len(d.lib.names) == before


@pytest.mark.parametrize("prompt,n_new,draft,kept", [([1, 2], 4, 17, 0), ([], 4, 4, 0), ([1] * 300, 200, 16, 0),
                                                     ([1, 2], 100, 8, 405)])
def test_generation_that_does_not_fit_is_refused(prompt, n_new, draft, kept):
    """More drafted nodes than rows, no prompt, or more tokens than the cache has slots left."""
    d = TreeDecoder(HostModel(), capi.Q8_0, 16)
    d.len = kept
    before = len(d.lib.names)
    with pytest.raises(ValueError):
        d.generate(prompt, n_new, draft)
    assert len(d.lib.names) == before


class CountingDecoder(TreeDecoder):
    """The model's choice after a token is a fixed function of it, in a cycle of five, so that drafts are accepted."""

    def forward(self, tokens, parents):
        assert self.len + len(tokens) <= self.model.spec["max_seq_len"] and len(tokens) <= self.max_rows
        return [(t + 1) % 5 for t in tokens]


@pytest.mark.parametrize("draft", [1, 3, 8, 16])
@pytest.mark.parametrize("n_new", [1, 6, 23, 24, 25])
def test_the_cache_holds_what_was_returned(draft, n_new):
    """A pass may accept more tokens than are asked for: those are not kept, and a further call goes on from the text."""
    d = CountingDecoder(HostModel(), capi.Q8_0, 16)
    prompt = [0, 1, 2, 3, 4] * 3
    text, _ = d.generate(prompt, n_new, draft)
    assert text == [i % 5 for i in range(n_new)]
    assert d.len == len(prompt) + n_new - 1
    more, _ = d.generate(text[-1:], 7, draft)
    assert more == [(n_new + i) % 5 for i in range(7)]
    assert d.len == len(prompt) + n_new + 6
