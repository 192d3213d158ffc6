"""Decoding with drafted tokens on the GPU: the same greedy text as without drafts, and as the decode session
(whose cache is fp32); the cache holds what plain decoding leaves there."""
import numpy as np
import pytest

from mini_llama_b200 import capi, synth
from mini_llama_b200.device import Model, Session
from mini_llama_b200.tree_decode import SPECS, TreeDecoder

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny(mlb, gpu):
    m = Model(mlb, gpu, SPECS["tiny"])
    m.synthesize(seed=7, tied=True)
    yield m
    m.close()


@pytest.mark.parametrize("cache", [capi.F32, capi.Q8_0, capi.Q4_0], ids=["f32", "q8_0", "q4_0"])
def test_drafts_leave_the_text_unchanged(mlb, gpu, tiny, cache):
    prompt = synth.tokens(40, 11, SPECS["tiny"]["vocab_size"])
    plain = TreeDecoder(tiny, cache, 16)
    text, passes = plain.generate(prompt, 96, 1)
    assert passes == 96
    drafted = TreeDecoder(tiny, cache, 16)
    again, fewer = drafted.generate(prompt, 96, 12)
    assert again == text
    assert fewer < passes  # a random model falls into repetition, which the drafts find
    if cache == capi.F32:
        s = Session(tiny)
        try:
            assert list(s.generate(prompt, 96)) == text
        finally:
            s.close()


def test_kept_rows_are_in_place(mlb, gpu, tiny):
    """After keeping a path that skips nodes, the cache holds the path's rows at the next slots: attention from
    there equals that over a cache that was fed the path as a chain."""
    tokens, parents, path = [3, 9, 14, 20, 33], [-1, 0, 0, 2, 2], [0, 2, 4]
    a, b = TreeDecoder(tiny, capi.Q8_0, 8), TreeDecoder(tiny, capi.Q8_0, 8)
    for d in (a, b):
        d.forward([1, 2, 5], [-1, 0, 1])
        d.len = 3
    tree = a.forward(tokens, parents)
    chain = b.forward([tokens[i] for i in path], [-1, 0, 1])
    assert [tree[i] for i in path] == chain
    a.keep(path)
    b.len += 3
    assert a.len == b.len == 6
    one, two = (d.forward([7], [-1]) for d in (a, b))
    la, lb = (d.logits.download()[0] for d in (a, b))
    assert one == two and np.abs(la - lb).max() <= 1e-4 * np.abs(lb).max()
