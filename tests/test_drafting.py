"""The host side of decoding with drafted tokens: guesses from a text, how a tree attention is cut, what is refused before a launch."""
import random

import pytest
import torch

from mini_llm_b200 import ops
from mini_llm_b200.engine.drafting import DraftRunner, PromptLookup
from mini_llm_b200.engine.runner import StepError


def paths(tokens, parents):
    """Every root-to-leaf path of a tree, as tuples of tokens behind the root."""
    kids = {i: [j for j, p in enumerate(parents) if p == i] for i in range(len(tokens))}
    def walk(i):
        return [(tokens[i],) + rest for k in [kids[i]] for rest in ([p for j in k for p in walk(j)] or [()])]
    return sorted(p[1:] for p in walk(0))


def test_a_lookup_follows_the_longest_suffix_and_the_latest_occurrence_first():
    text = [1, 2, 3, 4, 5, 9, 2, 3, 7, 7, 8, 1, 2, 3]
    tokens, parents = PromptLookup(ngram=3, branches=2).draft(text, rows=16, depth=4)
    assert tokens[0] == 3 and parents[0] == -1
    assert paths(tokens, parents) == [(4, 5, 9), (7, 7, 8)]       # 1 2 3 -> 4 5 9, then 2 3 -> 7 7 8
    tokens, parents = PromptLookup(ngram=3, branches=1).draft(text, rows=16, depth=4)
    assert paths(tokens, parents) == [(4, 5, 9)]
    tokens, parents = PromptLookup(ngram=1, branches=2).draft(text, rows=16, depth=3)
    assert paths(tokens, parents) == [(4, 5), (7, 7)]


def test_continuations_that_begin_alike_share_rows():
    text = [5, 6, 7, 8, 5, 6, 7, 9, 5]
    tokens, parents = PromptLookup(ngram=1, branches=4).draft(text, rows=16, depth=4)
    assert paths(tokens, parents) == [(6, 7, 8), (6, 7, 9)] and len(tokens) == 5


@pytest.mark.parametrize("rows,depth", [(1, 1), (2, 2), (3, 8), (8, 2), (16, 8), (64, 5)])
def test_trees_stay_within_their_rows_and_depth(rows, depth):
    rng = random.Random(rows * 100 + depth)
    for _ in range(60):
        text = [rng.randrange(4) for _ in range(rng.randrange(1, 60))]
        tokens, parents = PromptLookup(rng.randrange(1, 5), rng.randrange(1, 6)).draft(text, rows, depth)
        assert 1 <= len(tokens) == len(parents) <= rows and tokens[0] == text[-1] and parents[0] == -1
        level = []
        for i, p in enumerate(parents):
            assert -1 <= p < i and (p >= 0 or i == 0)
            level.append(0 if p < 0 else level[p] + 1)
        assert max(level) < depth
        seen = {(p, t) for p, t in zip(parents, tokens)}
        assert len(seen) == len(tokens)                     # no two children of a row with the same token


def test_a_text_that_repeats_nothing_drafts_nothing():
    assert PromptLookup().draft([1, 2, 3, 4], 16, 8) == ([4], [-1])
    assert PromptLookup().draft([7], 16, 8) == ([7], [-1])


def test_lookup_refusals():
    for kw in (dict(ngram=0), dict(branches=0)):
        with pytest.raises(ValueError):
            PromptLookup(**kw)


# ------------------------------------------------------------------------------------------------ how the work is cut
def test_a_plan_for_every_shape():
    """Every plan names a kernel that exists, and a few requests with long texts share their keys out."""
    for f32 in (False, True):
        for dim in (16, 48, 64, 80, 128, 256):
            for boxes in (False, True):
                for S in (1, 3, 64, 1000):
                    for heads, kv in ((1, 1), (12, 12), (12, 4), (32, 8), (16, 1)):
                        for nodes in (1, 8, 17, 64, 256):
                            for length in (0, 1, 500, 100000):
                                tile, rows, blocks, least, wide = ops.tree_plan(f32, S, heads, kv, dim, nodes, length, boxes, 148)
                                v = ops._tree_variant(f32, dim, tile, wide)
                                assert v is not None and rows == nodes * (heads // kv) and least >= 1
                                assert blocks in (0, 148 * v[0])
                                assert tile <= 64 or (not f32 and boxes and dim <= 128)
    assert ops.tree_plan(False, 1, 8, 2, 128, 8, 30000, True, 148)[2] > 0
    assert ops.tree_plan(False, 64, 12, 12, 64, 8, 500, True, 148)[2] == 0


def test_slices_of_logits():
    for rows in (1, 8, 300, 5000):
        for vocab in (1, 2047, 50257, 200000):
            n = ops.accept_slices(rows, vocab)
            assert 1 <= n <= max(1, -(-vocab // 2048)) and (n == 1 or rows * n <= 4736 + rows)


def test_tensors_that_are_not_on_the_device_are_refused():
    t = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.draft_tables(t, t, t, t, t, 16, block_table=t, slot_mapping=t, positions=t, token_seq=t, ctx_len=t),
                 lambda: ops.tree_attention(t, t, t, t, t, t, t, t, num_heads=1, num_kv_heads=1, head_dim=16, scale=1.0),
                 lambda: ops.accept_drafts(t, t, t, t, chosen=t, path=t, accepted=t, next_token=t, new_lengths=t),
                 lambda: ops.keep_accepted(t, t, t, t, t), lambda: ops.draft_tables(None, t, t, t, t, 16, block_table=t, slot_mapping=t,
                                                                                    positions=t, token_seq=t, ctx_len=t)):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()


# ------------------------------------------------------------------------------------------------ which models take drafts
def fake_runner(mixers, window=None, states=()):
    from types import SimpleNamespace as N
    return N(model=N(layers=[N(mixer=m) for m in mixers]), spec=None,
             cache=N(groups=[N(need=N(window=window, chunk=None))], state_layers=list(states)))


def test_models_that_take_no_drafts_are_refused():
    class Tree:
        takes_trees = True
    class Scan:
        pass
    DraftRunner(fake_runner([Tree()]))
    for bad in (fake_runner([Tree(), Scan()]), fake_runner([Tree()], window=64), fake_runner([Tree()], states=[1])):
        with pytest.raises(StepError, match="drafts need"):
            DraftRunner(bad)
    for rows, depth in ((0, 1), (4, 5), (257, 8), (4, 0)):
        with pytest.raises(ValueError, match="depth"):
            DraftRunner(fake_runner([Tree()]), rows, depth)
