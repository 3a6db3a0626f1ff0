"""Guesses for drafted trees (CPU)."""
from hymt2_b200.draft import PromptLookup


def test_lookup_follows_the_latest_repetition_first():
    tokens, parents = PromptLookup(nodes=8, match=2, depth=3)([1, 2, 3, 4, 9, 1, 2, 7, 8, 1, 2])
    assert tokens[0] == 2 and parents[0] == -1
    assert tokens[1:4] == [7, 8, 1] and parents[1:4] == [0, 1, 2]   # after the later "1 2"
    assert tokens[4:7] == [3, 4, 9] and parents[4:7] == [0, 4, 5]   # after the earlier one
    assert len(tokens) <= 8 and all(p < i for i, p in enumerate(parents))


def test_lookup_shares_prefixes_and_keeps_its_bounds():
    ids = [5, 6, 7, 5, 6, 8, 5, 6, 7, 5, 6]
    tokens, parents = PromptLookup(nodes=64, match=2, depth=2)(ids)
    kids = [t for t, p in zip(tokens, parents) if p == 0]
    assert sorted(kids) == sorted(set(kids))                        # no child twice
    assert PromptLookup(nodes=1)(ids) == ([6], [-1])
    assert PromptLookup()([3]) == ([3], [-1])
    assert PromptLookup()([3, 4]) == ([4], [-1])                    # nothing to go by
    tokens, _ = PromptLookup(nodes=4, match=1, depth=8)([1] * 50)
    assert len(tokens) == 4
