"""draft.generate within the bounds of an engine (CPU: a stand-in that refuses what hyc_tree_forward refuses)."""
import pytest

from hymt2_b200.draft import PromptLookup, generate


class Engine:
    """Rows and positions as the engine counts them; the token after t at position p is (31 t + 7 p) mod 89."""

    def __init__(self, slots=1, slot_ctx=64, max_tokens=64, max_out=None, nodes=16, ctx=1 << 20):
        self.batch_slots, self.batch_ctx, self.batch_tokens, self.tree_nodes, self.ctx = slots, slot_ctx, max_tokens, nodes, ctx
        self.batch_out = max_out or max_tokens
        self.rows, self.pos, self.cuts, self.counted = [0] * slots, [0] * slots, 0, [0] * slots

    @staticmethod
    def after(t, p):
        return (31 * t + 7 * p) % 89

    def batch_forward(self, tokens, slots, positions, out_rows):
        assert len(tokens) <= self.batch_tokens and all(p < self.batch_ctx for p in positions)

    def tree_open(self, s, rows):
        assert 0 <= rows <= self.batch_ctx
        self.rows[s] = self.pos[s] = rows
        self.counted[s] = 0

    def tree_state(self, s):
        return self.rows[s], self.pos[s], None

    def tree_evict(self, budget, sinks, recent):
        assert sinks + recent <= budget <= self.batch_ctx
        self.cuts += 1
        self.rows = [min(r, budget) for r in self.rows]

    def tree_forward(self, trees, slots, forced=None):
        assert slots == self.batch_slots and 1 <= sum(len(t) for t, _ in trees.values()) <= min(self.batch_tokens, self.batch_out)
        got = {}
        for s, (tk, pa) in trees.items():
            assert 1 <= len(tk) == len(pa) <= self.tree_nodes
            assert self.rows[s] + len(tk) <= self.batch_ctx, "a tree does not fit its slot's context"
            assert pa[0] == -1 and all(0 <= p < i for i, p in enumerate(pa) if i)
            pos = [self.pos[s]]
            for p in pa[1:]:
                pos.append(pos[p] + 1)
            assert max(pos) < self.ctx, "a position is past the prepared context"
            if forced and s in forced:
                path = list(range(len(tk)))
                assert list(pa) == list(range(-1, len(tk) - 1))
            else:
                path = [0]
                while True:
                    want = self.after(tk[path[-1]], pos[path[-1]])
                    kid = [i for i in range(len(tk)) if pa[i] == path[-1] and tk[i] == want]
                    if not kid:
                        break
                    path.append(kid[0])
            self.rows[s] += len(path)
            self.pos[s] += len(path)
            self.counted[s] += len(path)
            got[s] = [tk[i] for i in path], self.after(tk[path[-1]], pos[path[-1]])
        return got


def plain(prompt, n):
    ids = list(prompt)
    for _ in range(n):
        ids.append(Engine.after(ids[-1], len(ids) - 1))
    return ids[len(prompt):]


def oracle_draft(wrong=0):
    """The right continuation, up to 12 tokens, with `wrong` wrong siblings before each."""
    def draft(ids):
        tokens, parents, node, t, p = [ids[-1]], [-1], 0, ids[-1], len(ids) - 1
        for _ in range(12):
            t, p = Engine.after(t, p), p + 1
            tokens += [(t + 1 + i) % 89 for i in range(wrong)] + [t]
            parents += [node] * (wrong + 1)
            node = len(tokens) - 1
        return tokens, parents
    return draft


PROMPT = [int(x) for x in "31415926535897932384626433832795028841971693993751"]
DRAFTS = [PromptLookup(nodes=16), oracle_draft(), oracle_draft(1), lambda ids: ([ids[-1]], [-1])]


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("slot_ctx,budget,slack", [(64, 60, 32), (64, 63, 32), (64, 40, 32), (64, 62, 0), (70, 50, 10), (64, 40, 200)])
def test_a_cache_sized_just_above_its_bound(slot_ctx, budget, slack, draft):
    """The cut comes before the slot is full, whatever the slack."""
    dm = Engine(slot_ctx=slot_ctx)
    out, st = generate(dm, [PROMPT], 100, draft, budget=budget, recent=8, slack=slack)
    assert out == [plain(PROMPT, 100)] and dm.cuts == st.evictions >= 1


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("kw,most", [(dict(slot_ctx=64), 64), (dict(slot_ctx=128, ctx=70), 70)])
def test_a_slot_without_room_ends_early(kw, most, draft):
    """No bound, and the slot's rows or the positions run out: the ids so far, as the plain loop has them."""
    dm = Engine(slots=2, **kw)
    out, _ = generate(dm, [PROMPT, PROMPT[:20]], 100, draft)
    want = [plain(PROMPT, 100), plain(PROMPT[:20], 100)]
    assert [len(o) for o in out] == [most - 50 + 1, most - 20 + 1]   # the last row's token too
    assert all(o == w[:len(o)] for o, w in zip(out, want))


@pytest.mark.parametrize("nodes", [1, 3, 8, 15])
@pytest.mark.parametrize("window", [0, 1, 7, 16, 100])
def test_a_window_wider_than_a_tree(nodes, window):
    """The prompt's last tokens go in as chains of as many nodes as a tree has, each query counted once."""
    dm = Engine(nodes=nodes)
    out, _ = generate(dm, [PROMPT], 5, budget=60, window=window)
    assert out == [plain(PROMPT, 5)]
    assert dm.counted[0] == min(window, len(PROMPT) - 1) + dm.pos[0] - (len(PROMPT) - 1)


@pytest.mark.parametrize("max_tokens,max_out", [(64, 64), (64, 17), (6, 6)])
def test_windows_of_more_tokens_than_a_pass(max_tokens, max_out):
    dm = Engine(slots=6, max_tokens=max_tokens, max_out=max_out)
    prompts = [PROMPT[i:] for i in range(6)]
    out, _ = generate(dm, prompts, 1, lambda ids: ([ids[-1]], [-1]), budget=60)
    assert out == [plain(p, 1) for p in prompts]
    assert all(c >= 16 for c in dm.counted)


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("slots,max_tokens,max_out", [(16, 128, 128), (5, 64, 20), (6, 6, 6), (6, 5, 5), (6, 64, 4), (3, 1, 1)])
def test_trees_of_more_nodes_than_a_pass(slots, max_tokens, max_out, draft):
    """The live slots share a pass's tokens; where there are fewer tokens than slots, slots take turns."""
    dm = Engine(slots=slots, max_tokens=max_tokens, max_out=max_out, slot_ctx=128)
    prompts = [PROMPT[i:] for i in range(slots)]
    out, st = generate(dm, prompts, 20, draft, budget=100)
    assert out == [plain(p, 20) for p in prompts]
    assert st.nodes <= st.passes * min(max_tokens, max_out)
