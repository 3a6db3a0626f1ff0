"""Greedy decoding with drafted token trees over a bounded KV cache.

The reference generates one token per step (src/model.c:943-954).  `generate`
feeds every slot a tree of guesses in one pass (DeviceModel.tree_forward), keeps
the path the model agrees with, and returns the ids of the plain greedy loop (up
to near ties: passes of other sizes sum in another order).  Whether that is
faster goes by the tree and the guesses: on the 32-layer STQ1_0 model a plain
token takes 0.81 ms, a pass of one node 1.76, of 16 nodes 8.9, of 32 to 64 nodes
3.3, so a pass of 32 or more should yield over four tokens.  With a budget, the cache of every
slot is cut back to its heaviest rows as it grows (DeviceModel.tree_evict).

    python -m hymt2_b200.draft MODEL.gguf --budget 512
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np


@dataclass
class PromptLookup:
    """Guesses by repetition: the continuations that followed earlier occurrences of the text's last `match` ids (then
    of fewer), merged into one tree of up to `nodes` nodes, the latest occurrences first."""
    nodes: int = 16
    match: int = 3
    depth: int = 8

    def __call__(self, ids: list[int]) -> tuple[list[int], list[int]]:
        tokens, parents, child = [int(ids[-1])], [-1], {}
        for m in range(min(self.match, len(ids) - 1), 0, -1):
            tail = ids[-m:]
            for at in range(len(ids) - m - 1, -1, -1):
                if ids[at:at + m] != tail:
                    continue
                node = 0
                for t in ids[at + m:at + m + self.depth]:
                    nxt = child.get((node, int(t)))
                    if nxt is None:
                        if len(tokens) >= self.nodes:
                            return tokens, parents
                        nxt = child[(node, int(t))] = len(tokens)
                        tokens.append(int(t))
                        parents.append(node)
                    node = nxt
        return tokens, parents


def _shares(want: list[int], most: int) -> list[int]:
    """Of `most` nodes, what each gets: an equal share, or what it wants where that is less, and what those leave in turn."""
    got = [min(w, most // len(want)) for w in want]
    left = most - sum(got)
    for i, w in enumerate(want):
        more = min(w - got[i], left)
        got[i] += more
        left -= more
    return got


@dataclass
class DraftStats:
    passes: int = 0
    nodes: int = 0
    tokens: int = 0
    evictions: int = 0
    rows: list[int] = field(default_factory=list)


def generate(dm, prompts, max_new: int, draft=None, stop=(), budget: int = 0, sinks: int = 4, recent: int = 32,
             window: int = 16, slack: int = 32):
    """Greedy ids for a few prompts at once, one slot each (dm.batch_prepare and dm.tree_prepare done before).

    draft(ids) -> (tokens, parents): a tree whose node 0 is ids[-1].  budget > 0 bounds every slot's cache: it is cut
    back to budget rows when it has over `slack` more, or more and no room for the next tree (a cut copies what stays).
    The last `window` prompt tokens then go through tree passes, so that their queries' weights are counted.  The slots
    share a pass's tokens; one that has no row or position left ends early, with the ids so far.  Returns (ids per
    prompt, DraftStats)."""
    draft = draft or PromptLookup()
    stop, n = set(int(t) for t in stop), len(prompts)
    ids = [[int(t) for t in p] for p in prompts]
    stats = DraftStats()
    # the prompts but their last tokens; with a budget the window is fed below, as a given chain
    keep = [len(p) - 1 - (min(window, len(p) - 1) if budget else 0) for p in ids]
    flat = [(t, s, i) for s, p in enumerate(ids) for i, t in enumerate(p[:keep[s]])]
    for a in range(0, len(flat), dm.batch_tokens):
        part = flat[a:a + dm.batch_tokens]
        dm.batch_forward([t for t, _, _ in part], [s for _, s, _ in part], [i for _, _, i in part], [])
    for s in range(n):
        dm.tree_open(s, keep[s])
    if budget:
        chain = {s: p[keep[s]:-1] for s, p in enumerate(ids)}
        while any(chain.values()):  # in passes of as many nodes as a tree and a pass may have
            part, left = {}, min(dm.batch_tokens, dm.batch_out)
            for s, c in chain.items():
                m = min(len(c), dm.tree_nodes, left)
                if m > 0:
                    part[s] = c[:m], list(range(-1, m - 1))
                    chain[s], left = c[m:], left - m
            dm.tree_forward(part, dm.batch_slots, forced=part)
    out: list[list[int]] = [[] for _ in range(n)]
    live = [s for s in range(n) if max_new > 0]
    while live:
        drafts = {s: draft(ids[s] + out[s]) for s in live}
        state = {s: dm.tree_state(s) for s in live}
        if budget and any(state[s][0] > min(budget + slack, max(budget, dm.batch_ctx - min(len(drafts[s][0]), dm.tree_nodes)))
                          for s in live):
            dm.tree_evict(budget, sinks, recent)
            stats.evictions += 1
            state = {s: dm.tree_state(s) for s in live}
        # as many nodes as the slot and the context have room for
        room = {s: min(dm.tree_nodes, dm.batch_ctx - state[s][0], dm.ctx - state[s][1]) for s in live}
        live = [s for s in live if room[s] > 0]
        if not live:
            break
        share = _shares([min(room[s], len(drafts[s][0])) for s in live], min(dm.batch_tokens, dm.batch_out))
        trees = {s: (drafts[s][0][:m], drafts[s][1][:m]) for s, m in zip(live, share) if m > 0}
        live = [s for s in live if s not in trees] + list(trees)  # who had to wait is first in the next pass
        got = dm.tree_forward(trees, dm.batch_slots)
        stats.passes += 1
        stats.nodes += sum(len(t) for t, _ in trees.values())
        for s in trees:
            path, nxt = got[s]
            for t in path[1:] + [nxt]:
                if t in stop:
                    live.remove(s)
                    break
                out[s].append(t)
                if len(out[s]) == max_new:
                    live.remove(s)
                    break
    stats.tokens = sum(len(o) for o in out)
    stats.rows = [dm.tree_state(s)[0] for s in range(n)]
    return out, stats


def main(argv=None) -> None:
    import argparse
    import time

    from .device import DeviceModel
    ap = argparse.ArgumentParser(description="greedy decoding with drafted token trees on a synthetic prompt")
    ap.add_argument("model")
    ap.add_argument("--prompt", type=int, default=256, help="prompt tokens (a phrase repeated with changes)")
    ap.add_argument("--new", type=int, default=128)
    ap.add_argument("--nodes", type=int, default=16)
    ap.add_argument("--budget", type=int, default=0, help="most cached rows (0: no bound)")
    a = ap.parse_args(argv)
    ctx = a.prompt + a.new + 64
    dm = DeviceModel(a.model, ctx=ctx)
    dm.batch_prepare(slots=1, slot_ctx=ctx, max_tokens=256, max_out=64)
    dm.tree_prepare(64, weights=a.budget > 0)
    rng = np.random.default_rng(7)
    phrase = rng.integers(0, min(1000, dm.vocab_out), 24)
    prompt = np.where(rng.random(a.prompt) < 0.05, rng.integers(0, min(1000, dm.vocab_out), a.prompt), np.resize(phrase, a.prompt))
    generate(dm, [prompt[:64].tolist()], 2, PromptLookup(nodes=a.nodes), budget=a.budget)  # first uses lay weights out
    t = time.perf_counter()
    out, st = generate(dm, [prompt.tolist()], a.new, PromptLookup(nodes=a.nodes), budget=a.budget)
    dt = time.perf_counter() - t
    print(f"{st.tokens} tokens in {st.passes} passes ({st.nodes / max(st.passes, 1):.1f} nodes a pass), {st.tokens / dt:.0f} tok/s, "
          f"{st.rows[0]} cached rows, {st.evictions} evictions")
    dm.close()


if __name__ == "__main__":
    main()
