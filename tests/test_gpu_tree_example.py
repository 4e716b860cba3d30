"""GPU: examples/tree_step.py, the operators of a step with drafted trees together. The drafted trees hold the tokens that a plain decoder of the
same weights takes, scattered among others, and those are what is picked: so all of them are accepted, and their logits, of every step,
agree with the plain decoder's to the accuracy that test_gpu_decode_example.py derives (projections that quantise their inputs to 8 bits:
an input next to a border of two codes may take the other). Entries that were moved, pages given back and taken again are read by the steps behind."""
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


def scatter(r, chain, vocab, more):
    """A tree that holds `chain` from its root on, and `more` other tokens hung up anywhere; the chain's places."""
    tokens, parents, places = [chain[0]], [-1], [0]
    rest = list(chain[1:])
    extra = more
    while rest or extra:
        if extra and (not rest or r.random() < 0.6):
            at = int(r.integers(0, len(tokens)))
            tokens.append(int(r.integers(0, vocab)) + vocab)   # never what is picked
            parents.append(at)
            extra -= 1
        else:
            tokens.append(rest.pop(0))
            parents.append(places[-1])
            places.append(len(tokens) - 1)
    return tokens, parents, places


@pytest.mark.parametrize("kind", ["F16", "Q8_0", "Q4_0"])
def test_trees_follow_a_plain_decoder(kind):
    import decode_step as E
    import torch
    import tree_step as X
    from qxotic_amd.jam import JAM, HipJAM
    print("tree example", kind, file=sys.stderr, flush=True)
    r = np.random.default_rng(4)
    prompts = [r.integers(0, E.VOCAB, n).tolist() for n in (1, 40, 17)]
    plain, jam = HipJAM(), HipJAM()
    try:
        a, b = E.Decoder(plain, pages=64, cache_type=getattr(JAM, kind), seed=5), E.Decoder(jam, pages=40, cache_type=getattr(JAM, kind), seed=5)
        try:
            chats = E.Conversations(a, [], prompts, shared=False)
            trees = X.Trees(b, 40, prompts)
            b.stream.synchronize()
            assert int(trees.n_free) == 40 - sum(-(-len(p) // E.PAGE) for p in prompts)

            def near(x, y):
                x, y = x.cpu().numpy(), y.cpu().numpy()
                assert np.isfinite(x).all() and np.abs(x - y).max() <= 0.05 * np.abs(y).max()

            near(trees.logits, chats.logits)
            for step in range(5):
                lengths = r.integers(1, 8, 3)
                chains, seen = [[] for _ in prompts], [[] for _ in prompts]
                for k in range(max(lengths)):   # the plain decoder's tokens, and its logits after each
                    nxt = chats.logits.argmax(-1).tolist()
                    new = [[t] if k < lengths[i] else [] for i, t in enumerate(nxt)]
                    live = [i for i in range(3) if new[i]]
                    keep = chats.logits
                    for i in live:
                        chats.own[i] += 1
                        chats._grow(chats.pages[i], chats.own[i])
                    got = chats._call([new[i] for i in live], [chats.pages[i] for i in live], [chats.own[i] for i in live], 0, [])
                    chats.logits = keep.clone()
                    for row, i in enumerate(live):
                        chains[i].append(nxt[i])
                        seen[i].append(got[row])
                        chats.logits[i] = got[row]
                torch.cuda.synchronize()
                drafts, places, picked = [], [], []
                for i, c in enumerate(chains):
                    tokens, parents, at = scatter(r, c, E.VOCAB, int(r.integers(0, 30)))
                    picks = [-1] * len(tokens)   # the token after each of the chain's, and what no token is
                    for k, p in enumerate(at[:-1]):
                        picks[p] = c[k + 1]
                    picks[at[-1]] = 7
                    drafts.append(([t % E.VOCAB for t in tokens], parents))
                    # an unlucky neighbour must not be accepted for the chain's: none of the others carries a picked token
                    for k, t in enumerate(tokens):
                        if t >= E.VOCAB and drafts[-1][0][k] in [picks[p] for p in at]:
                            drafts[-1][0][k] = next(v for v in range(E.VOCAB) if v not in c and v != 7)
                    places.append(at)
                    picked += picks
                out, logits = trees.step(drafts, picked=torch.tensor(picked, dtype=torch.int32).cuda())
                b.stream.synchronize()
                off = np.cumsum([0] + [len(t) for t, _ in drafts])
                for i, (path, after) in enumerate(out):
                    assert path == places[i] and after == 7
                    near(logits[(torch.tensor(path) + off[i]).cuda()], torch.stack(seen[i]))
                assert trees.lens.cpu().tolist() == chats.own and trees.held.cpu().tolist() == [-(-v // E.PAGE) for v in chats.own]
                assert int(trees.n_free) == 40 - sum(-(-v // E.PAGE) for v in chats.own)
                table, free = trees.table.cpu().numpy(), trees.free.cpu().tolist()[:int(trees.n_free)]
                held = [int(p) for i, h in enumerate(trees.held.cpu().tolist()) for p in table[i, :h]]
                assert sorted(held + free) == list(range(40))   # every page is held once or free
        finally:
            a.close()
            b.close()
    finally:
        plain.close()
        jam.close()


def test_example_runs():
    import tree_step as X
    X.main(steps=3)
