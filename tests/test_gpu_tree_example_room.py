"""GPU: examples/tree_step.py where pages run out: prompts that find no room are an error, a conversation whose tree finds none stays as it was."""
import sys

import pytest
from test_gpu_tree_example_streams import PROMPTS, chain, decoder

pytestmark = pytest.mark.gpu


def test_prompts_without_room():
    import tree_step as X
    print("prompts without room", file=sys.stderr, flush=True)
    jam, d = decoder(5)   # the prompts take 2, 1 and 3 pages of 16
    try:
        with pytest.raises(RuntimeError, match="out of pages"):
            X.Trees(d, 5, PROMPTS)
    finally:
        d.close()
        jam.close()


def test_a_step_without_room():
    """The conversations that fit go on; the one that does not, and the one behind it that would grow, stay as they were, and go on where a later
    step has room for them."""
    import torch
    import tree_step as X
    print("a step without room", file=sys.stderr, flush=True)

    def steps(pages, drafts):
        jam, d = decoder(pages)
        try:
            t = X.Trees(d, pages, PROMPTS)
            out, logits = [], []
            for s in drafts:
                a, b = t.step(s)
                out.append(a)
                logits.append(b.cpu())
            held = t.held.cpu().tolist()
            table, free = t.table.cpu(), t.free.cpu().tolist()[:int(t.n_free)]
            assert sorted(free + [int(p) for i, h in enumerate(held) for p in table[i, :h]]) == list(range(pages))
            return out, logits, t.lens.cpu().tolist()
        finally:
            d.close()
            jam.close()

    wide = chain([5, 6, 7], ((1,), tuple(range(100, 120)), (3,)))
    narrow = chain([5, 6, 7], ((1,), (2,), (3,)))
    out, logits, lens = steps(6, [wide, narrow])   # 6 pages are held; the second's tree takes one more
    assert out[0][0][0] and out[0][1:] == [([], 6), ([], 7)]
    assert all(p for p, _ in out[1]) and lens == [len(p) + len(out[0][i][0]) + len(out[1][i][0]) for i, p in enumerate(PROMPTS)]
    # the same with room: the conversations that were refused have their second step's logits as their first
    want = steps(40, [narrow])[1][0]
    assert torch.isfinite(logits[1]).all()
    assert (logits[1][2:] - want[2:]).abs().max() <= 0.05 * want[2:].abs().max()   # as in test_gpu_decode_example.py
