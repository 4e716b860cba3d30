"""GPU: examples/tree_step.py where streams are busy. A step's own work is in the order of the decoder's stream, behind what the caller has
queued, so neither what that stream nor what the caller's still has to do changes a result."""
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
PROMPTS = [list(range(3, 21)), [7, 5, 900], list(range(40, 80))]
BUSY = 200_000_000   # clock cycles, a tenth of a second and more: longer than the host takes to queue a step


def decoder(pages):
    import decode_step as E
    from qxotic_amd.jam import HipJAM
    jam = HipJAM()
    return jam, E.Decoder(jam, pages=pages, seed=5)


def chain(roots, more=((), (), ())):
    return [([r, *m], [-1, *range(len(m))]) for r, m in zip(roots, more)]


def run(busy):
    """Logits of the prompts and of a step; `busy`: which stream has work queued before each of them."""
    import torch
    import tree_step as X
    jam, d = decoder(40)

    def wait():
        if busy != "no":
            with torch.cuda.stream(d.stream if busy == "decoder" else torch.cuda.current_stream()):
                torch.cuda._sleep(BUSY)

    try:
        torch.cuda.synchronize()
        wait()
        t = X.Trees(d, 40, PROMPTS)
        first = t.logits.clone()
        wait()
        picked = torch.arange(7, dtype=torch.int32, device="cuda") * 0 - 1   # on the caller's stream
        out, logits = t.step(chain([5, 6, 7], ((1, 2), (), (3, 4))), picked=picked)
        second = logits.clone()
        torch.cuda.synchronize()
        return first.cpu(), second.cpu(), out, t.lens.cpu().tolist()
    finally:
        d.close()
        jam.close()


@pytest.mark.parametrize("busy", ["decoder", "caller"])
def test_busy_streams(busy):
    import torch
    print("busy streams", busy, file=sys.stderr, flush=True)
    want, got = run("no"), run(busy)
    assert torch.isfinite(want[0]).all() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert got[2:] == want[2:] and want[2] == [([0], -1)] * 3 and want[3] == [len(p) + 1 for p in PROMPTS]
