"""GPU: examples/decode_step.py, the operators together. A prefix that conversations share and one that each keeps in pages of its own
give the same tokens, and logits that agree to the accuracy of f32 sums carried through two layers whose projections quantise their
inputs to 8 bits (an input next to a border of two codes may take the other: 1 / 127 of a block's largest, in a few of the 256 to 512
terms of a product)."""
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


@pytest.mark.parametrize("kind", ["F16", "Q8_0", "Q4_0"])
def test_shared_and_private_prefixes_agree(kind):
    import decode_step as E
    import torch
    from qxotic_amd.jam import JAM, HipJAM
    print("decode example", kind, file=sys.stderr, flush=True)
    rng = np.random.default_rng(3)
    prefix = rng.integers(0, E.VOCAB, 141).tolist()
    prompts = [rng.integers(0, E.VOCAB, n).tolist() for n in (1, 40, 17)]
    numbers = [(rng.random(3) * (1 - 2.0 ** -24)).astype(np.float32) for _ in range(4)]
    seen = []
    jam = HipJAM()
    try:
        for shared in (True, False):
            d = E.Decoder(jam, pages=64, cache_type=getattr(JAM, kind), seed=5)
            try:
                c = E.Conversations(d, prefix, prompts, shared)
                logits, tokens = [c.logits.cpu().numpy()], []
                for u in numbers:
                    tokens.append(c.step(torch.from_numpy(u).cuda()))
                    logits.append(c.logits.cpu().numpy())
                seen.append((tokens, logits))
            finally:
                d.close()
    finally:
        jam.close()
    assert seen[0][0] == seen[1][0]
    for a, b in zip(seen[0][1], seen[1][1]):
        assert np.isfinite(a).all() and np.abs(a - b).max() <= 0.05 * np.abs(b).max()
