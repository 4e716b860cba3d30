"""GPU: the factor of the head norm, 1 / sqrt(mean(x²) + eps), where everything beside it is exact: elements are powers of two, head_dim
is one, there is no rotation, weights are 1. The definition rounds it once; a correction by a few roundings of the last bit of a
value that is itself off by an ulp leaves it within 0.51 units of the last place."""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [32, 64, 128, 256, 512])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -20])
def test_norm_factor(hip, dim, eps):
    import torch
    from qxotic_amd.jam import QkSpec
    print("norm factor", dim, eps, file=sys.stderr, flush=True)
    r = np.random.default_rng(dim)
    n, heads = 700, 4
    # at most 9 + 8 bits of a sum of squares above its last, and eps within 24 of its first
    x = (2.0 ** r.integers(-3, 2, (n, heads, dim)) * r.choice([-1, 1], (n, heads, dim))).astype(np.float32)
    one = torch.ones(dim, device="cuda")
    xd = torch.from_numpy(x.reshape(n, -1)).cuda()
    out = torch.empty_like(xd)
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    s = QkSpec(q_heads=heads, kv_heads=0, head_dim=dim, rope_dim=0, eps=eps, scale=1.0, q_weight=one.data_ptr(), k_weight=None)
    assert hip.qk_norm_rope(s, xd.data_ptr(), heads * dim, out.data_ptr(), heads * dim, None, 0, None, 0, pos.data_ptr(), n) == 0, hip.last_error()
    hip.synchronize()
    got = out.cpu().numpy().reshape(x.shape)
    mean = (x.astype(np.float64) ** 2).mean(-1, keepdims=True)
    v = (mean.astype(np.float32) + np.float32(eps)).astype(np.float64)   # exact but for eps's rounding, which the definition in f32 has
    want = np.abs(x) / np.sqrt(v)
    off = np.abs(np.abs(got.astype(np.float64)) - want) / np.spacing(want.astype(np.float32)).astype(np.float64)
    assert np.array_equal(np.sign(got), np.sign(x)) and float(off.max()) <= 0.51, float(off.max())


def test_norm_of_zeros_and_infinities(hip):
    """A head of zeros is zeros with eps above 0; one whose squares pass f32 is 0 where it is finite, as x · rsqrt(Inf)."""
    import torch
    from qxotic_amd.jam import QkSpec
    x = np.zeros((3, 64), np.float32)
    x[1] = 1e25
    x[2] = 1e-30
    one = torch.ones(64, device="cuda")
    xd, out, pos = torch.from_numpy(x).cuda(), torch.full((3, 64), -5.0, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    s = QkSpec(q_heads=1, kv_heads=0, head_dim=64, rope_dim=0, eps=1e-6, scale=1.0, q_weight=one.data_ptr(), k_weight=None)
    assert hip.qk_norm_rope(s, xd.data_ptr(), 64, out.data_ptr(), 64, None, 0, None, 0, pos.data_ptr(), 3) == 0
    hip.synchronize()
    got = out.cpu().numpy()
    assert (got[0] == 0).all() and (got[1] == 0).all()
    assert (np.abs(got[2] / np.float32(1e-27) - 1) < 2.0 ** -20).all()
