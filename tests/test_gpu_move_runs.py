"""GPU: jamhip_kv_move with more workgroups than go out in one launch (2^23), most of them without entries."""
import sys

import pytest

from oracle import decode as D

pytestmark = pytest.mark.gpu


def test_move_in_several_launches(hip):
    import torch
    from qxotic_amd.jam import KvCache
    print("move in several launches", file=sys.stderr, flush=True)
    groups, layers, slots, row = 1 << 20, 9, 64, 128
    bufs = [torch.randint(0, 256, (slots * row,), dtype=torch.uint8, device="cuda") for _ in range(2 * layers)]
    caches = (KvCache * layers)(*(KvCache(type=D.F16, kv_heads=1, head_dim=64, page_tokens=16, n_pages=4, k=bufs[2 * i].data_ptr(),
                                          v=bufs[2 * i + 1].data_ptr()) for i in range(layers)))
    # an entry in each of these groups: on both sides of the launches' border, (1 << 23) / 9, and at the ends
    at = [0, 1, 932066, 932067, 932068, 932069, groups - 2, groups - 1]
    counts = torch.zeros(groups + 1, dtype=torch.int64)
    counts[[g + 1 for g in at]] = 1
    off = counts.cumsum(0).int().cuda()
    src = torch.arange(len(at), dtype=torch.int32, device="cuda")
    dst = src + 32
    want = [b.clone() for b in bufs]
    for b in want:
        v = b.view(slots, row)
        v[32:32 + len(at)] = v[:len(at)].clone()
    torch.cuda.synchronize()
    assert hip.kv_move(caches, layers, off.data_ptr(), groups, src.data_ptr(), dst.data_ptr(), len(at)) == 0, hip.last_error()
    hip.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(bufs, want))
