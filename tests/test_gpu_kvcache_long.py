"""GPU: the cache read back where a thread takes eight tokens, the call's length cut into eight strides (from 4194304 pieces of four
elements on): numbers of tokens that are no multiple of eight, slots outside the cache in the last stride, unaligned rows."""
import sys

import numpy as np
import pytest

from oracle import decode as D

pytestmark = pytest.mark.gpu
NAMES = {D.F16: "F16", D.Q8_0: "Q8_0", D.Q4_0: "Q4_0"}


def values(kind, buf, slots, kv, dim, page, pages):
    """What the slots of a buffer stand for, [n, kv, dim] f32."""
    row = {D.F16: 2 * dim, D.Q8_0: dim, D.Q4_0: dim // 2}[kind]
    cut = pages * kv * page * row
    codes = buf[:cut].reshape(pages, kv, page, row)[slots // page, :, slots % page]
    if kind == D.F16:
        return codes.view(np.float16).astype(np.float32)
    scales = buf[cut:].view(np.float16).reshape(pages, kv, page, dim // 32)[slots // page, :, slots % page].astype(np.float32)
    if kind == D.Q8_0:
        c = codes.view(np.int8).reshape(*scales.shape, 32)
    else:
        b = codes.reshape(*scales.shape, 16)
        c = np.concatenate([b & 15, b >> 4], -1).astype(np.int8) - 8
    return (c * scales[..., None]).astype(np.float16).astype(np.float32).reshape(len(slots), kv, dim)   # at most 19 bits, then rounded once


@pytest.mark.parametrize("kind", [D.F16, D.Q8_0, D.Q4_0])
@pytest.mark.parametrize("n,kv,dim,page", [(16384, 8, 128, 16), (16389, 8, 128, 16), (16391, 8, 128, 48), (87389, 2, 96, 64)])
def test_read_many(hip, kind, n, kv, dim, page):
    import torch
    from qxotic_amd.jam import KvCache
    print("read many", NAMES[kind], n, kv, dim, page, file=sys.stderr, flush=True)
    assert n * kv * dim // 4 >= 4194304
    pages = -(-n // page) + 3
    r = np.random.default_rng(n + kind)
    c = KvCache(type=kind, kv_heads=kv, head_dim=dim, page_tokens=page, n_pages=pages)
    size = hip.kv_cache_bytes(c)
    rows = pages * page * kv
    bufs = []
    for _ in range(2):
        if kind == D.F16:
            b = r.standard_normal(rows * dim, dtype=np.float32).astype(np.float16).view(np.uint8)
        else:   # any codes, scales of either sign
            b = np.concatenate([r.integers(0, 256, rows * (dim if kind == D.Q8_0 else dim // 2), dtype=np.uint8),
                                (0.1 * r.standard_normal(rows * dim // 32, dtype=np.float32)).astype(np.float16).view(np.uint8)])
        assert b.size == size
        bufs.append(b)
    slots = r.permutation(pages * page)[:n].astype(np.int32)
    bad = np.array([0, n // 8, n // 2, n - n // 9, n - 4, n - 2, n - 1])   # in the first stride and the last ones
    slots[bad] = [-1, pages * page, -(1 << 31), (1 << 31) - 1, pages * page + 5, -7, -1]
    live = (slots >= 0) & (slots < pages * page)
    want = [values(kind, b, np.where(live, slots, 0), kv, dim, page, pages) for b in bufs]
    for w in want:
        w[~live] = 0
    dev = [torch.from_numpy(b).cuda() for b in bufs]
    c.k, c.v = dev[0].data_ptr(), dev[1].data_ptr()
    sd = torch.from_numpy(slots).cuda()
    for odd in (0, 1):   # rows at 16-byte and at 4-byte alignment
        ld = kv * dim + odd
        outs = [torch.full((n + 1, ld), -5.0, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        assert hip.kv_read(c, sd.data_ptr(), n, outs[0].data_ptr(), ld, outs[1].data_ptr(), ld) == 0, hip.last_error()
        hip.synchronize()
        for o, w in zip(outs, want):
            got = o.cpu().numpy()
            assert np.array_equal(got[:n, :kv * dim].reshape(n, kv, dim), w)
            assert (got[n] == -5.0).all() and (got[:, kv * dim:] == -5.0).all()
    one = torch.full((n, kv * dim), -5.0, device="cuda")
    torch.cuda.synchronize()
    assert hip.kv_read(c, sd.data_ptr(), n, None, 0, one.data_ptr(), kv * dim) == 0
    hip.synchronize()
    assert np.array_equal(one.cpu().numpy().reshape(n, kv, dim), want[1])
