"""A small decoder on one MI355X, every step of it through qxotic_amd.jam.HipJAM: quantised projections, head norm and rotation with
the keys and values written into a paged cache, attention over the cache with a prefix that several sequences share, gated
feed-forward, and the next token of each sequence.

    python examples/decode_step.py

The weights are random. One system prompt is read once into its own pages; three conversations of different lengths go on from it,
first their prompts in one ragged call, then a token each per step."""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from qxotic_amd import ggml                                                                  # noqa: E402
from qxotic_amd.jam import JAM, AttnBatch, HipJAM, KvCache, QkSpec, Sampling, Segment         # noqa: E402

HIDDEN, HEADS, KV, DIM, FFN, VOCAB, LAYERS, PAGE = 256, 8, 2, 64, 512, 1024, 2, 16


class Decoder:
    def __init__(self, jam: HipJAM, pages: int, cache_type: int = JAM.Q8_0, seed: int = 0):
        self.jam, self.stream = jam, torch.cuda.Stream()
        jam.set_stream(self.stream.cuda_stream)   # torch's work and the kernels in one order
        rng = np.random.default_rng(seed)
        self.weights = []

        def weight(rows, cols):
            w = ggml.quantize("Q8_0", (rng.standard_normal((rows, cols)) / np.sqrt(cols)).astype(np.float32))
            self._ok(jam.pin(Segment.of(w), JAM.Q8_0, cols, rows))
            self.weights.append(w)
            return w, rows, cols

        self.layers = [{"qkv": weight((HEADS + 2 * KV) * DIM, HIDDEN), "o": weight(HIDDEN, HEADS * DIM), "up": weight(2 * FFN, HIDDEN),
                        "down": weight(HIDDEN, FFN)} for _ in range(LAYERS)]
        self.head = weight(VOCAB, HIDDEN)
        with torch.cuda.stream(self.stream):
            g = torch.Generator(device="cuda").manual_seed(seed)
            self.embedding = torch.randn((VOCAB, HIDDEN), generator=g, device="cuda")
            self.norms = [1 + 0.1 * torch.randn(DIM, generator=g, device="cuda") for _ in range(2)]
            self.freq = torch.tensor([10000.0 ** (-2 * i / DIM) for i in range(DIM // 2)], device="cuda")
            self.spec = QkSpec(q_heads=HEADS, kv_heads=KV, head_dim=DIM, rope_dim=DIM, eps=1e-6, scale=1.0,
                               q_weight=self.norms[0].data_ptr(), k_weight=self.norms[1].data_ptr(), inv_freq=self.freq.data_ptr())
            self.caches, self.buffers = [], []
            for _ in range(LAYERS):
                c = KvCache(type=cache_type, kv_heads=KV, head_dim=DIM, page_tokens=PAGE, n_pages=pages)
                kv = [torch.zeros(jam.kv_cache_bytes(c), dtype=torch.uint8, device="cuda") for _ in range(2)]
                c.k, c.v = kv[0].data_ptr(), kv[1].data_ptr()
                self.caches.append(c)
                self.buffers.append(kv)

    def _ok(self, status):
        if status != JAM.OK:
            raise RuntimeError(self.jam.last_error())

    def _mm(self, weight, x, out=None):
        """x · Wᵀ; with `out` given the product is added to it."""
        w, rows, cols = weight
        c = torch.empty((x.shape[0], rows), device="cuda") if out is None else out
        self._ok(self.jam.mm_device_ex(Segment.of(w), JAM.Q8_0, cols, x.data_ptr(), cols, c.data_ptr(), rows, rows, x.shape[0], cols,
                                       None, out is not None))
        return c

    @staticmethod
    def _norm(x):
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).contiguous()

    def forward(self, tokens, positions, slots, batch: AttnBatch, masks=None):
        """Logits [n, VOCAB] of the call's tokens: int32 device tensors [n], the batch's arrays on the device too. masks int64 [n, words]: the
        tokens are drafted trees (examples/tree_step.py)."""
        with torch.cuda.stream(self.stream):
            n, q_dim, kv_dim = tokens.numel(), HEADS * DIM, KV * DIM
            x = self.embedding[tokens.long()].clone()
            for layer, cache in zip(self.layers, self.caches):
                qkv = self._mm(layer["qkv"], self._norm(x))
                ld, q = q_dim + 2 * kv_dim, qkv.data_ptr()
                k, v = q + 4 * q_dim, q + 4 * (q_dim + kv_dim)
                self._ok(self.jam.qkv_norm_rope_write(self.spec, cache, q, ld, q, ld, k, ld, v, ld, positions.data_ptr(), slots.data_ptr(), n))
                seen = torch.zeros((n, q_dim), device="cuda")
                if masks is None:
                    self._ok(self.jam.attn_shared_prefix(cache, batch, q, ld, HEADS, DIM ** -0.5, seen.data_ptr(), q_dim))
                else:
                    self._ok(self.jam.attn_tree(cache, batch, masks.data_ptr(), masks.shape[1], q, ld, HEADS, DIM ** -0.5, seen.data_ptr(), q_dim))
                self._mm(layer["o"], seen, x)
                up = self._mm(layer["up"], self._norm(x))
                self._ok(self.jam.glu_device(HipJAM.ACT_SWIGLU, up.data_ptr(), 2 * FFN, up.data_ptr() + 4 * FFN, 2 * FFN, n, FFN))
                self._mm(layer["down"], up[:, :FFN].contiguous(), x)
            return self._mm(self.head, self._norm(x))

    def sample(self, logits, temperature=0.8, top_k=40, top_p=0.95, min_p=0.02, u=None):
        """The next token of each row, int32 [rows]."""
        with torch.cuda.stream(self.stream):
            rows = logits.shape[0]
            full = lambda value, kind: torch.full((rows,), value, dtype=kind, device="cuda")   # noqa: E731
            arrays = [full(temperature, torch.float32), full(top_k, torch.int32), full(top_p, torch.float32), full(min_p, torch.float32), u]
            token = torch.empty(rows, dtype=torch.int32, device="cuda")
            self._ok(self.jam.sample(logits.data_ptr(), VOCAB, rows, VOCAB, Sampling(*(a.data_ptr() for a in arrays)), token.data_ptr()))
            return token

    def close(self):
        self.stream.synchronize()
        for w in self.weights:
            self.jam.evict(Segment.of(w))
        self.jam.set_stream(None)


class Conversations:
    """Sequences behind one shared prompt: their pages, lengths and the batches that the calls take."""

    def __init__(self, decoder: Decoder, prefix, prompts, shared=True):
        """shared=False: every conversation keeps the prefix in pages of its own."""
        self.d, self.free = decoder, iter(range(10 ** 9))
        self.pages = [[] for _ in prompts]
        self.own = [0] * len(prompts)
        self.base = len(prefix) if shared else 0
        self.prefix_pages = []
        if shared:
            self.prefix_pages = self._grow([], len(prefix))
            self._call([prefix], [self.prefix_pages], [len(prefix)], 0, [])
        self.logits = self._extend(prompts if shared else [list(prefix) + list(p) for p in prompts])

    def _grow(self, pages, length):
        while len(pages) * PAGE < length:
            pages.append(next(self.free))
        return pages

    def _call(self, new, tables, lengths, base, prefix_pages):
        """new[i] tokens of sequence i, the last of its lengths[i] own ones."""
        flat = [t for s in new for t in s]
        at = [(tables[i], lengths[i] - len(s) + k) for i, s in enumerate(new) for k in range(len(s))]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()   # noqa: E731
        width = max(len(t) for t in tables)
        self.held = a = [i32(flat), i32([base + p for _, p in at]), i32([t[p // PAGE] * PAGE + p % PAGE for t, p in at]),
                         i32(np.cumsum([0] + [len(s) for s in new]).tolist()), i32(lengths), i32([t + [0] * (width - len(t)) for t in tables]),
                         i32([0, len(new)]), i32([base]), i32([prefix_pages or [0]])]
        torch.cuda.synchronize()
        b = AttnBatch(n_tokens=len(flat), n_seqs=len(new), n_prefixes=int(bool(prefix_pages)), max_q=max(len(s) for s in new),
                      max_seq_len=max(lengths), max_prefix_len=base, q_offsets=a[3].data_ptr(), seq_lens=a[4].data_ptr(),
                      seq_pages=a[5].data_ptr(), ld_seq_pages=width, prefix_seqs=a[6].data_ptr(), prefix_lens=a[7].data_ptr(),
                      prefix_pages=a[8].data_ptr(), ld_prefix_pages=max(1, len(prefix_pages)))
        logits = self.d.forward(a[0], a[1], a[2], b)
        self.d.stream.synchronize()
        return logits[(a[3][1:] - 1).long()].contiguous()

    def _extend(self, new):
        for i, s in enumerate(new):
            self.own[i] += len(s)
            self._grow(self.pages[i], self.own[i])
        return self._call(new, self.pages, self.own, self.base, self.prefix_pages)

    def step(self, u):
        """One more token of every conversation from the random numbers u [sequences]; returns them."""
        torch.cuda.synchronize()
        tokens = self.d.sample(self.logits, u=u)
        self.d.stream.synchronize()
        out = tokens.tolist()
        self.logits = self._extend([[t] for t in out])
        return out


def main(steps=8):
    rng = np.random.default_rng(1)
    prefix = rng.integers(0, VOCAB, 75).tolist()
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (5, 33, 18)]
    jam = HipJAM()
    decoder = Decoder(jam, pages=64)
    try:
        chats = Conversations(decoder, prefix, prompts)
        for step in range(steps):
            u = torch.from_numpy(rng.random(len(prompts)).astype(np.float32) * np.float32(1 - 2 ** -24)).cuda()
            print(step, chats.step(u))
    finally:
        decoder.close()
        jam.close()


if __name__ == "__main__":
    main()
