"""Decoding with drafted trees on one MI355X, through qxotic_amd.jam.HipJAM: every step a few guesses of each conversation's next tokens
go through the model in one pass, and the ones that agree with what it picks are kept.

    python examples/tree_step.py

The decoder is the one of decode_step.py. Lengths, page tables, free pages and slots live on the device: a step hands out pages for the
drafted tokens, attends to each tree by its mask, picks after every drafted token, keeps a path, moves its entries to their places in all
layers' caches, and takes the pages that are too many back. The drafts are of the simplest kind: what followed the last token earlier on."""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))

from decode_step import LAYERS, PAGE, VOCAB, Decoder                             # noqa: E402

from qxotic_amd.jam import AttnBatch, HipJAM, KvCache, KvPages, Tree, TreePath   # noqa: E402


class Trees:
    """Conversations whose state is on the device: [n] lengths and pages held, [n, width] page tables, the list of free pages. All of it is made
    and used on the decoder's stream, which waits for nothing by itself and nothing for it."""

    def __init__(self, decoder: Decoder, pages: int, prompts, width: int = 16):
        self.d, self.n, self.pages, self.width = decoder, len(prompts), pages, width
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")   # noqa: E731
        with torch.cuda.stream(decoder.stream):
            self.lens, self.held, self.table, self.status = i32(self.n), i32(self.n), i32(self.n, width), i32(self.n)
            self.free = torch.arange(pages, dtype=torch.int32, device="cuda")
            self.n_free = torch.full((1,), pages, dtype=torch.int32, device="cuda")
            self.offsets = i32(self.n + 1)
            self.caches = (KvCache * LAYERS)(*decoder.caches)
            self.longest = 0   # of a conversation, as the host knows it: at most
            logits = self._pass(prompts, None)[0]
            if self.status.any():
                raise RuntimeError("out of pages")
            logits = logits[(self.offsets[1:] - 1).long()].contiguous()   # after each prompt's last token
        self.logits = self._out(logits)

    def _out(self, t):
        """A tensor of the decoder's stream for the caller's, which waits for it; it is not used again while that one still reads it."""
        caller = torch.cuda.current_stream()
        caller.wait_stream(self.d.stream)
        t.record_stream(caller)
        return t

    def _resize(self, targets, rows=0, pos=None, slots=None, old=None):
        """To `targets` [n] tokens each; `old`: where the lengths before stay (else they are followed in place)."""
        p = KvPages(n_seqs=self.n, n_tokens=rows, page_tokens=PAGE, n_pages=self.pages, free_cap=self.pages, ld_seq_pages=self.width)
        lens = self.lens if old is None else old
        arrays = dict(lens=lens, targets=targets, held=self.held, n_free=self.n_free, free_pages=self.free, seq_pages=self.table,
                      lens_out=self.lens, held_out=self.held, n_free_out=self.n_free, status=self.status, q_offsets=self.offsets, pos=pos, slots=slots)
        for k, t in arrays.items():
            setattr(p, k, None if t is None else t.data_ptr())
        self.d._ok(self.d.jam.kv_resize(p))

    def _pass(self, tokens, parents):
        """New tokens of every conversation through the model, as prompts or (with parents) as trees: the logits of all rows, and what the
        step's end needs."""
        counts, rows = [len(t) for t in tokens], sum(len(t) for t in tokens)
        with torch.cuda.stream(self.d.stream):
            up = lambda v: torch.tensor(v, dtype=torch.int32).pin_memory().cuda(non_blocking=True)   # noqa: E731
            flat = up([t for s in tokens for t in s])
            pos, slots = torch.empty_like(flat), torch.empty_like(flat)
            before = self.lens.clone()
            targets = before + up(counts)
            offsets = self.offsets if parents is None else torch.empty_like(self.offsets)
            self.offsets = offsets
            self._resize(targets, rows, pos, slots, before)
            self.longest += max(counts)
            batch = AttnBatch(n_tokens=rows, n_seqs=self.n, max_q=max(counts), max_seq_len=min(self.longest, self.width * PAGE),
                              q_offsets=offsets.data_ptr(), seq_lens=self.lens.data_ptr(), seq_pages=self.table.data_ptr(), ld_seq_pages=self.width)
            masks = tree = None
            if parents is not None:
                links = up([p for s in parents for p in s])
                tree = Tree(n_tokens=rows, n_seqs=self.n, max_q=max(counts), q_offsets=offsets.data_ptr(), parents=links.data_ptr())
                masks = torch.zeros((rows, -(-max(counts) // 64)), dtype=torch.int64, device="cuda")
                self.d._ok(self.d.jam.tree_masks(tree, masks.data_ptr(), masks.shape[1], pos.data_ptr()))
                self.kept = links
            logits = self.d.forward(flat, pos, slots, batch, masks)
        return logits, flat, slots, before, tree

    def step(self, drafts, temperature=0.0, u=None, picked=None):
        """drafts: each conversation's (tokens, parents), token 0 the one that was picked last. Returns (path, next token) of each, and the
        logits of all drafted tokens. A conversation without room for its tree stays as it was: its path is empty, its next token the same one.
        `picked`: the model's picks given from outside, int32 [rows]."""
        tokens, parents = [t for t, _ in drafts], [p for _, p in drafts]
        self.d.stream.wait_stream(torch.cuda.current_stream())   # u and picked are the caller's
        for t in (u, picked):
            if t is not None:
                t.record_stream(self.d.stream)
        logits, flat, slots, before, tree = self._pass(tokens, parents)
        most = max(len(t) for t in tokens)
        with torch.cuda.stream(self.d.stream):
            if picked is None:
                u = torch.zeros(flat.numel(), device="cuda") if u is None else u
                picked = self.d.sample(logits, temperature=temperature, u=u)
            path = torch.empty((self.n, most), dtype=torch.int32, device="cuda")
            accepted, after, lens = (torch.empty(self.n, dtype=torch.int32, device="cuda") for _ in range(3))
            src, dst = torch.empty_like(flat), torch.empty_like(flat)
            p = TreePath(ld_path=most, path=path.data_ptr(), accepted=accepted.data_ptr(), next=after.data_ptr(), lens=before.data_ptr(),
                         lens_out=lens.data_ptr(), slots=slots.data_ptr(), move_from=src.data_ptr(), move_to=dst.data_ptr())
            self.d._ok(self.d.jam.tree_accept(tree, flat.data_ptr(), picked.data_ptr(), p))
            self.d._ok(self.d.jam.kv_move(self.caches, LAYERS, self.offsets.data_ptr(), self.n, src.data_ptr(), dst.data_ptr(), flat.numel()))
            self.offsets = torch.empty_like(self.offsets)   # the next call's own; this one's are still read
            self._resize(lens)   # refuses none: no length grows
            out = [t.cpu() for t in (path, accepted, after, self.lens)]
        path, accepted, after, held = (t.tolist() for t in out)
        self.longest = max(held)
        return [(p[:k], t) for p, k, t in zip(path, accepted, after)], self._out(logits)


def draft(history, root, width=3, depth=4):
    """A tree behind `root`: what followed it in the history, up to `width` times, `depth` tokens each."""
    tokens, parents = [root], [-1]
    for at in [i for i, t in enumerate(history[:-1]) if t == root][-width:]:
        parent = 0
        for t in history[at + 1:at + 1 + depth]:
            tokens.append(t)
            parents.append(parent)
            parent = len(tokens) - 1
    return tokens, parents


def main(steps=8):
    rng = np.random.default_rng(1)
    phrase = rng.integers(0, VOCAB, 12).tolist()
    prompts = [phrase * 3, phrase[3:] + phrase, rng.integers(0, VOCAB, 18).tolist()]
    jam = HipJAM()
    decoder = Decoder(jam, pages=64)
    try:
        trees = Trees(decoder, 64, prompts)
        decoder.stream.synchronize()
        roots = trees.logits.argmax(-1).tolist()
        text = [list(p) for p in prompts]
        for step in range(steps):
            drafts = [draft(h, r) for h, r in zip(text, roots)]
            paths, _ = trees.step(drafts)
            for h, (tokens, _), (path, _) in zip(text, drafts, paths):
                h += [tokens[i] for i in path]
            roots = [t for _, t in paths]
            print(step, [len(p) for p, _ in paths], roots)
    finally:
        decoder.close()
        jam.close()


if __name__ == "__main__":
    main()
