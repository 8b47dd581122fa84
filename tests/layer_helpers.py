"""Batches and bounds for the tests of the operators around the expert block."""
from __future__ import annotations

import numpy as np
import torch

from moe_stream_amd import synth

BF16, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
# half a step, relative to the value
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
# half the step of a type's subnormal range, absolute
TINY = {BF16: 0.0, F16: 2.0 ** -25}


def randn(shape, seed, dtype=BF16, scale=1.0):
    g = synth.generator("cuda", seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def f64(t) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def within(got, ref, bound):
    """got (a tensor) is within bound of ref everywhere; the worst share of the bound."""
    g = f64(got)
    assert np.isfinite(g).all(), "not finite"
    share = np.abs(g - ref) / np.maximum(bound, 1e-300)
    worst = float(share.max()) if share.size else 0.0
    assert worst <= 1.0, (f"{worst:.3g} of the bound at "
                          f"{np.unravel_index(int(share.argmax()), share.shape)}")
    return worst


class Batch:
    """Sequences of (new tokens, whole length) over pages in random order; pages hold
    `fill` where no token is."""

    def __init__(self, seqs, heads, kv_heads, dim, page=16, dtype=BF16, seed=1, fill=None,
                 extra_rows=0, extra_width=1):
        self.seqs, self.dtype, self.page = seqs, dtype, page
        rng = np.random.default_rng(seed)
        used = [-(-L // page) for _, L in seqs]
        n_pages = sum(used) + 2
        order = rng.permutation(n_pages)
        self.np_table = np.zeros((len(seqs), max(max(used), 1) + extra_width), dtype=np.int32)
        at = 0
        for s, u in enumerate(used):
            self.np_table[s, :u] = order[at:at + u]
            at += u
        starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.rows = int(starts[-1])
        self.T = self.rows + extra_rows
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table = torch.tensor(self.np_table, **i32)
        self.starts = torch.tensor(starts, **i32)
        self.lens = torch.tensor([L for _, L in seqs], **i32)
        self.np_starts = starts
        shape = (n_pages, kv_heads, page, dim)
        self.kp = randn(shape, seed + 1, dtype)
        self.vp = randn(shape, seed + 2, dtype)
        self.q = randn((self.T, heads, dim), seed + 3, dtype, 1.5)
        if fill is not None:   # every place past a sequence's end, and the spare pages
            live = np.zeros((n_pages, page), dtype=bool)
            for s, (_, L) in enumerate(seqs):
                j = np.arange(L)
                live[self.np_table[s, j // page], j % page] = True
            dead = torch.tensor(~live, device="cuda")[:, None, :, None].expand(shape)
            self.kp[dead] = fill
            self.vp[dead] = fill

    def pages(self):
        return self.kp, self.vp, self.table, self.starts, self.lens

    def cached(self, s, pages):
        """Sequence s's [L, HK, D] in 64 bits."""
        L = self.seqs[s][1]
        j = np.arange(L)
        p = f64(pages)
        return p[self.np_table[s, j // self.page], :, j % self.page]

    def span(self, s):
        n, L = self.seqs[s]
        return slice(int(self.np_starts[s]), int(self.np_starts[s]) + n), np.arange(L - n, L)
