"""Inputs that the tests of the paged key-value cache share, made on the CPU."""
import math
import random

import torch

from oracle import paged_oracle as O

BF, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn


class Case:
    """Random pages with the given lengths; what no sequence has is NaN (e4m3: NaN with the largest scale)."""

    def __init__(self, lengths, hkv, hd, page, e4m3, seed=0, new=None, spare=2, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.page, self.hkv, self.hd, self.e4m3 = page, hkv, hd, e4m3
        self.lengths = list(lengths)
        self.new = new
        self.starts = None if new is None else [sum(new[:b]) for b in range(len(new) + 1)]
        self.rows = len(lengths) if new is None else self.starts[-1]
        used = [-(-max(n, 0) // page) for n in lengths]
        self.n_pages = sum(used) + spare
        order = list(range(self.n_pages))
        random.Random(seed).shuffle(order)
        self.table = torch.full((len(lengths), max(used + [1]) + 1), -7, dtype=torch.int32)
        mine = torch.zeros(self.n_pages, page, dtype=torch.bool)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            for i in range(n):
                mine[order[at + i], :min(page, max(lengths[b], 0) - i * page)] = True
            at += n
        k, v = (torch.randn(self.n_pages, hkv, page, hd, generator=g) * spread for _ in range(2))
        self.scales = None
        if e4m3:
            (k, ke), (v, ve) = O.quantise(k), O.quantise(v)
            self.scales = torch.where(mine[:, None, None, :], torch.stack([ke, ve], 2), torch.tensor(254, dtype=torch.uint8))
        nan = torch.tensor(math.nan)
        self.k, self.v = (torch.where(mine[:, None, :, None], x.to(F32), nan).to(E4M3 if e4m3 else BF) for x in (k, v))

    def on(self, device, hq, rows=None):
        from gpt_fast.utils import PagedKVCache

        t = lambda x: None if x is None else torch.as_tensor(x, dtype=torch.int32).to(device)
        cache = PagedKVCache.from_pages(self.k.to(device), self.v.to(device), None if self.scales is None else self.scales.to(device))
        return cache, cache.batch(t(self.table), t(self.lengths), hq, starts=t(self.starts),
                                  rows=None if self.starts is None else rows or max(1, self.rows))

    def oracle(self, q, hq, scale=None):
        """(y, sum of weights * |v|, size of the scores) of O.attention."""
        clean = lambda x: torch.nan_to_num(x, nan=0.0)
        return O.attention(q.view(-1, hq, self.hd), clean(O.values(self.k, self.scales, 0)), clean(O.values(self.v, self.scales, 1)),
                           self.table, self.lengths, self.starts, scale or self.hd ** -0.5)


def bound(want, spread, size, keys, hd, weight):
    """How far y may be off: its own rounding to bf16 (half a step is 2^-8 of the value); a score's fp32 sum of hd products, each
    addition off by 2^-24 of what has been added up to there, and its product with scale and log2(e), 2^-23 of it: a weight is off by the
    factor e^(that); exponential and sums of `keys` weights 2^-23 each; a weight's rounding to what the matrix cores take,
    `weight`.  The last three enter numerator and denominator."""
    score = (hd * 2.0 ** -24 + 2.0 ** -22) * size
    return 2.0 ** -8 * want.abs() + 2 * (score + (keys + 8) * 2.0 ** -23 + weight) * spread + 1e-30
