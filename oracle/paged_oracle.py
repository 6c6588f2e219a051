"""Restatement of the paged key-value cache in plain PyTorch: test infrastructure.

A case is plain tensors on the CPU: pages [n_pages, heads, page, head_dim] as the values they stand for (float64), table, lengths,
starts.  Rounding to e4m3 and the fp32 rotation are written out, since the cache's bytes are defined by them."""
import math

import torch

F32, F64 = torch.float32, torch.float64


def places(table, lengths, starts, page):
    """[(row, sequence, position, page number, slot)] of a call's rows that have a place in the table."""
    got = []
    for b, n in enumerate(lengths):
        first, end = (b, b + (n > 0)) if starts is None else (starts[b], starts[b + 1])
        for r in range(first, end):
            pos = n - (end - r)
            if 0 <= pos < table.shape[1] * page:
                got.append((r, b, pos, int(table[b, pos // page]), pos % page))
    return got


def turn(x, angles, rot, interleaved, dtype=F32):
    """x [heads, head_dim] turned by angles [rot / 2, 2]: products and sums of `dtype`, one rounding each."""
    x, c, s = x.to(dtype).clone(), angles[:, 0].to(dtype), angles[:, 1].to(dtype)
    a, b = (x[:, 0:rot:2], x[:, 1:rot:2]) if interleaved else (x[:, :rot // 2], x[:, rot // 2:rot])
    p, q = a * c - b * s, b * c + a * s
    if interleaved:
        x[:, 0:rot:2], x[:, 1:rot:2] = p, q
    else:
        x[:, :rot // 2], x[:, rot // 2:rot] = p, q
    return x


def exponent(x):
    """Per row of fp32 values: the smallest e with max|x| <= 448 * 2^e, at least -126, over what is finite."""
    top = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1).to(F64)
    return torch.tensor([max(-126, math.ceil(math.log2(t / 448))) if t > 0 else -126 for t in top.reshape(-1).tolist()]).view(top.shape)


def quantise(x):
    """fp32 rows -> (e4m3 numbers, e + 127)."""
    e = exponent(x)
    y = (x.to(F64) * torch.exp2(-e.to(F64))[..., None])
    return torch.where(torch.isfinite(y), y, torch.full_like(y, math.nan)).to(F32).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def values(pages, scales=None, which=0):
    """What pages stand for, in float64."""
    x = pages.to(F32).to(F64)
    return x if scales is None else x * torch.exp2(scales[:, :, which].to(F64) - 127)[..., None]


def attention(q, k, v, table, lengths, starts, scale):
    """q [rows, Hq, head_dim] on pages k, v of values -> (y, sum of weight * |v|, largest sum |q k| * scale), rows without a
    sequence NaN, keys of bad pages not there."""
    rows, hq, hd = q.shape
    n_pages, hkv, page, _ = k.shape
    y = torch.full((rows, hq, hd), math.nan, dtype=F64)
    spread, size = torch.zeros(rows, hq, hd, dtype=F64), 0.0
    for b, length in enumerate(lengths):
        n = min(max(length, 0), table.shape[1] * page)     # (a position is the length's, whether or not the table has all of the keys)
        first, end = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        if end <= first:
            continue
        ids = table[b, :-(-n // page)].tolist()
        ok = torch.tensor([0 <= p < n_pages for p in ids for _ in range(page)][:n], dtype=torch.bool)
        safe = [p if 0 <= p < n_pages else 0 for p in ids]
        ks, vs = ((x[safe].transpose(0, 1).reshape(hkv, -1, hd)[:, :n] if n else x.new_zeros(hkv, 0, hd)) for x in (k, v))
        vs = torch.where(ok[None, :, None], vs, torch.zeros_like(vs))
        for r in range(first, end):
            see = ok & (torch.arange(n) <= length - (end - r))
            for h in range(hq):
                kh, vh = ks[h // (hq // hkv)][see], vs[h // (hq // hkv)][see]
                if not see.any():
                    y[r, h] = 0
                    continue
                s = kh @ q[r, h].to(F64) * scale
                w = torch.softmax(s, 0)
                y[r, h], spread[r, h] = w @ vh, w @ vh.abs()
                size = max(size, float((kh.abs() @ q[r, h].to(F64).abs()).max()) * scale)
    return y, spread, size


def attention_of_sequences(q, k, v, table, lengths, starts, scale):
    """attention() of a call with starts, all rows of a sequence and head at once."""
    rows, hq, hd = q.shape
    n_pages, hkv, page, _ = k.shape
    y = torch.full((rows, hq, hd), math.nan, dtype=F64)
    spread, size = torch.zeros(rows, hq, hd, dtype=F64), 0.0
    for b, length in enumerate(lengths):
        first, end = starts[b], starts[b + 1]
        if end <= first:
            continue
        there = min(max(length, 0), table.shape[1] * page)
        ids = table[b, :-(-there // page)].long()
        ok = ((ids >= 0) & (ids < n_pages)).repeat_interleave(page)[:there]
        safe = torch.where((ids >= 0) & (ids < n_pages), ids, torch.zeros_like(ids))
        see = ok & (torch.arange(there) <= length - end + torch.arange(first, end)[:, None])
        for h in range(hq):
            kh, vh = (x[safe, h // (hq // hkv)].reshape(-1, hd)[:there] for x in (k, v))
            qh = q[first:end, h].to(F64)
            score = torch.where(see, qh @ kh.t() * scale, -math.inf)
            top = score.amax(-1, keepdim=True) if there else score.new_zeros(end - first, 1)
            w = torch.where(see, torch.exp(score - torch.where(top > -math.inf, top, 0.0)), 0.0)
            total = w.sum(-1, keepdim=True)
            w = w / torch.where(total > 0, total, 1.0)
            y[first:end, h], spread[first:end, h] = w @ vh, w @ vh.abs()
            if there:
                size = max(size, float((qh.abs() @ kh.abs().t()).max()) * scale)
    return y, spread, size
