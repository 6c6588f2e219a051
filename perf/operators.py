"""Operators of a paged key-value cache: what is timed of them, in their plain form and through gpt_fast.utils.PagedKVCache.

A cache holds k and v as pages [n_pages, kv heads, page, head_dim], bf16 or e4m3; e4m3 rows have a power of two each, its exponent
as a byte (value + 127) in scales [n_pages, kv heads, 2, page] (k's, then v's).  A batch is a table of page numbers [B, P], the
sequences' lengths (the call's tokens among them) and, where a sequence may have several rows in the call, starts [B + 1].

A case: `op` ("write", "read", "decode", "prefill"), `q_heads`, `kv_heads`, `head_dim`, `page`, `cache` ("bf16" or "e4m3"), `batch`
sequences of which the longest has `longest` tokens ahead of the call's own, up to `new` of those each, `even`: all as long as the
longest, else ragged; write: `rope` ("pairs" or "halves"), `rotary` dimensions, `table` of angles ("bf16" or "fp32").

exact() restates the operators in float64, sequence by sequence."""
import math
import os
import random
import sys

import torch

own = False

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------------------------------------ the cases

def _case(op, heads, page, cache, batch, longest, new, even=False, rope="pairs", rotary=None, table="bf16"):
    c = dict(op=op, q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2], page=page, cache=cache, batch=batch, longest=longest,
             new=new, even=even)
    if op == "write":
        c.update(rope=rope, rotary=rotary or heads[2], table=table)
    return c


H1B, H8B, H70B, H405B = (32, 8, 64), (32, 8, 128), (8, 1, 128), (16, 1, 128)   # the last two: one rank of eight


def listed():
    named = [
        # one user's token enters the cache of a 70B rank shard: the smallest call there is
        ("write_70b_b1", _case("write", H70B, 16, "bf16", 1, 2047, 1)),
        # a decode step of 64 users, quantised as it is written; angles in fp32, half of each head turned
        ("write_8b_b64_e4m3", _case("write", H8B, 64, "e4m3", 64, 4095, 1, rope="halves", rotary=64, table="fp32")),
        # six prompts of ragged lengths enter a quantised cache
        ("write_8b_prompts_e4m3", _case("write", H8B, 32, "e4m3", 6, 0, 2048)),
        # one short sequence read back, small heads, odd length
        ("read_1b_b1", _case("read", H1B, 16, "bf16", 1, 0, 333)),
        # sixteen sequences of a quantised cache read back, as they move to another machine
        ("read_8b_b16_e4m3", _case("read", H8B, 64, "e4m3", 16, 0, 4096)),
        # the headline's shard, one user: latency of a token's attention
        ("decode_70b_b1", _case("decode", H70B, 16, "bf16", 1, 2048, 1)),
        # a serving batch whose sequences have lengths of their own, some places empty
        ("decode_8b_b24_ragged", _case("decode", H8B, 16, "bf16", 24, 4096, 1)),
        # a large serving batch on a quantised cache
        ("decode_8b_b64_e4m3", _case("decode", H8B, 64, "e4m3", 64, 2048, 1, even=True)),
        # one user with a long document
        ("decode_8b_long", _case("decode", H8B, 64, "bf16", 1, 131071, 1)),
        # three short prompts to a small model: time to the first token
        ("prefill_1b_short", _case("prefill", H1B, 16, "bf16", 3, 0, 100)),
        # prompts of ragged lengths together in one call
        ("prefill_8b_ragged", _case("prefill", H8B, 64, "bf16", 5, 0, 2048)),
        # the next portion of a long document on a rank shard, history quantised
        ("prefill_70b_portion_e4m3", _case("prefill", H70B, 32, "e4m3", 1, 8111, 256)),
    ]
    return [dict(c, name=n) for n, c in named]


def _spread(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    """Head layouts from one kv head to as many as q heads, pages of 16 to 256, 1 to 64 sequences; decode up to 32768 keys of a sequence
    (131072 of all; fewer where there are more than 8 kv heads), prompts up to 2048 tokens (6000 of all), portions behind up to 8192."""
    op = rng.choice(["write", "read", "decode", "decode", "prefill", "prefill"])
    heads = rng.choice([H1B, H8B, H8B, H70B, H405B, (12, 12, 64), (14, 2, 64), (24, 24, 128)])
    many = max(1, heads[1] // 8)
    page, cache, even = rng.choice([16, 32, 64, 128, 256]), rng.choice(["bf16", "e4m3"]), rng.random() < 0.3
    if op == "write":
        batch = _spread(rng, 1, 64)
        new = 1 if rng.random() < 0.5 else _spread(rng, 2, max(2, 8192 // batch))
        rot = rng.choice([heads[2], heads[2], heads[2] // 2, 16])
        return _case(op, heads, page, cache, batch, _spread(rng, 1, 4096) - 1, new, even, rng.choice(["pairs", "halves"]), rot,
                     rng.choice(["bf16", "fp32"]))
    if op == "read":
        batch = _spread(rng, 1, 32)
        return _case(op, heads, page, cache, batch, 0, _spread(rng, 1, 32768 // (batch * many)), even)
    if op == "decode":
        batch = _spread(rng, 1, 64)
        return _case(op, heads, page, cache, batch, _spread(rng, 1, min(32768, 131072 // (batch * many))), 1, even)
    if rng.random() < 0.5:
        batch = _spread(rng, 1, 8)
        return _case(op, heads, page, cache, batch, 0, _spread(rng, 2, min(2048, 6000 // batch)), even)
    batch = _spread(rng, 1, 4)
    return _case(op, heads, page, cache, batch, _spread(rng, 16, 8192 // batch), _spread(rng, 2, 256), even)


def _sizes(case):
    """[(tokens ahead of the call's, the call's)] per sequence: the first is the longest, the others anything below it (one in three by
    its logarithm: many users have just begun), in a decode step every ninth place is empty.  A write of single tokens has no empty place."""
    r = random.Random(case["batch"] * 1000003 + case["longest"] * 131 + case["new"])
    got = []
    for b in range(case["batch"]):
        if b == 0 or case["even"]:
            ahead, new = case["longest"], case["new"]
        else:
            below = (lambda n: _spread(r, 1, n)) if r.random() < 0.33 else (lambda n: r.randint(1, n))
            ahead, new = below(case["longest"] + 1) - 1, below(case["new"])
            if case["op"] == "decode" and b % 9 == 5:
                ahead = new = 0
        if case["op"] == "decode" and new:
            ahead = max(ahead - 1, 0)
        got.append((ahead, new))
    return got


def work(case):
    hq, hkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    c = 2 if case["cache"] == "bf16" else 1
    row = hkv * (2 * hd * c + (2 if c == 1 else 0))      # bytes of a token in the cache
    sizes = _sizes(case)
    rows, keys = sum(n for _, n in sizes), sum(a + n for a, n in sizes)
    pages = 4 * sum(-(-(a + n) // case["page"]) for a, n in sizes) + 8 * len(sizes)
    if case["op"] == "write":
        positions = len({p for a, n in sizes for p in range(a, a + n)}) * case["rotary"] * (2 if case["table"] == "bf16" else 4)
        return {"bytes": rows * ((2 * hq + 2 * hkv) * hd * 2 + row) + positions + pages, "flops": rows * (hq + hkv) * case["rotary"] * 3}
    if case["op"] == "read":
        return {"bytes": rows * (2 * hkv * hd * 2 + row) + pages, "flops": 0}
    seen = sum(a * n + n * (n + 1) // 2 for a, n in sizes)
    return {"bytes": keys * row + 2 * rows * hq * hd * 2 + pages, "flops": 4 * hq * hd * seen}


# ------------------------------------------------------------------------------------------------ inputs

def _exponents(x):
    """The smallest e with max|x| <= 448 * 2^e over the last dimension; -126 at least."""
    m, e = torch.frexp(x.abs().amax(-1))          # m * 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    return torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)


def _power(e):
    """2^e in fp32, exactly; e from -126 to 127."""
    return ((e.to(torch.int32) + 127) << 23).view(F32)


def _quantised(x):
    """(x / 2^e as e4m3, e + 127 as bytes) of fp32 rows."""
    e = _exponents(x)
    return (x * _power(-e)[..., None]).to(E4M3), (e + 127).to(torch.uint8)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    hq, hkv, hd, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    sizes = _sizes(case)
    lengths = [a + n for a, n in sizes]
    starts = [sum(n for _, n in sizes[:b]) for b in range(len(sizes) + 1)]
    rows = starts[-1]
    width = max(1, -(-max(lengths) // page)) + 1
    used = [-(-n // page) for n in lengths]
    n_pages = sum(used) + 3
    # pages in the order in which an allocator that has run for a while hands them out: any
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(sizes), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    single = case["op"] == "decode" or (case["op"] == "write" and case["new"] == 1)    # one row per sequence
    s = dict(case=case, table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device=dev),
             starts=None if single else torch.tensor(starts, dtype=torch.int32, device=dev))
    rows = len(sizes) if single else rows
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)
    # a few channels of keys are several times the others, as in trained models
    channel = torch.exp(0.5 * normal(hkv, 1, hd))
    if case["op"] == "write":
        qkv = normal(rows, (hq + 2 * hkv) * hd)
        qkv[:, hq * hd:(hq + hkv) * hd] *= channel.reshape(-1)
        s["qkv"] = qkv.to(BF)
        s["q"] = torch.zeros(rows, hq * hd, dtype=BF, device=dev)
        half = case["rotary"] // 2
        freq = 500000.0 ** (-torch.arange(half, dtype=F64, device=dev) / half)
        angle = torch.arange(max(lengths) + 5, dtype=F64, device=dev)[:, None] * freq
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).to(BF if case["table"] == "bf16" else F32)
        k, v = (torch.zeros(n_pages, hkv, page, hd, dtype=F32, device=dev) for _ in range(2))
    else:
        k, v = normal(n_pages, hkv, page, hd), normal(n_pages, hkv, page, hd)
        k *= channel / channel.square().mean().sqrt()
        s["q"] = normal(rows, hq * hd).to(BF)
    s["scales"] = None
    if case["cache"] == "e4m3":
        (s["k"], ke), (s["v"], ve) = _quantised(k), _quantised(v)
        s["scales"] = torch.stack([ke, ve], 2).contiguous()
        if case["op"] == "write":
            s["scales"].zero_()
    else:
        s["k"], s["v"] = k.to(BF), v.to(BF)
    s["kv"] = s["k"], s["v"]
    if case["op"] == "read":
        s["rows"] = tuple(torch.empty(rows, hkv * hd, dtype=BF, device=dev) for _ in range(2))
    elif case["op"] != "write":
        s["y"] = torch.empty(rows, hq * hd, dtype=BF, device=dev)
    if own:   # the cache and the batch's plan, which a program keeps from step to step
        PagedKVCache = _package()
        s["cache"] = PagedKVCache.from_pages(s["k"], s["v"], s["scales"])
        s["batch"] = s["cache"].batch(s["table"], s["lengths"], hq, starts=s["starts"], rows=rows)
    return s


def _package():
    at = os.path.abspath("ladder-residual-inference_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from gpt_fast.utils import PagedKVCache

    return PagedKVCache


# ------------------------------------------------------------------------------------------------ the plain form

def _where(s, rows):
    """(sequence, position) of each row of the call."""
    row = torch.arange(rows, device="cuda")
    if s["starts"] is None:
        return row, s["lengths"].long() - 1
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    return seq, s["lengths"].long()[seq] - s["starts"].long()[seq + 1] + row


def _slots(s, seq, pos):
    page = s["case"]["page"]
    return s["table"][seq, pos // page].long(), pos % page


def _as_fp32(x, scales):
    """Cache rows [..., head_dim] as the values they stand for."""
    return x.float() if scales is None else x.float() * _power(scales.int() - 127)[..., None]


def _gather(s, which, pages, slots):
    """Rows [n, kv heads, head_dim] of k (0) or v (1) at [n] places."""
    x = s["kv"[which]]
    raw = x.view(torch.uint8)[pages, :, slots].view(x.dtype) if x.dtype == E4M3 else x[pages, :, slots]
    return _as_fp32(raw, None if s["scales"] is None else s["scales"][pages, :, which, slots])


def _sequences(s, which):
    """All of k or v of every sequence, [B, kv heads, page * P, head_dim]; pages that are not there: page 0's."""
    x, at = s["kv"[which]], s["table"].clamp(min=0).long()
    raw = x.view(torch.uint8)[at].view(x.dtype) if x.dtype == E4M3 else x[at]
    rows = _as_fp32(raw, None if s["scales"] is None else s["scales"][at][:, :, :, which])
    return rows.transpose(1, 2).reshape(at.shape[0], x.shape[1], -1, x.shape[3])


def _turn(x, cos, sin, rotary, style):
    """fp32 rows [n, heads, head_dim] turned by [n, rotary / 2] angles."""
    out, cos, sin = x.clone(), cos[:, None], sin[:, None]
    if style == "pairs":
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        out[..., 0:rotary:2], out[..., 1:rotary:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        out[..., :rotary // 2], out[..., rotary // 2:rotary] = a * cos - b * sin, b * cos + a * sin
    return out


def _plain_write(s):
    c = s["case"]
    hq, hkv, hd = c["q_heads"], c["kv_heads"], c["head_dim"]
    rows = s["qkv"].shape[0]
    x = s["qkv"].float().view(rows, hq + 2 * hkv, hd)
    seq, pos = _where(s, rows)
    angles = s["rope"].float()[pos]
    turned = _turn(x[:, :hq + hkv], angles[..., 0], angles[..., 1], c["rotary"], c["rope"])
    s["q"].copy_(turned[:, :hq].reshape(rows, -1))
    pages, slots = _slots(s, seq, pos)
    k, v = turned[:, hq:], x[:, hq + hkv:]
    if s["scales"] is None:
        s["k"][pages, :, slots], s["v"][pages, :, slots] = k.to(BF), v.to(BF)
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    (k8, ke), (v8, ve) = _quantised(k), _quantised(v)
    s["k"].view(torch.uint8)[pages, :, slots] = k8.view(torch.uint8)
    s["v"].view(torch.uint8)[pages, :, slots] = v8.view(torch.uint8)
    s["scales"][pages, :, :, slots] = torch.stack([ke, ve], -1)
    return {"q": s["q"], "k": s["k"], "v": s["v"], "scales": s["scales"]}


def _plain_read(s):
    k, v = s["rows"]
    pages, slots = _slots(s, *_where(s, k.shape[0]))
    k.copy_(_gather(s, 0, pages, slots).reshape(k.shape))
    v.copy_(_gather(s, 1, pages, slots).reshape(v.shape))
    return {"k": k, "v": v}


def _attend(q, k, v, seen):
    """q [B, kv heads, n, head_dim] on k, v [B, kv heads, L, head_dim]; seen [B, 1, n, L]."""
    there = seen.any(-2)[..., None]              # keys that nobody sees hold anything
    k, v = torch.where(there, k, torch.zeros_like(k)), torch.where(there, v, torch.zeros_like(v))
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * q.shape[-1] ** -0.5
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight, v) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_decode(s):
    c = s["case"]
    B, hkv, hd = c["batch"], c["kv_heads"], c["head_dim"]
    k, v = _sequences(s, 0), _sequences(s, 1)
    seen = torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None]
    y = _attend(s["q"].float().view(B, hkv, -1, hd), k, v, seen[:, None, None, :])
    return s["y"].copy_(y.reshape(B, -1))


def _plain_prefill(s):
    c = s["case"]
    B, hq, hkv, hd = c["batch"], c["q_heads"], c["kv_heads"], c["head_dim"]
    rows, n, group = s["q"].shape[0], c["new"], c["q_heads"] // c["kv_heads"]
    seq, pos = _where(s, rows)
    at = torch.arange(rows, device="cuda") - s["starts"].long()[seq]
    q = torch.zeros(B, n, hq, hd, device="cuda")
    q[seq, at] = s["q"].float().view(rows, hq, hd)
    place = torch.full((B, n), -1, device="cuda")
    place[seq, at] = pos
    k, v = _sequences(s, 0), _sequences(s, 1)
    seen = torch.arange(k.shape[2], device="cuda") <= place[..., None]
    # the q heads of a kv head one after the other: [B, kv heads, group * n, head_dim]
    y = _attend(q.view(B, n, hkv, group, hd).permute(0, 2, 3, 1, 4).reshape(B, hkv, group * n, hd), k, v,
                seen.repeat(1, group, 1)[:, None])
    y = y.view(B, hkv, group, n, hd).permute(0, 3, 1, 2, 4).reshape(B, n, hq * hd)
    return s["y"].copy_(y[seq, at])


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    op = s["case"]["op"]
    if own:
        cache, batch = s["cache"], s["batch"]
        if op == "write":
            cache.write(batch, s["qkv"], s["q"], s["rope"], interleaved=s["case"]["rope"] == "pairs")
            got = {"q": s["q"], "k": s["k"], "v": s["v"]}
            return got if s["scales"] is None else dict(got, scales=s["scales"])
        if op == "read":
            cache.read(batch, *s["rows"])
            return {"k": s["rows"][0], "v": s["rows"][1]}
        return cache.attend(batch, s["q"], s["y"])
    return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "prefill": _plain_prefill}[op](s)


# ------------------------------------------------------------------------------------------------ in 64 bits

def _rows64(s, which, b, n):
    """The first n keys or values of sequence b, [kv heads, n, head_dim]."""
    page = s["case"]["page"]
    ids = s["table"][b, :-(-n // page)].tolist()
    parts = []
    for i, p in enumerate(ids):
        part = s["kv"[which]][p].to(F32).to(F64)
        if s["scales"] is not None:
            part = part * torch.exp2(s["scales"][p, :, which].to(F64) - 127)[..., None]
        parts.append(part[:, :min(page, n - i * page)])
    return torch.cat(parts, 1)


def _nearest_e4m3(x):
    """float64 to the nearest of e4m3's numbers, ties to even."""
    _, e = torch.frexp(x.abs())
    step = torch.exp2((e - 1).clamp(min=-6).to(F64) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    sizes = _sizes(case)
    if case["op"] == "write":
        q, rope = torch.zeros_like(s["q"], dtype=F64), s["rope"].to(F64)
        out = [s["k"].to(F32).to(F64), s["v"].to(F32).to(F64)]
        scales = None if s["scales"] is None else s["scales"].to(F64)
        r = case["rotary"]
        lo = torch.arange(0, r, 2, device="cuda") if case["rope"] == "pairs" else torch.arange(r // 2, device="cuda")
        hi = lo + (1 if case["rope"] == "pairs" else r // 2)
        row = 0
        for b, (ahead, new) in enumerate(sizes):
            x = s["qkv"][row:row + new].to(F64).view(new, -1, hd)
            turn = torch.view_as_complex(rope[ahead:ahead + new].contiguous())[:, None]
            z = torch.complex(x[:, :hq + hkv][..., lo].contiguous(), x[:, :hq + hkv][..., hi].contiguous()) * turn
            x[:, :hq + hkv, lo], x[:, :hq + hkv, hi] = z.real, z.imag
            q[row:row + new] = x[:, :hq].reshape(new, -1)
            pos = torch.arange(ahead, ahead + new, device="cuda")
            page, slot = s["table"][b].long()[pos // case["page"]], pos % case["page"]
            for which in (0, 1):
                y = x[:, hq + which * hkv:hq + (which + 1) * hkv]
                if scales is not None:
                    e = torch.ceil(torch.log2(y.abs().amax(-1) / 448))
                    scales[page, :, which, slot] = e + 127
                    y = _nearest_e4m3(y * torch.exp2(-e)[..., None])
                out[which][page, :, slot] = y
            row += new
        got = {"q": q, "k": out[0], "v": out[1]}
        return got if scales is None else dict(got, scales=None)
    if case["op"] == "read":
        got = [[_rows64(s, w, b, n).transpose(0, 1).reshape(n, -1) for b, (_, n) in enumerate(sizes)] for w in (0, 1)]
        return {"k": torch.cat(got[0]), "v": torch.cat(got[1])}
    y = torch.zeros(s["q"].shape[0], hq, hd, dtype=F64, device="cuda")
    row, group = 0, hq // hkv
    for b, (ahead, new) in enumerate(sizes):
        first = b if case["op"] == "decode" else row
        row += new
        if ahead + new == 0:
            continue
        k, v = _rows64(s, 0, b, ahead + new), _rows64(s, 1, b, ahead + new)
        q = s["q"][first:first + new].to(F64).view(new, hq, hd)
        late = torch.arange(ahead + new, device="cuda") > torch.arange(ahead, ahead + new, device="cuda")[:, None]
        for h in range(hkv):
            qh = q[:, h * group:(h + 1) * group].transpose(0, 1).reshape(group * new, hd)
            score = (qh @ k[h].t().contiguous() / math.sqrt(hd)).view(group, new, -1).masked_fill(late, -math.inf)
            w = torch.softmax(score, -1).view(group * new, -1)
            y[first:first + new, h * group:(h + 1) * group] = (w @ v[h]).view(group, new, hd).transpose(0, 1)
    return y.view(y.shape[0], -1)
