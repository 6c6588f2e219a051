"""The kernels of the paged key-value cache against their restatement in float64 (bits where the definition gives them).

What no sequence has in the pages is NaN, with the largest scale where rows have one; lengths lie around the edges of tiles and pages."""
import math
import random

import pytest
import torch

from oracle import paged_oracle as O
from paged_cases import BF, E4M3, F32, F64, Case, bound
from paged_schedule import SCHEDULED

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def hip():
    from gpt_fast import _hip

    _hip.load()
    return _hip


@pytest.fixture(autouse=True)
def _no_device_error():
    from gpt_fast import _hip

    yield
    _hip.raise_on_device_error()


def rnd(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF)


def bits(t):
    return t.cpu().contiguous().view(torch.uint8)


# ------------------------------------------------------------------------------------------------ write

def written(case, hq, rope, rot, interleaved, qkv, dtype=F32):
    """(q, {(page, slot): (k, v)}) in `dtype` of the rows that have a place."""
    hkv, hd = case.hkv, case.hd
    q, rows = {}, {}
    for r, _, pos, page, slot in O.places(case.table, case.lengths, case.starts, case.page):
        x = qkv[r].view(hq + 2 * hkv, hd).to(dtype)
        if rope is not None:
            x = torch.cat([O.turn(x[:hq + hkv], rope[pos], rot, interleaved, dtype), x[hq + hkv:]])
        q[r], rows[page, slot] = x[:hq], (x[hq:hq + hkv], x[hq + hkv:])
    return q, rows


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("hq,hkv,hd,page,rot,table,lengths,new", [
    (8, 1, 128, 16, 128, BF, [17], None),                                # a rank shard's decode step
    (4, 2, 64, 32, 32, F32, [1, 0, 33, 64, 31], None),                   # empty places, first and last slots of pages
    (3, 3, 64, 16, 64, F32, [5, 40, 16, 16], [5, 3, 0, 16]),             # prompts, a portion, a sequence without rows
    (14, 2, 64, 256, 16, BF, [300, 2], [299, 2]),
    (2, 1, 128, 64, None, BF, [70, 64], [70, 1]),                        # nothing turned
    (16, 8, 128, 128, 64, F32, [129] + [3] * 69, None),                  # more sequences than a wave has lanes
    (2, 1, 64, 64, 48, F32, [1500, 700, 1103], [1500, 0, 1101]),         # workgroups of several tokens
    (1, 1, 128, 16, 128, BF, [1300, 30], [1290, 30]),
])
def test_write(hip, e4m3, interleaved, hq, hkv, hd, page, rot, table, lengths, new):
    case = Case(lengths, hkv, hd, page, e4m3, seed=3, new=new)
    cache, batch = case.on(DEV, hq, rows=case.rows + 3)
    width = (hq + 2 * hkv) * hd
    behind = 0 if new is None else 3
    buf = rnd(case.rows + behind, width + 24, seed=4)
    buf[0, hq * hd:hq * hd + 8] *= 100.0
    qkv = buf[:, 8:8 + width]
    rope = None
    if rot:
        g = torch.Generator().manual_seed(5)
        angle = torch.rand(max(lengths), rot // 2, generator=g) * 6.28
        rope = torch.stack([angle.cos(), angle.sin()], -1).to(table)
    k0, v0 = case.k.clone(), case.v.clone()
    s0 = None if case.scales is None else case.scales.clone()
    dev = buf.to(DEV)
    q = torch.full((case.rows + behind, hq * hd + 8), 7.0, dtype=BF, device=DEV)
    cache.write(batch, dev[:, 8:8 + width], q[:, :hq * hd], None if rope is None else rope.to(DEV), interleaved)
    assert torch.equal(bits(dev), bits(buf)), "qkv is read only"
    want_q, rows = written(case, hq, rope, rot, interleaved, qkv)
    exact_q, exact_rows = written(case, hq, rope, rot, interleaved, qkv, F64)
    expect = torch.full(q.shape, 7.0, dtype=BF)
    for r, x in want_q.items():
        expect[r, :hq * hd] = x.reshape(-1).to(BF)
        # against 64 bits: half a step of bf16, and 2^-24 of each product and the sum (products of at most |x| each)
        near = 2.0 ** -8 * exact_q[r].abs() + 4 * 2.0 ** -24 * qkv[r].view(-1, hd)[:hq].double().abs().amax(-1, keepdim=True)
        assert ((q[r, :hq * hd].cpu().double().view(hq, hd) - exact_q[r]).abs() <= near).all()
    assert torch.equal(bits(q), bits(expect)), "q, and nothing besides"
    for (p, slot), kv in rows.items():
        for which, pages in enumerate((k0, v0)):
            if e4m3:
                pages[p, :, slot], s0[p, :, which, slot] = O.quantise(kv[which])
            else:
                pages[p, :, slot] = kv[which].to(BF)
    assert torch.equal(bits(cache.k_pages), bits(k0)) and torch.equal(bits(cache.v_pages), bits(v0)), "pages: these rows, nothing besides"
    if e4m3:
        assert torch.equal(cache.scales.cpu(), s0)
        for (p, slot), kv in exact_rows.items():
            got = O.values(cache.k_pages[p:p + 1, :, slot:slot + 1].cpu(), cache.scales[p:p + 1, :, :, slot:slot + 1].cpu())[0, :, 0]
            step = torch.exp2(s0[p, :, 0, slot].double() - 127)[:, None]
            near = torch.maximum(2.0 ** -4 * kv[0].abs(), 2.0 ** -10 * step) * (1 + 2.0 ** -20) + 2.0 ** -20 * step
            assert ((got - kv[0]).abs() <= near).all()


@pytest.mark.parametrize("interleaved", [True, False])
def test_write_in_place_gives_the_same_bits(hip, interleaved):
    hq, hkv, hd = 6, 2, 128
    case = Case([40, 21], hkv, hd, 16, False, new=[17, 21])
    cache, batch = case.on(DEV, hq)
    other, _ = case.on(DEV, hq)
    qkv = rnd(case.rows, (hq + 2 * hkv) * hd, seed=1).to(DEV)
    rope = torch.randn(64, hd // 2, 2, generator=torch.Generator().manual_seed(2)).to(DEV)
    q = torch.empty(case.rows, hq * hd, dtype=BF, device=DEV)
    cache.write(batch, qkv, q, rope, interleaved)
    mine = qkv.clone()
    other.write(batch, mine, mine[:, :hq * hd], rope, interleaved)
    assert torch.equal(bits(mine[:, :hq * hd]), bits(q)) and torch.equal(mine[:, hq * hd:], qkv[:, hq * hd:])
    assert torch.equal(bits(other.k_pages), bits(cache.k_pages)) and torch.equal(bits(other.v_pages), bits(cache.v_pages))


def test_write_of_values_that_are_not_finite_or_far_apart(hip):
    """Rows of zeros, with infinities and NaN, of the smallest and the largest numbers."""
    hq, hkv, hd = 1, 1, 64
    n = 9
    case = Case([n], hkv, hd, 16, True, new=[n])
    cache, batch = case.on(DEV, hq)
    qkv = rnd(n, 3 * hd, seed=1)
    k = qkv[:, hd:2 * hd]
    k[0] = 0
    k[1, 3], k[1, 60] = math.inf, -math.inf
    k[2, 5] = math.nan
    k[3] = math.nan
    k[4] *= 1e-38
    k[5] *= 3e37
    k[6] = 448.0
    k[7, 0] = 452.0          # the exponent is one larger: 226
    k[8] = torch.logspace(-6, 2, hd).to(BF)
    cache.write(batch, qkv.to(DEV), torch.empty(n, hd, dtype=BF, device=DEV))
    page = int(case.table[0, 0])
    for which, pages in enumerate((cache.k_pages, cache.v_pages)):
        want, byte = O.quantise(qkv[:, (1 + which) * hd:(2 + which) * hd].float())
        got = pages[page, 0, :n].cpu()
        assert torch.equal(cache.scales[page, 0, which, :n].cpu(), byte)
        assert torch.equal(got.float().isnan(), want.float().isnan())
        assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))


def test_rows_and_pages_out_of_range_are_left_alone(hip):
    hq, hkv, hd, page = 2, 1, 64, 16
    case = Case([20, 20, 20, 20], hkv, hd, page, False, new=[2, 2, 2, 2])
    cache, batch = case.on(DEV, hq)
    batch.table[0, 1] = -1                     # both rows of sequence 0
    batch.table[1, 1] = case.n_pages           # and of 1
    batch.lengths[2] = 1                       # its first row would be at position -1
    batch.lengths[3] = case.table.shape[1] * page + 1     # its last row has no page in the table
    table, lengths = batch.table.cpu(), batch.lengths.tolist()
    table[3, 2:] = table[3, 0]
    batch.table[3, 2:] = table[3, 0]
    qkv = rnd(8, 4 * hd, seed=2)
    q = torch.full((8, hq * hd), 5.0, dtype=BF, device=DEV)
    k0 = cache.k_pages.clone()
    cache.write(batch, qkv.to(DEV), q)
    with pytest.raises(hip.LadderHipError, match="outside"):
        hip.raise_on_device_error(DEV)
    there = [(r, p, s) for r, b, pos, p, s in O.places(table, lengths, case.starts, page) if 0 <= p < case.n_pages]
    assert [t[0] for t in there] == [5, 6]
    want_q, want_k = torch.full((8, hq * hd), 5.0, dtype=BF), k0.cpu()
    for r, p, s in there:
        want_q[r], want_k[p, :, s] = qkv[r, :hq * hd], qkv[r, hq * hd:(hq + 1) * hd].view(1, hd)
    assert torch.equal(bits(q), bits(want_q)) and torch.equal(bits(cache.k_pages), bits(want_k))
    # read back: the same two rows
    a, b = (torch.full((8, hd), 9.0, dtype=BF, device=DEV) for _ in range(2))
    cache.read(batch, a, b)
    with pytest.raises(hip.LadderHipError, match="outside"):
        hip.raise_on_device_error(DEV)
    assert [r for r in range(8) if not (a[r] == 9).all()] == [5, 6]
    # positions without an angle
    case = Case([9], hkv, hd, page, False)
    cache, batch = case.on(DEV, hq)
    q.fill_(5.0)
    cache.write(batch, qkv[:1].to(DEV), q[:1], torch.ones(8, hd // 2, 2, device=DEV))
    with pytest.raises(hip.LadderHipError, match="position"):
        hip.raise_on_device_error(DEV)
    assert (q == 5).all()


# ------------------------------------------------------------------------------------------------ read

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hkv,hd,page,lengths,new", [
    (1, 128, 16, [1], None), (2, 64, 32, [33, 0, 32, 5], None), (8, 128, 64, [130, 64, 1], [130, 64, 1]), (3, 64, 16, [50, 7], [20, 0]),
    (1, 64, 256, [1] * 130, [1] * 130), (24, 128, 128, [300], [300]), (1, 64, 32, [1700, 3, 0, 1000], [1700, 2, 0, 999]),
])
def test_read(hip, e4m3, hkv, hd, page, lengths, new):
    case = Case(lengths, hkv, hd, page, e4m3, seed=6, new=new)
    cache, batch = case.on(DEV, hkv, rows=case.rows + 2)
    n = case.rows + (0 if new is None else 2)
    k, v = (torch.full((n, hkv * hd + 8 * i), 3.0, dtype=BF, device=DEV) for i in (1, 2))
    cache.read(batch, k[:, :hkv * hd], v[:, :hkv * hd])
    for which, got in enumerate((k, v)):
        want = torch.full(got.shape, 3.0, dtype=BF)
        x = O.values((case.k, case.v)[which], case.scales, which)
        for r, _, _, p, slot in O.places(case.table, case.lengths, case.starts, page):
            want[r, :hkv * hd] = x[p, :, slot].reshape(-1).to(BF)       # (exact)
        assert torch.equal(bits(got), bits(want))


# ------------------------------------------------------------------------------------------------ attention

WEIGHT = 2.0 ** -16     # decode: a weight enters as two bf16 numbers; prompts see the tests below


def attend(case, hq, seed=11, scale=None, q_scale=1.0, weight=WEIGHT, behind=0, pad=8):
    cache, batch = case.on(DEV, hq, rows=None if case.starts is None else case.rows + behind)
    q = rnd(case.rows + behind, hq * case.hd, seed=seed, scale=q_scale)
    buf = torch.full((q.shape[0], hq * case.hd + pad), 3.0, dtype=BF, device=DEV)
    src = torch.full((q.shape[0], hq * case.hd + 2 * pad), 3.0, dtype=BF, device=DEV)
    src[:, pad:pad + q.shape[1]] = q.to(DEV)
    cache.attend(batch, src[:, pad:pad + q.shape[1]], buf[:, :q.shape[1]], scale)
    got = buf.cpu()
    assert (got[:, q.shape[1]:] == 3).all()
    y, spread, size = case.oracle(q, hq, scale)
    got = got[:, :q.shape[1]].double().view(y.shape)
    rows = ~y.isnan().all(-1).all(-1)
    assert (got[~rows] == 3).all(), "rows behind the last sequence are left as they were"
    near = bound(y, spread, size, max(case.lengths + [1]), case.hd, weight)
    off = ((got - y).abs() / near)[rows]
    assert not off.isnan().any() and (off.numel() == 0 or off.max() <= 1), f"{off.max():.2f} of what rounding explains"
    return cache, batch, q, got


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 1, 128), (1, 1, 64), (6, 2, 128), (14, 2, 64), (16, 1, 128), (3, 3, 64), (40, 2, 64), (17, 1, 128)])
@pytest.mark.parametrize("page,lengths", [(16, [1, 0, 15, 16, 17, 33]), (64, [128, 31, 32, 0, 257, 63]), (256, [513, 255])])
def test_decode(hip, e4m3, hq, hkv, hd, page, lengths):
    attend(Case(lengths, hkv, hd, page, e4m3, seed=hq + page), hq)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths,hq,hkv,hd,page", [
    ([9001], 4, 1, 128, 16), ([5000, 1, 0, 700], 2, 2, 64, 32), ([33] * 300, 2, 1, 64, 16), ([0] * 70 + [100], 4, 4, 128, 64),
    ([2049, 4095], 8, 1, 128, 128), ([0, 0], 8, 1, 128, 16),
    ([20000, 300, 0, 9000], 2, 1, 128, 64), ([700] * 5 + [3], 20, 1, 64, 16), ([1500, 3, 40, 900] * 7, 8, 8, 64, 32), ([26000], 17, 1, 128, 256),
])
def test_decode_of_long_and_of_many_sequences(hip, e4m3, lengths, hq, hkv, hd, page):
    attend(Case(lengths, hkv, hd, page, e4m3, seed=5), hq)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 1, 128), (12, 4, 64), (17, 1, 128)])
def test_decode_of_one_sequence(hip, e4m3, hq, hkv, hd):
    """Around a tile, a tile for each wave, two workers, and from single tiles of a worker's waves to several."""
    for n in (0, 1, 32, 33, 96, 128, 129, 160, 161, 200, 255, 256, 257, 300, 511, 513, 2047, 2049, 2100, 4000, 8192, 8193, 8300):
        attend(Case([n], hkv, hd, 64, e4m3, seed=n), hq)


PROMPT = 2.0 ** -8      # prompts: a weight enters as one bf16 number


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hq,hkv,hd,page,lengths,new", [
    (8, 1, 128, 16, [1], [1]), (4, 1, 64, 32, [33, 5], [33, 5]), (2, 2, 128, 64, [200, 64, 65], [70, 0, 65]),
    (6, 2, 64, 16, [31, 32, 33, 0, 1], [31, 32, 33, 0, 1]), (12, 4, 128, 256, [300, 17], [40, 17]), (5, 1, 64, 16, [90, 250], [90, 129]),
    (16, 1, 128, 128, [700], [3]), (1, 1, 128, 16, [64] * 70, [1, 2] * 35), (32, 8, 64, 16, [100, 77], [100, 77]),
    (8, 1, 128, 32, [3000], [65]), (4, 4, 64, 64, [0, 0, 2], [0, 0, 2]), (7, 1, 128, 16, [150], [150]),
])
def test_prompts(hip, e4m3, hq, hkv, hd, page, lengths, new):
    attend(Case(lengths, hkv, hd, page, e4m3, seed=7, new=new), hq, weight=PROMPT, behind=3)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,page,lengths,new", [
    (128, 16, [(37 * b) % 150 for b in range(90)], [min((37 * b) % 150, 1 + b % 7) for b in range(90)]),
    (64, 32, [5] * 100, [b % 12 for b in range(100)]),                                                      # many of them see no key at all
    (64, 64, [1100, 0, 700, 1], [90, 0, 400, 1]),
    (128, 32, [1300, 20], [1300, 20]),
])
def test_prompts_of_many_blocks(hip, e4m3, hd, page, lengths, new):
    """More than the chip holds at once, most of them short; the same bits again, also replayed."""
    hq, hkv = (16, 8) if len(lengths) > 10 else (32, 16)
    case = Case(lengths, hkv, hd, page, e4m3, seed=41, new=new)
    if len(lengths) > 10:
        cache, batch, q, got = attend(case, hq, weight=PROMPT, behind=2)
    else:
        cache, batch = case.on(DEV, hq)
        q = rnd(case.rows, hq * hd, seed=1)
    x = q.to(DEV)
    y = torch.full_like(x, 3)
    cache.attend(batch, x, y)
    want = y.clone()
    # against one sequence at a time, whose blocks are few
    for b, n in enumerate(new):
        if n:
            i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
            one = cache.batch(batch.table[b:b + 1], batch.lengths[b:b + 1], hq, starts=i(0, n), rows=n)
            at = slice(case.starts[b], case.starts[b] + n)
            off = (cache.attend(one, x[at], torch.empty_like(x[at])).float() - want[at].float()).abs()
            assert off.max() <= 2.0 ** -6 * 4 and want[at].isfinite().all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(batch, x, y)
    for _ in range(5):
        y.fill_(3)
        cache.attend(batch, x, y)
        assert torch.equal(y, want)
        y.fill_(3)
        graph.replay()
        assert torch.equal(y, want)


def test_rows_ahead_of_a_sequences_first_token_see_nothing(hip):
    """More rows than tokens: those at negative positions are zeros."""
    for e4m3 in (False, True):
        case = Case([3, 40], 1, 64, 16, e4m3, new=[5, 2])
        *_, got = attend(case, 2, weight=PROMPT)
        assert (got[:2] == 0).all() and (got[2] != 0).any()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [None, [40, 17]])
def test_scores_far_apart(hip, e4m3, new):
    """Scores of some hundreds, of both signs; a scale of one's own."""
    attend(Case([500, 77], 1, 128, 16, e4m3, seed=8, new=new, spread=4.0), 4, q_scale=6.0, weight=PROMPT if new else WEIGHT)
    attend(Case([500, 77], 1, 64, 16, e4m3, seed=9, new=new), 4, scale=1e-3, weight=PROMPT if new else WEIGHT)
    attend(Case([500, 77], 1, 64, 16, e4m3, seed=9, new=new), 4, scale=1.0, weight=PROMPT if new else WEIGHT)


@pytest.mark.parametrize("new", [None, [2, 30]])
@pytest.mark.parametrize("e4m3", [False, True])
def test_one_key_that_stands_out(hip, e4m3, new):
    """The winning key first, last, at a tile's or a page's edge: the output is its value, whatever stood before and after."""
    hq, hkv, hd, page = 2, 1, 128, 16
    n = 300
    for at in (0, 15, 16, 31, 32, 127, 128, 255, 269 if new else 299):
        case = Case([5, n], hkv, hd, page, e4m3, seed=at, new=new)
        k = torch.zeros(hd)
        k[7] = 256.0
        p, slot = int(case.table[1, at // page]), at % page
        case.k[p, 0, slot] = (k / 64.0 if e4m3 else k).to(case.k.dtype)
        if e4m3:
            case.scales[p, 0, 0, slot] = 127 + 6
        cache, batch = case.on(DEV, hq)
        q = torch.zeros(case.rows, hq * hd, dtype=BF)
        q[:, 7::hd] = 64.0
        y = torch.empty(case.rows, hq * hd, dtype=BF, device=DEV)
        cache.attend(batch, q.to(DEV), y)
        want = O.values(case.v, case.scales, 1)[p, 0, slot].to(BF)
        assert torch.equal(y[-1].cpu(), want.repeat(hq)), at


@pytest.mark.parametrize("new", [None, [1, 20]])
@pytest.mark.parametrize("e4m3", [False, True])
def test_pages_out_of_range_are_not_there(hip, e4m3, new):
    case = Case([40, 70], 2, 64, 16, e4m3, seed=3, new=new)
    case.table[1, 1], case.table[1, 3] = case.n_pages, -1
    attend(case, 4, weight=PROMPT if new else WEIGHT)
    with pytest.raises(hip.LadderHipError, match="page"):
        hip.raise_on_device_error(DEV)
    case.table[0, :] = 1 << 30       # none of a sequence's: zeros
    *_, got = attend(case, 4, weight=PROMPT if new else WEIGHT)
    assert (got[0] == 0).all()
    with pytest.raises(hip.LadderHipError, match="page"):
        hip.raise_on_device_error(DEV)
    # a length beyond the table's pages: as many keys as these hold
    case = Case([64, 64], 2, 64, 16, e4m3, seed=3, new=new)
    case.table = case.table[:, :4].contiguous()
    full = case.on(DEV, 4)
    q = rnd(case.rows, 4 * 64).to(DEV)
    want = full[0].attend(full[1], q, torch.empty_like(q)).clone()
    if new is None:
        full[1].lengths[1] = 65
        assert torch.equal(full[0].attend(full[1], q, torch.empty_like(q)), want)
        with pytest.raises(hip.LadderHipError, match="position"):
            hip.raise_on_device_error(DEV)
        full[1].lengths[1] = -3
        y = full[0].attend(full[1], q, torch.empty_like(q))
        assert torch.equal(y[0], want[0]) and (y[1] == 0).all()


def test_not_a_number_where_it_is_seen(hip):
    """NaN in a key or a value of one sequence is that sequence's alone; an infinite value goes through."""
    for new in (None, [3, 4]):
        case = Case([40, 50], 1, 64, 16, False, seed=4, new=new)
        page = int(case.table[0, 0])
        case.v[page, 0, 2, 5] = math.nan
        case.v[page, 0, 3, 6] = math.inf
        cache, batch = case.on(DEV, 2)
        q = rnd(case.rows, 128).to(DEV)
        y = cache.attend(batch, q, torch.empty_like(q)).view(case.rows, 2, 64)
        first = 1 if new is None else 3
        assert y[:first, :, 5].isnan().all() and (y[:first, :, 6] == math.inf).all()
        assert y[:first, :, :5].isfinite().all() and y[first:].isfinite().all()
        case.k[page, 0, 1, 0] = math.nan
        cache, batch = case.on(DEV, 2)
        y = cache.attend(batch, q, torch.empty_like(q))
        assert y[:first].isnan().all() and y[first:].isfinite().all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hq,hkv,hd,page,lengths,new", [
    (8, 1, 128, 16, [90, 5], [90, 5]), (2, 2, 64, 32, [200], [200]), (4, 1, 128, 64, [700], [700]), (3, 1, 64, 16, [900, 60], [900, 60]),
    (8, 1, 128, 32, [3000], [65]), (1, 1, 64, 64, [2000], [100]),
])
def test_what_later_tokens_hold_does_not_reach_earlier_rows(hip, e4m3, hq, hkv, hd, page, lengths, new):
    """NaN and infinities in keys and values of a prompt's later tokens, the first of them in the middle of its rows."""
    weight = PROMPT
    clean = Case(lengths, hkv, hd, page, e4m3, seed=21, new=new)
    q = rnd(clean.rows, hq * hd, seed=22)
    y, spread, size = clean.oracle(q, hq)
    near = bound(y, spread, size, max(lengths), hd, weight)
    for back in (1, 2, new[0] // 2, new[0] - 1):
        case = Case(lengths, hkv, hd, page, e4m3, seed=21, new=new)
        at = lengths[0] - back                # the first such token
        for pos in range(at, lengths[0], 3 if back > 2 else 1):
            p, slot = int(case.table[0, pos // page]), pos % page
            case.v[p, :, slot, 3] = math.nan
            if not e4m3:
                case.v[p, :, slot, hd - 1] = -math.inf
            if pos % 2:
                case.k[p, :, slot, 1] = math.nan
        cache, batch = case.on(DEV, hq)
        got = cache.attend(batch, q.to(DEV), torch.empty(case.rows, hq * hd, dtype=BF, device=DEV)).cpu().double().view(y.shape)
        first = new[0] - back                 # the first row that sees it
        rows = torch.ones(case.rows, dtype=torch.bool)
        rows[first:new[0]] = False
        off = ((got - y).abs() / near)[rows]
        assert not off.isnan().any() and off.max() <= 1, (back, f"{off.max():.2f} of what rounding explains")
        assert got[first:new[0], :, 3].isnan().all()
        assert e4m3 or not got[first:new[0], :, hd - 1].isfinite().any()


@pytest.mark.parametrize("new", [None, [40, 17]])
@pytest.mark.parametrize("scale", [1e-37, 1.2e-38, 1e38])
def test_smallest_and_largest_scales(hip, new, scale):
    """A scale that makes all weights alike gives means of the values; one beyond 2^64 is refused."""
    case = Case([100, 77], 1, 64, 16, False, seed=30, new=new)
    if scale > 1:
        with pytest.raises(hip.LadderHipError):
            attend(case, 2, scale=scale)
    else:
        attend(case, 2, scale=scale, weight=PROMPT if new else WEIGHT)


def test_fewer_rows_than_starts_says(hip):
    """They are what they are in the whole call, and the others stay as they were."""
    for e4m3 in (False, True):
        case = Case([30, 90, 20], 2, 64, 16, e4m3, seed=31, new=[30, 40, 20])
        cache, batch = case.on(DEV, 4)
        q = rnd(90, 256, seed=1).to(DEV)
        whole = cache.attend(batch, q, torch.empty_like(q)).clone()
        for rows in (1, 29, 30, 31, 69, 71):
            y = torch.full_like(q, 3)
            cache.attend(batch, q[:rows], y[:rows])
            y0, spread, size = case.oracle(q.cpu(), 4)
            near = bound(y0, spread, size, 90, 64, PROMPT)
            assert ((y.cpu().double().view(90, 4, 64) - y0).abs() <= near)[:rows].all() and (y[rows:] == 3).all()
        assert whole.isfinite().all()


def test_batches_are_not_changed_under_their_addresses(hip):
    case = Case([20, 20], 2, 64, 16, False)
    cache, batch = case.on(DEV, 4)
    with pytest.raises(AttributeError, match="replaced"):
        batch.lengths = batch.lengths.clone()
    with pytest.raises(AssertionError, match="expanded"):
        cache.batch(batch.table[:1].expand(2, -1), batch.lengths, 4)
    one = cache.batch(batch.table[:1].expand(1, -1), batch.lengths[:1], 4)      # a single row is its own
    q = rnd(2, 256).to(DEV)
    assert torch.equal(cache.attend(one, q[:1], torch.empty_like(q[:1])), cache.attend(batch, q, torch.empty_like(q))[:1])
    wide = torch.cat([batch.table, batch.table * 0 - 5], 1)                     # rows of a wider table
    view = cache.batch(wide[:, :batch.table.shape[1]], batch.lengths, 4)
    assert torch.equal(cache.attend(view, q, torch.empty_like(q)), cache.attend(batch, q, torch.empty_like(q)))
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="capture"):
            cache.batch(batch.table, batch.lengths, 4)
    with pytest.raises(hip.LadderHipError):
        cache.attend(batch, q, q)


def test_offsets_beyond_32_bits(hip):
    """Pages whose bytes and whose elements lie beyond 2^32."""
    hq, hkv, hd, page = 8, 8, 128, 256
    n_pages = (1 << 32) // (hkv * page * hd) + 3
    from gpt_fast.utils import PagedKVCache
    for dtype in (BF, E4M3):
        cache = PagedKVCache(n_pages, page, hkv, hd, dtype, device=DEV)
        table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32, device=DEV)
        n = 2 * page + 9
        i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
        batch = cache.batch(table, i(n), hq, starts=i(0, n), rows=n)
        qkv = rnd(n, (hq + 2 * hkv) * hd, seed=1).to(DEV)
        q, k, v, y = (torch.empty(n, hq * hd, dtype=BF, device=DEV) for _ in range(4))
        cache.write(batch, qkv, q)
        cache.read(batch, k, v)
        cache.attend(batch, q, y)
        one = cache.batch(table, i(n), hq)
        y1 = cache.attend(one, q[-1:], torch.empty_like(q[-1:]))
        small = PagedKVCache(3, page, hkv, hd, dtype, device=DEV)
        t2 = i(1, 2, 0)[None]
        b2 = small.batch(t2, i(n), hq, starts=i(0, n), rows=n)
        q2, k2, v2, y2 = (torch.empty_like(q) for _ in range(4))
        small.write(b2, qkv, q2)
        small.read(b2, k2, v2)
        small.attend(b2, q2, y2)
        for a, b in ((q, q2), (k, k2), (v, v2), (y, y2), (y1, small.attend(small.batch(t2, i(n), hq), q2[-1:], torch.empty_like(q2[-1:])))):
            assert torch.equal(a, b)
        if dtype == BF:
            assert torch.equal(k, qkv[:, hq * hd:(hq + hkv) * hd])
        del cache, batch, one
        torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", [BF, E4M3])
def test_prompts_then_tokens_as_a_server_runs_them(hip, dtype):
    """Three sequences: prompts together in one call, a portion for one of them, then tokens in a captured graph whose table and
    lengths advance on the device, one sequence leaving and its page going to another; every step against the oracle on what the
    cache holds, read back."""
    from gpt_fast.utils import PagedKVCache
    hq, hkv, hd, page = 4, 2, 64, 16
    cache = PagedKVCache(24, page, hkv, hd, dtype, device=DEV)
    g = torch.Generator().manual_seed(1)
    angle = torch.rand(200, hd // 2, generator=g) * 6.28
    rope = torch.stack([angle.cos(), angle.sin()], -1).to(BF).to(DEV)
    table = torch.randperm(24, generator=g).to(torch.int32).view(3, 8)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    dev_table = table.to(DEV)

    def check(batch, q, y, lengths, starts, weight):
        whole = cache.batch(dev_table, i(lengths), hq, starts=i([sum(lengths[:b]) for b in range(4)]), rows=max(1, sum(lengths)))
        k, v = (torch.empty(sum(lengths), hkv * hd, dtype=BF, device=DEV) for _ in range(2))
        cache.read(whole, k, v)
        kp, vp = (torch.zeros(24, hkv, page, hd, dtype=F64) for _ in range(2))
        for r, _, _, p, s in O.places(table, lengths, whole.starts.tolist(), page):
            kp[p, :, s], vp[p, :, s] = k[r].cpu().double().view(hkv, hd), v[r].cpu().double().view(hkv, hd)
        want, spread, size = O.attention(q.cpu().view(-1, hq, hd), kp, vp, table, lengths, starts, hd ** -0.5)
        off = (y.cpu().double().view(want.shape) - want).abs() / bound(want, spread, size, max(lengths), hd, weight)
        assert off.max() <= 1

    lengths, new = [30, 17, 50], [30, 17, 50]
    for lengths, new in (([30, 17, 50], [30, 17, 50]), ([30, 37, 50], [0, 20, 0])):
        starts = [sum(new[:b]) for b in range(4)]
        batch = cache.batch(dev_table, i(lengths), hq, starts=i(starts), rows=starts[-1])
        qkv = rnd(starts[-1], (hq + 2 * hkv) * hd, seed=sum(lengths)).to(DEV)
        q, y = (torch.empty(starts[-1], hq * hd, dtype=BF, device=DEV) for _ in range(2))
        cache.write(batch, qkv, q, rope)
        cache.attend(batch, q, y)
        check(batch, q, y, lengths, starts, PROMPT)
    step = cache.batch(dev_table, i(lengths), hq)
    qkv = torch.zeros(3, (hq + 2 * hkv) * hd, dtype=BF, device=DEV)
    y = torch.empty(3, hq * hd, dtype=BF, device=DEV)

    def once():
        cache.write(step, qkv, qkv[:, :hq * hd], rope)
        cache.attend(step, qkv[:, :hq * hd], y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    k0, v0 = cache.k_pages.clone(), cache.v_pages.clone()
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    cache.k_pages.copy_(k0)
    cache.v_pages.copy_(v0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once()
    for n in range(12):
        fresh = rnd(3, qkv.shape[1], seed=100 + n).to(DEV)
        lengths = [x + 1 if x else 0 for x in lengths]
        if n == 5:
            lengths[0] = 0                        # leaves
            table[1, 5:7] = table[0, :2]          # its pages are another's
            dev_table.copy_(table)
        step.lengths.copy_(i(lengths))
        qkv.copy_(fresh)
        graph.replay()
        check(step, qkv[:, :hq * hd], y, lengths, None, WEIGHT)
        graph_y = y.clone()
        qkv.copy_(fresh)
        once()                                    # eagerly: the same bits
        assert torch.equal(y, graph_y)
    hip.raise_on_device_error(DEV)


def test_two_batches_on_two_streams(hip):
    """Each with a scratch of its own, at once, over and over: the bits of each alone."""
    case = Case([3000, 17, 900], 2, 128, 16, False, seed=2)
    q = rnd(3, 8 * 128).to(DEV)
    work = []
    for _ in range(2):
        cache, batch = case.on(DEV, 8)
        work.append((cache, batch, torch.empty_like(q), torch.cuda.Stream()))
    want = work[0][0].attend(work[0][1], q, torch.empty_like(q)).clone()
    torch.cuda.synchronize()
    for _ in range(20):
        for cache, batch, y, stream in work:
            with torch.cuda.stream(stream):
                y.zero_()
                cache.attend(batch, q, y)
    torch.cuda.synchronize()
    assert all(torch.equal(w[2], want) for w in work)


def test_the_contiguous_caches_numbers(hip):
    """On one sequence the paged operators do what lr_rope_kv_write, lr_attn_prefill and lr_attn_decode do: the same cached bits, and outputs
    within the rounding of either."""
    from gpt_fast.utils import precompute_freqs_cis
    hq, hkv, hd, page, n = 8, 2, 128, 32, 150
    case = Case([n], hkv, hd, page, False, new=[n])
    cache, batch = case.on(DEV, hq)
    rope = precompute_freqs_cis(256, hd, 500000).to(DEV)
    qkv = rnd(n, (hq + 2 * hkv) * hd, seed=3).to(DEV)
    q, y, y0 = (torch.empty(n, hq * hd, dtype=BF, device=DEV) for _ in range(3))
    cache.write(batch, qkv, q, rope)
    kc, vc = (torch.zeros(1, hkv, 160, hd, dtype=BF, device=DEV) for _ in range(2))
    dense = qkv.clone()
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    hip.rope_kv_write(dense, rope, False, pos, kc, vc, 1, n, hq, hkv, hd)
    k, v = (torch.empty(n, hkv * hd, dtype=BF, device=DEV) for _ in range(2))
    cache.read(batch, k, v)
    assert torch.equal(q, dense[:, :hq * hd])
    assert torch.equal(k.view(n, hkv, hd).transpose(0, 1), kc[0, :, :n]) and torch.equal(v.view(n, hkv, hd).transpose(0, 1), vc[0, :, :n])
    cache.attend(batch, q, y)
    hip.attn_prefill(dense, kc, vc, pos, y0, 1, n, hq, hkv, hd)
    clean = lambda t: torch.nan_to_num(t.cpu().double())
    want, spread, size = O.attention(q.cpu().view(n, hq, hd), clean(cache.k_pages), clean(cache.v_pages), case.table, [n], [0, n], hd ** -0.5)
    near = bound(want, spread, size, n, hd, PROMPT)
    for got in (y, y0):
        assert ((got.cpu().double().view(want.shape) - want).abs() <= near).all()


def test_refusals(hip):
    case = Case([20, 20], 2, 64, 16, False)
    cache, batch = case.on(DEV, 4)
    q = rnd(2, 256).to(DEV)
    y = torch.empty_like(q)
    for bad in (q.float(), q[:, :128], q.t().contiguous().t(), q.cpu()):
        with pytest.raises(ValueError):
            cache.attend(batch, bad, y)
        with pytest.raises(ValueError):
            cache.attend(batch, q, bad)
    with pytest.raises(ValueError):
        cache.attend(batch, q[:1], y)
    with pytest.raises(hip.LadderHipError):
        cache.attend(batch, q[:1], y[:1])                # one row per sequence
    with pytest.raises(hip.LadderHipError):
        cache.attend(batch, q, y, scale=0.0)
    with pytest.raises(ValueError, match="rows"):
        cache.attend(batch, q.repeat(2, 1), y.repeat(2, 1))
    other, _ = Case([20, 20], 1, 64, 16, False).on(DEV, 4)
    with pytest.raises(ValueError, match="pages"):
        other.attend(batch, q, y)
    with pytest.raises(ValueError):
        cache.write(batch, rnd(2, 8 * 64).to(DEV), q, torch.zeros(8, 32, 2, dtype=torch.float16, device=DEV))
    with pytest.raises(hip.LadderHipError):
        cache.write(batch, rnd(2, 8 * 64).to(DEV), q, torch.zeros(8, 12, 2, device=DEV))
    with pytest.raises(hip.LadderHipError, match="not served"):
        cache.batch(batch.table, batch.lengths, 5)
    with pytest.raises(AssertionError):
        cache.batch(batch.table.long(), batch.lengths, 4)


# ------------------------------------------------------------------------------------------------ precision

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hq,hkv,hd,page,lengths,new", [
    (4, 1, 128, 16, [90, 33], [90, 33]), (2, 2, 64, 32, [200, 65], [70, 65]),        # four waves
    (12, 1, 64, 64, [700], [700]), (2, 2, 128, 16, [640, 130], [400, 1]),            # eight
    (8, 1, 128, 32, [3000], [65]), (4, 1, 64, 16, [2500, 700], [9, 40]),             # parts joined
])
def test_prompts_weights_have_two_numbers(hip, e4m3, hq, hkv, hd, page, lengths, new):
    """A weight enters the matrix cores with 2^-16 of it lost, as in decode and as in lr_attn_prefill: one bf16 number would lose 2^-8."""
    attend(Case(lengths, hkv, hd, page, e4m3, seed=51, new=new), hq, weight=WEIGHT)


def test_both_caches_prompts_are_as_precise(hip):
    """lr_attn_prefill on dense keys and the paged operator on the same ones, both within what two bf16 numbers per weight explain."""
    hq, hkv, hd, n = 8, 2, 128, 150
    case = Case([n], hkv, hd, 32, False, new=[n])
    cache, batch, q, _ = attend(case, hq, weight=WEIGHT)
    k, v = (torch.empty(n, hkv * hd, dtype=BF, device=DEV) for _ in range(2))
    cache.read(batch, k, v)
    kc, vc = (torch.zeros(1, hkv, 160, hd, dtype=BF, device=DEV) for _ in range(2))
    kc[0, :, :n], vc[0, :, :n] = k.view(n, hkv, hd).transpose(0, 1), v.view(n, hkv, hd).transpose(0, 1)
    qkv = torch.zeros(n, (hq + 2 * hkv) * hd, dtype=BF, device=DEV)
    qkv[:, :hq * hd] = q.to(DEV)
    y = torch.empty(n, hq * hd, dtype=BF, device=DEV)
    hip.attn_prefill(qkv, kc, vc, torch.arange(n, dtype=torch.int32, device=DEV), y, 1, n, hq, hkv, hd)
    want, spread, size = case.oracle(q, hq)
    assert ((y.cpu().double().view(want.shape) - want).abs() <= bound(want, spread, size, n, hd, WEIGHT)).all()


@pytest.mark.parametrize("lengths,new,hq,hkv", [([90], [20], 4, 1), ([700], [300], 4, 2), ([3000], [40], 8, 1), ([700], [700], 12, 1)])
def test_infinite_values_go_through_prompts(hip, lengths, new, hq, hkv):
    """An infinite value that all of a call's rows see, or some of them: infinite for those, nothing to the others, the other dimensions as they are."""
    n, first = lengths[0], lengths[0] - new[0]
    for at in (0, 37, first, first + new[0] // 2, n - 1):
        case = Case(lengths, hkv, 64, 16, False, seed=52, new=new)
        q = rnd(case.rows, hq * 64, seed=53)
        want, spread, size = case.oracle(q, hq)
        page, slot = int(case.table[0, at // 16]), at % 16
        case.v[page, :, slot, 7], case.v[page, :, slot, 9] = math.inf, -math.inf
        cache, batch = case.on(DEV, hq)
        y = cache.attend(batch, q.to(DEV), torch.empty(case.rows, hq * 64, dtype=BF, device=DEV)).cpu().double().view(want.shape)
        sees = torch.arange(new[0]) + first >= at
        assert (y[sees][:, :, 7] == math.inf).all() and (y[sees][:, :, 9] == -math.inf).all(), at
        near = bound(want, spread, size, n, 64, WEIGHT)
        off = (y - want).abs() / near
        others = [d for d in range(64) if d not in (7, 9)]
        assert off[:, :, others].max() <= 1 and (not (~sees).any() or off[~sees].max() <= 1), at


# ------------------------------------------------------------------------------------------------ what nobody has written

@pytest.mark.parametrize("new", [None, [3, 1, 0, 16, 20, 33]])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 1, 128), (6, 2, 64)])
@pytest.mark.parametrize("page,lengths", [(16, [1, 0, 15, 16, 17, 33]), (64, [128, 31, 32, 0, 257, 63]), (256, [513, 255, 0, 1, 20, 40])])
@pytest.mark.parametrize("byte", [255, 0])
def test_scales_of_slots_that_no_sequence_has(hip, new, hq, hkv, hd, page, lengths, byte):
    """Memory that was there already holds any byte behind a sequence's last token: 255 stands for no power of two."""
    new = None if new is None else [min(a, b) for a, b in zip(new, lengths)]
    case = Case(lengths, hkv, hd, page, True, seed=54, new=new)
    case.scales = torch.where(case.scales == 254, torch.tensor(byte, dtype=torch.uint8), case.scales)
    attend(case, hq)


# ------------------------------------------------------------------------------------------------ lengths and starts that a table or a call does not hold

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hq,hkv,hd,page,pages,lengths,new", [
    (4, 2, 64, 16, 4, [70, 64], [10, 5]),               # four rows of sequence 0 have a place
    (4, 1, 128, 16, 4, [64, 100], [64, 40]), (2, 1, 64, 64, 20, [1300, 1281], [30, 2]), (4, 1, 128, 16, 3, [200], [20]),
])
def test_rows_of_a_sequence_longer_than_its_table(hip, e4m3, hq, hkv, hd, page, pages, lengths, new):
    """A row's position is what the length says, whether or not the table has all of the sequence: the keys that it has are those up to there."""
    held = [min(n, pages * page) for n in lengths]
    case = Case(held, hkv, hd, page, e4m3, seed=57, new=new)
    case.table = case.table[:, :pages].contiguous()
    case.lengths = lengths
    attend(case, hq)
    with pytest.raises(hip.LadderHipError, match="position"):
        hip.raise_on_device_error(DEV)


# ------------------------------------------------------------------------------------------------ long prompts

def long_prompts(hip, lengths, new, hq, hkv, hd, page, e4m3, gone=()):
    """attend() with the oracle over whole sequences at once; `gone`: (sequence, place in its table) of pages that are not there."""
    case = Case(lengths, hkv, hd, page, e4m3, seed=55, new=new)
    for b, i in gone:
        case.table[b, i] = case.n_pages + 7
    cache, batch = case.on(DEV, hq)
    q = rnd(case.rows, hq * hd, seed=56)
    y = cache.attend(batch, q.to(DEV), torch.empty(case.rows, hq * hd, dtype=BF, device=DEV)).cpu().double().view(-1, hq, hd)
    if gone:
        with pytest.raises(hip.LadderHipError, match="page"):
            hip.raise_on_device_error(DEV)
    clean = lambda x: torch.nan_to_num(x, nan=0.0)
    want, spread, size = O.attention_of_sequences(q.view(-1, hq, hd), clean(O.values(case.k, case.scales, 0)), clean(O.values(case.v, case.scales, 1)),
                                                  case.table, case.lengths, case.starts, hd ** -0.5)
    off = (y - want).abs() / bound(want, spread, size, max(lengths), hd, WEIGHT)
    assert off.max() <= 1, f"{off.max():.2f} of what rounding explains"


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths,new,hq,hkv,hd,page", [
    ([1300, 20], [1300, 20], 32, 8, 128, 32), ([2048], [600], 64, 8, 64, 64),                           # four waves: more blocks than CUs
    ([1100, 0, 700, 1], [90, 0, 400, 1], 32, 16, 64, 64),                                               # eight: a block for more than every other CU, not cut
    ([1300, 20], [1300, 20], 16, 8, 64, 16), ([2100], [1200], 16, 8, 128, 128),
])
def test_long_prompts_that_are_not_cut(hip, e4m3, lengths, new, hq, hkv, hd, page):
    """Keys beyond the 1024 whose pages a wave holds at a time, in one part; the second time with pages missing on either side of there."""
    long_prompts(hip, lengths, new, hq, hkv, hd, page, e4m3)
    if lengths[0] > 1100:
        long_prompts(hip, lengths, new, hq, hkv, hd, page, e4m3, gone=[(0, 1), (0, 1024 // page), (0, (lengths[0] - 40) // page)])


def test_rows_ahead_of_the_first_sequence_are_left_alone(hip):
    """starts[0] beyond 0: by write, read and attention alike."""
    hq, hkv, hd, page = 4, 1, 64, 16
    case = Case([40, 33], hkv, hd, page, False, seed=58, new=[4, 33])
    cache, batch = case.on(DEV, hq, rows=case.rows + 3)
    batch.starts.add_(3)
    n = case.rows + 3
    qkv = rnd(n, (hq + 2 * hkv) * hd, seed=59).to(DEV)
    q = torch.full((n, hq * hd), 3.0, dtype=BF, device=DEV)
    k0 = cache.k_pages.clone()
    cache.write(batch, qkv, q)
    assert (q[:3] == 3).all() and torch.equal(q[3:], qkv[3:, :hq * hd])
    for r, _, pos, p, s in O.places(case.table, case.lengths, [3, 7, 40], page):
        k0[p, :, s] = qkv[r, hq * hd:(hq + hkv) * hd].view(hkv, hd)
    assert torch.equal(bits(cache.k_pages), bits(k0))
    k, v = (torch.full((n, hkv * hd), 5.0, dtype=BF, device=DEV) for _ in range(2))
    cache.read(batch, k, v)
    assert (k[:3] == 5).all() and (v[:3] == 5).all() and torch.equal(k[3:], qkv[3:, hq * hd:(hq + hkv) * hd])
    y = torch.full_like(q, 7)
    cache.attend(batch, q, y)
    assert (y[:3] == 7).all() and y[3:].isfinite().all()


def test_pages_exchanged_under_a_cache(hip):
    """Whichever way another tensor comes into the cache's place, calls go to that one."""
    import copy
    hq = 4
    cases = [Case([40, 33], 2, 64, 16, e4m3, seed=s) for e4m3 in (False, True) for s in (61, 62)]
    for first, second in (cases[:2], cases[2:]):
        cache, batch = first.on(DEV, hq)
        batch.table.copy_(second.table)
        other, _ = second.on(DEV, hq)
        q = rnd(2, hq * 64).to(DEV)
        attended = lambda c: c.attend(batch, q, torch.empty_like(q))
        want, kept = attended(other), [b for b in cache.buffers()]
        assert not torch.equal(attended(cache), want)
        names = ["k_pages", "v_pages"] + ([] if cache.scales is None else ["scales"])

        def restore():
            for n, t in zip(names, kept):
                setattr(cache, n, t)
            assert not torch.equal(attended(cache), want)

        for n in names:
            setattr(cache, n, getattr(other, n))
        assert torch.equal(attended(cache), want)
        restore()
        for n in names:
            cache._buffers[n] = getattr(other, n)
        assert torch.equal(attended(cache), want)
        restore()
        twin = copy.copy(cache)
        for n in names:
            setattr(twin, n, getattr(other, n))
        assert torch.equal(attended(twin), attended(cache))      # (a shallow copy has the same buffers)
        restore()
        old = [t.data for t in kept]                            # (the memory stays while the tensors have other)
        for n in names:
            getattr(cache, n).data = getattr(other, n)
        assert torch.equal(attended(cache), want)
        del old


def test_a_batch_given_up_while_another_stream_works(hip):
    """Its memory and that of its tables is not handed out before the work has ended: later tensors of the same sizes lie elsewhere."""
    case = Case([3000, 900], 2, 128, 16, False, seed=63)
    q = rnd(2, 8 * 128).to(DEV)
    cache, first = case.on(DEV, 8)
    want = cache.attend(first, q, torch.empty_like(q)).clone()
    side = torch.cuda.Stream()
    for _ in range(3):
        y = torch.empty_like(q)
        i = lambda x: torch.as_tensor(x, dtype=torch.int32).to(DEV)
        batch = cache.batch(i(case.table), i(case.lengths), 8)
        tensors = [batch.table, batch.lengths, batch.scratch]
        sizes, at = [(t.shape, t.dtype) for t in tensors], {t.data_ptr() for t in tensors}
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            cache.attend(batch, q, y)
        del batch, tensors
        later = [torch.full(shape, 77, dtype=dtype, device=DEV) for shape, dtype in sizes for _ in range(4)]
        assert not side.query() and not at & {t.data_ptr() for t in later}
        side.synchronize()
        assert torch.equal(y, want)
        del later
    # in a graph: captured with a batch made before, replayed while that is kept
    graph, y = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        cache.attend(first, q, y)
    for _ in range(3):
        y.zero_()
        graph.replay()
        assert torch.equal(y, want)


# ------------------------------------------------------------------------------------------------ how a step is dealt out

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths,hq,hkv,hd,page,way", SCHEDULED, ids=[f"{c[5]}{i}" for i, c in enumerate(SCHEDULED)])
def test_every_way_of_dealing_out_a_step(hip, e4m3, lengths, hq, hkv, hd, page, way):
    """The ways that tests/paged_schedule.py tells apart, each against the oracle; the same bits the second time."""
    cache, batch, q, got = attend(Case(lengths, hkv, hd, page, e4m3, seed=64), hq)
    again = cache.attend(batch, q.to(DEV), torch.empty(len(lengths), hq * hd, dtype=BF, device=DEV))
    assert torch.equal(again.cpu().double().view(got.shape), got)


# ------------------------------------------------------------------------------------------------ bytes

def test_every_byte_with_every_power_is_read_back(hip):
    """All 256 e4m3 numbers with all powers that a write gives: the values they stand for, which are bf16 numbers but below 2^-133 and from 2^128 on."""
    from gpt_fast.utils import PagedKVCache
    hd, page = 128, 256
    codes = torch.arange(256, dtype=torch.uint8).view(2, 1, 1, hd).expand(2, 1, page, hd).contiguous()      # page 0: codes 0..127, 1: the rest
    scales = torch.arange(256, dtype=torch.uint8).clamp(1, 247).view(1, 1, 1, page).expand(2, 1, 2, page).contiguous()
    cache = PagedKVCache.from_pages(codes.view(E4M3).to(DEV), codes.view(E4M3).to(DEV), scales.to(DEV))
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    batch = cache.batch(i(0, 1)[None], i(512), 1, starts=i(0, 512), rows=512)
    k, v = (torch.empty(512, hd, dtype=BF, device=DEV) for _ in range(2))
    cache.read(batch, k, v)
    want = O.values(codes.view(E4M3), scales, 0).reshape(512, hd).to(F32).to(BF)
    for got in (k.cpu(), v.cpu()):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))


def test_rows_of_the_largest_and_smallest_numbers_are_written_as_defined(hip):
    """At both ends of bf16's range: the exponent and the rounding as the definition says, read back as bf16 rounds what is kept."""
    hd = 64
    qkv = torch.zeros(4, 3 * hd, dtype=BF)
    most = torch.finfo(BF).max
    qkv[0, hd:] = torch.linspace(-1, 1, 2 * hd).to(BF) * most
    qkv[1, hd:] = torch.linspace(-1, 1, 2 * hd).to(BF) * 2.0 ** -118
    qkv[2, hd:] = torch.arange(2 * hd, dtype=torch.int16).view(BF)                # subnormal numbers: multiples of 2^-133
    qkv[3, hd:] = torch.tensor([248.0, 247.0]).to(BF).repeat(hd) * 2.0 ** 120
    case = Case([4], 1, hd, 16, True, new=[4])
    cache, batch = case.on(DEV, 1)
    cache.write(batch, qkv.to(DEV), torch.empty(4, hd, dtype=BF, device=DEV))
    k, v = (torch.empty(4, hd, dtype=BF, device=DEV) for _ in range(2))
    cache.read(batch, k, v)
    page = int(case.table[0, 0])
    for which, (pages, got) in enumerate(((cache.k_pages, k), (cache.v_pages, v))):
        x, byte = O.quantise(qkv[:, (1 + which) * hd:(2 + which) * hd].float())
        assert torch.equal(cache.scales[page, 0, which, :4].cpu(), byte) and torch.equal(pages[page, 0, :4].cpu().float(), x.float())
        want = (x.double() * torch.exp2(byte.double() - 127)[:, None]).to(F32).to(BF)
        assert torch.equal(got.cpu(), want) and want[0].isinf().any() and want[3].isinf().any() and want[1:3].isfinite().all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,lengths,new", [(64, [90, 33], None), (128, [2500], None), (64, [90, 33], [60, 33]), (128, [900], [9]), (128, [700], [700])])
@pytest.mark.parametrize("scale,q_scale", [(2.0 ** 30, 1.0), (2.0 ** 40, 1.0), (2.0 ** 64, 1.0), (None, 2.0 ** 40)])
def test_scores_beyond_what_exponents_tell_apart(hip, e4m3, hd, lengths, new, scale, q_scale):
    """Scores of 2^30 and more: the value of a row's largest one, where that is clear of the next.  fp32 sums of hd products are off by hd * 2^-24 of
    the sum of their sizes, at most; a gap of 2^-10 of it, times scale 2^20 and more, leaves the others no weight."""
    hq = 2
    case = Case(lengths, 1, hd, 16, e4m3, seed=65, new=new)
    cache, batch = case.on(DEV, hq)
    q = rnd(case.rows, hq * hd, seed=66, scale=q_scale)
    y = cache.attend(batch, q.to(DEV), torch.empty(case.rows, hq * hd, dtype=BF, device=DEV), scale).cpu().view(-1, hq, hd)
    assert y.isfinite().all()
    k, v = (torch.nan_to_num(O.values(x, case.scales, i), nan=0.0)[:, 0] for i, x in enumerate((case.k, case.v)))
    clear = 0
    for b, n in enumerate(lengths):
        ids = case.table[b, :-(-n // 16)].long()
        ks, vs = k[ids].reshape(-1, hd)[:n], v[ids].reshape(-1, hd)[:n]
        first, end = (b, b + 1) if new is None else case.starts[b:b + 2]
        for r in range(first, end):
            seen = n - (end - r) + 1
            for h in range(hq):
                x = q[r, h * hd:(h + 1) * hd].double()
                s, size = ks[:seen] @ x, float((ks[:seen].abs() @ x.abs()).max())
                top = s.argmax()
                others = s[torch.arange(seen) != top]
                if seen == 1 or s[top] - others.max() > size * 2.0 ** -10:
                    assert torch.equal(y[r, h], vs[top].to(BF)), (r, h)
                    clear += 1
    assert clear >= case.rows * hq // 2


def test_a_sequence_without_rows_has_no_position_out_of_range(hip):
    """A sequence that takes no part may be longer than the table: nobody is told of it."""
    case = Case([64, 33, 20], 2, 64, 16, False, seed=67, new=[0, 33, 0])
    case.table, case.lengths = case.table[:, :4].contiguous(), [4000, 33, 65]
    attend(case, 4)
    hip.raise_on_device_error(DEV)


# ------------------------------------------------------------------------------------------------ calls that are allowed

@pytest.mark.parametrize("e4m3", [False, True])
def test_captured_prompts_follow_what_the_device_holds(hip, e4m3):
    """write, attend and read of a call with starts, captured once: lengths, starts and the table change between replays, the program's own
    eager calls run between them."""
    hq, hkv, hd, page, rows, B = 8, 2, 64, 16, 90, 5
    from gpt_fast.utils import PagedKVCache
    dtype = E4M3 if e4m3 else BF
    caches = [PagedKVCache(400, page, hkv, hd, dtype, device=DEV) for _ in range(2)]
    g = torch.Generator().manual_seed(70)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(DEV)
    table, lengths, starts = i32(torch.zeros(B, 80)), i32(torch.ones(B)), i32(torch.arange(B + 1))
    batch = caches[0].batch(table, lengths, hq, starts=starts, rows=rows)
    qkv = torch.zeros(rows, (hq + 2 * hkv) * hd, dtype=BF, device=DEV)
    angle = torch.rand(1300, hd // 2, generator=g) * 6.28
    rope = torch.stack([angle.cos(), angle.sin()], -1).to(DEV)
    outs = [[torch.zeros(rows, w, dtype=BF, device=DEV) for w in (hq * hd, hq * hd, hkv * hd, hkv * hd)] for _ in range(2)]

    def once(cache, b, q, y, k, v):
        cache.write(b, qkv, q, rope)
        cache.attend(b, q, y)
        cache.read(b, k, v)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once(caches[0], batch, *outs[0])
    r = random.Random(71)
    for _ in range(8):
        new = [r.choice([0, 1, r.randint(0, 17)]) for _ in range(B)]
        ahead = [r.choice([0, r.randint(0, 40), r.randint(0, 1180)]) for _ in range(B)]
        at = [sum(new[:b]) for b in range(B + 1)]
        table.copy_(torch.randperm(400, generator=g)[:B * 80].view(B, 80).to(torch.int32))
        lengths.copy_(i32([a + n for a, n in zip(ahead, new)]))
        starts.copy_(i32(at))
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        for a, b in zip(caches[0].buffers(), caches[1].buffers()):
            b.copy_(a)
        for out in outs:
            for t in out:
                t.fill_(3)
        once(caches[1], caches[1].batch(table.clone(), lengths.clone(), hq, starts=starts.clone(), rows=rows), *outs[1])
        graph.replay()
        for a, b in zip((*caches[0].buffers(), *outs[0]), (*caches[1].buffers(), *outs[1])):
            assert torch.equal(bits(a), bits(b))
        assert all((t[at[-1]:] == 3).all() and t[:at[-1]].isfinite().all() for t in outs[0])


@pytest.mark.parametrize("new", [None, [1, 40]])
def test_rows_side_by_side_in_one_matrix(hip, new):
    """q and y as columns of the same matrix, and k and v that are read back: what lies between stays."""
    hq, hkv, hd = 4, 2, 64
    case = Case([30, 77], hkv, hd, 16, False, seed=72, new=new)
    cache, batch = case.on(DEV, hq)
    width = hq * hd
    m = torch.full((case.rows, 2 * width + 2 * hkv * hd + 24), 3.0, dtype=BF, device=DEV)
    m[:, 8:8 + width] = rnd(case.rows, width, seed=73).to(DEV)
    want = cache.attend(batch, m[:, 8:8 + width].contiguous(), torch.empty(case.rows, width, dtype=BF, device=DEV)).clone()
    k0, v0 = (torch.empty(case.rows, hkv * hd, dtype=BF, device=DEV) for _ in range(2))
    cache.read(batch, k0, v0)
    before = m.clone()
    cache.attend(batch, m[:, 8:8 + width], m[:, 16 + width:16 + 2 * width])
    cache.read(batch, m[:, 16 + 2 * width:16 + 2 * width + hkv * hd], m[:, 24 + 2 * width + hkv * hd:])
    before[:, 16 + width:16 + 2 * width] = want
    before[:, 16 + 2 * width:16 + 2 * width + hkv * hd], before[:, 24 + 2 * width + hkv * hd:] = k0, v0
    assert torch.equal(bits(m), bits(before))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("single", [True, False])
def test_as_many_sequences_as_a_call_has(hip, e4m3, single):
    """65535 sequences of one or two tokens, every ninth of none."""
    from gpt_fast.utils import PagedKVCache
    B, hq, hd, page = 65535, 2, 64, 16
    cache = PagedKVCache(B, page, 1, hd, E4M3 if e4m3 else BF, device=DEV)
    g = torch.Generator().manual_seed(74)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(DEV)
    table = torch.randperm(B, generator=g).to(torch.int32)[:, None]
    lengths = torch.randint(1, 3, (B,), generator=g)
    lengths[::9] = 0
    ends = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    rows = int(ends[-1])
    whole = cache.batch(i32(table), i32(lengths), hq, starts=i32(ends), rows=rows)
    qkv = torch.randn(rows, (hq + 2) * hd, generator=g).to(BF).to(DEV)
    q = torch.empty(rows, hq * hd, dtype=BF, device=DEV)
    cache.write(whole, qkv, q)
    k, v = (torch.empty(rows, hd, dtype=BF, device=DEV) for _ in range(2))
    cache.read(whole, k, v)
    if not e4m3:
        assert torch.equal(k, qkv[:, hq * hd:(hq + 1) * hd]) and torch.equal(v, qkv[:, (hq + 1) * hd:])
    last = ends[1:][lengths > 0].to(DEV) - 1
    if single:
        x = torch.zeros(B, hq * hd, dtype=BF, device=DEV)
        there = (lengths > 0).to(DEV)
        x[there] = q[last]
        y = cache.attend(cache.batch(i32(table), i32(lengths), hq), x, torch.full_like(x, 3))
        assert (y[~there] == 0).all()
        y = y[there]
    else:
        y = cache.attend(whole, q, torch.full_like(q, 3))
        first = ends[:-1][lengths > 0].to(DEV)
        assert torch.equal(y[first], v[first].repeat(1, hq))        # a first token sees itself alone
        y = y[last]
    # a second token: two keys
    two = (lengths[lengths > 0] == 2).to(DEV)
    assert torch.equal(y[~two], v[last][~two].repeat(1, hq))
    qf, kf, vf = q[last][two].double().view(-1, hq, hd), k.double(), v.double()
    k1, k0, v1, v0 = kf[last][two], kf[last - 1][two], vf[last][two], vf[last - 1][two]
    d = ((qf * (k1 - k0)[:, None]).sum(-1, keepdim=True) * hd ** -0.5).sigmoid()
    want, spread = d * v1[:, None] + (1 - d) * v0[:, None], d * v1[:, None].abs() + (1 - d) * v0[:, None].abs()
    size = float(torch.maximum((qf.abs() * k1.abs()[:, None]).sum(-1), (qf.abs() * k0.abs()[:, None]).sum(-1)).max()) * hd ** -0.5
    assert ((y[two].double().view(want.shape) - want).abs() <= bound(want, spread, size, 2, hd, WEIGHT)).all()
