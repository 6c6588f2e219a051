"""The paged key-value cache without a GPU: refusals of the C entry points, the oracle's own definitions, the module's bookkeeping."""
import copy
import ctypes
import math

import pytest
import torch

from oracle import paged_oracle as O

E_NULL, E_ALIGN, E_SHAPE, E_UNSUPPORTED = -1, -2, -3, -4


@pytest.fixture(scope="module")
def hip():
    from gpt_fast import _hip

    _hip.load()
    return _hip


def descs(hip, **change):
    """(cache, batch) that are served, with some fields changed.  The addresses are nobody's: only calls that are refused are made."""
    c = dict(k=4096, v=8192, scales=12288, n_pages=10, page=16, n_kv_head=2, head_dim=128, format=1)
    b = dict(table=64, ld_table=4, lengths=128, starts=192, err=None, B=3, pages=4)
    for k, v in change.items():
        (c if k in c else b)[k] = v
    return hip._PagedCache(**c), hip._PagedBatch(**b)


WRITE, READ, ATTEND = range(3)


def address(d):
    return 0 if d is None else ctypes.addressof(d)


def write(hip, cache, batch, qkv, ldqkv, q, ldq, rows, Hq, rope, rope_len, rot, interleaved, rope_dtype):
    return hip.load().lr_paged_write(hip._PAGED_WRITE.pack(address(cache), address(batch), qkv or 0, ldqkv, q, ldq, rope or 0, rows, Hq, rope_len, rot,
                                                           interleaved, rope_dtype), None)


def read(hip, cache, batch, k, ldk, v, ldv, rows):
    return hip.load().lr_paged_read(hip._PAGED_READ.pack(address(cache), address(batch), k or 0, ldk, v, ldv, rows), None)


def attend(hip, cache, batch, q, ldq, y, ldy, rows, Hq, scale, scratch, scratch_bytes):
    return hip.load().lr_paged_attention(hip._PAGED_ATTENTION.pack(address(cache), address(batch), q or 0, ldq, y, ldy, scratch, scratch_bytes, rows, Hq,
                                                                   scale), None)


def calls(hip, cache, batch, which=(WRITE, READ, ATTEND), rows=5, Hq=8, ld=None, scale=0.1, x=1 << 20, rope=None, rot=128, rope_dtype=0,
          scratch_bytes=1 << 30):
    """What the entry points `which` return, one value where they agree."""
    hd, hkv = max(cache.head_dim, 1), max(cache.n_kv_head, 1)
    width = ld or (Hq + 2 * hkv) * hd
    got = set()
    if WRITE in which:
        got.add(write(hip, cache, batch, x, width, 1 << 21, Hq * hd, rows, Hq, rope, 64, rot, 1, rope_dtype))
    if READ in which:
        got.add(read(hip, cache, batch, x, ld or hkv * hd, 1 << 21, ld or hkv * hd, rows))
    if ATTEND in which:
        got.add(attend(hip, cache, batch, x, ld or Hq * hd, 1 << 21, ld or Hq * hd, rows, Hq, scale, 1 << 22, scratch_bytes))
    return got


@pytest.mark.parametrize("change,code", [
    (dict(k=None), E_NULL), (dict(v=None), E_NULL), (dict(scales=None), E_NULL), (dict(table=None), E_NULL), (dict(lengths=None), E_NULL),
    (dict(k=4100), E_ALIGN), (dict(v=4104), E_ALIGN), (dict(scales=12290), E_ALIGN), (dict(table=66), E_ALIGN), (dict(lengths=129), E_ALIGN),
    (dict(starts=193), E_ALIGN), (dict(err=6), E_ALIGN),
    (dict(n_pages=0), E_SHAPE), (dict(n_kv_head=0), E_SHAPE), (dict(page=0), E_SHAPE), (dict(head_dim=-64), E_SHAPE), (dict(B=0), E_SHAPE),
    (dict(pages=0), E_SHAPE), (dict(ld_table=3), E_SHAPE), (dict(n_kv_head=3), E_SHAPE),
    (dict(page=8), E_UNSUPPORTED), (dict(page=24), E_UNSUPPORTED), (dict(page=512), E_UNSUPPORTED), (dict(head_dim=96), E_UNSUPPORTED),
    (dict(head_dim=256), E_UNSUPPORTED), (dict(format=2), E_UNSUPPORTED), (dict(B=65536), E_UNSUPPORTED), (dict(n_pages=1 << 30), E_UNSUPPORTED),
    (dict(page=256, pages=(1 << 22) + 1, ld_table=1 << 23), E_UNSUPPORTED),
    (dict(starts=None), E_SHAPE),      # one row per sequence: 3, not 5
])
def test_descriptors_are_checked_by_every_entry_point(hip, change, code):
    which = (WRITE, ATTEND) if change == dict(n_kv_head=3) else (WRITE, READ, ATTEND)    # 8 q heads on 3: a read has no q heads
    assert calls(hip, *descs(hip, **change), which) == {code}
    cache, batch = descs(hip, **change)
    if change not in (dict(starts=None),):
        assert hip.load().lr_paged_attention_scratch_bytes(ctypes.byref(cache), ctypes.byref(batch), 5, 8) == 0


def test_arguments_are_checked(hip):
    d = descs(hip)
    lib = hip.load()
    assert lib.lr_paged_write(None, None) == lib.lr_paged_read(None, None) == lib.lr_paged_attention(None, None) == E_NULL
    assert write(hip, None, d[1], 16, 8, 16, 8, 1, 8, None, 0, 0, 0, 0) == E_NULL
    assert read(hip, d[0], None, 16, 8, 16, 8, 1) == E_NULL
    assert attend(hip, None, None, 16, 8, 16, 8, 1, 8, 1.0, 16, 1 << 30) == E_NULL
    heads = WRITE, ATTEND
    assert calls(hip, *d, rows=0) == {E_SHAPE}
    assert calls(hip, *d, x=None) == {E_NULL}
    assert calls(hip, *d, x=(1 << 20) + 8) == {E_ALIGN}
    assert calls(hip, *d, ld=248) == {E_SHAPE} and calls(hip, *d, ld=12 * 128 + 4) == {E_ALIGN}
    assert calls(hip, *d, heads, ld=8) == {E_SHAPE}
    assert calls(hip, *d, heads, Hq=7) == {E_SHAPE}
    for scale in (0.0, -1.0, math.nan, math.inf, 3e38, 2e19):
        assert calls(hip, *d, (ATTEND,), scale=scale) == {E_SHAPE}
    assert calls(hip, *d, (ATTEND,), scratch_bytes=0) == {E_SHAPE}
    assert calls(hip, *d, (WRITE,), rope=64, rot=144) == {E_SHAPE} and calls(hip, *d, (WRITE,), rope=64, rot=0) == {E_SHAPE}
    assert calls(hip, *d, (WRITE,), rope=64, rot=24) == {E_UNSUPPORTED} and calls(hip, *d, (WRITE,), rope=64, rope_dtype=2) == {E_UNSUPPORTED}
    assert calls(hip, *d, (WRITE,), rope=68) == {E_ALIGN}


def test_scratch_grows_with_what_is_served(hip):
    lib = hip.load()
    size = lambda rows, Hq, **c: (lambda d: lib.lr_paged_attention_scratch_bytes(ctypes.byref(d[0]), ctypes.byref(d[1]), rows, Hq))(descs(hip, **c))
    assert size(5, 8) > 0
    assert size(0, 8) == 0 and size(5, 7) == 0
    for kw in (dict(), dict(starts=None)):
        for a, b in (((1, 8), (64, 8)), ((64, 8), (500, 8)), ((8, 8), (8, 16))):
            assert size(*a, **kw) <= size(*b, **kw)


def test_module_bookkeeping():
    from gpt_fast.utils import PagedKVCache

    c = PagedKVCache(5, 32, 2, 64)
    assert c.scales is None and c.shape == (2, 32, 64, torch.bfloat16, torch.device("cpu"))
    c = PagedKVCache(5, 32, 2, 64, torch.float8_e4m3fn)
    assert tuple(c.scales.shape) == (5, 2, 2, 32) and c.scales.dtype == torch.uint8
    c.to(torch.float32)          # a model's type is not its cache's
    assert c.k_pages.dtype == torch.float8_e4m3fn and c.scales.dtype == torch.uint8
    assert set(c.state_dict()) == {"k_pages", "v_pages", "scales"}
    with pytest.raises(AssertionError):
        PagedKVCache(5, 32, 2, 64, torch.float32)
    twin = copy.deepcopy(c)
    assert twin.k_pages.data_ptr() != c.k_pages.data_ptr() and twin.shape == c.shape
    t = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(AssertionError, match="rows"):
        c.batch(t, t[:, 0], 4, starts=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(AssertionError):      # device tensors only
        c.batch(t, torch.zeros(2, dtype=torch.int32), 4)


def test_the_oracle_quantises_as_defined():
    x = torch.tensor([[448.0, -1.0], [449.0, 1.0], [0.0, 0.0], [448 * 2.0 ** -20, 1e-9], [math.inf, 3.0], [1e-40, 0.0], [-896.0, 0.875]])
    q, byte = O.quantise(x)
    assert byte.tolist() == [127, 128, 1, 107, 120, 1, 128]
    v = O.values(q[:, None, None], torch.stack([byte, byte], 1)[:, None, :, None])[:, 0, 0]
    assert v[0].tolist() == [448, -1] and v[1].tolist() == [448, 1] and v[2].tolist() == [0, 0] and v[6].tolist() == [-896, 0.875]
    assert math.isnan(v[4, 0]) and v[4, 1] == 3
    y = torch.randn(400, 64, generator=torch.Generator().manual_seed(1))
    q, byte = O.quantise(y)
    back = O.values(q[:, None, None], torch.stack([byte, byte], 1)[:, None, :, None])[:, 0, 0]
    step = torch.exp2(byte.double() - 127)[:, None]
    assert ((back - y.double()).abs() <= torch.maximum(2.0 ** -4 * y.double().abs(), 2.0 ** -10 * step)).all()
    assert torch.equal(back.to(torch.bfloat16).double(), back)     # exact in bf16


def test_the_oracle_places_rows():
    table = torch.tensor([[4, 2, 9], [1, 0, 3]])
    assert O.places(table, [17, 0], None, 16) == [(0, 0, 16, 2, 0)]
    assert O.places(table, [17, 3], [0, 2, 5], 16) == [(0, 0, 15, 4, 15), (1, 0, 16, 2, 0), (2, 1, 0, 1, 0), (3, 1, 1, 1, 1), (4, 1, 2, 1, 2)]


def test_operands_that_overlap_are_refused(hip):
    """(rows, widths of both, their row strides, how far apart in elements) -> whether they share memory; and the calls that check it."""
    cache, batch = descs(hip)
    at, hd, hq = 1 << 20, 128, 8
    width = (hq + 4) * hd
    for off, ldq in ((8, width), (hd, hq * hd), (width * 5 - 8, hq * hd), (0, hq * hd), (-8, width), (width, width), (width - 8, 2 * width)):
        assert write(hip, cache, batch, at, width, at + 2 * off, ldq, 5, hq, None, 0, 0, 0, 0) == E_SHAPE, (off, ldq)
    for off, ld in ((0, hq * hd), (8, hq * hd), (hq * hd, hq * hd), (-8, 3 * hd * hq), (hq * hd - 8, 3 * hq * hd), (3 * hd * hq - 8, 3 * hd * hq)):
        assert attend(hip, cache, batch, at, ld, at + 2 * off, ld, 5, hq, 0.1, 1 << 24, 1 << 30) == E_SHAPE, (off, ld)
    assert attend(hip, cache, batch, at, hq * hd, at + 2 * hq * hd, 2 * hq * hd, 5, hq, 0.1, 1 << 24, 1 << 30) == E_SHAPE
    for off, ld in ((0, 2 * hd), (8, 2 * hd), (2 * hd - 8, 4 * hd), (-8, 4 * hd)):
        assert read(hip, cache, batch, at, ld, at + 2 * off, ld, 5) == E_SHAPE, (off, ld)


def test_more_workgroups_than_a_launch_has_threads_for(hip):
    """2^30 rows of q heads: 2^23 workgroups of four waves fit; with as many short sequences as go by a head's blocks on top they do not."""
    lib = hip.load()
    size = lambda rows, Hq, **c: (lambda d: lib.lr_paged_attention_scratch_bytes(ctypes.byref(d[0]), ctypes.byref(d[1]), rows, Hq))(descs(hip, **c))
    assert size(1 << 20, 1 << 10, n_kv_head=1, B=16) > 0
    assert size(1 << 16, 1 << 10, n_kv_head=1 << 10, B=65535) == 0


def test_the_oracles_two_forms_agree():
    from paged_cases import Case

    for lengths, new, gone in (([40, 33, 0, 5], [20, 33, 0, 1], (0, 1)), ([64, 70], [10, 3], (1, 0)), ([2, 9], [5, 9], (1, 0))):
        case = Case(lengths, 2, 64, 16, True, new=new)
        case.table[gone] = case.n_pages
        if lengths[1] == 70:
            case.table = case.table[:, :4]
        q = torch.randn(case.rows, 4 * 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        clean = [torch.nan_to_num(O.values(x, case.scales, i), nan=0.0) for i, x in enumerate((case.k, case.v))]
        y, spread, size = case.oracle(q, 4)
        y2, spread2, size2 = O.attention_of_sequences(q.view(-1, 4, 64), *clean, case.table, lengths, case.starts, 64 ** -0.5)
        assert (y - y2).abs().max() < 1e-12 and (spread - spread2).abs().max() < 1e-12
        assert size <= size2 + 1e-9      # (it looks at keys that a row does not see, too)


def test_sizes_have_no_scratch_where_the_call_refuses_them(hip):
    """lr_paged_attention_scratch_bytes and lr_paged_attention agree on every size (its calls have no scratch: none of them is made)."""
    served = refused = 0
    for starts in (192, None):
        for B in (1, 3, 65535):
            for rows in (-1, 0, 1, 3, 65535, 1 << 20, (1 << 20) + 1, (1 << 31) - 1):
                for Hq in (-2, 0, 2, 7, 8, 1024, 65534, 65536, 1 << 24):
                    cache, batch = descs(hip, starts=starts, B=B)
                    size = hip.load().lr_paged_attention_scratch_bytes(ctypes.byref(cache), ctypes.byref(batch), rows, Hq)
                    ld = max(Hq, 1) * 128
                    code = attend(hip, cache, batch, 1 << 20, ld, 1 << 60, ld, rows, Hq, 0.1, 1 << 22, 0)     # (q ends below 2^56)
                    bad = rows <= 0 or Hq <= 0 or Hq > 65535 or Hq % 2 or (starts is None and rows != B)
                    big = rows * Hq > 1 << 30
                    assert (size == 0) == (bad or big), (starts, B, rows, Hq, size)
                    assert code == (E_SHAPE if bad or not big else E_UNSUPPORTED), (starts, B, rows, Hq, code)    # (not big: no room)
                    served += size > 0
                    refused += big and not bad
    assert served > 20 and refused > 5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_casts_leave_the_pages_bytes(dtype):
    """A model's .half() is not its cache's: every 16-bit (8-bit) number stays what it was, in the same memory."""
    from gpt_fast.utils import PagedKVCache

    n = 16 * 64
    raw = torch.arange(64 * n).to(torch.int16).view(torch.uint8) if dtype == torch.bfloat16 else torch.arange(2 * n).to(torch.uint8)
    pages = lambda: raw.clone().view(dtype).view(-1, 1, 16, 64)
    scales = None if dtype == torch.bfloat16 else torch.arange(2 * 32).to(torch.uint8).view(2, 1, 2, 16)
    held = lambda c: [b.contiguous().view(torch.uint8).flatten().tolist() for b in c.buffers()]
    cache = PagedKVCache.from_pages(pages(), pages(), scales)
    want, at = held(cache), cache.k_pages.data_ptr()
    for cast in (lambda m: m.half(), lambda m: m.to(torch.float16), lambda m: m.double(), lambda m: m.to(torch.float32), lambda m: m.bfloat16(),
                 lambda m: m.type(torch.float16), lambda m: m.to("cpu", torch.half), lambda m: m.cpu()):
        outer = torch.nn.ModuleDict(dict(cache=cache, other=torch.nn.Linear(2, 2)))
        cast(outer)
        assert held(cache) == want and cache.k_pages.dtype == dtype and cache.k_pages.data_ptr() == at
    cache.to("meta")
    assert cache.k_pages.device.type == "meta" and cache.k_pages.dtype == dtype and cache.k_pages.shape[1:] == (1, 16, 64)


def test_more_rows_than_a_launch_has_threads_for(hip):
    """2^24 workgroups of 256: a write of many heads and a read of 16 kv heads have one token each."""
    cache, batch = descs(hip, n_kv_head=16)
    ld = 64 * 128
    for rows in (1 << 24, (1 << 31) - 1):
        assert write(hip, cache, batch, 1 << 20, ld, 1 << 60, ld, rows, 32, None, 0, 0, 1, 0) == E_UNSUPPORTED
        assert read(hip, cache, batch, 1 << 20, ld, 1 << 60, ld, rows) == E_UNSUPPORTED


def test_the_batches_of_the_gpu_tests_take_every_way():
    """What the steps of tests/test_gpu_paged.py over SCHEDULED are there for, worked out from the rules."""
    from paged_schedule import SCHEDULED, facts, workers_of

    got = []
    for lengths, hq, hkv, hd, page, way in SCHEDULED:
        f = facts(lengths, workers_of(len(lengths), max(-(-n // page) for n in lengths) + 1, page, hq, hkv, hd))
        assert f[0] == way, (f, way)
        got.append((len(lengths) <= 64, *f))
    assert any(few and way == "line" and two == 2 for few, way, _, _, two, _ in got)                   # two open parts, up to 64 sequences
    assert any(not few and way == "line" and two == 2 for few, way, _, _, two, _ in got)               # and beyond
    assert any(few and way == "line" and n >= w for few, way, n, w, _, _ in got)                       # more sequences than workers, as a line
    assert sum(way == "whole" and n > w for _, way, n, w, _, _ in got) == 2                            # and whole
    assert any(way == "cut" and parts > 32 for _, way, _, _, _, parts in got)                          # joined in blocks
    assert any(way == "line" and parts > 32 for _, way, _, _, _, parts in got)
