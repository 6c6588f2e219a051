"""How k_paged_decode deals a batch's tiles out to the workers of a kv head, restated: which of its ways a case takes."""
import random


def workers_of(B, pages, page, hq, hkv, hd, cus=256):
    """The grid's width: as many workgroups as the chip holds at once, no more than the table's pages could give four tiles each."""
    groups = hkv * -(-(hq // hkv) // 16)
    tiles = B * (pages * page // 32 + 1)
    return max(1, min(cus * (2 if hd == 64 else 1) // groups, (tiles + 3) // 4))


def schedule(lengths, grid):
    """(way, [per worker: [(sequence, first tile, tiles, is all of it)]]) of a batch: "alone", "cut", "whole" or "line"."""
    tiles = [-(-max(n, 0) // 32) for n in lengths]
    total, sequences = sum(tiles), sum(t > 0 for t in tiles)
    some = [b for b, t in enumerate(tiles) if t]
    few = lambda t: max(4, -(-t // 16)) if t <= 256 else 4
    workers = min(grid, max(-(-total // 4), sequences))
    if sequences == 1 and few(total) > 4:
        workers = min(workers, 16)
    many = len(lengths) > 1
    longest = max(tiles) if many and len(lengths) <= 64 and sequences > 1 else 0
    if longest and sequences < workers:
        even = max(-(-total // workers), few(longest))
        most = even if (even + 8) * (grid - sequences // 2) >= total else even + 9
        while most <= even + 8:
            parts = {b: -(-tiles[b] // most) for b in some}
            if sum(parts.values()) <= grid:
                got = []
                for b in some:
                    each, larger = divmod(tiles[b], parts[b])
                    at = 0
                    for i in range(parts[b]):
                        n = each + (i < larger)
                        got.append([(b, at, n, parts[b] == 1)])
                        at += n
                return "cut", got
            most += 1 + most // 8
    extra = 6 if many and 2 * sequences >= workers else 0
    line, begin = 0, {}
    for b in some:
        begin[b] = line
        line += tiles[b] + extra
    each, larger = divmod(line, workers)
    got = []
    for w in range(workers):
        at = w * each + min(w, larger)
        end = at + each + (w < larger)
        if longest and longest <= 16:
            got.append([(b, 0, tiles[b], True) for b in some if at <= begin[b] + tiles[b] + extra - (tiles[b] + extra) // 2 < end])
            continue
        mine = []
        for b in some:
            first = begin[b] + extra
            lo, hi = max(0, at - first), min(tiles[b], end - first)
            if lo < hi:
                mine.append((b, lo, hi - lo, hi - lo == tiles[b]))
        got.append(mine)
    return ("alone" if sequences <= 1 else "whole" if longest and longest <= 16 else "line"), got


def facts(lengths, grid):
    """(way, sequences, workers, most open parts of a worker, most parts of a sequence); the parts have to be all tiles, once each."""
    way, got = schedule(lengths, grid)
    parts = {}
    for mine in got:
        for b, at, n, _ in mine:
            parts.setdefault(b, []).append((at, n))
    for b, n in enumerate(lengths):
        at = 0
        for first, k in sorted(parts.get(b, [])):
            assert first == at
            at += k
        assert at == -(-max(n, 0) // 32)
    return (way, sum(n > 0 for n in lengths), len(got), max((sum(not p[3] for p in mine) for mine in got), default=0),
            max((len(p) for p in parts.values()), default=0))


def _ragged(seed, n, most, least=1):
    return [random.Random(seed * 1000 + i).randint(least, most) for i in range(n)]


# lengths, q heads, kv heads, head_dim, page, way
SCHEDULED = [
    (_ragged(1, 20, 1500), 8, 8, 128, 16, "line"),          # workers with a sequence that began before them and one that goes on behind
    (_ragged(2, 28, 1500), 32, 8, 128, 64, "line"),
    (_ragged(3, 30, 700), 16, 16, 128, 32, "line"),         # more sequences than workers
    ([700] * 20, 32, 32, 64, 16, "line"),                   # equal ones
    ([3000] + _ragged(4, 30, 60), 16, 16, 128, 16, "line"),
    (_ragged(5, 40, 270), 24, 24, 128, 16, "whole"),        # short ones, four to a worker
    (_ragged(6, 40, 270, 0), 16, 16, 64, 16, "whole"),
    ([40, 9000, 33] + [20] * 9, 4, 4, 128, 16, "cut"),      # parts joined in blocks
    (_ragged(7, 100, 500), 8, 8, 128, 16, "line"),          # more than a wave has lanes
    ([0, 20000, 0] + [300] * 70, 2, 1, 128, 64, "line"),    # and one of them joined in blocks
    ([31] * 65 + [1200] * 3 + [0] * 70 + [64, 65] * 20, 6, 6, 64, 32, "line"),
]
