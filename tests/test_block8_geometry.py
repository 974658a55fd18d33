"""Which warp of the append writes which rows, and how the decode kernel cuts a batch into pieces: the device
arithmetic restated line for line, over random batches."""
import random


def _append_writes(start, lens, T, chunk, max_blocks):
    """(sequence, block, first row of the call, rows, row in the block) of every warp's writes of one head and side."""
    out, n = [], len(lens)
    for t0 in range(0, T, chunk):
        t, end = t0, min(t0 + chunk, T)
        s = sum(start[i + 1] <= t for i in range(n))
        while t < end:
            while s < n and start[s + 1] <= t:
                s += 1
            if s >= n:
                break
            a, b = start[s], min(start[s + 1], T)
            if t < a:
                t = a
                continue
            pos = lens[s] - (b - t)
            if pos < 0:
                t += min(b - t, -pos)
                continue
            step = 0 if t == a else (16 - (pos & 15)) & 15
            t, pos = t + step, pos + step
            if t >= b:
                t = b
                continue
            if t >= end:
                break
            r = pos & 15
            cnt = min(16 - r, b - t)
            if pos >> 4 < max_blocks:
                out.append((s, pos >> 4, t, cnt, r))
            t += cnt
    return out


def test_every_row_is_written_once_and_every_block_by_one_warp():
    rng = random.Random(5)
    for _ in range(4000):
        n = rng.randint(1, 9)
        new = [rng.choice((0, 1, 1, rng.randint(1, 80))) for _ in range(n)]
        old = [rng.choice((0, rng.randint(0, 70), -rng.randint(1, 20) if rng.random() < 0.1 else 3)) for _ in range(n)]
        gap = rng.choice((0, 0, 3))
        start = [gap]
        for x in new:
            start.append(start[-1] + x)
        lens = [o + x for o, x in zip(old, new)]
        T = start[-1] + rng.choice((0, 0, 5))
        writes = _append_writes(start, lens, T, rng.choice((1, 2, 4, 16)), 1000)
        want = {(s, old[s] + i, start[s] + i) for s in range(n) for i in range(new[s]) if old[s] + i >= 0}
        got = [(s, blk * 16 + r + i, t + i) for s, blk, t, cnt, r in writes for i in range(cnt)]
        assert len(got) == len(set(got)) and set(got) == want
        assert len({(s, blk) for s, blk, *_ in writes}) == len(writes)
        for s, blk, t, cnt, r in writes:
            assert cnt >= 1 and r + cnt <= 16 and 0 <= t and t + cnt <= T
            assert r == 0 or (t == start[s] and old[s] % 16 == r)     # rows in front of it were there before the call


def _pieces(counts, target, min_piece, grid, one_wave):
    cut = lambda piece: [max(1, -(-c // piece)) for c in counts]
    hi = max(min_piece, -(-sum(counts) // target))
    if one_wave:
        lo = max(min_piece, -(-sum(counts) // grid))
        if (hi - lo) * 8 < hi:
            return hi, cut(hi)
        while lo < hi:
            mid = (lo + hi) // 2
            if sum(cut(mid)) <= grid:
                hi = mid
            else:
                lo = mid + 1
    return hi, cut(hi)


def test_pieces_fit_the_grid_and_cover_every_block():
    rng = random.Random(6)
    for _ in range(4000):
        B = rng.randint(1, 70)
        most = rng.choice((1, 5, 40, 700, 8192))
        counts = [rng.choice((0, most, rng.randint(0, most))) for _ in range(B)]
        wave = rng.choice((1, 18, 37, 74, 296))
        target = max(1, wave - B if 2 * B <= wave else 3 * wave)
        min_piece = rng.choice((8, 20, 64))
        grid = min(target + B, -(-most // min_piece) * B)
        piece, n = _pieces(counts, target, min_piece, grid, 1 < B <= 32 and 2 * B <= grid and rng.random() < 0.7)
        assert sum(n) <= grid
        for c, k in zip(counts, n):
            each = -(-c // k)                                     # a sequence's pieces are of one length
            covered = [min(i * each + each, c) - i * each for i in range(k)]
            assert each <= piece and sum(max(0, x) for x in covered) == c


def _cluster_size(columns, places, blocks):
    c = 1
    while c < 8 and c * 8 < blocks and 2 * c * columns <= places:
        c *= 2
    return c if blocks <= c * 8 * (2 if 8 * c * columns <= places else 6) else 0


def test_the_blocks_of_a_cluster_share_what_there_is():
    rng = random.Random(8)
    for _ in range(4000):
        columns, places = rng.choice((1, 2, 8, 64, 512)) * rng.randint(1, 70), rng.choice((148, 296))
        most = rng.choice((1, 8, 9, 65, 250, 385, 8192))
        c = _cluster_size(columns, places, most)
        assert c in (0, 1, 2, 4, 8) and (c <= 1 or c * columns <= places) and most <= 8 * c * 6 or c == 0
        if c == 0:
            continue
        count, heads = rng.randint(0, most), rng.randint(1, 16)
        each = -(-count // c)
        spans = [(i * each, min(i * each + each, count)) for i in range(c)]   # the last may be empty, with an end in front of its start
        assert [x for b, e in spans for x in range(b, e)] == list(range(count))
        share = -(-heads * 32 // c)                                # (head, four channels) that a block joins
        assert [x for i in range(c) for x in range(i * share, min(i * share + share, heads * 32))] == list(range(heads * 32))
