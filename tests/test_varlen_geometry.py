"""Which key tiles a work item of the packed-prompt kernel goes through, which of them it masks, and which block takes which
item: the device arithmetic restated line for line, over random prompts, windows and prefixes.  Every tile in an
item's list has to be used by one of its two row tiles (the buffers it is loaded into are freed by their products)."""
import random

ROWS, KEYS = 128, 128


class Item:
    def __init__(self, length, q0, apart, two, prefix, causal, window):
        self.len, self.q0, self.apart, self.two, self.prefix, self.causal, self.window = length, q0, apart, two, prefix, causal, window
        self.span = ROWS + apart

    def first_key(self, row):
        return max(0, row - self.window + 1) if self.window > 0 else 0

    def end_key(self, row):
        if self.causal:
            return row + 1
        return min(self.len, row + self.window) if self.window > 0 else self.len

    def sees(self, row, j):
        return j < self.len and (j < self.prefix or self.first_key(row) <= j < self.end_key(row))

    def tiles(self, t):
        """(some_p, lo, hi, all_p, all_lo, all_hi) of a row tile."""
        if t == 1 and not self.two:
            return (0,) * 6
        q0 = self.q0 + t * self.apart
        r1 = min(q0 + ROWS, self.len) - 1
        return (-(-self.prefix // KEYS), self.first_key(q0) // KEYS, -(-self.end_key(r1) // KEYS), self.prefix // KEYS,
                -(-self.first_key(r1) // KEYS), min(self.end_key(q0), self.len) // KEYS)

    def keys(self):
        r0 = self.q0
        r1 = min(r0 + self.span, self.len) - 1
        np_, frm, to = -(-self.prefix // KEYS), self.first_key(r0) // KEYS, -(-self.end_key(r1) // KEYS)
        a = min(np_, frm)
        count = a + max(to, np_) - frm
        return [(j if j < a else frm + j - a) for j in (count - 1 - i for i in range(count))]


def _uses(t, k):
    return k < t[0] or t[1] <= k < t[2]


def _masked(t, k):
    return k >= t[3] and (k < t[4] or k >= t[5])


def test_key_tiles_of_every_item():
    rng = random.Random(11)
    for _ in range(700):
        length = rng.choice((1, 127, 128, 129, 256, 257, rng.randint(1, 1500)))
        prefix = rng.choice((0, 0, 1, 128, rng.randint(0, length), length))
        apart = rng.choice((0, ROWS))         # two heads of the same rows, or 256 rows of one
        q0 = rng.randrange(-(-length // (ROWS + apart))) * (ROWS + apart)
        two = q0 + apart < length if apart else rng.random() < 0.7
        it = Item(length, q0, apart, two, min(prefix, length), rng.random() < 0.7, rng.choice((0, 0, 1, 2, 100, 128, 129, rng.randint(1, 2000))))
        tiles = [it.tiles(0), it.tiles(1)]
        keys = it.keys()
        assert keys and len(set(keys)) == len(keys) and min(keys) >= 0 and max(keys) * KEYS < length
        for k in keys:
            assert any(_uses(t, k) for t in tiles)
        for t, start, there in zip(tiles, (q0, q0 + apart), (True, two)):
            rows = range(start, min(start + ROWS, length)) if there else ()
            probe = sorted({r for r in (*rows[:2], *rows[-2:], *(rng.choice(rows) for _ in range(3)))} if rows else ())
            assert bool(rows) == any(_uses(t, k) for k in keys)          # a row tile with rows sees at least itself
            for k in range(-(-length // KEYS)):
                span = range(k * KEYS, (k + 1) * KEYS)
                if _uses(t, k):
                    assert k in keys
                    if not _masked(t, k):                                # then every row sees every key of it
                        assert all(it.sees(r, j) for r in probe for j in (span[0], span[-1], rng.choice(span)))
                else:
                    assert not any(it.sees(r, j) for r in probe for j in span)


def _schedule(lens, H_kv, G, block, grid):
    """(sequence, first row, head) of the row tiles of a block's items, in order."""
    apart = 0 if G > 1 else ROWS
    span, pairs = ROWS + apart, (G + 1) // 2
    units = H_kv * pairs if G > 1 else H_kv
    out, want, before = [], block, 0
    for level in range(-(-max(lens, default=0) // span) - 1, -1, -1):
        for c in range(0, len(lens), 32):
            has = [s for s in range(c, min(c + 32, len(lens))) if lens[s] > level * span]
            n = len(has) * units
            while want < before + n:
                s, unit, q0 = has[(want - before) // units], (want - before) % units, level * span
                head = unit if apart else unit // pairs * G + unit % pairs * 2
                two = q0 + apart < lens[s] if apart else unit % pairs * 2 + 1 < G
                assert not two or apart or head // G == (head + 1) // G      # two heads of one KV head
                out += [(s, q0 + t * apart, head + (0 if apart else t)) for t in range(2 if two else 1)]
                want += grid
            before += n
    return out


def test_every_row_tile_is_taken_once():
    rng = random.Random(12)
    for _ in range(200):
        lens = [rng.choice((0, 1, 127, 128, 129, 256, 257, rng.randint(0, 3000))) for _ in range(rng.choice((1, 3, 32, 33, 70)))]
        H_kv, G = rng.choice((1, 2, 8)), rng.choice((1, 1, 2, 3, 4, 9))
        span, units = (128, H_kv * ((G + 1) // 2)) if G > 1 else (256, H_kv)
        grid = min(148, (sum(lens) // span + min(len(lens), max(1, sum(lens)))) * units) or 1
        got = [x for b in range(grid) for x in _schedule(lens, H_kv, G, b, grid)]
        want = [(s, r, h) for s, n in enumerate(lens) for r in range(0, n, ROWS) for h in range(H_kv * G)]
        assert len(got) == len(set(got)) and sorted(got) == sorted(want)
