"""Which key tiles a work item of the packed-prompt kernel goes through, which of them it masks, and which block takes which
item: the device arithmetic restated line for line, over random prompts, windows and prefixes.  Every tile in an
item's list has to be used by one of its two row tiles (the buffers it is loaded into are freed by their products)."""
import random

ROWS, KEYS = 128, 128


class Item:
    def __init__(self, length, pair, prefix, causal, window):
        self.len, self.pair, self.prefix, self.causal, self.window = length, pair, prefix, causal, window

    def first_key(self, row):
        return max(0, row - self.window + 1) if self.window > 0 else 0

    def end_key(self, row):
        if self.causal:
            return row + 1
        return min(self.len, row + self.window) if self.window > 0 else self.len

    def sees(self, row, j):
        return j < self.len and (j < self.prefix or self.first_key(row) <= j < self.end_key(row))

    def tiles(self, q0):
        """(some_p, lo, hi, all_p, all_lo, all_hi) of a row tile."""
        if q0 >= self.len:
            return (0,) * 6
        r1 = min(q0 + ROWS, self.len) - 1
        return (-(-self.prefix // KEYS), self.first_key(q0) // KEYS, -(-self.end_key(r1) // KEYS), self.prefix // KEYS,
                -(-self.first_key(r1) // KEYS), min(self.end_key(q0), self.len) // KEYS)

    def keys(self):
        r0 = self.pair * 2 * ROWS
        r1 = min(r0 + 2 * ROWS, self.len) - 1
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
        it = Item(length, rng.randrange(-(-length // (2 * ROWS))), min(prefix, length), rng.random() < 0.7,
                  rng.choice((0, 0, 1, 2, 100, 128, 129, rng.randint(1, 2000))))
        q0 = it.pair * 2 * ROWS
        tiles = [it.tiles(q0), it.tiles(q0 + ROWS)]
        keys = it.keys()
        assert keys and len(set(keys)) == len(keys) and min(keys) >= 0 and max(keys) * KEYS < length
        for k in keys:
            assert any(_uses(t, k) for t in tiles)
        for t, start in zip(tiles, (q0, q0 + ROWS)):
            rows = range(start, min(start + ROWS, length))
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


def _schedule(lens, heads, block, grid):
    """Items (sequence, pair, head) of a block, in order."""
    out, want, before = [], block, 0
    most = max(lens, default=0)
    for level in range(-(-most // 256) - 1, -1, -1):
        for c in range(0, len(lens), 32):
            has = [s for s in range(c, min(c + 32, len(lens))) if lens[s] > level * 256]
            n = len(has) * heads
            while want < before + n:
                at = want - before
                out.append((has[at // heads], level, at % heads))
                want += grid
            before += n
    return out


def test_every_item_is_taken_once():
    rng = random.Random(12)
    for _ in range(200):
        lens = [rng.choice((0, 1, 255, 256, 257, rng.randint(0, 3000))) for _ in range(rng.choice((1, 3, 32, 33, 70)))]
        heads = rng.choice((1, 4, 9, 32))
        grid = min(148, (sum(lens) // 256 + min(len(lens), max(1, sum(lens)))) * heads) or 1
        got = [x for b in range(grid) for x in _schedule(lens, heads, b, grid)]
        want = [(s, p, h) for s, n in enumerate(lens) for p in range(-(-n // 256)) for h in range(heads)]
        assert len(got) == len(set(got)) and sorted(got) == sorted(want)
