"""The shared-prefix kernel's cut of the work, its order of waits and its operand layout, restated on the CPU."""
import pytest


def cut(units, grid, c):
    return c * units // grid, (c + 1) * units // grid


@pytest.mark.parametrize("items, tiles, grid", [(1, 1, 1), (4, 64, 128), (8, 5, 20), (64, 512, 148), (3, 7, 10), (16, 256, 148), (1, 300, 148), (148, 1, 74), (5, 3, 7)])
def test_a_row_s_results_are_found_by_the_join(items, tiles, grid):
    """Thread blocks leave results as (block + item); the join takes those of the blocks between its item's first and last unit."""
    units = items * tiles
    left = {}
    for c in range(grid):
        u, end = cut(units, grid, c)
        while u < end:
            item, first = divmod(u, tiles)
            n = min(tiles - first, end - u)
            assert (c + item) not in left            # no two results share a place
            left[c + item] = (item, first, n)
            u += n
    assert all(0 <= p < grid + items for p in left)
    for item in range(items):
        u0, u1 = item * tiles, item * tiles + tiles - 1
        c0, c1 = ((u0 + 1) * grid - 1) // units, ((u1 + 1) * grid - 1) // units
        got = [left[c + item] for c in range(c0, c1 + 1)]
        assert all(g[0] == item for g in got)
        seen = sorted(t for _, first, n in got for t in range(first, first + n))
        assert seen == list(range(tiles))


@pytest.mark.parametrize("two", [True, False])
@pytest.mark.parametrize("n", list(range(1, 12)) + [37])
def test_conversion_and_products_never_wait_for_one_another(two, n):
    """K and V tiles through two places each; scores of job j + 2 behind the products of job j; with two row tiles a K or V tile is
    left by the second, with one by whoever has it."""
    jobs = 2 * n if two else n
    tile = (lambda j: j >> 1) if two else (lambda j: j)
    program = [("S", j) for j in range(min(2, jobs))]
    for j in range(jobs):
        program.append(("P", j))
        if j + 2 < jobs:
            program.append(("S", j + 2))
    converts = [(side, g) for g in range(n) for side in "KV"]
    ready, left, scored, c, m = set(), set(), set(), 0, 0
    while c < len(converts) or m < len(program):
        before = (c, m)
        while c < len(converts) and (converts[c][1] < 2 or (converts[c][0], converts[c][1] - 2) in left):
            ready.add(converts[c])
            c += 1
        while m < len(program):
            what, j = program[m]
            g = tile(j)
            if ("K" if what == "S" else "V", g) not in ready or (what == "P" and j not in scored):
                break
            if what == "S":
                scored.add(j)
            if not two or j & 1:
                left.add(("K" if what == "S" else "V", g))
            m += 1
        assert (c, m) != before


def test_the_converting_threads_meet_all_banks_and_all_chunks():
    seen = set()
    for group in range(8):
        read, low, high = set(), set(), set()
        for l in range(8):
            tid = group * 8 + l
            row, cc = tid >> 4 << 1 | (tid >> 2 & 1), ((tid >> 2 ^ tid >> 3) & 1) << 2 | (tid & 3)
            j0, sw, base = (cc & 3) * 2, row & 7, (cc >> 2) * 16384 + row * 128
            seen.add((row, cc))
            read.add((row * 128 + cc * 16) // 16 % 8)
            low.add((base + ((j0 ^ sw) << 4)) // 16 % 8)
            high.add((base + (((j0 + 1) ^ sw) << 4)) // 16 % 8)
        assert len(read) == len(low) == len(high) == 8
    assert seen == {(r, c) for r in range(8) for c in range(8)}      # rows 8 .. 15 of a block: the same eight rows on

