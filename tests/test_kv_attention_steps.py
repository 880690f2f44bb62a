"""The steps of 128 tokens that kv_prompt.cuh's two tiles take, as ranges, against the masks themselves: the same arithmetic in Python, no GPU needed."""
import random


def steps_of(low, high, window, sinks, size):
    """KvSteps: (steps of sinks alone, first step behind them, all)."""
    sink = first = 0
    if high < 0:
        return 0, 0, 0
    if window > 0 and low - window + 1 > 0:
        first = (low - window + 1) // size
        sink = min((sinks + size - 1) // size, high // size + 1)
        if sink >= first:
            sink = first = 0
    return sink, first, sink + high // size + 1 - first


def begins(s, k, size):
    return (k if k < s[0] else k - s[0] + s[1]) * size


def prompt_steps(s, low, high, window, sinks):
    """KvPromptSteps: (sinks' steps, from, to, whole from, whole to)."""
    first, total = s[1], s[2]
    add = first - s[0]
    sink = s[0] if s[0] > 0 else min((sinks + 127) // 128, total)
    to = 0 if high < 0 else min(total, min(s[0], high // 128 + 1) if high < 128 * first else high // 128 + 1 - add)
    frm = (low - window + 1) // 128 - add if window > 0 and low - window + 1 > 0 else 0
    whole_to = min(to, 0 if low < 127 else (low - 127) // 128 + 1 - add)
    whole_from = max(s[0], (high - window + 1 + 127) // 128 - add if window > 0 and high - window + 1 > 0 else 0)
    return sink, frm, to, whole_from, whole_to


def seen(j, i, window, sinks):
    return j <= i and (window == 0 or j > i - window or j < sinks)


def cases(n):
    rng = random.Random(1)
    for _ in range(n):
        first, group, rows, row0 = rng.randint(-300, 3000), rng.choice([1, 2, 5, 8]), rng.randint(1, 256), rng.randint(0, 3) * 256
        yield (first, group, rows, row0, rng.choice([0, 0, 1, 5, 64, 128, 129, 300, 1000, 2 ** 31 - 1]), rng.choice([0, 0, 1, 4, 100, 128, 200, 700, 2 ** 31 - 1]))


def test_every_token_that_a_row_sees_is_in_a_step():
    for first, group, rows, row0, window, sinks in cases(300):
        low, high = max(first + row0 // group, -1), max(first + (row0 + rows - 1) // group, -1)
        for size in (16, 32, 128):
            s = steps_of(low, high, window, sinks, size)
            held = [range(begins(s, k, size), begins(s, k, size) + size) for k in range(s[2])]
            assert len({r.start for r in held}) == len(held)
            have = {j for r in held for j in r}
            for i in {low, high, (low + high) // 2}:
                assert all(j in have for j in range(0, i + 1) if seen(j, i, window, sinks))


def test_a_tiles_ranges_are_its_steps():
    for first, group, rows, row0, window, sinks in cases(20000):
        tiles = [(max(first + row0 // group, -1), max(first + (row0 + min(rows, 128) - 1) // group, -1)),
                 (max(first + (row0 + 128) // group, -1), -1 if rows <= 128 else max(first + (row0 + rows - 1) // group, -1))]
        s = steps_of(tiles[0][0], max(tiles[0][1], tiles[1][1]), window, sinks, 128)
        for low, high in tiles:
            sink, frm, to, whole_from, whole_to = prompt_steps(s, low, high, window, sinks)
            active = []
            for k in range(s[2]):
                t = begins(s, k, 128)
                needed = t <= high and (window == 0 or t + 127 > low - window or t < sinks)
                takes, whole = k < to and (k < sink or k >= frm), whole_from <= k < whole_to
                assert takes or not needed
                if whole:                             # all rows see all of it
                    assert takes and t + 127 <= low and (window == 0 or t > high - window)
                if needed and t + 127 <= low and (window == 0 or t > high - window):
                    assert whole or k < s[0]
                if takes:
                    active.append(k)
            assert (active[-1] if active else -1) == to - 1
