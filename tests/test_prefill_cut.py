"""Where a prefill launch cuts its row blocks' keys: the search against a plain
restatement, and that its answer depends on the launch alone."""
import heapq
import os
import random
import subprocess
import sys

import pytest

from ttsxabe_b200 import InvalidArgument, prefill_cut

SMS = 148


def plain_cut(lens, columns, sms):
    """Every candidate played through, none remembered, none left out by a bound."""
    work, longest = sum(lens), max(lens, default=0)
    share = work * columns / sms
    blocks = len(lens) * columns
    few = longest > 1.25 * share
    uneven = not few and longest >= 16 and blocks <= 3 * sms
    if longest < 8 or not (few or uneven):
        return 0

    def makespan(c):
        items = []
        for n in lens:
            k = -(-n // c) if c and n > c else 1
            items += [(i + 1) * n // k - i * n // k for i in range(k)]
        if len(items) > 2048:
            return 1e30
        free = [0.0] * sms
        for n in sorted(items, reverse=True):
            for _ in range(columns):
                heapq.heapreplace(free, free[0] + n + 4.0)
        return max(free) + (5.0 if c else 0.0)

    cut, best = 0, makespan(0)
    candidates = []
    if uneven and best > 1.15 * (share + 4.0 * blocks / sms):
        candidates = [c for c in (-(-longest // k) for k in (2, 3, 4, 6)) if c >= 6]
    c = (longest + 1) // 2
    while few and c >= 6 and -(-longest // c) <= 255:
        candidates.append(c)
        c -= max(2 if c > 24 else 1, c // 16)
    for c in candidates:
        t = makespan(c)
        if t < 0.95 * best and (cut == 0 or t < best):
            cut, best = c, t
    return cut


def row_blocks(past, rows):
    return [(past + min(rows, 128 * (i + 1)) + 127) // 128 for i in range((rows + 127) // 128)]


def shapes(seed, n):
    rng = random.Random(seed)
    for _ in range(n):
        lens = []
        for _ in range(rng.choice([1, 1, 2, 4, 11, 20])):
            lens += row_blocks(int(2.718 ** rng.uniform(0, 10)), int(2.718 ** rng.uniform(0, 6.5)))
        yield lens, rng.choice([1, 2, 4, 8, 16])


def test_the_search_is_the_plain_one():
    seen = set()
    for lens, columns in shapes(0, 150):
        want = plain_cut(lens, columns, SMS)
        assert prefill_cut(lens, columns, SMS) == want, (lens, columns)
        seen.add(want > 0)
    assert seen == {False, True}


def test_the_order_of_the_sequences_does_not_matter():
    rng = random.Random(1)
    for lens, columns in shapes(2, 40):
        want = prefill_cut(lens, columns)
        rng.shuffle(lens)
        assert prefill_cut(lens, columns) == want


def test_a_launch_is_cut_as_it_is_however_like_it_an_earlier_one_was():
    rng = random.Random(3)
    pairs = 0
    for _ in range(4000):
        n, longest = rng.choice([2, 3, 5, 8, 12]), rng.choice([40, 90, 172])
        a = [longest] + [rng.randint(1, longest) for _ in range(n - 1)]
        b = [longest] + [rng.randint(1, longest) for _ in range(n - 1)]
        b[-1] += sum(a) - sum(b)
        if not 1 <= b[-1] <= longest:
            continue
        columns = rng.choice([2, 4, 8])
        x, y = plain_cut(a, columns, SMS), plain_cut(b, columns, SMS)
        if x != y:
            pairs += 1
            assert prefill_cut(a, columns) == x and prefill_cut(b, columns) == y, (a, b, columns)
            assert prefill_cut(a, columns) == x
        if pairs == 12:
            break
    assert pairs == 12


def test_the_same_in_a_process_of_its_own():
    lens, columns = [172, 60, 30, 9], 8
    out = subprocess.run([sys.executable, "-c", f"from ttsxabe_b200 import prefill_cut; print(prefill_cut({lens}, {columns}))"],
                         capture_output=True, text=True, check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    for other, c in shapes(5, 70):
        prefill_cut(other, c)
    assert prefill_cut(lens, columns) == int(out.stdout) == plain_cut(lens, columns, SMS)


def test_refusals():
    assert prefill_cut([], 4) == 0
    for args in (([0], 4), ([-3], 4), ([5], 0), ([5], 4, 0), ([(1 << 22) + 1], 1)):
        with pytest.raises(InvalidArgument):
            prefill_cut(*args)
