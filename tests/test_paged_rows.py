"""CPU model of how the prompt kernel reads row_start: 32 entries at a time, once
over the list and again at look-ups (kestrel_b200/csrc/attn_prompt.cu). Whatever
the list holds, the entries taken share no row, so that their row tiles stay
within what the launch reckons with; and a look-up takes what the first time over
the list took."""
import random

import pytest


class Reader:
    def __init__(self, row_start, n, n_rows):
        self.rows, self.n, self.n_rows = row_start, n, n_rows
        self.ascend, self.known = True, False

    def chunk(self, b, last):
        """[(lo, hi)] of entries b .. b + 31, and `last` after them."""
        at = [(self.rows[i], self.rows[i + 1]) if i < self.n else (last, last) for i in range(b, b + 32)]
        wrong = [lo < last or hi < lo or hi > self.n_rows for lo, hi in at]
        if not self.ascend or (not self.known and any(wrong)):
            self.ascend = False
            top = last
            for l, (lo, hi) in enumerate(at):
                top = max(top, lo)
                if wrong[l] or lo < top:
                    at[l] = (0, 0)
            last = top
        return at, last

    def read(self):
        out, last = [], 0
        for b in range(0, self.n, 32):
            at, last = self.chunk(b, last)
            out += at
        return out[:self.n]


def lists(rng):
    n, n_rows = rng.choice([1, 2, 5, 31, 32, 33, 64, 65, 100, 200]), rng.choice([1, 3, 40, 1000])
    rows = sorted(rng.randint(0, n_rows) for _ in range(n + 1))
    for _ in range(rng.choice([0, 0, 1, 1, 2, 5, n])):
        i = rng.randrange(n + 1)
        rows[i] = rng.choice([rng.randint(-5, n_rows + 5), 0, n_rows, -2 ** 31, 2 ** 31 - 1])
    if rng.random() < 0.2:
        rows = [n_rows * (i % 2) for i in range(n + 1)]
    return rows, n, n_rows


@pytest.mark.parametrize("seed", range(4))
def test_entries_share_no_row(seed):
    rng = random.Random(seed)
    for _ in range(3000):
        rows, n, n_rows = lists(rng)
        r = Reader(rows, n, n_rows)
        first = r.read()
        r.known = True
        assert r.read() == first == r.read()
        taken = [(lo, hi) for lo, hi in first if hi > lo]
        assert all(0 <= lo and hi <= n_rows for lo, hi in taken)
        assert all(a[1] <= b[0] for a, b in zip(taken, taken[1:]))
        if all(0 <= a <= b <= n_rows for a, b in zip(rows, rows[1:])):
            assert first == list(zip(rows, rows[1:]))
        for group, tile in ((1, 128), (8, 128), (8, 256), (3, 128), (128, 256)):
            tiles = sum(-(-(hi - lo) * group // tile) for lo, hi in first)
            assert tiles <= n_rows * group // tile + min(n, n_rows)


def test_a_reader_without_the_rule_would_pass_the_bound():
    """Each entry by itself, as in 0, N, 0, N, ...: rows counted many times."""
    rows = [1280 * (i % 2) for i in range(10)]
    tiles = sum(-(-(hi - lo) // 128) for lo, hi in zip(rows, rows[1:]) if 0 <= lo <= hi <= 1280)
    assert tiles == 50 > 1280 // 128 + 9
