"""Outputs may lie between the rows of an input (column slices of one buffer) but
not share its memory: d1._rows.apart against the bytes themselves."""
import random

import pytest
import torch


def test_against_the_bytes():
    from d1._rows import apart, rows_meet
    rng = random.Random(8)
    seen = [0, 0]
    for _ in range(20000):
        size = rng.choice([1, 2, 4])
        ld = rng.randrange(0, 20)
        a = [1000 + size * rng.randrange(60), rng.randrange(0, 6), rng.randrange(1, 8), ld]
        b = [1000 + size * rng.randrange(60), rng.randrange(0, 6), rng.randrange(1, 8), ld if rng.random() < 0.6 else rng.randrange(0, 20)]
        cells = [{p + (i * step + k) * size for i in range(rows) for k in range(n)} for p, rows, n, step in (a, b)]
        want = bool(cells[0] & cells[1])
        spans = [(p, rows, n * size, step * size) for p, rows, n, step in (a, b)]
        assert rows_meet(*spans[0], *spans[1]) == rows_meet(*spans[1], *spans[0]) == want, (size, a, b)
        seen[want] += 1
        if want:
            with pytest.raises(ValueError):
                apart(a, b, size, 'a', 'b')
        else:
            apart(a, b, size, 'a', 'b')
    assert min(seen) > 3000


def test_column_slices_of_one_buffer():
    from d1._rows import apart, matrix
    buf = torch.zeros(50, 64, dtype=torch.bfloat16)
    left, right = matrix(buf[:, :32], 'x'), matrix(buf[:, 32:], 'y')
    apart(left, right, 2, 'x', 'y')
    for bad in (buf[:, 31:63], buf[:, :32], buf[1:, :32], buf[:, 20:40]):
        with pytest.raises(ValueError):
            apart(matrix(bad, 'y'), left, 2, 'y', 'x')
