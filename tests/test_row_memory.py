"""Rows in memory against every byte written out."""

from __future__ import annotations

import itertools
import random

from marathon_amd.row_memory import Rows, share


def starts(r: Rows) -> list:
    return [r.base + sum(i * s for i, (s, _) in zip(at, r.dims))
            for at in itertools.product(*(range(n) for _, n in r.dims))]


def bytes_of(r: Rows) -> set:
    return {x + i for x in starts(r) for i in range(r.width)}


def nested(rng) -> Rows:
    """Random rows that do not lie in one another, strides in a random order."""
    width, dims = rng.randint(1, 4), []
    reach = width
    for _ in range(3):
        s, n = reach + rng.randint(0, 5), rng.randint(1, 4)
        dims.append((s, n))
        reach += s * (n - 1)
    rng.shuffle(dims)
    return Rows(rng.randint(0, 60), width, tuple(dims))


def test_rows_of_one_stride_share_memory_exactly():
    rng = random.Random(1)
    seen = set()
    for _ in range(20000):
        a = nested(rng)
        b = Rows(rng.randint(0, 200), rng.randint(1, 4),
                 tuple((s, rng.randint(1, 4)) for s, _ in a.dims))
        want = bool(bytes_of(a) & bytes_of(b))
        assert share(a, b) == share(b, a) == want, (a, b)
        seen.add((want, a.end > b.base and b.end > a.base))
    assert {(True, True), (False, True), (False, False)} <= seen


def test_a_dimension_of_one_has_any_stride():
    rng = random.Random(2)
    for _ in range(5000):
        a = nested(rng)
        b = Rows(rng.randint(0, 120), a.width, tuple((rng.choice([0, 7, 999]), 1) for _ in a.dims))
        assert share(a, b) == share(b, a) == bool(bytes_of(a) & bytes_of(b))


def test_strides_that_differ_are_never_taken_for_apart():
    rng = random.Random(3)
    for _ in range(5000):
        a, b = nested(rng), nested(rng)
        if bytes_of(a) & bytes_of(b):
            assert share(a, b)
        if a.end <= b.base or b.end <= a.base:
            assert not share(a, b)


def test_rows_that_are_repeated_or_missing():
    a = Rows(100, 8, ((0, 5), (16, 4)))  # expanded: one row over and over
    assert share(a, Rows(116, 8, ((0, 5), (16, 1)))) and not share(a, Rows(108, 8, ((0, 5), (16, 4))))
    none = Rows(100, 8, ((16, 0), (16, 4)))
    assert not share(none, a) and not share(a, none) and none.end == 100


def test_apart_is_true_of_nested_rows_alone():
    rng = random.Random(4)
    both = set()
    for _ in range(5000):
        a = nested(rng)
        assert a.apart()
        b = Rows(0, rng.randint(1, 5), tuple((rng.randint(0, 12), rng.randint(1, 4)) for _ in range(3)))
        if b.apart():
            assert len(bytes_of(b)) == b.width * len(starts(b))
        both.add(b.apart())
    assert both == {True, False}
