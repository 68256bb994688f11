"""CPU tests of fa::may_overlap, by which the binding refuses results over what a
call reads: never false where two sets of rows share an element, and exact for
views of one buffer (the same strides)."""
from __future__ import annotations

import ctypes
import itertools
import os
import random
import subprocess

import pytest

import abi_ctypes as A

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(A.REPO_ROOT, "flash-attention_amd", "csrc")


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("overlap") / "libfa_row_overlap.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(A.REPO_ROOT, "include"),
                    "-I", CSRC, os.path.join(HERE, "plan", "fa_row_overlap.cpp"), A.LIB_PATH,
                    f"-Wl,-rpath,{os.path.dirname(A.LIB_PATH)}", "-o", out], check=True)
    f = ctypes.CDLL(out).row_overlap
    V = ctypes.c_int64 * 3

    def call(a, b):
        args = []
        for base, strides, sizes, row in (a, b):
            args += [ctypes.c_int64(2 * base), V(*strides), V(*sizes), len(strides), ctypes.c_int64(row)]
        got = bool(f(*args))
        args = args[5:] + args[:5]
        assert bool(f(*args)) == got
        return got

    return call


def elements(x):
    base, strides, sizes, row = x
    return {base + sum(i * s for i, s in zip(at, strides)) + e
            for at in itertools.product(*(range(n) for n in sizes)) for e in range(row)}


def test_views_of_one_buffer_exactly(overlap):
    """The same strides, any order of them, sizes of each view's own."""
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        row = rng.choice([1, 3, 4])
        sizes, strides, reach = [], [], row
        for _ in range(rng.randint(1, 3)):
            s = reach + rng.choice([0, 0, 1, row, 2 * row, 5])
            n = rng.randint(1, 4)
            strides.append(s)
            sizes.append(n)
            reach = s * n
        order = rng.sample(range(len(strides)), len(strides))
        strides, sizes = [strides[i] for i in order], [sizes[i] for i in order]
        a = (100 + rng.randint(0, 20), strides, sizes, row)
        other = [max(0, n - rng.choice([0, 0, 0, 1, n])) if rng.random() < 0.3 else n for n in sizes]
        b = (100 + rng.randint(-20, 20) + rng.choice([0, 0, *strides]), strides, other, row)
        want = bool(elements(a) & elements(b))
        assert overlap(a, b) == want, (a, b)
        seen[want] += 1
    assert min(seen.values()) > 500


def test_never_missed_for_any_two_layouts(overlap):
    rng = random.Random(2)
    hits = clear = 0
    for _ in range(6000):
        sets = []
        for _ in range(2):
            n = rng.randint(1, 3)
            sets.append((100 + rng.randint(0, 40), [rng.choice([0, 2, 4, 6, 8, 12, 16, 24, 40]) for _ in range(n)],
                         [rng.randint(0, 4) for _ in range(n)], rng.choice([1, 2, 4])))
        a, b = sets
        got = overlap(a, b)
        if elements(a) & elements(b):
            assert got, (a, b)
            hits += 1
        clear += not got
    assert hits > 500 and clear > 500


def test_the_layouts_of_a_program(overlap):
    D, T, H, KH = 64, 45, 4, 2
    row = (2 * H + 2 * KH) * D
    head = lambda i, n: (i * D, [row, D], [T, n], D)  # noqa: E731  heads i.. of a projection
    assert not overlap(head(0, H), head(H, KH)) and not overlap(head(H, KH), head(H + KH, KH))
    assert overlap(head(0, H), head(H - 1, KH)) and overlap(head(0, H), head(0, 1))
    page = 16 * D
    pool = lambda i: (i * KH * page, [2 * KH * page, page, D], [9, KH, 16], D)  # noqa: E731  [pages, 2, KH, 16, D]
    assert not overlap(pool(0), pool(1)) and overlap(pool(0), pool(2)) and overlap(pool(1), pool(1))
    half = lambda i: (i * D, [KH * 2 * page, 2 * page, 2 * D], [9, KH, 16], D)  # noqa: E731  [pages, KH, 16, 2 D]
    assert not overlap(half(0), half(1)) and overlap(half(0), half(2))
    keys = lambda i: (i * D, [16 * KH * 2 * D, 2 * D, KH * 2 * D], [9, KH, 16], D)  # noqa: E731  [pages, 16, KH, 2, D]
    assert not overlap(keys(0), keys(1)) and overlap(keys(0), keys(2))
    # one token, whose stride means nothing; expanded rows beside a buffer of their own
    assert not overlap((0, [0, D], [1, H], D), (H * D, [0, D], [1, H], D))
    assert overlap((0, [0, D], [1, H], D), (H * D - 1, [0, D], [1, H], D))
    assert not overlap((0, [0, 0], [T, H], D), (D, [H * D, D], [T, H], D))
    # huge pools, far apart and interleaved
    big = 2 ** 40
    assert not overlap((0, [2 * big, D], [2 ** 20, 16], D), (big, [2 * big, D], [2 ** 20, 16], D))
    assert overlap((0, [2 * big, D], [2 ** 20, 16], D), (big, [big, D], [2 ** 20, 16], D))
