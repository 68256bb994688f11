"""The LDS layout of tiles that are read both by rows and transposed (lds::TileBoth), on a host build of the
kernels' own functions: every read finds what was staged for it, and neither kind has a bank conflict: 64 banks of
4 bytes; a cycle of the transposing reads serves 32 lanes, one of the 16-byte reads 16, lanes 0 to 3, 12 to 15 and 20
to 27 or the others (of each 32), as SQ_LDS_BANK_CONFLICT shows for swizzles that tell such groups apart."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "flash-attention_amd", "csrc")


@pytest.fixture(scope="module")
def at(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("lds") / "both.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, os.path.join(HERE, "lds", "fa_lds_both.cpp"),
                    "-o", out], check=True)
    return ctypes.CDLL(out).fa_lds_both


def place(at, d, row, element):
    """Byte of an element: chunk c of a row at position c ^ swz(row), rows 16 apart alike."""
    return row * 2 * d + (((element // 8) ^ at(d, 0, 0, row % 16)) << 4) + element % 8 * 2


def conflict_free(addresses, size):
    banks = [b for a in set(addresses) for b in range(a // 4, (a + size) // 4)]
    return len({b % 64 for b in banks}) == len(banks)


@pytest.mark.parametrize("d", [64, 128])
def test_swizzle(at, d):
    chunks = d // 8
    for row in range(16):
        assert 0 <= at(d, 0, 0, row) < chunks


@pytest.mark.parametrize("d", [64, 128])
def test_row_reads(at, d):
    for step in range(d // 32):
        got = [at(d, 1, lane, step) for lane in range(64)]
        assert got == [place(at, d, lane % 16, 32 * step + 8 * (lane // 16)) for lane in range(64)]
        first = [*range(4), *range(12, 16), *range(20, 28)]
        for lanes in (first, [i for i in range(32) if i not in first]):
            for half in (0, 32):
                assert conflict_free([got[half + i] for i in lanes], 16), (step, lanes[0], half)


@pytest.mark.parametrize("d", [64, 128])
def test_turned_reads(at, d):
    for block in range(d // 16):
        got = [at(d, 2, lane, block) for lane in range(64)]
        assert got == [place(at, d, 4 * (lane // 16) + lane % 16 // 4, 16 * block + 4 * (lane % 4)) for lane in range(64)]
        for half in range(2):
            assert conflict_free(got[32 * half:32 * half + 32], 8), (block, half)
