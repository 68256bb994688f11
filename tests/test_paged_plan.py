"""CPU tests of the paged calls' plans: what the host allocates and launches holds
every tile and piece that the kernels make of the offsets they read, whatever
those are.  The plan is the library's; the kernels' arithmetic is theirs, built
for the host (tests/plan/fa_paged_plan.cpp)."""
from __future__ import annotations

import ctypes
import os
import random
import subprocess

import pytest

import abi_ctypes as A

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(A.REPO_ROOT, "flash-attention_amd", "csrc")
CUS = 256
CHUNK_ROWS = 128


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("plan") / "libfa_paged_plan.so")
    lib_dir = os.path.dirname(A.LIB_PATH)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__=1",
                    "-I", os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"), "-I", CSRC,
                    os.path.join(HERE, "plan", "fa_paged_plan.cpp"), A.LIB_PATH, f"-Wl,-rpath,{lib_dir}",
                    "-o", out], check=True)
    lib = ctypes.CDLL(out)
    lib.partial_tile.restype = ctypes.c_int64
    return lib


def plan(lib, tokens, batch, kv_heads, group, d, max_q, max_kv, causal=True, cus=CUS):
    out = (ctypes.c_int64 * 8)()
    lib.paged_plan(tokens, batch, kv_heads, group, d, max_q, max_kv, int(causal), cus, out)
    return dict(zip(("rows", "slots", "splits", "chunk", "conc", "pieces", "ws_rows", "bytes"), out))


def found_tiles(cu, tokens, max_q, group):
    """Tiles that a list of up to 64 sequences counts, offsets limited as the kernels do."""
    n = 0
    for a, b in zip(cu, cu[1:]):
        c0 = min(max(a, 0), tokens)
        c1 = min(max(b, c0), tokens)
        n += -(-min(c1 - c0, max_q) * group // CHUNK_ROWS)
    return n


def check(lib, cu, tokens, kv_heads, group, max_q, max_kv, causal=True):
    """Every piece has rows in the workspace and a place in the grid, every cut tile a place in the join."""
    batch = len(cu) - 1
    p = plan(lib, tokens, batch, kv_heads, group, 64, max_q, max_kv, causal)
    if p["rows"] != CHUNK_ROWS:
        return None
    out = (ctypes.c_int * 4)()
    found = found_tiles(cu, tokens, max_q, group) if batch <= 64 else p["slots"]
    lib.last_round(found, p["slots"], p["conc"], p["pieces"], max_kv, out)
    count, whole, rest, pieces = out
    assert count <= p["slots"] and whole + rest * pieces <= p["slots"] + p["pieces"]
    if pieces > 1:
        last = lib.partial_tile(kv_heads - 1, p["pieces"], rest - 1, pieces, pieces - 1)
        assert (last + 1) * CHUNK_ROWS <= p["ws_rows"], (cu, tokens, group, max_kv, out[:], p)
        # a kv head's pieces end before the next one's begin
        assert rest * pieces <= p["pieces"]
        assert rest <= min(p["conc"] - 1, p["slots"])
    return found, p["slots"], pieces


def test_descending_offsets_that_make_more_tiles_than_slots(plans):
    """Two sequences on the same rows: eight tiles, where the launch counts on seven."""
    found, slots, pieces = check(plans, [0, 64, 0, 64], 64, 1, 8, 64, 40000)
    assert found > slots and pieces > 1


@pytest.mark.parametrize("kind", ["descending", "ascending", "any"])
def test_any_offsets_stay_in_the_workspace(plans, kind):
    rng = random.Random(7)
    cut = 0
    for _ in range(4000):
        batch, tokens = rng.choice([1, 2, 3, 5, 9, 33, 64]), rng.choice([1, 17, 64, 100, 999, 5000])
        kv_heads, group = rng.choice([1, 2, 3, 4, 8, 40]), rng.choice([1, 2, 5, 8, 40])
        cu = [rng.randint(0, tokens) for _ in range(batch + 1)]
        if kind == "ascending":
            cu.sort()
        elif kind == "descending":
            cu = [0 if i % 2 == 0 else tokens for i in range(batch + 1)]
        else:
            cu = [rng.choice([x, -x, x * 7, 2 ** 31 - 1, -2 ** 31]) for x in cu]
        got = check(plans, cu, tokens, kv_heads, group, rng.choice([1, 40, tokens]),
                    rng.choice([1, 700, 1025, 9000, 131072]), rng.random() < 0.8)
        cut += got is not None and got[2] > 1
    assert cut > 200


@pytest.mark.parametrize("kv_heads,cus", [(257, 256), (512, 256), (513, 256), (1000, 256), (64, 32), (33, 32), (5, 2)])
@pytest.mark.parametrize("batch", [1, 9, 70])
def test_as_many_heads_as_compute_units_cut_nothing(plans, kv_heads, cus, batch):
    """Where a kv head has one workgroup at a time, every round is a whole one: no
    pieces, no workspace and no launch that joins them (its grid would be empty)."""
    p = plan(plans, 400, batch, kv_heads, 1, 64, 100, 4096, cus=cus)
    assert p["rows"] == CHUNK_ROWS and (p["conc"] == 1) == (kv_heads > cus)
    if p["conc"] == 1:
        assert p["pieces"] == 0 and p["ws_rows"] == 0 and p["bytes"] == 0


def test_a_call_that_may_cut_has_tiles_to_join(plans):
    rng = random.Random(8)
    for _ in range(3000):
        p = plan(plans, rng.choice([40, 400, 5000]), rng.choice([1, 4, 9, 64, 200]), rng.randint(1, 600), 1, 64,
                 rng.choice([33, 400, 5000]), rng.choice([64, 1025, 100000]), rng.random() < 0.5, rng.choice([8, 32, 256]))
        assert p["pieces"] == 0 or min(p["conc"] - 1, p["slots"]) > 0, p
