"""TMEM loads are executed by a whole warp.  A wait that each lane makes for itself can leave the lanes apart (the barrier completes
between the looks of two of them), so in the text of every tensor-core kernel something that brings the warp together stands between
the last such wait and the load."""
import re

import pytest

from .conftest import PKG_ROOT

WAIT = re.compile(r"\bmbar_(?:wait|wait_cluster|test|try_wait|try_wait_cluster)\(")
REJOIN = re.compile(r"\b(?:__syncwarp|__syncthreads|__all_sync|__any_sync|__shfl_sync|named_barrier_sync|named_barrier_any)\(")
LOAD = re.compile(r"\btmem_ld_(?!wait)\w+\(")
FILES = sorted(p.name for p in (PKG_ROOT / "csrc").glob("tc_gemm*"))


def loads_apart(text):
    """Lines with a load whose nearest wait or rejoin in front of it is a wait.  (A vote or barrier around a wait comes after it.)"""
    last, bad = "rejoin", []
    for number, line in enumerate(text.splitlines(), 1):
        code = line.split("//")[0]
        if "__device__" in code:
            last = "rejoin"
            continue
        if LOAD.search(code) and last == "wait":
            bad.append(number)
        if REJOIN.search(code):
            last = "rejoin"
        elif WAIT.search(code):
            last = "wait"
    return bad


@pytest.mark.parametrize("name", FILES)
def test_warps_are_together_at_their_tmem_loads(name):
    text = (PKG_ROOT / "csrc" / name).read_text()
    assert loads_apart(text) == []


def test_the_check_finds_a_load_behind_a_wait():
    body = "if (!mbar_wait(&full, ph)) break;\n{}tmem_ld_32x32(taddr, v);\n"
    assert loads_apart(body.format("")) == [2]
    assert loads_apart(body.format("__syncwarp();\n")) == []
    assert sum(len(LOAD.findall((PKG_ROOT / "csrc" / n).read_text())) for n in FILES) >= 8
