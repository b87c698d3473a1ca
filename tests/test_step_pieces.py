"""How lists of tensors are dealt out to launches (jax-gs_amd/csrc/gs_pieces.h): no launch of more work
items than HIP takes, whatever the sizes, and every element in one launch."""
import os
import subprocess

import pytest

from test_cull import _CSRC, HIPCC

_HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def pieces_bin(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not found")
    out = str(tmp_path_factory.mktemp("pieces") / "step_pieces")
    subprocess.run([HIPCC, "-O2", "-std=c++17", "-I", _CSRC, os.path.join(_HERE, "step_pieces.cpp"), "-o", out],
                   check=True, capture_output=True)
    return out


@pytest.mark.parametrize("seed", [1, 2])
def test_launches_take_every_workgroup_once_and_none_too_many(pieces_bin, seed):
    res = subprocess.run([pieces_bin, "2000", str(seed)], capture_output=True, text=True)
    lists, launches, most, faults = (int(v) for v in res.stdout.split())
    assert faults == 0 and res.returncode == 0
    # full launches are among them
    assert launches > lists and (1 << 24) - (1 << 20) <= most < 1 << 24
