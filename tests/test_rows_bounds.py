"""Bounds of the row operators' C entries: every call ends, with an error where it asks for too much."""
import subprocess
import sys

import pytest

from jax_gs_amd import _lib

CHILD = """
import sys
from array import array
from jax_gs_amd import _lib
i64 = lambda x: array("q", [x]).tobytes()
row, size = int(sys.argv[1]), int(sys.argv[2])
rc = _lib.lib().gs_take_rows(None, 1, i64(4096), i64(row), i64(row), 10, i64(4096), i64(size), None, 4096, 32, 10)
print(rc, _lib.lib().gs_last_error().decode())
"""


@pytest.mark.parametrize("row", [1, 4, 5, 15, 16, 17])
def test_outputs_of_too_many_workgroups_are_refused(row):
    """A workgroup writes 512 rows of fewer than 16 bytes, else 8192 bytes, and a launch has 2^24 - 1 of them.
    In a process of its own, as a call that does not end cannot be stopped from within."""
    size = ((1 << 24) - 1) * (512 * row if row < 16 else 8192) + 1
    child = subprocess.run([sys.executable, "-c", CHILD, str(row), str(size)], capture_output=True, text=True, timeout=30,
                           cwd=_lib.__file__.rsplit("/", 2)[0])
    assert child.returncode == 0, child.stderr
    assert child.stdout.startswith(f"1 gs_take_rows: output 0 of {size} bytes"), child.stdout
