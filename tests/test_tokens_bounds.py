"""Sizes that no call takes, at the workspace function of the embedding's
gradient: an answer at once, and none to allocate (CPU test)."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_workspace_of_sizes_that_are_refused():
    from src.model import _hip
    if not os.path.exists(_hip.LIB_PATH):
        pytest.skip("libwalsh_hip.so not built (run __graft_entry__.build())")
    # (in a process of its own, which ends if the function does not)
    code = f"""
import ctypes
f = ctypes.CDLL({_hip.LIB_PATH!r}).walsh_embedding_bwd_workspace_bytes
f.restype, f.argtypes = ctypes.c_int64, [ctypes.c_int64] * 3
big = 2 ** 63 - 1
for s in ((big, 1, 1), (big, big, big), (2 ** 62, 5, 8), (2 ** 28, 1, 1), (1, 2 ** 31 - 2047, 1), (1, 1, 2 ** 31 - 8),
          (2 ** 27, 1, 2 ** 13)):
    assert f(*s) == 0, s
for s in ((2 ** 28 - 1, 1, 1), (1, 2 ** 31 - 2049, 1), (0, 1, 0), (16384, 50257, 4096)):
    assert f(*s) > 0, s
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=60)
