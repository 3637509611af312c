"""The entry points for several continuations of one prompt under a tracer: an error in
Python, whatever the tensors are (a C++ exception that crosses the interpreter would end
the process, so each case runs in one of its own)."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

from kempnerforge_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import sys, torch
from torch.fx.experimental.proxy_tensor import make_fx
from kempnerforge_amd import _lib, ops
_lib.native()
z = torch.zeros
calls = {
    "reorder": (lambda k, v, l, p: ops.cache_reorder_raw([k], [v], l, p),
                (z(2, 2, 8, 64), z(2, 2, 8, 64), z(2).int(), z(1, 2).int())),
    "branch": (lambda *t: ops.branch_decode_raw(*t, rope_row_offset=0, max_prefix=4, max_len=8),
               (z(2, 1, 4, 64), z(2, 1, 2, 64), z(2, 1, 2, 64), z(1, 2, 4, 64), z(1, 2, 4, 64),
                z(1).int(), z(2, 2, 8, 64), z(2, 2, 8, 64), z(2).int(), z(12, 32), z(12, 32))),
    "select": (lambda *t: ops.beam_select_raw(*t, select=2), (z(1, 3, 9), z(1, 3))),
}
for name, (f, args) in calls.items():
    try:
        make_fx(f, tracing_mode=sys.argv[1])(*args)
    except RuntimeError as e:
        print("refused", name, flush=True)
"""


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_a_traced_call_raises(mode):
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    got = subprocess.run([sys.executable, "-c", CODE, mode], cwd=ROOT, capture_output=True,
                         text=True, timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]
    assert got.stdout.split("\n")[:3] == ["refused reorder", "refused branch", "refused select"]
