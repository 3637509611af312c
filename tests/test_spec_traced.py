"""Speculative decoding's entry points under a tracer: an error in Python, whatever the
tensors are (a C++ exception that crosses the interpreter would end the process, so each
case runs in one of its own)."""

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
    "keep": (lambda k, v, l, p, n: ops.cache_keep_raw([k], [v], [l], p, n),
             (z(1, 2, 8, 64), z(1, 2, 8, 64), z(1).int(), z(1, 3).int(), z(1).int())),
    "tree": (lambda *t: ops.tree_decode_raw(*t, rope_row_offset=0, max_len=8),
             (z(1, 2, 4, 64), z(1, 2, 2, 64), z(1, 2, 2, 64), z(1, 2, 8, 64), z(1, 2, 8, 64),
              z(1).int(), z(8, 32), z(8, 32))),
    "verify": (lambda *t: ops.verify_drafts_raw(*t), (z(1, 3, 9), z(1, 3).long(), z(1, 3))),
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
    assert got.stdout.split("\n")[:3] == ["refused keep", "refused tree", "refused verify"]
