"""What speculative decoding's entry points refuse on the host, each by its own message
(the test for a device put aside, so that nothing else can be what refuses)."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from kempnerforge_amd import _lib, ops
from test_speculative import no_device  # noqa: F401

BIG = (1 << 32) + 8  # 8 in a C int


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("what,size", [("batch", 0), ("n_heads", 2), ("n_kv_heads", 1),
                                       ("max_seq_len", 2), ("head_dim", 3)])
def test_sizes_past_a_c_int(no_device, what, size):  # noqa: F811
    """They would reach the library as other sizes."""
    B, N, Hq, Hkv, S, D = 1, 2, 8, 8, 16, 8
    if what == "batch":
        B = BIG
    elif what == "n_heads":
        Hq = BIG
    elif what == "n_kv_heads":
        Hkv = BIG
    elif what == "max_seq_len":
        S = BIG
    else:
        D = BIG
    i32, f32 = torch.int32, torch.float32
    caches = [_meta(B, Hkv, S, D) for _ in range(2)]
    with pytest.raises(ValueError, match=f"{what} is at most"):
        ops.tree_decode_raw(_meta(B, N, Hq, D), _meta(B, N, Hkv, D), _meta(B, N, Hkv, D), *caches,
                            _meta(B, dtype=i32), _meta(16, D // 2, dtype=f32),
                            _meta(16, D // 2, dtype=f32), rope_row_offset=0, max_len=10)
    if what != "n_heads":
        with pytest.raises(ValueError, match=f"{what} is at most"):
            ops.cache_keep_raw(caches[:1], caches[1:], [_meta(B, dtype=i32)],
                               _meta(B, 3, dtype=i32), _meta(B, dtype=i32))


@pytest.mark.parametrize("B,V,what", [(BIG, 9, "batch"), (1, BIG, "vocabulary")])
def test_logits_past_a_c_int(no_device, B, V, what):  # noqa: F811
    with pytest.raises(ValueError, match=f"{what} is at most"):
        ops.verify_drafts_raw(_meta(B, 3, V), _meta(B, 3, dtype=torch.int64),
                              _meta(B, 3, dtype=torch.float32))


@pytest.mark.parametrize("n", [2, 300])
@pytest.mark.parametrize("what", ["k", "v", "k and v", "own k and v", "lens_out", "lens", "own lens",
                                  "lens shared"])
def test_views_that_overlap(what, n):
    """Not the same tensors, but memory that one cache's workgroups write and another's
    read: views a row, or a sequence's length, apart.  (The addresses are never read.)"""
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib = _lib.load()
    B, H, S, D = 2, 2, 64, 64
    size, row = B * H * S * D * 2, D * 2
    base = 1 << 40
    k = [base + 2 * c * size for c in range(n)]
    v = [base + (2 * c + 1) * size for c in range(n)]
    lens = [(1 << 50) + 8 * c for c in range(n)]
    out = list(lens)
    if what == "k":
        k[-1] = k[0] + row
    elif what == "v":
        v[0] = v[-1] + size - row
    elif what == "k and v":
        k[-1] = v[0] - row
    elif what == "own k and v":
        v[-1] = k[-1] + row
    elif what == "lens_out":
        out[-1] = lens[-1] = out[0] + 4
    elif what == "lens":
        lens[-1] = out[0] - 4
    elif what == "own lens":
        lens[-1] = out[-1] + 4
    else:  # several caches may read one tensor that none writes, but not lens_out
        lens = [1 << 49] * n
        out[1] = lens[1]
    arr = ctypes.c_void_p * n
    p = ctypes.c_void_p(1 << 20)

    def call(B=B):
        return lib.kf_kv_cache_keep(arr(*k), arr(*v), arr(*lens), arr(*out), n, p, p, 8, B, H, S, D,
                                    1, None)

    assert call() == 1 and b"share" in lib.kf_last_error()


z = torch.zeros
CACHE, LENS = z(1, 2, 8, 64), z(1).int()
PATH, KEPT = z(1, 3).int(), z(1).int()


@pytest.mark.parametrize("change,kind,word", [
    (dict(k=[]), ValueError, "one tensor per cache"), (dict(v=[]), ValueError, "one tensor per cache"),
    (dict(lens=[LENS, LENS]), ValueError, "one tensor per cache"),
    (dict(lens=[LENS.long()]), TypeError, "int32"), (dict(lens=[z(2).int()]), TypeError, "int32"),
    (dict(out=[LENS.long()]), TypeError, "int32"), (dict(lens=[z(1, 1).int()]), TypeError, "int32"),
    (dict(path=PATH.long()), TypeError, "must be int32"), (dict(kept=KEPT.long()), TypeError, "must be int32"),
    (dict(kept=z(2).int()), TypeError, "must be int32"), (dict(path=z(2, 3).int()), ValueError, "path must be"),
    (dict(path=z(3).int()), ValueError, "path must be"), (dict(path=z(1, 0).int()), ValueError, "path must be"),
    (dict(path=z(1, 257).int()), ValueError, "path must be"),
    (dict(v=[CACHE.half()]), ValueError, "share a dtype"), (dict(v=[z(1, 2, 9, 64)]), ValueError, "share a shape"),
    (dict(v=[z(1, 8, 2, 64).transpose(1, 2)]), ValueError, "contiguous tensors"),
    (dict(k=[CACHE[0]], v=[CACHE[0].clone()]), ValueError, r"must be \[B, n_kv_heads"),
    (dict(k=[5]), ValueError, "tensors are needed"), (dict(lens=["x"]), ValueError, "must be alike"),
    (dict(), AssertionError, "nothing was refused"),
], ids=lambda x: "-".join(x) if isinstance(x, dict) else x if isinstance(x, str) else x.__name__)
def test_keep_arguments(no_device, monkeypatch, change, kind, word):  # noqa: F811
    """With the tensors taken for ones on the device."""
    class Native:
        keep = staticmethod(lambda *a: None)

        @staticmethod
        def same(*a, same=_lib.native().same):
            same(*a)
            return 0

    class OnDevice(torch.Tensor):
        def get_device(self):
            return 0

    monkeypatch.setattr(_lib, "native", lambda: Native)
    a = dict(k=[CACHE], v=[CACHE.clone()], lens=[LENS], out=None, path=PATH, kept=KEPT) | change
    path, kept = (t.as_subclass(OnDevice) for t in (a["path"], a["kept"]))
    with pytest.raises(kind, match=word):
        ops.cache_keep_raw(a["k"], a["v"], a["lens"], path, kept, lens_out=a["out"])
