"""What speculative decoding's entry points refuse on the host, each by its own message
(the test for a device put aside, so that nothing else can be what refuses)."""

from __future__ import annotations

import pytest
import torch

from kempnerforge_amd import ops
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
