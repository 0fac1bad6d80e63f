"""Edges of the serving operators' arguments, without a GPU: the wrappers run on fake tensors, a launch is counted instead of made;
the C entry points get pointers that are never followed."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from musicgeneration_amd import ops
from musicgeneration_amd._lib import lib

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture
def launches(monkeypatch):
    made, seen = [], {}
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: seen.setdefault(id(t), (t, 16 * (len(seen) + 1)))[1])
    monkeypatch.setattr(ops, "_on", lambda device, entry, args: made.append(entry) or 0)
    with FakeTensorMode():
        yield made


def E(*shape, dtype=F32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _cache(B, dtype=BF16, pages=6, Hkv=2, page=16, dh=64, width=4):
    return dict(kcache=E(pages, Hkv, page, dh, dtype=dtype), vcache=E(pages, Hkv, page, dh, dtype=dtype),
                table=E(B, width, dtype=I32), lens=E(B, dtype=I32))


def test_empty_batches_need_no_launch(launches):
    """A batch whose last sequence has ended, as rotary and verify_draft take it."""
    cache, c = _cache(0), E(99, 32)
    for tables in ({}, {"cos": c, "sin": c}):
        assert ops.paged_append(E(0, 2, 512, dtype=BF16), **cache, n_heads=4, **tables).shape == (0, 2, 4, 64)
        # ragged rows that belong to no sequence
        for T in (0, 3):
            assert ops.paged_append(E(T, 512, dtype=BF16), **cache, n_heads=4, cu_rows=E(1, dtype=I32), **tables).shape == (T, 4, 64)
    assert ops.paged_attn(E(0, 2, 4, 64, dtype=BF16), **cache).shape == (0, 2, 4, 64)
    for T in (0, 3):
        assert ops.paged_attn(E(T, 4, 64, dtype=BF16), **cache, cu_rows=E(1, dtype=I32)).shape == (T, 4, 64)
    assert ops.rotary(E(0, 2, 4, 64), c, c).shape == (0, 2, 4, 64)
    out, accepted = ops.verify_draft(E(0, 3, 9), E(0, 2, dtype=I32), E(0, 3))
    assert out.shape == (0, 3) and accepted.shape == (0,)
    assert not launches
    with pytest.raises(ValueError, match="table"):
        ops.paged_attn(E(0, 2, 4, 64, dtype=BF16), **{**cache, "table": E(0, 0, dtype=I32)})
