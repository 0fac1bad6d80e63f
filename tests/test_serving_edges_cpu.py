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


def test_scales_that_fp32_does_not_hold_are_refused(launches):
    """The kernel works in fp32, with the scale times log2 e: beyond 2^127 there would be NaN."""
    cache, q = _cache(3), E(3, 2, 4, 64, dtype=BF16)
    for scale in (2.0 ** 127, -1e39, 1e300, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            ops.paged_attn(q, **cache, scale=scale)
    assert not launches
    for scale in (1e38, -1e38, 0.0, 1e-300):
        ops.paged_attn(q, **cache, scale=scale)
    assert len(launches) == 4


def test_c_entry_point_refuses_such_scales():
    a, b, n = 16, 32, None
    for scale in (2.0 ** 127, -2.0 ** 127, math.inf, -math.inf, math.nan):
        assert lib.mgx_paged_attn(a, 8, a, b, a, a, n, n, n, a, a, 2, 2, 1, 1, 1, 8, 4, 2, 2, 0, 1, 8, scale, 1, n) == -1
        assert b"scale" in lib.mgx_last_error_string()
