"""What autograd is told by rotary, rotary_, paged_append, paged_attn and verify_draft, without a GPU: the wrappers run on fake
tensors, a launch is counted instead of made."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

from musicgeneration_amd import ops

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    made, seen = [], {}
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: seen.setdefault(id(t), (t, 16 * (len(seen) + 1)))[1])
    monkeypatch.setattr(ops, "_on", lambda device, entry, args: made.append(entry) or 0)
    with FakeTensorMode():
        yield made


def E(*shape, dtype=F32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _cache(dtype=BF16, pages=6, Hkv=2, page=16, dh=64, B=3, width=4):
    return dict(kcache=E(pages, Hkv, page, dh, dtype=dtype), vcache=E(pages, Hkv, page, dh, dtype=dtype),
                table=E(B, width, dtype=I32), lens=E(B, dtype=I32))


def _dual(t):
    return fwd.make_dual(t, E(*t.shape, dtype=t.dtype))


@pytest.mark.parametrize("on_graph", [False, True])
def test_rotary_carries_tangents(launches, on_graph):
    x, c = E(2, 5, 3, 16).requires_grad_(on_graph), E(8, 4)
    with fwd.dual_level():
        y, tangent = fwd.unpack_dual(ops.rotary(_dual(x), c, c))
        assert y.requires_grad == on_graph and tangent is not None and tangent.shape == x.shape
        assert len(launches) == 2
        # a tangent with a graph of its own keeps it
        t = E(2, 5, 3, 16).requires_grad_()
        assert fwd.unpack_dual(ops.rotary(fwd.make_dual(x, t), c, c)).tangent.requires_grad
    y = ops.rotary(E(2, 5, 3, 16).requires_grad_(on_graph), c, c)
    assert y.requires_grad == on_graph


def test_what_forms_no_tangent_refuses_one(launches):
    c = E(8, 4)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            ops.rotary_(_dual(E(2, 5, 3, 16)), c, c)
        for cos, sin in ((_dual(c), c), (c, _dual(c))):
            with pytest.raises(ValueError, match="no gradient"):
                ops.rotary(E(2, 5, 3, 16), cos, sin)
        qkv, q, cache = E(3, 2, 8 * 64, dtype=BF16), E(3, 2, 4, 64, dtype=BF16), _cache()
        refuse = lambda fn, *a, **kw: pytest.raises(RuntimeError, fn, *a, **kw).match("tangent")     # noqa: E731
        refuse(ops.paged_append, _dual(qkv), **cache, n_heads=4)
        refuse(ops.paged_attn, _dual(q), **cache)
        refuse(ops.paged_attn, q, **cache, slopes=_dual(E(4)))
        for which in ("kcache", "vcache"):
            with_tangent = {**cache, which: _dual(cache[which])}
            refuse(ops.paged_append, qkv, **with_tangent, n_heads=4)
            refuse(ops.paged_attn, q, **with_tangent)
        p, d, x, u = E(3, 5, 100), E(3, 4, 100), E(3, 4, dtype=I32), E(3, 5)
        refuse(ops.verify_draft, _dual(p), x, u, d)
        refuse(ops.verify_draft, p, x, u, _dual(d))
    assert not launches


def test_writes_in_place_raise_the_version(launches):
    """What an earlier operation saved for its backward must not be taken for the values it saw."""
    x, c = E(2, 5, 3, 16), E(8, 4)
    before = x._version
    ops.rotary_(x[:, 1:], c, c)
    assert x._version > before
    qkv, cache = E(3, 2, 8 * 64, dtype=BF16), _cache()
    for tables in ({}, {"cos": E(9, 32), "sin": E(9, 32)}):
        before = {n: t._version for n, t in {**cache, "qkv": qkv}.items()}
        ops.paged_append(qkv, **cache, n_heads=4, **tables)
        after = {n: t._version for n, t in {**cache, "qkv": qkv}.items()}
        assert {n for n in after if after[n] > before[n]} == {"kcache", "vcache"}
    q = E(3, 2, 4, 64, dtype=BF16)
    before = {n: t._version for n, t in {**cache, "q": q}.items()}
    ops.paged_attn(q, **cache)
    assert before == {n: t._version for n, t in {**cache, "q": q}.items()}
