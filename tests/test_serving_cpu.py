"""What rotary, rope_tables, paged_append, paged_attn and verify_draft refuse: checked without a GPU.

The Python checks run on fake tensors (no memory, no launch: every call here must raise before it comes to one), the C
entry points on pointers that are never followed."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from musicgeneration_amd import ops
from musicgeneration_amd._lib import lib

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture(autouse=True)
def fake():
    with FakeTensorMode():
        yield


def E(*shape, dtype=F32, device="cuda"):
    return torch.empty(*shape, dtype=dtype, device=device)


def refuse(error, text, fn, *a, **kw):
    with pytest.raises(error, match=text):
        fn(*a, **kw)


@pytest.mark.parametrize("fn", [ops.rotary, ops.rotary_])
def test_rotary_refuses(fn):
    x, c = E(2, 5, 3, 16), E(8, 4)
    refuse(RuntimeError, "GPU only", fn, E(2, 5, 3, 16, device="cpu"), c, c)
    refuse(TypeError, "float32 or bfloat16", fn, E(2, 5, 3, 16, dtype=torch.float16), c, c)
    refuse(ValueError, "batch, seq, heads", fn, E(5, 3, 16), c, c)
    refuse(ValueError, "unit stride", fn, E(2, 5, 16, 3).transpose(2, 3), c, c)
    refuse(ValueError, "even head dim", fn, E(2, 5, 3, 15), c, c)
    refuse(ValueError, "layout", fn, x, c, c, None, "neox")
    refuse(ValueError, "rd <=", fn, x, E(8, 9), E(8, 9))
    refuse(ValueError, "rd <=", fn, x, E(8, 0), E(8, 0))
    refuse(ValueError, "rd <=", fn, x, c, E(8, 3))
    refuse(TypeError, "cos", fn, x, E(8, 4, dtype=BF16), c)
    refuse(RuntimeError, "sin is on", fn, x, c, E(8, 4, device="cpu"))
    refuse(ValueError, "contiguous", fn, x, E(4, 8).t(), c)
    refuse(ValueError, "tables of 4", fn, x, E(4, 4), E(4, 4))
    refuse(ValueError, "no gradient", fn, x, c.clone().requires_grad_(), c)
    refuse(ValueError, "positions", fn, x, c, c, E(2, 4, dtype=I32))
    refuse(TypeError, "positions", fn, x, c, c, E(2, 5))
    refuse(ValueError, "contiguous", fn, x, c, c, E(5, 2, dtype=I32).t())


def test_rotary_in_place_refuses():
    c = E(8, 4)
    refuse(RuntimeError, "autograd", ops.rotary_, E(2, 5, 3, 16).requires_grad_(), c, c)
    refuse(ValueError, "share memory", ops.rotary_, E(1, 5, 3, 16).expand(2, 5, 3, 16), c, c)
    refuse(ValueError, "share memory", ops.rotary_, E(200).as_strided((2, 5, 3, 16), (60, 24, 8, 1)), c, c)


def test_rope_tables_refuse():
    for kw in ({"n": 0}, {"rotary_dim": 7}, {"rotary_dim": 0}, {"base": 1.0}, {"base": float("nan")}, {"factor": 0.5},
               {"factor": float("inf")}, {"scaling": "other"}, {"scaling": "by_parts", "factor": 2.0},
               {"scaling": "ntk", "rotary_dim": 2}):
        refuse(ValueError, "rope_tables", ops.rope_tables, **{"n": 4, "rotary_dim": 8, **kw})
    refuse(RuntimeError, "GPU only", ops.rope_tables, 4, 8, device="cpu")


def _cache(dtype=BF16, pages=6, Hkv=2, page=16, dh=64, B=3, width=4):
    return dict(kcache=E(pages, Hkv, page, dh, dtype=dtype), vcache=E(pages, Hkv, page, dh, dtype=dtype),
                table=E(B, width, dtype=I32), lens=E(B, dtype=I32))


def _bad_caches():
    ok = _cache()
    yield RuntimeError, "kcache is on", {**ok, "kcache": E(6, 2, 16, 64, dtype=BF16, device="cpu")}
    yield TypeError, "vcache", {**ok, "vcache": E(6, 2, 16, 64)}
    yield ValueError, "contiguous", {**ok, "kcache": E(6, 16, 2, 64, dtype=BF16).transpose(1, 2)}
    yield ValueError, "two", {**ok, "vcache": E(6, 2, 8, 64, dtype=BF16)}
    yield ValueError, "two", {**ok, "kcache": E(0, 2, 16, 64, dtype=BF16), "vcache": E(0, 2, 16, 64, dtype=BF16)}
    yield TypeError, "table", {**ok, "table": E(3, 4, dtype=torch.int64)}
    yield ValueError, "table", {**ok, "table": E(2, 4, dtype=I32)}
    yield ValueError, "table", {**ok, "table": E(3, 0, dtype=I32)}
    yield TypeError, "lens", {**ok, "lens": E(3, dtype=torch.int64)}
    yield ValueError, "lens", {**ok, "lens": E(3, 1, dtype=I32)}


@pytest.fixture
def pointers(monkeypatch):
    """data_ptr of fake tensors: distinct multiples of 16, never followed (every call that gets one raises first)."""
    seen = {}
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: seen.setdefault(id(t), 16 * (len(seen) + 1)))
    keep = []
    yield keep


def test_append_refuses_shapes(pointers):
    ok, qkv, c = _cache(), E(3, 2, 8 * 64, dtype=BF16), E(99, 32)
    call = lambda q=qkv, n=4, cos=None, sin=None, cache=ok, **kw: ops.paged_append(q, **cache, n_heads=n, cos=cos, sin=sin, **kw)  # noqa: E731
    for error, text, cache in _bad_caches():
        pointers.append(cache)
        refuse(error, text, call, cache=cache)
    refuse(RuntimeError, "GPU only", call, E(3, 2, 512, dtype=BF16, device="cpu"))
    refuse(TypeError, "float32 or bfloat16", call, E(3, 2, 512, dtype=torch.float16))
    refuse(RuntimeError, "no gradient", call, E(3, 2, 512, dtype=BF16).requires_grad_())
    refuse(ValueError, "contiguous", call, E(3, 512, 2, dtype=BF16).transpose(1, 2))
    refuse(ValueError, "qkv", call, n=5)
    refuse(ValueError, "qkv", call, n=0)
    refuse(ValueError, "qkv", call, E(4, 2, 512, dtype=BF16))
    refuse(ValueError, "qkv", call, E(6, 512, dtype=BF16))
    refuse(ValueError, "ragged", call, cu_rows=E(4, dtype=I32))
    refuse(ValueError, "4 offsets", call, E(6, 512, dtype=BF16), cu_rows=E(3, dtype=I32))
    refuse(TypeError, "cu_rows", call, E(6, 512, dtype=BF16), cu_rows=E(4, dtype=torch.int64))
    refuse(ValueError, "together", call, cos=c)
    refuse(ValueError, "layout", call, cos=c, sin=c, layout="other")
    refuse(ValueError, "offset", call, cos=c, sin=c, offset=-1)
    refuse(ValueError, "rd <=", call, cos=E(99, 33), sin=E(99, 33))
    pointers.append(c)


def test_attn_refuses(pointers):
    ok, q = _cache(), E(3, 2, 4, 64, dtype=BF16)
    call = lambda q=q, cache=ok, **kw: ops.paged_attn(q, **cache, **kw)  # noqa: E731
    refuse(RuntimeError, "GPU only", call, E(3, 2, 4, 64, dtype=BF16, device="cpu"))
    refuse(RuntimeError, "no gradient", call, E(3, 2, 4, 64, dtype=BF16).requires_grad_())
    for error, text, cache in _bad_caches():
        pointers.append(cache)
        refuse(error, text, call, cache=cache)
    for dh in (4, 12, 264):
        cache = _cache(dh=dh)
        pointers.append(cache)
        refuse(ValueError, "head dim", call, E(3, 2, 4, dh, dtype=BF16), cache)
    refuse(ValueError, "q \\(", call, E(2, 2, 4, 64, dtype=BF16))
    refuse(ValueError, "q \\(", call, E(3, 2, 4, 32, dtype=BF16))
    refuse(ValueError, "ragged", call, cu_rows=E(4, dtype=I32))
    refuse(ValueError, "query heads", call, E(3, 2, 5, 64, dtype=BF16))
    refuse(ValueError, "query heads", call, E(3, 2, 0, 64, dtype=BF16))
    refuse(ValueError, "slopes", call, slopes=E(3))
    refuse(TypeError, "slopes", call, slopes=E(4, dtype=BF16))
    refuse(ValueError, "prefix", call, prefix_len=3)
    refuse(ValueError, "prefix", call, prefix=E(2, dtype=I32), prefix_len=-1)
    refuse(ValueError, "prefix", call, prefix=E(2, dtype=I32), prefix_len=33)
    refuse(TypeError, "prefix", call, prefix=E(2, dtype=torch.int64), prefix_len=3)
    refuse(ValueError, "scale", call, scale=float("nan"))


def test_verify_refuses():
    p, x, u, d = E(3, 5, 100), E(3, 4, dtype=torch.int64), E(3, 5), E(3, 4, 100)
    v = ops.verify_draft
    refuse(RuntimeError, "GPU only", v, E(3, 5, 100, device="cpu"), x, u)
    refuse(TypeError, "float32 or bfloat16", v, E(3, 5, 100, dtype=torch.float16), x, u)
    refuse(RuntimeError, "no gradient", v, E(3, 5, 100).requires_grad_(), x, u)
    refuse(ValueError, "target", v, E(5, 100), x, u)
    refuse(ValueError, "target", v, E(3, 5, 0), x, u)
    refuse(ValueError, "target", v, E(3, 100, 5).transpose(1, 2), x, u)
    refuse(ValueError, "tokens", v, p, E(3, 5, dtype=I32), u)
    refuse(TypeError, "tokens", v, p, E(3, 4), u)
    refuse(ValueError, "uniforms", v, p, x, E(3, 4))
    refuse(TypeError, "uniforms", v, p, x, E(3, 5, dtype=torch.float64))
    refuse(TypeError, "draft", v, p, x, u, E(3, 4, 100, dtype=BF16))
    refuse(ValueError, "draft", v, p, x, u, E(3, 5, 100))
    refuse(ValueError, "counts", v, p, x, u, d, E(2, dtype=I32))
    refuse(TypeError, "counts", v, p, x, u, d, E(3, dtype=torch.int64))


def test_c_entry_points_refuse():
    """Bad arguments come back as codes; nothing is launched (the pointers are not memory)."""
    a, b, n = 16, 32, None
    rot = lambda x=a, y=b, cos=a, B=1, S=2, H=1, dh=8, rd=8, rows=4, xs=(16, 8, 8), ys=(16, 8, 8), half=0, dt=0: \
        lib.mgx_rotary(x, y, cos, a, n, 0, B, S, H, dh, rd, rows, *xs, *ys, half, 0, dt, n)       # noqa: E731
    for kw in ({"x": n}, {"cos": n}, {"B": 0}, {"S": -1}, {"rd": 0}, {"rd": 3}, {"rd": 10}, {"dh": 7, "rd": 2}, {"rows": 1}, {"dt": 2},
               {"y": a, "ys": (32, 8, 8)}):
        assert rot(**kw) < 0, kw
    app = lambda qkv=a, q=a, k=a, T=2, B=2, R=1, Hq=1, Hkv=1, dh=8, rd=8, page=4, pages=2, width=2, rows=4, off=0, dt=1, cos=a: \
        lib.mgx_paged_append(qkv, q, k, b, a, a, n, cos, cos, T, B, R, Hq, Hkv, dh, rd, page, pages, width, rows, off, 0, dt, n)   # noqa: E731
    for kw in ({"qkv": n}, {"q": n}, {"T": 0}, {"T": 3}, {"B": 0}, {"Hkv": 0}, {"dh": 12}, {"rd": 9}, {"rd": 16}, {"page": 0}, {"pages": 0},
               {"width": 0}, {"rows": 0}, {"off": -1}, {"dt": 7}, {"qkv": 8}, {"k": 24}, {"page": 2 ** 30, "width": 4}):
        assert app(**kw) < 0, kw
    att = lambda q=a, qs=8, k=a, prefix=n, T=2, B=2, R=1, Hq=1, Hkv=1, dh=8, page=4, pages=2, width=2, P=0, mr=1, ml=8, dt=1: \
        lib.mgx_paged_attn(q, qs, k, b, a, a, n, n, prefix, a, n, T, B, R, Hq, Hkv, dh, page, pages, width, P, mr, ml, 1.0, dt, n)   # noqa: E731
    for kw in ({"q": n}, {"qs": 7}, {"qs": 12}, {"T": 0}, {"T": 5}, {"Hq": 0}, {"Hq": 3, "Hkv": 2}, {"dh": 20}, {"dh": 264, "qs": 264}, {"P": 3},
               {"P": -1}, {"mr": 0}, {"ml": 0}, {"dt": 5}, {"q": 4}, {"page": 2 ** 28, "width": 4}):
        assert att(**kw) < 0, kw
    ver = lambda t=a, tok=a, B=1, k=1, V=4, dt=0: lib.mgx_verify_draft(t, n, tok, 0, a, n, a, a, B, k, V, 8, 4, 0, 0, dt, n)   # noqa: E731
    for kw in ({"t": n}, {"tok": n}, {"B": 0}, {"k": -1}, {"V": 0}, {"V": 2 ** 31}, {"dt": 3}):
        assert ver(**kw) < 0, kw
    tab = lambda f=a, nn=4, half=2: lib.mgx_rope_tables(f, a, a, nn, half, 1.0, n)      # noqa: E731
    for kw in ({"f": n}, {"nn": 0}, {"half": 0}):
        assert tab(**kw) < 0, kw
    assert lib.mgx_last_error_string()


def test_caches_and_weights_that_want_a_gradient_are_refused(pointers):
    """Filing and attention form no gradient: of the caches no more than of q."""
    qkv, q = E(3, 2, 8 * 64, dtype=BF16), E(3, 2, 4, 64, dtype=BF16)
    for which in ("kcache", "vcache"):
        cache = _cache()
        cache[which].requires_grad_()
        pointers.append(cache)
        refuse(RuntimeError, "no gradient", ops.paged_append, qkv, **cache, n_heads=4)
        refuse(RuntimeError, "no gradient", ops.paged_attn, q, **cache)
    refuse(RuntimeError, "no gradient", ops.paged_attn, q, **_cache(), slopes=E(4).requires_grad_())


def test_launches_beyond_the_grid_are_refused():
    """2^32 threads a launch dimension: more is refused as unsupported, before a launch is tried (the pointers are not memory)."""
    a, b, n, unsupported = 16, 32, None, -2
    big = 1 << 24
    assert lib.mgx_rotary(a, a, a, a, n, 0, 1, 2 ** 31 - 1, 1, 64, 64, 2 ** 31 - 1, 64, 64, 64, 64, 64, 64, 0, 0, 1, n) == unsupported
    assert lib.mgx_rope_tables(a, a, a, 1 << 31, 2, 1.0, n) == unsupported
    assert lib.mgx_verify_draft(a, n, a, 0, a, n, a, a, 1 << 22, 1, 4, 8, 4, 0, 0, 0, n) == unsupported
    append = lambda T, dh, rd: lib.mgx_paged_append(a, a, a, b, a, a, n, a, a, T, T, 1, 8, 8, dh, rd, 4, 2, 2, 4, 0, 0, 1, n)   # noqa: E731
    assert append(1 << 28, 128, 128) == unsupported
    attn = lambda T, Hq, dh, cu=n, R=1, B=None, mr=1: lib.mgx_paged_attn(   # noqa: E731
        a, Hq * dh, a, b, a, a, cu, n, n, a, a, T, T if B is None else B, R, Hq, 1, dh, 4, 2, 2, 0, mr, 8, 1.0, 1, n)
    assert attn(big, 1, 136) == unsupported             # a workgroup a row
    assert attn(big, 1, 64) == unsupported              # a workgroup a sequence
