"""Rotary positions (mgx_rotary, mgx_rope_tables) against the 64-bit forms of serving_oracle."""
import math

import pytest
import torch

from serving_oracle import assert_turned, turn

pytestmark = pytest.mark.gpu


def _tables(n, rd):
    a = torch.arange(n).double()[:, None] * 10000.0 ** (-torch.arange(0, rd, 2).double() / rd)
    return a.cos().float(), a.sin().float()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,S,H,dh,rd", [(1, 1, 1, 2, 2), (2, 7, 3, 64, 64), (3, 33, 9, 80, 40), (1, 129, 4, 96, 20),
                                         (2, 5, 5, 128, 16), (1, 3, 2, 66, 6), (2, 260, 1, 256, 256)])
def test_rotary_forward_and_gradient(dtype, layout, B, S, H, dh, rd):
    from musicgeneration_amd import ops
    g = torch.Generator().manual_seed(B * 1000 + S)
    cos, sin = _tables(S + 3, rd)
    x = torch.randn(B, S, H, dh, generator=g).to(dtype)
    dy = torch.randn(B, S, H, dh, generator=g).to(dtype)
    for positions in (None, torch.randint(0, S + 3, (B, S), generator=g), torch.randint(0, S + 3, (B, S), generator=g).int()):
        at = torch.arange(S).expand(B, S) if positions is None else positions.long()
        c, s = cos[at][:, :, None], sin[at][:, :, None]
        xg = x.cuda().requires_grad_()
        y = ops.rotary(xg, cos.cuda(), sin.cuda(), None if positions is None else positions.cuda(), layout)
        assert_turned(y.detach(), *turn(x, c, s, layout))
        dx, = torch.autograd.grad(y, xg, dy.cuda())
        assert_turned(dx, *turn(dy, c, -s, layout))
        z = x.cuda()
        assert ops.rotary_(z, cos.cuda(), sin.cuda(), None if positions is None else positions.cuda(), layout) is z
        assert torch.equal(z, y)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary_gradient_is_that_of_differences(layout):
    from musicgeneration_amd import ops
    cos, sin = (t.cuda() for t in _tables(6, 8))
    x = torch.randn(2, 3, 2, 12, generator=torch.Generator().manual_seed(4)).cuda().requires_grad_()
    # fp32 rounding 2^-24 of values below 8 over a step of 2^-4: 2 * 8 * 2^-24 / 2^-4 < 2^-15, sums of 2 values
    assert torch.autograd.gradcheck(lambda t: ops.rotary(t, cos, sin, None, layout), (x,), eps=2.0 ** -4, atol=2.0 ** -13, rtol=0,
                                    nondet_tol=0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary_strides_alignment_and_broadcast_inputs(dtype, layout):
    from musicgeneration_amd import ops
    g = torch.Generator().manual_seed(9)
    B, S, H, dh, rd = 2, 9, 5, 64, 32
    cos, sin = _tables(S, rd)
    c, s = cos[None, :, None], sin[None, :, None]
    big = torch.randn(B, S + 2, H + 3, dh + 9, generator=g).to(dtype)
    views = [big[:, :S, :H, :dh], big[:, 1:S + 1, 2:H + 2, 8:dh + 8], big[:, :S, :H, 1:dh + 1],
             big[:, :S, :H, :dh].transpose(1, 2).contiguous().transpose(1, 2), big[:1, :1, :H, :dh].expand(B, S, H, dh)]
    for v in views:
        gpu = v.cuda() if v.stride(0) == 0 else torch.empty_strided(v.shape, v.stride(), dtype=dtype, device="cuda").copy_(v)
        if v.stride(0) == 0:
            gpu = v[:1, :1].cuda().expand(B, S, H, dh)
        assert_turned(ops.rotary(gpu, cos.cuda(), sin.cuda(), layout=layout), *turn(v, c, s, layout))
    # in place: the neighbours of the view stay as they were
    z = big.cuda()
    w = z[:, 1:S + 1, 2:H + 2, 1:dh + 1]
    ops.rotary_(w, cos.cuda(), sin.cuda(), layout=layout)
    assert_turned(w, *turn(big[:, 1:S + 1, 2:H + 2, 1:dh + 1], c, s, layout))
    w.copy_(big[:, 1:S + 1, 2:H + 2, 1:dh + 1].cuda())
    assert torch.equal(z.cpu(), big)
    # a broadcast leaf collects the gradients of its copies; an expanded incoming gradient is read as it is
    leaf = torch.randn(1, 1, H, dh, generator=g).cuda().requires_grad_()
    y = ops.rotary(leaf.expand(B, S, H, dh), cos.cuda(), sin.cuda(), layout=layout)
    y.sum().backward()
    want, size = turn(torch.ones(1, S, H, dh), c, -s, layout)
    err = (leaf.grad.double().cpu() - B * want.sum(1, keepdim=True)).abs().max()
    assert float(err) <= 4 * B * S * 2.0 ** -24 * B * float(size.sum(1).max())


def test_rotary_clamps_positions_and_takes_empty_batches():
    from musicgeneration_amd import ops
    cos, sin = _tables(5, 8)
    x = torch.randn(1, 4, 2, 8)
    pos = torch.tensor([[-3, 4, 5, 2 ** 40]])
    y = ops.rotary(x.cuda(), cos.cuda(), sin.cuda(), pos.cuda())
    at = pos.clamp(0, 4)
    assert_turned(y, *turn(x, cos[at][:, :, None], sin[at][:, :, None], "interleaved"))
    for shape in ((0, 4, 2, 8), (1, 0, 2, 8), (1, 4, 0, 8)):
        e = torch.empty(shape, device="cuda").requires_grad_()
        z = ops.rotary(e, cos.cuda(), sin.cuda())
        assert z.shape == shape
        z.sum().backward()
        assert e.grad.shape == shape


@pytest.mark.parametrize("kw", [{}, {"scaling": "linear", "factor": 8.0}, {"scaling": "ntk", "factor": 4.0},
                                {"scaling": "by_parts", "factor": 16.0, "original": 2048}, {"base": 500000.0}])
def test_rope_tables_are_those_of_64_bits_far_out(kw):
    from musicgeneration_amd import ops
    n, rd = 131072, 64
    cos, sin = ops.rope_tables(n, rd, **kw)
    base, f = kw.get("base", 10000.0), kw.get("factor", 1.0)
    i = torch.arange(rd // 2, dtype=torch.float64)
    if kw.get("scaling") == "ntk":
        base = base * f ** (rd / (rd - 2))
    theta, m = base ** (-2 * i / rd), 1.0
    if kw.get("scaling") == "linear":
        theta = theta / f
    if kw.get("scaling") == "by_parts":
        turns = kw["original"] * theta / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        theta, m = theta * (keep + (1 - keep) / f), 1 + 0.1 * math.log(f)
    angle = torch.arange(n, dtype=torch.float64)[:, None] * theta
    for got, want in ((cos, m * angle.cos()), (sin, m * angle.sin())):
        # one rounding to fp32, and the fp64 angle itself: 131072 * a few 2^-53 relative
        bound = 2.0 ** -24 * want.abs() + 131072 * 2.0 ** -50
        assert got.shape == (n, rd // 2) and float(((got.double().cpu() - want).abs() - bound).max()) <= 0


def test_rotary_in_a_graph_and_on_a_side_stream():
    from musicgeneration_amd import ops
    cos, sin = ops.rope_tables(64, 32)
    x = torch.randn(2, 9, 4, 64, device="cuda").bfloat16()
    pos = torch.randint(0, 64, (2, 9), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = ops.rotary(x, cos, sin, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rotary(x, cos, sin, pos)
    for step in range(3):
        x.copy_(torch.randn_like(x))
        pos.copy_((pos + 7) % 64)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, ops.rotary(x, cos, sin, pos)), step
    assert want.shape == x.shape


def test_rotary_gradient_beside_an_eager_graph_of_the_same_leaf():
    from musicgeneration_amd import ops
    cos, sin = ops.rope_tables(64, 64)
    x = torch.randn(1, 8, 2, 64, device="cuda").requires_grad_()
    dy = torch.randn_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.rotary(x, cos, sin), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, = torch.autograd.grad(ops.rotary(x, cos, sin), x, dy)
    for _ in range(3):
        dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, torch.autograd.grad(ops.rotary(x, cos, sin), x, dy)[0])
