"""Forward-mode derivatives and version counters of the rotary and serving operators on the GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from serving_oracle import assert_turned, turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("on_graph", [False, True])
def test_rotary_tangent_is_the_turned_tangent(dtype, layout, on_graph):
    from musicgeneration_amd import ops
    g = torch.Generator().manual_seed(5)
    cos, sin = ops.rope_tables(20, 32)
    pos = torch.randint(0, 20, (2, 7), generator=g)
    c, s = cos.cpu()[pos][:, :, None], sin.cpu()[pos][:, :, None]
    x, t, dy = (torch.randn(2, 7, 3, 64, generator=g).to(dtype) for _ in range(3))
    with fwd.dual_level():
        leaf = x.cuda().requires_grad_(on_graph)
        # (a tangent whose head dim is not dense)
        tangent = t.cuda().transpose(2, 3).contiguous().transpose(2, 3)
        y, dx = fwd.unpack_dual(ops.rotary(fwd.make_dual(leaf, tangent), cos, sin, pos.cuda(), layout))
        assert_turned(y.detach(), *turn(x, c, s, layout))
        assert_turned(dx.detach(), *turn(t, c, s, layout))
        if on_graph:
            assert_turned(torch.autograd.grad(y, leaf, dy.cuda())[0], *turn(dy, c, -s, layout))
    # the gradient's tangent is the turned-back tangent of the incoming gradient
    leaf = x.cuda().requires_grad_()
    y = ops.rotary(leaf, cos, sin, pos.cuda(), layout)
    with fwd.dual_level():
        grad, tangent = fwd.unpack_dual(torch.autograd.grad(y, leaf, fwd.make_dual(dy.cuda(), t.cuda()))[0])
        assert_turned(grad, *turn(dy, c, -s, layout))
        assert_turned(tangent, *turn(t, c, -s, layout))


def test_rotary_tangent_is_that_of_differences():
    from musicgeneration_amd import ops
    cos, sin = ops.rope_tables(6, 8)
    x = torch.randn(2, 3, 2, 12, generator=torch.Generator().manual_seed(4)).cuda().requires_grad_()
    # fp32 rounding 2^-24 of values below 8 over a step of 2^-4: 2 * 8 * 2^-24 / 2^-4 < 2^-15, sums of 2 values
    assert torch.autograd.gradcheck(lambda z: ops.rotary(z, cos, sin), (x,), eps=2.0 ** -4, atol=2.0 ** -13, rtol=0, nondet_tol=0.0,
                                    check_forward_ad=True)


def test_dispatched_operators_refuse_tangents():
    from musicgeneration_amd import ops, torch_ops  # noqa: F401
    cos, sin = ops.rope_tables(8, 8)
    x = torch.randn(1, 4, 2, 8, device="cuda")
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            torch.ops.mgx.rotary(fwd.make_dual(x, x), cos, sin)
        p = torch.rand(1, 3, 9, device="cuda")
        with pytest.raises(RuntimeError, match="tangent"):
            torch.ops.mgx.verify_draft(fwd.make_dual(p, p), torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.rand(1, 3, device="cuda"))


def test_a_backward_that_saved_what_was_written_over_raises():
    from musicgeneration_amd import ops
    cos, sin = ops.rope_tables(40, 64)
    w = torch.randn(64, device="cuda").requires_grad_()
    x = torch.randn(1, 4, 2, 64, device="cuda")
    z = w * x
    ops.rotary_(x, cos, sin)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    kc, vc = (torch.zeros(3, 2, 16, 64, device="cuda") for _ in range(2))
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
    for which in (kc, vc):
        z = w * which
        ops.paged_append(torch.randn(1, 4, 6 * 64, device="cuda"), kc, vc, table, lens, 2, cos, sin)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
    # tensors made in inference mode have no counter
    with torch.inference_mode():
        y = torch.randn(1, 4, 2, 64, device="cuda")
        want = ops.rotary(y, cos, sin)
        assert torch.equal(ops.rotary_(y, cos, sin), want)
