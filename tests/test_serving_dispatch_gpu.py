"""torch.ops.mgx.{rotary, paged_append, paged_attention, verify_draft}: schema, fake kernel and autograd registration pass
torch.library.opcheck; results and gradients are those of the wrappers."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache():
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(9, 2, 16, 64, generator=g).bfloat16().cuda() for _ in range(2))
    table = torch.randperm(9, generator=g)[:6].int().view(2, 3).cuda()
    return k, v, table, torch.tensor([20, 33], dtype=torch.int32).cuda()


def test_rotary_dispatch():
    from musicgeneration_amd import ops, torch_ops  # noqa: F401
    cos, sin = ops.rope_tables(32, 32)
    x = torch.randn(2, 5, 3, 64).cuda()
    pos = torch.randint(0, 32, (2, 5)).cuda()
    torch.library.opcheck(torch.ops.mgx.rotary.default, (x.requires_grad_(), cos, sin, pos, "half"),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    dy = torch.randn_like(x)
    want = ops.rotary(x, cos, sin, pos, "half")
    got = torch.ops.mgx.rotary(x, cos, sin, pos, "half")
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got, x, dy)[0], torch.autograd.grad(want, x, dy)[0])
    # linear in x: the gradient's gradient is the rotation again
    z = dy.clone().requires_grad_()
    dx, = torch.autograd.grad(ops.rotary(x, cos, sin, pos, "half"), x, z, create_graph=True)
    assert torch.equal(torch.autograd.grad(dx, z, x.detach())[0], want.detach())


@pytest.mark.parametrize("rotated", [True, False])
def test_paged_dispatch(rotated):
    from musicgeneration_amd import ops, torch_ops  # noqa: F401
    k, v, table, lens = _cache()
    cos, sin = ops.rope_tables(64, 64) if rotated else (None, None)
    qkv = torch.randn(2, 3, (4 + 2 * 2) * 64).bfloat16().cuda()
    args = (qkv, k, v, table, lens, 4, cos, sin)
    torch.library.opcheck(torch.ops.mgx.paged_append.default, args, test_utils=("test_schema", "test_faketensor"))
    k2, v2 = k.clone(), v.clone()
    q = torch.ops.mgx.paged_append(*args)
    assert torch.equal(q, ops.paged_append(qkv, k2, v2, table, lens, 4, cos, sin))
    assert torch.equal(k, k2) and torch.equal(v, v2)
    torch.library.opcheck(torch.ops.mgx.paged_attention.default, (q, k, v, table, lens), test_utils=("test_schema", "test_faketensor"))
    assert torch.equal(torch.ops.mgx.paged_attention(q, k, v, table, lens), ops.paged_attn(q, k, v, table, lens))


def test_verify_dispatch():
    from musicgeneration_amd import ops, torch_ops  # noqa: F401
    p, d = torch.rand(3, 4, 50).softmax(-1).cuda(), torch.rand(3, 3, 50).softmax(-1).cuda()
    x, u = torch.randint(0, 50, (3, 3)).cuda(), torch.rand(3, 4).cuda()
    torch.library.opcheck(torch.ops.mgx.verify_draft.default, (p, x, u, d), test_utils=("test_schema", "test_faketensor"))
    for a, b in zip(torch.ops.mgx.verify_draft(p, x, u, d), ops.verify_draft(p, x, u, d)):
        assert torch.equal(a, b)
