"""Edges of the serving operators' arguments on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rotated", [False, True])
def test_ragged_rows_of_no_sequence(rotated):
    """No sequence is left, the rows of a padded batch are: q zero where it is rotated, outputs zero, the cache as it was."""
    from musicgeneration_amd import ops
    kc, vc = (torch.randn(3, 2, 16, 64, device="cuda").bfloat16() for _ in range(2))
    k, v = kc.clone(), vc.clone()
    table, lens, cu = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((0, 2), (0,), (1,)))
    cos, sin = ops.rope_tables(8, 64) if rotated else (None, None)
    qkv = torch.randn(5, 8 * 64, device="cuda").bfloat16()
    q = ops.paged_append(qkv, kc, vc, table, lens, 4, cos, sin, cu_rows=cu)
    assert torch.equal(q, torch.zeros_like(q) if rotated else qkv[:, :256].view(5, 4, 64))
    out = ops.paged_attn(q, kc, vc, table, lens, cu_rows=cu)
    assert out.shape == (5, 4, 64) and not out.any()
    assert torch.equal(kc, k) and torch.equal(vc, v)
