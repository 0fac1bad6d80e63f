"""Every form of paged_attn's kernel (private and shared tiles, prefix taken apart or not, ranges split or whole) against the 64-bit
loop, at sizes of which tests/test_paged_plan_cpu.py asserts that they reach it."""
import pytest
import torch

from paged_sizes import ALL, NAMES, rows_of_sequences
from serving_oracle import assert_attended, attend
from test_paged_gpu import _pool

pytestmark = pytest.mark.gpu
SPARE = 3


def _inputs(case, ragged, seed=0, size=1.0):
    """q, caches, page table, prefix pages, lengths, offsets of one call; lengths spread up to the announced one."""
    dtype, dh, _, _, _, B, R, Hq, Hkv, P, longest = case
    ns = rows_of_sequences(B, R, ragged)
    g = torch.Generator().manual_seed(seed)
    past = torch.randint(0, longest - R + 1, (B,), generator=g).tolist()
    past[0] = longest - R
    lens = [n + p for n, p in zip(ns, past)]
    k, v, table, prefix, g = _pool(lens, Hkv, 16, dh, dtype, P, seed=seed + 1)
    cu = [0]
    for n in ns:
        cu.append(cu[-1] + n)
    q = size * torch.randn(*((cu[-1] + SPARE,) if ragged else (B, R)), Hq, dh, generator=g)
    return q.to(dtype), k, v, table, lens, cu if ragged else None, prefix


def _call(case, q, k, v, table, lens, cu, prefix, slopes=None):
    from musicgeneration_amd import ops
    return ops.paged_attn(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                          slopes=None if slopes is None else slopes.cuda(), cu_rows=None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda(),
                          max_rows=case[6], max_len=case[10], prefix=prefix.cuda() if case[9] else None, prefix_len=case[9])


def _slopes(Hq):
    return 2.0 ** (-8.0 * torch.arange(1, Hq + 1) / Hq)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", ALL, ids=NAMES)
def test_every_form(case, ragged):
    """Without slopes, and with them: forms of their own of the shared tiles."""
    q, k, v, table, lens, cu, prefix = _inputs(case, ragged, seed=sum(case[5:]))
    for slopes in (None, _slopes(case[7])):
        got = _call(case, q, k, v, table, lens, cu, prefix, slopes)
        want, bound = attend(q, k, v, table, lens, slopes, cu, prefix if case[9] else None, case[9])
        assert_attended(got, want, bound)
        if ragged:
            assert not got[cu[-1]:].any()
