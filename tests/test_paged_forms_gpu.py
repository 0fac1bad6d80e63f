"""Every form of paged_attn's kernel (private and shared tiles, prefix taken apart or not, ranges split or whole) against the 64-bit
loop, at sizes of which tests/test_paged_plan_cpu.py asserts that they reach it."""
import math

import pytest
import torch

from paged_sizes import ALL, BF16, F32, NAMES, NEIGHBOURS, PROMPTS, rows_of_sequences
from serving_oracle import assert_attended, attend
from test_paged_gpu import _pool

pytestmark = pytest.mark.gpu
SPARE = 3
NAN = float("nan")


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


def _bits(x):
    """x as whole numbers: equal bit for bit, NaN too."""
    return x.view(torch.int16 if x.dtype is BF16 else torch.int32)


@pytest.mark.parametrize("dtype,dh", list(NEIGHBOURS))
@pytest.mark.parametrize("size", PROMPTS, ids=str)
def test_prompts_see_no_value_behind_their_row(dtype, dh, size):
    """Infinities and NaN in the v (and NaN in the k) of rows of the same prompt, in the first, a middle and the last tile and in several
    at once: earlier rows stay the same, bit for bit; later ones are not finite in the v's channel alone, or anywhere where k is bad."""
    B, R, Hq, Hkv, longest = size
    case = (dtype, dh, 0, 0, 0, B, R, Hq, Hkv, 0, longest)
    q, k, v, table, lens, _, prefix = _inputs(case, False, seed=dh + B, size=4.0)
    clean = _call(case, q, k, v, table, lens, None, prefix).cpu()
    others = [d for d in range(dh) if d != 5]
    for rows, bad, in_k in (((0,), NAN, False), ((R // 2,), math.inf, False), ((R - 1,), -math.inf, False), ((3, R // 2, R - 2), math.inf, False),
                            ((1,), NAN, True), ((R // 2 + 1, R - 1), NAN, True)):
        k2, v2 = k.clone(), v.clone()
        for b, n in enumerate(lens):
            for row in rows:
                j = n - R + row
                (k2 if in_k else v2)[table[b, j // 16], :, j % 16, 5] = bad
        got = _call(case, q, k2, v2, table, lens, None, prefix).cpu()
        first = rows[0]
        assert torch.equal(_bits(got[:, :first]), _bits(clean[:, :first])), (rows, bad, in_k)
        if in_k:
            assert torch.isnan(got[:, first:]).all(), (rows, bad)
        else:
            assert not torch.isfinite(got[:, first:, :, 5].float()).any(), (rows, bad)
            assert torch.equal(_bits(got[..., others]), _bits(clean[..., others])), (rows, bad)


def _rows_stay_alone(case, seed):
    dtype, dh, B, R = case[0], case[1], case[5], case[6]
    q, k, v, table, lens, _, prefix = _inputs(case, False, seed=seed, size=4.0)
    clean = _call(case, q, k, v, table, lens, None, prefix)
    q[1], q[B - 1, 0] = NAN, math.inf
    got = _call(case, q, k, v, table, lens, None, prefix)
    stay = torch.ones(B, R, dtype=torch.bool)
    stay[1], stay[B - 1, 0] = False, False
    stay = stay.cuda()
    assert torch.equal(_bits(got[stay]), _bits(clean[stay]))
    assert not torch.isfinite(got[~stay].float()).any()


@pytest.mark.parametrize("case", [(*at, 1, 0, 0, *size) for at, sizes in NEIGHBOURS.items() for size in sizes], ids=str)
def test_a_row_that_is_not_a_number_leaves_its_neighbours_in_a_tile_alone(case):
    """The tiles of a prefix hold rows of many sequences (a padded batch: some are NaN or infinite): the others stay the same, bit for
    bit, over many tiles of keys, where the running maxima move."""
    _rows_stay_alone(case, 7)


@pytest.mark.parametrize("dtype,dh", list(NEIGHBOURS))
@pytest.mark.parametrize("size", PROMPTS, ids=str)
def test_a_row_of_a_prompt_that_is_not_a_number_leaves_the_others_alone(dtype, dh, size):
    _rows_stay_alone((dtype, dh, 0, 0, 0, *size[:4], 0, size[4]), 8)


PRIVATE = [c for c in ALL if c[0] is BF16 and (c[3] in (0, 1) or not c[2]) and c[4] in (0, 1, 4)]


@pytest.mark.parametrize("case", PRIVATE, ids=str)
def test_private_tiles_keep_the_weights_precise(case):
    """bf16 calls of few rows: the weights enter the product with V as a bf16 value and the bf16 rounding of what it leaves, which is at
    most 2^-7 of it: off by 2^-8 x 2^-7 (and the 2^-24 that the remainder is raised by), where `attend` allows two roundings of 2^-8."""
    q, k, v, table, lens, cu, prefix = _inputs(case, False, seed=3)
    args = (table, lens, None, cu, prefix if case[9] else None, case[9])
    want, bound = attend(q, k, v, *args)
    weighed, _ = attend(q, k, v.abs(), *args)             # sum_j p_j |v_j|
    got = _call(case, q, k, v, table, lens, cu, prefix)
    assert_attended(got, want, bound - (2 * 2.0 ** -8 - 2.0 ** -15 - 2.0 ** -23) * weighed)


@pytest.mark.parametrize("dtype,dh", list(NEIGHBOURS))
@pytest.mark.parametrize("B,R", [(3, 1), (2, 20), (2, 150)])
def test_infinite_values_come_out_infinite(dtype, dh, B, R):
    """out = sum_j p_j v_j, p_j > 0: where a row sees one infinite v, wherever in a tile it lies, that is the result; where it sees
    infinities of both signs or a NaN, NaN.  (Weights far from underflow: |scores| < 10.)"""
    from musicgeneration_amd import ops
    n, page = 330, 16
    k, v, table, _, g = _pool([n] * B, 1, page, dh, dtype, seed=dh)
    q = torch.randn(B, R, 2, dh, generator=g).to(dtype)
    last = n - R                                          # own index of the first row
    keys = {1: (0, math.inf), 2: (last, -math.inf), 3: (n - 1, math.inf), 4: (last - 40, math.inf), 6: (last + R // 2, NAN)}
    for channel, (j, bad) in keys.items():
        for b in range(B):
            v[table[b, j // page], :, j % page, channel] = bad
    for b in range(B):                                    # channel 7: both signs, the second from row R / 2 on
        v[table[b, 2 // page], :, 2 % page, 7] = math.inf
        j = last + R // 2
        v[table[b, j // page], :, j % page, 7] = -math.inf
    got = ops.paged_attn(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.full((B,), n, dtype=torch.int32).cuda()).float().cpu()
    sees = torch.arange(R)[None, :, None].expand(B, R, 2) + last      # last key of a row
    for channel, (j, bad) in keys.items():
        x, seen = got[..., channel], sees >= j
        assert torch.isfinite(x[~seen]).all(), channel
        assert torch.isnan(x[seen]).all() if bad != bad else (x[seen] == bad).all(), channel
    both = sees >= last + R // 2
    assert torch.isnan(got[..., 7][both]).all() and (got[..., 7][~both] == math.inf).all()
    assert torch.isfinite(got[..., [0, 5]]).all()
