"""How mgx_paged_attn takes a call apart (mgx_paged_attn_plan, host only): the sizes that the GPU tests of the kernel's forms use do
reach those forms."""
import ctypes

import pytest

from paged_sizes import ALL, BF16, F32, NAMES, NEIGHBOURS, PROMPTS, SIZES, plan, plan_of_case

# every form the launcher has an instance of: (dtype, dh) -> {(share, tiles of prefix items, of own items)}
FORMS = {
    (F32, 64): {(0, 0, 0), (0, 1, 1), (0, 2, 2), (0, 0, 4), (1, 0, 0), (1, 1, 1), (1, 2, 0), (1, 2, 1), (1, 2, 2)},
    (F32, 128): {(0, 0, 0), (0, 1, 1), (0, 2, 2), (1, 0, 0), (1, 1, 1), (1, 2, 0), (1, 2, 1), (1, 2, 2)},
    (F32, 256): {(0, 0, 0), (1, 0, 0)},
    (BF16, 64): {(0, 0, 0), (0, 1, 1), (0, 2, 2), (0, 3, 3), (0, 0, 4), (1, 0, 0), (1, 1, 1), (1, 2, 0), (1, 2, 1), (1, 2, 2), (1, 3, 0),
                 (1, 3, 1), (1, 3, 3)},
    (BF16, 128): {(0, 0, 0), (0, 1, 1), (0, 2, 2), (0, 0, 4), (1, 0, 0), (1, 1, 1), (1, 2, 0), (1, 2, 1), (1, 2, 2)},
    (BF16, 256): {(0, 0, 0), (0, 2, 2), (1, 0, 0)},
}


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", ALL, ids=NAMES)
def test_sizes_reach_their_form(case, ragged):
    p = plan_of_case(case, ragged)
    assert (p["share"], p["body_p"] if p["share"] else case[3], p["body_o"]) == case[2:5], p


def test_every_form_is_reached_with_whole_and_split_ranges():
    assert {(k, f[2:]) for k in FORMS for f in SIZES if f[:2] == k} == {(k, f) for k, fs in FORMS.items() for f in fs}
    plans = [(c, plan_of_case(c, False)) for c in ALL]
    for dtype in (F32, BF16):
        for tiles in (0, 1, 2, 3, 4):
            own = [p for c, p in plans if c[0] is dtype and p["body_o"] == tiles]
            if own:
                assert {p["So"] > 1 for p in own} == {False, True}, (dtype, tiles)
        # prefix parts of one tile and of several
        assert any(p["share"] and p["chunk_p"] == 64 for c, p in plans if c[0] is dtype)
        assert any(p["share"] and p["body_p"] >= 2 and p["chunk_p"] > 64 for c, p in plans if c[0] is dtype)
    assert any(p["share"] and p["body_p"] == 2 and p["chunk_p"] >= 512 for c, p in plans) and any(p["share"] and p["body_p"] == 3 and p["chunk_p"] >= 512 for c, p in plans)


def test_prompts_and_neighbours_fill_tiles():
    own, prefix = {}, {}
    for at, sizes in NEIGHBOURS.items():
        for B, R, Hq, Hkv, longest in PROMPTS:
            p = plan(B * R, B, Hq, Hkv, at[1], 0, R, longest, at[0])
            own.setdefault((*at, p["body_o"]), set()).add(p["So"] > 1)
        for B, R, Hq, Hkv, P, longest in sizes:
            p = plan(B * R, B, Hq, Hkv, at[1], P, R, longest, at[0])
            assert p["share"] and p["chunk_p"] >= 192, (at, B, R, p)
            prefix.setdefault(at, set()).add((p["body_p"], p["body_o"]))
    # shared tiles of every kind, with whole and with split ranges
    assert all(own[at] == {False, True} for at in ((F32, 64, 2), (F32, 128, 2), (BF16, 128, 2), (BF16, 64, 3), (BF16, 256, 2))), own
    assert (BF16, 64, 2) in own and (F32, 256, 0) in own
    assert prefix == {(F32, 64): {(2, 0), (2, 1), (2, 2)}, (F32, 128): {(2, 0), (2, 2)}, (F32, 256): {(0, 0)}, (BF16, 64): {(2, 0), (3, 0), (3, 1), (3, 3)},
                      (BF16, 128): {(2, 0), (2, 1), (2, 2)}, (BF16, 256): {(0, 0)}}


def test_plan_refuses():
    from musicgeneration_amd._lib import lib
    out = (ctypes.c_int * 7)()
    ok = (4, 4, 2, 1, 64, 0, 1, 8, 1)
    assert lib.mgx_paged_attn_plan(*ok, out) == 0 and lib.mgx_paged_attn_plan(*ok, None) < 0
    for at, bad in ((0, 0), (1, 0), (2, 0), (2, 3), (3, 0), (4, 0), (4, 264), (5, -1), (6, 0), (7, 0), (8, 2)):
        args = list(ok)
        args[at] = bad
        if at == 2 and bad == 3:
            args[3] = 2
        assert lib.mgx_paged_attn_plan(*args, out) < 0, args
