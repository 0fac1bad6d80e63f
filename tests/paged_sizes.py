"""Sizes of paged_attn calls that reach every form of its kernel, and what mgx_paged_attn_plan has to say of each.

SIZES: (dtype, dh, share, tiles of prefix items, of own items) -> [(sequences, rows, Hq, Hkv, prefix, longest own length)]; share 0: no
prefix items.  The tiles are those of mgx_paged_attn_plan: 0 / 1 / 4 private, 2 / 3 shared by a workgroup's waves."""
import ctypes

import torch

F32, BF16 = torch.float32, torch.bfloat16

SIZES = {
    (F32, 64, 0, 0, 0): [(24, 1, 4, 4, 0, 601)], (F32, 64, 0, 1, 1): [(1, 6, 4, 1, 0, 6), (1, 6, 4, 1, 100, 106)],
    (F32, 64, 0, 2, 2): [(1, 6, 8, 1, 0, 6), (2, 40, 4, 1, 0, 300)], (F32, 64, 0, 0, 4): [(1, 1, 1, 1, 0, 601), (24, 1, 8, 8, 0, 1)],
    (F32, 64, 1, 0, 0): [(16, 1, 8, 8, 100, 1501), (2, 1, 8, 8, 4100, 1), (6, 1, 8, 8, 1003, 601)], (F32, 64, 1, 1, 1): [(24, 1, 4, 4, 517, 601)],
    (F32, 64, 1, 2, 0): [(100, 1, 8, 8, 100, 601), (48, 1, 2, 2, 100, 601)], (F32, 64, 1, 2, 1): [(6, 6, 32, 8, 100, 1506)],
    (F32, 64, 1, 2, 2): [(3, 33, 8, 8, 100, 633), (24, 33, 4, 4, 100, 33)],
    (F32, 128, 0, 0, 0): [(1, 1, 1, 1, 100, 101)], (F32, 128, 0, 1, 1): [(1, 6, 4, 1, 100, 106)], (F32, 128, 0, 2, 2): [(1, 6, 8, 1, 0, 106), (2, 40, 4, 1, 0, 300)],
    (F32, 128, 1, 0, 0): [(2, 1, 1, 1, 517, 601)], (F32, 128, 1, 1, 1): [(6, 1, 3, 1, 100, 101), (6, 1, 4, 1, 1003, 601)],
    (F32, 128, 1, 2, 0): [(48, 1, 4, 4, 100, 1501), (48, 1, 2, 2, 100, 601)], (F32, 128, 1, 2, 1): [(6, 6, 32, 8, 100, 1506)],
    (F32, 128, 1, 2, 2): [(3, 6, 32, 4, 100, 606), (6, 33, 8, 8, 100, 33)],
    (F32, 256, 0, 0, 0): [(1, 6, 2, 1, 100, 101)], (F32, 256, 1, 0, 0): [(2, 1, 2, 1, 517, 601), (48, 1, 8, 8, 517, 1501)],
    (BF16, 64, 0, 0, 0): [(6, 1, 16, 2, 2050, 601)], (BF16, 64, 0, 1, 1): [(1, 6, 4, 1, 0, 606), (1, 6, 4, 1, 0, 6)],
    (BF16, 64, 0, 2, 2): [(1, 6, 8, 1, 0, 606), (2, 60, 2, 1, 0, 60)], (BF16, 64, 0, 3, 3): [(1, 33, 8, 1, 0, 33), (1, 300, 2, 1, 100, 400)],
    (BF16, 64, 0, 0, 4): [(1, 1, 1, 1, 100, 101), (1, 1, 1, 1, 517, 601)],
    (BF16, 64, 1, 0, 0): [(2, 1, 8, 8, 1003, 1501), (16, 1, 8, 8, 100, 1501)], (BF16, 64, 1, 1, 1): [(16, 1, 4, 2, 517, 601), (24, 1, 4, 4, 100, 1501)],
    (BF16, 64, 1, 2, 0): [(24, 1, 4, 2, 517, 601), (64, 1, 8, 8, 517, 1501)], (BF16, 64, 1, 2, 1): [(2, 6, 8, 2, 100, 1506)],
    (BF16, 64, 1, 2, 2): [(3, 6, 16, 2, 100, 606), (2, 33, 8, 8, 1003, 33)], (BF16, 64, 1, 3, 0): [(150, 1, 8, 4, 1003, 1501), (150, 1, 16, 8, 100, 101)],
    (BF16, 64, 1, 3, 1): [(24, 6, 12, 4, 100, 606), (48, 6, 32, 8, 517, 606)], (BF16, 64, 1, 3, 3): [(3, 33, 6, 2, 1003, 1533)],
    (BF16, 128, 0, 0, 0): [(6, 1, 8, 8, 0, 601)], (BF16, 128, 0, 1, 1): [(1, 6, 4, 1, 0, 606), (1, 6, 4, 1, 0, 6)],
    (BF16, 128, 0, 2, 2): [(1, 6, 8, 1, 100, 106), (2, 300, 2, 1, 0, 300)], (BF16, 128, 0, 0, 4): [(1, 1, 1, 1, 100, 101), (1, 1, 1, 1, 0, 601)],
    (BF16, 128, 1, 0, 0): [(2, 1, 8, 8, 1003, 1501), (6, 1, 8, 8, 100, 601)], (BF16, 128, 1, 1, 1): [(16, 1, 4, 2, 517, 601), (24, 1, 2, 2, 100, 601)],
    (BF16, 128, 1, 2, 0): [(24, 1, 4, 2, 100, 601), (100, 1, 8, 8, 100, 601)], (BF16, 128, 1, 2, 1): [(2, 6, 4, 1, 100, 606), (16, 6, 32, 8, 100, 1506)],
    (BF16, 128, 1, 2, 2): [(2, 6, 8, 1, 100, 1506), (16, 33, 16, 8, 100, 633)],
    (BF16, 256, 0, 0, 0): [(1, 6, 2, 1, 100, 101)], (BF16, 256, 0, 2, 2): [(1, 33, 8, 1, 0, 33), (1, 200, 2, 1, 100, 300)],
    (BF16, 256, 1, 0, 0): [(2, 1, 2, 1, 517, 601), (24, 1, 8, 8, 517, 1501)],
}
ALL = [(*form, *size) for form, sizes in SIZES.items() for size in sizes]
NAMES = ["%s-%d-%d%d%d-%dx%d-%d+%d-P%d-%d" % (str(c[0])[6:], *c[1:]) for c in ALL]


def rows_of_sequences(B, R, ragged):
    """Rows of each sequence: R of each, or R and fewer (none among them) in turn."""
    return [(R, R // 2, R)[b % 3] for b in range(B)] if ragged else [R] * B


def plan(T, B, Hq, Hkv, dh, P, max_rows, max_len, dtype):
    """{share, prefix tiles, own tiles, prefix parts, own parts, prefix keys a part, own keys a part}"""
    from musicgeneration_amd._lib import lib
    got = (ctypes.c_int * 7)()
    assert lib.mgx_paged_attn_plan(T, B, Hq, Hkv, dh, P, max_rows, max_len, 0 if dtype is F32 else 1, got) == 0
    return dict(zip(("share", "body_p", "body_o", "Sp", "So", "chunk_p", "chunk_o"), got))


def plan_of_case(case, ragged, spare=3):
    dtype, dh, _, _, _, B, R, Hq, Hkv, P, longest = case
    T = sum(rows_of_sequences(B, R, ragged)) + (spare if ragged else 0)
    return plan(T, B, Hq, Hkv, dh, P, R, longest, dtype)


# (sequences, rows, Hq, Hkv, longest own length): prompts whose rows fill several tiles, over several tiles of keys
PROMPTS = [(2, 150, 2, 1, 400), (40, 130, 2, 1, 300), (60, 130, 2, 2, 400)]
# (dtype, dh) -> [(sequences, rows, Hq, Hkv, prefix, longest own length)]: prefix items of many sequences' rows, several tiles of keys each
NEIGHBOURS = {(dtype, dh): [(64, 1, 8, 8, 2050, 700), (150, 1, 8, 4, 2050, 700), (30, 33, 8, 8, 2050, 133)] for dtype in (F32, BF16) for dh in (64, 128, 256)}
for _at in ((F32, 64), (BF16, 64), (BF16, 128), (F32, 256)):
    NEIGHBOURS[_at].append((48, 6, 16, 4, 2050, 106))
