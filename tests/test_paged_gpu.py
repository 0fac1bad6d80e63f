"""Paged cache: paged_append and paged_attn against the 64-bit loops of serving_oracle, and a serving run of them together."""
import math

import pytest
import torch

from serving_oracle import append, assert_attended, assert_turned, attend, turn, verify

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NAN = float("nan")


def _tables(n, rd):
    a = torch.arange(n).double()[:, None] * 10000.0 ** (-torch.arange(0, rd, 2).double() / rd)
    return a.cos().float(), a.sin().float()


def _pool(lens, Hkv, page, dh, dtype, P=0, spare=2, seed=0, wide=1):
    """Caches whose every slot that no key occupies holds NaN; tables whose unused entries lie outside the pool."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    shared = -(-P // page)
    ids = torch.randperm(sum(need) + shared + spare, generator=g).int()
    table = torch.full((len(lens), max(need + [0]) + wide), 2 ** 31 - 1, dtype=torch.int32)
    table[:, -1] = -7
    k, v = (torch.full((ids.numel(), Hkv, page, dh), NAN, dtype=dtype) for _ in range(2))
    at = shared

    def fill(pages, n):
        for i, pg in enumerate(pages):
            m = min(page, n - i * page)
            for c in (k, v):
                c[pg, :, :m] = torch.randn(Hkv, m, dh, generator=g).to(dtype)

    fill(ids[:shared], P)
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        fill(ids[at:at + n], lens[b])
        at += n
    return k, v, table, ids[:shared].clone(), g


def _attend_both(q, k, v, table, lens, slopes=None, cu=None, prefix=None, P=0, scale=None, **hints):
    from musicgeneration_amd import ops
    dev = lambda t: None if t is None else t.cuda()     # noqa: E731
    got = ops.paged_attn(q if q.is_cuda else q.cuda(), dev(k), dev(v), dev(table), torch.tensor(lens, dtype=torch.int32).cuda(),
                         slopes=dev(slopes), cu_rows=None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda(),
                         prefix=dev(prefix), prefix_len=P, scale=scale, **hints)
    assert got.shape == q.shape and got.is_contiguous()
    want, bound = attend(q.cpu(), k, v, table, lens, slopes, cu, prefix, P, scale)
    assert_attended(got, want, bound)
    return got


HEADS = [(1, 1, 64), (8, 8, 64), (6, 2, 128), (12, 1, 32), (5, 1, 80), (4, 2, 256), (2, 2, 8), (3, 1, 200)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Hq,Hkv,dh", HEADS)
@pytest.mark.parametrize("R,page,P", [(1, 16, 0), (3, 32, 45), (6, 64, 130), (1, 1, 7)])
def test_attn_few_rows(dtype, Hq, Hkv, dh, R, page, P):
    lens = [R, R + 1, R + 63, R + 64, 131 + R, R - 1, 0]         # (the last two have rows that see no own key)
    k, v, table, prefix, g = _pool(lens, Hkv, page, dh, dtype, P, seed=Hq * dh + R)
    q = torch.randn(len(lens), R, Hq, dh, generator=g).to(dtype)
    slopes = 2.0 ** (-8.0 * torch.arange(1, Hq + 1) / Hq) if R != 3 else None
    _attend_both(q, k, v, table, lens, slopes, prefix=prefix, P=P)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Hq,Hkv,dh", [(4, 4, 64), (8, 1, 128), (6, 2, 96)])
@pytest.mark.parametrize("P", [0, 77])
def test_attn_ragged_prompts(dtype, Hq, Hkv, dh, P):
    ns, past = [1, 0, 130, 37, 5, 257], [0, 9, 3, 64, 0, 0]
    lens = [n + p for n, p in zip(ns, past)]
    cu = [0]
    for n in ns:
        cu.append(cu[-1] + n)
    k, v, table, prefix, g = _pool(lens, Hkv, 16, dh, dtype, P, seed=dh)
    q = torch.randn(cu[-1] + 6, Hq, dh, generator=g).to(dtype)     # six rows behind the last sequence: zeros
    q[cu[-1]:] = NAN
    got = _attend_both(q, k, v, table, lens, None, cu=cu, prefix=prefix, P=P)
    assert not got[cu[-1]:].any()
    # the hints shape the launch, not the result
    for hints in ({"max_rows": 1, "max_len": 1}, {"max_rows": 100000, "max_len": 10 ** 9}, {"max_rows": 33, "max_len": 70}):
        _attend_both(q, k, v, table, lens, None, cu=cu, prefix=prefix, P=P, **hints)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,R,Hq,Hkv,dh,P,own", [(40, 1, 8, 2, 64, 700, 90), (70, 3, 4, 2, 64, 515, 10), (3, 2, 4, 4, 128, 2100, 1500)])
def test_attn_shared_prefix_of_many_rows(dtype, B, R, Hq, Hkv, dh, P, own):
    g = torch.Generator().manual_seed(B)
    lens = (torch.randint(0, own, (B,), generator=g) + R).tolist()
    k, v, table, prefix, g = _pool(lens, Hkv, 32, dh, dtype, P, seed=B)
    q = torch.randn(B, R, Hq, dh, generator=g).to(dtype)
    _attend_both(q, k, v, table, lens, 2.0 ** (-8.0 * torch.arange(1, Hq + 1) / Hq), prefix=prefix, P=P, max_len=own + R)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attn_large_scores_and_scale(dtype):
    """Scores of +-60 and more that rise and fall along the keys: the running maximum has to move, weights underflow."""
    lens = [300, 129]
    k, v, table, prefix, g = _pool(lens, 2, 16, 64, dtype, 200, seed=8)
    q = 8 * torch.randn(2, 2, 4, 64, generator=g).to(dtype)
    _attend_both(q, k, v, table, lens, prefix=prefix, P=200)
    _attend_both(q, k, v, table, lens, prefix=prefix, P=200, scale=0.02)
    _attend_both(q, k, v, table, lens, prefix=prefix, P=200, scale=-0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attn_pages_outside_the_pool_hide_their_keys(dtype):
    lens = [100, 33]
    k, v, table, prefix, g = _pool(lens, 2, 16, 64, dtype, 70, seed=5)
    table[0, 2], table[0, 4], prefix[1] = -1, k.shape[0], 2 ** 30
    q = torch.randn(2, 4, 4, 64, generator=g).to(dtype)
    _attend_both(q, k, v, table, lens, torch.tensor([0.5, 0.1, 0.0, 2.0]), prefix=prefix, P=70)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dh", [64, 128])
def test_attn_what_a_row_does_not_see_has_no_effect(dtype, dh):
    """Infinities and NaN in the k and v of a later row of the same call: the earlier rows' outputs stay the same, bit for
    bit; the rows that see them are not finite."""
    from musicgeneration_amd import ops
    lens, R = [70, 64, 40], 4
    k, v, table, prefix, g = _pool(lens, 2, 16, dh, dtype, 37, seed=3)
    q = torch.randn(3, R, 4, dh, generator=g).to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    call = lambda kk, vv: ops.paged_attn(q.cuda(), kk.cuda(), vv.cuda(), table.cuda(), lens_t, prefix=prefix.cuda(), prefix_len=37)   # noqa: E731
    clean = call(k, v)
    for bad in (NAN, math.inf, -math.inf):
        for row in range(R):
            k2, v2 = k.clone(), v.clone()
            for b, n in enumerate(lens):
                j = n - R + row
                v2[table[b, j // 16], :, j % 16, 5] = bad
                if bad is NAN:
                    k2[table[b, j // 16], :, j % 16, 1] = bad
            got = call(k2, v2)
            assert torch.equal(got[:, :row], clean[:, :row]), (bad, row)
            assert not torch.isfinite(got[:, row:, :, 5].float()).any(), (bad, row)


def test_attn_q_of_a_packed_projection_and_other_strides():
    lens = [50, 20, 9]
    k, v, table, _, g = _pool(lens, 2, 16, 64, BF16, seed=6)
    packed = torch.randn(3, 2, 4 + 4, 64, generator=g).bfloat16().cuda()
    got = _attend_both(packed[:, :, :4], k, v, table, lens)
    for q in (packed[:, :, :4].contiguous(), packed[:, :, :4].transpose(1, 2).contiguous().transpose(1, 2),
              torch.empty(3 * 2 * 4 * 64 + 1, dtype=BF16, device="cuda")[1:].view(3, 2, 4, 64).copy_(packed[:, :, :4])):
        assert torch.equal(_attend_both(q, k, v, table, lens), got)


def test_attn_replays_in_two_graphs_with_other_lengths():
    """Two captured calls of one shape, replayed in turn with lengths and rows that changed on the device."""
    from musicgeneration_amd import ops
    B, R, Hq, Hkv, dh, P, cap = 5, 2, 4, 2, 64, 300, 900
    k, v, table, prefix, g = _pool([cap] * B, Hkv, 16, dh, BF16, P, seed=11)
    kc, vc, tc, pc = k.cuda(), v.cuda(), table.cuda(), prefix.cuda()
    qs = [torch.randn(B, R, Hq, dh, generator=g).bfloat16().cuda() for _ in range(2)]
    lens = torch.full((B,), R, dtype=torch.int32, device="cuda")
    run = lambda q: ops.paged_attn(q, kc, vc, tc, lens, prefix=pc, prefix_len=P, max_len=cap)     # noqa: E731
    graphs, outs = [], []
    for q in qs:
        run(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(q))
        graphs.append(graph)
    for step in range(4):
        lens.copy_((torch.randint(0, cap - R, (B,), generator=g) + R).int())
        for q in qs:
            q.copy_(torch.randn(q.shape, generator=g).bfloat16())
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for q, out in zip(qs, outs):
            assert torch.equal(out, run(q)), step
            want, bound = attend(q.cpu(), k, v, table, lens.tolist(), None, None, prefix, P)
            assert_attended(out, want, bound)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [7, 48])
def test_attn_one_sequence_and_pages_of_any_size(dtype, page):
    """Nothing to share with a batch of one: prefix and own keys meet inside a tile.  The hints' smallest values."""
    for R, n, P in ((1, 1, 1), (3, 90, 50), (40, 40, 129), (2, 300, 0)):
        k, v, table, prefix, g = _pool([n], 2, page, 64, dtype, P, seed=page + n)
        q = torch.randn(1, R, 4, 64, generator=g).to(dtype)
        _attend_both(q, k, v, table, [n], torch.tensor([1.0, 0.25, 0.0, 0.01]), prefix=prefix, P=P)
        _attend_both(q, k, v, table, [n], prefix=prefix, P=P, max_len=0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dh", [64, 136])
def test_attn_lengths_that_no_table_holds(dtype, dh):
    """Lengths beyond the table and below zero: keys end where the table does, and begin at the first."""
    k, v, table, prefix, g = _pool([48, 48, 48, 48], 2, 16, dh, dtype, 20, seed=dh)
    table = table[:, :3].contiguous()
    q = torch.randn(4, 2, 4, dh, generator=g).to(dtype)
    for lens in ([48, 49, 50, 1000], [0, 1, -1, -50], [2 ** 31 - 1, -2 ** 31, 48, 47]):
        _attend_both(q, k, v, table, lens, prefix=prefix, P=20)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_beyond_the_table_files_nothing(dtype):
    from musicgeneration_amd import ops
    k, v, table, _, g = _pool([48, 48, 48, 48], 2, 16, 64, dtype, seed=4)
    table = table[:, :3].contiguous().cuda()
    qkv = torch.randn(4, 3, 6 * 64, generator=g).to(dtype).cuda()
    kc, vc = k.cuda(), v.cuda()
    ops.paged_append(qkv, kc, vc, table, torch.tensor([51, 2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32).cuda(), 2)
    assert torch.equal(torch.nan_to_num(kc), torch.nan_to_num(k.cuda())) and torch.equal(torch.nan_to_num(vc), torch.nan_to_num(v.cuda()))


def test_pool_past_32_bits():
    """A pool of 6.4 GB a cache: pages at its far end serve as those of a small pool do, bit for bit."""
    from musicgeneration_amd import ops
    n, Hkv, page, dh = 48000, 4, 128, 128
    cos, sin = ops.rope_tables(300, dh)
    qkv = torch.randn(2, 200, (8 + 2 * Hkv) * dh, device="cuda").bfloat16()
    lens = torch.tensor([200, 260], dtype=torch.int32).cuda()
    outs = []
    for pages, first in ((n, n - 6), (6, 0)):
        kc, vc = (torch.empty(pages, Hkv, page, dh, dtype=BF16, device="cuda") for _ in range(2))
        kc[first:].zero_(), vc[first:].zero_()
        table = torch.arange(first, first + 6, dtype=torch.int32).view(2, 3).cuda()
        q = ops.paged_append(qkv, kc, vc, table, lens, 8, cos, sin)
        outs.append((ops.paged_attn(q, kc, vc, table, lens), ops.paged_attn(q[:, :1], kc, vc, table, lens), kc[first:].clone(), vc[first:].clone()))
        del kc, vc
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and outs[0][2].any()


# ---- paged_append -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["interleaved", "half", None])
@pytest.mark.parametrize("Hq,Hkv,dh,rd,page", [(8, 8, 64, 64, 16), (6, 2, 96, 48, 32), (5, 1, 80, 20, 1), (2, 1, 8, 2, 7), (16, 4, 128, 128, 64)])
@pytest.mark.parametrize("ragged", [False, True])
def test_append(dtype, layout, Hq, Hkv, dh, rd, page, ragged):
    from musicgeneration_amd import ops
    if ragged:
        ns, past = [3, 0, 41, 1, 18], [0, 12, 5, 64, 1]
    else:
        ns, past = [5] * 4, [0, 30, 7, -3]             # (the last: rows before the cache's begin are not filed)
    lens = [n + p for n, p in zip(ns, past)]
    cu = [0]
    for n in ns:
        cu.append(cu[-1] + n)
    offset = 19
    k, v, table, _, g = _pool(lens, Hkv, page, dh, dtype, seed=rd + page)
    table[2, 0] = -1                                   # a page outside the pool files nothing
    cos, sin = _tables(max(lens) + offset - 4, rd)     # (the last positions are clamped to the tables' end)
    lead = (cu[-1] + 3,) if ragged else (4, 5)
    qkv = torch.randn(*lead, (Hq + 2 * Hkv) * dh, generator=g).to(dtype)
    if layout is None:
        cos = sin = None
    want_q, want_k, want_v, qs, ks = append(qkv, k, v, table, lens, Hq, cos, sin, layout, cu if ragged else None, offset)
    kc, vc = k.cuda(), v.cuda()
    dev = lambda t: None if t is None else t.cuda()    # noqa: E731
    q = ops.paged_append(qkv.cuda(), kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), Hq, dev(cos), dev(sin),
                         layout=layout or "half", cu_rows=torch.tensor(cu, dtype=torch.int32).cuda() if ragged else None, offset=offset)
    assert q.shape == (*lead, Hq, dh)
    if layout is None:
        assert torch.equal(q.cpu(), qkv[..., :Hq * dh].unflatten(-1, (Hq, dh)))
    else:
        assert_turned(q.reshape(-1, Hq, dh), want_q, qs, "q")
    # v and everything that was not written: exactly; k: to its rounding
    assert torch.equal(torch.nan_to_num(vc.double().cpu(), 9e9), torch.nan_to_num(want_v, 9e9))
    filed = ks > 0 if layout else torch.zeros_like(ks, dtype=torch.bool)
    same = torch.nan_to_num(kc.double().cpu(), 9e9) == torch.nan_to_num(want_k, 9e9)
    assert bool(same[~filed].all())
    if layout:
        got = torch.where(filed, kc.cpu().float(), torch.zeros(())).to(dtype)
        assert_turned(got, torch.where(filed, want_k, torch.zeros((), dtype=torch.float64)), ks, "k")


def test_append_moves_with_the_lengths_in_a_graph():
    from musicgeneration_amd import ops
    B, H, dh, page = 3, 2, 64, 16
    table = torch.randperm(B * 4, generator=torch.Generator().manual_seed(2)).int().view(B, 4)
    cos, sin = _tables(80, dh)
    qkv = torch.randn(B, 2, 3 * H * dh, device="cuda").bfloat16()
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    pools = [torch.zeros(B * 4, H, page, dh, dtype=BF16, device="cuda") for _ in range(4)]
    args = (table.cuda(), lens, H, cos.cuda(), sin.cuda())
    ops.paged_append(qkv, pools[0], pools[1], *args)
    pools[0].zero_(), pools[1].zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens.add_(2)
        q = ops.paged_append(qkv, pools[0], pools[1], *args)
    lens.zero_()
    for step in range(6):
        qkv.copy_(torch.randn_like(qkv))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.paged_append(qkv, pools[2], pools[3], *args)
        assert torch.equal(q, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3]), step
    assert lens.tolist() == [12] * B


# ---- together ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,layout", [(F32, "interleaved"), (BF16, "half")])
def test_serving_run_equals_one_causal_pass(dtype, layout):
    """A primer filed once, then per-sequence prompts of other lengths, then steps of several rows of which some are taken
    back (as rejected drafts are): each row's attention equals the 64-bit causal attention of its whole sequence."""
    from musicgeneration_amd import ops
    B, Hq, Hkv, dh, rd, page, P = 4, 6, 2, 64, 32, 16, 53
    g = torch.Generator().manual_seed(21)
    width = (Hq + 2 * Hkv) * dh
    cos, sin = ops.rope_tables(400, rd, scaling="by_parts", factor=4.0, original=64)
    kc, vc = (torch.full((40, Hkv, page, dh), NAN, dtype=dtype, device="cuda") for _ in range(2))
    ids = torch.randperm(40, generator=g).int()
    prefix, table = ids[:4].cuda(), ids[4:].view(B, 9).contiguous().cuda()
    pages_of_prefix = prefix.view(1, 4)
    history = [[] for _ in range(B)]

    primer = torch.randn(1, P, width, generator=g).to(dtype)
    q = ops.paged_append(primer.cuda(), kc, vc, pages_of_prefix, torch.tensor([P], dtype=torch.int32).cuda(), Hq, cos, sin, layout)
    out = ops.paged_attn(q, kc, vc, pages_of_prefix, torch.tensor([P], dtype=torch.int32).cuda())

    def reference(rows, n):
        """attention of the last n rows of a sequence whose packed rows are `rows` [S, width]: fp64 over the values as the
        cache holds them"""
        S = rows.shape[0]
        x = rows.view(S, -1, dh)
        turned, _ = turn(x[:, :Hq + Hkv], cos.cpu()[:S, None], sin.cpu()[:S, None], layout)
        turned = turned.to(dtype)
        pages = -(-S // page)
        pool = [torch.zeros(pages, Hkv, page, dh, dtype=dtype) for _ in range(2)]
        flat = torch.arange(S)
        pool[0][flat // page, :, flat % page] = turned[:, Hq:]
        pool[1][flat // page, :, flat % page] = x[:, Hq + Hkv:]
        return attend(turned[None, S - n:, :Hq], *pool, torch.arange(pages).int()[None], [S], None, None, None, 0)

    # one step of a rounding more than the bound: the kernel's rotated q and k may differ from the 64-bit ones rounded here
    # in a last bit (a tie), 2 U relative in q and in k, so in a score by 4 U scale sum |q||k| <= 4 U 8 (|q|,|k| < 4.5)
    slack = 2 * 4 * (2.0 ** -8 if dtype == BF16 else 2.0 ** -24) * 8

    def check(got, rows, n):
        want, bound = reference(rows, n)
        assert_attended(got, want, bound + slack * 4.5)

    check(out, primer[0], P)
    ns = [7, 0, 33, 1]
    cu = [0, 7, 7, 40, 41]
    prompts = torch.randn(41, width, generator=g).to(dtype)
    lens = torch.tensor(ns, dtype=torch.int32).cuda()
    cu_t = torch.tensor(cu, dtype=torch.int32).cuda()
    q = ops.paged_append(prompts.cuda(), kc, vc, table, lens, Hq, cos, sin, layout, cu_rows=cu_t, offset=P)
    out = ops.paged_attn(q, kc, vc, table, lens, cu_rows=cu_t, prefix=prefix, prefix_len=P, max_rows=33, max_len=33)
    for b, n in enumerate(ns):
        history[b] = prompts[cu[b]:cu[b + 1]]
        if n:
            check(out[None, cu[b]:cu[b + 1]], torch.cat((primer[0], history[b])), n)
    for step in range(4):
        k = 3
        rows = torch.randn(B, k + 1, width, generator=g).to(dtype)
        lens += k + 1
        q = ops.paged_append(rows.cuda(), kc, vc, table, lens, Hq, cos, sin, layout, offset=P)
        out = ops.paged_attn(q, kc, vc, table, lens, prefix=prefix, prefix_len=P, max_len=144)
        for b in range(B):
            check(out[b:b + 1], torch.cat((primer[0], history[b], rows[b])), k + 1)
        V = 50
        p = torch.randn(B, k + 1, V, generator=g).softmax(-1)
        d = torch.randn(B, k, V, generator=g).softmax(-1)
        x, u = torch.randint(0, V, (B, k), generator=g), torch.rand(B, k + 1, generator=g)
        tokens, taken = ops.verify_draft(p.cuda(), x.cuda(), u.cuda(), d.cuda())
        want, n = verify(p, x, u, d)
        assert torch.equal(tokens.cpu(), want) and torch.equal(taken.cpu(), n)
        lens -= k - taken                      # the rejected rows' slots are filed over in the next step
        history = [torch.cat((history[b], rows[b, :1 + int(n[b])])) for b in range(B)]


def test_attn_many_ragged_sequences_without_a_bound_of_their_rows():
    """More row tiles (8192 sequences x all rows) than a launch holds: keys of zero weigh the same, so a row's output is the
    mean of its sequence's values, whole numbers: sums of them are exact, the division is off by at most 2 x 2^-24."""
    from musicgeneration_amd import ops
    B, T, dh, page = 8192, 300000, 64, 64
    n = torch.full((B,), T // B, dtype=torch.int64)
    n[5], n[4000] = 0, T - int(n.sum()) + int(n[4000]) - 100 + int(n[5])         # one empty, one long, 100 rows behind the last
    cu = torch.cat((torch.zeros(1, dtype=torch.int64), n.cumsum(0))).int().cuda()
    width = int(-(-n.max() // page))
    value = torch.arange(B, device="cuda") % 61 + 1
    kc = torch.zeros(61, 1, page, dh, device="cuda")
    vc = torch.arange(1, 62, device="cuda").float().view(61, 1, 1, 1).expand(61, 1, page, dh).contiguous()
    table = (value - 1).int()[:, None].expand(B, width).contiguous()
    out = ops.paged_attn(torch.randn(T, 1, dh, device="cuda"), kc, vc, table, n.int().cuda(), cu_rows=cu)
    last = int(cu[-1])
    want = value.repeat_interleave(n.cuda(), output_size=last).double()[:, None, None]
    assert last == T - 100 and not out[last:].any()
    assert float(((out[:last].double() - want).abs() / want).max()) <= 2 * 2.0 ** -24


def test_attn_a_row_that_is_not_a_number_stays_alone():
    """A padded batch: q of one sequence is NaN.  The prefix's tiles hold rows of all sequences; the others' outputs are the same."""
    from musicgeneration_amd import ops
    for dtype, B, R, Hq, Hkv, dh, P in ((BF16, 48, 1, 8, 2, 64, 700), (F32, 12, 3, 4, 2, 64, 300), (BF16, 70, 6, 4, 2, 64, 515), (BF16, 40, 4, 8, 2, 128, 600),
                                        (BF16, 3, 2, 4, 2, 136, 40)):
        k, v, table, prefix, g = _pool([70] * B, Hkv, 16, dh, dtype, P, seed=B)
        q = torch.randn(B, R, Hq, dh, generator=g).to(dtype).cuda()
        lens = torch.full((B,), 70, dtype=torch.int32).cuda()
        call = lambda x: ops.paged_attn(x, k.cuda(), v.cuda(), table.cuda(), lens, prefix=prefix.cuda(), prefix_len=P)   # noqa: E731
        clean = call(q)
        q[1], q[B - 1, 0] = NAN, math.inf
        got = call(q)
        stay = [b for b in range(B) if b not in (1, B - 1)]
        assert torch.equal(got[stay], clean[stay]), (dtype, B, R, dh)
        assert not torch.isfinite(got[1].float()).any()


def test_serving_on_two_streams_from_two_threads():
    """Calls of two threads, each on a stream of its own behind work that fills its inputs late, equal the same calls alone."""
    import threading
    from musicgeneration_amd import ops
    B, R, Hq, Hkv, dh, P = 6, 2, 8, 2, 64, 200
    cos, sin = ops.rope_tables(P + 400, dh)

    def run(seed, out):
        k, v, table, prefix, g = _pool([330] * B, Hkv, 16, dh, BF16, P, seed=seed)
        src = torch.randn(B, R, (Hq + 2 * Hkv) * dh, generator=g).bfloat16().cuda()
        k, v, table, prefix = k.cuda(), v.cuda(), table.cuda(), prefix.cuda()
        lens = torch.full((B,), 330, dtype=torch.int32, device="cuda")
        big = torch.ones(1 << 24, device="cuda")
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream), torch.no_grad():
            for _ in range(8):
                for _ in range(6):
                    big = big * 1.0
                qkv = src * big[:1].bfloat16()
                q = ops.paged_append(qkv, k, v, table, lens, Hq, cos, sin, offset=P)
                res = ops.paged_attn(q, k, v, table, lens, prefix=prefix, prefix_len=P)
                prob = res.float().reshape(B, R, -1).softmax(-1)
                tok, acc = ops.verify_draft(prob, torch.zeros(B, R - 1, dtype=torch.int64, device="cuda"), torch.full((B, R), 0.5, device="cuda"))
                out.append((res, ops.rotary(res, cos, sin), tok, acc))
            stream.synchronize()

    alone, both = [[], []], [[], []]
    for i in range(2):
        run(i, alone[i])
    threads = [threading.Thread(target=run, args=(i, both[i])) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for a, b in zip(alone, both):
        assert len(a) == len(b) == 8
        for x, y in zip(a, b):
            assert all(torch.equal(s, t) for s, t in zip(x, y))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Hq,Hkv,dh", [(4, 1, 256), (6, 2, 136), (3, 3, 192)])
@pytest.mark.parametrize("P", [0, 77])
def test_attn_wide_heads_of_many_rows(dtype, Hq, Hkv, dh, P):
    """Heads wider than 128: prompts whose rows fill tiles of every size (alone, and many short ones behind a prefix)."""
    cu, lens = [0, 1, 1, 70, 81], [1, 5, 69, 140]
    k, v, table, prefix, g = _pool(lens, Hkv, 16, dh, dtype, P, seed=dh + P)
    q = torch.randn(85, Hq, dh, generator=g).to(dtype)
    slopes = torch.rand(Hq, generator=g)
    for s in (None, slopes):
        out = _attend_both(q, k, v, table, lens, s, cu, prefix=prefix, P=P)
        assert not out[81:].any()
        _attend_both(q, k, v, table, lens, s, cu, prefix=prefix, P=P, max_rows=1, max_len=1)
    lens = [20] * 24
    k, v, table, prefix, g = _pool(lens, Hkv, 16, dh, dtype, P, seed=dh)
    _attend_both(torch.randn(24, 3, Hq, dh, generator=g).to(dtype), k, v, table, lens, slopes, prefix=prefix, P=P)


def test_attn_wide_heads_what_a_row_does_not_see_has_no_effect():
    """As above for narrower heads, with enough rows for the shared tiles."""
    from musicgeneration_amd import ops
    R, n, dh = 48, 90, 256
    k, v, table, _, g = _pool([n], 1, 16, dh, BF16, seed=2)
    q = torch.randn(1, R, 2, dh, generator=g).bfloat16().cuda()
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    clean = ops.paged_attn(q, k.cuda(), v.cuda(), table.cuda(), lens)
    for row in (1, 20, 47):
        j = n - R + row
        k2, v2 = k.clone(), v.clone()
        v2[table[0, j // 16], :, j % 16, 200] = math.inf
        got = ops.paged_attn(q, k2.cuda(), v2.cuda(), table.cuda(), lens)
        assert torch.equal(got[:, :row], clean[:, :row]) and not torch.isfinite(got[:, row:, :, 200].float()).any()
