"""Cases for the operators of rotary, paged serving: rotation, filing into a paged cache, attention over a shared prefix
and the sequences' own pages, and the verification of drafted tokens.

`run` computes each operator in its plain form (elementary torch operations, 32-bit) or, where `own` is set, through
`musicgeneration_amd.ops`.  `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one sampling step of a batch of 32: q and k heads of one token each, every sequence at its own position
        {"name": "rotary_step", "op": "rotary", "batch": 32, "seq": 1, "heads": 12, "spare": 4, "dh": 64, "rd": 64,
         "layout": "interleaved", "dtype": "bf16", "far": 32768, "positions": True, "grad": False},
        # training: q | k heads of a packed projection of 16 sequences of 2048 tokens, forward and gradient
        {"name": "rotary_train", "op": "rotary", "batch": 16, "seq": 2048, "heads": 16, "spare": 8, "dh": 64, "rd": 64,
         "layout": "interleaved", "dtype": "bf16", "far": 2048, "positions": False, "grad": True},
        # parity mode: fp32, half layout over part of the head, odd lengths, windows that begin far into a piece
        {"name": "rotary_far", "op": "rotary", "batch": 3, "seq": 1371, "heads": 10, "spare": 5, "dh": 80, "rd": 40,
         "layout": "half", "dtype": "fp32", "far": 131072, "positions": True, "grad": True},
        # one sampling step of 64 sequences: a row each into pages of 16
        {"name": "append_step", "op": "append", "seqs": 64, "least": 1, "most": 1, "past": 4000, "hq": 8, "hkv": 8, "dh": 64,
         "rd": 64, "page": 16, "layout": "interleaved", "dtype": "bf16", "offset": 0},
        # primers of 1 to 3000 tokens, filed behind a shared prefix before the first step
        {"name": "append_prompts", "op": "append", "seqs": 11, "least": 1, "most": 3000, "past": 0, "hq": 32, "hkv": 8,
         "dh": 128, "rd": 128, "page": 64, "layout": "half", "dtype": "bf16", "offset": 4001},
        # a sampling step of the ALiBi model without a shared prefix
        {"name": "attn_step", "op": "attn", "seqs": 16, "least": 1, "most": 1, "past": 2047, "hq": 8, "hkv": 8, "dh": 64,
         "page": 16, "prefix": 0, "alibi": True, "dtype": "bf16"},
        # 64 continuations of one 8192-token primer, one row each
        {"name": "attn_shared_step", "op": "attn", "seqs": 64, "least": 1, "most": 1, "past": 1023, "hq": 32, "hkv": 8,
         "dh": 128, "page": 64, "prefix": 8192, "alibi": False, "dtype": "bf16"},
        # 128 continuations of a long primer that ends inside a page, six rows each (a token and five drafted ones)
        {"name": "attn_shared_draft", "op": "attn", "seqs": 128, "least": 6, "most": 6, "past": 2000, "hq": 20, "hkv": 4,
         "dh": 64, "page": 32, "prefix": 16385, "alibi": False, "dtype": "bf16"},
        # ragged prompts behind a shared instruction-like opening
        {"name": "attn_prompts", "op": "attn", "seqs": 9, "least": 1, "most": 1500, "past": 200, "hq": 16, "hkv": 2,
         "dh": 128, "page": 64, "prefix": 4001, "alibi": False, "dtype": "bf16"},
        # parity mode: fp32, three rows each (the sampling loop's), ALiBi
        {"name": "attn_fp32", "op": "attn", "seqs": 24, "least": 3, "most": 3, "past": 700, "hq": 12, "hkv": 4, "dh": 64,
         "page": 16, "prefix": 1000, "alibi": True, "dtype": "fp32"},
        # the unified MIDI vocabulary (rows padded to a multiple of 64 by the model's head)
        {"name": "verify_midi", "op": "verify", "seqs": 4, "drafts": 4, "vocab": 618, "pad": 22, "dtype": "fp32",
         "drafted": True, "agree": 0.7},
        # a large vocabulary and batch
        {"name": "verify_wide", "op": "verify", "seqs": 128, "drafts": 5, "vocab": 50257, "pad": 0, "dtype": "fp32",
         "drafted": True, "agree": 0.7},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(8, 8, 64), (12, 4, 64), (16, 2, 128), (32, 8, 128), (6, 6, 96), (20, 4, 64), (6, 6, 128), (4, 1, 80)]


def draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "append", "attn", "attn", "attn", "verify"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    layout = rng.choice(["interleaved", "half"])
    if op == "rotary":
        dh = rng.choice([64, 80, 96, 128])
        batch = _spread(rng, 1, 32)
        return {"op": op, "batch": batch, "seq": _spread(rng, 1, 16384 // batch), "heads": rng.randint(1, 16),
                "spare": rng.choice([0, 3, 8]), "dh": dh, "rd": rng.choice([dh, dh // 2, dh // 4 * 2]), "layout": layout,
                "dtype": dtype, "far": 131072, "positions": rng.random() < 0.5, "grad": rng.random() < 0.6}
    if op == "verify":
        return {"op": op, "seqs": _spread(rng, 1, 96), "drafts": rng.randint(1, 5), "vocab": _spread(rng, 128, 50000),
                "pad": rng.choice([0, 1, 22, 64]), "dtype": dtype, "drafted": rng.random() < 0.8, "agree": rng.uniform(0.2, 1.0)}
    hq, hkv, dh = rng.choice(_HEADS)
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        if rng.random() < 0.5:
            n = rng.randint(1, 8)
            seqs, least, most, past = _spread(rng, 1, 128), n, n, _spread(rng, 16, 4000)
        else:
            seqs, least, most, past = rng.randint(1, 8), 1, _spread(rng, 16, 3000), _spread(rng, 1, 500)
        return {"op": op, "seqs": seqs, "least": least, "most": most, "past": past, "hq": hq, "hkv": hkv, "dh": dh,
                "rd": rng.choice([dh, dh // 2]), "page": page, "layout": layout, "dtype": dtype,
                "offset": _spread(rng, 1, 16000) - 1}
    prefix = rng.choice([0, _spread(rng, 1, 200), _spread(rng, 200, 8000)])
    if rng.random() < 0.7:
        n = rng.randint(1, 6)
        seqs, least, most, past = _spread(rng, 1, 64), n, n, _spread(rng, 1, 2000)
    else:
        seqs, least, most, past = rng.randint(1, 6), 1, _spread(rng, 8, 1000), _spread(rng, 1, 300)
    return {"op": op, "seqs": seqs, "least": least, "most": most, "past": past, "hq": hq, "hkv": hkv, "dh": dh, "page": page,
            "prefix": prefix, "alibi": rng.random() < 0.4, "dtype": dtype}


def _stairs(lo, hi, n):
    """n whole numbers from lo to hi, evenly apart: a batch's lengths (the seed only shuffles them)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "rotary":
        values = case["batch"] * case["seq"] * case["heads"] * case["dh"]
        passes = 2 if case["grad"] else 1
        return {"bytes": 2 * passes * values * size, "flops": 3 * passes * values * case["rd"] // case["dh"]}
    if case["op"] == "append":
        rows = sum(_stairs(case["least"], case["most"], case["seqs"]))
        width = (case["hq"] + 2 * case["hkv"]) * case["dh"]
        return {"bytes": 2 * rows * width * size, "flops": 3 * rows * (case["hq"] + case["hkv"]) * case["rd"]}
    if case["op"] == "verify":
        rows = 2 if case["drafted"] else 1
        return {"bytes": case["seqs"] * rows * case["vocab"] * size, "flops": case["seqs"] * (rows + 1) * case["vocab"]}
    ns, past = _stairs(case["least"], case["most"], case["seqs"]), sum(_stairs(0, case["past"], case["seqs"]))
    rows, keys = sum(ns), sum(ns) + past
    pairs = rows * case["prefix"] + sum(n * (n + 1) // 2 for n in ns) + past * rows // len(ns)
    kv = 2 * case["hkv"] * case["dh"] * size
    return {"bytes": 2 * rows * case["hq"] * case["dh"] * size + (case["prefix"] + keys) * kv,
            "flops": 4 * pairs * case["hq"] * case["dh"]}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _tables(n, rd):
    """cos, sin [n, rd/2] of position * 10000^(-2i/rd): angles in 64 bits, kept in 32."""
    freq = 10000.0 ** (-torch.arange(0, rd, 2, dtype=torch.float64, device="cuda") / rd)
    angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen).tolist()
    return [values[i] for i in order]


def _pages(case, lens, gen, dev):
    """A pool of pages in shuffled order, the sequences' page tables, and the shared prefix's."""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    shared = -(-case.get("prefix", 0) // page)
    ids = torch.randperm(sum(need) + shared + 3, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    at = shared
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    shape = (ids.numel(), case["hkv"], page, case["dh"])
    cache = [torch.randn(shape, generator=dev, device="cuda").to(_DT[case["dtype"]]) for _ in range(2)]
    return table.cuda(), ids[:shared].cuda(), cache


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DT[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rotary":
        B, S, H, dh = case["batch"], case["seq"], case["heads"], case["dh"]
        packed = torch.randn(B, S, H + case["spare"], dh, generator=dev, device="cuda").to(dtype)
        s["x"] = packed[:, :, :H].detach().requires_grad_(case["grad"])
        s["dy"] = torch.randn(B, S, H, dh, generator=dev, device="cuda").to(dtype) if case["grad"] else None
        s["cos"], s["sin"] = _tables(max(case["far"], S), case["rd"])
        s["positions"] = None
        if case["positions"]:       # every sequence a window of its own
            first = torch.randint(0, max(case["far"], S) - S + 1, (B, 1), generator=gen)
            s["positions"] = (first + torch.arange(S)).cuda()
        return s
    if case["op"] == "verify":
        B, k, V = case["seqs"], case["drafts"], case["vocab"]
        logits = 2.0 * torch.randn(B, k + 1, V, generator=dev, device="cuda")
        other = case["agree"] * logits[:, :k] + 2.0 * (1 - case["agree"]) * torch.randn(B, k, V, generator=dev, device="cuda")
        q = other.softmax(-1)
        s["tokens"] = torch.multinomial(q.view(B * k, V), 1, generator=dev).view(B, k)
        s["target"] = _padded(logits.softmax(-1), case["pad"], dtype)
        s["draft"] = _padded(q, case["pad"], dtype) if case["drafted"] else None
        s["u"] = torch.rand(B, k + 1, generator=dev, device="cuda")
        return s
    ns = _shuffled(_stairs(case["least"], case["most"], case["seqs"]), gen)
    past = _shuffled(_stairs(0, case["past"], case["seqs"]), gen)
    lens = [n + p for n, p in zip(ns, past)]
    s["uniform"] = case["least"] == case["most"]
    s["max_rows"], s["max_len"] = max(ns), max(lens)
    s["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    s["cu"] = torch.tensor([0] + ns).cumsum(0).to(torch.int32).cuda()
    s["table"], s["prefix"], (s["k"], s["v"]) = _pages(case, lens, gen, dev)
    lead = (len(ns), ns[0]) if s["uniform"] else (sum(ns),)
    if case["op"] == "append":
        width = (case["hq"] + 2 * case["hkv"]) * case["dh"]
        s["qkv"] = torch.randn(*lead, width, generator=dev, device="cuda").to(dtype)
        s["cos"], s["sin"] = _tables(case["offset"] + max(lens), case["rd"])
        return s
    s["q"] = (1.5 * torch.randn(*lead, case["hq"], case["dh"], generator=dev, device="cuda")).to(dtype)
    s["slopes"] = None
    if case["alibi"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, case["hq"] + 1, dtype=torch.float32, device="cuda") / case["hq"])
    return s


def _padded(p, pad, dtype):
    """The [..., :V] view of rows that are `pad` values longer, as a head with a padded class dimension leaves them."""
    return torch.nn.functional.pad(p.to(dtype), (0, pad), value=0.5)[..., :p.shape[-1]]


# ---------------------------------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"rotary": _rotary, "append": _append, "attn": _attn, "verify": _verify}[state["case"]["op"]](state)


def _rotary(s):
    c = s["case"]
    if own:
        from musicgeneration_amd import ops
        y = ops.rotary(s["x"], s["cos"], s["sin"], s["positions"], layout=c["layout"])
        if not c["grad"]:
            return y
        return y, torch.autograd.grad(y, s["x"], s["dy"])[0]
    x = s["x"].detach()
    if s["positions"] is None:
        cos, sin = s["cos"][:c["seq"], None], s["sin"][:c["seq"], None]
    else:
        cos, sin = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
    y = _turn(x.float(), cos, sin, c["rd"], c["layout"]).to(x.dtype)
    if not c["grad"]:
        return y
    return y, _turn(s["dy"].float(), cos, -sin, c["rd"], c["layout"]).to(x.dtype)


def _turn(x, cos, sin, rd, layout):
    """The first rd values of each head, turned pair by pair; the rest as it is."""
    if layout == "interleaved":
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rd:]), -1)


def _rows(s):
    """(sequence, own index) of every row of the batch, in order."""
    ns = s["cu"][1:] - s["cu"][:-1]
    total = s["qkv" if "qkv" in s else "q"].numel() // (s["qkv"].shape[-1] if "qkv" in s else s["q"].shape[-1] * s["q"].shape[-2])
    row = torch.arange(total, device="cuda")
    b = torch.searchsorted(s["cu"], row, right=True, out_int32=False) - 1
    return b, row - s["cu"][b] + (s["lens"] - ns)[b]


def _append(s):
    c = s["case"]
    if own:
        from musicgeneration_amd import ops
        q = ops.paged_append(s["qkv"], s["k"], s["v"], s["table"], s["lens"], c["hq"], s["cos"], s["sin"],
                             layout=c["layout"], cu_rows=None if s["uniform"] else s["cu"], offset=c["offset"])
        return q, s["k"], s["v"]
    hq, hkv, dh = c["hq"], c["hkv"], c["dh"]
    x = s["qkv"].reshape(-1, hq + 2 * hkv, dh)
    b, index = _rows(s)
    at = index + c["offset"]
    turned = _turn(x[:, :hq + hkv].float(), s["cos"][at][:, None], s["sin"][at][:, None], c["rd"], c["layout"]).to(x.dtype)
    page = s["table"][b, index // c["page"]].long()
    s["k"][page, :, index % c["page"]] = turned[:, hq:]
    s["v"][page, :, index % c["page"]] = x[:, hq + hkv:]
    return turned[:, :hq].reshape(*s["qkv"].shape[:-1], hq, dh).contiguous(), s["k"], s["v"]


def _gathered(cache, table):
    """Pages of a table [..., n] as rows of keys: [..., heads, n * page, dh] in 32 bits."""
    x = cache[table.clamp(min=0).long()].float()
    return x.transpose(-4, -3).flatten(-3, -2)


def _attn(s):
    c = s["case"]
    if own:
        from musicgeneration_amd import ops
        return ops.paged_attn(s["q"], s["k"], s["v"], s["table"], s["lens"], slopes=s["slopes"],
                              cu_rows=None if s["uniform"] else s["cu"], max_rows=s["max_rows"], max_len=s["max_len"],
                              prefix=s["prefix"] if c["prefix"] else None, prefix_len=c["prefix"])
    hq, hkv, dh, P = c["hq"], c["hkv"], c["dh"], c["prefix"]
    G, B, R, scale = hq // hkv, c["seqs"], s["max_rows"], 1.0 / math.sqrt(c["dh"])
    q = s["q"].reshape(-1, hkv, G, dh).float() * scale
    T = q.shape[0]
    b, index = _rows(s)
    r = torch.arange(T, device="cuda") - s["cu"][b]
    # own keys, the rows padded to R a sequence: [B, hkv, R, G, keys]
    k, v = _gathered(s["k"], s["table"]), _gathered(s["v"], s["table"])
    L = k.shape[2]
    padded = torch.zeros(B, R, hkv, G, dh, device="cuda")
    padded[b, r] = q
    padded = padded.permute(0, 2, 1, 3, 4).reshape(B, hkv, R * G, dh)
    so = torch.matmul(padded, k.transpose(-1, -2).contiguous()).view(B, hkv, R, G, L)
    at = (s["lens"] - (s["cu"][1:] - s["cu"][:-1]))[:, None] + torch.arange(R, device="cuda")       # [B, R]
    off = torch.arange(L, device="cuda") - at[..., None]                                           # [B, R, L]
    if s["slopes"] is not None:
        slopes = s["slopes"].view(hkv, 1, G, 1)
        so = so + slopes * off[:, None, :, None].float()
    so = so.masked_fill((off > 0)[:, None, :, None], -math.inf)
    top = so.amax(-1)
    if P:
        kp, vp = _gathered(s["k"], s["prefix"])[:, :P], _gathered(s["v"], s["prefix"])[:, :P]
        qp = q.permute(1, 0, 2, 3).reshape(hkv, T * G, dh)
        sp = torch.matmul(qp, kp.transpose(-1, -2).contiguous()).view(hkv, T, G, P)
        if s["slopes"] is not None:
            sp = sp + slopes * (torch.arange(P, device="cuda") - (P + index)[:, None])[None, :, None].float()
        top_rows = torch.maximum(sp.amax(-1), top[b, :, r].permute(1, 0, 2))                        # [hkv, T, G]
        sp = (sp - top_rows[..., None]).exp()
        top = top.clone()
        top[b, :, r] = top_rows.permute(1, 0, 2)
    so = (so - top[..., None]).exp()
    out = torch.matmul(so.view(B, hkv, R * G, L), v.contiguous()).view(B, hkv, R, G, dh)[b, :, r]   # [T, hkv, G, dh]
    mass = so.sum(-1)[b, :, r]
    if P:
        out = out + torch.matmul(sp.view(hkv, T * G, P), vp.contiguous()).view(hkv, T, G, dh).permute(1, 0, 2, 3)
        mass = mass + sp.sum(-1).permute(1, 0, 2)
    return (out / mass[..., None]).to(s["q"].dtype).view(s["q"].shape)


def _verify(s):
    if own:
        from musicgeneration_amd import ops
        return ops.verify_draft(s["target"], s["tokens"], s["u"], draft=s["draft"])
    p, x, u = s["target"], s["tokens"], s["u"]
    B, k = x.shape
    px = p[:, :k].gather(-1, x[..., None])[..., 0].double()
    if s["draft"] is None:
        qx = torch.ones_like(px)
    else:
        qx = s["draft"].gather(-1, x[..., None])[..., 0].double()
    taken = (u[:, :k].double() * qx < px).long().cumprod(-1).sum(-1)
    at = torch.arange(B, device="cuda")
    row = p[at, taken].double()
    last = taken.clamp(max=k - 1)
    if s["draft"] is None:
        lost = torch.zeros_like(row).scatter_(-1, x[at, last][:, None], math.inf)
    else:
        lost = s["draft"][at, last].double()
    rest = (row - lost).clamp(min=0)
    use = (taken < k) & (rest.sum(-1) > 0)
    rest = torch.where(use[:, None], rest, row)
    run_sum = rest.cumsum(-1)
    over = run_sum > u[:, k, None].double() * run_sum[:, -1:]
    drawn = over.long().argmax(-1)
    place = torch.arange(k + 1, device="cuda")
    out = torch.cat((x, x[:, :1]), -1)
    out = torch.where(place == taken[:, None], drawn[:, None], out).masked_fill(place > taken[:, None], -1)
    return out, taken.to(torch.int32)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        at = s["positions"] if s["positions"] is not None else torch.arange(case["seq"], device="cuda").expand(case["batch"], -1)
        w = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, :, None]
        y = _complex_turn(s["x"].detach().double(), w, case)
        return (y, _complex_turn(s["dy"].double(), w.conj(), case)) if case["grad"] else y
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "attn":
        return _exact_attn(s, case)
    return _exact_verify(s)


def _complex_turn(x, w, case):
    """A pair (a, b) as a + ib, times cos + i sin."""
    rd, half = case["rd"], case["rd"] // 2
    pair = (half, 2) if case["layout"] == "interleaved" else (2, half)
    z = x[..., :rd].unflatten(-1, pair)
    z = z if case["layout"] == "interleaved" else z.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * w)
    z = z if case["layout"] == "interleaved" else z.transpose(-1, -2)
    x = x.clone()
    x[..., :rd] = z.flatten(-2)
    return x


def _exact_append(s, case):
    hq, hkv, dh, page = case["hq"], case["hkv"], case["dh"], case["page"]
    k, v = s["k"].double(), s["v"].double()
    x = s["qkv"].reshape(-1, hq + 2 * hkv, dh).double()
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    queries = []
    for b, last in enumerate(lens):
        rows = x[cu[b]:cu[b + 1]]
        index = torch.arange(last - rows.shape[0], last, device="cuda")
        angle = torch.complex(s["cos"][index + case["offset"]].double(), s["sin"][index + case["offset"]].double())
        turned = _complex_turn(rows[:, :hq + hkv], angle[:, None], case)
        slot = s["table"][b].long()[index // page] * page + index % page
        k[slot // page, :, slot % page] = turned[:, hq:]
        v[slot // page, :, slot % page] = rows[:, hq + hkv:]
        queries.append(turned[:, :hq])
    return torch.cat(queries).view(*s["qkv"].shape[:-1], hq, dh), k, v


def _exact_attn(s, case):
    hq, hkv, dh, P = case["hq"], case["hkv"], case["dh"], case["prefix"]
    q = s["q"].reshape(-1, hq, dh).double()
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    out = torch.zeros_like(q)
    for b, last in enumerate(lens):
        n = cu[b + 1] - cu[b]
        keys = [[], []]
        for side, cache in enumerate((s["k"], s["v"])):
            for table, length in ((s["prefix"], P), (s["table"][b], last)):
                used = cache[table[:-(-length // case["page"])].long()].double()        # [pages, hkv, page, dh]
                keys[side].append(used.permute(1, 0, 2, 3).reshape(hkv, -1, dh)[:, :length])
        k, v = torch.cat(keys[0], 1), torch.cat(keys[1], 1)
        place = torch.arange(P + last, device="cuda")
        at = P + last - n + torch.arange(n, device="cuda")
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            score = q[cu[b]:cu[b + 1], heads].transpose(0, 1) @ k[h].t() / math.sqrt(dh)
            if s["slopes"] is not None:
                score = score + s["slopes"][heads].double()[:, None, None] * (place - at[:, None]).double()
            score = score.masked_fill(place > at[:, None], -math.inf)
            out[cu[b]:cu[b + 1], heads] = (score.softmax(-1) @ v[h]).transpose(0, 1)
    return out.view(s["q"].shape)


def _exact_verify(s):
    p, x, u = s["target"].cpu().double(), s["tokens"].cpu(), s["u"].cpu().double()
    q = None if s["draft"] is None else s["draft"].cpu().double()
    B, k = x.shape
    out = torch.full((B, k + 1), -1, dtype=torch.int64)
    count = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = 0
        while n < k and u[b, n] * (1.0 if q is None else q[b, n, x[b, n]]) < p[b, n, x[b, n]]:
            out[b, n] = x[b, n]
            n += 1
        rest = p[b, n].clone()
        if n < k and q is None:
            rest[x[b, n]] = 0.0
        elif n < k:
            rest = (rest - q[b, n]).clamp(min=0)
        if not rest.sum() > 0:
            rest = p[b, n]
        total = rest.cumsum(0)
        out[b, n] = torch.searchsorted(total, u[b, k] * total[-1], right=True)
        count[b] = n
    return out.cuda(), count.cuda()
