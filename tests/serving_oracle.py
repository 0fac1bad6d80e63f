"""Plain 64-bit forms of rotary, paged_append, paged_attn and verify_draft (CPU, loops), and error bounds for their tests.

A rounding is off by at most half a step: U[t] = finfo(t).eps / 2 of the value.
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def turn(x, cos, sin, layout):
    """x [..., dh], cos / sin broadcast to [..., rd/2] -> (rotated fp64, sum of the magnitudes of the two products)."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    rd = 2 * cos.shape[-1]
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if layout == "interleaved" else (x[..., :rd // 2], x[..., rd // 2:rd])
    y, size = x.clone(), torch.zeros_like(x)
    parts = (a * cos - b * sin, b * cos + a * sin)
    sizes = ((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs())
    if layout == "interleaved":
        y[..., 0:rd:2], y[..., 1:rd:2] = parts
        size[..., 0:rd:2], size[..., 1:rd:2] = sizes
    else:
        y[..., :rd // 2], y[..., rd // 2:rd] = parts
        size[..., :rd // 2], size[..., rd // 2:rd] = sizes
    return y, size


def assert_turned(got, want, size, name=""):
    """Two fp32 products and their sum (each off by 2^-24 of its size: at most 3 x 2^-24 of |ac| + |bs|), then one
    rounding to the storage type."""
    bound = U[got.dtype] * (want.abs() + 3 * 2.0 ** -24 * size) + 3 * 2.0 ** -24 * size
    over = (got.double().cpu() - want).abs() - bound
    assert not torch.isnan(got.float()).any() and float(over.max()) <= 0, (name, float(over.max()))


def rows_of(T, lens, cu, R):
    """[(sequence, own index)] of every row, None for rows of no sequence."""
    out = [None] * T
    for b, last in enumerate(lens):
        first, n = (cu[b], cu[b + 1] - cu[b]) if cu is not None else (b * R, R)
        for r in range(n):
            out[first + r] = (b, last - n + r)
    return out


def append(qkv, kc, vc, table, lens, Hq, cos, sin, layout, cu, offset):
    """fp64 (q, k, v, their product sizes) after the call; kc, vc are copied."""
    n_pages, Hkv, page, dh = kc.shape
    x = qkv.reshape(-1, Hq + 2 * Hkv, dh)
    R = None if cu is not None else qkv.shape[1]
    k, v = kc.double().clone(), vc.double().clone()
    q, qs, ks = torch.zeros(x.shape[0], Hq, dh, dtype=torch.float64), torch.zeros(x.shape[0], Hq, dh, dtype=torch.float64), torch.zeros_like(k)
    for t, place in enumerate(rows_of(x.shape[0], lens, cu, R)):
        if place is None:
            continue
        b, index = place
        if cos is None:
            y, size = x[t].double(), torch.zeros(Hq + 2 * Hkv, dh, dtype=torch.float64)
        else:
            at = min(max(offset + index, 0), cos.shape[0] - 1)
            y, size = turn(x[t], cos[at], sin[at], layout)
        q[t], qs[t] = y[:Hq], size[:Hq]
        if index < 0 or index // page >= table.shape[1]:
            continue
        pg = int(table[b, index // page])
        if 0 <= pg < n_pages:
            k[pg, :, index % page], ks[pg, :, index % page] = y[Hq:Hq + Hkv], size[Hq:Hq + Hkv]
            v[pg, :, index % page] = x[t, Hq + Hkv:].double()
    return q, k, v, qs, ks


def attend(q, kc, vc, table, lens, slopes, cu, prefix, P, scale=None):
    """fp64 (out, bound): the definition, row by row, and how far a kernel in dtype q.dtype may be off:
      scores  dh products and sums in fp32, the scale and the slope term: d = (dh + 4) 2^-24 max_j (scale sum |q||k| + |bias|)
      weights exp of scores off by d: 2 d relative; their rounding to the storage type for the matrix product: 2 U; fp32
              sums of n weights in blocks: (n / 16 + 64) 2^-24
      each on sum_j p_j |v_j|, then the output's own rounding."""
    n_pages, Hkv, page, dh = kc.shape
    Hq = q.shape[-2]
    x = q.reshape(-1, Hq, dh).double()
    R = None if cu is not None else q.shape[1]
    scale = dh ** -0.5 if scale is None else scale
    out, bound = torch.zeros_like(x), torch.zeros_like(x)
    for t, place in enumerate(rows_of(x.shape[0], lens, cu, R)):
        if place is None:
            continue
        b, index = place
        ks, vs, js = [], [], []
        own = min(max(index + 1, 0), table.shape[1] * page)
        i = P + own - 1                               # (own index + 1 keys: i of the definition wherever any own key is seen)
        for j in range(P + own):
            pg = int(prefix[j // page]) if j < P else int(table[b, (j - P) // page])
            if 0 <= pg < n_pages:
                ks.append((pg, (j if j < P else j - P) % page))
                js.append(j)
        if not js:
            continue
        pgs, slots = torch.tensor([p for p, _ in ks]), torch.tensor([s for _, s in ks])
        k, v = kc[pgs, :, slots].double(), vc[pgs, :, slots].double()                 # [n, Hkv, dh]
        off = torch.tensor(js, dtype=torch.float64) - i
        for h in range(Hq):
            kk, vv = k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)]
            bias = off * (float(slopes[h]) if slopes is not None else 0.0)
            s = kk @ x[t, h] * scale + bias
            p = s.softmax(0)
            out[t, h] = p @ vv
            size = kk.abs() @ x[t, h].abs() * abs(scale) + bias.abs()
            d = (dh + 4) * 2.0 ** -24 * float(size.max())
            u = U[q.dtype]
            n = len(js)
            bound[t, h] = (2 * u + 2 * d + (n / 16 + 64) * 2.0 ** -24) * (p @ vv.abs()) + u * out[t, h].abs()
    return out.view(q.shape), bound.view(q.shape)


def assert_attended(got, want, bound):
    assert torch.isfinite(got.float()).all()
    over = (got.double().cpu() - want).abs() - bound
    worst = int(over.argmax())
    assert float(over.max()) <= 0, (float(over.max()), worst, float(got.flatten()[worst]), float(want.flatten()[worst]))


def verify(target, tokens, u, draft=None, counts=None):
    B, k = tokens.shape
    V = target.shape[-1]
    out, acc = torch.full((B, k + 1), -1, dtype=tokens.dtype), torch.zeros(B, dtype=torch.int32)

    def clean(r):
        r = r.double()
        return torch.where((r > 0) & (r < math.inf), r, torch.zeros_like(r))

    for b in range(B):
        n = k if counts is None else min(max(int(counts[b]), 0), k)
        a = 0
        while a < n:
            c = int(tokens[b, a])
            if not 0 <= c < V:
                break
            q = 1.0 if draft is None else float(draft[b, a, c])
            if not float(u[b, a]) * q < float(target[b, a, c]) or not float(clean(target[b, a, c])) > 0:
                break
            out[b, a] = c
            a += 1
        rest = clean(target[b, a])
        if a < n and draft is not None:
            rest = (rest - clean(draft[b, a])).clamp(min=0)
        elif a < n and 0 <= int(tokens[b, a]) < V:
            rest[int(tokens[b, a])] = 0.0
        if not float(rest.sum()) > 0:
            rest = clean(target[b, a])
        run = 0.0
        goal = float(u[b, k]) * float(rest.sum())
        found = last = 0
        hit = False
        for c, w in enumerate(rest.tolist()):
            run += w
            if w > 0:
                last = c
            if not hit and w > 0 and run > goal:
                found, hit = c, True
        out[b, a] = found if hit else last
        acc[b] = a
    return out, acc
