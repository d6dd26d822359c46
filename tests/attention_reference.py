"""The attention block in 64 bits, element by element of its definition, on the CPU; and inputs for its tests."""

import math

import numpy as np
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# half a unit in the last place of a number, relative to it (at most)
HALF_ULP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def cdiv(a, b):
    return -(-a // b)


def sees(at, key, window, sinks):
    """Which of the keys (a vector of positions) the query at position ``at`` sees."""
    seen = key <= at
    return seen & ((at - key < window) | (key < sinks)) if window else seen


def attention(q, k, v, first, scale, window=0, sinks=0):
    """One request: q [n, hq, d] at positions first.., k, v [keys, hk, d] -> (out, lse, spread), spread = sum of p |v|."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    n, hq, d = q.shape
    keys, hk, _ = k.shape
    out, spread = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    for i in range(n):
        seen = torch.nonzero(sees(first + i, torch.arange(keys), window, sinks)).flatten()
        if first + i < 0 or len(seen) == 0:
            continue
        for h in range(hq):
            ks, vs = k[seen, h // (hq // hk)], v[seen, h // (hq // hk)]
            s = (ks @ q[i, h]) * scale
            p = torch.softmax(s, 0)
            out[i, h], spread[i, h] = p @ vs, p @ vs.abs()
            lse[i, h] = torch.logsumexp(s, 0)
    return out, lse, spread


def attention_error(dtype, out, spread, dim):
    """How far a kernel may be off: the result's rounding; the weights' rounding to 16 bits, each of which is off by half
    a place of itself; and fp32 scores, off by some 2^-24 of sums of dim products, whose exponentials
    are off by as much of themselves (scores here stay below 64)."""
    weights = 0.0 if dtype == F32 else HALF_ULP[dtype]
    return out.abs() * HALF_ULP[dtype] * 1.01 + spread * (weights * 1.01 + 64 * math.sqrt(dim) * 2.0 ** -23) + 1e-30 + (2.0 ** -25 if dtype == F16 else 0)


def norm(x, weight, eps):
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y * weight.double()


def rotate(y, positions, cos, sin, interleaved, back=False):
    """y [tokens, heads, d] in 64 bits; one pair at a time."""
    y = y.double().clone()
    if cos is None:
        return y
    half = cos.shape[1]
    c, s = cos.double()[positions.long()], sin.double()[positions.long()]
    s = -s if back else s
    out = y.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        ci, si = c[:, i, None], s[:, i, None]
        out[..., a] = y[..., a] * ci - y[..., b] * si
        out[..., b] = y[..., b] * ci + y[..., a] * si
    return out


def norm_rope(x, weight, positions, cos, sin, eps, interleaved):
    y = x.double() if weight is None else norm(x, weight, eps)
    return rotate(y, positions, cos, sin, interleaved)


def norm_rope_gradient(dz, x, weight, positions, cos, sin, eps, interleaved):
    """The formula's gradient: (dx, dweight)."""
    g = rotate(dz.double(), positions, cos, sin, interleaved, back=True)
    if weight is None:
        return g, None
    x, w = x.double(), weight.double()
    d = x.shape[-1]
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    dx = r * g * w - x * r ** 3 * (g * w * x).sum(-1, keepdim=True) / d
    return dx, (g * x * r).sum((0, 1))


def block_tables(cached, new, table, pool, state, page, tokens):
    """A step, request by request, on lists; returns what the call writes."""
    table, pool, ring = np.array(table), list(pool), list(pool)
    width = table.shape[1] if len(cached) else 0
    taken, returned = state
    free, asked = returned - taken, 0
    lengths, starts, positions, slots, refused = [], [0], [], [], False
    for i, (c, n) in enumerate(zip(cached, new)):
        held = cdiv(c, page)
        if n < 0:
            for j in range(min(held, width)):
                pool[returned % len(pool)] = int(table[i, j])
                returned += 1
            lengths.append(0)
            starts.append(starts[-1])
            continue
        need, ok = cdiv(c + n, page) - held, cdiv(c + n, page) <= width
        if ok and need:
            asked += need
            ok = asked <= free
        if ok:
            for j in range(held, held + need):
                table[i, j] = ring[taken % len(ring)]
                taken += 1
        refused |= not ok
        lengths.append(c + n if ok else c)
        starts.append(starts[-1] + n)
        for p in range(c, c + n):
            positions.append(p)
            slots.append(int(table[i, p // page]) * page + p % page if ok else -1)
    total = len(positions)
    positions = (positions + [0] * tokens)[:tokens]
    slots = (slots + [-1] * tokens)[:tokens]
    return {"table": table, "pool": pool, "state": [taken, returned], "lengths": lengths, "starts": starts,
            "positions": positions, "slots": slots, "refused": refused, "short": total > tokens}
