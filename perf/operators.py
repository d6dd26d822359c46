"""The attention block of one rank of a tensor-parallel decoder, as cases to be timed.

Between the shard of the query / key / value projection and the output
projection's K-shard a rank works on its own heads:

* ``tables``   block tables, positions and slots of a step, from request lengths;
* ``rope``     norms of query and key heads, their rotation, the write into the cache;
* ``grad``     the gradient of norms and rotation;
* ``decode``   attention of one new token a request over the paged cache;
* ``prompt``   attention of many new tokens a request over the same cache.

``own`` False computes them with elementary torch operations in 32 bits,
``own`` True calls ``iris_amd.attention``.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def _tables(name, requests, prompts, ended, new, cached, page):
    """A step of ``requests`` requests: ``prompts`` of them bring up to ``new`` tokens, ``ended`` give their pages
    back, the others bring one token; up to ``cached`` tokens are there already."""
    case = {"op": "tables", "requests": requests, "prompts": prompts, "ended": ended, "new": new, "cached": cached,
            "page": page}
    return dict(case, name=name) if name else case


def _rope(name, op, dtype, tokens, hq, hk, dim, rotary, interleaved, norm, cache=False, page=16):
    """``cache``: keys and values go to their slots of the paged cache (serving), else k_out is written."""
    case = {"op": op, "dtype": dtype, "tokens": tokens, "hq": hq, "hk": hk, "dim": dim, "rotary": rotary,
            "interleaved": interleaved, "norm": norm, "cache": cache, "page": page}
    return dict(case, name=name) if name else case


def _attention(name, op, dtype, requests, new, cached, hq, hk, dim, page, window=0, sinks=0):
    """decode: ``requests`` contexts of up to ``cached`` tokens; prompt: up to ``new`` tokens behind up to ``cached``."""
    case = {"op": op, "dtype": dtype, "requests": requests, "new": new, "cached": cached, "hq": hq, "hk": hk,
            "dim": dim, "page": page, "window": window, "sinks": sinks}
    return dict(case, name=name) if name else case


def listed():
    return [
        # A decode step of 64 requests: latency of one small launch.
        _tables("tables_step", 64, 0, 0, 1, 8192, 16),
        # A thousand requests, some of them new prompts, some ended.
        _tables("tables_mixed", 1000, 24, 15, 2000, 8192, 16),
        # Sixteen tokens of a 6.7B decoder cut over eight ranks (4 heads of 128 a rank): rotation and cache write.
        _rope("rope_step", "rope", "bf16", 16, 4, 4, 128, 128, False, False, cache=True),
        # A batch of prompts, normed heads, grouped keys, a number of tokens that is a multiple of nothing.
        _rope("norm_rope_prompts", "rope", "bf16", 8191, 8, 2, 128, 128, False, True, cache=True),
        # Training: the gradient for a whole layer's heads on one GPU.
        _rope("norm_rope_grad", "grad", "bf16", 8192, 32, 8, 128, 128, False, True),
        # fp32, an odd head size, interleaved pairs over part of the head.
        _rope("norm_rope_grad_fp32", "grad", "fp32", 1000, 6, 2, 80, 32, True, True),
        # One request of odd length, 4 heads of their own keys: the smallest call of a server.
        _attention("decode_one", "decode", "bf16", 1, 1, 1999, 4, 4, 128, 16),
        # A batch of requests of very different lengths, eight query heads to one key head (one rank of eight).
        _attention("decode_batch", "decode", "bf16", 64, 1, 8192, 8, 1, 128, 16),
        # Long contexts: the whole cache of a few requests is read once.
        _attention("decode_long", "decode", "fp16", 16, 1, 131072, 8, 2, 128, 64),
        # A layer with a sliding window and visible first tokens, many requests.
        _attention("decode_window", "decode", "bf16", 128, 1, 16384, 8, 2, 64, 32, window=1024, sinks=4),
        # Prompts and pieces of prompts behind cached tokens, causal.
        _attention("prompt_causal", "prompt", "bf16", 4, 8192, 2048, 8, 1, 128, 16),
        # Prompts through a layer with a sliding window and visible first tokens, ten heads of 64.
        _attention("prompt_window", "prompt", "fp16", 4, 8192, 1000, 10, 2, 64, 32, window=1024, sinks=4),
    ]


# ---- sizes -------------------------------------------------------------------


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _avoid(n):
    return n + 1 if n == 3072 else n


def _shape_rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _contexts(case):
    """Context lengths of a decode batch: the longest, one idle slot, one first token, the rest ragged."""
    rng, count, hi = _shape_rng(case), case["requests"], case["cached"]
    lengths = [_avoid(_log(rng, max(1, hi // 64), hi)) for _ in range(count)]
    lengths[0] = hi
    if count >= 8:
        lengths[1], lengths[2] = 0, 1
    return lengths


def _prompts(case):
    """(new, cached) tokens of each request of a prompt batch."""
    rng, count, new, cached = _shape_rng(case), case["requests"], case["new"], case["cached"]
    pairs = [(_avoid(_log(rng, max(1, new // 16), new)), _avoid(rng.randint(0, cached))) for _ in range(count)]
    pairs[0] = (new, 0)
    if count >= 4:
        pairs[1] = (1, cached)  # a request that decodes beside the prompts
    return pairs


def _step(case):
    """(cached, new) tokens of each request of a step; new is -1 where the request has ended."""
    rng, count = _shape_rng(case), case["requests"]
    pairs = []
    for i in range(count):
        cached = rng.randint(0, case["cached"])
        if i < case["ended"]:
            pairs.append((cached, -1))
        elif i < case["ended"] + case["prompts"]:
            pairs.append((rng.choice([0, 0, cached]), _log(rng, max(1, case["new"] // 16), case["new"])))
        else:
            pairs.append((cached, 1))
    return [(_avoid(c), _avoid(n)) for c, n in pairs]


def _cdiv(a, b):
    return (a + b - 1) // b


def _visible(length, window, sinks):
    """Keys that the token at position length - 1 sees."""
    if length <= 0 or not window or length <= window:
        return max(length, 0)
    return window + min(sinks, length - window)


def _reach(new, cached, window, sinks):
    """Keys that any of ``new`` tokens behind ``cached`` sees."""
    lo = max(0, cached + 1 - window) if window else 0
    return cached + new - lo + min(sinks, lo)


_MOST_BYTES, _MOST_FLOPS, _MOST_PADDED = 6.0e8, 1.5e11, 16 * 131072 * 2 * 128


def _too_much(case):
    w = work(case)
    if w["bytes"] > _MOST_BYTES or w["flops"] > _MOST_FLOPS:
        return True
    if case["op"] == "decode":
        return case["requests"] * case["cached"] * case["hk"] * case["dim"] > _MOST_PADDED
    if case["op"] == "prompt":
        return sum(n * (n + c) for n, c in _prompts(case)) * case["hq"] > 8e9
    return False


def draw(rng):
    while True:
        op = rng.choices(["tables", "rope", "grad", "decode", "prompt"], [10, 20, 15, 30, 25])[0]
        dtype = rng.choices(["bf16", "fp16", "fp32"], [50, 30, 20])[0]
        dim = rng.choices([64, 80, 96, 128, 192, 256], [25, 8, 10, 40, 7, 10])[0]
        hk = rng.choice([1, 1, 2, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 8, 12, 16])
        page = rng.choices([16, 32, 64, 128, 8, 20], [35, 20, 20, 10, 8, 7])[0]
        window = rng.choice([0, 0, 0, _log(rng, 16, 8192)])
        sinks = rng.choice([0, 1, 4, 16, 100]) if window else 0
        if op == "tables":
            count = _log(rng, 1, 4096)
            ended, prompts = int(count * rng.uniform(0, 0.1)), int(count * rng.choice([0, 0, 0.02, 0.2]))
            new = _log(rng, 2, 4096)
            if prompts * new > 1 << 18:
                continue
            case = _tables(None, count, prompts, ended, new, _log(rng, 1, 16384), page)
        elif op in ("rope", "grad"):
            rotary = rng.choice([dim, dim, dim // 2, 32])
            tokens = _log(rng, 1, 16384)
            norm = rng.random() < 0.7
            cache = op == "rope" and rng.random() < 0.6
            case = _rope(None, op, dtype, tokens, hq, hk, dim, rotary, rng.random() < 0.3, norm, cache, page)
        elif op == "decode":
            case = _attention(None, op, dtype, _log(rng, 1, 256), 1, _log(rng, 1, 131072), hq, hk, dim, page, window, sinks)
        else:
            case = _attention(None, op, dtype, rng.choice([1, 1, 2, 3, 4, 8]), _log(rng, 2, 8192),
                              rng.choice([0, 0, 1, 100, _log(rng, 1, 16384)]), hq, hk, dim, page, window, sinks)
        sizes = [case.get("tokens"), case.get("cached"), case.get("new"), case.get("requests"), window]
        if op != "tables":
            sizes += [hq * dim, hk * dim, (hq + hk) * dim, (hq + 2 * hk) * dim]
        if 3072 in sizes or _too_much(case):
            continue
        return case


# ---- inputs ------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, dtype, gen, std=1.0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=gen)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _block_tables(lengths, page, seed, spare=8):
    """(table [requests, width], pages): pages in no order, as a server's cache has them after a while."""
    rng = np.random.default_rng(seed)
    counts = [_cdiv(n, page) for n in lengths]
    pages = sum(counts) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.zeros((len(lengths), max(1, max(counts))), dtype=np.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), pages


def _rope_table(positions, rotary):
    """cos and sin of every position's angles, as a server keeps them."""
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _prepare_tables(case, seed):
    pairs, page = _step(case), case["page"]
    random.Random(seed).shuffle(pairs)
    held = [_cdiv(c, page) for c, _ in pairs]
    width = max(_cdiv(c + max(n, 0), page) for c, n in pairs) + 8
    need = sum(_cdiv(c + max(n, 0), page) - h for (c, n), h in zip(pairs, held))
    pages = sum(held) + need + 64
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.zeros((len(pairs), max(1, width)), dtype=np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    # the ring of free pages: those that no request holds, from wherever the ring stands
    free = order[at:]
    taken = random.Random(seed).randrange(5 * pages)
    ring = np.zeros(pages, dtype=np.int32)
    ring[(taken + np.arange(len(free))) % pages] = free
    total = sum(max(n, 0) for _, n in pairs)
    tokens = _cdiv(max(total, 1), 64) * 64  # (padded, as a captured step's buffers are)
    state = {"cached": _ints([c for c, _ in pairs]), "new": _ints([n for _, n in pairs]),
             "table": torch.from_numpy(table).cuda(), "pool": torch.from_numpy(ring).cuda(),
             "pool_state": _ints([taken, taken + len(free)], torch.int64), "tokens": tokens}
    if own:
        state["lengths"] = torch.empty_like(state["cached"])
        state["pool_state_out"] = torch.empty_like(state["pool_state"])
        state["query_starts"] = torch.empty(len(pairs) + 1, dtype=torch.int32, device="cuda")
        state["positions"] = torch.empty(tokens, dtype=torch.int32, device="cuda")
        state["slots"] = torch.empty(tokens, dtype=torch.int64, device="cuda")
    return state


def _prepare_rope(case, seed):
    gen, dtype, t, hq, hk, d = _gen(seed), DTYPES[case["dtype"]], case["tokens"], case["hq"], case["hk"], case["dim"]
    qkv = _normal((t, (hq + 2 * hk) * d), dtype, gen)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split((hq * d, hk * d, hk * d), 1))
    # tokens of requests that stand somewhere in their contexts
    positions = torch.randint(0, 16384, (t,), device="cuda", dtype=torch.int32, generator=gen)
    cos, sin = _rope_table(16384, case["rotary"])
    state = {"q": q, "k": k, "v": v, "positions": positions, "cos": cos, "sin": sin, "q_weight": None, "k_weight": None}
    if case["norm"]:
        state["q_weight"] = 1 + _normal((d,), dtype, gen, 0.1)
        state["k_weight"] = 1 + _normal((d,), dtype, gen, 0.1)
    if case["op"] == "grad":
        state["dq_out"], state["dk_out"] = _normal((t, hq, d), dtype, gen), _normal((t, hk, d), dtype, gen)
        if own:
            from iris_amd import attention

            dqkv = torch.empty((t, (hq + hk) * d), dtype=dtype, device="cuda")
            state["dq"], state["dk"] = (x.unflatten(1, (-1, d)) for x in dqkv.split((hq * d, hk * d), 1))
            if case["norm"]:
                state["dq_weight"], state["dk_weight"] = (torch.empty(d, device="cuda") for _ in range(2))
                state["workspace"] = attention.make_gradient_workspace(d, device="cuda")
        return state
    if case["cache"]:
        pages = _cdiv(t, case["page"]) + 8
        shape = (pages, case["page"], hk, d)
        state["k_cache"], state["v_cache"] = torch.zeros(shape, dtype=dtype, device="cuda"), torch.zeros(shape, dtype=dtype, device="cuda")
        slots = torch.randperm(pages * case["page"] - 1, device="cuda", generator=gen)[:t].contiguous()
        if t > 8:
            slots[t // 2] = -1  # a padded token: it has no slot
        state["slots"] = slots
    if own:
        state["q_out"] = torch.empty((t, hq, d), dtype=dtype, device="cuda")
        if not case["cache"]:
            state["k_out"] = torch.empty((t, hk, d), dtype=dtype, device="cuda")
    return state


def _prepare_attention(case, seed):
    gen, dtype, hq, hk, d = _gen(seed), DTYPES[case["dtype"]], case["hq"], case["hk"], case["dim"]
    if case["op"] == "decode":
        lengths, news = _contexts(case), None
        random.Random(seed).shuffle(lengths)
        tokens = len(lengths)
    else:
        pairs = _prompts(case)
        random.Random(seed).shuffle(pairs)
        lengths, news = [n + c for n, c in pairs], [n for n, _ in pairs]
        tokens = sum(news)
    table, pages = _block_tables(lengths, case["page"], seed)
    cache = (pages, case["page"], hk, d)
    state = {"case": case, "table": table, "lengths": _ints(lengths), "host_lengths": lengths,
             # queries are larger than one: attention in earnest has few keys with most of the weight
             "q": _normal((tokens, hq, d), dtype, gen, 2.0),
             "k_cache": _normal(cache, dtype, gen), "v_cache": _normal(cache, dtype, gen)}
    if news is not None:
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        state["starts"], state["host_starts"] = _ints(starts), starts
    if own:
        from iris_amd import attention

        state["out"] = torch.empty_like(state["q"])
        state["workspace"] = attention.make_workspace(d, device="cuda")
    return state


def prepare(case, seed):
    if case["op"] == "tables":
        state = _prepare_tables(case, seed)
    elif case["op"] in ("rope", "grad"):
        state = _prepare_rope(case, seed)
    else:
        state = _prepare_attention(case, seed)
    state["case"] = case
    return state


# ---- plain forms -------------------------------------------------------------


def _plain_tables(s):
    page, table, pool = s["case"]["page"], s["table"].long(), s["pool"].long()
    c, n = s["cached"].long(), s["new"].long()
    taken, returned = s["pool_state"][0], s["pool_state"][1]
    ended, add = n < 0, n.clamp(min=0)
    held, want = (c + page - 1) // page, (c + add + page - 1) // page
    fits = (want <= table.shape[1]) & ~ended
    need = torch.where(fits, want - held, 0)
    after = need.cumsum(0)
    served = fits & ((need == 0) | (after <= returned - taken))
    need = torch.where(served, need, 0)
    lengths = torch.where(ended, 0, torch.where(served, c + add, c))
    j = torch.arange(table.shape[1], device=table.device)
    first = (after - torch.where(fits, want - held, 0))[:, None]
    fresh = (j >= held[:, None]) & (j < want[:, None]) & served[:, None]
    new_table = torch.where(fresh, pool[(taken + first + j - held[:, None]) % len(pool)], table)
    back = torch.where(ended, held, 0)
    gone = (j < back[:, None]) & ended[:, None]
    at = (returned + (back.cumsum(0) - back)[:, None] + j) % len(pool)
    new_pool = torch.cat((pool, pool[:1])).scatter(0, torch.where(gone, at, len(pool)).flatten(), table.flatten())[:-1]
    starts = torch.cat((add.new_zeros(1), add.cumsum(0)))
    t = torch.arange(s["tokens"], device=table.device)
    i = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=len(c) - 1)
    live = t < starts[-1]
    position = torch.where(live, c[i] + t - starts[i], 0)
    slot = new_table[i, (position // page).clamp(max=table.shape[1] - 1)] * page + position % page
    slot = torch.where(live & served[i], slot, -1)
    state = torch.stack((taken + need.sum(), returned + back.sum()))
    return {"table": new_table.int(), "pool": new_pool.int(), "pool_state": state, "lengths": lengths.int(),
            "query_starts": starts.int(), "positions": position.int(), "slots": slot}


def _halves(x, rotary, interleaved):
    return (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:rotary])


def _joined(a, b, rest, interleaved):
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, rest), -1)


def _plain_norm_rope(x, weight, cos, sin, interleaved):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    rotary = 2 * cos.shape[-1]
    a, b = _halves(y, rotary, interleaved)
    return _joined(a * cos - b * sin, b * cos + a * sin, y[..., rotary:], interleaved).to(x.dtype)


def _plain_rope(s):
    case = s["case"]
    where = s["positions"].long()
    cos, sin = s["cos"][where][:, None], s["sin"][where][:, None]
    out = {"q": _plain_norm_rope(s["q"], s["q_weight"], cos, sin, case["interleaved"])}
    k = _plain_norm_rope(s["k"], s["k_weight"], cos, sin, case["interleaved"])
    if not case["cache"]:
        return dict(out, k=k)
    for name, rows in (("k_cache", k), ("v_cache", s["v"])):
        flat = s[name].flatten(0, 1)
        # (a padded token's slot is -1: it writes the last one, which no token has and which is put back)
        last = flat[-1].clone()
        flat[s["slots"]] = rows
        flat[-1] = last
    return dict(out, k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_norm_rope_grad(dz, x, weight, cos, sin, interleaved):
    rotary = 2 * cos.shape[-1]
    dz, x32 = dz.float(), x.float()
    a, b = _halves(dz, rotary, interleaved)
    g = _joined(a * cos + b * sin, b * cos - a * sin, dz[..., rotary:], interleaved)
    if weight is None:
        return g.to(x.dtype), None
    r = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS)
    gw = g * weight.float()
    dx = r * gw - x32 * (r * r * r) * (gw * x32).mean(-1, keepdim=True)
    return dx.to(x.dtype), (g * x32 * r).sum((0, 1))


def _plain_grad(s):
    where = s["positions"].long()
    cos, sin = s["cos"][where][:, None], s["sin"][where][:, None]
    turned = s["case"]["interleaved"]
    dq, dqw = _plain_norm_rope_grad(s["dq_out"], s["q"], s["q_weight"], cos, sin, turned)
    dk, dkw = _plain_norm_rope_grad(s["dk_out"], s["k"], s["k_weight"], cos, sin, turned)
    out = {"dq": dq, "dk": dk}
    return dict(out, dq_weight=dqw, dk_weight=dkw) if s["case"]["norm"] else out


def _softmax_rows(scores, mask):
    """Rows of weights; zeros where the mask leaves nothing."""
    scores = scores.masked_fill(~mask, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _seen(at, key, window, sinks):
    mask = (key <= at) & (at >= 0)
    return mask & ((at - key < window) | (key < sinks)) if window else mask


def _plain_decode(s):
    case, q, table = s["case"], s["q"], s["table"].long()
    hq, hk, d = case["hq"], case["hk"], case["dim"]
    n = len(q)
    k, v = (c[table].flatten(1, 2).float() for c in (s["k_cache"], s["v_cache"]))  # [requests, keys, hk, d]
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    rows = q.float().view(n, hk, hq // hk, d)
    scores = torch.matmul(k, rows.transpose(2, 3).contiguous()).transpose(2, 3) * (1.0 / math.sqrt(d))
    at = (s["lengths"].long() - 1)[:, None, None, None]
    key = torch.arange(k.shape[2], device=q.device)
    p = _softmax_rows(scores, _seen(at, key, case["window"], case["sinks"]))
    return torch.matmul(p, v).view(n, hq, d).to(q.dtype)


def _plain_prompt(s):
    case, q = s["case"], s["q"]
    hq, hk, d, page = case["hq"], case["hk"], case["dim"], case["page"]
    out = torch.empty_like(q)
    for i, length in enumerate(s["host_lengths"]):
        lo, hi = s["host_starts"][i], s["host_starts"][i + 1]
        if lo == hi:
            continue
        pages = s["table"][i, :_cdiv(length, page)].long()
        k, v = (c[pages].flatten(0, 1)[:length].float().transpose(0, 1) for c in (s["k_cache"], s["v_cache"]))
        key = torch.arange(length, device=q.device)
        mask = _seen(torch.arange(length - (hi - lo), length, device=q.device)[:, None], key, case["window"], case["sinks"])
        rows = q[lo:hi].float().view(hi - lo, hk, hq // hk, d).permute(1, 2, 0, 3)
        for h in range(hk):
            p = _softmax_rows(torch.matmul(rows[h], k[h].T) * (1.0 / math.sqrt(d)), mask)
            out[lo:hi, h * (hq // hk):(h + 1) * (hq // hk)] = torch.matmul(p, v[h]).transpose(0, 1).to(q.dtype)
    return out


# ---- the passes --------------------------------------------------------------


def _own(s):
    from iris_amd import attention

    case, op = s["case"], s["case"]["op"]
    if op == "tables":
        attention.build_block_tables(s["cached"], s["new"], s["table"], s["pool"], s["pool_state"], case["page"],
                                     lengths=s["lengths"], pool_state_out=s["pool_state_out"],
                                     query_starts=s["query_starts"], positions=s["positions"], slots=s["slots"])
        return {"table": s["table"], "pool": s["pool"], "pool_state": s["pool_state_out"], "lengths": s["lengths"],
                "query_starts": s["query_starts"], "positions": s["positions"], "slots": s["slots"]}
    if op == "rope":
        if not case["cache"]:
            attention.qk_norm_rope(s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["q_out"], s["k_out"],
                                   q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, interleaved=case["interleaved"])
            return {"q": s["q_out"], "k": s["k_out"]}
        attention.qk_norm_rope(s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["q_out"], None, q_weight=s["q_weight"],
                               k_weight=s["k_weight"], eps=EPS, interleaved=case["interleaved"], v=s["v"],
                               k_cache=s["k_cache"], v_cache=s["v_cache"], slots=s["slots"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "grad":
        attention.qk_norm_rope_backward(s["dq_out"], s["dk_out"], s["q"], s["k"], s["positions"], s["cos"], s["sin"],
                                        s["dq"], s["dk"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                                        dq_weight=s.get("dq_weight"), dk_weight=s.get("dk_weight"), eps=EPS,
                                        interleaved=case["interleaved"], workspace=s.get("workspace"))
        out = {"dq": s["dq"], "dk": s["dk"]}
        return dict(out, dq_weight=s["dq_weight"], dk_weight=s["dk_weight"]) if case["norm"] else out
    if op == "decode":
        attention.decode_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["out"],
                                   window=case["window"], sinks=case["sinks"], workspace=s["workspace"])
    else:
        attention.prompt_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["starts"], s["out"],
                                   window=case["window"], sinks=case["sinks"], workspace=s["workspace"])
    return s["out"]


_PLAIN = {"tables": _plain_tables, "rope": _plain_rope, "grad": _plain_grad, "decode": _plain_decode, "prompt": _plain_prompt}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "tables":
        pairs, page = _step(case), case["page"]
        tokens = sum(max(n, 0) for _, n in pairs)
        moved = sum(_cdiv(c + max(n, 0), page) - _cdiv(c, page) if n >= 0 else _cdiv(c, page) for c, n in pairs)
        # lengths in and out, starts; a page taken or given back is read and written; position and slot of a token
        return {"bytes": 16 * len(pairs) + 8 * moved + 12 * tokens + 32, "flops": 0}
    e, d, hq, hk = SIZES[case["dtype"]], case["dim"], case["hq"], case["hk"]
    if op in ("rope", "grad"):
        t = case["tokens"]
        angles = min(t, 16384) * case["rotary"] * 4 + 4 * t
        if op == "rope":
            heads = hq + hk + (hk if case["cache"] else 0)
            return {"bytes": 2 * t * heads * d * e + angles + (8 * t if case["cache"] else 0), "flops": 10 * t * (hq + hk) * d}
        return {"bytes": 3 * t * (hq + hk) * d * e + angles, "flops": 20 * t * (hq + hk) * d}
    window, sinks = case["window"], case["sinks"]
    if op == "decode":
        keys = pairs = sum(_visible(n, window, sinks) for n in _contexts(case))
        tokens = case["requests"]
    else:
        both = _prompts(case)
        keys = sum(_reach(n, c, window, sinks) for n, c in both)
        pairs = sum(sum(_visible(c + i + 1, window, sinks) for i in range(n)) for n, c in both)
        tokens = sum(n for n, _ in both)
    return {"bytes": 2 * keys * hk * d * e + 2 * tokens * hq * d * e + 4 * _cdiv(keys, case["page"]), "flops": 4 * pairs * hq * d}


# ---- the definitions in 64 bits ----------------------------------------------


def _exact_tables(s):
    page, tokens = s["case"]["page"], s["tokens"]
    cached, new = s["cached"].tolist(), s["new"].tolist()
    table, pool = s["table"].cpu().numpy().copy(), s["pool"].cpu().numpy().copy()
    taken, returned = s["pool_state"].tolist()
    ring, free, first_free, wanted = pool.copy(), returned - taken, taken, 0
    lengths, starts, positions, slots = [], [0], [], []
    for i, (c, n) in enumerate(zip(cached, new)):
        held = -(-c // page)
        if n < 0:
            for j in range(held):
                pool[returned % len(pool)] = table[i, j]
                returned += 1
            lengths.append(0)
            starts.append(starts[-1])
            continue
        need = -(-(c + n) // page) - held
        served = held + need <= table.shape[1]
        if served and need:
            wanted += need
            served = wanted <= free
        if served:
            for j in range(need):
                table[i, held + j] = ring[taken % len(ring)]
                taken += 1
        lengths.append(c + n if served else c)
        starts.append(starts[-1] + n)
        for p in range(c, c + n):
            positions.append(p)
            slots.append(int(table[i, p // page]) * page + p % page if served else -1)
    positions += [0] * (tokens - len(positions))
    slots += [-1] * (tokens - len(slots))
    return {"table": torch.from_numpy(table), "pool": torch.from_numpy(pool),
            "pool_state": torch.tensor([taken, returned]), "lengths": torch.tensor(lengths, dtype=torch.int32),
            "query_starts": torch.tensor(starts, dtype=torch.int32),
            "positions": torch.tensor(positions[:tokens], dtype=torch.int32), "slots": torch.tensor(slots[:tokens])}


def _turn(x, positions, s):
    """Each pair of coordinates as a complex number, times the position's unit number."""
    rotary = 2 * s["cos"].shape[1]
    unit = torch.complex(s["cos"].double(), s["sin"].double())[positions][:, None, :]
    if s["case"]["interleaved"]:
        z = torch.view_as_complex(x[..., :rotary].unflatten(-1, (-1, 2)).contiguous()) * unit
        turned = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :rotary // 2].contiguous(), x[..., rotary // 2:rotary].contiguous()) * unit
        turned = torch.cat((z.real, z.imag), -1)
    return torch.cat((turned, x[..., rotary:]), -1)


def _normed(x, weight):
    if weight is None:
        return x
    return x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight


def _exact_rope(s):
    where = s["positions"].long()
    wide = [None if w is None else w.double() for w in (s["q_weight"], s["k_weight"])]
    q = _turn(_normed(s["q"].double(), wide[0]), where, s)
    k = _turn(_normed(s["k"].double(), wide[1]), where, s)
    if not s["case"]["cache"]:
        return {"q": q, "k": k}
    caches = {"q": q, "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
    kept = [t for t, slot in enumerate(s["slots"].tolist()) if slot >= 0]
    slots, kept = s["slots"][kept], torch.tensor(kept, device="cuda")
    page = s["case"]["page"]
    caches["k_cache"][slots // page, slots % page] = k[kept]
    caches["v_cache"][slots // page, slots % page] = s["v"].double()[kept]
    return caches


def _exact_grad(s):
    where, out = s["positions"].long(), {}
    for name in ("q", "k"):
        x = s[name].double().requires_grad_()
        w = s[name + "_weight"]
        w = None if w is None else w.double().requires_grad_()
        with torch.enable_grad():
            z = _turn(_normed(x, w), where, s)
            grads = torch.autograd.grad(z, [x] if w is None else [x, w], s[f"d{name}_out"].double())
        out["d" + name] = grads[0]
        if w is not None:
            out[f"d{name}_weight"] = grads[1]
    return out


def _exact_attention(s):
    case = s["case"]
    hq, hk, d, page, window, sinks = (case[n] for n in ("hq", "hk", "dim", "page", "window", "sinks"))
    starts = s.get("host_starts") or list(range(len(s["host_lengths"]) + 1))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(s["host_lengths"]):
        lo, hi = starts[i], starts[i + 1]
        if length == 0 or lo == hi:
            continue
        t = torch.arange(length, device="cuda")
        where = s["table"][i].long()[t // page], t % page
        at = torch.arange(hi - lo, device="cuda") + length - (hi - lo)
        hidden = t[None, :] > at[:, None]
        if window:
            hidden |= (t[None, :] <= at[:, None] - window) & (t[None, :] >= sinks)
        for h in range(hk):
            k, v = s["k_cache"][where[0], where[1], h].double(), s["v_cache"][where[0], where[1], h].double()
            for g in range(h * (hq // hk), (h + 1) * (hq // hk)):
                scores = s["q"][lo:hi, g].double() @ k.T / math.sqrt(d)
                scores[hidden] = -math.inf
                out[lo:hi, g] = torch.softmax(scores, -1) @ v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "tables":
        return _exact_tables(state)
    if case["op"] == "rope":
        return _exact_rope(state)
    if case["op"] == "grad":
        return _exact_grad(state)
    return _exact_attention(state)
