"""A key-value cache in 8 bits, as cases to be timed.

A server that keeps its cache in 8 bits has room for twice the context and reads
half the bytes a step.  The cache holds codes (8-bit floats) and, for
each block of tokens and key head, a scale that is a power of two:

* ``write``    keys and values of new tokens are quantised into their slots of the cache;
* ``read``     cached tokens are read back, as 16-bit or fp32 heads;
* ``decode``   attention of one new token a request over the cache;
* ``prompt``   attention of many new tokens a request over the cache.

The scale of a block is the smallest power of two (2^-100 at least) by which the largest of its values
fits the codes.  Tokens that come to a block later may make its scale grow, and then the codes that are there are
rounded to the new one; it shrinks when the block is begun anew.

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
CODES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
# (the largest code is 0.875 times this power of two)
TOP = {"e4m3": 9, "e5m2": 16}
LEAST = -100  # exponent of the smallest scale


def _case(name, op, dtype, code, requests, new, cached, hq, hk, dim, page, block, window=0, sinks=0):
    """``requests`` requests: up to ``new`` tokens behind up to ``cached`` in the cache (decode: contexts of up to ``cached``;
    read: the last ``new`` tokens at most of up to ``cached``)."""
    case = {"op": op, "dtype": dtype, "code": code, "requests": requests, "new": new, "cached": cached, "hq": hq, "hk": hk,
            "dim": dim, "page": page, "block": block, "window": window, "sinks": sinks}
    return dict(case, name=name) if name else case


def listed():
    return [
        # A decode step's tokens of 64 requests, one key head of 128 (one rank of eight): latency of one small launch.
        _case("write_step", "write", "bf16", "e4m3", 64, 1, 8192, 8, 1, 128, 16, 16),
        # A batch of prompts of odd lengths, some behind tokens that are cached, eight key heads.
        _case("write_prompts", "write", "bf16", "e4m3", 4, 4096, 999, 16, 8, 128, 16, 16),
        # fp32, the other code, an odd head size, long blocks: a scale for a whole page of 64 tokens.
        _case("write_fp32", "write", "fp32", "e5m2", 3, 500, 1000, 6, 6, 80, 64, 64),
        # One request's context of odd length read back, 4 heads of 128.
        _case("read_one", "read", "bf16", "e4m3", 1, 1999, 1999, 4, 4, 128, 16, 16),
        # The prefixes of 16 requests, as they are handed to a server whose cache is in 16 bits.
        _case("read_prefixes", "read", "fp16", "e5m2", 16, 16384, 16384, 2, 2, 128, 64, 32),
        # One request of odd length, 4 heads of their own keys: the smallest call of a server.
        _case("decode_one", "decode", "bf16", "e4m3", 1, 1, 1999, 4, 4, 128, 16, 16),
        # A batch of requests of very different lengths, eight query heads to one key head (one rank of eight).
        _case("decode_batch", "decode", "bf16", "e4m3", 64, 1, 8192, 8, 1, 128, 16, 16),
        # Long contexts: the whole cache of a few requests is read once.
        _case("decode_long", "decode", "fp16", "e4m3", 16, 1, 131072, 8, 2, 128, 64, 64),
        # A layer with a sliding window and visible first tokens, many requests, the other code.
        _case("decode_window", "decode", "bf16", "e5m2", 128, 1, 16384, 8, 2, 64, 32, 16, window=1024, sinks=4),
        # Pieces of a few tokens behind cached ones.
        _case("prompt_pieces", "prompt", "bf16", "e4m3", 8, 30, 4000, 8, 1, 128, 16, 16),
        # Prompts and pieces of prompts behind cached tokens, causal.
        _case("prompt_causal", "prompt", "bf16", "e4m3", 4, 8192, 2048, 8, 1, 128, 16, 16),
        # Prompts through a layer with a sliding window and visible first tokens, ten heads of 64.
        _case("prompt_window", "prompt", "fp16", "e4m3", 4, 8192, 1000, 10, 2, 64, 32, 32, window=1024, sinks=4),
    ]


# ---- sizes -------------------------------------------------------------------


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cdiv(a, b):
    return (a + b - 1) // b


def _spans(case):
    """(length, new) of each request: its tokens, and how many of the last are written, read or asked about."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    count, new, cached = case["requests"], case["new"], case["cached"]
    if case["op"] == "decode":
        lengths = [_log(rng, max(1, cached // 64), cached) for _ in range(count)]
        lengths[0] = cached
        if count >= 8:
            lengths[1], lengths[2] = 0, 1  # an idle slot, a first token
        return [(n, 1) for n in lengths]
    if case["op"] == "read":
        lengths = [cached] + [_log(rng, max(1, cached // 16), cached) for _ in range(count - 1)]
        return [(n, min(n, new)) for n in lengths]
    pairs = [(_log(rng, max(1, new // 16), new), rng.randint(0, cached)) for _ in range(count)]
    pairs[0] = (new, 0 if new > 1 else cached)
    if count >= 4:
        pairs[1] = (1, cached)  # a request that decodes beside the prompts
    return [(n + c, n) for n, c in pairs]


def _visible(length, window, sinks):
    """Keys that the token at position length - 1 sees."""
    if length <= 0 or not window or length <= window:
        return max(length, 0)
    return window + min(sinks, length - window)


def _reach(new, cached, window, sinks):
    """Keys that any of ``new`` tokens behind ``cached`` sees."""
    lo = max(0, cached + 1 - window) if window else 0
    return cached + new - lo + min(sinks, lo)


def work(case):
    spans, e, hq, hk, d = _spans(case), SIZES[case["dtype"]], case["hq"], case["hk"], case["dim"]
    tokens = sum(n for _, n in spans)
    if case["op"] in ("write", "read"):
        blocks = sum(_cdiv(length, case["block"]) - (length - n) // case["block"] for length, n in spans)
        # heads in 8 bits on one side and whole on the other, a scale a block, a slot or a page's number
        index = 8 * tokens if case["op"] == "write" else 4 * _cdiv(tokens, case["page"])
        return {"bytes": 2 * tokens * hk * d * (1 + e) + 2 * blocks * hk + index, "flops": 2 * tokens * hk * d}
    window, sinks = case["window"], case["sinks"]
    keys = sum(_reach(n, length - n, window, sinks) if length else 0 for length, n in spans)
    pairs = sum(sum(_visible(length - n + i + 1, window, sinks) for i in range(n)) for length, n in spans)
    scales = 2 * _cdiv(keys, case["block"]) * hk
    return {"bytes": 2 * keys * hk * d + scales + 2 * tokens * hq * d * e + 4 * _cdiv(keys, case["page"]), "flops": 4 * pairs * hq * d}


_MOST_BYTES, _MOST_FLOPS, _MOST_PADDED = 3.1e8, 1.5e11, 16 * 131072 * 2 * 128


def _too_much(case):
    w = work(case)
    if w["bytes"] > _MOST_BYTES or w["flops"] > _MOST_FLOPS:
        return True
    if case["op"] == "decode":
        return case["requests"] * case["cached"] * case["hk"] * case["dim"] > _MOST_PADDED
    if case["op"] == "prompt":
        return sum(n * length for length, n in _spans(case)) * case["hq"] > 8e9
    return sum(length for length, _ in _spans(case)) * case["hk"] * case["dim"] > 2.5e8


def draw(rng):
    while True:
        op = rng.choices(["write", "read", "decode", "prompt"], [25, 15, 35, 25])[0]
        dtype = rng.choices(["bf16", "fp16", "fp32"], [50, 30, 20])[0]
        code = rng.choices(["e4m3", "e5m2"], [70, 30])[0]
        dim = rng.choices([64, 80, 96, 128, 192, 256], [25, 8, 10, 40, 7, 10])[0]
        hk = rng.choice([1, 1, 2, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 8, 12, 16])
        page = rng.choices([16, 32, 48, 64, 128, 256], [30, 25, 7, 20, 10, 8])[0]
        block = rng.choice([b for b in (16, 32, 48, 64, 128, 256) if page % b == 0])
        window = rng.choice([0, 0, 0, _log(rng, 16, 8192)])
        sinks = rng.choice([0, 1, 4, 16, 100]) if window else 0
        if op == "decode":
            case = _case(None, op, dtype, code, _log(rng, 1, 256), 1, _log(rng, 1, 131072), hq, hk, dim, page, block, window, sinks)
        elif op == "prompt":
            case = _case(None, op, dtype, code, rng.choice([1, 1, 2, 3, 4, 8]), _log(rng, 2, 8192),
                         rng.choice([0, 0, 1, 100, _log(rng, 1, 16384)]), hq, hk, dim, page, block, window, sinks)
        elif op == "read":
            cached = _log(rng, 1, 32768)
            case = _case(None, op, dtype, code, _log(rng, 1, 64), rng.choice([cached, _log(rng, 1, cached)]), cached, hk, hk, dim, page, block)
        else:
            new = rng.choice([1, _log(rng, 1, 8192)])
            case = _case(None, op, dtype, code, _log(rng, 1, 256 if new == 1 else 16), new, rng.choice([0, _log(rng, 1, 8192)]), hk, hk, dim,
                         page, block)
        if not _too_much(case):
            return case


# ---- inputs ------------------------------------------------------------------


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _block_tables(lengths, page, seed, spare=8):
    """(table [requests, width], pages): pages in no order, as a server's cache has them after a while."""
    counts = [_cdiv(n, page) for n in lengths]
    pages = sum(counts) + spare
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.zeros((len(lengths), max(1, max(counts))), dtype=np.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    spans, dtype, page, block = _spans(case), DTYPES[case["dtype"]], case["page"], case["block"]
    hq, hk, d, op = case["hq"], case["hk"], case["dim"], case["op"]
    random.Random(seed).shuffle(spans)
    lengths, news = [n for n, _ in spans], [n for _, n in spans]
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    tokens = starts[-1]
    table, pages = _block_tables(lengths, page, seed)
    state = {"case": case, "table": table, "lengths": _ints(lengths), "host_lengths": lengths, "starts": _ints(starts), "host_starts": starts}

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen)

    # Values of about one: codes of about a quarter of the largest, scales that bring them back, a power of two more or less apart.
    shift = 7 if case["code"] == "e4m3" else 14
    for name in ("k", "v"):
        codes = torch.empty((pages, page, hk, d), dtype=CODES[case["code"]], device="cuda")
        for p in range(0, pages, 4096):  # (a piece at a time: the codes are a quarter of what they are made from)
            some = normal(min(4096, pages - p), page, hk, d, std=2.0 ** (shift - 1))
            codes[p:p + 4096] = some.clamp_(-0.875 * 2 ** TOP[case["code"]], 0.875 * 2 ** TOP[case["code"]]).to(codes.dtype)
        power = torch.randint(127 - shift, 129 - shift, (pages, page // block, hk), device="cuda", generator=gen)
        state[name + "_cache"], state[name + "_scales"] = codes, power.to(torch.uint8).view(torch.float8_e8m0fnu)
    if op == "write":
        # A fused projection's output; now and then a token is larger than those before it.
        padded = _cdiv(tokens, 16) * 16 if tokens > 8 else tokens
        qkv = normal(padded, (hq + 2 * hk) * d) * torch.exp(0.7 * normal(padded, 1))
        qkv = qkv.to(dtype)
        _, state["k"], state["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split((hq * d, hk * d, hk * d), 1))
        request = torch.repeat_interleave(torch.arange(len(news), device="cuda"), _ints(news, torch.int64))
        at = state["lengths"].long()[request] - state["starts"].long()[request + 1] + torch.arange(tokens, device="cuda")
        slots = table.long()[request, at // page] * page + at % page
        # a captured step's buffers are padded: behind the last token are some that have no slot
        state["slots"] = torch.cat((slots, torch.full((padded - tokens,), -1, device="cuda")))
    elif op == "read":
        if own:
            state["k_out"], state["v_out"] = (torch.empty((tokens, hk, d), dtype=dtype, device="cuda") for _ in range(2))
    else:
        # queries are larger than one: attention in earnest has few keys with most of the weight
        state["q"] = normal(tokens, hq, d, std=2.0).to(dtype)
        if own:
            from iris_amd import attention

            state["out"] = torch.empty_like(state["q"])
            state["workspace"] = attention.make_workspace(d, device="cuda")
    return state


# ---- plain forms -------------------------------------------------------------


def _powers(scales):
    """Scales in 32 bits: their bytes are the exponents of fp32 numbers."""
    return (scales.view(torch.uint8).int() << 23).view(torch.float32)


def _gathered(codes, where):
    # (8-bit floats are looked up as bytes)
    return codes.view(torch.uint8)[where].view(codes.dtype)


def _two_to(n):
    return ((n + 127) << 23).view(torch.float32)


def _write_one(x, cache, scales, s):
    case = s["case"]
    block, hk, d = case["block"], case["hk"], case["dim"]
    codes, powers = cache.view(-1, block, hk, d), scales.view(torch.uint8).view(-1, hk)
    starts = s["starts"].long()
    # (a padded token does again what the first token does)
    t = torch.arange(len(s["slots"]), device=x.device)
    source = torch.where(s["slots"] >= 0, t, 0)
    slots = s["slots"][source]
    into, row = slots // block, slots % block
    x32 = x.float()
    # the largest value that comes to each block, and the smallest scale that holds it
    most = torch.zeros((len(codes), hk), device=x.device)
    most.scatter_reduce_(0, into[:, None].expand(-1, hk), x32.abs().amax(-1)[source], "amax")
    fraction, exponent = torch.frexp(most)
    wanted = (exponent - TOP[case["code"]] + (fraction > 0.875).int()).clamp(min=LEAST)
    # a block that holds earlier tokens keeps its scale or takes a larger one: a request's first new tokens may come to such a one
    first = slots[starts[:-1]]
    blocks, older = first // block, first % block
    before = powers.int() - 127
    begun = torch.zeros(len(codes), dtype=torch.bool, device=x.device)
    begun[into] = True
    kept = ~begun
    kept[blocks] = older > 0
    now = torch.where(begun[:, None], wanted, before)
    now = torch.where(kept[:, None], torch.maximum(now, before), now)
    # its older rows, at the scale that the block has from now on
    old = _gathered(codes, blocks)
    again = (old.float() * _two_to(before[blocks] - now[blocks])[:, None, :, None]).to(cache.dtype)
    mine = torch.arange(block, device=x.device) < older[:, None]
    flat = codes.view(torch.uint8)
    flat[blocks] = torch.where(mine[:, :, None, None], again.view(torch.uint8), old.view(torch.uint8))
    new = (x32 * _two_to(-now[into])[..., None]).to(cache.dtype)
    flat.view(-1, hk, d)[slots] = new.view(torch.uint8)[source]
    powers[:] = (now + 127).to(torch.uint8)


def _plain_write(s):
    out = {}
    for name in ("k", "v"):
        cache, scales = s[name + "_cache"], s[name + "_scales"]
        _write_one(s[name], cache, scales, s)
        out[name + "_cache"], out[name + "_scales"] = cache, scales.view(torch.uint8)
    return out


def _where(s, request, at):
    """Page, row and block of positions ``at`` of a request (tensors of one shape)."""
    page = s["case"]["page"]
    return s["table"].long()[request, at // page], at % page, at % page // s["case"]["block"]


def _plain_read(s):
    dtype = DTYPES[s["case"]["dtype"]]
    t = torch.arange(s["host_starts"][-1], device="cuda")
    request = torch.searchsorted(s["starts"][1:].contiguous(), t.int(), right=True)
    at = s["lengths"].long()[request] - s["starts"].long()[request + 1] + t
    page, row, block = _where(s, request, at)
    out = {}
    for name in ("k", "v"):
        scale = _powers(s[name + "_scales"])[page, block][..., None]
        out[name] = (_gathered(s[name + "_cache"], (page, row)).float() * scale).to(dtype)
    return out


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


def _cached(s, name, pages):
    """The heads of pages (a tensor of their numbers), in 32 bits: [..., keys, hk, d]."""
    block = s["case"]["block"]
    codes = _gathered(s[name + "_cache"], pages).float().unflatten(-3, (-1, block))
    heads = codes * _powers(s[name + "_scales"])[pages][..., None, :, None]
    return heads.flatten(-5, -3)


def _plain_decode(s):
    case, q = s["case"], s["q"]
    hq, hk, d = case["hq"], case["hk"], case["dim"]
    k, v = (_cached(s, name, s["table"].long()).transpose(1, 2).contiguous() for name in ("k", "v"))  # [requests, hk, keys, d]
    rows = q.float().view(len(q), hk, hq // hk, d)
    scores = torch.matmul(k, rows.transpose(2, 3).contiguous()).transpose(2, 3) * (1.0 / math.sqrt(d))
    at = (s["lengths"].long() - 1)[:, None, None, None]
    key = torch.arange(k.shape[2], device=q.device)
    p = _softmax_rows(scores, _seen(at, key, case["window"], case["sinks"]))
    return torch.matmul(p, v).view(len(q), hq, d).to(q.dtype)


def _plain_prompt(s):
    case, q = s["case"], s["q"]
    hq, hk, d, page = case["hq"], case["hk"], case["dim"], case["page"]
    out = torch.empty_like(q)
    for i, length in enumerate(s["host_lengths"]):
        lo, hi = s["host_starts"][i], s["host_starts"][i + 1]
        if lo == hi:
            continue
        pages = s["table"][i, :_cdiv(length, page)].long()
        k, v = (_cached(s, name, pages)[:length].transpose(0, 1) for name in ("k", "v"))
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
    if op == "write":
        attention.write_quantized_cache(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["slots"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scales": s["k_scales"].view(torch.uint8),
                "v_scales": s["v_scales"].view(torch.uint8)}
    if op == "read":
        attention.read_quantized_cache(s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["table"], s["lengths"], s["starts"],
                                       s["k_out"], s["v_out"])
        return {"k": s["k_out"], "v": s["v_out"]}
    if op == "decode":
        attention.decode_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["out"], window=case["window"],
                                   sinks=case["sinks"], workspace=s["workspace"], k_scales=s["k_scales"], v_scales=s["v_scales"])
    else:
        attention.prompt_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["starts"], s["out"],
                                   window=case["window"], sinks=case["sinks"], workspace=s["workspace"], k_scales=s["k_scales"],
                                   v_scales=s["v_scales"])
    return s["out"]


_PLAIN = {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "prompt": _plain_prompt}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- the definitions in 64 bits ----------------------------------------------


def _power(n):
    """2^n in 64 bits, exactly."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _nearest(x, code):
    """x rounded to the codes' numbers: three (two) places behind the first, the last one even at a tie, subnormal ones alike."""
    places, lowest = (3, -6) if code == "e4m3" else (2, -14)
    step = _power((torch.frexp(x)[1] - 1).clamp(min=lowest) - places)
    return torch.round(x / step) * step


def _exact_write(s):
    case = s["case"]
    page, block, code = case["page"], case["block"], case["code"]
    largest = 0.875 * 2.0 ** TOP[code]
    out = {}
    for name in ("k", "v"):
        codes = s[name + "_cache"].double()
        power = s[name + "_scales"].view(torch.uint8).long() - 127
        x = s[name].double()
        slots, t = s["slots"].tolist(), 0
        while t < len(slots):
            if slots[t] < 0:
                t += 1
                continue
            end = t + 1
            while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % block:
                end += 1
            p, b, r = slots[t] // page, slots[t] % page // block, slots[t] % block
            rows = codes[p, b * block:(b + 1) * block]  # (a view)
            most = x[t:end].abs().amax((0, 2))
            need = torch.full_like(power[p, b], LEAST)
            for off in (1, 0, -1):  # the smallest that holds it, next to where the logarithm says
                near = torch.ceil(torch.log2(most.clamp(min=1e-300) / largest)).long() + off
                holds = largest * _power(near.clamp(min=-1000)) >= most
                need = torch.where(holds & (near >= LEAST), near, need)
            now = torch.maximum(need, power[p, b]) if r else need
            if r:
                rows[:r] = _nearest(rows[:r] * _power(power[p, b] - now)[None, :, None], code)
            rows[r:r + end - t] = _nearest(x[t:end] * _power(-now)[None, :, None], code)
            power[p, b] = now
            t = end
        out[name + "_cache"], out[name + "_scales"] = codes, (power + 127).to(torch.uint8)
    return out


def _positions(s, i):
    """Page, row and block of every token of request i."""
    t = torch.arange(s["host_lengths"][i], device="cuda")
    page = s["case"]["page"]
    return s["table"][i].long()[t // page], t % page, t % page // s["case"]["block"]


def _heads(s, name, i):
    page, row, block = _positions(s, i)
    return s[name + "_cache"].double()[page, row] * _power(s[name + "_scales"].view(torch.uint8).long()[page, block][..., None] - 127)


def _exact_read(s):
    starts = s["host_starts"]
    out = {"k": [], "v": []}
    for i in range(len(s["host_lengths"])):
        for name in out:
            out[name].append(_heads(s, name, i)[s["host_lengths"][i] - (starts[i + 1] - starts[i]):])
    return {name: torch.cat(rows) for name, rows in out.items()}


def _exact_attention(s):
    case = s["case"]
    hq, hk, d, window, sinks = (case[n] for n in ("hq", "hk", "dim", "window", "sinks"))
    starts = s["host_starts"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    wide = {n: s[n + "_cache"].double() for n in ("k", "v")}
    for i, length in enumerate(s["host_lengths"]):
        lo, hi = starts[i], starts[i + 1]
        if length == 0 or lo == hi:
            continue
        page, row, block = _positions(s, i)
        t = torch.arange(length, device="cuda")
        at = torch.arange(hi - lo, device="cuda") + length - (hi - lo)
        hidden = t[None, :] > at[:, None]
        if window:
            hidden |= (t[None, :] <= at[:, None] - window) & (t[None, :] >= sinks)
        for h in range(hk):
            k, v = (wide[n][page, row, h] * _power(s[n + "_scales"].view(torch.uint8).long()[page, block, h][:, None] - 127) for n in ("k", "v"))
            for g in range(h * (hq // hk), (h + 1) * (hq // hk)):
                scores = s["q"][lo:hi, g].double() @ k.T / math.sqrt(d)
                scores[hidden] = -math.inf
                out[lo:hi, g] = torch.softmax(scores, -1) @ v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "write":
        return _exact_write(state)
    if case["op"] == "read":
        return _exact_read(state)
    return _exact_attention(state)
