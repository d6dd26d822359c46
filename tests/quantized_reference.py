"""A key-value cache in 8 bits by its definition, in 64 bits on the CPU; and attention problems over one."""

import math

import torch

from test_paged_attention_gpu import Problem

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
LARGEST = {E4M3: 448.0, E5M2: 57344.0}
NOT_A_NUMBER, LEAST = 255, -100


def nearest(x, code):
    """x (64 bits) rounded to the numbers of a code, ties to even; what is past them is not met here."""
    places, lowest = (3, -6) if code == E4M3 else (2, -14)
    exponent = (torch.frexp(x)[1] - 1).clamp(min=lowest)
    step = torch.ldexp(torch.ones_like(x), exponent - places)  # (of the CPU: exact)
    return torch.round(x / step) * step


def scale_exponent(x, code):
    """The exponent of the smallest scale that the finite elements of x fit."""
    most = x[torch.isfinite(x)].abs().max().item() if torch.isfinite(x).any() else 0.0
    e = LEAST
    while LARGEST[code] * 2.0 ** e < most:
        e += 1
    return e


class Cache:
    """Numbers of codes [slots, heads, dim] and bytes of scales [blocks, heads] of K or of V."""

    def __init__(self, codes, scales, block, code):
        self.numbers = codes.cpu().double().flatten(0, 1).clone()
        self.bytes = scales.cpu().view(torch.uint8).flatten(0, 1).int().clone()
        self.block, self.code = block, code

    def write(self, x, slots):
        x, slots, t = x.cpu().double(), slots.tolist(), 0
        while t < len(slots):
            if not 0 <= slots[t] < len(self.numbers):
                t += 1
                continue
            end = t + 1
            while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % self.block:
                end += 1
            b, older = divmod(slots[t], self.block)
            for h in range(x.shape[1]):
                new = x[t:end, h]
                now, was = scale_exponent(new, self.code) + 127, int(self.bytes[b, h])
                if older:
                    now = max(now, was)
                    if now != was:
                        old = self.numbers[b * self.block:slots[t], h]
                        self.numbers[b * self.block:slots[t], h] = nearest(old * 2.0 ** (was - now), self.code)
                codes = nearest(new * 2.0 ** (127 - now), self.code)
                self.numbers[slots[t]:slots[t] + end - t, h] = torch.where(torch.isfinite(new), codes, math.nan)
                self.bytes[b, h] = now
            while end < len(slots) and 0 <= slots[end] < len(self.numbers) and slots[end] // self.block == b:
                end += 1  # (reported, and skipped)
            t = end

    def elements(self):
        scale = torch.ldexp(torch.ones(self.bytes.shape, dtype=torch.float64), self.bytes - 127)
        scale[self.bytes == NOT_A_NUMBER] = math.nan
        return self.numbers * scale.repeat_interleave(self.block, 0)[..., None]


def same(got, want):
    """Whether a cache's numbers are what they should be (64 bits, NaN where NaN)."""
    got = got.cpu().double().flatten(0, 1)
    return bool(((got == want) | (got.isnan() & want.isnan())).all())


class Quantized(Problem):
    """A problem whose keys and values are what a cache in 8 bits holds; its other places are no numbers, and neither are their scales."""

    def __init__(self, lengths, news, hq, hk, d, dtype, page, *, code=E4M3, block=None, spread=0.0, strided=False, **kw):
        super().__init__(lengths, news, hq, hk, d, dtype, page, **kw)
        block = block or page
        pages = self.k_cache.shape[0]
        table, gen = self.table.cpu(), torch.Generator().manual_seed(kw.get("seed", 0) + 1)
        for name in ("k", "v"):
            shape = (pages, hk, page, d) if kw.get("heads_first") else (pages, page, hk, d)
            codes = torch.full(shape, math.nan).to(code)
            view = codes.transpose(1, 2) if kw.get("heads_first") else codes
            scales = torch.full((pages, page // block, hk), NOT_A_NUMBER, dtype=torch.uint8)
            rows = getattr(self, name)
            for i, n in enumerate(lengths):
                held = rows[i].double()
                for at in range(0, n, block):
                    where = int(table[i, at // page])
                    for h in range(hk):
                        x = rows[i][at:at + block, h].double()
                        if spread:  # blocks of very different sizes
                            x = x * 2.0 ** torch.randint(-int(spread), int(spread) + 1, (1,), generator=gen).item()
                        e = scale_exponent(x, code)
                        numbers = nearest(x * 2.0 ** -e, code)
                        view[where, at % page:at % page + len(x), h] = numbers.float().to(code)
                        scales[where, at % page // block, h] = e + 127
                        held[at:at + block, h] = numbers * 2.0 ** e
                rows[i] = held  # (kept in 64 bits: what the cache stands for)
            scales = scales.cuda()
            if strided:  # scales as a view of something wider
                wide = torch.full((pages, hk, 2 * (page // block) + 1), NOT_A_NUMBER, dtype=torch.uint8, device="cuda")
                into = wide[:, :, 1::2].transpose(1, 2)
                into.copy_(scales)
                scales = into
            setattr(self, name + "_cache", codes.cuda().transpose(1, 2) if kw.get("heads_first") else codes.cuda())
            setattr(self, name + "_scales", scales.view(torch.float8_e8m0fnu))

    def launch(self, workspace="own", scale=None):
        from iris_amd import attention

        if isinstance(workspace, str):
            workspace = attention.make_workspace(self.shape[2])
        args = dict(scale=scale, window=self.window, sinks=self.sinks, lse=self.lse, workspace=workspace, status=self.word, k_scales=self.k_scales,
                    v_scales=self.v_scales)
        if self.news is None:
            attention.decode_attention(self.q, self.k_cache, self.v_cache, self.table, self.lens, self.out, **args)
        else:
            attention.prompt_attention(self.q, self.k_cache, self.v_cache, self.table, self.lens, self.starts, self.out, **args)
        return workspace
