"""Keys and values written into a cache in 8 bits, and read back: code by code, for every rounding is to nearest and nothing is left to a tolerance."""

import math
import random

import pytest
import torch

import attention_reference as R
from attention_reference import BF16, F16, F32
from iris_amd import attention
from quantized_reference import E4M3, E5M2, LARGEST, Cache, same

pytestmark = pytest.mark.gpu

CODES, E8M0 = [E4M3, E5M2], torch.float8_e8m0fnu


class Written:
    """Requests with ``cached`` tokens to which ``new`` ones come, in a cache of shuffled pages; what is in no request's rows holds a mark."""

    def __init__(self, spans, heads, dim, dtype, code, page, block, seed=0, heads_first=False, fused=True, padding=0):
        self.spans, self.block, self.code, self.dtype = spans, block, code, dtype
        rng = random.Random(seed)
        counts = [R.cdiv(c + n, page) for c, n in spans]
        pages = sum(counts) + 2
        order = list(range(pages))
        rng.shuffle(order)
        g = torch.Generator().manual_seed(seed)
        shape = (pages, heads, page, dim) if heads_first else (pages, page, heads, dim)
        self.caches, self.scales, self.before = {}, {}, {}
        for name in "kv":
            codes = (torch.randn(shape, generator=g) * LARGEST[code] / 8).clamp(-LARGEST[code], LARGEST[code]).to(code).cuda()
            self.caches[name] = codes.transpose(1, 2) if heads_first else codes
            self.scales[name] = torch.randint(110, 120, (pages, page // block, heads), generator=g).to(torch.uint8).cuda().view(torch.float8_e8m0fnu)
        slots, at = [], 0
        for (c, n), count in zip(spans, counts):
            mine = order[at:at + count]
            at += count
            slots += [mine[p // page] * page + p % page for p in range(c, c + n)]
        self.slots = torch.tensor(slots + [-1] * padding, dtype=torch.int64, device="cuda")
        tokens = len(slots) + padding
        wide = torch.randn((tokens, 3 * heads * dim), generator=g) * torch.exp2(torch.randint(-6, 7, (tokens, 1), generator=g).float())
        wide = wide.to(dtype).cuda()
        if fused:
            _, self.k, self.v = (x.unflatten(1, (heads, dim)) for x in wide.split(heads * dim, 1))
        else:
            self.k, self.v = (wide[:, i * heads * dim:(i + 1) * heads * dim].unflatten(1, (heads, dim)).contiguous() for i in (0, 1))
        self.word = torch.zeros(1, dtype=torch.int32, device="cuda")

    def want(self):
        out = {}
        for name, x in (("k", self.k), ("v", self.v)):
            out[name] = Cache(self.caches[name], self.scales[name], self.block, self.code)
            out[name].write(x, self.slots)
        return out

    def launch(self):
        attention.write_quantized_cache(self.k, self.v, self.caches["k"], self.caches["v"], self.scales["k"], self.scales["v"], self.slots, status=self.word)

    def check(self, want):
        for name in "kv":
            assert torch.equal(self.scales[name].view(torch.uint8).cpu().flatten(0, 1).int(), want[name].bytes), name
            assert same(self.caches[name], want[name].numbers), name


def run(*args, status=0, **kw):
    p = Written(*args, **kw)
    want = p.want()
    p.launch()
    p.check(want)
    assert p.word.item() == status
    p.launch()  # the same tokens again: nothing moves
    p.check(want)
    return p


SPANS = [(0, 1), (0, 16), (0, 40), (5, 1), (15, 1), (16, 1), (15, 2), (37, 100), (3, 12), (100, 17)]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 192, 256])
def test_types_and_head_sizes(dtype, code, dim):
    run(SPANS, 2, dim, dtype, code, 32, 16)


@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (48, 48), (64, 32), (128, 128), (256, 64), (80, 80)])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F32, 256), (F16, 64)])
def test_blocks(page, block, dtype, dim):
    """(Blocks of more rows than a wave holds are read twice.)"""
    run(SPANS + [(0, 300), (70, 300), (127, 2), (255, 70)], 3, dim, dtype, E4M3, page, block, heads_first=page == 64, fused=page != 16)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F32, 256), (F16, 64)])
@pytest.mark.parametrize("block", [192, 256, 512])
def test_long_blocks(block, dtype, dim):
    """Blocks that sixteen waves share; of 512 tokens some rows are read twice."""
    run([(0, 1), (0, 700), (block - 3, 5), (100, block + 60), (block, 33), (block - 1, 1)], 2, dim, dtype, E5M2, block, block)


@pytest.mark.parametrize("page,block,requests", [(32, 16, 700), (64, 64, 150), (256, 256, 40)])
def test_many_tokens_of_many_heads(page, block, requests):
    """More tokens than waves: a wave, or the waves that share blocks, look after several."""
    run([(7, 1)] * requests + [(0, 901), (30, 1003), (0, 16), (0, 16), (17, 300)], 8, 64, BF16, E4M3, page, block, padding=29)


def test_scales_as_views():
    """Scales as every other byte of something wider, heads before blocks, whose other bytes stay."""
    p = Written([(5, 40), (0, 17), (70, 3)], 2, 64, BF16, E4M3, 64, 16)
    pages = p.caches["k"].shape[0]
    wide = torch.full((2, pages, 2, 9), 77, dtype=torch.uint8, device="cuda")
    for i, name in enumerate("kv"):
        view = wide[i, :, :, 1::2].transpose(1, 2)
        view.copy_(p.scales[name].view(torch.uint8))
        p.scales[name] = view.view(E8M0)
    want = p.want()
    p.launch()
    p.check(want)
    assert bool((wide[..., ::2] == 77).all())
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([pages * 64], [0, pages * 64]))
    outs, word = read((p.caches["k"], p.caches["v"], p.scales["k"], p.scales["v"]), table, lengths, starts, pages * 64, 2, 64, BF16)
    assert word.item() == 0
    for got, name in zip(outs, "kv"):
        assert torch.equal(got.cpu(), Cache(p.caches[name], p.scales[name], 16, E4M3).elements().to(BF16))


def test_padded_tokens_and_slots_outside():
    p = Written([(0, 20), (3, 5)], 2, 64, BF16, E4M3, 16, 16, padding=3)
    p.slots = torch.cat((p.slots[:20], p.slots[25:], p.slots[20:25]))  # the padding between two requests
    p.slots[21] = 1 << 40
    p.slots[22] = p.caches["k"].shape[0] * 16
    want = p.want()
    p.launch()
    p.check(want)
    assert p.word.item() == attention.STATUS_BAD_INDEX


def test_a_block_whose_slots_are_not_in_a_row_is_reported():
    p = Written([(0, 16), (0, 16), (0, 16)], 1, 64, F16, E5M2, 32, 32)
    p.slots[5] += 1   # a hole, and the next one twice
    p.slots[20:24] = p.slots[20:24].flip(0)
    want = p.want()
    p.launch()
    p.check(want)
    assert p.word.item() == attention.STATUS_BAD_INDEX


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_every_rounding(dtype, code):
    """Every fp16 (or bf16; for fp32 every tie between neighbours and what is next to it) number up to the largest code in blocks of scale 1."""
    if dtype == F32:
        points = torch.arange(256, dtype=torch.uint8).view(code).float()
        points = points[points.isfinite() & (points >= 0)].unique()
        ties = (points[1:].double() + points[:-1].double()).div(2).float()
        x = torch.cat([points, ties, torch.nextafter(ties, torch.tensor(math.inf)), torch.nextafter(ties, torch.tensor(0.0))])
    else:
        x = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
        x = x[x.isfinite() & (x.float() <= LARGEST[code])]
    x = torch.cat([x, -x])
    rows = x.new_zeros((R.cdiv(len(x), 15 * 256) * 16, 256))
    at = torch.arange(len(rows)) % 16 != 0
    rows[at] = torch.cat([x, x.new_zeros(int(at.sum()) * 256 - len(x))]).view(-1, 256)
    rows[~at] = LARGEST[code]
    tokens = len(rows)
    k = rows.view(tokens, 1, 256).cuda()
    caches = attention.make_quantized_cache(tokens // 16, 16, 1, 256, dtype=code)
    attention.write_quantized_cache(k, k, *caches, torch.arange(tokens, device="cuda"))
    for cache, scales in zip(caches[:2], caches[2:]):
        assert bool((scales.view(torch.uint8) == 127).all())
        want = Cache(cache, scales, 16, code)
        want.write(k, torch.arange(tokens))
        assert same(cache, want.numbers)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_scales_at_their_borders(dtype, code):
    """Largest elements at, next to and between the borders of scales, from the smallest numbers to the largest."""
    top, low = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    values = [0.0, top, top / 2, low, low / 4]
    for e in range(-126, 127):
        for x in (1.75 * 2.0 ** e, 2.0 ** e):
            y = torch.tensor(x, dtype=torch.float64).to(dtype)
            if bool(y.isfinite()) and y > 0:
                bits = y.view(torch.int32 if dtype == F32 else torch.int16)
                values += [y.item(), (bits + 1).view(dtype).item(), (bits - 1).view(dtype).item()]
    x = torch.zeros((len(values) * 16, 1, 16), dtype=torch.float64)
    x[7::16, 0, 5] = torch.tensor(values, dtype=torch.float64)
    x[8::16, 0, 9] = torch.tensor(values, dtype=torch.float64) / 37
    k = x.to(dtype).cuda()
    caches = attention.make_quantized_cache(len(values), 16, 1, 16, dtype=code)
    attention.write_quantized_cache(k, -k, *caches, torch.arange(len(k), device="cuda"))
    for cache, scales, y in zip(caches[:2], caches[2:], (k, -k)):
        want = Cache(cache, scales, 16, code)
        want.write(y, torch.arange(len(k)))
        assert torch.equal(scales.view(torch.uint8).cpu().flatten().int(), want.bytes.flatten())
        assert same(cache, want.numbers)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block", [16, 128])
def test_what_is_not_finite_is_no_number_and_has_no_part_in_a_scale(dtype, block):
    p = Written([(0, 128), (4, 12), (0, 128)], 2, 64, dtype, E4M3, 128, block)
    p.k[3, 0, 7], p.k[9, 1, 0], p.v[100, 0, 63], p.v[130, 1, 5] = math.nan, math.inf, -math.inf, math.nan
    p.k[140:156, 0] = math.nan
    want = p.want()
    p.launch()
    p.check(want)


@pytest.mark.parametrize("code", CODES)
def test_a_scale_grows_token_by_token(code):
    """A decoding request: each token in a call of its own, every block's scale as large as its tokens so far want."""
    p = Written([(0, 70)], 2, 64, BF16, code, 32, 32)
    want = p.want()
    whole = {name: (Cache(p.caches[name], p.scales[name], 32, code)) for name in "kv"}
    for t in range(70):
        attention.write_quantized_cache(p.k[t:t + 1], p.v[t:t + 1], p.caches["k"], p.caches["v"], p.scales["k"], p.scales["v"], p.slots[t:t + 1])
        for name, x in (("k", p.k), ("v", p.v)):
            whole[name].write(x[t:t + 1], p.slots[t:t + 1])
    p.check(whole)
    for name in "kv":  # the scales are those of all the tokens at once, for one only grows while its block fills
        assert torch.equal(whole[name].bytes, want[name].bytes)


def test_a_scale_that_is_no_number_stays_until_its_block_is_begun_anew():
    p = Written([(3, 5), (0, 5)], 1, 64, BF16, E4M3, 16, 16)
    for name in "kv":
        p.scales[name].view(torch.uint8).fill_(255)
    p.launch()
    blocks = (p.slots[[0, 5]] // 16).tolist()
    for name in "kv":
        got = p.scales[name].view(torch.uint8).flatten()
        assert got[blocks[0]] == 255 and got[blocks[1]] != 255


def read(p_caches, table, lengths, starts, tokens, heads, dim, dtype, fill=-7.0, **kw):
    outs = [torch.full((tokens, heads, dim), fill, dtype=dtype, device="cuda") for _ in range(2)]
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    attention.read_quantized_cache(*p_caches, table, lengths, starts, *outs, status=word, **kw)
    return outs, word


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_every_code_at_every_scale(dtype, code):
    """Products are exact in 64 bits; past fp32's ordinary numbers (scales below 2^-100 are never written) a result may be flushed to 0."""
    codes = torch.arange(256, dtype=torch.uint8).view(16, 1, 16).expand(256, 16, 1, 16).contiguous().view(code).cuda()
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1, 1).contiguous().cuda().view(torch.float8_e8m0fnu)
    table = torch.arange(256, dtype=torch.int32, device="cuda")[None]
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([4096], [0, 4096]))
    (k, v), word = read((codes, codes, scales, scales), table, lengths, starts, 4096, 1, 16, dtype)
    elements = Cache(codes, scales, 16, code).elements()
    want = elements.to(dtype)
    kept = (elements.abs() >= 2.0 ** -126) | (elements == 0) | elements.isnan()
    for got in (k.cpu(), v.cpu()):
        assert bool(((got == want) | (got.isnan() & want.isnan()) | ~kept).all())
        assert bool((got[~kept].abs() <= 2.0 ** -126).all())
    assert word.item() == 0


@pytest.mark.parametrize("dtype,dim,code", [(BF16, 128, E4M3), (F16, 80, E5M2), (F32, 256, E4M3), (BF16, 16, E5M2)])
@pytest.mark.parametrize("page,block", [(16, 16), (96, 48), (64, 64)])
def test_reading(dtype, dim, code, page, block):
    lengths, news = [0, 1, 15, 16, 17, 100, 500, 64, 0, 33], [0, 1, 3, 16, 17, 100, 41, 0, 0, 33]
    p = Written([(0, n) for n in lengths], 3, dim, F32, code, page, block)
    p.launch()
    table = torch.zeros((len(lengths), R.cdiv(500, page) + 1), dtype=torch.int32)
    at = 0
    for i, n in enumerate(lengths):
        for j in range(R.cdiv(n, page)):
            table[i, j] = p.slots[at + j * page] // page
        at += n
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for counts in (lengths, news):
        starts = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).int().cuda()
        tokens = sum(counts)
        (k, v), word = read((p.caches["k"], p.caches["v"], p.scales["k"], p.scales["v"]), table.cuda(), lens, starts, tokens + 5, 3, dim, dtype)
        assert word.item() == 0
        slots = torch.cat([p.slots.cpu()[sum(lengths[:i + 1]) - n:sum(lengths[:i + 1])] for i, n in enumerate(counts)])
        for got, name in ((k, "k"), (v, "v")):
            want = Cache(p.caches[name], p.scales[name], block, code).elements()[slots].to(dtype)
            assert torch.equal(got[:tokens].cpu(), want)
            assert bool((got[tokens:] == -7).all())  # rows of no request


def test_reading_many_requests_into_views():
    """More requests than a workgroup holds the starts of; outputs as parts of something wider."""
    requests, page = 3000, 16
    caches = attention.make_quantized_cache(requests, page, 2, 64)
    k = torch.randn((requests * page, 2, 64), device="cuda", dtype=BF16)
    attention.write_quantized_cache(k, k, *caches, torch.arange(requests * page, device="cuda"))
    lengths = torch.arange(requests, dtype=torch.int32, device="cuda") % 17
    starts = torch.cat((lengths.new_zeros(1), lengths.cumsum(0).int()))
    table = torch.arange(requests, dtype=torch.int32, device="cuda").flip(0)[:, None].contiguous()
    tokens = int(starts[-1])
    wide = torch.zeros((tokens, 4, 64), dtype=BF16, device="cuda")
    attention.read_quantized_cache(*caches, table, lengths, starts, wide[:, :2], wide[:, 2:])
    request = torch.repeat_interleave(torch.arange(requests, device="cuda"), lengths.long())
    slots = table[request, 0].long() * page + torch.arange(tokens, device="cuda") - starts[request].long()
    want = Cache(caches[0], caches[2], page, E4M3).elements()[slots.cpu()].to(BF16)
    assert torch.equal(wide[:, :2].cpu(), want) and torch.equal(wide[:, 2:].cpu(), want)


def test_rows_that_have_no_place_are_reported():
    caches = attention.make_quantized_cache(4, 16, 1, 64)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.tensor([[0, 1], [9, -1], [2, 3]], dtype=torch.int32, device="cuda")
    # more rows than tokens; a page that is none; longer than the table
    (k, v), word = read(caches, table, ints(2, 3, 33), ints(0, 3, 6, 8), 8, 1, 64, BF16)
    assert word.item() == attention.STATUS_BAD_INDEX
    bad = [True, False, False, True, True, True, False, True]
    for got in (k, v):
        assert got.isnan().all(-1).flatten().tolist() == bad
        assert bool((got[[1, 2, 6]] == 0).all())


def test_in_a_captured_graph_on_another_stream():
    """A step recorded once: slots change from replay to replay."""
    p = Written([(0, 48)], 2, 64, BF16, E4M3, 16, 16)
    whole = {name: Cache(p.caches[name], p.scales[name], 16, E4M3) for name in "kv"}
    k, v, slots = p.k[:1].clone(), p.v[:1].clone(), torch.full((1,), -1, dtype=torch.int64, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        attention.write_quantized_cache(k, v, p.caches["k"], p.caches["v"], p.scales["k"], p.scales["v"], slots)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            attention.write_quantized_cache(k, v, p.caches["k"], p.caches["v"], p.scales["k"], p.scales["v"], slots)
    torch.cuda.current_stream().wait_stream(stream)
    for t in range(48):
        k.copy_(p.k[t:t + 1])
        v.copy_(p.v[t:t + 1])
        slots.copy_(p.slots[t:t + 1])
        graph.replay()
        for name, x in (("k", p.k), ("v", p.v)):
            whole[name].write(x[t:t + 1], p.slots[t:t + 1])
        if t % 5 == 0 or t > 45:
            torch.cuda.synchronize()
            p.check(whole)


def test_addresses_past_32_bits():
    """A cache of 6 GB of codes, its last page."""
    pages = (6 << 30) // (64 * 8 * 128)
    caches = [torch.empty((pages, 64, 8, 128), dtype=E4M3, device="cuda") for _ in range(2)]
    scales = [torch.empty((pages, 4, 8), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    k = torch.randn((64, 8, 128), device="cuda", dtype=BF16)
    slots = torch.arange(64, device="cuda") + (pages - 1) * 64
    attention.write_quantized_cache(k, k, *caches, *scales, slots)
    table, length, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[pages - 1]], [64], [0, 64]))
    (got, also), word = read((*caches, *scales), table, length, starts, 64, 8, 128, BF16)
    small = [c[-1:].clone() for c in caches] + [s.view(torch.uint8)[-1:].clone().view(torch.float8_e8m0fnu) for s in scales]
    want = Cache(small[0], small[2], 16, E4M3)
    assert torch.equal(got.cpu(), want.elements().to(BF16)) and torch.equal(got, also) and word.item() == 0
    want.write(k, slots - (pages - 1) * 64)
    assert same(small[0], want.numbers) and bool((got - k).abs().max() <= 2.0 ** -4 * k.abs().max())


def test_nothing_to_do():
    caches = attention.make_quantized_cache(2, 16, 2, 64)
    none = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    attention.write_quantized_cache(none, none, *caches, torch.empty(0, dtype=torch.int64, device="cuda"))
    table, zero = torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    attention.read_quantized_cache(*caches, table, zero, torch.zeros(2, dtype=torch.int32, device="cuda"), none, none.clone())
    # a cache without a page: no slot lies in it, and no token
    caches = attention.make_quantized_cache(0, 16, 2, 64)
    some, word = torch.ones((2, 2, 64), dtype=BF16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    attention.write_quantized_cache(some, some.clone(), *caches, torch.tensor([-1, 0], device="cuda"), status=word)
    assert word.item() == attention.STATUS_BAD_INDEX
    outs, word = read(caches, table, zero + 1, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 2, 2, 64, BF16)
    assert word.item() == attention.STATUS_BAD_INDEX and bool(outs[0][0].isnan().all()) and bool((outs[0][1] == -7).all())
