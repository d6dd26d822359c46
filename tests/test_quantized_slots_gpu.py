"""Slots that a write into a cache in 8 bits takes, skips and reports: compared with calls that leave the skipped tokens out."""

import pytest
import torch

from iris_amd import attention
from quantized_reference import E4M3, E5M2, Cache

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SKIPPED = -1


class Slots:
    """A cache with something in it, tokens of very different sizes, and what becomes of them."""

    def __init__(self, slots, *, page=32, block=16, pages=8, heads=2, dim=64, dtype=BF16, code=E4M3):
        g = torch.Generator().manual_seed(len(slots))
        self.caches = attention.make_quantized_cache(pages, page, heads, dim, block=block, dtype=code)
        self.slots = torch.tensor(slots, dtype=torch.int64, device="cuda")
        x = torch.randn((len(slots), 2 * heads, dim), generator=g) * torch.exp2(torch.randint(-6, 7, (len(slots), 1, 1), generator=g).float())
        self.k, self.v = x.to(dtype).cuda().split(heads, 1)
        old = torch.randn((pages * page, heads, dim), generator=g).to(dtype).cuda()
        attention.write_quantized_cache(old, -old, *self.caches, torch.arange(pages * page, device="cuda"))
        self.word = torch.zeros(1, dtype=torch.int32, device="cuda")

    def write(self, caches, slots):
        attention.write_quantized_cache(self.k, self.v, *caches, slots, status=self.word)

    def check(self, written, status):
        """``written``: the tokens that are to be; the others are skipped, whatever they are."""
        want = [t.clone() for t in self.caches]
        self.write(self.caches, self.slots)
        assert self.word.item() == status
        keep = torch.zeros(len(self.slots), dtype=torch.bool, device="cuda")
        keep[torch.tensor(written, dtype=torch.int64, device="cuda")] = True
        self.k, self.v = self.k[keep], self.v[keep]  # (a call of these alone)
        self.word.zero_()
        self.write(want, self.slots[keep])
        assert self.word.item() == 0
        for got, expected in zip(self.caches, want):
            assert torch.equal(got.view(torch.uint8), expected.view(torch.uint8))


TYPES = [(BF16, 64, E4M3), (F32, 256, E5M2), (F16, 128, E4M3)]


@pytest.mark.parametrize("dtype,dim,code", TYPES)
@pytest.mark.parametrize("slots,written", [
    ([0, 1, 5, 6, 7], [0, 1]),                      # the rest of a block behind a hole
    ([0, 1, 5, 6, 7, 16, 17], [0, 1, 5, 6]),        # ... and the next block
    ([35, 36, 36, 37, 38], [0, 1]),                 # a slot twice
    ([9, 8, 7, 6], [0]),                            # backwards
    ([3, 5, 4, 32, 33, 35, 34, 36, 48], [0, 3, 4, 8]),
])
def test_the_rest_of_a_block_is_skipped_behind_a_slot_that_is_not_the_next(slots, written, dtype, dim, code):
    Slots(slots, dtype=dtype, dim=dim, code=code).check(written, attention.STATUS_BAD_INDEX)


@pytest.mark.parametrize("block", [64, 192, 512])
def test_the_same_in_blocks_that_waves_share(block):
    slots = [*range(40, 60), 61, 62, 63, *range(block, block + 20), block + 19, *range(block + 20, block + 30)]
    Slots(slots, page=block, block=block, pages=3).check([*range(20), *range(23, 43)], attention.STATUS_BAD_INDEX)


@pytest.mark.parametrize("dtype,dim,code", TYPES)
@pytest.mark.parametrize("slots,written", [
    ([0, 1, -1, 2, 3], [0, 1]),                              # padding inside a block
    ([5, -1, 7], [0]),
    ([-1, 5, -1, 5, -1, 16], [1, 5]),
    ([0, 1, 1 << 40, 2, 3, 20, -7, 21], [0, 1, 5]),          # what lies outside of the cache is skipped, too
    ([3, 256, 4], [0]),
    ([3, 5, -1, 6, -1, -1, 7, 33, -1, 48], [0, 7, 9]),       # behind a token that is skipped itself
])
def test_no_block_goes_on_behind_skipped_tokens(slots, written, dtype, dim, code):
    Slots(slots, dtype=dtype, dim=dim, code=code).check(written, attention.STATUS_BAD_INDEX)


@pytest.mark.parametrize("dtype,dim,code", TYPES)
def test_padding_between_blocks_is_no_mistake(dtype, dim, code):
    slots = [14, 15, -1, -1, 16, 17, -1, 32, -1, 67, 68, -1]
    Slots(slots, dtype=dtype, dim=dim, code=code).check([i for i, s in enumerate(slots) if s >= 0], 0)


@pytest.mark.parametrize("page,block", [(16, 16), (64, 64), (256, 256), (512, 512)])
@pytest.mark.parametrize("gap", [1, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128, 129, 700, 1086, 1087, 1088, 1089, 2112, 5000])
def test_skipped_tokens_of_any_number_between_two_of_a_block(gap, page, block):
    """At every place of the waves' chunks, and before other blocks, which are written."""
    for ahead in (0, 3, 29, 64):
        front = [block * 20 + i for i in range(min(ahead, block))]  # another block's tokens
        slots = [*front, 2, 3, *[SKIPPED] * gap, 4, 5, block, block + 1, *[SKIPPED] * gap, 2 * block + 9]
        n = len(front)
        Slots(slots, page=page, block=block, pages=24, heads=1).check([*range(n + 2), n + gap + 4, n + gap + 5, len(slots) - 1], attention.STATUS_BAD_INDEX)


@pytest.mark.parametrize("page,block", [(16, 16), (64, 64), (256, 256)])
def test_a_padded_batch(page, block):
    """Every request padded to the longest: many begin far behind the last slot."""
    longest, lengths = 2500, [3, 2500, 1, 17, 900]
    slots = []
    for i, n in enumerate(lengths):
        start = i * 2560 + (7 if n < 20 else 0)
        slots += [*range(start, start + n), *[SKIPPED] * (longest - n)]
    Slots(slots, page=page, block=block, pages=5 * 2560 // page, heads=1).check([i for i, s in enumerate(slots) if s >= 0], 0)


def test_reading_more_requests_than_half_of_what_31_bits_count():
    """Most of them without a token."""
    requests, page, some = (1 << 30) + 9, 16, 7
    caches = attention.make_quantized_cache(some, page, 1, 64)
    x = torch.randn((some * page, 1, 64), device="cuda", dtype=BF16)
    attention.write_quantized_cache(x, x, *caches, torch.arange(some * page, device="cuda"))
    table, lengths = (torch.zeros((requests, 1) if wide else requests, dtype=torch.int32, device="cuda") for wide in (True, False))
    starts = torch.zeros(requests + 1, dtype=torch.int32, device="cuda")
    news = torch.tensor([1, 16, 0, 3, 9, 16, 2], dtype=torch.int32, device="cuda")
    table[-some:, 0] = torch.arange(some, dtype=torch.int32, device="cuda").flip(0)
    lengths[-some:] = news
    starts[-some:] = news.cumsum(0).int()
    tokens = int(news.sum())
    outs, word = [torch.zeros((tokens, 1, 64), dtype=F32, device="cuda") for _ in range(2)], torch.zeros(1, dtype=torch.int32, device="cuda")
    attention.read_quantized_cache(*caches, table, lengths, starts, *outs, status=word)
    assert word.item() == 0
    numbers = Cache(caches[0], caches[2], page, E4M3).elements().float().unflatten(0, (some, page)).flip(0)
    want = torch.cat([numbers[i, :n] for i, n in enumerate(news.tolist())])
    for got in outs:
        assert torch.equal(got.cpu(), want)
