"""Slots that a write into a cache in 8 bits takes, skips and reports: compared with calls that leave the skipped tokens out."""

import pytest
import torch

from iris_amd import attention
from quantized_reference import E4M3, E5M2

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
