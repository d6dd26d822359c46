"""Calls over a cache in 8 bits that run at the same time."""

import pytest
import torch

from attention_reference import BF16
from iris_amd import attention
from quantized_reference import Quantized

pytestmark = pytest.mark.gpu


def test_one_cache_from_two_streams_while_a_third_writes_another():
    """Single tokens, prompts and a reading of the same cache at once, each with its own workspace; what was written meanwhile is looked at, too."""
    lengths = [5000, 700, 3001]
    p = Quantized(lengths, None, 8, 2, 128, BF16, 16)
    q = Quantized(lengths, [300, 200, 41], 8, 2, 128, BF16, 16)
    for name in ("k_cache", "v_cache", "k_scales", "v_scales", "table", "k", "v"):
        setattr(q, name, getattr(p, name))
    ends = torch.tensor([0, *lengths], dtype=torch.int32).cumsum(0).int().cuda()
    outs = [torch.full((sum(lengths), 2, 128), -7.0, dtype=torch.float32, device="cuda") for _ in range(2)]
    spare = attention.make_quantized_cache(64, 16, 2, 128)
    x = torch.randn((1000, 2, 128), device="cuda", dtype=BF16)
    word, slots = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.arange(1000, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(3)]
    spaces = [attention.make_workspace(128) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            p.launch(spaces[0])
        with torch.cuda.stream(streams[1]):
            q.launch(spaces[1])
            attention.read_quantized_cache(p.k_cache, p.v_cache, p.k_scales, p.v_scales, p.table, p.lens, ends, *outs, status=word)
        with torch.cuda.stream(streams[2]):
            attention.write_quantized_cache(x, -x, *spare, slots, status=word)
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    p.check()
    q.check()
    assert word.item() == 0
    for got, rows in zip(outs, (p.k, p.v)):
        assert torch.equal(got.cpu().double(), torch.cat([r.cpu().double() for r in rows]))
    alone = attention.make_quantized_cache(64, 16, 2, 128)
    attention.write_quantized_cache(x, -x, *alone, slots)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(spare, alone))
