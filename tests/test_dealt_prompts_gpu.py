"""Prompts over a cache in 8 bits whose row tiles fill the chip and are dealt out in another order than their own."""

import ctypes

import pytest
import torch

from attention_reference import BF16, F16
from iris_amd import _native, attention
from quantized_reference import E4M3, E5M2, Quantized
from test_attention_edges_gpu import Declining

pytestmark = pytest.mark.gpu


def items(p, monkeypatch):
    """The items that a launch's places take, as the library plans it on this device."""
    got = []
    with monkeypatch.context() as m:
        m.setattr(_native, "host", lambda: Declining())
        m.setattr(attention, "_launch", lambda name, args, device: got.append(args))
        p.launch()
    lib, info, item = _native.lib(), _native.AttentionPlanInfo(), ctypes.c_int64()
    args = [ctypes.byref(x) for x in got[0]] + [0]
    assert lib.iris_quantized_attention_plan(*args, ctypes.byref(info)) == 0 and info.kernel == _native.ATTENTION_PROMPT_TILES and info.parts == 1
    out = []
    for place in range(info.workgroups // p.k_cache.shape[2]):
        assert lib.iris_quantized_attention_item(*args, place, ctypes.byref(item)) == 0
        out.append(item.value)
    return out


# (16 tokens of 8 query heads a key head are a row tile: two items a request, the second of them empty)
@pytest.mark.parametrize("requests,hk,dim,dtype,code,left", [(256, 1, 128, BF16, E4M3, 0), (300, 1, 128, F16, E5M2, 1), (150, 2, 128, BF16, E4M3, 1),
                                                             (401, 1, 64, F16, E4M3, 1), (130, 1, 256, BF16, E5M2, 1)])
@pytest.mark.parametrize("window", [0, 24])
def test_prompts_that_are_dealt_out(requests, hk, dim, dtype, code, left, window, monkeypatch):
    """(``left``: their number is no multiple of 256.)"""
    lengths, news = [16 + (7 * i) % 53 for i in range(requests)], [16] * requests
    if left:
        news[-1] = 13
    p = Quantized(lengths, news, 8 * hk, hk, dim, dtype, 16, code=code, window=window)
    order = items(p, monkeypatch)
    assert sorted(order) == list(range(len(order))) and order != sorted(order) and (len(order) % 256 != 0) == bool(left)
    p.launch()
    p.check()


def test_dealt_out_in_a_captured_graph(monkeypatch):
    """Recorded once, replayed over other queries and lengths with eager work in between."""
    requests = 260
    p = Quantized([40 + i % 30 for i in range(requests)], [16] * requests, 8, 1, 128, BF16, 16)
    order = items(p, monkeypatch)
    assert order != sorted(order)
    workspace = attention.make_workspace(128)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        p.launch(workspace)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            p.launch(workspace)
    torch.cuda.current_stream().wait_stream(stream)
    longest = p.lens.clone()
    for shorter in (0, 9, 3, 0):
        p.lens.copy_(longest - shorter)
        p.q.copy_(torch.randn_like(p.q) if shorter else p.q_host)
        p.out.fill_(-7)
        graph.replay()
        got = p.out.clone()
        p.out.fill_(-7)
        p.launch(workspace)
        assert torch.equal(got, p.out) and p.word.item() == 0
    p.check()
    got, p.lse = p.out.clone(), None  # (a kernel of its own)
    p.out.fill_(-7)
    p.launch(workspace)
    assert torch.equal(got, p.out) and p.word.item() == 0
