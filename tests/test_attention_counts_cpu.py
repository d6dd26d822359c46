"""Tokens, heads, pages and requests that 32-bit fields of the launches' arguments do not hold: refused, and not taken for what is left of them."""

import pytest
import torch

from iris_amd import attention
from test_attention_checks_cpu import BF16, calls, decode, operands  # noqa: F401  (a fixture)
from test_quantized_cache_cpu import E4M3, E8M0, CALLS, attend_operands, read_operands, write_operands

MANY = (1 << 32) + 5  # (5, were it cut to 32 bits; expanded tensors of no memory)


def refused(run, o, change):
    with pytest.raises(ValueError, match="31 bits"):
        run(**dict(o, **change))


def test_tokens_and_heads(calls):  # noqa: F811
    heads = torch.zeros((1, 2, 64), dtype=BF16).expand(MANY, 2, 64)
    write, read = CALLS["write"][0], CALLS["read"][0]
    refused(write, write_operands(), dict(k=heads, v=heads))
    refused(write, write_operands(), dict(k=torch.zeros((5, 1, 64), dtype=BF16).expand(5, MANY, 64)))
    refused(read, read_operands(), dict(k_out=heads, v_out=heads))
    refused(decode, attend_operands(), dict(q=heads))
    refused(decode, operands(), dict(q=heads, out=heads))
    with pytest.raises(ValueError, match="31 bits"):
        attention.qk_norm_rope(heads, heads, None, None, None, heads, heads)
    assert not calls.launched


def test_pages(calls):  # noqa: F811
    cache = torch.zeros((1, 32, 2, 64), dtype=torch.uint8).view(E4M3).expand(MANY, 32, 2, 64)
    scales = torch.zeros((1, 2, 2), dtype=torch.uint8).view(E8M0).expand(MANY, 2, 2)
    many = dict(k_cache=cache, v_cache=cache, k_scales=scales, v_scales=scales)
    for name, (run, ops) in CALLS.items():
        refused(run, ops(), many)
    wide = torch.zeros((1, 16, 2, 64), dtype=BF16).expand(MANY, 16, 2, 64)
    refused(decode, operands(), dict(k_cache=wide, v_cache=wide))
    assert not calls.launched


def test_requests(calls):  # noqa: F811
    table = torch.zeros((1, 4), dtype=torch.int32).expand(MANY, 4)
    for run, o in ((CALLS["read"][0], read_operands()), (decode, attend_operands()), (decode, operands())):
        refused(run, o, dict(block_table=table))
    assert not calls.launched
