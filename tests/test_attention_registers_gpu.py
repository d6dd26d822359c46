"""Registers of the attention kernels: those of 16 rows keep everything in them; those of tiles, whose waves take all that a SIMD has,
spill some words a lane (heads of up to 128 outside of their loop), and no more than when they were measured."""

import ctypes

import pytest
import torch

from attention_reference import BF16, F16, F32
from iris_amd import _native, attention
from test_attention_edges_gpu import Declining
from test_paged_attention_gpu import Problem

pytestmark = pytest.mark.gpu


def scratch(dtype, dim, news, monkeypatch, *, lse=True, page=16, kernel):
    """Scratch bytes a lane of the kernel that a call would run."""
    got = []
    p = Problem([n + 10 for n in news] if news else [40, 50], news, 8, 8, dim, dtype, page)
    with monkeypatch.context() as m:
        m.setattr(_native, "host", lambda: Declining())
        m.setattr(attention, "_launch", lambda name, args, device: got.append(args))
        if not lse:
            p.lse = None
        p.launch()
    info, registers, spills = _native.AttentionPlanInfo(), ctypes.c_int(), ctypes.c_int()
    assert _native.lib().iris_attention_plan(ctypes.byref(got[0]), 0, ctypes.byref(info)) == 0 and info.kernel == kernel
    assert _native.lib().iris_attention_kernel_info(ctypes.byref(got[0]), ctypes.byref(registers), ctypes.byref(spills)) == 0
    assert 0 < registers.value <= 512
    return spills.value


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 20])
def test_no_scratch_in_tiles_of_16_rows(dtype, dim, page, monkeypatch):
    assert scratch(dtype, dim, None, monkeypatch, page=page, kernel=_native.ATTENTION_DECODE) == 0
    assert scratch(dtype, dim, [3, 9], monkeypatch, page=page, kernel=_native.ATTENTION_PROMPT_ROWS) == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,lse,most", [(64, True, 64), (64, False, 88), (128, True, 88), (128, False, 108), (256, True, 372), (256, False, 364)])
def test_scratch_of_tiles_of_128_rows(dtype, dim, lse, most, monkeypatch):
    assert scratch(dtype, dim, [900, 1300], monkeypatch, lse=lse, kernel=_native.ATTENTION_PROMPT_TILES) <= most
