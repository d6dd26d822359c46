"""The order in which workgroups of prompts over a cache in 8 bits take their row tiles: every tile once, and dealt out where they fill the chip."""

import ctypes

import pytest

from iris_amd import _native
from test_attention_plans_cpu import COUNTERS, CUS, call

INVALID = _native.HIP_ERROR_INVALID_VALUE


def order(cus=CUS, code=_native.DTYPE_E4M3, **kw):
    """(plan, the items that the places take)"""
    a, s = call(**kw), _native.CacheScales()
    s.k_scales = s.v_scales = 1 << 20
    s.block, s.code = 16, code
    info, item, lib = _native.AttentionPlanInfo(), ctypes.c_int64(-1), _native.lib()
    args = ctypes.byref(a), ctypes.byref(s), cus
    assert lib.iris_quantized_attention_plan(*args, ctypes.byref(info)) == 0
    places = info.workgroups if info.kernel == _native.ATTENTION_DECODE else info.workgroups // a.k_heads
    items = []
    for place in range(places):
        assert lib.iris_quantized_attention_item(*args, place, ctypes.byref(item)) == 0
        items.append(item.value)
    for place in (-1, places):
        assert lib.iris_quantized_attention_item(*args, place, ctypes.byref(item)) == INVALID
    return info, items


def prompts(row_tiles, *, hk=1, dim=128, requests=65, **kw):
    """Requests whose prompts leave room for ``row_tiles`` tiles of 128 rows of each key head."""
    return dict(requests=requests, tokens=16 * (row_tiles - requests), hq=8 * hk, hk=hk, dim=dim, **kw)


def test_every_item_is_taken_once_whatever_their_number():
    """(A device of few units has room for few row tiles, and deals out all these.)"""
    moved = set()
    for n in [*range(200, 1100), 1 << 11, (1 << 12) + 255]:
        info, items = order(cus=2, **prompts(n))
        assert info.kernel == _native.ATTENTION_PROMPT_TILES and len(items) == n
        assert sorted(items) == list(range(n)), n
        if items != list(range(n)):
            moved.add(n)
    assert moved == {*range(200, 1100), 1 << 11, (1 << 12) + 255}


@pytest.mark.parametrize("n", [512, 600, 767, 1024])
def test_every_engine_gets_items_of_every_kind(n):
    """Where requests have one row tile each every other item is empty, where they have three every fourth.  XCDs get workgroups in turn, and the four
    engines of each in turn, so places 32 apart are one engine's: of 256 places these are eight, whose numbers differ in their upper three
    bits, which reversed are the items' lower three."""
    _, items = order(**prompts(n))
    for batch in range(0, n // 256 * 256, 256):
        for engine in range(32):
            mine = items[batch + engine:batch + 256:32]
            assert sorted(i % 8 for i in mine) == list(range(8))


@pytest.mark.parametrize("dim,hk,places", [(128, 1, 512), (64, 1, 768), (256, 1, 256), (128, 2, 512)])
@pytest.mark.parametrize("code", [_native.DTYPE_E4M3, _native.DTYPE_E5M2])
def test_they_are_dealt_out_where_they_fill_the_places(dim, hk, places, code):
    for tiles in (places // hk - 1, places // hk, places // hk + 77):
        _, items = order(code=code, **prompts(tiles, hk=hk, dim=dim))
        assert (items != list(range(tiles))) == (tiles * hk >= places), tiles


def test_other_launches_take_their_work_in_its_own_order():
    for kw in (dict(requests=300), dict(requests=2, tokens=4000, hq=8, dim=128),                                # single tokens; by length
               dict(requests=1, tokens=2000, hq=8, dim=128, workspace=COUNTERS + 4096 * 16 * 132),              # in parts
               dict(requests=100, tokens=200, hq=8), dict(requests=600, tokens=9600, hq=8, dim=128, dtype="fp32")):  # rows of 16
        info, items = order(**kw)
        assert items == list(range(len(items))) and len(items) > 1


def test_refusals():
    lib, item = _native.lib(), ctypes.c_int64()
    a, s = call(**prompts(600)), _native.CacheScales()
    s.k_scales = s.v_scales = 1 << 20
    s.block, s.code = 16, _native.DTYPE_E4M3
    entry = lib.iris_quantized_attention_item
    args = ctypes.byref(a), ctypes.byref(s)
    assert entry(*args, CUS, 0, ctypes.byref(item)) == 0
    assert entry(None, args[1], CUS, 0, ctypes.byref(item)) == entry(args[0], None, CUS, 0, ctypes.byref(item)) == INVALID
    assert entry(*args, CUS, 0, None) == entry(*args, -1, 0, ctypes.byref(item)) == INVALID
    s.code = _native.DTYPE_BF16
    assert entry(*args, CUS, 0, ctypes.byref(item)) == INVALID
    s.code, a.tokens = _native.DTYPE_E4M3, 0
    assert entry(*args, CUS, 0, ctypes.byref(item)) == INVALID  # nothing to do: no item
