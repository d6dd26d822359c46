"""Element types of the C-ABI: each has a value of its own, and a cache in 8 bits takes its two codes and no other."""

import ctypes
import os
import re

import pytest

from iris_amd import _native, ops
from test_attention_plans_cpu import CUS, call

HEADER = os.path.join(os.path.dirname(__file__), "..", "include", "iris_amd.h")
INVALID = _native.HIP_ERROR_INVALID_VALUE
ADDRESS = 4096  # (never followed)


def types():
    return {name: int(value) for name, value in re.findall(r"#define IRIS_DTYPE_(\w+) (\d+)", open(HEADER).read())}


def test_every_type_has_a_value_of_its_own():
    values = types()
    assert set(values) >= {"F32", "F16", "BF16", "I8", "I16", "I32", "I64", "E4M3", "E5M2"}
    assert len(set(values.values())) == len(values)
    assert (values["E4M3"], values["E5M2"]) == (_native.DTYPE_E4M3, _native.DTYPE_E5M2)
    assert not {values["E4M3"], values["E5M2"]} & {*ops._DTYPES.values(), *ops._RMA_DTYPES.values()}


@pytest.mark.parametrize("name", [name for name in types() if name not in ("E4M3", "E5M2")])
def test_other_types_are_no_codes(name):
    lib, code = _native.lib(), types()[name]
    for struct, entry, operands in ((_native.WriteCacheArgs, lib.iris_write_quantized_cache_launch, "k v slots"),
                                    (_native.ReadCacheArgs, lib.iris_read_quantized_cache_launch, "k_out v_out block_table lengths starts")):
        a = struct()
        for operand in (operands + " k_cache v_cache k_scales v_scales").split():
            setattr(a, operand, ADDRESS)
        a.dtype, a.head_dim, a.page_size, a.block, a.heads = _native.DTYPE_BF16, 64, 32, 16, 2  # (and no token)
        for accepted in (_native.DTYPE_E4M3, _native.DTYPE_E5M2):
            a.code = accepted
            assert entry(ctypes.byref(a), None) == 0
        a.code = code
        assert entry(ctypes.byref(a), None) == INVALID
    a, s, info, n = call(page=32), _native.CacheScales(), _native.AttentionPlanInfo(), ctypes.c_int()
    s.k_scales = s.v_scales = ADDRESS
    s.block, s.code = 16, _native.DTYPE_E5M2
    args = ctypes.byref(a), ctypes.byref(s)
    assert lib.iris_quantized_attention_plan(*args, CUS, ctypes.byref(info)) == 0
    s.code = code
    assert lib.iris_quantized_attention_plan(*args, CUS, ctypes.byref(info)) == INVALID
    assert lib.iris_quantized_attention_launch(*args, None) == INVALID
    assert lib.iris_quantized_attention_kernel_info(*args, ctypes.byref(n), ctypes.byref(n)) == INVALID
