"""The attention block's host side without a device: argument structs, the launchers' own checks, angle tables."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

from iris_amd import _native, attention

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
STRUCTS = {"iris_block_tables_args": _native.BlockTablesArgs, "iris_qk_norm_rope_args": _native.QkNormRopeArgs,
           "iris_qk_norm_rope_backward_args": _native.QkNormRopeBackwardArgs, "iris_attention_args": _native.AttentionArgs}
INVALID = _native.HIP_ERROR_INVALID_VALUE


def test_struct_layouts_match_the_c_compiler(tmp_path):
    lines = []
    for cname, struct in STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{name} %zu\\n", offsetof({cname}, {name}));' for name, _ in struct._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "iris_amd.h"\nint main(void){\n' + "\n".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    rows = iter(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n"))
    for cname, struct in STRUCTS.items():
        assert next(rows) == f"{cname} {ctypes.sizeof(struct)}"
        for name, _ in struct._fields_:
            assert next(rows) == f"{name} {getattr(struct, name).offset}"


def test_launchers_reject_bad_arguments_without_a_device():
    lib = _native.lib()
    for launch in (lib.iris_block_tables_launch, lib.iris_qk_norm_rope_launch, lib.iris_qk_norm_rope_backward_launch, lib.iris_attention_launch):
        assert launch(None, None) == INVALID
    t = _native.BlockTablesArgs()
    assert lib.iris_block_tables_launch(ctypes.byref(t), None) == INVALID  # no page size, no ring
    t.page_size, t.pool_size, t.requests = 16, 4, attention.MAX_REQUESTS + 1
    assert lib.iris_block_tables_launch(ctypes.byref(t), None) == INVALID
    for args, launch in ((_native.QkNormRopeArgs(), lib.iris_qk_norm_rope_launch),
                         (_native.QkNormRopeBackwardArgs(), lib.iris_qk_norm_rope_backward_launch)):
        args.dtype, args.head_dim = _native.DTYPE_BF16, 64
        assert launch(ctypes.byref(args), None) == 0  # no token: nothing to do
        args.tokens, args.q_heads, args.k_heads = 4, 2, 1
        assert launch(ctypes.byref(args), None) == INVALID  # no tensors
        for field, value in (("dtype", 7), ("head_dim", 63), ("head_dim", 514), ("rotary_dim", 66), ("rotary_dim", 3), ("tokens", -1)):
            old = getattr(args, field)
            setattr(args, field, value)
            assert launch(ctypes.byref(args), None) == INVALID, field
            setattr(args, field, old)
    a = _native.AttentionArgs()
    a.dtype, a.head_dim, a.page_size, a.scale = _native.DTYPE_BF16, 64, 16, 0.125
    assert lib.iris_attention_launch(ctypes.byref(a), None) == 0  # no query
    a.requests, a.tokens, a.q_heads, a.k_heads, a.table_width, a.num_pages = 2, 2, 4, 2, 3, 9
    assert lib.iris_attention_launch(ctypes.byref(a), None) == INVALID  # no tensors
    # (addresses that are never followed: every call here is refused before a launch)
    for field in ("q", "k_cache", "v_cache", "block_table", "lengths", "out"):
        setattr(a, field, 4096)
    a.stride_table = 3
    for field, value in (("dtype", 5), ("head_dim", 60), ("head_dim", 264), ("k_heads", 3), ("page_size", 0), ("window", -1), ("sinks", -1),
                         ("scale", 0.0), ("scale", math.nan), ("scale", math.inf), ("tokens", 3), ("stride_table", 2), ("q", 4104),
                         ("stride_qt", 4), ("stride_kc_row", 12), ("workspace", 4100), ("table_width", 1 << 28), ("num_pages", 0)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert lib.iris_attention_launch(ctypes.byref(a), None) == INVALID, (field, value)
        setattr(a, field, old)


def test_workspace_sizes():
    sizes = [_native.lib().iris_attention_workspace_elems(d) for d in (8, 64, 72, 128, 256)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert [_native.lib().iris_attention_workspace_elems(d) for d in (0, -1, 257)] == [0, 0, 0]


def test_tensors_of_the_host_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be on|got cpu"):
        attention.qk_norm_rope(x, x, None, None, None, x, x)
    with pytest.raises(RuntimeError):
        attention.decode_attention(x, x[None], x[None], i[:, None], i, x)
    with pytest.raises(RuntimeError):
        attention.build_block_tables(i, i, i[:, None], i, i.long(), 16, lengths=i, pool_state_out=i.long(), query_starts=i, positions=i, slots=i.long())


def angles(tables, position, pair):
    return math.atan2(tables[1][position, pair].item(), tables[0][position, pair].item())


def turns(x):
    return (x + math.pi) % (2 * math.pi) - math.pi


@pytest.mark.parametrize("rotary,base", [(64, 10000.0), (128, 500000.0), (2, 10000.0), (20, 10000.0)])
def test_rope_tables(rotary, base):
    tables = attention.rope_tables(5000, rotary, base=base, device="cpu")
    assert tables[0].shape == tables[1].shape == (5000, rotary // 2) and tables[0].dtype == torch.float32
    for position in (0, 1, 777, 4999):
        for pair in {0, 1 % (rotary // 2), rotary // 2 - 1}:
            want = position * base ** (-2 * pair / rotary)
            assert abs(tables[0][position, pair].item() - math.cos(want)) <= 2.0 ** -24 + 1e-9
            assert abs(tables[1][position, pair].item() - math.sin(want)) <= 2.0 ** -24 + 1e-9


def test_rope_tables_for_longer_contexts():
    plain = attention.rope_tables(4000, 64, device="cpu")
    linear = attention.rope_tables(16000, 64, scaling={"type": "linear", "factor": 4}, device="cpu")
    assert torch.allclose(linear[0][::4], plain[0], atol=1e-6) and torch.allclose(linear[1][::4], plain[1], atol=1e-6)
    # the base grows: the fastest pair keeps its angle, the slowest is divided by the factor
    grown = attention.rope_tables(16000, 64, scaling={"type": "base", "factor": 4}, device="cpu")
    assert torch.equal(grown[0][:4000, 0], plain[0][:, 0])
    assert torch.allclose(grown[1][::4, 31], plain[1][:, 31], atol=1e-6)
    for kind, growth in (("by_parts", 1 + 0.1 * math.log(4)), ("by_wavelength", 1.0)):
        t = attention.rope_tables(16000, 64, scaling={"type": kind, "factor": 4, "trained": 4000}, device="cpu")
        assert torch.allclose(t[0] ** 2 + t[1] ** 2, torch.full_like(t[0], growth ** 2), atol=1e-5)
        for pair in range(32):
            freq = 10000.0 ** (-2 * pair / 64)
            got = turns(angles(t, 1, pair)) / freq  # 1: kept, 1/4: divided
            assert 0.25 - 1e-5 <= got <= 1 + 1e-5
            if 4000 * freq / (2 * math.pi) >= 33:
                assert abs(got - 1) < 1e-5
            if 4000 * freq / (2 * math.pi) <= (0.7 if kind == "by_parts" else 1):
                assert abs(got - 0.25) < 1e-5
    fixed = attention.rope_tables(10, 64, scaling={"type": "by_parts", "factor": 4, "trained": 4000, "attention_factor": 1.0}, device="cpu")
    assert torch.allclose(fixed[0] ** 2 + fixed[1] ** 2, torch.ones(10, 32), atol=1e-6)


def test_rope_tables_refusals():
    for args, kw in [((0, 64), {}), ((8, 63), {}), ((8, 0), {}), ((8, 64), {"base": 0}), ((8, 64), {"scaling": {"type": "what", "factor": 2}}),
                     ((8, 64), {"scaling": {"type": "linear", "factor": 0.5}}), ((8, 64), {"scaling": {"type": "linear"}}),
                     ((8, 64), {"scaling": {"type": "by_parts", "factor": 2}}), ((8, 64), {"scaling": {"type": "linear", "factor": 2, "trained": 8}}),
                     ((8, 64), {"scaling": {"type": "by_wavelength", "factor": 2, "trained": 8, "fast": 1, "slow": 2}})]:
        with pytest.raises(ValueError):
            attention.rope_tables(*args, device="cpu", **kw)
