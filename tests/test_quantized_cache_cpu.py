"""The cache in 8 bits without a device: struct layouts, refusals by the C-ABI and by the Python checks, plans."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

from iris_amd import _native, attention
from test_attention_checks_cpu import BF16, calls  # noqa: F401  (a fixture)
from test_attention_plans_cpu import COUNTERS, CUS, call, slot

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
STRUCTS = {"iris_cache_scales": _native.CacheScales, "iris_write_cache_args": _native.WriteCacheArgs, "iris_read_cache_args": _native.ReadCacheArgs}
INVALID = _native.HIP_ERROR_INVALID_VALUE
E4M3, E5M2, E8M0 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu


def test_struct_layouts_match_the_c_compiler(tmp_path):
    lines = []
    for cname, struct in STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{name} %zu\\n", offsetof({cname}, {name}));' for name, _ in struct._fields_]
    lines.append('printf("%d %d\\n", IRIS_DTYPE_E4M3, IRIS_DTYPE_E5M2);')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "iris_amd.h"\nint main(void){\n' + "\n".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    rows = iter(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n"))
    for cname, struct in STRUCTS.items():
        assert next(rows) == f"{cname} {ctypes.sizeof(struct)}"
        for name, _ in struct._fields_:
            assert next(rows) == f"{name} {getattr(struct, name).offset}"
    assert next(rows) == f"{_native.DTYPE_E4M3} {_native.DTYPE_E5M2}"


def refused(launch, args, cases):
    for field, value in cases:
        old = getattr(args, field)
        setattr(args, field, value)
        assert launch() == INVALID, (field, value)
        setattr(args, field, old)


def test_the_write_and_the_read_reject_bad_arguments_without_a_device():
    lib = _native.lib()
    for struct, entry, names in ((_native.WriteCacheArgs, lib.iris_write_quantized_cache_launch, "k v k_cache v_cache k_scales v_scales slots"),
                                 (_native.ReadCacheArgs, lib.iris_read_quantized_cache_launch,
                                  "k_out v_out k_cache v_cache k_scales v_scales block_table lengths starts")):
        assert entry(None, None) == INVALID
        a = struct()
        launch = lambda: entry(ctypes.byref(a), None)  # noqa: E731
        assert launch() == INVALID
        a.dtype, a.code, a.head_dim, a.page_size, a.block = _native.DTYPE_BF16, _native.DTYPE_E4M3, 64, 32, 16
        assert launch() == 0  # no token
        a.tokens, a.heads = 4, 2
        if struct is _native.WriteCacheArgs:
            a.num_slots = 96
        else:
            a.requests, a.num_pages, a.table_width, a.stride_table = 2, 3, 4, 4
        assert launch() == INVALID  # no tensors
        for name in names.split():  # (addresses that are never followed: every call here is refused before a launch)
            setattr(a, name, 4096)
        common = [("dtype", 3), ("code", 5), ("code", 0), ("head_dim", 72), ("head_dim", 272), ("head_dim", 0), ("page_size", 0), ("page_size", 40), ("page_size", 1 << 21), ("block", 8),
                  ("block", 0), ("block", 64), ("block", 24), ("tokens", -1), ("heads", -1), ("k_cache", 4104), ("v_cache", 4097), ("stride_kc_row", 72),
                  ("stride_vc_page", 8), ("stride_kt", 4), ("stride_vh", 7)] + [(name, 0) for name in names.split()]
        refused(launch, a, common)
        if struct is _native.WriteCacheArgs:
            refused(launch, a, [("num_slots", -1), ("num_slots", 1 << 31), ("k", 4100)])
        else:
            refused(launch, a, [("requests", -1), ("num_pages", -1), ("table_width", -1), ("table_width", 1 << 28), ("stride_table", 3), ("v_out", 4100)])


def quantized(code=_native.DTYPE_E4M3, block=16, **kw):
    a, s = call(**kw), _native.CacheScales()
    s.k_scales = s.v_scales = 1 << 20
    s.block, s.code = block, code
    return a, s


def test_attention_rejects_bad_arguments_without_a_device():
    lib = _native.lib()
    a, s = quantized(page=32, dim=64)
    launch = lambda: lib.iris_quantized_attention_launch(ctypes.byref(a), ctypes.byref(s), None)  # noqa: E731
    assert lib.iris_quantized_attention_launch(None, ctypes.byref(s), None) == INVALID
    assert lib.iris_quantized_attention_launch(ctypes.byref(a), None, None) == INVALID
    refused(launch, s, [("code", 2), ("code", 0), ("block", 0), ("block", 8), ("block", 64), ("block", 24), ("k_scales", 0), ("v_scales", 0)])
    refused(launch, s, [("stride_ks_page", 1 << 32), ("stride_vs_block", 1 << 32), ("stride_vs_page", -1)])
    refused(launch, a, [("head_dim", 72), ("head_dim", 264), ("page_size", 20), ("page_size", 1 << 21), ("stride_kc_page", 1 << 36), ("stride_vc_page", -16), ("stride_kc_row", 72), ("stride_vc_page", 8), ("q", 4104), ("k_cache", 4104),
                        ("stride_qt", 4), ("scale", math.nan), ("k_heads", 3), ("dtype", 6), ("num_pages", 0), ("stride_table", 2)])
    info, n = _native.AttentionPlanInfo(), ctypes.c_int()
    assert lib.iris_quantized_attention_plan(ctypes.byref(a), None, CUS, ctypes.byref(info)) == INVALID
    assert lib.iris_quantized_attention_plan(ctypes.byref(a), ctypes.byref(s), -1, ctypes.byref(info)) == INVALID
    assert lib.iris_quantized_attention_kernel_info(ctypes.byref(a), None, ctypes.byref(n), ctypes.byref(n)) == INVALID
    a.tokens = 0
    assert launch() == 0


@pytest.mark.parametrize("code", [_native.DTYPE_E4M3, _native.DTYPE_E5M2])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("problem", [dict(requests=4), dict(requests=1, width=2000, hq=8), dict(requests=64, width=512, dim=128, hq=8),
                                     dict(requests=300, dim=256, width=40), dict(requests=4, tokens=600), dict(requests=1, tokens=2000, dim=128, hq=8),
                                     dict(requests=8, tokens=30, width=300), dict(requests=2, tokens=900, dim=256)])
def test_no_part_lies_outside_the_workspace(problem, dtype, code):
    dim = problem.get("dim", 64)
    for behind in (-COUNTERS, -1, 0, 1, slot(dim) - 1, slot(dim), 2 * slot(dim) - 1, 2 * slot(dim), 5 * slot(dim), 33 * slot(dim) - 1, 1000 * slot(dim) + 7):
        info = _native.AttentionPlanInfo()
        a, s = quantized(code, dtype=dtype, workspace=COUNTERS + behind, **problem)
        assert _native.lib().iris_quantized_attention_plan(ctypes.byref(a), ctypes.byref(s), CUS, ctypes.byref(info)) == 0
        assert info.workspace_elems <= COUNTERS + max(behind, 0)


# ---- the Python checks -------------------------------------------------------


def cache(pages=6, page=32, heads=2, dim=64, code=E4M3, blocks=2):
    tensors = [torch.zeros((pages, page, heads, dim), dtype=code) for _ in range(2)]
    tensors += [torch.zeros((pages, blocks, heads), dtype=torch.uint8).view(E8M0) for _ in range(2)]
    return dict(zip(("k_cache", "v_cache", "k_scales", "v_scales"), tensors))


def write_operands(tokens=5, heads=2, dim=64, dtype=BF16, **kw):
    return dict(k=torch.zeros((tokens, heads, dim), dtype=dtype), v=torch.zeros((tokens, heads, dim), dtype=dtype), **cache(heads=heads, dim=dim, **kw),
                slots=torch.zeros(tokens, dtype=torch.int64))


def read_operands(tokens=5, requests=3, width=4, dtype=BF16, **kw):
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return dict(**cache(**kw), block_table=ints(requests, width), lengths=ints(requests), starts=ints(requests + 1),
                k_out=torch.zeros((tokens, 2, 64), dtype=dtype), v_out=torch.zeros((tokens, 2, 64), dtype=dtype))


def attend_operands(requests=3, width=4, dtype=BF16, **kw):
    c = cache(**kw)
    return dict(q=torch.zeros((requests, 4, 64), dtype=dtype), k_cache=c["k_cache"], v_cache=c["v_cache"],
                block_table=torch.zeros((requests, width), dtype=torch.int32), lengths=torch.zeros(requests, dtype=torch.int32),
                out=torch.zeros((requests, 4, 64), dtype=dtype), k_scales=c["k_scales"], v_scales=c["v_scales"])


def write(**a):
    attention.write_quantized_cache(*[a.pop(n) for n in ("k", "v", "k_cache", "v_cache", "k_scales", "v_scales", "slots")], **a)


def read(**a):
    attention.read_quantized_cache(*[a.pop(n) for n in ("k_cache", "v_cache", "k_scales", "v_scales", "block_table", "lengths", "starts", "k_out", "v_out")], **a)


def decode(**a):
    attention.decode_attention(*[a.pop(n) for n in ("q", "k_cache", "v_cache", "block_table", "lengths", "out")], **a)


CALLS = {"write": (write, write_operands), "read": (read, read_operands), "decode": (decode, attend_operands)}


@pytest.mark.parametrize("name", list(CALLS))
def test_what_the_checks_hand_over(calls, name):  # noqa: F811
    run, operands = CALLS[name]
    run(**operands())
    entry, args = calls.launched.pop()
    scales = args
    if name == "decode":
        assert entry == "iris_quantized_attention_launch"
        args, scales = args
    else:
        assert entry == f"iris_{name}_quantized_cache_launch"
    assert (scales.block, scales.code, args.page_size, args.head_dim) == (16, _native.DTYPE_E4M3, 32, 64)
    assert (scales.stride_ks_page, scales.stride_ks_block, scales.stride_ks_head) == (4, 2, 1)
    assert (args.stride_kc_page, args.stride_kc_row, args.stride_kc_head) == (32 * 128, 128, 64)
    run(**operands(code=E5M2, blocks=1, dtype=torch.float32))
    args = calls.launched.pop()[1]
    args, scales = args if name == "decode" else (args, args)
    assert (scales.block, scales.code, args.dtype) == (32, _native.DTYPE_E5M2, _native.DTYPE_F32)
    # what the native code launched is not launched again
    calls.answer = 0
    run(**operands())
    calls.answer = INVALID
    with pytest.raises(ValueError, match="rejected"):
        run(**operands())
    assert not calls.launched


@pytest.mark.parametrize("name", list(CALLS))
def test_refusals_of_a_cache(calls, name):  # noqa: F811
    run, operands = CALLS[name]
    o = operands()
    scales = lambda pages=6, blocks=2, heads=2: torch.zeros((pages, blocks, heads), dtype=torch.uint8).view(E8M0)  # noqa: E731
    wrong = [
        (TypeError, dict(k_cache=o["k_cache"].view(torch.uint8))), (TypeError, dict(v_cache=o["v_cache"].view(E5M2))),
        (TypeError, dict(k_cache=o["k_cache"].to(BF16), v_cache=o["v_cache"].to(BF16))),
        (TypeError, dict(k_scales=o["k_scales"].view(torch.uint8))), (TypeError, dict(v_scales=torch.ones(6, 2, 2))),
        (TypeError, dict(v_scales=scales()[0])), (ValueError, dict(k_scales=scales(pages=5))), (ValueError, dict(k_scales=scales(heads=1))),
        (ValueError, dict(k_scales=scales(blocks=3))), (ValueError, dict(k_scales=scales(blocks=4), v_scales=scales(blocks=4))),
        (ValueError, dict(k_scales=scales(blocks=0), v_scales=scales(blocks=0))), (ValueError, dict(v_scales=scales(blocks=1))),
        (ValueError, dict(v_scales=None)), (ValueError, dict(k_scales=None)),
        (ValueError, dict(k_cache=torch.zeros((6, 64, 2, 64), dtype=E4M3))),
        (ValueError, dict(k_cache=torch.zeros((6, 32, 2, 80), dtype=E4M3), v_cache=torch.zeros((6, 32, 2, 80), dtype=E4M3))),
        (ValueError, dict(k_cache=torch.zeros(6 * 32 * 128 + 8, dtype=E4M3)[8:].view(6, 32, 2, 64))),
        (ValueError, dict(k_cache=torch.zeros((6, 32, 2, 128), dtype=E4M3)[..., ::2])),
        (TypeError, dict(status=torch.zeros(1))),
    ]
    for kind, change in wrong:
        with pytest.raises(kind):
            run(**dict(o, **change))
    assert not calls.launched


def test_refusals_of_heads_and_vectors(calls):  # noqa: F811
    o = write_operands()
    for kind, change in [(TypeError, dict(k=o["k"].double())), (TypeError, dict(v=o["v"].half())), (ValueError, dict(v=o["v"][:4])), (ValueError, dict(k=o["k"][:, :1])),
                         (ValueError, dict(k=o["k"][0])), (TypeError, dict(slots=o["slots"].int())), (ValueError, dict(slots=o["slots"][:4])),
                         (ValueError, dict(k=torch.zeros(5 * 128 + 1, dtype=BF16)[1:].view(5, 2, 64))),
                         (ValueError, dict(k=torch.zeros((5, 64, 2), dtype=BF16).transpose(1, 2)))]:
        with pytest.raises(kind):
            write(**dict(o, **change))
    o = read_operands()
    for kind, change in [(TypeError, dict(k_out=o["k_out"].to(E4M3))), (TypeError, dict(v_out=o["v_out"].float())), (ValueError, dict(v_out=o["v_out"][:3])),
                         (TypeError, dict(block_table=o["block_table"].long())), (ValueError, dict(block_table=o["block_table"][:1].expand(3, 4))),
                         (TypeError, dict(lengths=o["lengths"].long())), (ValueError, dict(lengths=o["lengths"][:2])), (ValueError, dict(starts=o["starts"][:3])),
                         (ValueError, dict(k_out=o["k_out"][:1].expand(5, 2, 64)))]:
        with pytest.raises(kind):
            read(**dict(o, **change))
    # head sizes that heads in 8 bits do not come in
    for dim in (8, 72, 272):
        with pytest.raises(ValueError, match="multiple of 16"):
            write(**write_operands(dim=dim))
    with pytest.raises(ValueError):
        decode(**dict(attend_operands(), q=torch.zeros((3, 3, 64), dtype=BF16), out=torch.zeros((3, 3, 64), dtype=BF16)))
    # a cache in 8 bits without its scales is no cache
    o = attend_operands()
    with pytest.raises(TypeError):
        decode(**{n: t for n, t in o.items() if "scales" not in n})
    assert not calls.launched


def test_outputs_lie_apart(calls):  # noqa: F811
    o = write_operands()
    room = torch.zeros(4 * 6 * 32 * 128, dtype=torch.uint8)
    apart = room.view(6, 32, 2, 256)
    write(**dict(o, k_cache=apart[..., :64].view(E4M3), v_cache=apart[..., 64:128].view(E4M3)))  # (keys and values side by side)
    done = len(calls.launched)
    both = room[:6 * 32 * 128].view(6, 32, 2, 64).view(E4M3)
    inside = room[:24].view(6, 2, 2).view(E8M0)
    for change in (dict(k_cache=both, v_cache=both), dict(v_scales=o["k_scales"]), dict(k_cache=both, v_scales=inside),
                   dict(k=room[:5 * 256].view(BF16).view(5, 2, 64), k_cache=both), dict(slots=room[:40].view(torch.int64), v_cache=both),
                   dict(k_cache=both[:1].expand(6, 32, 2, 64))):
        with pytest.raises(ValueError):
            write(**dict(o, **change))
    o = read_operands()
    for change in (dict(v_out=o["k_out"]), dict(k_out=room[:5 * 256].view(BF16).view(5, 2, 64), k_cache=both), dict(k_out=room[:5 * 256].view(BF16).view(5, 2, 64), k_scales=inside)):
        with pytest.raises(ValueError):
            read(**dict(o, **change))
    o = attend_operands()
    with pytest.raises(ValueError):
        decode(**dict(o, out=room[:3 * 512].view(BF16).view(3, 4, 64), v_scales=inside))
    assert len(calls.launched) == done


def test_gradients_and_tangents_that_would_be_lost_are_refused(calls):  # noqa: F811
    forward_ad = torch.autograd.forward_ad
    for run, o, names in ((write, write_operands(), ("k", "v")), (decode, attend_operands(), ("q", "out")), (read, read_operands(), ("k_out", "v_out"))):
        for name in names:
            with pytest.raises(RuntimeError, match="gradient"):
                run(**dict(o, **{name: o[name].clone().requires_grad_()}))
            with forward_ad.dual_level():
                with pytest.raises(RuntimeError, match="gradient"):
                    run(**dict(o, **{name: forward_ad.make_dual(o[name].clone(), torch.ones_like(o[name]))}))
    assert not calls.launched


def test_tensors_of_the_host_are_refused():
    for run, operands in CALLS.values():
        with pytest.raises(RuntimeError, match="must be on"):
            run(**operands())


def test_make_quantized_cache():
    k, v, ks, vs = attention.make_quantized_cache(3, 64, 2, 80, device="cpu")
    assert k.shape == v.shape == (3, 64, 2, 80) and k.dtype == E4M3 and ks.shape == vs.shape == (3, 1, 2) and ks.dtype == E8M0
    assert not k.float().any() and bool((ks.float() == 1).all())
    wide = cache(page=1, blocks=1)  # (expanded, so that it takes no memory)
    o = dict(read_operands(), **{n: t.expand(6, 1 << 21, 2, 64) for n, t in wide.items() if "cache" in n}, k_scales=wide["k_scales"], v_scales=wide["v_scales"])
    with pytest.raises(ValueError, match="at most 1048576"), pytest.MonkeyPatch.context() as m:
        m.setattr(attention, "_require_cuda", lambda what, t, device: None)
        read(**o)
    assert attention.make_quantized_cache(3, 64, 2, 80, block=16, dtype=E5M2, device="cpu")[3].shape == (3, 4, 2)
    for bad in (dict(block=8), dict(block=48), dict(block=0), dict(page_size=24), dict(page_size=1 << 21), dict(head_dim=72), dict(head_dim=512), dict(head_dim=0), dict(pages=-1)):
        with pytest.raises(ValueError):
            attention.make_quantized_cache(**dict(dict(pages=3, page_size=64, heads=2, head_dim=80, device="cpu"), **bad))
    with pytest.raises(TypeError):
        attention.make_quantized_cache(3, 64, 2, 80, dtype=BF16, device="cpu")
