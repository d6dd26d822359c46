"""What the attention launcher plans, without a device: which kernel, how many workgroups, how much of the workspace."""

import ctypes

import pytest

from iris_amd import _native

COUNTERS = 4096  # arrival counters at a workspace's start
CUS = 256
DTYPES = {"bf16": (_native.DTYPE_BF16, 2), "fp16": (_native.DTYPE_F16, 2), "fp32": (_native.DTYPE_F32, 4)}
ADDRESS = 1 << 20  # (never followed)


def call(*, dtype="bf16", dim=64, requests=4, tokens=None, hq=4, hk=1, page=16, width=200, workspace=None, window=0, sinks=0, **other):
    """Arguments of a launch; ``tokens``: a prompt's, ``workspace``: its elements."""
    a = _native.AttentionArgs()
    for name in ("q", "k_cache", "v_cache", "block_table", "lengths", "out"):
        setattr(a, name, ADDRESS)
    a.dtype = DTYPES[dtype][0]
    a.requests, a.tokens, a.q_heads, a.k_heads, a.head_dim = requests, tokens or requests, hq, hk, dim
    if tokens is not None:
        a.query_starts = ADDRESS
    a.page_size, a.table_width, a.num_pages, a.stride_table = page, width, requests * width, width
    a.stride_qt, a.stride_qh, a.stride_ot, a.stride_oh = hq * dim, dim, hq * dim, dim
    a.stride_kc_page, a.stride_kc_row, a.stride_kc_head = page * hk * dim, hk * dim, dim
    a.stride_vc_page, a.stride_vc_row, a.stride_vc_head = page * hk * dim, hk * dim, dim
    a.window, a.sinks, a.scale = window, sinks, 0.125
    if workspace is not None:
        a.workspace, a.workspace_elems = ADDRESS, workspace
    for name, value in other.items():
        setattr(a, name, value)
    return a


def plan(**kw):
    info = _native.AttentionPlanInfo()
    assert _native.lib().iris_attention_plan(ctypes.byref(call(**kw)), CUS, ctypes.byref(info)) == 0
    return info


def slot(dim):
    """Elements of a partial result of 16 rows."""
    padded = 64 if dim <= 64 else 128 if dim <= 128 else 256
    return 16 * (padded + 4)


PROBLEMS = [dict(requests=4), dict(requests=1, width=2000, hq=8), dict(requests=64, width=512, dim=128, hq=8), dict(requests=300, dim=256, width=40),
            dict(requests=2, hq=40, hk=2, dim=128, width=4000), dict(requests=1, width=1), dict(requests=4, tokens=600),
            dict(requests=1, tokens=2000, dim=128, hq=8), dict(requests=8, tokens=30, width=300), dict(requests=2, tokens=900, dim=256),
            dict(requests=1, tokens=500, page=20, dim=128), dict(requests=16, width=4000, window=1000, sinks=4)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("problem", PROBLEMS, ids=lambda p: "-".join(f"{k}{v}" for k, v in p.items()))
def test_no_part_lies_outside_the_workspace(problem, dtype):
    """Of any size, among them those with room for the counters and less than one partial result."""
    dim = problem.get("dim", 64)
    for behind in sorted({-COUNTERS, -1, 0, 1, 500, slot(dim) - 1, slot(dim), slot(dim) + 1, 2 * slot(dim) - 1, 2 * slot(dim), 3 * slot(dim), 5 * slot(dim),
                          33 * slot(dim) - 1, 200 * slot(dim), 1000 * slot(dim) + 7, 4096 * slot(dim)}):
        p = plan(dtype=dtype, workspace=COUNTERS + behind, **problem)
        assert p.workspace_elems <= max(COUNTERS + behind, 0), f"{behind} elements behind the counters"
        assert p.workgroups >= 1 and p.parts >= 1
    assert plan(dtype=dtype, **problem).workspace_elems == 0


@pytest.mark.parametrize("behind", [1, 500, 16 * 68 - 1, 16 * 68, 2 * 16 * 68 - 1])
def test_less_workspace_than_two_parts_is_none(behind):
    full, none = plan(workspace=COUNTERS + 4096 * slot(64), hq=8), plan(hq=8)
    few = plan(workspace=COUNTERS + behind, hq=8)
    assert few.workspace_elems == 0 and few.workgroups == none.workgroups and few.kernel == none.kernel == _native.ATTENTION_DECODE
    assert full.workspace_elems > COUNTERS


def test_kernels():
    kernels = _native.ATTENTION_NOTHING, _native.ATTENTION_DECODE, _native.ATTENTION_PROMPT_TILES, _native.ATTENTION_PROMPT_ROWS
    assert [p.kernel for p in (plan(hq=0), plan(), plan(tokens=4000, requests=2, hq=8), plan(tokens=40, requests=8))] == list(kernels)
    assert plan(tokens=4000, requests=2, hq=8, dtype="fp32").kernel == _native.ATTENTION_PROMPT_ROWS
    assert plan(tokens=4000, requests=2, hq=8, page=20).kernel == _native.ATTENTION_PROMPT_ROWS
    info, lib = _native.AttentionPlanInfo(), _native.lib()
    for bad in (call(dim=60), call(scale=0.0), call(q=ADDRESS + 8)):
        assert lib.iris_attention_plan(ctypes.byref(bad), CUS, ctypes.byref(info)) == _native.HIP_ERROR_INVALID_VALUE
    assert lib.iris_attention_plan(ctypes.byref(call()), -1, ctypes.byref(info)) == _native.HIP_ERROR_INVALID_VALUE
    assert lib.iris_attention_plan(None, CUS, ctypes.byref(info)) == _native.HIP_ERROR_INVALID_VALUE


@pytest.mark.parametrize("page,row,kernel", [(1 << 20, 64, "TILES"), (1 << 20, 1 << 11, "ROWS"), (1 << 30, 1, "ROWS"), ((1 << 31) - 16, 8, "ROWS")])
def test_pages_past_what_31_bits_address_are_not_for_the_tiles(page, row, kernel):
    """The tiles address a page's rows with 31 bits: the others do with 64."""
    p = plan(tokens=4000, requests=2, hq=8, dim=8, width=1, page=page, stride_kc_row=row * 8, stride_vc_row=8)
    assert p.kernel == getattr(_native, f"ATTENTION_PROMPT_{kernel}")


@pytest.mark.parametrize("requests,hk", [(1, 1), (4, 1), (64, 1), (64, 8), (300, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_small_workspace_leaves_no_less_workgroups_than_none(requests, hk, dim):
    """Equal runs of the line for fewer workgroups than there are units would be slower than a unit a workgroup."""
    problem = dict(requests=requests, hq=8 * hk, hk=hk, dim=dim, width=400)
    none, units = plan(**problem), requests * hk
    for slots in (0, 1, 2, 3, 5, 9, 40, 64, 65, 200, 600, 1000, 4096):
        p = plan(workspace=COUNTERS + slots * slot(dim), **problem)
        assert p.workgroups >= min(units, none.workgroups)
        # split where that is more workgroups than units, or as many as there are without a workspace
        assert (p.workspace_elems > 0) == (slots // 2 >= min(units + 1, none.workgroups))
