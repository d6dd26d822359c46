"""Attention over a paged cache at the edges of what a caller may hand in."""

import ctypes

import pytest
import torch

import attention_reference as R
from attention_reference import BF16, F16, F32
from iris_amd import _native, attention
from test_block_tables_gpu import mixed, step
from test_paged_attention_gpu import Problem, dense_on_gpu

pytestmark = pytest.mark.gpu

COUNTERS = 4096  # arrival counters at a workspace's start


def slot(dim):
    """Elements of a partial result of 16 rows."""
    return 16 * ((64 if dim <= 64 else 128 if dim <= 128 else 256) + 4)


@pytest.mark.parametrize("news", [None, [40, 9]])
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128), (F32, 64)])
def test_nothing_is_written_behind_a_workspace(dtype, dim, news):
    for behind in (1, 500, slot(dim) - 1, slot(dim), 2 * slot(dim) - 1, 2 * slot(dim), 5 * slot(dim)):
        p = Problem([3000, 700], news, 8, 1, dim, dtype, 16)
        room = torch.zeros(COUNTERS + behind + 200 * slot(dim), device="cuda")
        room[COUNTERS + behind:] = -7
        for _ in range(2):
            p.out.fill_(-7)
            p.launch(room[:COUNTERS + behind])
            p.check()
        assert bool((room[COUNTERS + behind:] == -7).all()), f"{behind} elements behind the counters"
        assert bool((room[:COUNTERS].view(torch.int32) == 0).all())


def forget(p, first_row_at, page, entries=(-1, 1 << 30)):
    """Table entries of pages that no query of a request sees (its first one stands at ``first_row_at[i]``) become none."""
    for i, first in enumerate(first_row_at):
        for j in range(p.table.shape[1]):
            lo, hi = j * page, (j + 1) * page - 1  # its keys
            if lo >= p.sinks and hi < first - p.window + 1:
                p.table[i, j] = entries[j % 2]


@pytest.mark.parametrize("page", [16, 20, 64, 8])
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128), (F32, 64), (BF16, 256)])
@pytest.mark.parametrize("window,sinks", [(50, 0), (50, 3), (16, 0), (200, 70), (1, 0)])
def test_pages_behind_the_window_may_be_gone_for_single_tokens(window, sinks, dtype, dim, page):
    lengths = [500, 40, 51, 300, 0, 129]
    p = Problem(lengths, None, 4, 2, dim, dtype, page, window=window, sinks=sinks)
    forget(p, [n - 1 for n in lengths], page)
    p.launch()
    p.check()


@pytest.mark.parametrize("dtype,dim,page,hq,hk", [
    (BF16, 64, 16, 4, 2), (F16, 128, 16, 4, 2), (F32, 64, 16, 4, 2), (BF16, 256, 16, 4, 2), (BF16, 64, 20, 4, 2), (F16, 128, 20, 4, 2), (F32, 64, 20, 4, 2),
    (F16, 128, 64, 4, 2), (BF16, 64, 16, 48, 24), (F16, 128, 16, 48, 24), (BF16, 256, 64, 48, 24)])  # (tiles of 16 rows, and of 128)
@pytest.mark.parametrize("window,sinks", [(50, 0), (50, 3), (200, 70)])
def test_pages_behind_the_window_may_be_gone_for_prompts(window, sinks, dtype, dim, page, hq, hk):
    lengths, news = [500, 40, 700, 300], [40, 40, 130, 1]
    p = Problem(lengths, news, hq, hk, dim, dtype, page, window=window, sinks=sinks)
    forget(p, [n - new for n, new in zip(lengths, news)], page)
    p.launch()
    p.check()


@pytest.mark.parametrize("dtype,dim,heads", [(BF16, 128, 1), (F16, 64, 1), (F32, 64, 1), (BF16, 128, 20), (F16, 64, 20)])
def test_a_page_that_is_none_reaches_the_tiles_whose_rows_see_it(dtype, dim, heads):
    n, window, page = 700, 100, 16
    p = Problem([n], [n], heads, heads, dim, dtype, page, window=window)
    lo, hi = 304, 304 + page - 1  # its keys: rows 304 .. 418 see some of them
    p.table[0, lo // page] = -1
    p.launch()
    assert p.word.item() == attention.STATUS_BAD_INDEX
    out = p.out[:, 0].isnan()
    assert bool(out[lo:hi + window].all())
    assert not bool(out[:lo // 128 * 128].any()) and not bool(out[-(-(hi + window) // 128) * 128:].any())


@pytest.mark.parametrize("window,sinks", [(2 ** 32 + 16, 0), (2 ** 31 - 1, 0), (16, 2 ** 32), (16, 2 ** 31 - 1), (2 ** 31, 2 ** 40)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_windows_and_first_tokens_past_31_bits_are_all_keys(window, sinks, dtype):
    for news, heads in ((None, (4, 2)), ([200, 30], (4, 2)), ([200, 30], (80, 40))):
        p = Problem([300, 40], news, *heads, 64, dtype, 16, window=window, sinks=sinks)
        p.launch()
        p.check()


@pytest.mark.parametrize("size", [1e20, 1e25, 1e35])
@pytest.mark.parametrize("news", [70, 650, 1])
@pytest.mark.parametrize("room", [2, 30000], ids=["tight", "roomy"])
@pytest.mark.parametrize("steps", [14, 7])
def test_large_values_under_scores_that_grow(size, news, room, steps):
    """Averages of finite values are finite, whatever the scores of the keys before: bf16 has fp32's range, and products of weights and
    values must not leave it."""
    n, d = 700, 64
    p = Problem([n], [news] if news > 1 else None, 1, 1, d, BF16, 16, room=room)
    p.q_host[:] = 0
    p.q_host[..., 0] = 16
    p.q.copy_(p.q_host)
    p.k[0][..., 0] = (torch.arange(n) * steps // n).to(BF16)[:, None] * (19 / steps)  # 38 more at the end than at the beginning
    p.k[0][..., 0] = p.k[0][..., 0].float().round().to(BF16)
    p.v[0] = (p.v[0].float() * size).to(BF16)
    for j in range(-(-n // 16)):
        for cache, rows in ((p.k_cache, p.k[0]), (p.v_cache, p.v[0])):
            part = rows[16 * j:16 * j + 16].cuda()
            cache[p.table[0, j], :len(part)] = part
    p.launch()
    p.check()
    p.out.fill_(-7)
    p.launch(None)  # (in one part)
    p.check()


def test_tangents_are_refused():
    forward_ad = torch.autograd.forward_ad
    p = Problem([20, 30], None, 4, 2, 64, BF16, 16)
    k, cos = torch.zeros((2, 2, 64), dtype=BF16, device="cuda"), torch.ones((4, 32), device="cuda")
    positions = torch.zeros(2, dtype=torch.int32, device="cuda")

    def attend(q):
        attention.decode_attention(q, p.k_cache, p.v_cache, p.table, p.lens, p.out)

    def turn(q):
        attention.qk_norm_rope(q, k, positions, cos, cos, p.out, torch.empty_like(k))

    def back(q):
        attention.qk_norm_rope_backward(q, k, p.q, k, positions, cos, cos, p.out, torch.empty_like(k))

    for call in (attend, turn, back):
        call(p.q)
        p.out.fill_(-7)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="gradient"):
            call(forward_ad.make_dual(p.q, torch.ones_like(p.q)))
        assert bool((p.out == -7).all())
        call(p.q.detach())


def test_outputs_over_other_operands_are_refused():
    """(What is refused and what is not: the checks' own tests, without a GPU.)"""
    wide = torch.zeros((6, 10, 64), dtype=BF16, device="cuda")
    q, k, fresh = wide[:, :4], wide[:, 4:6], torch.zeros((6, 4, 64), dtype=BF16, device="cuda")
    positions, cos = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.ones((4, 32), device="cuda")
    attention.qk_norm_rope(q, k, positions, cos, cos, q, k)
    with pytest.raises(ValueError, match="shares memory"):
        attention.qk_norm_rope(q, k, positions, cos, cos, wide[:, 1:5], k)
    attention.qk_norm_rope_backward(fresh, fresh[:, :2], q, k, positions, cos, cos, q, k)
    with pytest.raises(ValueError, match="shares memory"):
        attention.qk_norm_rope_backward(fresh, fresh[:, :2], q, k, positions, cos, cos, fresh[:, :4], fresh[:, 1:3])
    p = Problem([20, 30], None, 4, 2, 64, BF16, 16)
    with pytest.raises(ValueError, match="shares memory"):
        attention.decode_attention(p.q, p.k_cache, p.v_cache, p.table, p.lens, p.k_cache.view(-1, 4, 64)[:2])


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F32, 64)])
def test_outputs_in_place_of_the_queries(dtype, dim):
    for lengths, news in (([3000, 700, 0], None), ([900, 300], [900, 40]), ([4000], [20])):
        p = Problem(lengths, news, 8, 1, dim, dtype, 16)
        p.out = p.q
        p.launch()
        p.check()


# ---- which launch a call is --------------------------------------------------


def planned(p, workspace, monkeypatch):
    """What the launcher does with a problem's call (which is not made)."""
    got = []
    with monkeypatch.context() as m:
        m.setattr(_native, "host", lambda: Declining())
        m.setattr(attention, "_launch", lambda name, args, device: got.append(args))
        p.launch(workspace)
    info = _native.AttentionPlanInfo()
    assert _native.lib().iris_attention_plan(ctypes.byref(got[0]), 0, ctypes.byref(info)) == 0
    return info


class Declining:
    """A native module that takes no call."""

    overlap = staticmethod(_native.host().overlap)

    def __getattr__(self, name):
        return lambda *args: attention.DECLINED


@pytest.mark.parametrize("requests", [63, 64, 65, 150])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_prompts_of_about_as_many_requests_as_are_put_in_order(dtype, dim, requests, monkeypatch):
    """Up to 64 requests' row tiles start by the keys they see, those of more in the requests' order."""
    news = [60 + (7 * i) % 41 for i in range(requests)]
    lengths = [n + (13 * i) % 200 for i, n in enumerate(news)]
    p = Problem(lengths, news, 40, 8, dim, dtype, 16)
    assert planned(p, None, monkeypatch).kernel == _native.ATTENTION_PROMPT_TILES
    p.launch()
    assert p.word.item() == 0
    want, spread = dense_on_gpu(p)
    off, bound = (p.out.double().cpu() - want).abs(), R.attention_error(dtype, want, spread, dim)
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item()} times the bound"


@pytest.mark.parametrize("news,hq,hk,kernel", [([300, 200], 8, 1, _native.ATTENTION_PROMPT_TILES), ([9, 4], 4, 2, _native.ATTENTION_PROMPT_ROWS)])
def test_prompts_in_a_captured_graph_whose_parts_join(news, hq, hk, kernel, monkeypatch):
    most = [3000, 2100]
    p = Problem(most, news, hq, hk, 128, BF16, 16)
    workspace = attention.make_workspace(128)
    info = planned(p, workspace, monkeypatch)
    assert info.kernel == kernel and info.parts > 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            p.launch(workspace)
    torch.cuda.synchronize()
    k, v, tokens = p.k, p.v, sum(news)
    for lengths, first in ((most, news[0]), ([1000, 700], tokens - 1), ([3000, 40], 3), ([500, 0], tokens), (most, news[0])):
        news = [first, tokens - first]
        p.lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        p.starts.copy_(torch.tensor([0, first, tokens], dtype=torch.int32))
        p.lengths, p.news = lengths, news
        p.k, p.v = [x[:n] for x, n in zip(k, lengths)], [x[:n] for x, n in zip(v, lengths)]
        p.out.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        p.check()
        eager = p.out.clone()
        p.launch(workspace)
        assert torch.equal(p.out, eager)
    assert bool((workspace[:COUNTERS].view(torch.int32) == 0).all())


# ---- the Python code's own launches: what the native module declines ----------


@pytest.mark.parametrize("news", [None, [300, 20]])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F32, 64)])
def test_attention_launched_by_the_python_code_is_the_same(dtype, dim, news, monkeypatch):
    p = Problem([1500, 200], news, 8, 2, dim, dtype, 16, window=400, sinks=3, fused=True)
    workspace = p.launch()
    out, lse = p.out.clone(), p.lse.clone()
    p.out.fill_(-7)
    p.lse.fill_(-7)
    monkeypatch.setattr(_native, "host", lambda: Declining())
    p.launch(workspace)
    assert torch.equal(p.out, out) and torch.equal(p.lse, lse)
    p.check()


def test_heads_launched_by_the_python_code_are_the_same(monkeypatch):
    t, hq, hk, d = 50, 6, 2, 128
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn((t, (hq + 2 * hk) * d), generator=g).to(BF16).cuda()
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split((hq * d, hk * d, hk * d), 1))
    wq, wk = (1 + torch.randn(d, generator=g).cuda() * 0.1 for _ in range(2))
    cos, sin = attention.rope_tables(64, d)
    positions, slots = torch.arange(t, device="cuda", dtype=torch.int32), torch.randperm(64, generator=g)[:t].cuda()

    def run():
        caches = torch.zeros((2, 4, 16, hk, d), dtype=BF16, device="cuda")
        q_out, k_out, dq, dk = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, q, k))
        attention.qk_norm_rope(q, k, positions, cos, sin, q_out, k_out, q_weight=wq, k_weight=wk, v=v, k_cache=caches[0], v_cache=caches[1], slots=slots)
        dwq, dwk = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
        attention.qk_norm_rope_backward(q, k, q, k, positions, cos, sin, dq, dk, q_weight=wq, k_weight=wk, dq_weight=dwq, dk_weight=dwk,
                                        workspace=attention.make_gradient_workspace(d))
        return caches, q_out, k_out, dq, dk, dwq, dwk

    native = run()
    monkeypatch.setattr(_native, "host", lambda: Declining())
    assert all(torch.equal(a, b) for a, b in zip(native, run()))


def test_block_tables_launched_by_the_python_code_are_right(monkeypatch):
    monkeypatch.setattr(_native, "host", lambda: Declining())
    step(mixed(70, 5), 16, seed=5, table_stride=3)


@pytest.mark.parametrize("dtype,dim", [(BF16, 8), (F16, 16), (BF16, 24), (F16, 72), (BF16, 120), (F16, 136), (BF16, 248), (F32, 4), (F32, 60), (F32, 132), (F32, 252)])
def test_odd_head_sizes(dtype, dim):
    for lengths, news, heads in (([300, 40, 0], None, (6, 2)), ([200, 33, 7], [150, 33, 1], (6, 2)), ([400, 200], [300, 130], (40, 20))):
        p = Problem(lengths, news, *heads, dim, dtype, 16)
        p.launch()
        p.check()


@pytest.mark.parametrize("slots", [6, 7, 33, 100, 513, 1000])
def test_single_tokens_in_parts_of_a_small_workspace(slots, monkeypatch):
    p = Problem([3000, 700], None, 8, 1, 64, BF16, 16)
    workspace = torch.zeros(COUNTERS + slots * slot(64), device="cuda")
    info = planned(p, workspace, monkeypatch)
    assert COUNTERS < info.workspace_elems <= len(workspace) and info.workgroups > 2
    p.launch(workspace)
    p.check()
    first = p.out.clone()
    p.launch(workspace)
    assert torch.equal(p.out, first) and bool((workspace[:COUNTERS].view(torch.int32) == 0).all())


def test_an_error_that_an_earlier_call_left_is_not_a_launchs(monkeypatch):
    """What a call reports is its own launch's status, by the native module's way and by the Python code's."""
    t, hq, hk, d = 5, 4, 2, 64
    q, k, dq_out, dk_out = (torch.randn((t, h, d), device="cuda").to(BF16) for h in (hq, hk, hq, hk))
    cos, sin = attention.rope_tables(16, d)
    positions, weight = torch.arange(t, device="cuda", dtype=torch.int32), torch.ones(d, device="cuda")
    q_out, k_out, dq, dk, dw = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty_like(k), torch.empty(d, device="cuda")
    room = attention.make_gradient_workspace(d)
    p, prompts = Problem([50, 20], None, 4, 2, 64, BF16, 16), Problem([50, 20], [30, 20], 4, 2, 64, BF16, 16)
    workspace = attention.make_workspace(64)
    i32, i64 = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    tables = [i32.clone() for _ in range(2)] + [torch.zeros((3, 4), dtype=torch.int32, device="cuda"), i32.clone(), i64[:2].clone(), 16]
    written = dict(lengths=i32.clone(), pool_state_out=i64[:2].clone(), query_starts=torch.zeros(4, dtype=torch.int32, device="cuda"),
                   positions=i32.clone(), slots=i64.clone())
    calls = [lambda: p.launch(workspace), lambda: prompts.launch(workspace), lambda: attention.qk_norm_rope(q, k, positions, cos, sin, q_out, k_out),
             lambda: attention.qk_norm_rope_backward(dq_out, dk_out, q, k, positions, cos, sin, dq, dk, q_weight=weight, dq_weight=dw, workspace=room),
             lambda: attention.build_block_tables(*tables, **written)]
    torch.cuda.synchronize()
    loaded = {line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line}
    assert len(loaded) == 1
    hip = ctypes.CDLL(loaded.pop())
    for host in (_native.host(), Declining()):
        monkeypatch.setattr(_native, "host", lambda: host)
        for call in calls:
            call()
            assert _native.lib().iris_hip_set_device(9999) != 0
            call()
            assert hip.hipGetLastError() == 101  # (still there for whom it concerns; cleared)
    torch.cuda.synchronize()
    p.check()
    prompts.check()
