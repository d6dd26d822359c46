"""Attention over a cache in 8 bits against the definition in 64 bits.  What codes and scales stand for is exact in the heads' type, so
the bound is that of attention over a cache of that type."""

import ctypes
import math

import pytest
import torch

import attention_reference as R
from attention_reference import BF16, F16, F32
from iris_amd import _native, attention
from quantized_reference import E4M3, E5M2, Quantized
from test_attention_edges_gpu import Declining, forget

pytestmark = pytest.mark.gpu


def run(*args, scale=None, workspace="own", **kw):
    p = Quantized(*args, **kw)
    p.launch(workspace, scale)
    p.check(scale)
    return p


LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 300, 700]


@pytest.mark.parametrize("code", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 192, 256])
def test_decode_types_and_head_sizes(dtype, dim, code):
    run(LENGTHS, None, 4, 2, dim, dtype, 16, code=code)


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 1), (16, 1), (17, 1), (40, 2), (6, 3)])
def test_decode_heads(hq, hk):
    run(LENGTHS, None, hq, hk, 128, BF16, 32, block=16)


@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (48, 48), (64, 32), (128, 128), (256, 64), (80, 80)])
@pytest.mark.parametrize("heads_first,strided", [(False, True), (True, False)])
def test_decode_pages_and_blocks(page, block, heads_first, strided):
    run(LENGTHS, None, 4, 2, 64, BF16, page, block=block, heads_first=heads_first, strided=strided, spread=3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (100, 4), (256, 70), (1000, 3)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_decode_window_and_first_tokens(window, sinks, dtype):
    run(LENGTHS, None, 8, 2, 128, dtype, 32, block=16, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_blocks_of_very_different_sizes(dtype):
    """Scales 2^-12 to 2^12 apart; in fp16 some of the values are subnormal."""
    run([33, 300, 90], None, 4, 2, 64, dtype, 16, spread=6 if dtype == F16 else 12, scale=2.0 ** -12)
    run([33, 300, 90], [20, 300, 3], 4, 2, 64, dtype, 16, spread=6 if dtype == F16 else 12, scale=2.0 ** -12)


def test_decode_long_contexts_are_split():
    run([20011, 1, 9000, 64], None, 8, 2, 128, BF16, 16, code=E5M2)
    run([9001], None, 4, 1, 256, F16, 64, block=32)


def test_decode_many_requests():
    run([(37 * i) % 301 for i in range(400)], None, 4, 1, 64, F16, 16, strided=True)


def test_decode_with_little_or_no_workspace_gives_the_same():
    args = ([5000, 700, 0, 3001], None, 8, 2, 64, BF16, 32)
    for workspace in ("own", None, torch.zeros(4096 + 12 * 16 * 68, device="cuda")):
        run(*args, workspace=workspace)


def test_a_workspace_serves_many_launches_and_gives_the_same_bits():
    p = run([7000, 300, 2000], None, 8, 1, 128, BF16, 16)
    workspace = p.launch()
    first = p.out.clone()
    for _ in range(5):
        p.out.fill_(-7)
        p.launch(workspace)
        assert torch.equal(first, p.out)
    q = run([900, 1200], [900, 1100], 8, 2, 128, F16, 16, workspace=workspace)
    assert q.word.item() == 0


@pytest.fixture(params=[True, False])
def room(request):
    """A workspace, or none: then the rows of few tiles are not split."""
    return "own" if request.param else None


PROMPTS = ([3, 18, 200, 64, 0, 500, 129], [3, 5, 200, 1, 0, 130, 129])


@pytest.mark.parametrize("code", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 192, 256])
def test_prompt_types_and_head_sizes(dtype, dim, code, room):
    run(*PROMPTS, 4, 2, dim, dtype, 16, code=code, workspace=room)


@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (48, 48), (64, 32), (128, 128), (80, 80)])
@pytest.mark.parametrize("heads_first,strided", [(False, True), (True, False)])
def test_prompt_pages_and_blocks(page, block, heads_first, strided):
    run([300, 190, 77], [300, 140, 77], 6, 2, 128, BF16, page, block=block, heads_first=heads_first, strided=strided, spread=3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (100, 4), (256, 70)])
@pytest.mark.parametrize("dtype,hq,hk,dim", [(BF16, 8, 1, 128), (F16, 10, 2, 64), (BF16, 4, 2, 256), (F32, 4, 2, 64)])
def test_prompt_window_and_first_tokens(window, sinks, dtype, hq, hk, dim):
    run([700, 333, 90], [600, 100, 90], hq, hk, dim, dtype, 32, block=16, window=window, sinks=sinks)


def test_prompt_pieces_behind_a_long_context(room):
    run([3000, 2800, 41, 1999], [30, 9, 3, 1], 8, 1, 128, BF16, 16, workspace=room)


def test_prompt_of_more_queries_than_keys_leaves_rows_empty(room):
    p = run([5, 40, 0], [9, 300, 4], 8, 2, 64, BF16, 16, workspace=room)
    assert bool((p.out[:4] == 0).all())


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 256), (F32, 64)])
@pytest.mark.parametrize("window", [0, 48])
@pytest.mark.parametrize("what", ["code", "scale", "range"])
def test_a_value_that_is_no_number_reaches_only_the_queries_that_see_it(dtype, dim, window, what, room):
    """A code, or the scale of its block, is no number; or a code times its scale is past the type's numbers."""
    p = Quantized([400, 90], [380, 90], 8, 2, dim, dtype, 16, window=window)
    at, block = 333, range(320, 336)
    page = int(p.table[0, at // 16])
    if what == "code":
        p.v_cache.view(torch.uint8)[page, at % 16, 1, 3] = 0x7F
        block = [at]
    elif what == "scale":
        p.v_scales.view(torch.uint8)[page, 0, 1] = 255
    else:
        p.v_cache.view(torch.uint8)[page, at % 16, 1, 3] = 0x7E
        p.v_scales.view(torch.uint8)[page, 0, 1] = 254
    p.launch(room)
    sees = lambda position: any(k <= position and (not window or position - k < window) for k in block)  # noqa: E731
    p.check(skip=lambda request, position: request == 0 and sees(position))
    if what != "range":
        hit = torch.tensor([sees(20 + i) for i in range(380)])
        got = p.out[:380, 4:].float().cpu()
        assert bool(got[hit, :, 3].isnan().all()) and not bool(got[~hit].isnan().any())


@pytest.mark.parametrize("what", ["code", "scale"])
def test_a_key_that_is_no_number_reaches_only_the_queries_that_see_it(what, room):
    p = Quantized([400, 90], [380, 90], 8, 2, 128, BF16, 16)
    page = int(p.table[0, 20])
    if what == "code":
        p.k_cache.view(torch.uint8)[page, 15, 0, 100] = 0xFF
    else:
        p.k_scales.view(torch.uint8)[page, 0, 0] = 255
    first = 335 if what == "code" else 320
    p.launch(room)
    p.check(skip=lambda request, position: request == 0 and position >= first)
    assert bool(p.out[first - 20:380, :4].isnan().all())


def test_decode_hidden_keys_are_not_read_as_numbers():
    for what in ("codes", "scales"):
        p = Quantized([100, 64, 33], None, 4, 2, 128, BF16, 16, window=20)
        for name in ("k", "v"):  # pages behind the windows: they may hold anything
            for r, gone in ((0, 5), (1, 2)):
                if what == "codes":
                    getattr(p, name + "_cache").view(torch.uint8)[p.table[r, :gone].long()] = 0x7F
                else:
                    getattr(p, name + "_scales").view(torch.uint8)[p.table[r, :gone].long()] = 255
        p.launch()
        p.check()


@pytest.mark.parametrize("dtype,dim,news", [(BF16, 128, None), (F32, 64, None), (F16, 64, [200, 30]), (BF16, 256, [200, 30]), (BF16, 128, [3, 1])])
def test_pages_behind_the_window_may_be_gone(dtype, dim, news):
    lengths = [300, 90]
    p = Quantized(lengths, news, 4, 2, dim, dtype, 16, window=40, sinks=3)
    firsts = [n - (1 if news is None else m) for n, m in zip(lengths, news or [1, 1])]
    forget(p, firsts, 16)
    p.launch()
    p.check()


@pytest.mark.parametrize("news", [None, [200, 41]])
def test_a_page_outside_the_cache_is_reported(news):
    p = Quantized([300, 41], news, 4, 2, 128, BF16, 16)
    p.table[0, 3] = p.k_cache.shape[0]
    p.launch()
    assert p.word.item() == attention.STATUS_BAD_INDEX
    rows = 1 if news is None else 200
    assert bool(p.out[:rows].isnan().all())
    p.word.zero_()
    p.check(skip=lambda request, position: request == 0)


def test_views_streams_and_scale():
    p = Quantized([300, 41, 0, 77], [300, 2, 0, 77], 6, 2, 64, F16, 32, block=16, fused=True, strided=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        p.launch(scale=0.3)
    torch.cuda.current_stream().wait_stream(stream)
    p.check(0.3)
    q = Quantized([300, 41, 0, 77], None, 6, 2, 64, F16, 32, block=16, fused=True)
    q.launch(scale=0.3)
    q.check(0.3)


@pytest.mark.parametrize("dtype,dim,news", [(BF16, 128, None), (F32, 80, None), (F16, 64, [100, 300]), (BF16, 192, [100, 300])])
def test_launched_by_the_python_code_it_is_the_same(dtype, dim, news, monkeypatch):
    p = run([400, 300], news, 8, 2, dim, dtype, 32, block=16, strided=True)
    first = p.out.clone()
    p.out.fill_(-7)
    with monkeypatch.context() as m:
        m.setattr(_native, "host", lambda: Declining())
        p.launch()
    assert torch.equal(first, p.out)


def test_a_server_steps_in_a_captured_graph():
    """Tables, norms and rotation, the write into the cache and attention over it, recorded once and replayed as the contexts grow; eager
    work stands between the replays, and every one is checked."""
    page, block, hq, hk, d, requests, steps = 16, 16, 8, 2, 64, 3, 40
    g = torch.Generator().manual_seed(5)
    x = torch.randn((steps, requests, (hq + 2 * hk), d), generator=g).to(BF16).cuda()
    cos, sin = attention.rope_tables(256, d)
    ints = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    cached, new, lengths, starts = ints(requests), ints(requests) + 1, ints(requests), ints(requests + 1)
    cached += torch.tensor([0, 15, 3], device="cuda")
    pages = 16
    caches = attention.make_quantized_cache(pages, page, hk, d, block=block)
    table, pool = ints(requests, 5), torch.randperm(pages, generator=g).int().cuda()
    state, state_out = torch.tensor([0, pages], device="cuda"), ints(2, dtype=torch.int64)
    positions, slots = ints(requests), ints(requests, dtype=torch.int64)
    heads, out, word = x[0].clone(), torch.zeros((requests, hq, d), dtype=BF16, device="cuda"), ints(1)
    keys, workspace = torch.zeros((requests, hk, d), dtype=BF16, device="cuda"), attention.make_workspace(d)
    # the first tokens of requests 1 and 2
    first = torch.randn((18, hk, d), generator=g).to(BF16).cuda()
    attention.build_block_tables(ints(requests), cached.clone(), table, pool, state, page, lengths=lengths, pool_state_out=state_out,
                                 query_starts=starts, positions=ints(18), slots=(early := ints(18, dtype=torch.int64)), status=word)
    attention.write_quantized_cache(first, first, *caches, early, status=word)
    state.copy_(state_out)

    def step():
        attention.build_block_tables(cached, new, table, pool, state, page, lengths=lengths, pool_state_out=state_out, query_starts=starts,
                                     positions=positions, slots=slots, status=word)
        q, k, v = heads.split((hq, hk, hk), 1)
        attention.qk_norm_rope(q, k, positions, cos, sin, q, keys, status=word)
        attention.write_quantized_cache(keys, v, *caches, slots, status=word)
        attention.decode_attention(q, caches[0], caches[1], table, lengths, out, workspace=workspace, status=word, k_scales=caches[2], v_scales=caches[3])

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    saved = [t.clone() for t in (table, pool, *(c.view(torch.uint8) for c in caches))]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        for t, was in zip((table, pool, *(c.view(torch.uint8) for c in caches)), saved):
            t.copy_(was)
        with torch.cuda.graph(graph, stream=stream):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    for t in range(steps):
        heads.copy_(x[t])
        graph.replay()
        torch.cuda.synchronize()
        assert word.item() == 0
        # the same over what the cache holds now, in 64 bits
        total = int(lengths.sum())
        whole = [torch.empty((total, hk, d), dtype=F32, device="cuda") for _ in range(2)]
        ends = torch.cat((ints(1), lengths.cumsum(0).int()))
        attention.read_quantized_cache(*caches, table, lengths, ends, *whole, status=word)
        for i in range(requests):
            k, v = (w[int(ends[i]):int(ends[i + 1])] for w in whole)
            want, _, spread = R.attention(heads[i:i + 1, :hq], k, v, len(k) - 1, d ** -0.5)
            assert bool(((out[i:i + 1].double().cpu() - want).abs() <= R.attention_error(BF16, want, spread, d)).all())
        assert bool((whole[1][ends[1:].long() - 1] - x[t, :, hq + hk:]).abs().max() <= 2.0 ** -4 * x.abs().max())
        cached.copy_(lengths)
        state.copy_(state_out)


@pytest.mark.parametrize("news", [None, [300], [9]])
def test_addresses_past_32_bits(news):
    """A cache of 6 GB of codes a side, whose last pages are a request's."""
    p = Quantized([500], news, 4, 2, 128, BF16, 64, block=32)
    pages, held = (6 << 30) // (64 * 2 * 128), p.k_cache.shape[0]
    for name in ("k", "v"):
        cache = torch.empty((pages, 64, 2, 128), dtype=E4M3, device="cuda")
        scales = torch.empty((pages, 2, 2), dtype=torch.uint8, device="cuda")
        cache.view(torch.uint8)[-held:] = getattr(p, name + "_cache").view(torch.uint8)
        scales[-held:] = getattr(p, name + "_scales").view(torch.uint8)
        setattr(p, name + "_cache", cache)
        setattr(p, name + "_scales", scales.view(torch.float8_e8m0fnu))
    count = R.cdiv(500, 64)
    p.table[0, :count] += pages - held
    p.launch()
    p.check()


@pytest.mark.parametrize("news", [None, [3, 2, 0]])
def test_without_a_page(news):
    """A cache or a table without a page: rows that would see a key are NaN and reported, the others zeros."""
    p = Quantized([0, 5, 0], news, 4, 2, 64, BF16, 16)
    caches = attention.make_quantized_cache(0, 16, 2, 64)
    p.k_cache, p.v_cache, p.k_scales, p.v_scales = caches
    p.table = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    p.launch()
    sees = [False, True, False] if news is None else [False] * 3 + [True] * 2
    assert p.out.isnan().all(-1).all(-1).tolist() == sees and p.word.item() == attention.STATUS_BAD_INDEX
    assert bool((p.out[~torch.tensor(sees, device="cuda")] == 0).all())


@pytest.mark.parametrize("dtype,dim,news", [(BF16, 128, [300, 90]), (F16, 64, [300, 90]), (F32, 64, None), (BF16, 256, None)])
def test_outputs_in_place_of_the_queries(dtype, dim, news):
    p = run([400, 90], news, 8, 2, dim, dtype, 16)
    want = p.out.clone()
    p.out = p.q
    p.launch()
    assert torch.equal(p.q, want)


def test_nothing_is_written_behind_a_workspace():
    for news in (None, [40, 9]):
        for behind in (1, 16 * 132 - 1, 2 * 16 * 132, 5 * 16 * 132 + 3):
            p = Quantized([3000, 700], news, 8, 1, 128, BF16, 16)
            room = torch.zeros(4096 + behind + 200 * 16 * 132, device="cuda")
            room[4096 + behind:] = -7
            for _ in range(2):
                p.out.fill_(-7)
                p.launch(room[:4096 + behind])
                p.check()
            assert bool((room[4096 + behind:] == -7).all()) and bool((room[:4096].view(torch.int32) == 0).all())


@pytest.mark.parametrize("news,hq,hk,kernel", [([400, 130], 8, 1, _native.ATTENTION_PROMPT_TILES), ([9, 3], 8, 1, _native.ATTENTION_PROMPT_ROWS)])
def test_prompts_in_a_captured_graph(news, hq, hk, kernel):
    """Parts that join, replayed over other numbers and shorter contexts with eager work in between; rows past the last request's stay."""
    p = Quantized([1500, 900], news, hq, hk, 128, BF16, 16)
    tokens = sum(news)
    q = torch.zeros((tokens + 7, hq, 128), dtype=BF16, device="cuda")
    out = torch.full_like(q, -7.0)
    q[:tokens] = p.q
    p.q, p.out, p.lse = q, out, torch.full((tokens + 7, hq), -7.0, device="cuda")
    if kernel == _native.ATTENTION_PROMPT_TILES:  # (a table this wide has many keys to see)
        p.table = torch.cat((p.table, torch.full((2, 400), 1 << 30, dtype=torch.int32, device="cuda")), 1)
    workspace = attention.make_workspace(128)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        p.launch(workspace)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            p.launch(workspace)
    torch.cuda.current_stream().wait_stream(stream)
    for shorter in (0, 100, 0, 333, 700):
        p.lens.copy_(torch.tensor([1500 - shorter, 900 - shorter // 2], device="cuda"))
        p.q[:tokens] = torch.randn_like(p.q[:tokens]) * 1.5
        p.out.fill_(-7)
        graph.replay()
        got = p.out.clone()
        p.out.fill_(-7)
        p.launch(workspace)  # eager, the same
        assert torch.equal(got, p.out) and p.word.item() == 0
        assert bool((got[tokens:] == -7).all()) and bool((p.lse[tokens:] == -7).all())
        at = 0
        for i, (n, new) in enumerate(zip(p.lens.tolist(), news)):
            rows = slice(at, at + 2), slice(at + new - 2, at + new)
            for r, first in zip(rows, (n - new, n - 2)):
                want, _, spread = R.attention(p.q[r], p.k[i][:n], p.v[i][:n], first, 128 ** -0.5)
                assert bool(((got[r].double().cpu() - want).abs() <= R.attention_error(BF16, want, spread, 128)).all())
            at += new


def test_calls_on_two_streams_at_once():
    """Single tokens, prompts and reads over one cache from two streams, each with its own workspace, while a third call writes another cache."""
    p, q = Quantized([5000, 700, 3001], None, 8, 2, 128, BF16, 16), Quantized([900, 1200], [900, 300], 8, 2, 128, BF16, 16, seed=3)
    spare = attention.make_quantized_cache(64, 16, 2, 128)
    k = torch.randn((1000, 2, 128), device="cuda", dtype=BF16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [attention.make_workspace(128) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            p.launch(spaces[0])
            attention.write_quantized_cache(k, k, *spare, torch.arange(1000, device="cuda"))
        with torch.cuda.stream(streams[1]):
            q.launch(spaces[1])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    p.check()
    q.check()


@pytest.mark.parametrize("requests,new,hq,hk", [(140, 32, 8, 2), (270, 16, 8, 1)])
def test_prompts_of_one_row_tile_each(requests, new, hq, hk):
    """As many row tiles as places, every other one empty: they are dealt out in another order."""
    lengths = [new + (7 * i) % 53 for i in range(requests)]
    run(lengths, [new] * (requests - 1) + [new - 3], hq, hk, 64, BF16, 16)


@pytest.mark.parametrize("requests", [65, 150])
def test_prompts_of_many_requests(requests):
    lengths = [40 + 17 * (i % 23) for i in range(requests)]
    run(lengths, [n - (11 * i) % 40 for i, n in enumerate(lengths)], 4, 2, 64, F16, 16)


@pytest.mark.parametrize("code", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim,most", [(64, 0), (128, 64), (256, 372)])
def test_scratch_of_the_kernels(dtype, code, dim, most, monkeypatch):
    """Scratch bytes a lane: none in tiles of 16 rows, and no more than when they were measured in those of 128."""
    for news, kernel in ((None, _native.ATTENTION_DECODE), ([3, 9], _native.ATTENTION_PROMPT_ROWS), ([900, 1300], _native.ATTENTION_PROMPT_TILES)):
        if dtype == F32 and kernel == _native.ATTENTION_PROMPT_TILES:
            continue
        got = []
        p = Quantized([1500, 1500], news, 8, 8, dim, dtype, 16, code=code)
        with monkeypatch.context() as m:
            m.setattr(_native, "host", lambda: Declining())
            m.setattr(attention, "_launch", lambda name, args, device: got.append(args))
            p.launch()
        info, registers, spills = _native.AttentionPlanInfo(), ctypes.c_int(), ctypes.c_int()
        args = [ctypes.byref(x) for x in got[0]]
        assert _native.lib().iris_quantized_attention_plan(*args, 0, ctypes.byref(info)) == 0 and info.kernel == kernel
        assert _native.lib().iris_quantized_attention_kernel_info(*args, ctypes.byref(registers), ctypes.byref(spills)) == 0
        assert 0 < registers.value <= 512
        assert spills.value <= (most if kernel == _native.ATTENTION_PROMPT_TILES else 0)
