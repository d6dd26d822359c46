"""Attention over a paged cache, of single tokens and of prompts, against the definition in 64 bits."""

import math
import random

import pytest
import torch

import attention_reference as R
from attention_reference import BF16, F16, F32
from iris_amd import attention

pytestmark = pytest.mark.gpu


class Problem:
    """Requests with ``lengths`` keys and ``news`` queries each (None: one each), in a cache whose other places hold NaN."""

    def __init__(self, lengths, news, hq, hk, d, dtype, page, *, window=0, sinks=0, seed=0, heads_first=False, fused=False, spare=3, room=2):
        self.lengths, self.news, self.dtype, self.window, self.sinks = lengths, news, dtype, window, sinks
        self.shape = (hq, hk, d)
        g = torch.Generator().manual_seed(seed)
        tokens = sum(news) if news is not None else len(lengths)
        self.q_host = (torch.randn((tokens, hq, d), generator=g) * 1.5).to(dtype)
        self.k = [torch.randn((n, hk, d), generator=g).to(dtype) for n in lengths]
        self.v = [torch.randn((n, hk, d), generator=g).to(dtype) for n in lengths]
        counts = [R.cdiv(n, page) for n in lengths]
        pages = sum(counts) + spare
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
        caches = [torch.full(shape, math.nan, dtype=dtype) for _ in range(2)]
        width = max(counts + [1]) + room
        table = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32)  # (entries past a request's pages are not read)
        at = 0
        for i, n in enumerate(counts):
            table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
            for c, rows in zip(caches, (self.k[i], self.v[i])):
                view = c.transpose(1, 2) if heads_first else c
                for j in range(n):
                    part = rows[j * page:(j + 1) * page]
                    view[table[i, j], :len(part)] = part
        self.k_cache, self.v_cache = (c.cuda().transpose(1, 2) if heads_first else c.cuda() for c in caches)
        self.table = table.cuda()
        self.lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        if fused:  # queries as a view of a wider projection, outputs into a wider tensor
            wide = torch.zeros((tokens, (hq + 2 * hk) * d), dtype=dtype, device="cuda")
            self.q = wide[:, :hq * d].unflatten(1, (hq, d))
            self.q.copy_(self.q_host)
            self.out = torch.full((tokens, hq + 1, d), -7.0, dtype=dtype, device="cuda")[:, 1:]
        else:
            self.q = self.q_host.cuda()
            self.out = torch.full((tokens, hq, d), -7.0, dtype=dtype, device="cuda")
        self.lse = torch.full((tokens, hq), -7.0, device="cuda")
        self.word = torch.zeros(1, dtype=torch.int32, device="cuda")
        if news is not None:
            starts = [0]
            for n in news:
                starts.append(starts[-1] + n)
            self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")

    def launch(self, workspace="own", scale=None):
        if isinstance(workspace, str):
            workspace = attention.make_workspace(self.shape[2])
        args = dict(scale=scale, window=self.window, sinks=self.sinks, lse=self.lse, workspace=workspace, status=self.word)
        if self.news is None:
            attention.decode_attention(self.q, self.k_cache, self.v_cache, self.table, self.lens, self.out, **args)
        else:
            attention.prompt_attention(self.q, self.k_cache, self.v_cache, self.table, self.lens, self.starts, self.out, **args)
        return workspace

    def check(self, scale=None, skip=lambda request, position: False):
        assert self.word.item() == 0
        hq, hk, d = self.shape
        scale = scale or d ** -0.5
        out, lse = self.out.double().cpu(), self.lse.double().cpu()
        at = 0
        for i, n in enumerate(self.lengths):
            new = 1 if self.news is None else self.news[i]
            want, want_lse, spread = R.attention(self.q_host[at:at + new], self.k[i], self.v[i], n - new, scale, self.window, self.sinks)
            keep = [j for j in range(new) if not skip(i, n - new + j)]
            off, bound = (out[at:at + new] - want).abs()[keep], R.attention_error(self.dtype, want, spread, d)[keep]
            assert bool((off <= bound).all()), f"request {i}: off by up to {(off / bound).max().item()} times the bound"
            got = lse[at:at + new][keep]
            empty = want_lse[keep] == -math.inf
            assert torch.equal(got == -math.inf, empty)
            assert bool(((got - want_lse[keep]).abs()[~empty] <= 64 * math.sqrt(d) * 2.0 ** -23 + 2.0 ** -18).all())
            at += new


def run(*args, scale=None, workspace="own", **kw):
    p = Problem(*args, **kw)
    p.launch(workspace, scale)
    p.check(scale)
    return p


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300, 700]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256, 80, 96, 192, 8])
def test_decode_types_and_head_sizes(dtype, dim):
    run(LENGTHS, None, 4, 2, dim, dtype, 16)


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (3, 1), (8, 1), (5, 1), (14, 2), (16, 1), (17, 1), (40, 1), (24, 8)])
def test_decode_heads(hq, hk):
    run([0, 1, 40, 333], None, hq, hk, 64, BF16, 32)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 20, 48, 64, 512])
@pytest.mark.parametrize("heads_first", [False, True])
def test_decode_pages(page, heads_first):
    run([5, 130, 257, 600], None, 2, 1, 128, F16, page, heads_first=heads_first)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (100, 130), (128, 128), (300, 5), (1000, 4)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_window_and_first_tokens(window, sinks, dtype):
    run([0, 1, 2, 99, 100, 101, 128, 300, 555, 900], None, 4, 2, 64, dtype, 16, window=window, sinks=sinks)


def test_decode_hidden_keys_are_not_read_as_numbers():
    window, sinks = 50, 3
    p = Problem([40, 200, 500], None, 4, 2, 64, BF16, 16, window=window, sinks=sinks)
    for i, n in enumerate(p.lengths):
        for key in range(sinks, n - window):
            page, row = p.table[i, key // 16], key % 16
            p.k_cache[page, row] = math.inf
            p.v_cache[page, row] = math.nan
    p.launch()
    p.check()


def test_decode_long_contexts_are_split():
    run([9000, 3, 0, 20000], None, 8, 2, 128, BF16, 16)
    run([9000, 3, 0, 20000], None, 8, 2, 64, F32, 64, window=5000, sinks=2)


def test_decode_many_requests():
    rng = random.Random(2)
    run([rng.choice([0, 1, rng.randrange(200)]) for _ in range(600)], None, 2, 1, 64, BF16, 16)


def test_decode_with_little_or_no_workspace_gives_the_same():
    lengths = [3000, 10, 0, 700]
    full = run(lengths, None, 4, 1, 64, BF16, 16)
    none = run(lengths, None, 4, 1, 64, BF16, 16, workspace=None)
    small = torch.zeros(4096 + 5 * 16 * 68, device="cuda")
    few = run(lengths, None, 4, 1, 64, BF16, 16, workspace=small)
    for other in (none, few):
        # (the parts' weights are rounded against other maxima)
        assert bool(((full.out.double() - other.out.double()).abs() <= 2.0 ** -6).all())
    tiny = torch.zeros(8, device="cuda")
    run(lengths, None, 4, 1, 64, BF16, 16, workspace=tiny)


def test_a_workspace_serves_many_launches_and_gives_the_same_bits():
    p = Problem([5000, 40, 900], None, 8, 1, 128, BF16, 16)
    workspace = p.launch()
    p.check()
    first = p.out.clone()
    for _ in range(5):
        p.out.fill_(-7)
        p.launch(workspace)
        assert torch.equal(p.out, first)
    assert bool((workspace[:4096].view(torch.int32) == 0).all())


def test_scores_far_apart():
    """One key with almost all weight and thousands with almost none: in fp16 the small weights still count."""
    n, d = 4096, 64
    p = Problem([n], None, 1, 1, d, F16, 16)
    p.q_host = torch.zeros(1, 1, d, dtype=F16)
    p.q_host[..., 0] = 8
    p.q.copy_(p.q_host)
    p.k[0][..., 0] = 0
    p.k[0][7, 0, 0] = 9.0  # 9 more than the others: they have e^-9 of its weight, 4095 of them half of it
    p.v[0].fill_(1)
    p.v[0][7] = -1
    for j in range(n // 16):
        p.k_cache[p.table[0, j]] = p.k[0][16 * j:16 * j + 16].cuda()
        p.v_cache[p.table[0, j]] = p.v[0][16 * j:16 * j + 16].cuda()
    p.launch()
    p.check()


def test_decode_scale_views_and_streams():
    p = Problem([100, 37, 512], None, 6, 2, 64, BF16, 16, fused=True)
    workspace = attention.make_workspace(64)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        p.launch(workspace, scale=0.3)
    side.synchronize()
    p.check(scale=0.3)
    assert bool((p.out._base[:, 0] == -7).all())


def test_decode_in_a_captured_graph_with_growing_contexts():
    p = Problem([600, 600, 600], None, 8, 1, 128, BF16, 16)
    workspace = attention.make_workspace(128)
    full = [600, 600, 600]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            p.launch(workspace)
    torch.cuda.synchronize()
    k, v = p.k, p.v
    for lengths in ([1, 0, 5], [400, 599, 130], full, [17, 600, 0]):
        p.lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        p.lengths, p.k, p.v = lengths, [x[:n] for x, n in zip(k, lengths)], [x[:n] for x, n in zip(v, lengths)]
        graph.replay()
        torch.cuda.synchronize()
        p.check()


def test_a_page_outside_the_cache_is_reported():
    p = Problem([100, 100, 100], None, 2, 1, 64, BF16, 16)
    p.table[1, 3] = 1 << 30
    p.table[2, 2] = -1
    p.launch()
    assert p.word.item() == attention.STATUS_BAD_INDEX
    assert bool(p.out[1:].isnan().all()) and not bool(p.out[0].isnan().any())


def test_a_length_beyond_the_table_is_reported():
    p = Problem([100, 100], None, 2, 1, 64, BF16, 16)
    p.table = p.table[:, :7]
    p.lens[0] = 1000
    p.launch()
    assert p.word.item() == attention.STATUS_BAD_INDEX


def test_decode_addresses_past_32_bits():
    """A cache of more than 4 GiB (and 2^31 elements) whose last pages are used."""
    d, hk, page = 128, 8, 64
    pages = (2 ** 31 + 2 ** 28) // (d * hk * page)
    p = Problem([200, 70], None, hk, hk, d, BF16, page)
    k_cache = torch.empty((pages, page, hk, d), dtype=BF16, device="cuda")
    v_cache = torch.empty((pages, page, hk, d), dtype=BF16, device="cuda")
    used = len(p.k_cache)
    k_cache[pages - used:], v_cache[pages - used:] = p.k_cache, p.v_cache
    p.k_cache, p.v_cache = k_cache, v_cache
    p.table = torch.where(p.table < used, p.table + (pages - used), p.table)
    p.launch()
    p.check()


# ---- prompts -----------------------------------------------------------------
# (Few rows of few keys at most go in tiles of 16 rows; block tables with room for more keys take the same problems to tiles of 128.)

@pytest.fixture(params=[2, 30000], ids=["tight", "roomy"])
def room(request):
    return request.param


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256, 80, 96, 192])
def test_prompt_types_and_head_sizes(dtype, dim, room):
    run([70, 33, 1, 0, 150], [70, 5, 1, 0, 1], 4, 2, dim, dtype, 16, room=room)


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (3, 1), (8, 1), (7, 1), (16, 1), (20, 1), (6, 2)])
def test_prompt_heads(hq, hk, room):
    run([90, 20], [40, 20], hq, hk, 64, BF16, 32, room=room)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 20, 64])
@pytest.mark.parametrize("heads_first", [False, True])
def test_prompt_pages(page, heads_first, room):
    run([150, 31, 64], [130, 31, 2], 2, 1, 128, BF16, page, heads_first=heads_first, room=room)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (50, 70), (64, 64), (200, 5)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hk", [(4, 2), (32, 16)])  # (tiles of 16 rows, and of 128)
def test_prompt_window_and_first_tokens(window, sinks, dtype, hq, hk):
    run([260, 100, 7], [260, 30, 7], hq, hk, 64, dtype, 16, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 64), (F16, 128), (BF16, 96)])
def test_prompts_of_many_tiles(dtype, dim, room):
    run([700, 513], [700, 257], 2, 1, dim, dtype, 16, room=room)
    run([700, 513], [700, 257], 2, 1, dim, dtype, 16, window=100, sinks=3)
    run([700, 513], [700, 257], 10, 5, dim, dtype, 16, window=100, sinks=3)


def test_prompt_pieces_behind_a_long_context(room):
    run([5000, 3000], [9, 64], 4, 1, 128, BF16, 16, room=room)
    run([5000, 3000], [9, 64], 4, 1, 128, BF16, 16, workspace=None, room=room)
    run([5000, 3500], [300, 310], 4, 1, 64, F16, 16, window=3000, sinks=4, room=room)
    run([5000, 3000], [9, 64], 4, 1, 64, F16, 16, window=900, sinks=4)


def test_prompt_of_more_queries_than_keys_leaves_rows_empty(room):
    p = run([3, 40], [10, 12], 2, 1, 64, BF16, 16, room=room)
    assert bool((p.out[:7] == 0).all())
    run([0, 40], [4, 12], 2, 1, 128, BF16, 16, room=room)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128), (F32, 64), (BF16, 192)])
@pytest.mark.parametrize("hq,hk", [(2, 1), (64, 32)])
def test_a_value_that_is_no_number_reaches_only_the_queries_that_see_it(dtype, dim, window, hq, hk, room):
    n = 150
    p = Problem([n], [n], hq, hk, dim, dtype, 16, window=window, room=room)
    bad = {60: math.nan, 100: math.inf, 101: -math.inf, n - 1: math.nan}
    for key, value in bad.items():
        p.v_cache[p.table[0, key // 16], key % 16, :, ::2] = value
        p.v[0][key, :, ::2] = value
    p.launch()

    def reached(request, at):
        return any(bool(R.sees(at, torch.tensor(key), window, 0)) for key in bad)

    p.check(skip=reached)
    out = p.out.cpu()
    touched = torch.tensor([reached(0, at) for at in range(n)])
    assert bool((~out[touched][..., ::2].isfinite()).all()) and bool(out[..., 1::2].isfinite().all())


def test_a_key_that_is_no_number_reaches_only_the_queries_that_see_it(room):
    n = 140
    p = Problem([n], [n], 2, 1, 64, BF16, 16, room=room)
    p.k_cache[p.table[0, 90 // 16], 90 % 16] = math.nan
    p.launch()
    p.check(skip=lambda request, at: at >= 90)
    assert bool(p.out[90:].isnan().all())


def test_prompt_views_padding_and_repeats(room):
    p = Problem([200, 90], [150, 90], 6, 2, 128, BF16, 16, fused=True, room=room)
    pad = 20  # tokens of no request behind the last one's
    q, out = torch.zeros((260, 6, 128), dtype=BF16, device="cuda"), torch.full((260, 6, 128), -7.0, dtype=BF16, device="cuda")
    lse = torch.full((260, 6), -7.0, device="cuda")
    q[:240] = p.q
    p.launch()
    p.check()
    workspace = attention.make_workspace(128)
    for _ in range(3):
        attention.prompt_attention(q, p.k_cache, p.v_cache, p.table, p.lens, p.starts, out, lse=lse, workspace=workspace)
        assert torch.equal(out[:240], p.out) and torch.equal(lse[:240], p.lse)
        assert bool((out[240:] == -7).all()) and bool((lse[240:] == -7).all()) and pad == 20


def test_one_token_prompts_are_decode():
    lengths = [5, 200, 77]
    a, b = Problem(lengths, None, 4, 2, 64, F32, 16), Problem(lengths, [1, 1, 1], 4, 2, 64, F32, 16)
    a.launch()
    b.launch()
    a.check()
    b.check()


def test_refusals():
    p = Problem([20, 30], [4, 5], 4, 2, 64, BF16, 16)
    base = dict(q=p.q, k_cache=p.k_cache, v_cache=p.v_cache, block_table=p.table, lengths=p.lens, query_starts=p.starts, out=p.out)

    def call(decode=False, **other):
        args = dict(base, **other)
        names = ["q", "k_cache", "v_cache", "block_table", "lengths", "query_starts", "out"]
        if decode:
            names.remove("query_starts")
            args.pop("query_starts")
        operands = [args.pop(n) for n in names]
        (attention.decode_attention if decode else attention.prompt_attention)(*operands, **args)

    call()
    k = p.k_cache
    wide = torch.zeros((9, 4, 68), dtype=BF16, device="cuda")
    for wrong, error in [
            (dict(q=p.q.double()), TypeError), (dict(q=p.q.half()), TypeError), (dict(out=p.out.float()), TypeError), (dict(out=p.out[:3]), ValueError),
            (dict(out=p.out[:1].expand(9, 4, 64)), ValueError), (dict(q=p.q[:, :3], out=p.out[:, :3]), ValueError),
            (dict(v_cache=p.v_cache[:2]), ValueError), (dict(k_cache=k[..., :32]), ValueError), (dict(k_cache=k.transpose(0, 3)), ValueError),
            (dict(q=wide[..., 2:66]), ValueError), (dict(q=wide[..., :64]), ValueError), (dict(q=wide[..., :60], out=wide[..., :60].clone()), ValueError),
            (dict(block_table=p.table.long()), TypeError), (dict(block_table=p.table.T), TypeError), (dict(lengths=p.lens[:1]), ValueError),
            (dict(lengths=p.lens.long()), TypeError), (dict(query_starts=p.starts[:2]), ValueError), (dict(scale=0.0), ValueError),
            (dict(scale=-1.0), ValueError), (dict(scale=math.inf), ValueError), (dict(scale=math.nan), ValueError), (dict(window=-1), ValueError),
            (dict(sinks=-1), ValueError), (dict(lse=p.lse.half()), TypeError), (dict(lse=p.lse[:, :3]), TypeError), (dict(workspace=p.out), TypeError),
            (dict(status=p.lse), TypeError), (dict(q=p.q.cpu()), RuntimeError), (dict(lengths=p.lens.cpu()), RuntimeError),
            (dict(decode=True), ValueError), (dict(q=p.q.clone().requires_grad_()), RuntimeError)]:
        with pytest.raises(error):
            call(**wrong)
    big = torch.zeros((1, 1, 264), dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="at most"):
        attention.decode_attention(big, big[None], big[None], p.table[:1], p.lens[:1], big.clone())
    with pytest.raises(ValueError, match="at most"):
        attention.make_workspace(264)


def test_nothing_to_do():
    e = torch.empty((0, 4, 64), dtype=BF16, device="cuda")
    cache = torch.zeros((1, 16, 2, 64), dtype=BF16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    attention.decode_attention(e, cache, cache, torch.zeros((0, 1), dtype=torch.int32, device="cuda"), none, e)
    q, out = torch.ones((2, 4, 64), dtype=BF16, device="cuda"), torch.ones((2, 4, 64), dtype=BF16, device="cuda")
    attention.decode_attention(q, cache[:0], cache[:0], torch.zeros((2, 1), dtype=torch.int32, device="cuda"),
                               torch.zeros(2, dtype=torch.int32, device="cuda"), out)
    assert bool((out == 0).all())


# ---- many prompts, against the definition on the GPU ---------------------------


def dense_on_gpu(p):
    """The definition in 64 bits with whole score matrices, one head at a time: for problems too large for the CPU's."""
    hq, hk, d = p.shape
    out, at = [], 0
    for i, n in enumerate(p.lengths):
        new = p.news[i]
        q, k, v = p.q[at:at + new].double(), p.k[i].double().cuda(), p.v[i].double().cuda()
        rows, keys = torch.arange(n - new, n, device="cuda")[:, None], torch.arange(n, device="cuda")
        heads = []
        for h in range(hq):
            s = (q[:, h] @ k[:, h // (hq // hk)].T) * d ** -0.5
            weights = torch.softmax(s.masked_fill(~R.sees(rows, keys, p.window, p.sinks), -math.inf), -1)
            heads.append((weights @ v[:, h // (hq // hk)], weights @ v[:, h // (hq // hk)].abs()))
        out.append(tuple(torch.stack([h[j] for h in heads], 1) for j in (0, 1)))
        at += new
    return tuple(torch.cat([o[j] for o in out]).cpu() for j in (0, 1))


@pytest.mark.parametrize("lengths,news,hq,hk,dim,dtype,window", [
    # more row tiles than run at once: those that see the most keys start first
    ([900, 700, 1300, 64, 2000], [900, 500, 300, 64, 1999], 40, 8, 128, BF16, 0),
    ([800, 1500, 700], [800, 1500, 1], 40, 8, 64, F16, 0),
    ([2100], [2100], 36, 4, 64, BF16, 200),
    ([700, 650], [600, 650], 32, 4, 256, BF16, 0),
])
def test_more_prompts_than_run_at_once(lengths, news, hq, hk, dim, dtype, window):
    p = Problem(lengths, news, hq, hk, dim, dtype, 16, window=window, sinks=3 if window else 0)
    p.launch()
    assert p.word.item() == 0
    want, spread = dense_on_gpu(p)
    off, bound = (p.out.double().cpu() - want).abs(), R.attention_error(dtype, want, spread, dim)
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item()} times the bound"
    first = p.out.clone()
    p.launch()
    assert torch.equal(p.out, first)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 256), (F32, 64)])
def test_a_page_outside_the_cache_is_reported_for_prompts(dtype, dim, room):
    for lengths, news in (([300, 300], [300, 300]), ([3000, 3000], [40, 40])):  # (the second: keys split over workgroups)
        p = Problem(lengths, news, 4, 1, dim, dtype, 16, room=room)
        p.table[1, 5] = 1 << 30
        p.launch()
        assert p.word.item() == attention.STATUS_BAD_INDEX
        at = news[0]
        reached = 5 * 16 - (lengths[1] - news[1])  # the first query that sees the page
        assert bool(p.out[at + max(reached, 0):].isnan().all())
        assert not bool(p.out[:at].isnan().any())


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_values_that_are_no_numbers_where_keys_are_split(dtype, dim, room):
    n, new = 2500, 40
    p = Problem([n], [new], 4, 1, dim, dtype, 16, room=room)
    p.v_cache[p.table[0, (n - 20) // 16], (n - 20) % 16, 0, 1] = math.nan
    p.v[0][n - 20, 0, 1] = math.nan
    p.launch()
    p.check(skip=lambda request, at: at >= n - 20)
    assert bool(p.out[new - 20:, :, 1].isnan().all()) and bool(p.out[new - 20:, :, 2:].isfinite().all())


def test_scores_that_grow_along_the_context(room):
    """Each stretch of keys outweighs those before it: the reference of the weights moves again and again."""
    for dtype, new in ((F16, 70), (BF16, 70), (F16, 1)):
        n, d = 700, 64
        p = Problem([n], [new], 1, 1, d, dtype, 16, room=room)
        p.q_host[:] = 0
        p.q_host[..., 0] = 16
        p.q.copy_(p.q_host)
        p.k[0][..., 0] = (torch.arange(n) // 50).to(dtype)[:, None]  # two more a stretch, 28 in all
        for j in range(R.cdiv(n, 16)):
            part = p.k[0][16 * j:16 * j + 16].cuda()
            p.k_cache[p.table[0, j], :len(part)] = part
        p.launch()
        p.check()
