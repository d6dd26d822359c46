"""Block tables, positions and slots built on the GPU against the definition request by request: every number equal."""

import random

import pytest
import torch

import attention_reference as R
from iris_amd import attention

pytestmark = pytest.mark.gpu


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def step(pairs, page, *, spare=8, width=None, tokens=None, wrap=0, seed=0, table_stride=0, status=True):
    """Runs one step of (cached, new) requests and compares everything it writes."""
    rng = random.Random(seed)
    held = [R.cdiv(c, page) for c, _ in pairs]
    width = width or max([R.cdiv(c + max(n, 0), page) for c, n in pairs] + [1])
    need = sum(R.cdiv(c + max(n, 0), page) - h for (c, n), h in zip(pairs, held))
    total_pages = sum(held) + need + 8
    order = list(range(total_pages))
    rng.shuffle(order)
    table = [[-7] * width for _ in pairs]
    for i, h in enumerate(held):
        for j in range(min(h, width)):
            table[i][j] = order.pop()
    free = order[:max(need + spare, 0)]
    pool = [-9] * total_pages
    for x, page_id in enumerate(free):
        pool[(wrap + x) % total_pages] = page_id
    state = [wrap, wrap + len(free)]
    total = sum(max(n, 0) for _, n in pairs)
    tokens = total + 5 if tokens is None else tokens
    want = R.block_tables([c for c, _ in pairs], [n for _, n in pairs], table, pool, state, page, tokens)
    wide = torch.full((max(len(pairs), 1), width + table_stride), -5, dtype=torch.int32, device="cuda")
    table_d = wide[:len(pairs), :width]
    if pairs:
        table_d.copy_(ints(table))
    pool_d = ints(pool)
    lengths, starts = ints([-1] * len(pairs)), ints([-1] * (len(pairs) + 1))
    positions, slots = ints([-1] * tokens), ints([-2] * tokens, torch.int64)
    state_out, word = ints([0, 0], torch.int64), ints([0])
    attention.build_block_tables(ints([c for c, _ in pairs]), ints([n for _, n in pairs]), table_d, pool_d,
                                 ints(state, torch.int64), page, lengths=lengths, pool_state_out=state_out, query_starts=starts,
                                 positions=positions, slots=slots, status=word if status else None)
    assert lengths.tolist() == want["lengths"]
    assert starts.tolist() == want["starts"]
    assert positions.tolist() == want["positions"]
    assert slots.tolist() == want["slots"]
    assert state_out.tolist() == want["state"]
    assert pool_d.tolist() == want["pool"]
    assert table_d.tolist() == want["table"].tolist()
    assert bool((wide[:, width:] == -5).all())
    if status:
        bits = (attention.STATUS_NO_PAGES if want["refused"] else 0) | (attention.STATUS_NO_ROOM if want["short"] else 0)
        assert word.item() == bits
    return want


def mixed(count, seed, most=300):
    rng = random.Random(seed)
    pairs = []
    for _ in range(count):
        cached = rng.choice([0, 1, 15, 16, 17, rng.randrange(most)])
        pairs.append((cached, rng.choice([1, 1, 1, 0, -1, rng.randrange(most)])))
    return pairs


@pytest.mark.parametrize("count", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 1024, 1025, 2500])
def test_numbers_of_requests(count):
    step(mixed(count, count), 16, seed=count)


@pytest.mark.parametrize("page", [1, 3, 16, 20, 128])
def test_page_sizes(page):
    step(mixed(70, page), page, seed=page, wrap=12345, table_stride=3)


def test_the_most_requests_of_a_call():
    step([(i % 40, 1) for i in range(attention.MAX_REQUESTS)], 16)


def test_no_request_and_no_token():
    step([], 16)
    step([], 16, tokens=0)
    step([(5, 0), (0, 0), (17, -1)], 16, tokens=0)


def test_the_ring_wraps():
    pairs = mixed(90, 3)
    for wrap in (1, 200, 10 ** 9, 5 * 10 ** 9):
        step(pairs, 16, wrap=wrap)


def test_a_ring_that_runs_out_serves_the_first_requests_and_those_that_need_nothing():
    pairs = [(16, 40), (3, 1), (32, 1), (16, 1), (15, 1), (0, 100), (31, 1)]
    for spare in range(-11, 1):
        want = step(pairs, 16, spare=spare)
        assert want["refused"] == (spare < 0)


def test_a_table_row_that_is_too_short():
    want = step([(0, 40), (10, 60), (0, 8)], 16, width=3)
    assert want["lengths"] == [40, 10, 8] and want["refused"]


def test_more_tokens_than_room():
    want = step([(4, 30), (0, 30)], 16, tokens=40)
    assert want["short"]
    step([(4, 30), (0, 30)], 16, tokens=40, status=False)


def test_a_long_prompt_among_many():
    step([(0, 40000)] + [(i, 1) for i in range(200)] + [(100, 3001)], 16)


def test_steps_in_a_captured_graph_on_another_stream():
    """Two buffers in turn, as a captured serving loop has them: every replay takes and gives pages."""
    page, count = 16, 10
    lengths = [ints([15] * count), ints([0] * count)]
    new = ints([1] * count)
    pages = 64
    table = torch.zeros((count, 8), dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(count, dtype=torch.int32, device="cuda")
    pool = torch.arange(pages, dtype=torch.int32, device="cuda")
    states = [ints([count, pages], torch.int64), ints([0, 0], torch.int64)]
    starts, positions, slots = ints([0] * (count + 1)), ints([0] * count), ints([0] * count, torch.int64)

    def one(i):
        attention.build_block_tables(lengths[i], new, table, pool, states[i], page, lengths=lengths[1 - i],
                                     pool_state_out=states[1 - i], query_starts=starts, positions=positions, slots=slots)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            one(0)
            one(1)
    torch.cuda.synchronize()
    for replay in range(1, 12):
        graph.replay()
        torch.cuda.synchronize()
        n = 15 + 2 * replay
        assert lengths[0].tolist() == [n] * count
        taken = count * R.cdiv(n, page)
        assert states[0].tolist() == [taken, pages]
        want = [table[i, (n - 1) // page].item() * page + (n - 1) % page for i in range(count)]
        assert slots.tolist() == want and positions.tolist() == [n - 1] * count
        assert len(set(table[:, :R.cdiv(n, page)].flatten().tolist())) == taken


def test_refusals():
    def call(**other):
        args = dict(cached=ints([1, 2]), new_tokens=ints([1, 1]), block_table=ints([[0, 0], [1, 1]]), pool=ints([2, 3, 4, 5]),
                    pool_state=ints([0, 4], torch.int64), page_size=16, lengths=ints([0, 0]), pool_state_out=ints([0, 0], torch.int64),
                    query_starts=ints([0, 0, 0]), positions=ints([0, 0]), slots=ints([0, 0], torch.int64))
        args.update(other)
        attention.build_block_tables(args.pop("cached"), args.pop("new_tokens"), args.pop("block_table"), args.pop("pool"),
                                     args.pop("pool_state"), args.pop("page_size"), **args)

    call()
    same = ints([1, 2])
    for wrong, error in [(dict(cached=same, lengths=same), ValueError), (dict(new_tokens=ints([1])), ValueError),
                         (dict(new_tokens=ints([1, 1], torch.int64)), TypeError), (dict(page_size=0), ValueError),
                         (dict(query_starts=ints([0, 0])), ValueError), (dict(slots=ints([0, 0])), TypeError),
                         (dict(slots=ints([0], torch.int64)), ValueError), (dict(pool=ints([])), ValueError),
                         (dict(block_table=ints([[0, 0]])), TypeError), (dict(block_table=ints([[0, 0], [1, 1]]).T), ValueError),
                         (dict(block_table=ints([[0, 0]]).expand(2, 2)), ValueError), (dict(status=ints([0], torch.int64)), TypeError),
                         (dict(positions=torch.zeros(2, dtype=torch.int32)), RuntimeError), (dict(pool_state=ints([0, 4])), TypeError)]:
        with pytest.raises(error):
            call(**wrong)
    n = attention.MAX_REQUESTS + 1
    with pytest.raises(ValueError, match="at most"):
        call(cached=ints([0] * n), new_tokens=ints([0] * n), block_table=torch.zeros((n, 1), dtype=torch.int32, device="cuda"),
             lengths=ints([0] * n), query_starts=ints([0] * (n + 1)))
