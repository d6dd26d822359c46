"""The attention block's Python checks, and what becomes of the native launch's answers, on tensors of the host: the native module
and the launch are replaced, and the check that tensors lie on the GPU is left out."""

import pytest
import torch

from iris_amd import _native, attention

BF16 = torch.bfloat16
DECLINED = -1
HOST = _native.host()


class Calls:
    """``answer``: what the native module says; ``launched``: (name, arguments) of the launches that the Python code makes."""

    def __init__(self):
        self.answer, self.launched = DECLINED, []
        self.overlap = HOST.overlap  # (of tensors anywhere)

    def __getattr__(self, name):  # the native module's functions
        return lambda *args: self.answer


@pytest.fixture()
def calls(monkeypatch):
    calls = Calls()
    monkeypatch.setattr(_native, "host", lambda: calls)
    monkeypatch.setattr(attention, "_require_cuda", lambda what, t, device: None)
    monkeypatch.setattr(attention, "_launch", lambda name, args, device: calls.launched.append((name, args)))
    return calls


def operands(requests=3, width=5, page=16, hq=4, hk=2, dim=64, tokens=None, dtype=BF16):
    tokens = tokens or requests
    cache = (requests * width, page, hk, dim)
    return dict(q=torch.zeros((tokens, hq, dim), dtype=dtype), k_cache=torch.zeros(cache, dtype=dtype), v_cache=torch.zeros(cache, dtype=dtype),
                block_table=torch.zeros((requests, width), dtype=torch.int32), lengths=torch.zeros(requests, dtype=torch.int32),
                out=torch.zeros((tokens, hq, dim), dtype=dtype))


def decode(**args):
    named = [args.pop(n) for n in ("q", "k_cache", "v_cache", "block_table", "lengths", "out")]
    attention.decode_attention(*named, **args)


def test_rows_of_a_block_table_lie_apart(calls):
    """A table whose rows share memory has no stride that the kernels take: with any other one they would read past its end."""
    base = operands()
    wide = torch.zeros((3, 9), dtype=torch.int32)
    decode(**dict(base, block_table=wide[:, :5]))
    assert calls.launched[-1][1].stride_table == 9
    decode(**dict(operands(requests=1), block_table=wide[:1, :5]))  # (one row has no next)
    assert calls.launched[-1][1].stride_table >= 5
    done = len(calls.launched)
    for table in (wide[:1, :5].expand(3, 5), wide.flatten().as_strided((3, 5), (2, 1))):
        with pytest.raises(ValueError, match="overlap"):
            decode(**dict(base, block_table=table))
    assert len(calls.launched) == done


def tables_operands(requests=3, width=5, tokens=6):
    i32, i64 = torch.int32, torch.int64
    return [torch.zeros(requests, dtype=i32), torch.zeros(requests, dtype=i32), torch.zeros((requests, width), dtype=i32), torch.zeros(16, dtype=i32),
            torch.zeros(2, dtype=i64), 16], dict(lengths=torch.zeros(requests, dtype=i32), pool_state_out=torch.zeros(2, dtype=i64),
                                                 query_starts=torch.zeros(requests + 1, dtype=i32), positions=torch.zeros(tokens, dtype=i32),
                                                 slots=torch.zeros(tokens, dtype=i64))


def rope_operands(tokens=5, hq=4, hk=2, dim=64):
    heads = [torch.zeros((tokens, h, dim), dtype=BF16) for h in (hq, hk, hq, hk)]
    cos = torch.zeros((10, dim // 2))
    return heads[:2] + [torch.zeros(tokens, dtype=torch.int32), cos, cos.clone()] + heads[2:]


CALLS = {
    "tables": lambda: (lambda args, kw: attention.build_block_tables(*args, **kw))(*tables_operands()),
    "rope": lambda: attention.qk_norm_rope(*rope_operands()),
    "in place": lambda: (lambda x: attention.qk_norm_rope(*x[:5], x[0], x[1]))(rope_operands()),
    "gradient": lambda: (lambda x, y: attention.qk_norm_rope_backward(*x[:2], *y))(rope_operands(), rope_operands()),
    "gradient in place": lambda: (lambda x, y: attention.qk_norm_rope_backward(*x[:2], *y[:5], *x[:2]))(rope_operands(), rope_operands()),
    "decode": lambda: decode(**operands()),
    "prompt": lambda: (lambda a: attention.prompt_attention(*[a[n] for n in ("q", "k_cache", "v_cache", "block_table", "lengths")],
                                                            torch.zeros(4, dtype=torch.int32), a["out"]))(operands(tokens=7)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_what_the_native_code_launched_is_not_launched_again(calls, name, monkeypatch):
    """A status that is an error may come from behind a launch (one that was left by an earlier call, a second launch that failed): work
    in place would be done twice."""
    calls.answer = 0
    CALLS[name]()
    assert not calls.launched
    calls.answer = _native.HIP_ERROR_INVALID_VALUE
    with pytest.raises(ValueError, match="rejected"):
        CALLS[name]()
    assert not calls.launched
    calls.answer = 719
    monkeypatch.setattr(_native, "hip_try", lambda err: (_ for _ in ()).throw(RuntimeError(f"HIP error code {err}")))
    with pytest.raises(RuntimeError, match="719"):
        CALLS[name]()
    assert not calls.launched
    calls.answer = DECLINED
    CALLS[name]()
    assert len(calls.launched) == 1


def test_what_the_launcher_refuses_is_explained_where_the_checks_know_it(calls):
    calls.answer = _native.HIP_ERROR_INVALID_VALUE
    with pytest.raises(ValueError, match="16 bytes"):
        decode(**dict(operands(), q=torch.zeros(3 * 4 * 64 + 1, dtype=BF16)[1:].view(3, 4, 64)))


def test_numbers_past_31_bits_keep_their_meaning(calls):
    """No context is longer than 31 bits count: a window or first tokens beyond it are all keys."""
    most = 2 ** 31 - 1
    for value, want in ((2 ** 32 + 16, most), (2 ** 32, most), (2 ** 31, most), (most, most), (2 ** 70, most), (17, 17), (0, 0)):
        decode(**dict(operands(), window=value, sinks=5))
        assert (calls.launched[-1][1].window, calls.launched[-1][1].sinks) == (want, 5)
        decode(**dict(operands(), window=9, sinks=value))
        assert (calls.launched[-1][1].window, calls.launched[-1][1].sinks) == (9, want)
    done = len(calls.launched)
    for wrong in (dict(window=-2 ** 32 + 16), dict(sinks=-1)):
        with pytest.raises(ValueError):
            decode(**dict(operands(), **wrong))
    args, kw = tables_operands(width=0)
    for page_size in (2 ** 32 + 16, 2 ** 31):
        with pytest.raises(ValueError, match="31 bits"):
            attention.build_block_tables(*args[:5], page_size, **kw)
    assert len(calls.launched) == done


def test_gradients_and_tangents_that_would_be_lost_are_refused(calls):
    """Of every operand that results depend on: heads, caches, weights, angles."""
    forward_ad = torch.autograd.forward_ad
    cache = torch.zeros((3, 16, 2, 64), dtype=BF16)
    serving = dict(v=torch.zeros((5, 2, 64), dtype=BF16), k_cache=cache, v_cache=cache.clone(), slots=torch.zeros(5, dtype=torch.int64),
                   q_weight=torch.ones(64), k_weight=torch.ones(64))
    q, k, positions, cos, sin, q_out, k_out = rope_operands()
    rope = dict(serving, q=q, k=k, cos=cos, sin=sin, q_out=q_out, k_out=k_out)
    heads = [torch.zeros_like(t) for t in (q, k)]
    gradient = dict(dq_out=heads[0], dk_out=heads[1], q=q, k=k, cos=cos, sin=sin, dq=q_out, dk=k_out, q_weight=torch.ones(64), k_weight=torch.ones(64))

    def run_rope(**a):
        first = [a.pop(n) for n in ("q", "k")] + [positions] + [a.pop(n) for n in ("cos", "sin", "q_out", "k_out")]
        attention.qk_norm_rope(*first, **a)

    def run_gradient(**a):
        first = [a.pop(n) for n in ("dq_out", "dk_out", "q", "k")] + [positions] + [a.pop(n) for n in ("cos", "sin", "dq", "dk")]
        attention.qk_norm_rope_backward(*first, **a)

    attended = {n: t for n, t in operands().items() if t.is_floating_point()}
    for run, names, args in ((run_rope, rope, rope), (decode, attended, operands()), (run_gradient, gradient, gradient)):
        run(**args)
        for name in names:
            if not args[name].is_floating_point():
                continue
            done = len(calls.launched)
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(args[name].clone(), torch.ones_like(args[name]))
                with pytest.raises(RuntimeError, match="gradient"):
                    run(**dict(args, **{name: dual}))
            if run is not run_gradient or name in ("dq", "dk"):  # (a gradient's inputs are what autograd holds)
                with pytest.raises(RuntimeError, match="gradient"):
                    run(**dict(args, **{name: args[name].clone().requires_grad_()}))
            assert len(calls.launched) == done, name
    with pytest.raises(RuntimeError, match="gradient"):
        attention.QkNormRope.apply(q, k, positions, cos.clone().requires_grad_(), sin)


def test_overlap_of_strided_tensors():
    """Against the elements' addresses one by one: nested axes in any order, windows into each other, expanded axes."""
    import random

    overlap = HOST.overlap
    rng = random.Random(1)
    both = [0, 0]
    for _ in range(3000):
        base = torch.zeros(20000, dtype=rng.choice([torch.int16, torch.int32]))

        def view(t):
            if rng.random() < 0.5:  # axes inside each other, with gaps
                sizes = [rng.randint(1, 4) for _ in range(rng.randint(1, 4))]
                strides, reach = [], 1
                for n in sizes:
                    strides.append(reach * rng.choice([1, 1, 2]) + rng.choice([0, 0, 1, 5]))
                    reach = strides[-1] * n
                order = list(range(len(sizes)))
                rng.shuffle(order)
                sizes, strides = [sizes[i] for i in order], [strides[i] for i in order]
            else:
                sizes = [rng.randint(0 if rng.random() < 0.1 else 1, 5) for _ in range(3)]
                strides = [rng.randint(0, 30) for _ in range(3)]
            return t.as_strided(sizes, strides, rng.randint(0, 300))

        a, b = view(base), view(base.view(torch.int16) if rng.random() < 0.3 else base)

        def touched(t):
            at = torch.zeros(t.shape, dtype=torch.int64)
            for d, (n, s) in enumerate(zip(t.shape, t.stride())):
                at = at + (torch.arange(n) * s).view([-1 if i == d else 1 for i in range(t.dim())])
            start = (t.data_ptr() - base.data_ptr()) + at.flatten() * t.element_size()
            return {x + i for x in start.tolist() for i in range(t.element_size())}

        want = not touched(a).isdisjoint(touched(b))
        assert overlap(a, b) == overlap(b, a) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        both[want] += 1
    assert min(both) > 500
    big = torch.zeros(1).expand(1 << 30)  # (nothing of that size is walked through)
    assert overlap(big, big)
    qkv = torch.zeros((1 << 16, 12, 64), dtype=BF16)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    assert not any(overlap(*pair) for pair in ((q, k), (q, v), (k, v))) and overlap(q, qkv[:, 7:9])
    by_head = qkv.view(1 << 16, 4, 3, 64)
    assert not overlap(by_head[:, :, 0], by_head[:, :, 1]) and overlap(by_head[:, :, 0], qkv[:, :1])
    assert not overlap(q[::2], q[1::2]) and overlap(q[::2], q[::3])


def test_outputs_lie_apart(calls):
    """In place is element by element; anything else that shares memory would be read by one workgroup while another writes it."""

    def check(good, bad):
        for call in good:
            done = len(calls.launched)
            call()
            assert len(calls.launched) == done + 1
        for call in bad:
            done = len(calls.launched)
            with pytest.raises(ValueError, match="memory"):
                call()
            assert len(calls.launched) == done

    tokens, hq, hk, d = 6, 4, 2, 64
    wide = torch.zeros((tokens, hq + 2 * hk + 2, d), dtype=BF16)  # a fused projection, and room behind it
    q, k, v = wide[:, :hq], wide[:, hq:hq + hk], wide[:, hq + hk:hq + 2 * hk]
    cos, sin, positions = torch.zeros((10, d // 2)), torch.zeros((10, d // 2)), torch.zeros(tokens, dtype=torch.int32)
    q_new, k_new = torch.zeros((tokens, hq, d), dtype=BF16), torch.zeros((tokens, hk, d), dtype=BF16)
    caches = torch.zeros((2, 4, 16, hk, d), dtype=BF16)
    cache = dict(v=v, k_cache=caches[0], v_cache=caches[1], slots=torch.zeros(tokens, dtype=torch.int64))
    pages = caches.view(4, 2, 16, hk, d)  # keys and values of a page beside each other

    def turn(q_out, k_out, **kw):
        attention.qk_norm_rope(q, k, positions, cos, sin, q_out, k_out, **kw)

    check([lambda: turn(q, k), lambda: turn(q, k, **cache), lambda: turn(q_new, k_new, **cache), lambda: turn(q, None, **cache),
           lambda: turn(q, wide[:, -hk:], **cache), lambda: turn(q_new, k, **dict(cache, k_cache=pages[:, 0], v_cache=pages[:, 1]))],
          [lambda: turn(wide[:, 1:1 + hq], k_new), lambda: turn(q_new, wide[:, hq + 1:hq + 1 + hk]), lambda: turn(q, q[:, :hk]),
           lambda: turn(wide[:, hk:hk + hq], k), lambda: turn(q, v, **cache), lambda: turn(q_new, q_new[:, 1:1 + hk]),
           lambda: turn(q, k, **dict(cache, v_cache=caches[0])), lambda: turn(q, k, **dict(cache, v=caches[1, 0, :tokens])),
           lambda: turn(q, caches[0, 0, :tokens], **cache)])

    dq_out, dk_out, room = torch.zeros((tokens, hq, d), dtype=BF16), torch.zeros((tokens, hk, d), dtype=BF16), torch.zeros(20 * d)
    weights = dict(q_weight=torch.ones(d), k_weight=torch.ones(d), dq_weight=torch.zeros(d), dk_weight=torch.zeros(d), workspace=room)

    def back(dq, dk, **kw):
        attention.qk_norm_rope_backward(dq_out, dk_out, q, k, positions, cos, sin, dq, dk, **kw)

    check([lambda: back(dq_out, dk_out), lambda: back(q, k), lambda: back(q_new, k_new, **weights), lambda: back(wide[:, -hq:], k_new),
           lambda: back(dq_out, dk_out, **dict(weights, dq_weight=weights["q_weight"]))],  # (written when all has been read)
          [lambda: back(q_new, q_new[:, :hk]), lambda: back(wide[:, 1:1 + hq], k_new), lambda: back(q_new, q[:, :hk]), lambda: back(q_new, dq_out[:, :hk]),
           lambda: back(q_new, k_new, **dict(weights, dk_weight=weights["dq_weight"])), lambda: back(q_new, k_new, **dict(weights, dq_weight=room[:d])),
           lambda: back(q_new, k_new, **dict(weights, workspace=cos.flatten()[:2 * d]))])

    a = operands(requests=3)
    flat, scratch = torch.zeros(768 + 64, dtype=BF16), torch.zeros(5000)
    check([lambda: decode(**dict(a, out=a["q"])), lambda: decode(**dict(a, lse=torch.zeros(3, 4), workspace=scratch)),
           lambda: decode(**dict(a, v_cache=a["k_cache"]))],
          [lambda: decode(**dict(a, q=flat[:768].view(3, 4, 64), out=flat[64:].view(3, 4, 64))), lambda: decode(**dict(a, out=a["k_cache"].view(-1, 4, 64)[:3])),
           lambda: decode(**dict(a, out=a["q"].as_strided((3, 4, 64), (64, 192, 1)))), lambda: decode(**dict(a, lse=scratch[100:112].view(3, 4), workspace=scratch)),
           lambda: decode(**dict(a, lse=a["block_table"].view(torch.float32).flatten()[:12].view(3, 4)))])


@pytest.mark.parametrize("width,pages", [(0, 4), (3, 0), (0, 0)])
def test_without_a_page_the_rows_are_as_with_one(calls, width, pages):
    """Rows that see a key have no page to read it from (NaN, reported) where the table has room for it; a length beyond the table's
    room is none (reported); rows of no request stay as they are."""
    q, nan, inf = torch.ones((9, 4, 64), dtype=BF16), float("nan"), float("inf")
    cache = torch.zeros((pages, 16, 2, 64), dtype=BF16)

    def run(lengths, starts):
        n = len(lengths)
        out, lse, word = torch.full((9, 4, 64), 7.0, dtype=BF16), torch.full((9, 4), 7.0), torch.tensor([64], dtype=torch.uint32)
        table = torch.zeros((n, width), dtype=torch.int32)
        args = [cache, cache, table, torch.tensor(lengths, dtype=torch.int32)]
        if starts is None:
            attention.decode_attention(q, *args, out, lse=lse, status=word)
        else:
            attention.prompt_attention(q, *args, torch.tensor(starts, dtype=torch.int32), out, lse=lse, status=word)
        return out, lse, word.item()

    def expect(got, rows, bits):
        """rows: what each row's elements are, 0 (no key), nan (no page) or 7 (untouched)."""
        want = torch.tensor(rows)
        torch.testing.assert_close(got[0].float(), want[:, None, None].expand(9, 4, 64), equal_nan=True, rtol=0, atol=0)
        torch.testing.assert_close(got[1], torch.where(want == 0, -inf, want)[:, None].expand(9, 4), equal_nan=True, rtol=0, atol=0)
        assert got[2] == 64 | bits

    bad = attention.STATUS_BAD_INDEX
    see = nan if width else 0.0
    expect(run([0] * 9, None), [0.0] * 9, 0)
    expect(run([0, 5] + [0] * 7, None), [0.0, see] + [0.0] * 7, bad)
    # the requests' tokens are 1 .. 2, 3 .. 6 (of which the last two have keys), none, and none is 0, 7 and 8
    expect(run([0, 0, 0], [1, 3, 7, 7]), [7.0] + [0.0] * 6 + [7.0] * 2, 0)
    expect(run([0, 2, 0], [1, 3, 7, 7]), [7.0] + [0.0] * 4 + [see] * 2 + [7.0] * 2, bad)
    expect(run([0, 1000, 0], [1, 3, 7, 7]), [7.0] + [0.0] * 2 + [see] * 4 + [7.0] * 2, bad)
    assert not calls.launched
