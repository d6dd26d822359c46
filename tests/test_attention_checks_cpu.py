"""The attention block's Python checks, and what becomes of the native launch's answers, on tensors of the host: the native module
and the launch are replaced, and the check that tensors lie on the GPU is left out."""

import pytest
import torch

from iris_amd import _native, attention

BF16 = torch.bfloat16
DECLINED = -1


class Calls:
    """``answer``: what the native module says; ``launched``: (name, arguments) of the launches that the Python code makes."""

    def __init__(self):
        self.answer, self.launched = DECLINED, []

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
