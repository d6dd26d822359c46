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
