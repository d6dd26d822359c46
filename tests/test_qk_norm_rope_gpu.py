"""Norms and rotation of query and key heads, the cache write, and their gradient, against the formulas in 64 bits."""

import math

import pytest
import torch

import attention_reference as R
from attention_reference import BF16, F16, F32, HALF_ULP
from iris_amd import attention

pytestmark = pytest.mark.gpu
EPS = 1e-6


def normal(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def angles(rotary, positions=64, seed=5):
    """Any angles will do for a rotation: the table's are the caller's."""
    g = torch.Generator().manual_seed(seed)
    angle = torch.rand((positions, rotary // 2), generator=g, dtype=torch.float64) * 6.3
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def close(got, want, dtype, dim):
    """One rounding of the result, and fp32 arithmetic on the way: a mean of dim squares, a root, five products."""
    got, want = got.double().cpu(), want.cpu()
    size = want.abs().amax(-1, keepdim=True)  # (a rotation mixes a pair: its elements are off by shares of the larger)
    bound = want.abs() * HALF_ULP[dtype] * 1.01 + size * (16 + math.sqrt(dim)) * 2.0 ** -24 + 2.0 ** -25 * (dtype == F16) + 1e-37
    off = (got - want).abs()
    assert bool((off <= bound).all()), f"off by {(off - bound).max().item()} more than {bound.max().item()}"


def cpu(*ts):
    return [None if t is None else t.cpu() for t in ts]


SHAPES = [  # tokens, q heads, k heads, head size, rotary size
    (1, 1, 1, 64, 64), (16, 4, 4, 128, 128), (17, 8, 2, 128, 64), (33, 5, 1, 96, 32), (7, 3, 3, 80, 20), (5, 2, 1, 256, 256),
    (9, 2, 2, 192, 96), (3, 1, 1, 512, 128), (4, 3, 1, 2, 2), (6, 2, 1, 50, 10), (1000, 7, 1, 128, 128), (2, 40, 8, 64, 16), (5, 2, 2, 24, 0)]


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype, interleaved, normed):
    t, hq, hk, d, rotary = shape
    q, k = normal((t, hq, d), dtype, 1), normal((t, hk, d), dtype, 2)
    cos, sin = angles(rotary) if rotary else (None, None)
    positions = torch.randint(0, 64, (t,), generator=torch.Generator().manual_seed(3)).int().cuda()
    wq = (1 + normal((d,), F32, 4, 0.2)).to(dtype) if normed else None
    wk = 1 + normal((d,), F32, 5, 0.2).to(dtype) if normed else None
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    attention.qk_norm_rope(q, k, positions, cos, sin, q_out, k_out, q_weight=wq, k_weight=wk, eps=EPS, interleaved=interleaved)
    for x, w, out in ((q, wq, q_out), (k, wk, k_out)):
        x, w, p, c, s = cpu(x, w, positions, cos, sin)
        close(out, R.norm_rope(x, w, p, c, s, EPS, interleaved), dtype, d)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page,heads_first", [(16, False), (5, False), (8, True)])
def test_the_cache_write_from_a_fused_projection_in_place(dtype, page, heads_first):
    t, hq, hk, d, rotary = 37, 6, 2, 64, 64
    qkv = normal((t, (hq + 2 * hk) * d), dtype, 7)
    before = qkv.clone()
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split((hq * d, hk * d, hk * d), 1))
    pages = 12
    shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
    caches = [torch.full(shape, -3.0, dtype=dtype, device="cuda") for _ in range(2)]
    k_cache, v_cache = (c.transpose(1, 2) if heads_first else c for c in caches)
    cos, sin = angles(rotary)
    positions = torch.arange(t, device="cuda")  # (int64)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:t].cuda()
    slots[5] = -1
    slots[6] = pages * page  # outside
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    wq, wk = (1 + normal((d,), F32, s, 0.2) for s in (1, 2))
    attention.qk_norm_rope(q, k, positions, cos, sin, q, k, q_weight=wq, k_weight=wk, eps=EPS, v=v, k_cache=k_cache, v_cache=v_cache,
                           slots=slots, status=word)
    assert word.item() == attention.STATUS_BAD_INDEX
    q0, k0, v0 = (x.unflatten(1, (-1, d)) for x in before.split((hq * d, hk * d, hk * d), 1))
    p, c, s = cpu(positions, cos, sin)
    close(q, R.norm_rope(q0.cpu(), wq.cpu(), p, c, s, EPS, False), dtype, d)
    want_k = R.norm_rope(k0.cpu(), wk.cpu(), p, c, s, EPS, False)
    close(k, want_k, dtype, d)
    assert torch.equal(v, v0)
    flat_k, flat_v = k_cache.flatten(0, 1), v_cache.flatten(0, 1)
    kept = [i for i in range(t) if 0 <= slots[i] < pages * page]
    assert torch.equal(flat_k[slots[kept]], k[kept]) and torch.equal(flat_v[slots[kept]], v0[kept])
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots[kept]] = False
    assert bool((flat_k[rest] == -3).all()) and bool((flat_v[rest] == -3).all())


def test_keys_into_the_cache_alone():
    t, d = 9, 128
    q, k, v = normal((t, 2, d), BF16, 1), normal((t, 1, d), BF16, 2), normal((t, 1, d), BF16, 3)
    cos, sin = angles(d)
    positions = torch.arange(t, device="cuda", dtype=torch.int32)
    k_cache, v_cache = torch.zeros((2, 16, 1, d), dtype=BF16, device="cuda"), torch.zeros((2, 16, 1, d), dtype=BF16, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    attention.qk_norm_rope(q, k, positions, cos, sin, q_out, k_out)
    attention.qk_norm_rope(q, k, positions, cos, sin, q_out, None, v=v, k_cache=k_cache, v_cache=v_cache, slots=torch.arange(t, device="cuda") + 8)
    assert torch.equal(k_cache.flatten(0, 1)[8:8 + t], k_out) and torch.equal(v_cache.flatten(0, 1)[8:8 + t], v)


def test_positions_outside_the_table_are_reported_and_marked():
    q, k = normal((4, 2, 64), BF16, 1), normal((4, 1, 64), BF16, 2)
    cos, sin = angles(32, positions=10)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    attention.qk_norm_rope(q, k, torch.tensor([0, 9, 10, -1], device="cuda"), cos, sin, q_out, k_out, status=word)
    assert word.item() == attention.STATUS_BAD_INDEX
    assert bool(q_out[2:, :, :32].isnan().all()) and bool(k_out[2:, :, :32].isnan().all())
    assert torch.equal(q_out[2:, :, 32:], q[2:, :, 32:]) and not bool(q_out[:2].isnan().any())


@pytest.mark.parametrize("offset", [1, 2])
def test_unaligned_heads(offset):
    t, hq, d = 6, 3, 64
    q = normal((t, hq * d + 1), F16, 1)[:, offset % 2:offset % 2 + hq * d].unflatten(1, (hq, d))
    buf = normal((t * 2 * d + 8,), F16, 2)
    k = buf[offset:offset + t * 2 * d].view(t, 2, d)
    cos, sin = angles(d)
    positions = torch.arange(t, device="cuda", dtype=torch.int32)
    q_out, k_out = torch.empty((t, hq, d), dtype=F16, device="cuda"), torch.empty((t, 2, d), dtype=F16, device="cuda")
    attention.qk_norm_rope(q, k, positions, cos, sin, q_out, k_out)
    for x, out in ((q, q_out), (k, k_out)):
        close(out, R.norm_rope(x.cpu(), None, positions.cpu(), cos.cpu(), sin.cpu(), EPS, False), F16, d)


# ---- the gradient ------------------------------------------------------------


def gradient(t, hq, hk, d, rotary, dtype, interleaved, normed, workspace_rows=None):
    q, k = normal((t, hq, d), dtype, 1), normal((t, hk, d), dtype, 2)
    dq_out, dk_out = normal((t, hq, d), dtype, 3), normal((t, hk, d), dtype, 4)
    cos, sin = angles(rotary) if rotary else (None, None)
    positions = torch.randint(0, 64, (t,), generator=torch.Generator().manual_seed(3)).int().cuda()
    wq, wk = ((1 + normal((d,), F32, s, 0.2)).to(dtype) if normed else None for s in (5, 6))
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    dwq, dwk = (torch.empty(d, device="cuda") if normed else None for _ in range(2))
    workspace = None
    if normed:
        workspace = torch.empty(workspace_rows * 2 * d, device="cuda") if workspace_rows else attention.make_gradient_workspace(d)

    def call():
        attention.qk_norm_rope_backward(dq_out, dk_out, q, k, positions, cos, sin, dq, dk, q_weight=wq, k_weight=wk, dq_weight=dwq,
                                        dk_weight=dwk, eps=EPS, interleaved=interleaved, workspace=workspace)
        return dq, dk, dwq, dwk

    call()
    want = []
    for x, dz, w in ((q, dq_out, wq), (k, dk_out, wk)):
        x, dz, w, p, c, s = cpu(x, dz, w, positions, cos, sin)
        want.append(R.norm_rope_gradient(dz, x, w, p, c, s, EPS, interleaved))
    return call, (dq, dk), (dwq, dwk), want


def check_gradient(shape, dtype, interleaved, normed, **kw):
    t, hq, hk, d, rotary = shape
    call, dx, dw, want = gradient(*shape, dtype, interleaved, normed, **kw)
    for x, w, (wx, ww), heads in zip(dx, dw, want, (hq, hk)):
        # (two sums over the head instead of one; what cancels is of the size of the gradient's largest elements)
        close(x, wx, dtype, 16 * d)
        if normed:
            # a sum of t * heads terms of a normed and a random number in fp32, partly in order
            terms = t * heads
            assert bool(((w.double().cpu() - ww).abs() <= 2.0 ** -24 * (terms + 60 * math.sqrt(terms) + 60)).all())
    first = [t.clone() for t in dx + dw if t is not None]
    call()
    assert all(torch.equal(a, b) for a, b in zip(first, [t for t in dx + dw if t is not None]))  # the same bits every time


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradient(shape, dtype, interleaved, normed):
    check_gradient(shape, dtype, interleaved, normed)


def test_gradient_of_many_tokens():
    check_gradient((9001, 3, 2, 128, 128), BF16, False, True)


def test_gradient_in_a_small_workspace():
    check_gradient((300, 3, 2, 64, 64), F32, False, True, workspace_rows=1)
    check_gradient((300, 3, 2, 64, 64), F32, False, True, workspace_rows=5)


def test_gradient_of_no_token_is_zero():
    e = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    w = torch.ones(64, device="cuda")
    dwq, dwk = torch.full((64,), 5.0, device="cuda"), torch.full((64,), 5.0, device="cuda")
    attention.qk_norm_rope_backward(e, e, e, e, None, None, None, e, e, q_weight=w, k_weight=w, dq_weight=dwq, dk_weight=dwk,
                                    workspace=attention.make_gradient_workspace(64))
    assert bool((dwq == 0).all()) and bool((dwk == 0).all())


def test_gradient_against_differences():
    """d loss / d x of loss = sum(z * r) along random directions, from the forward kernel in fp32: central differences with step h are
    off by h^2 / 6 times the third derivative, and by the forward's rounding over h."""
    t, hq, hk, d = 3, 2, 1, 64
    call, (dq, dk), (dwq, dwk), _ = gradient(t, hq, hk, d, 32, F32, True, True)
    q, k, r_q, r_k = normal((t, hq, d), F32, 1), normal((t, hk, d), F32, 2), normal((t, hq, d), F32, 3), normal((t, hk, d), F32, 4)
    cos, sin = angles(32)
    positions = torch.randint(0, 64, (t,), generator=torch.Generator().manual_seed(3)).int().cuda()
    wq, wk = (1 + normal((d,), F32, s, 0.2) for s in (5, 6))

    def loss(q, k, wq, wk):
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
        attention.qk_norm_rope(q, k, positions, cos, sin, q_out, k_out, q_weight=wq, k_weight=wk, eps=EPS, interleaved=True)
        return (q_out.double() * r_q.double()).sum() + (k_out.double() * r_k.double()).sum()

    h = 1e-2
    point = [q, k, wq, wk]
    for i, grad in enumerate((dq, dk, dwq, dwk)):
        direction = normal(point[i].shape, F32, 20 + i)
        direction = direction / direction.norm()
        ends = [loss(*[x + sign * h * direction if j == i else x for j, x in enumerate(point)]) for sign in (1, -1)]
        slope = ((ends[0] - ends[1]) / (2 * h)).item()
        want = (grad.double() * direction.double()).sum().item()
        # third derivatives of x / |x| * 8 along a unit vector are below 1 here; the sums are of some 400 terms of size 1
        assert abs(slope - want) <= h * h + 400 ** 0.5 * 2.0 ** -22 / h


def test_autograd():
    t, hq, hk, d = 11, 4, 2, 64
    leaves = [x.requires_grad_() for x in (normal((t, hq, d), BF16, 1), normal((t, hk, d), BF16, 2), 1 + normal((d,), BF16, 3, 0.2),
                                           1 + normal((d,), BF16, 4, 0.2))]
    q, k, wq, wk = leaves
    cos, sin = angles(d)
    positions = torch.arange(t, device="cuda")
    q_out, k_out = attention.QkNormRope.apply(q, k, positions, cos, sin, wq, wk, EPS)
    r = normal((t, hq, d), BF16, 9)
    (q_out * r).sum().backward()  # (no gradient arrives for k)
    want, ww = R.norm_rope_gradient(r.cpu(), q.detach().cpu(), wq.detach().cpu(), positions.cpu(), cos.cpu(), sin.cpu(), EPS, False)
    close(q.grad, want, BF16, 16 * d)
    assert bool(((wq.grad.double().cpu() - ww).abs() <= ww.abs() * HALF_ULP[BF16] * 1.01 + 1e-4).all())
    assert bool((k.grad == 0).all()) and bool((wk.grad == 0).all())
    q_out, k_out = attention.QkNormRope.apply(q.detach(), k, positions, cos, sin)
    k.grad = None
    k_out.sum().backward()  # (an expanded gradient)
    want, _ = R.norm_rope_gradient(torch.ones(t, hk, d), k.detach().cpu(), None, positions.cpu(), cos.cpu(), sin.cpu(), EPS, False)
    close(k.grad, want, BF16, 16 * d)


def test_a_rotation_in_a_captured_graph():
    t, d = 5, 128
    q, k = normal((t, 4, d), BF16, 1), normal((t, 4, d), BF16, 2)
    cos, sin = angles(d)
    positions = torch.zeros(t, dtype=torch.int32, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            attention.qk_norm_rope(q, k, positions, cos, sin, q_out, k_out)
    torch.cuda.synchronize()
    for step in range(4):
        positions.copy_(torch.arange(t) + 7 * step)
        graph.replay()
        torch.cuda.synchronize()
        close(q_out, R.norm_rope(q.cpu(), None, positions.cpu(), cos.cpu(), sin.cpu(), EPS, False), BF16, d)


def test_refusals():
    q, k = normal((4, 2, 64), BF16, 1), normal((4, 1, 64), BF16, 2)
    cos, sin = angles(64)
    positions = torch.zeros(4, dtype=torch.int32, device="cuda")
    base = dict(q=q, k=k, positions=positions, cos=cos, sin=sin, q_out=torch.empty_like(q), k_out=torch.empty_like(k))
    cache = torch.zeros((2, 4, 1, 64), dtype=BF16, device="cuda")
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")

    def call(**other):
        args = dict(base, **other)
        operands = [args.pop(n) for n in ("q", "k", "positions", "cos", "sin", "q_out", "k_out")]
        attention.qk_norm_rope(*operands, **args)

    call()
    for wrong, error in [
            (dict(q=q.double()), TypeError), (dict(k=k.half()), TypeError), (dict(k=k[:3]), ValueError), (dict(k=k[..., :32]), ValueError),
            (dict(q_out=torch.empty_like(q)[:, :1]), ValueError), (dict(q_out=torch.empty_like(q).half()), TypeError),
            (dict(q_out=q[:1].expand(4, 2, 64)), ValueError), (dict(q=q.transpose(1, 2)), ValueError), (dict(k_out=None), ValueError),
            (dict(sin=None), ValueError), (dict(cos=cos.half()), TypeError), (dict(cos=torch.cat((cos, cos), 1), sin=torch.cat((sin, sin), 1)), ValueError),
            (dict(positions=positions[:3]), ValueError), (dict(positions=positions.short()), TypeError), (dict(positions=None), ValueError),
            (dict(q_weight=torch.ones(32, device="cuda")), ValueError), (dict(q_weight=torch.ones(64, device="cuda").half()), TypeError),
            (dict(q_weight=torch.ones(64, device="cuda"), k_weight=torch.ones(64, device="cuda", dtype=BF16)), TypeError),
            (dict(slots=slots), ValueError), (dict(v=k), ValueError), (dict(slots=slots, v=k, k_cache=cache, v_cache=cache[:1]), ValueError),
            (dict(slots=slots, v=k, k_cache=cache, v_cache=cache.half()), TypeError), (dict(slots=slots.int(), v=k, k_cache=cache, v_cache=cache), TypeError),
            (dict(q=q.cpu()), RuntimeError), (dict(positions=positions.cpu()), RuntimeError), (dict(status=torch.zeros(1, device="cuda")), TypeError),
            (dict(q=q.clone().requires_grad_()), RuntimeError)]:
        with pytest.raises(error):
            call(**wrong)
    odd = torch.zeros((4, 2, 63), dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="even"):
        attention.qk_norm_rope(odd, odd, None, None, None, odd.clone(), odd.clone())
    with pytest.raises(ValueError, match="workspace"):
        w = torch.ones(64, device="cuda")
        attention.qk_norm_rope_backward(q, k, q, k, positions, cos, sin, q.clone(), k.clone(), q_weight=w, dq_weight=w.clone())
    with pytest.raises(ValueError, match="without a weight"):
        attention.qk_norm_rope_backward(q, k, q, k, positions, cos, sin, q.clone(), k.clone(), dq_weight=torch.ones(64, device="cuda"),
                                        workspace=attention.make_gradient_workspace(64))
