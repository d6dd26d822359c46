"""The attention block of one rank of a tensor-parallel decoder, over the C-ABI of ``libiris_amd.so``.

Between the shard of the query / key / value projection and the output
projection's K-shard a rank works on its own heads.  A serving step is

    build_block_tables   pages, positions and slots of the step's tokens
    qk_norm_rope         head norms, rotation, keys and values into the cache
    decode_attention     one new token a request over the paged cache
    prompt_attention     many new tokens a request over the same cache

and ``qk_norm_rope_backward`` (``QkNormRope`` under autograd) is the gradient
of the norms and the rotation for training.

Like ``iris_amd.ops`` these check operands against what the kernels assume
(types, shapes, strides, and that outputs share no memory with other operands, but for work in place)
*before* anything is launched, launch on torch's current stream, write into the
tensors they are given, and neither synchronise nor allocate.  What only the
device can see (an index outside of what it indexes, a ring of free pages
that runs out) is OR-ed into an optional ``status`` word, as ``STATUS_*`` bits.

A cache is a tensor ``[pages, page_size, key heads, head size]`` in any order
of memory whose head elements are contiguous; ``block_table[i, j]`` is the page of request i's
tokens ``[j * page_size, (j + 1) * page_size)``.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _native
from ._native import STATUS_BAD_INDEX, STATUS_NO_PAGES, STATUS_NO_ROOM
from .ops import _DTYPES, _ptr, _require_cuda

__all__ = [
    "rope_tables",
    "build_block_tables",
    "qk_norm_rope",
    "qk_norm_rope_backward",
    "QkNormRope",
    "decode_attention",
    "prompt_attention",
    "make_workspace",
    "make_gradient_workspace",
    "STATUS_BAD_INDEX",
    "STATUS_NO_PAGES",
    "STATUS_NO_ROOM",
]

MAX_REQUESTS = 8192  # of a call of build_block_tables (include/iris_amd.h)
MAX_HEAD_DIM = 512  # of the norms and the rotation
MAX_ATTENTION_HEAD_DIM = 256
INT32_MAX = (1 << 31) - 1


# ---- checks ------------------------------------------------------------------


def _heads(name, t, device, dtype=None, tokens=None, heads=None, dim=None):
    """A tensor [tokens, heads, head size] whose head elements are contiguous."""
    _require_cuda(name, t, device)
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head size], got {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    for what, want, got in (("tokens", tokens, t.shape[0]), ("heads", heads, t.shape[1]), ("elements a head", dim, t.shape[2])):
        if want is not None and want != got:
            raise ValueError(f"{name} has {got} {what}, expected {want}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: the elements of a head must be contiguous")
    return t


def _output(name, t):
    """Something that a kernel writes: its elements must not share memory with each other."""
    live = [(s, n) for s, n in zip(t.stride(), t.shape) if n > 1]
    reach = 0
    for stride, n in sorted(live):
        if stride <= reach:
            raise ValueError(f"{name}: elements of an output must not overlap")
        reach += stride * (n - 1)
    if _differentiated(t):
        raise RuntimeError(f"{name} requires a gradient; outputs are written in place")


def _same_view(a, b):
    return (a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and a.shape == b.shape
            and all(n <= 1 or s == z for n, s, z in zip(a.shape, a.stride(), b.stride())))


def _apart(outputs, inputs, in_place=()):
    """(name, tensor) outputs share no memory with each other or with the inputs, but for an output that is one of its own inputs,
    element by element: (output, input) names ``in_place``."""
    outputs, inputs = ([(name, t) for name, t in operands if t is not None] for operands in (outputs, inputs))
    for i, (name, t) in enumerate(outputs):
        others = outputs[:i] + [(other, x) for other, x in inputs if not ((name, other) in in_place and _same_view(t, x))]
        for other, x in others:
            if _native.host().overlap(t, x):
                raise ValueError(f"{name} shares memory with {other}: an output lies in memory of its own, or is its own input")


def _ints(name, t, device, dtype, numel, exact=True):
    _require_cuda(name, t, device)
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous vector of {dtype}")
    if t.numel() != numel if exact else t.numel() < numel:
        raise ValueError(f"{name} has {t.numel()} elements, expected {numel}")


def _status(t, device):
    if t is not None:
        _require_cuda("status", t, device)
        if t.dtype not in (torch.int32, torch.uint32) or t.numel() < 1:
            raise TypeError("status must be a 32-bit device word")


def _cache(name, t, device, dtype, heads, dim):
    _require_cuda(name, t, device)
    if t.dim() != 4:
        raise ValueError(f"{name} must be [pages, page_size, key heads, head size], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape[2] != heads or t.shape[3] != dim:
        raise ValueError(f"{name} holds {t.shape[2]} heads of {t.shape[3]}, expected {heads} of {dim}")
    if t.shape[1] < 1:
        raise ValueError(f"{name} has empty pages")
    if t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"{name}: the elements of a head must be contiguous")


def _tangent(t):
    return torch.autograd.forward_ad.unpack_dual(t).tangent is not None


def _differentiated(t):
    """Whether autograd has business with a tensor: a gradient, or a tangent (forward mode)."""
    return t is not None and ((torch.is_grad_enabled() and t.requires_grad) or _tangent(t))


def _no_gradient(*tensors):
    if any(_differentiated(t) for t in tensors):
        raise RuntimeError("no gradient flows through this call; QkNormRope is the differentiable form of qk_norm_rope "
                           "(in heads and weights), and attention over a cache has none")


DECLINED = -1  # the native module: not a call of the ordinary kind, nothing was launched


def _native_call(err):
    """Whether a call is done.  What the native code declined, or its launcher may have refused, goes through the full checks, which say
    what is wrong; then ``_rest``."""
    if err > 0 and err != _native.HIP_ERROR_INVALID_VALUE:
        _native.hip_try(err)
    return err == 0


def _rest(err, name, args, device):
    """Launches a call that the native code declined.  Any other status may have come from behind a launch, which is not made again."""
    if err != DECLINED:
        _rejected(name)
    _launch(name, args, device)


def _rejected(name):
    raise ValueError(f"{name} rejected the arguments (sizes, strides or alignment it does not take)")


def _launch(name, args, device):
    stream = torch.cuda.current_stream(device).cuda_stream
    with torch.cuda.device(device):
        err = getattr(_native.lib(), name)(ctypes.byref(args), stream)
    if err == _native.HIP_ERROR_INVALID_VALUE:
        _rejected(name)
    _native.hip_try(err)


# ---- block tables ------------------------------------------------------------


def build_block_tables(cached, new_tokens, block_table, pool, pool_state, page_size, *, lengths, pool_state_out, query_starts,
                       positions, slots, status=None):
    """Pages, positions and slots of a step, on the device, from request lengths.

    ``cached`` int32 [requests]: tokens in the cache; ``new_tokens`` int32:
    tokens that the step adds (0: none, -1: the request has ended and gives its
    pages back).  ``pool`` int32 is a ring of free pages and ``pool_state`` int64 [2]
    how many were ever (taken, put in): free is ``pool[x % len(pool)]`` for x in between; ``len(pool)`` is at
    least the number of pages.  Requests take pages in order; one that does not get
    all it needs (the ring runs out, or ``block_table`` [requests, width] is too narrow) gets
    none and sets ``STATUS_NO_PAGES``: its length stays and its tokens have slot -1.

    Writes the fresh entries of ``block_table`` and the returned pages of ``pool`` in place,
    ``lengths`` int32 [requests] (tokens after the step), ``pool_state_out``,
    ``query_starts`` int32 [requests + 1], and ``positions`` int32 and ``slots`` int64 of
    every token, up to their common length (0 and -1 past the last token).
    ``lengths`` and ``pool_state_out`` may not be ``cached`` and ``pool_state``.
    """
    err = _native.host().block_tables(cached, new_tokens, block_table, pool, pool_state, lengths, pool_state_out, query_starts,
                                      positions, slots, status, page_size)
    if _native_call(err):
        return
    device = cached.device
    requests = cached.numel()
    _ints("cached", cached, device, torch.int32, requests)
    _ints("new_tokens", new_tokens, device, torch.int32, requests)
    _ints("lengths", lengths, device, torch.int32, requests)
    _ints("query_starts", query_starts, device, torch.int32, requests + 1)
    _ints("pool", pool, device, torch.int32, 1, exact=False)
    _ints("pool_state", pool_state, device, torch.int64, 2)
    _ints("pool_state_out", pool_state_out, device, torch.int64, 2)
    _ints("positions", positions, device, torch.int32, positions.numel())
    _ints("slots", slots, device, torch.int64, positions.numel())
    _require_cuda("block_table", block_table, device)
    _status(status, device)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != requests:
        raise TypeError("block_table must be an int32 matrix with a row a request")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("the rows of block_table must be contiguous")
    if requests > 1:
        _output("block_table", block_table)
    if requests > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests, got {requests}")
    if page_size < 1:
        raise ValueError("page_size must be positive")
    if max(block_table.shape[1], 1) * page_size > INT32_MAX:
        raise ValueError("block_table has room for more tokens than 31 bits count")
    written = (block_table, pool, lengths, pool_state_out, query_starts, positions, slots)
    spans = [(t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape))))
             for t in written + (cached, new_tokens, pool_state) if t.numel()]
    spans.sort()
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("operands overlap: lengths and pool_state_out are tensors of their own")
    a = _native.BlockTablesArgs()
    a.cached, a.new_tokens, a.block_table, a.pool = _ptr(cached), _ptr(new_tokens), _ptr(block_table), _ptr(pool)
    a.pool_state, a.pool_state_out, a.lengths = _ptr(pool_state), _ptr(pool_state_out), _ptr(lengths)
    a.query_starts, a.positions, a.slots, a.status = _ptr(query_starts), _ptr(positions), _ptr(slots), _ptr(status)
    a.requests, a.table_width, a.page_size = requests, block_table.shape[1], page_size
    a.stride_table = max(block_table.stride(0), block_table.shape[1])
    a.pool_size, a.max_tokens = pool.numel(), positions.numel()
    _rest(err, "iris_block_tables_launch", a, device)


# ---- norms and rotation ------------------------------------------------------


def rope_tables(max_positions, rotary_dim, *, base=10000.0, scaling=None, device="cuda"):
    """(cos, sin) fp32 [max_positions, rotary_dim / 2] of the angles ``position * base ** (-2 i / rotary_dim)``,
    computed in 64 bits: made once, kept by the program.

    ``scaling`` stretches the positions for contexts longer than the trained
    ones; a dict with ``"type"`` and ``"factor"`` (how many times longer):

    * ``"linear"``: every angle is divided by the factor.
    * ``"base"``: the base grows by ``factor ** (rotary_dim / (rotary_dim - 2))``, so that
      the slowest angle is divided by the factor and the fastest stays.
    * ``"by_parts"``: pairs that turn at least ``fast`` (32) times within ``trained`` positions
      keep their angles, those that turn at most ``slow`` (1) times are divided by the
      factor, and between them the two are mixed by a ramp over the pair's index.  Queries and keys both grow
      by ``attention_factor`` (``1 + 0.1 ln factor``), as cos and sin do here.
    * ``"by_wavelength"``: the same with a ramp over the number of turns within ``trained`` positions
      between ``slow`` (1) and ``fast`` (4), and nothing grows.
    """
    if max_positions < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("max_positions must be positive and rotary_dim even")
    if base <= 0:
        raise ValueError("base must be positive")
    scaling = dict(scaling or {"type": "linear", "factor": 1.0})
    kind, factor = scaling.pop("type", None), float(scaling.pop("factor", 0))
    if kind not in ("linear", "base", "by_parts", "by_wavelength"):
        raise ValueError(f"unknown scaling type {kind!r}")
    if factor < 1:
        raise ValueError("scaling needs a factor of at least 1")
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    growth = 1.0
    if kind == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = float(base) ** (-2.0 * pair / rotary_dim)
    if kind == "linear":
        freq = freq / factor
    elif kind in ("by_parts", "by_wavelength"):
        trained = scaling.pop("trained", None)
        if not trained or trained < 1:
            raise ValueError(f"scaling {kind!r} needs the number of trained positions")
        fast = float(scaling.pop("fast", 32.0 if kind == "by_parts" else 4.0))
        slow = float(scaling.pop("slow", 1.0))
        if not fast > slow > 0:
            raise ValueError("scaling needs fast > slow > 0")
        if kind == "by_parts":
            growth = float(scaling.pop("attention_factor", 1.0 + 0.1 * math.log(factor)))

            def index(turns):  # the (fractional) pair that turns so often within the trained positions
                return rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

            lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
            keep = 1 - ((pair - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        else:
            keep = ((trained * freq / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    if scaling:
        raise ValueError(f"scaling {kind!r} does not take {sorted(scaling)}")
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return (growth * angle.cos()).float(), (growth * angle.sin()).float()


def _rope_operands(a, device, dtype, tokens, dim, positions, cos, sin, q_weight, k_weight, eps, interleaved):
    if dim % 2 or not 0 < dim <= MAX_HEAD_DIM:
        raise ValueError(f"the head size must be even and at most {MAX_HEAD_DIM}, got {dim}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            _require_cuda(name, t, device)
            if t.dtype != torch.float32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
                raise TypeError(f"{name} must be an fp32 matrix [positions, rotary size / 2] with contiguous rows")
        if cos.shape != sin.shape or cos.shape[0] < 1:
            raise ValueError("cos and sin must have the same shape and at least one position")
        if 2 * cos.shape[1] > dim:
            raise ValueError(f"angles for {2 * cos.shape[1]} elements, a head has {dim}")
        if positions is None:
            raise ValueError("positions are required to rotate")
        _require_cuda("positions", positions, device)
        if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 1 or not positions.is_contiguous():
            raise TypeError("positions must be a contiguous vector of int32 or int64")
        if positions.numel() != tokens:
            raise ValueError(f"{positions.numel()} positions for {tokens} tokens")
        if cos.shape[0] > INT32_MAX:
            raise ValueError("too many positions")
        a.cos, a.sin, a.positions = _ptr(cos), _ptr(sin), _ptr(positions)
        a.stride_cos, a.stride_sin = cos.stride(0), sin.stride(0)
        a.rotary_dim, a.max_positions = 2 * cos.shape[1], cos.shape[0]
        a.positions_64 = int(positions.dtype == torch.int64)
    kinds = set()
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            _require_cuda(name, w, device)
            if w.dtype not in (dtype, torch.float32):
                raise TypeError(f"{name} must be {dtype} or fp32, got {w.dtype}")
            if w.shape != (dim,) or not w.is_contiguous():
                raise ValueError(f"{name} must be a contiguous vector of {dim}")
            kinds.add(w.dtype)
    if len(kinds) > 1:
        raise TypeError("q_weight and k_weight must share a dtype")
    a.q_weight, a.k_weight = _ptr(q_weight), _ptr(k_weight)
    a.weight_fp32 = int(kinds == {torch.float32})
    a.interleaved, a.eps, a.dtype = int(bool(interleaved)), float(eps), _DTYPES[dtype]
    a.tokens, a.head_dim = tokens, dim


def _strides(a, prefix, t):
    token, head = _steps(t, 2)
    setattr(a, f"stride_{prefix}t", token)
    setattr(a, f"stride_{prefix}h", head)


def qk_norm_rope(q, k, positions, cos, sin, q_out, k_out, *, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, v=None,
                 k_cache=None, v_cache=None, slots=None, status=None):
    """Norm, rotate and store query and key heads in one pass.

    ``q`` [tokens, query heads, head size] and ``k`` [tokens, key heads, head size]
    (views of a fused projection's output will do; fp16, bf16 or fp32) become
    ``x / sqrt(mean(x^2) + eps) * weight`` per head, each where it has a weight
    ([head size], of the heads' type or fp32), and their first ``2 * cos.shape[1]`` elements turn by
    the angles of the token's position (``rope_tables``; ``cos`` None: no rotation): pairs are the
    two halves' elements, or neighbours if ``interleaved``.  fp32 inside, rounded once.

    Queries go to ``q_out``, keys to ``k_out`` (the inputs themselves, for
    work in place) and, with ``slots`` int64 [tokens], keys and values ``v`` to their
    slots of ``k_cache`` / ``v_cache`` [pages, page size, key heads, head size]; a negative
    slot is skipped, and with a cache ``k_out`` may be None.
    """
    err = _native.host().qk_norm_rope(q, k, positions, cos, sin, q_out, k_out, q_weight, k_weight, v, k_cache, v_cache, slots,
                                      status, eps, interleaved)
    if _native_call(err):
        return
    device, dtype = q.device, q.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"q: unsupported dtype {dtype}")
    _heads("q", q, device)
    tokens, hq, dim = q.shape
    _heads("k", k, device, dtype, tokens, None, dim)
    hk = k.shape[1]
    _heads("q_out", q_out, device, dtype, tokens, hq, dim)
    _no_gradient(q, k, v, cos, sin, q_weight, k_weight)
    outputs = [("q_out", q_out)]
    a = _native.QkNormRopeArgs()
    _rope_operands(a, device, dtype, tokens, dim, positions, cos, sin, q_weight, k_weight, eps, interleaved)
    _status(status, device)
    a.q_heads, a.k_heads = hq, hk
    a.q, a.k, a.q_out, a.status = _ptr(q), _ptr(k), _ptr(q_out), _ptr(status)
    _strides(a, "q", q)
    _strides(a, "k", k)
    _strides(a, "qo", q_out)
    if k_out is not None:
        _heads("k_out", k_out, device, dtype, tokens, hk, dim)
        outputs.append(("k_out", k_out))
        a.k_out = _ptr(k_out)
        _strides(a, "ko", k_out)
    if slots is not None:
        if v is None or k_cache is None or v_cache is None:
            raise ValueError("slots need v, k_cache and v_cache")
        _heads("v", v, device, dtype, tokens, hk, dim)
        _ints("slots", slots, device, torch.int64, tokens)
        for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
            _cache(name, t, device, dtype, hk, dim)
            outputs.append((name, t))
        if k_cache.shape != v_cache.shape:
            raise ValueError("k_cache and v_cache must have the same shape")
        a.num_slots = k_cache.shape[0] * k_cache.shape[1]
        if a.num_slots > INT32_MAX:
            raise ValueError("more slots than 31 bits count")
        a.v, a.slots, a.k_cache, a.v_cache = _ptr(v), _ptr(slots), _ptr(k_cache), _ptr(v_cache)
        _strides(a, "v", v)
        a.stride_kc_page, a.stride_kc_row, a.stride_kc_head = _steps(k_cache, 3)
        a.stride_vc_page, a.stride_vc_row, a.stride_vc_head = _steps(v_cache, 3)
        a.page_size = k_cache.shape[1]
    elif v is not None or k_cache is not None or v_cache is not None:
        raise ValueError("v, k_cache and v_cache need slots")
    elif k_out is None and hk:
        raise ValueError("k_out is required without a cache")
    for name, t in outputs:
        _output(name, t)
    _apart(outputs, [("q", q), ("k", k), ("v", v), ("positions", positions), ("cos", cos), ("sin", sin), ("q_weight", q_weight),
                     ("k_weight", k_weight), ("slots", slots)], [("q_out", "q"), ("k_out", "k")])
    _rest(err, "iris_qk_norm_rope_launch", a, device)


def make_gradient_workspace(head_dim, *, device="cuda"):
    """A workspace for the weight gradients of ``qk_norm_rope_backward``: a row of ``head_dim`` partial sums for each of the (at most)
    1024 workgroups of a launch."""
    return torch.empty(1024 * head_dim, dtype=torch.float32, device=device)


def qk_norm_rope_backward(dq_out, dk_out, q, k, positions, cos, sin, dq, dk, *, q_weight=None, k_weight=None, dq_weight=None,
                          dk_weight=None, eps=1e-6, interleaved=False, workspace=None, status=None):
    """The gradient of ``qk_norm_rope``: ``dq`` and ``dk`` from those of its outputs and its inputs ``q`` and ``k``.

    ``dq_weight`` / ``dk_weight`` fp32 [head size] (None: not wanted) are summed over tokens and
    heads in a fixed order, in ``workspace`` (``make_gradient_workspace``; fp32, as
    few as 2 * head size elements).  ``dq`` may be ``dq_out`` or ``q``, and ``dk`` ``dk_out`` or ``k``.
    """
    err = _native.host().qk_norm_rope_backward(dq_out, dk_out, q, k, positions, cos, sin, dq, dk, q_weight, k_weight, dq_weight,
                                               dk_weight, workspace, status, eps, interleaved)
    if _native_call(err):
        return
    device, dtype = q.device, q.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"q: unsupported dtype {dtype}")
    _heads("q", q, device)
    tokens, hq, dim = q.shape
    _heads("k", k, device, dtype, tokens, None, dim)
    hk = k.shape[1]
    for name, t, heads in (("dq_out", dq_out, hq), ("dq", dq, hq), ("dk_out", dk_out, hk), ("dk", dk, hk)):
        _heads(name, t, device, dtype, tokens, heads, dim)
    if any(t is not None and _tangent(t) for t in (dq_out, dk_out, q, k, cos, sin, q_weight, k_weight)):
        raise RuntimeError("no gradient flows through this call, and no tangent")
    a = _native.QkNormRopeBackwardArgs()
    _rope_operands(a, device, dtype, tokens, dim, positions, cos, sin, q_weight, k_weight, eps, interleaved)
    _status(status, device)
    a.q_heads, a.k_heads = hq, hk
    for name, t, w in (("dq_weight", dq_weight, q_weight), ("dk_weight", dk_weight, k_weight)):
        if t is not None:
            if w is None:
                raise ValueError(f"{name} without a weight")
            _require_cuda(name, t, device)
            if t.dtype != torch.float32 or t.shape != (dim,) or not t.is_contiguous():
                raise TypeError(f"{name} must be a contiguous fp32 vector of {dim}")
            _output(name, t)
    if dq_weight is not None or dk_weight is not None:
        if workspace is None:
            raise ValueError("weight gradients need a workspace")
        _require_cuda("workspace", workspace, device)
        if workspace.dtype != torch.float32 or not workspace.is_contiguous() or workspace.numel() < 2 * dim:
            raise TypeError(f"workspace must be contiguous fp32 of at least {2 * dim} elements")
        a.workspace, a.workspace_elems = _ptr(workspace), workspace.numel()
    for name, t in (("dq", dq), ("dk", dk)):
        _output(name, t)
    written = [("dq", dq), ("dk", dk), ("workspace", workspace)]
    _apart(written, [("dq_out", dq_out), ("dk_out", dk_out), ("q", q), ("k", k), ("positions", positions), ("cos", cos), ("sin", sin),
                     ("q_weight", q_weight), ("k_weight", k_weight)], [("dq", "dq_out"), ("dq", "q"), ("dk", "dk_out"), ("dk", "k")])
    # (the weights' gradients are written by a launch of their own, behind the last read of an input)
    _apart(written + [("dq_weight", dq_weight), ("dk_weight", dk_weight)], [])
    a.dq_out, a.dk_out, a.q, a.k, a.dq, a.dk = _ptr(dq_out), _ptr(dk_out), _ptr(q), _ptr(k), _ptr(dq), _ptr(dk)
    a.dq_weight, a.dk_weight, a.status = _ptr(dq_weight), _ptr(dk_weight), _ptr(status)
    for prefix, t in (("dqo", dq_out), ("dko", dk_out), ("q", q), ("k", k), ("dq", dq), ("dk", dk)):
        _strides(a, prefix, t)
    _rest(err, "iris_qk_norm_rope_backward_launch", a, device)


class QkNormRope(torch.autograd.Function):
    """``QkNormRope.apply(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved)`` -> (q, k), normed and rotated,
    under autograd: gradients for q, k and the weights."""

    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
        if any(ctx.needs_input_grad[3:5]):
            raise RuntimeError("no gradient flows to the angles")
        q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format)
        qk_norm_rope(q, k, positions, cos, sin, q_out, k_out, q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved)
        ctx.save_for_backward(q, k, positions, cos, sin, q_weight, k_weight)
        ctx.eps, ctx.interleaved = eps, interleaved
        return q_out, k_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, positions, cos, sin, q_weight, k_weight = ctx.saved_tensors
        dim = q.shape[2]
        wanted = ctx.needs_input_grad + (False,) * 2  # (weights that were left out have no entry)
        dq, dk = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format)
        dqw, dkw = (torch.empty(dim, dtype=torch.float32, device=q.device) if w is not None and asked else None
                    for w, asked in ((q_weight, wanted[5]), (k_weight, wanted[6])))
        workspace = make_gradient_workspace(dim, device=q.device) if dqw is not None or dkw is not None else None
        # (a gradient that arrives expanded or permuted is laid out first)
        dq_out, dk_out = (t if t.stride(2) == 1 else t.contiguous() for t in (dq_out, dk_out))
        qk_norm_rope_backward(dq_out, dk_out, q, k, positions, cos, sin, dq, dk, q_weight=q_weight, k_weight=k_weight,
                              dq_weight=dqw, dk_weight=dkw, eps=ctx.eps, interleaved=ctx.interleaved, workspace=workspace)
        dqw, dkw = (None if t is None else t.to(w.dtype) for t, w in ((dqw, q_weight), (dkw, k_weight)))
        return dq, dk, None, None, None, dqw, dkw, None, None


# ---- attention ---------------------------------------------------------------


def make_workspace(head_dim, *, device="cuda"):
    """A workspace for ``decode_attention`` and ``prompt_attention`` of heads of this size: the parts of long contexts meet in it.
    Zeroed here and left zeroed where it has to be by every launch; for one stream at a time."""
    elems = _native.lib().iris_attention_workspace_elems(head_dim)
    if elems <= 0:
        raise ValueError(f"the head size must be positive and at most {MAX_ATTENTION_HEAD_DIM}, got {head_dim}")
    return torch.zeros(elems, dtype=torch.float32, device=device)


def _without_a_page(out, lse, status, lengths, query_starts, room):
    """The rows of a call that has no page to read: NaN where one sees a key, else zeros, and reported as the kernels do."""
    tokens = torch.arange(out.shape[0], device=out.device)
    if query_starts is None:
        row, begin, new, mine = tokens, tokens, 1, torch.ones_like(tokens, dtype=torch.bool)
    else:
        row = torch.searchsorted(query_starts[1:].contiguous(), tokens, right=True).clamp(max=len(lengths) - 1)
        begin, new = query_starts[row], query_starts[row + 1] - query_starts[row]
        mine = (tokens >= query_starts[0]) & (tokens < query_starts[-1])
    sees = mine & (lengths.clamp(0, room)[row] - new + tokens - begin >= 0)
    for t, none in ((out, 0.0), (lse, -math.inf)):
        if t is not None:
            shape = [-1] + [1] * (t.dim() - 1)
            t.masked_fill_(mine.view(shape), none).masked_fill_(sees.view(shape), math.nan)
    if status is not None:
        bits = (sees.any() | (lengths > room).any()).int() * STATUS_BAD_INDEX
        status.view(torch.int32).as_strided((1,), (1,)).bitwise_or_(bits)


def _attention(q, k_cache, v_cache, block_table, lengths, query_starts, out, scale, window, sinks, lse, workspace, status):
    err = _native.host().attention(q, k_cache, v_cache, block_table, lengths, query_starts, out, lse, workspace, status, scale,
                                   window, sinks)
    if _native_call(err):
        return
    device, dtype = q.device, q.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"q: unsupported dtype {dtype}")
    _heads("q", q, device)
    tokens, hq, dim = q.shape
    _heads("out", out, device, dtype, tokens, hq, dim)
    _require_cuda("k_cache", k_cache, device)
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be [pages, page_size, key heads, head size], got {tuple(k_cache.shape)}")
    pages, page_size, hk, _ = k_cache.shape
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _cache(name, t, device, dtype, hk, dim)
    if v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    if hk == 0 or hq % hk:
        raise ValueError(f"{hq} query heads do not divide over {hk} key heads")
    vec = 16 // q.element_size()
    if dim % vec or not 0 < dim <= MAX_ATTENTION_HEAD_DIM:
        raise ValueError(f"the head size must be a multiple of {vec} and at most {MAX_ATTENTION_HEAD_DIM}, got {dim}")
    for name, t in (("q", q), ("out", out), ("k_cache", k_cache), ("v_cache", v_cache)):
        if t.data_ptr() % 16 or any(s % vec for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
            raise ValueError(f"{name}: every head must begin at a multiple of 16 bytes")
    _require_cuda("block_table", block_table, device)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise TypeError("block_table must be an int32 matrix with contiguous rows")
    requests, width = block_table.shape
    if requests > 1 and block_table.stride(0) < width:
        raise ValueError("the rows of block_table must not overlap")
    _ints("lengths", lengths, device, torch.int32, requests)
    if query_starts is None:
        if requests != tokens:
            raise ValueError(f"{tokens} queries for {requests} requests; decode_attention takes one each")
    else:
        _ints("query_starts", query_starts, device, torch.int32, requests + 1)
    if width * page_size > INT32_MAX:
        raise ValueError("block_table has room for more tokens than 31 bits count")
    if scale is None:
        scale = dim ** -0.5
    if not 0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    _no_gradient(q, k_cache, v_cache)
    _output("out", out)
    _status(status, device)
    a = _native.AttentionArgs()
    if lse is not None:
        _require_cuda("lse", lse, device)
        if lse.dtype != torch.float32 or lse.shape != (tokens, hq) or (hq > 1 and lse.stride(1) != 1):
            raise TypeError("lse must be an fp32 matrix [tokens, query heads] with contiguous rows")
        _output("lse", lse)
        a.lse, a.stride_lse = _ptr(lse), lse.stride(0)
    if workspace is not None:
        _require_cuda("workspace", workspace, device)
        if workspace.dtype != torch.float32 or not workspace.is_contiguous() or workspace.data_ptr() % 16:
            raise TypeError("workspace must be contiguous fp32 at a multiple of 16 bytes (make_workspace)")
        a.workspace, a.workspace_elems = _ptr(workspace), workspace.numel()
    _apart([("out", out), ("lse", lse), ("workspace", workspace)],
           [("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("block_table", block_table), ("lengths", lengths), ("query_starts", query_starts)],
           [("out", "q")])
    if tokens == 0 or hq == 0:
        return
    if requests == 0:
        raise ValueError("queries of no request")
    if width == 0 or pages == 0:
        _without_a_page(out, lse, status, lengths, query_starts, width * page_size)
        return
    a.q, a.k_cache, a.v_cache, a.out = _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out)
    a.block_table, a.lengths, a.query_starts, a.status = _ptr(block_table), _ptr(lengths), _ptr(query_starts), _ptr(status)
    a.stride_qt, a.stride_qh = _steps(q, 2)
    a.stride_ot, a.stride_oh = _steps(out, 2)
    a.stride_kc_page, a.stride_kc_row, a.stride_kc_head = _steps(k_cache, 3)
    a.stride_vc_page, a.stride_vc_row, a.stride_vc_head = _steps(v_cache, 3)
    a.stride_table = block_table.stride(0) if requests > 1 else width
    a.requests, a.tokens, a.q_heads, a.k_heads, a.head_dim = requests, tokens, hq, hk, dim
    a.page_size, a.table_width, a.num_pages = page_size, width, pages
    # (no context is longer than 31 bits count, so that the most they hold is all keys)
    a.window, a.sinks, a.dtype, a.scale = min(window, INT32_MAX), min(sinks, INT32_MAX), _DTYPES[dtype], scale
    _rest(err, "iris_attention_launch", a, device)


def _steps(t, n):
    # (the stride of an axis of one element is never taken, and need not be a multiple of anything)
    return [s if size > 1 else 0 for s, size in zip(t.stride()[:n], t.shape[:n])]


def decode_attention(q, k_cache, v_cache, block_table, lengths, out, *, scale: Optional[float] = None, window=0, sinks=0, lse=None,
                     workspace=None, status=None):
    """Attention of one new token a request over the paged cache.

    ``q`` and ``out`` [requests, query heads, head size] (fp16, bf16 or fp32);
    ``lengths`` int32 [requests]: keys of each request, the new token's own
    (written before, ``qk_norm_rope``) among them; 0 gives zeros.  Query head h reads key head ``h // (query heads // key heads)``.
    ``window`` > 0: only the last ``window`` keys are seen, and the first ``sinks``.
    ``scale`` is ``head size ** -0.5`` by default; ``lse`` fp32 [requests, query heads] takes the logarithms of the
    softmax sums.  With a ``workspace`` (``make_workspace``) long contexts are split over the GPU and joined; one too small for that is none.

    With heads of 16 bits the softmax's weights are rounded to the heads' type for the product with the values, and divided by
    the sum of the rounded ones; sums are fp32 (and values times the number of keys have to stay in its range).  A
    table's entry need be no page where no query sees one of its keys: pages behind a window may be given back.
    ``out`` may be ``q``, and shares no other memory with an operand.
    """
    _attention(q, k_cache, v_cache, block_table, lengths, None, out, scale, window, sinks, lse, workspace, status)


def prompt_attention(q, k_cache, v_cache, block_table, lengths, query_starts, out, *, scale: Optional[float] = None, window=0,
                     sinks=0, lse=None, workspace=None, status=None):
    """Causal attention of many new tokens a request over the paged cache.

    Request i's queries are the tokens ``query_starts[i] .. query_starts[i + 1]`` of ``q`` [tokens, query heads, head size] and stand at the last
    positions of its ``lengths[i]`` keys (written before): a query sees the
    keys up to its own position.  With ``window`` > 0 it sees the last ``window`` of
    them and the request's first ``sinks``.  Rows of ``out`` past the last request's stay as they are.  The rest is as in ``decode_attention``.
    """
    _attention(q, k_cache, v_cache, block_table, lengths, query_starts, out, scale, window, sinks, lse, workspace, status)
