#!/usr/bin/env python3
"""The attention half of a tensor-parallel decoder layer, serving: prompts, then one token a request a step.

One GPU plays ``--ranks`` ranks, as the GEMM examples do with
``--virtual_ranks``.  A rank holds its share of the heads, a paged cache of its key heads
and its shards of both projections.  A step is

    build_block_tables    pages, positions and slots (the same for every rank)
    gemm_launch           qkv = x @ W_qkv, the rank's shard
    qk_norm_rope          head norms, rotation, keys and values into the cache
    prompt_attention      or decode_attention: the rank's heads over the cache
    one-shot all-reduce   y = sum over ranks of heads @ W_o, the rank's K-shard

and requests that end give their pages back to the ring, from which later steps take them.
``--validate`` compares every step's output with the layer computed densely in 64 bits on the CPU.
"""

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.abspath(os.path.join(os.path.dirname(__file__), "..", "..")))

import iris_amd as iris  # noqa: E402
from iris_amd import attention, ops  # noqa: E402
from iris_amd.matmul import matmul_one_shot_all_reduce as all_reduce  # noqa: E402

DATATYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
PROGRAMS, TILE_M, TILE_N = 256, 64, 64
EPS = 1e-6


def parse_args(argv=None):
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0], formatter_class=argparse.ArgumentDefaultsHelpFormatter)
    p.add_argument("--ranks", type=int, default=4, help="Ranks played by this one GPU")
    p.add_argument("--hidden", type=int, default=1024, help="Width of the layer")
    p.add_argument("--heads", type=int, default=16, help="Query heads of the layer")
    p.add_argument("--key_heads", type=int, default=4, help="Key heads of the layer")
    p.add_argument("--head_dim", type=int, default=64, help="Elements of a head")
    p.add_argument("--prompts", type=int, nargs="+", default=[37, 1, 90, 300], help="Tokens of each request's prompt")
    p.add_argument("--steps", type=int, default=6, help="Single-token steps behind the prompts")
    p.add_argument("--page_size", type=int, default=16, help="Tokens of a cache page")
    p.add_argument("--pages", type=int, default=128, help="Pages of each rank's cache")
    p.add_argument("--window", type=int, default=0, help="Sliding window (0: none)")
    p.add_argument("--sinks", type=int, default=0, help="First tokens that stay visible outside of the window")
    p.add_argument("--datatype", choices=list(DATATYPES), default="bf16", help="Datatype of computation")
    p.add_argument("-v", "--validate", action="store_true", help="Compare with the dense layer in 64 bits")
    return p.parse_args(argv)


class Layer:
    """Every rank's shards and buffers, and the requests' state on the device."""

    def __init__(self, args):
        self.args, ranks, d = args, args.ranks, args.head_dim
        self.dtype = DATATYPES[args.datatype]
        self.hq, self.hk = args.heads // ranks, args.key_heads // ranks
        self.most = max(sum(args.prompts), len(args.prompts))  # tokens of the largest step
        wide = (self.hq + 2 * self.hk) * d
        heap = self.most * args.hidden * (4 + 2) + 4 * (ops.cdiv(self.most, TILE_M) * ops.cdiv(args.hidden, TILE_N) + PROGRAMS * (TILE_M * TILE_N + 1))
        self.shmem = iris.iris(heap + (1 << 20) & ~0xFFFFF, virtual_ranks=ranks)
        g = torch.Generator().manual_seed(123)

        def normal(*shape, std=1.0):
            return (torch.randn(shape, generator=g) * std).to(self.dtype).cuda()

        # weights as a linear layer keeps them ([out, in]); columns of the output projection belong to heads
        self.w_qkv = [normal(wide, args.hidden, std=args.hidden ** -0.5) for _ in range(ranks)]
        self.w_o = [normal(args.hidden, self.hq * d, std=(args.heads * d) ** -0.5) for _ in range(ranks)]
        self.q_weight, self.k_weight = 1 + normal(d, std=0.1), 1 + normal(d, std=0.1)
        self.cos, self.sin = attention.rope_tables(args.pages * args.page_size, d)
        cache = (args.pages, args.page_size, self.hk, d)
        self.caches = [(torch.zeros(cache, dtype=self.dtype, device="cuda"), torch.zeros(cache, dtype=self.dtype, device="cuda"))
                       for _ in range(ranks)]
        self.workspace = attention.make_workspace(d)
        # what peers touch lies in the symmetric heap: partial sums, results, ready flags
        self.partial = self.shmem.zeros((self.most, args.hidden), dtype=torch.float32)
        self.result = self.shmem.zeros((self.most, args.hidden), dtype=self.dtype)
        self.flags = self.shmem.zeros((ops.cdiv(self.most, TILE_M) * ops.cdiv(args.hidden, TILE_N),), dtype=torch.int32)
        self.P = self.shmem.zeros((PROGRAMS, TILE_M * TILE_N), dtype=torch.float32)
        self.locks = self.shmem.zeros((PROGRAMS,), dtype=torch.int32)
        # the requests: two buffers in turn, a table, and a ring with all pages free
        n = len(args.prompts)
        self.lengths = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2)]
        self.table = torch.zeros((n, args.pages), dtype=torch.int32, device="cuda")
        self.pool = torch.arange(args.pages, dtype=torch.int32, device="cuda")
        self.pool_state = [torch.tensor([0, args.pages], device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")]
        self.starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(self, x, new_tokens, single):
        """One step of all ranks: x [tokens, hidden] -> y; ``single``: one token a request."""
        args, tokens, d = self.args, x.shape[0], self.args.head_dim
        positions = torch.empty(tokens, dtype=torch.int32, device="cuda")
        slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
        attention.build_block_tables(self.lengths[0], new_tokens, self.table, self.pool, self.pool_state[0], args.page_size,
                                     lengths=self.lengths[1], pool_state_out=self.pool_state[1], query_starts=self.starts,
                                     positions=positions, slots=slots, status=self.status)
        self.lengths.reverse()
        self.pool_state.reverse()
        if tokens == 0:
            return x
        for phase in (ops.PHASE_PRODUCE, ops.PHASE_CONSUME):
            all_reduce.phase = phase
            for r in range(args.ranks):
                heads = self.heads(r, x, positions, slots, single) if phase == ops.PHASE_PRODUCE else self.no_heads
                partial, result = (self.shmem.on_rank(t, r)[:tokens] for t in (self.partial, self.result))
                all_reduce.apply(heads, self.w_o[r].T, partial, result, None, self.P, self.locks, self.shmem.on_rank(self.flags, r), r,
                                 args.ranks, PROGRAMS, TILE_M, TILE_N, 64, 6, "True", 2, 8, 0, 16, 2, self.shmem.get_heap_bases(),
                                 self.shmem.get_cu_count())
                self.no_heads = heads  # (the reduce takes shapes from its operands, and nothing else)
        return self.shmem.on_rank(self.result, args.ranks - 1)[:tokens]

    def heads(self, r, x, positions, slots, single):
        """Rank r's heads: [tokens, query heads * head size]."""
        args, tokens, d = self.args, x.shape[0], self.args.head_dim
        qkv = torch.empty((tokens, self.w_qkv[r].shape[0]), dtype=self.dtype, device="cuda")
        ops.gemm_launch(x, self.w_qkv[r].T, None, qkv, None, None, 0, 1, PROGRAMS, TILE_M, TILE_N, 64, 4, ops.EPI_ALL_SCATTER, notify=False,
                        num_xcds=8)
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((self.hq * d, self.hk * d, self.hk * d), 1))
        k_cache, v_cache = self.caches[r]
        attention.qk_norm_rope(q, k, positions, self.cos, self.sin, q, None, q_weight=self.q_weight, k_weight=self.k_weight, eps=EPS, v=v,
                               k_cache=k_cache, v_cache=v_cache, slots=slots, status=self.status)
        out = torch.empty((tokens, self.hq, d), dtype=self.dtype, device="cuda")
        options = dict(window=args.window, sinks=args.sinks, workspace=self.workspace, status=self.status)
        if single:
            attention.decode_attention(q, k_cache, v_cache, self.table, self.lengths[0], out, **options)
        else:
            attention.prompt_attention(q, k_cache, v_cache, self.table, self.lengths[0], self.starts, out, **options)
        return out.flatten(1)


def dense(layer, x):
    """The layer on one request's whole sequence x [tokens, hidden], in 64 bits on the CPU."""
    args, d, n = layer.args, layer.args.head_dim, len(x)
    cos, sin = layer.cos[:n, None].double().cpu(), layer.sin[:n, None].double().cpu()
    at = torch.arange(n)
    seen = at[None, :] <= at[:, None]
    if args.window:
        seen &= (at[:, None] - at[None, :] < args.window) | (at[None, :] < args.sinks)
    y = torch.zeros((n, args.hidden), dtype=torch.float64)

    def normed(t, weight):
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * weight.double().cpu()
        a, b = t.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    for r in range(args.ranks):
        qkv = x @ layer.w_qkv[r].double().cpu().T
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((layer.hq * d, layer.hk * d, layer.hk * d), 1))
        q, k = normed(q, layer.q_weight), normed(k, layer.k_weight)
        heads = []
        for h in range(layer.hq):
            g = h // (layer.hq // layer.hk)
            s = (q[:, h] @ k[:, g].T / math.sqrt(d)).masked_fill(~seen, -math.inf)
            heads.append(torch.softmax(s, -1) @ v[:, g])
        y += torch.cat(heads, -1) @ layer.w_o[r].double().cpu().T
    return y


def main(argv=None):
    args = parse_args(argv)
    if args.heads % args.ranks or args.key_heads % args.ranks or args.heads % args.key_heads:
        sys.exit("heads and key_heads must divide over the ranks, and heads over key_heads")
    layer, n = Layer(args), len(args.prompts)
    g = torch.Generator().manual_seed(7)
    history = [torch.zeros((0, args.hidden), dtype=torch.float64) for _ in range(n)]
    worst = 0.0
    for step in range(args.steps + 1):
        single = step > 0
        new = [1] * n if single else args.prompts
        x = torch.randn((sum(new), args.hidden), generator=g).to(layer.dtype)
        y = layer.step(x.cuda(), torch.tensor(new, dtype=torch.int32, device="cuda"), single).double().cpu()
        if layer.status.item():
            sys.exit(f"status {layer.status.item()}: out of pages, or an index that is none")
        for i, (rows, out) in enumerate(zip(x.double().split(new), y.split(new))):
            history[i] = torch.cat((history[i], rows))
            if args.validate:
                want = dense(layer, history[i])[-new[i]:]
                worst = max(worst, ((out - want).norm() / want.norm()).item())
        free = (layer.pool_state[0][1] - layer.pool_state[0][0]).item()
        print(f"step {step}: {sum(new)} tokens, contexts {layer.lengths[0].tolist()}, {free} pages free", flush=True)
    layer.step(x[:0].cuda(), torch.full((n,), -1, dtype=torch.int32, device="cuda"), True)
    free = (layer.pool_state[0][1] - layer.pool_state[0][0]).item()
    print(f"requests ended: {free} of {args.pages} pages free", flush=True)
    if args.validate:
        # roundings to 16 bits on the way: projections, heads, weights, outputs, a few half places each
        bound = 8 * (2.0 ** -8 if layer.dtype == torch.bfloat16 else 2.0 ** -11)
        ok = worst <= bound and free == args.pages
        print(f"largest error of a step {worst:.2e} of its norm: {'passed' if ok else 'FAILED'}", flush=True)
        return 0 if ok else 1
    return 0


if __name__ == "__main__":
    sys.exit(main())
