"""Attention over a paged cache at the edges of what a caller may hand in."""

import pytest
import torch

from attention_reference import BF16, F16, F32
from iris_amd import attention
from test_paged_attention_gpu import Problem

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
