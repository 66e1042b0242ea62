"""What a query does not see, or hardly weighs, leaves its output alone: sizes of other tokens' keys and values in the same block, in other blocks and in the same
tile of query rows.

The tolerances are those of test_cache_4bit_gpu.py, made of what the row itself sees."""
from __future__ import annotations

import math

import pytest
import torch

from test_cache_4bit_gpu import Step, queries

pytestmark = pytest.mark.gpu

DEV = "cuda"


# ----------------------------------------------------------------------------------------------- prompts over copies
def copies(step, window=0):
    """The step's blocks as float16 numbers with scales and marks, and the table that names them."""
    from thintensor_b200.kernels import api

    places = len(step.new) * step.table.shape[1]
    keys = torch.full((places, step.kv, 64, step.dim), math.nan, dtype=torch.float16, device=DEV)
    values, named = torch.full((places, step.kv, step.dim, 64), math.nan, dtype=torch.float16, device=DEV), torch.full_like(step.table, 5)
    scales, marks = torch.full((2, places, step.kv), 1.0, device=DEV), torch.full((places, step.kv, 64), 255, dtype=torch.uint8, device=DEV)
    api.expand_4bit(step.k_pool, step.v_pool, window=window, keys=keys, values=values, table_tmp=named, scales=scales, marks=marks, **step.common())
    return keys, values, scales, marks, named


def run_prompt(step, q, heads, window=0):
    from thintensor_b200.kernels import api

    keys, values, scales, marks, named = copies(step, window)
    out = torch.full_like(q, 7.0)
    api.attention_half(q, keys, values, scales, marks, n_tokens=q.shape[0], heads=heads, kv_heads=step.kv, head_dim=step.dim, scale=step.dim ** -0.5, window=window,
                       out=out, **(step.common() | dict(table=named)))
    return out


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_prompts_give_the_same_bits_every_time(dim):
    """More tiles than the GPU holds at once, two of them on an SM, whose warps store weights over each other's scores."""
    step = Step([700, 3], [1500, 400], 8, dim)
    q = queries(step, 32)
    first = run_prompt(step, q, 32)
    for _ in range(20):
        assert torch.equal(run_prompt(step, q, 32), first)
    assert int(step.status.item()) == 0
