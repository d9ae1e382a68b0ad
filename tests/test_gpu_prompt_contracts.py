"""What the packed-prompt calls promise beside their formulas: every stream's waits in the status,
lengths past the launch bound, rows that see nothing, tables that a cache manages, positions past
the rotation tables, and every form of the projection over many tiles a CTA."""
from __future__ import annotations

import math

import pytest
import torch

import rustllm_b200 as rb
from test_gpu_prompt import attention_case, gen, linear_case, randn

pytestmark = pytest.mark.gpu


# ---- prompt_linear: several tiles a CTA -------------------------------------------------
# Five tiles and more for every CTA (or pair), so that both accumulators, the ring of K steps and the
# staging buffers are used again; ragged rows and columns.
@pytest.mark.parametrize("rows,n,act", [
    (95001, 56, "gelu"), (95001, 104, "silu"), (60001, 264, "none"), (1080, 25000, "relu"),
    (385, 50000, "none"), (40003, 584, "gelu"),
    (95001, 56, "swiglu"), (1080, 12176, "swiglu"), (60001, 136, "swiglu")])
def test_prompt_linear_many_tiles_a_cta(cuda, rows, n, act):
    linear_case(cuda, rows, 200, n, act, bias=True, residual=True, seed=rows)
    linear_case(cuda, rows, 200, n, act, bias=True, seed=rows + 1, xpad=8)
    linear_case(cuda, rows, 72, n, act, residual=True, inplace=True, seed=rows + 2)


# ---- the status of the bounded waits ----------------------------------------------------
@pytest.mark.parametrize("name", ["prompt_status", "prefill_status", "linear_status"])
def test_status_waits_for_work_on_every_stream(cuda, name):
    """A status is that of all work launched before it, on streams that the default stream does
    not wait for, too."""
    from rustllm_b200.decoder import linear_status
    status = dict(prompt_status=rb.prompt_status, prefill_status=rb.prefill_status,
                  linear_status=linear_status)[name]
    g = gen(cuda, 1)
    q, k = randn(g, 8192, 32, 128), randn(g, 8192, 8, 128)
    starts = torch.tensor([0, 8192], dtype=torch.int32, device=cuda)
    out = torch.zeros_like(q)
    rb.prompt_attention(q, k, k, starts, 8192, out=out)
    status()  # (the first read loads its kernels, which waits)
    side, done = torch.cuda.Stream(cuda), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            rb.prompt_attention(q, k, k, starts, 8192, out=out)
        done.record()
    assert status() == 0
    assert done.query()


# ---- sizes past 32 bits -----------------------------------------------------------------
def test_prompt_linear_refuses_rows_past_32_bits(cuda):
    """2^32 rows are not 0 rows (the rows lie over one another: nothing may reach the GPU)."""
    x = torch.ones(1, 8, dtype=torch.float16, device=cuda)
    out = torch.zeros(1, 8, dtype=torch.float16, device=cuda)
    with pytest.raises(rb.InvalidShape):
        rb.prompt_linear(x.expand(2 ** 32, 8), torch.ones(8, 8, dtype=torch.float16, device=cuda),
                         out=out.expand(2 ** 32, 8))
