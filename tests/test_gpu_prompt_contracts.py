"""What the packed-prompt calls promise beside their formulas: every stream's waits in the status,
lengths past the launch bound, rows that see nothing, tables that a cache manages, positions past
the rotation tables, and every form of the projection over many tiles a CTA."""
from __future__ import annotations

import math

import pytest
import torch

import rustllm_b200 as rb
from test_gpu_prompt import attention_case, gen, linear_case, randn
from test_prompt_contracts import MANY_TILES

pytestmark = pytest.mark.gpu


# ---- prompt_linear: several tiles a CTA -------------------------------------------------
# Five tiles and more for every CTA (or pair), so that both accumulators, the ring of K steps and the
# staging buffers are used again; ragged rows and columns.
@pytest.mark.parametrize("rows,n,act,form", MANY_TILES)
def test_prompt_linear_many_tiles_a_cta(cuda, rows, n, act, form):
    if torch.cuda.get_device_properties(cuda).multi_processor_count == 148:
        assert rb.prompt_linear_form(rows, 200, n, act) == form
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


# ---- prompt_attention: values that are not finite ---------------------------------------
@pytest.mark.parametrize("dtype,d,out_dtype", [
    (torch.float16, 64, None), (torch.float16, 128, None), (torch.float16, 80, torch.float32),
    (torch.float16, 20, None), (torch.float32, 64, None), (torch.float32, 200, None)])
@pytest.mark.parametrize("hq,hkv,pad", [(2, 1, 0), (3, 1, 700), (24, 8, 0)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_prompt_attention_rows_without_a_key_are_zero(cuda, dtype, d, out_dtype, hq, hkv, pad, bad):
    """Every logit -inf gives zeros and lse -inf, also over values that are not finite, in the tiles
    that a row sees whole and in the others; in a row with a finite logit such a value shows."""
    g = gen(cuda, d + hq)
    dark, lens = 200, [70, 300, 40]
    rows, a = sum(lens) + pad, lens[0]
    q, k, v = randn(g, rows, hq, d, dtype=dtype).abs(), randn(g, rows, hkv, d, dtype=dtype), \
        randn(g, rows, hkv, d, dtype=dtype)
    k[a:a + dark] = -math.inf
    v[a + 3, :, 1], v[a + 150, :, 2], v[a + 250, :, 3] = bad, bad, bad
    clean = v.clone()
    clean[[a + 3, a + 150, a + 250]] = 0
    starts = torch.tensor([0, 70, 370, 410], dtype=torch.int32, device=cuda)
    out, lse = rb.prompt_attention(q, k, v, starts, 300, out_dtype=out_dtype, want_lse=True)
    want = rb.prompt_attention(q, k, clean, starts, 300, out_dtype=out_dtype)
    torch.cuda.synchronize()
    assert rb.prompt_status() == 0
    # a query element that was drawn as 0 makes its row's logits 0 * inf = NaN, not -inf
    none = torch.zeros(rows, hq, dtype=torch.bool, device=cuda)
    none[a:a + dark] = True
    odd = (q == 0).any(-1)
    odd[:a], odd[a + 300:] = False, False
    assert int(odd.sum()) < 9
    assert bool((out[none & ~odd] == 0).all()) and bool((lse[none & ~odd] == -math.inf).all())
    assert bool(torch.isnan(out[odd]).all()) and bool(torch.isnan(lse[odd]).all())
    sees = ~none & ~odd
    assert bool(torch.isfinite(lse[:sum(lens)][sees[:sum(lens)]]).all())
    sees[:a + dark], sees[a + 300:] = False, False
    assert not bool(torch.isfinite(out[sees][:, 1:3]).any())  # weight 0, not finite
    sees[:a + 250] = False
    shows = out[sees][:, 3]
    assert bool((torch.isnan(shows) if math.isnan(bad) else shows == bad).all())
    keep = ~odd[:, :, None].expand_as(out).clone()
    keep[a + dark:a + 300, :, 1:3] = False
    keep[a + 250:a + 300] = False  # the zeroed row of `clean` carries weight there
    assert torch.equal(out[keep], want[keep])


# ---- prompt_attention: sequences longer than the launch bound ---------------------------
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.float16, 128), (torch.float16, 136),
                                     (torch.float16, 20), (torch.float32, 64), (torch.float32, 128),
                                     (torch.float32, 256)])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (48, 4)])
def test_prompt_attention_longer_than_max_rows(cuda, dtype, d, hq, hkv):
    """max_rows sizes the launch: rows past it are computed all the same (a captured call meets
    longer prompts than it was captured with)."""
    for bound in (1, 70, 130):
        attention_case(cuda, [5, 300, 0, 131, 64], hq, hkv, d, dtype, seed=d, pad=3, lead=2,
                       max_rows=bound)
    attention_case(cuda, [200, 330], hq, hkv, d, dtype, seed=d, max_rows=1, inplace=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prompt_attention_captured_for_shorter_prompts(cuda, dtype):
    g = gen(cuda, 4)
    q, k, v = (randn(g, 400, h, 64, dtype=dtype) for h in (4, 2, 2))
    starts = torch.tensor([0, 40, 400], dtype=torch.int32, device=cuda)
    want = rb.prompt_attention(q, k, v, starts, 360)
    live = torch.tensor([0, 200, 400], dtype=torch.int32, device=cuda)
    out = torch.zeros_like(q)
    rb.prompt_attention(q, k, v, live, 200, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rb.prompt_attention(q, k, v, live, 200, out=out)
    live.copy_(starts)
    out.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ---- batch_tables: the tables of a cache ------------------------------------------------
def test_batch_tables_assigns_no_blocks_of_a_cache(cuda):
    """A cache hands out its own blocks: ids written into its table behind its back would be given
    to another sequence by the next reserve."""
    cache = rb.PagedKvCache(2, 2, 64, 2, 64, num_blocks=8, device=cuda)
    other = rb.PagedKvCache(1, 1, 64, 2, 64, device=cuda)
    new = torch.tensor([20, 5], dtype=torch.int32, device=cuda)
    free = torch.arange(8, dtype=torch.int32, device=cuda)
    for layer in (0, 1):
        with pytest.raises(rb.InvalidArgument):
            rb.batch_tables(cache.view(layer), new, 25, free_blocks=free)
    with pytest.raises(rb.InvalidArgument):
        rb.batch_tables(other.view(0), new[:1], 25, free_blocks=free)
    for s, n in enumerate((20, 5)):
        cache.reserve(s, n)
    m = rb.batch_tables(cache.view(0), new, 25)  # without a list: its own blocks
    blocks = cache.block_table(0) + cache.block_table(1)
    assert len(set(blocks)) == 3 and m.info.tolist() == [0, 25, 0, 0]
    assert m.slots.tolist() == [blocks[i // 16] * 16 + i % 16 for i in range(20)] + \
        [blocks[2] * 16 + i for i in range(5)]
    # the same memory in other hands is free to be assigned again
    view = cache.view(0)
    table = torch.full((2, view.max_blocks_per_seq), -1, dtype=torch.int32, device=cuda)
    view.block_table = table.data_ptr()
    rb.batch_tables(view, new, 25, free_blocks=free)
    assert table[:, :2].tolist() == [[0, 1], [2, -1]]


# ---- rope_append: positions past the tables ---------------------------------------------
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.float32, 128), (torch.float16, 6)])
def test_rope_append_reports_positions_past_the_tables(cuda, dtype, d):
    """Such rows are not rotated, which no output shows: the status does, once."""
    g = gen(cuda, 1)
    q, k = randn(g, 40, 4, d, dtype=dtype), randn(g, 40, 2, d, dtype=dtype)
    c = torch.zeros(4, 2, 16, d, dtype=dtype, device=cuda)
    kv = rb.paged_kv_from_tensors(c, c.clone(), torch.zeros((1, 4), dtype=torch.int32, device=cuda),
                                  torch.zeros(1, dtype=torch.int32, device=cuda))
    rope = rb.rope_tables(d, 60, 10000.0, device=cuda)
    slots = torch.arange(40, device=cuda)
    pos = torch.arange(20, 60, dtype=torch.int32, device=cuda)
    rb.append_status()  # whatever ran before
    rb.rope_append(kv, q, k, k, pos, slots, rope=rope)
    pos[3] = -5  # padding
    rb.rope_append(kv, q, k, k, pos, slots, rope=rope)
    rb.rope_append(kv, q, k, k, pos + 1, slots)  # no rotation asked for
    assert rb.append_status() == 0
    side = torch.cuda.Stream(cuda)
    pos[39] = 60
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        rb.rope_append(kv, q, k, k, pos, slots, rope=rope)
    assert rb.append_status() == rb.PositionOutOfRange.status
    assert rb.append_status() == 0
    assert rb.prompt_status() == 0  # that is the status of the bounded waits


# ---- the order of sums ------------------------------------------------------------------
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.float16, 128), (torch.float16, 136),
                                     (torch.float32, 64), (torch.float32, 128)])
def test_prompt_attention_repeats_bit_for_bit(cuda, dtype, d):
    """The order of a row's sums depends on the call, not on the run, nor on what other rows hold."""
    g = gen(cuda, d)
    lens = [300, 1, 0, 700, 129, 64]
    rows, starts = sum(lens) + 6, [3]
    for n in lens:
        starts.append(starts[-1] + n)
    q, k, v = (randn(g, rows, h, d, dtype=dtype) for h in (6, 2, 2))
    st = torch.tensor(starts, dtype=torch.int32, device=cuda)
    first = [t.clone() for t in rb.prompt_attention(q, k, v, st, 700, want_lse=True)]
    q[:3], k[-3:], v[-3:] = math.nan, math.nan, math.inf
    for _ in range(5):
        again = rb.prompt_attention(q, k, v, st, 700, want_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
