"""What the packed-prompt calls promise beside their formulas, as far as it shows without a GPU."""
from __future__ import annotations

import os
import re

import pytest
import torch

import rustllm_b200 as rb
from conftest import ROOT
from rustllm_b200 import _lib
from test_prompt_args import COS, K, O, POS, Q, SIN, SLOT, V, append, attention, lin, tables


def source(name: str) -> str:
    with open(os.path.join(ROOT, "rustllm_b200", "csrc", name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name,first,last", [
    ("prompt_linear.cu", "    if (warp == 0) {\n        if (lane == 0) {", "    __syncwarp();\n    if (SPLIT > 1) {"),
    ("prompt_attention.cu", "setmaxnreg.inc", "tcgen05.dealloc")])
def test_roles_of_a_cta_meet_at_no_barrier_without_a_limit(name, first, last):
    """A warp that gave up a wait leaves its loop by itself: a barrier inside the loops would keep
    the other warps for good.  They meet once, behind their loops."""
    text = source(name)
    lo, hi = text.index(first), text.index(last)
    assert lo < hi
    meets = re.findall(r"named_barrier|__syncthreads|bar\.sync|barrier\.cta|cluster_sync_all",
                       text[lo:hi])
    assert meets == (["__syncthreads"] if last == "tcgen05.dealloc" else [])


# ---- sizes past 32 bits -----------------------------------------------------------------
BIG = 2 ** 32  # 0 in its low 32 bits


@pytest.mark.parametrize("rows,k,n", [(BIG, 64, 128), (4, BIG + 64, 128), (4, 64, BIG + 128),
                                      (4, -BIG + 64, 128)])
def test_sizes_past_32_bits_are_refused_not_cut(rows, k, n):
    p = 1 << 20
    with pytest.raises(rb.InvalidShape):
        _lib.call("tmllm_prompt_linear", p, 64, 2 * p, 128, None, 0, None, 0, 3 * p, 128, rows, k, n,
                  None)


def test_older_calls_refuse_sizes_past_32_bits():
    with pytest.raises(rb.InvalidShape):
        _lib.call("tmllm_merge_lse", 16, 16, BIG, 1, 8, 8, 1, 16, 0, None, None)
    with pytest.raises(rb.InvalidShape):
        _lib.call("tmllm_cache_reserve", None, BIG, 1, None)


@pytest.mark.parametrize("make", [
    lambda: _lib.PagedKV(num_seqs=BIG + 1), lambda: _lib.PagedKV(num_blocks=BIG, block_size=BIG + 16),
    lambda: _lib.DecodeOpts(rope_len=BIG + 5), lambda: _lib.CacheConfig(max_seq_len=BIG + 64)])
def test_descriptor_fields_past_32_bits_are_refused(make):
    with pytest.raises(rb.InvalidShape):
        make()


def test_descriptors_keep_what_fits():
    kv = _lib.PagedKV(num_blocks=2 ** 40, num_seqs=2 ** 31 - 1, dtype=-1)
    assert (kv.num_blocks, kv.num_seqs, kv.dtype) == (2 ** 40, 2 ** 31 - 1, -1)
    assert _lib.DecodeOpts(max_len_hint=2 ** 40, rope_pos_offset=-3).rope_pos_offset == -3


# ---- descriptors over tensors -----------------------------------------------------------
def test_a_descriptor_keeps_its_tensors():
    """Arenas and tables that nobody else holds must not be freed under the descriptor."""
    import gc
    import weakref
    k = torch.zeros(2, 2, 4, 8, dtype=torch.float16)
    v, table, lens = k.clone(), torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    refs = [weakref.ref(t) for t in (v, table, lens)]
    kv = rb.paged_kv_from_tensors(k, v, table, lens)
    del v, table, lens
    gc.collect()
    assert all(r() is not None for r in refs) and refs[0]().data_ptr() == kv.v_cache
    del kv
    gc.collect()
    assert all(r() is None for r in refs)


# ---- what is written overlaps nothing else ----------------------------------------------
INVALID_ARGUMENT = 1
MB = 1 << 20


def refused(got: int, words: bytes) -> bool:
    return got == INVALID_ARGUMENT and words in _lib.load().tmllm_last_error()


@pytest.mark.parametrize("lse", [Q, Q + 64, K + 4, V + 128, O, O + 8 * 256 * 2 - 4, POS, O - 4])
def test_prompt_attention_lse_overlaps_nothing(lse):
    """8 rows of 4 query and 2 key heads of 64; lse has 128 bytes."""
    assert refused(attention(lse=lse), b"lse")


def test_prompt_attention_out_overlaps_no_starts():
    assert refused(attention(start=O + 16), b"q_start")
    assert refused(attention(start=O - 8), b"q_start")


def test_prompt_attention_lse_between_strided_rows_is_no_overlap():
    """Rows of q further apart (8192 bytes) than they are wide (512): lse may lie in a gap."""
    assert refused(attention(qs=4096, lse=Q + 512 - 4), b"lse")
    assert refused(attention(qs=4096, lse=Q + 8192 - 124), b"lse")  # reaches row 1
    assert refused(attention(qs=4096, lse=Q + 512, start=O), b"q_start")  # past that check


@pytest.mark.parametrize("bias,kw", [(O, {}), (O + 2, {}), (O - 254, {}), (O + 3 * 256 + 254, {}),
                                     (O + 1024, dict(ldo=512)), (O + 1024 - 2, dict(ldo=512))])
def test_prompt_linear_bias_lies_outside_out(bias, kw):
    """4 rows of 128 columns: 256 bytes a row, 1024 apart in the strided cases."""
    assert refused(lin(bias=bias, **kw), b"bias")


@pytest.mark.parametrize("kw", [
    dict(qo=20 * MB), dict(qo=20 * MB + 8 * 2 * 16 * 64 * 2 - 16), dict(qo=21 * MB - 16),
    dict(ko=21 * MB + 64), dict(qo=POS, pos=POS), dict(ko=SLOT - 16), dict(qo=COS), dict(ko=SIN),
    dict(pos=20 * MB + 4), dict(slots=21 * MB), dict(cos=20 * MB), dict(sin=21 * MB + 128)])
def test_rope_append_outputs_lie_apart(kw):
    assert append(**kw) == INVALID_ARGUMENT
    assert b"overlap" in _lib.load().tmllm_last_error()


@pytest.mark.parametrize("kw", [
    dict(new=3 * MB + 4), dict(q_start=23 * MB), dict(pos=23 * MB + 4), dict(seq=2 * MB + 12),
    dict(slots=MB), dict(info=2 * MB), dict(pos=3 * MB + 8), dict(seq=4 * MB + 28),
    dict(slots=5 * MB - 60), dict(info=6 * MB), dict(q_start=22 * MB), dict(free=22 * MB),
    dict(start=4 * MB), dict(pos=22 * MB + 28, free=None), dict(q_start=22 * MB + 16, free=None)])
def test_batch_tables_outputs_lie_apart(kw):
    assert tables(**kw) == INVALID_ARGUMENT
    assert b"overlap" in _lib.load().tmllm_last_error()


def test_batch_tables_empty_parts_overlap_nothing():
    """No rows and an empty free list have no bytes (only the null length is refused here)."""
    assert tables(rows=0, pos=3 * MB, seq=3 * MB, slots=3 * MB, free=7 * MB, num_free=0,
                  new=None) == INVALID_ARGUMENT
    assert b"null" in _lib.load().tmllm_last_error()


def test_append_status_refuses_null():
    assert _lib.load().tmllm_append_status(None) == INVALID_ARGUMENT


# ---- prompt_linear: the form each tested size takes -------------------------------------
# (rows, n, activation) of the GPU tests with five tiles and more for every CTA (or pair), whatever K,
# and their form: columns of a tile, CTAs that share one, CTAs that share its K
MANY_TILES = [
    (95001, 56, "gelu", (64, 1, 1)), (95001, 104, "silu", (128, 1, 1)),
    (60001, 264, "none", (192, 1, 1)), (1080, 25000, "relu", (256, 1, 1)),
    (385, 50000, "none", (256, 2, 1)), (40003, 584, "gelu", (256, 2, 1)),
    (95001, 56, "swiglu", (128, 1, 1)), (1080, 12176, "swiglu", (256, 1, 1)),
    (60001, 136, "swiglu", (256, 2, 1))]
# (rows, k, n, activation) of those that share K
SHARED_K = [
    (512, 1024, 1024, "none", (64, 1, 2)), (33, 4040, 1000, "silu", (64, 1, 4)),
    (33, 4096, 64, "none", (64, 1, 8)), (256, 4096, 4096, "gelu", (128, 1, 2)),
    (33, 4096, 4096, "none", (128, 1, 4)), (33, 8192, 1016, "silu", (128, 1, 8)),
    (300, 4096, 4088, "gelu", (192, 1, 2)), (500, 4104, 4096, "none", (256, 1, 2)),
    (9, 2048, 2560, "swiglu", (128, 1, 2)), (33, 4096, 2048, "swiglu", (128, 1, 4)),
    (70, 4104, 488, "swiglu", (128, 1, 8)), (300, 4096, 2040, "swiglu", (256, 1, 2))]


def test_prompt_linear_sizes_of_the_tests_reach_every_form():
    """A change of the rule must not leave a kernel without a test."""
    seen = set()
    for rows, n, act, form in MANY_TILES:
        for k in (72, 200):
            assert rb.prompt_linear_form(rows, k, n, act, sms=148) == form
        columns = form[0] // 2 if act == "swiglu" else form[0]
        tiles = -(-rows // (128 * form[1])) * -(-n // columns)
        assert tiles >= 5 * (148 // form[1])
        seen.add((act == "swiglu", *form))
    for rows, k, n, act, form in SHARED_K:
        assert rb.prompt_linear_form(rows, k, n, act, sms=148) == form
        seen.add((act == "swiglu", *form))
    assert len(seen) == 13 + 7  # all that tmllm_prompt_linear launches, plain and gated


def test_prompt_linear_form_refusals():
    with pytest.raises(rb.InvalidShape):
        rb.prompt_linear_form(0, 64, 64, sms=148)
    with pytest.raises(rb.InvalidShape):
        rb.prompt_linear_form(1, 64, 64, sms=-1)
    with pytest.raises(rb.InvalidArgument):
        rb.prompt_linear_form(1, 64, 64, "tanh")
    with pytest.raises(rb.InvalidShape):
        rb.prompt_linear_form(BIG + 1, 64, 64, sms=148)
    assert _lib.load().tmllm_prompt_linear_form(1, 64, 64, 0, 148, None) == INVALID_ARGUMENT


@pytest.mark.parametrize("scale", [3e38, 2.4e38])
def test_prompt_attention_scale_that_overflows_as_a_power_of_two(scale):
    """The kernels scale by log2(e) times as much: an infinite factor would make NaN of 0 scores."""
    assert attention(scale=scale) == 2
    assert b"scale" in _lib.load().tmllm_last_error()


@pytest.mark.parametrize("call", [
    lambda: lin(rows=1 << 28, ldo=1 << 34), lambda: lin(rows=1 << 28, ldx=1 << 34),
    lambda: lin(rows=1 << 28, res=V, ldr=1 << 34), lambda: lin(k=1 << 28, ldx=1 << 28, ldw=1 << 34),
    lambda: attention(rows=1 << 28, qs=1 << 33), lambda: append(rows=1 << 28, qs=1 << 33),
    lambda: append(rows=1 << 28, qos=1 << 33)])
def test_extents_whose_bytes_overflow_are_refused(call):
    """2^61 elements and more: their bytes do not fit the checks for overlaps."""
    assert call() == 2
    assert b"60 bits" in _lib.load().tmllm_last_error()
