"""What the packed-prompt calls promise beside their formulas, as far as it shows without a GPU."""
from __future__ import annotations

import os
import re

import pytest
import torch

import rustllm_b200 as rb
from conftest import ROOT
from rustllm_b200 import _lib


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
