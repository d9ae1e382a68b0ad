"""Refusals of the packed-prompt operators (batch_tables, rope_append, prompt_attention,
prompt_linear): every bad argument is reported on the host, before any device work.  No GPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import rustllm_b200 as rb
from rustllm_b200 import _lib

INVALID_ARGUMENT, INVALID_SHAPE, UNSUPPORTED, MODEL = 1, 2, 5, 8
P = 1 << 20  # aligned non-null dummies, far apart
Q, K, V, O, KO, POS, SLOT, COS, SIN = (P * (i + 1) for i in range(9))


def rc(name, *args):
    return getattr(_lib.load(), name)(*args)


def paged(**kw):
    base = dict(k_cache=P * 20, v_cache=P * 21, block_table=P * 22, seq_lens=P * 23, num_blocks=8,
                num_seqs=2, num_kv_heads=2, head_dim=64, block_size=16, max_blocks_per_seq=4,
                dtype=1)
    base.update(kw)
    return _lib.PagedKV(**base)


def tables(kv=None, new=P, free=P * 2, num_free=4, start=None, rows=8, q_start=P * 3, pos=P * 4,
           seq=P * 5, slots=P * 6, info=P * 7):
    return rc("tmllm_batch_tables", C.byref(kv or paged()), new, free, num_free, start, rows,
              q_start, pos, seq, slots, info, None)


@pytest.mark.parametrize("want,kw", [
    (INVALID_SHAPE, dict(kv=paged(num_seqs=0))),
    (INVALID_SHAPE, dict(kv=paged(block_size=0))),
    (INVALID_SHAPE, dict(kv=paged(max_blocks_per_seq=-1))),
    (INVALID_SHAPE, dict(kv=paged(num_blocks=0))),
    (INVALID_SHAPE, dict(kv=paged(max_blocks_per_seq=1 << 20, block_size=1 << 12))),
    (INVALID_SHAPE, dict(rows=-1)),
    (INVALID_SHAPE, dict(rows=1 << 31)),
    (INVALID_SHAPE, dict(num_free=-1)),
    (INVALID_ARGUMENT, dict(new=None)),
    (INVALID_ARGUMENT, dict(pos=None)),
    (INVALID_ARGUMENT, dict(q_start=None)),
    (INVALID_ARGUMENT, dict(info=None)),
    (INVALID_ARGUMENT, dict(kv=paged(block_table=None))),
    (INVALID_ARGUMENT, dict(kv=paged(seq_lens=None))),
    (INVALID_ARGUMENT, dict(start=P * 7 + 4)),  # inside info
])
def test_batch_tables_refusals(want, kw):
    assert tables(**kw) == want


def append(kv=None, q=Q, k=K, v=V, rows=4, hq=4, qs=0, ks=0, pos=POS, slots=SLOT, cos=COS,
           sin=SIN, rope_len=32, qo=O, qos=0, ko=KO, kos=0):
    return rc("tmllm_rope_append", C.byref(kv or paged()), q, k, v, rows, hq, qs, ks, pos, slots,
              cos, sin, rope_len, qo, qos, ko, kos, None)


@pytest.mark.parametrize("want,kw", [
    (UNSUPPORTED, dict(kv=paged(dtype=3))),
    (INVALID_SHAPE, dict(kv=paged(head_dim=63))),
    (INVALID_SHAPE, dict(kv=paged(num_kv_heads=0))),
    (MODEL, dict(hq=3)),
    (INVALID_SHAPE, dict(rows=-1)),
    (INVALID_SHAPE, dict(qs=255)),          # a row of q has 256 elements
    (INVALID_SHAPE, dict(ks=127)),
    (INVALID_SHAPE, dict(kos=100)),
    (INVALID_SHAPE, dict(qs=1 << 62)),
    (INVALID_ARGUMENT, dict(pos=None)),
    (INVALID_ARGUMENT, dict(slots=None)),
    (INVALID_ARGUMENT, dict(q=None)),
    (INVALID_ARGUMENT, dict(q=Q + 1)),
    (INVALID_ARGUMENT, dict(sin=None)),
    (INVALID_ARGUMENT, dict(rope_len=0)),
    (INVALID_ARGUMENT, dict(qo=Q + 512)),               # one row behind itself
    (INVALID_ARGUMENT, dict(qo=Q, qos=512)),            # itself, with other rows
    (INVALID_ARGUMENT, dict(ko=V)),
    (INVALID_ARGUMENT, dict(qo=K)),
    (INVALID_ARGUMENT, dict(qo=O, ko=O)),
])
def test_rope_append_refusals(want, kw):
    assert append(**kw) == want


def test_rope_append_fused_columns_do_not_overlap():
    """k behind q in one fused row is no overlap: only the null positions are refused here."""
    w = (4 + 2 + 2) * 64
    assert append(q=Q, k=Q + 512, v=Q + 768, qs=w, ks=w, qo=Q, qos=w, ko=Q + 512, kos=w,
                  pos=None) == INVALID_ARGUMENT
    assert b"null" in _lib.load().tmllm_last_error()
    assert append(q=Q, k=Q + 512, v=Q + 768, qs=w, ks=w, qo=Q, qos=w, ko=Q + 640,
                  kos=w) == INVALID_ARGUMENT  # shifted by half a key head
    assert b"overlap" in _lib.load().tmllm_last_error()


def attention(dtype=1, q=Q, qs=0, k=K, v=V, ks=0, start=POS, seqs=2, rows=8, max_rows=8, hq=4,
              hkv=2, d=64, scale=0.0, out=O, f32=0, lse=None):
    return rc("tmllm_prompt_attention", dtype, q, qs, k, v, ks, start, seqs, rows, max_rows, hq,
              hkv, d, scale, out, f32, lse, None)


@pytest.mark.parametrize("want,kw", [
    (UNSUPPORTED, dict(dtype=2)),
    (INVALID_SHAPE, dict(seqs=0)),
    (INVALID_SHAPE, dict(d=0)),
    (INVALID_SHAPE, dict(d=264)),
    (MODEL, dict(hkv=3)),
    (INVALID_SHAPE, dict(rows=-1)),
    (INVALID_SHAPE, dict(rows=1 << 31)),
    (INVALID_SHAPE, dict(max_rows=-1)),
    (INVALID_SHAPE, dict(qs=64)),
    (INVALID_SHAPE, dict(ks=64)),
    (INVALID_SHAPE, dict(scale=float("inf"))),
    (INVALID_SHAPE, dict(scale=float("nan"))),
    (INVALID_ARGUMENT, dict(f32=2)),
    (INVALID_ARGUMENT, dict(start=None)),
    (INVALID_ARGUMENT, dict(out=None)),
    (INVALID_ARGUMENT, dict(out=O + 1)),
    (INVALID_ARGUMENT, dict(lse=P + 2)),
    (INVALID_ARGUMENT, dict(out=K)),
    (INVALID_ARGUMENT, dict(out=V + 64)),
    (INVALID_ARGUMENT, dict(out=Q, f32=1)),             # in place, but wider
    (INVALID_ARGUMENT, dict(out=Q + 512)),
    (INVALID_ARGUMENT, dict(out=Q, qs=512)),
])
def test_prompt_attention_refusals(want, kw):
    assert attention(**kw) == want


def test_prompt_attention_without_rows_is_done():
    assert attention(rows=0, q=None, k=None, v=None, out=None) == 0
    assert attention(max_rows=0) == 0


def lin(x=Q, ldx=64, w=K, ldw=128, bias=None, act=0, res=None, ldr=0, out=O, ldo=128, rows=4,
        k=64, n=128):
    return rc("tmllm_prompt_linear", x, ldx, w, ldw, bias, act, res, ldr, out, ldo, rows, k, n,
              None)


@pytest.mark.parametrize("want,kw", [
    (INVALID_SHAPE, dict(rows=-1)),
    (INVALID_SHAPE, dict(k=60)),
    (INVALID_SHAPE, dict(n=0)),
    (INVALID_SHAPE, dict(n=124)),
    (INVALID_ARGUMENT, dict(act=5)),
    (INVALID_ARGUMENT, dict(act=-1)),
    (INVALID_SHAPE, dict(ldx=56)),
    (INVALID_SHAPE, dict(ldx=68)),
    (INVALID_SHAPE, dict(ldw=120)),
    (INVALID_SHAPE, dict(act=4)),                       # swiglu reads 2n columns
    (INVALID_SHAPE, dict(ldo=64)),
    (INVALID_SHAPE, dict(res=V, ldr=64)),
    (INVALID_SHAPE, dict(ldx=1 << 40)),
    (INVALID_ARGUMENT, dict(x=None)),
    (INVALID_ARGUMENT, dict(x=Q + 8)),
    (INVALID_ARGUMENT, dict(w=K + 2)),
    (INVALID_ARGUMENT, dict(out=O + 8)),
    (INVALID_ARGUMENT, dict(res=V + 8, ldr=128)),
    (INVALID_ARGUMENT, dict(bias=V + 1)),
    (INVALID_ARGUMENT, dict(out=Q)),
    (INVALID_ARGUMENT, dict(res=O + 256, ldr=128)),     # shifted by a row
    (INVALID_ARGUMENT, dict(res=O, ldr=256)),
    (INVALID_ARGUMENT, dict(out=K + 256)),              # inside W
])
def test_prompt_linear_refusals(want, kw):
    assert lin(**kw) == want


def test_prompt_linear_without_rows_is_done():
    assert lin(rows=0, x=None, out=None) == 0


def test_prompt_status_refuses_null():
    assert rc("tmllm_prompt_status", None) == INVALID_ARGUMENT


def test_host_tensors_are_refused():
    """A host pointer must never reach a kernel."""
    x = torch.zeros(4, 64, dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int32)
    h = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(rb.InvalidArgument):
        rb.prompt_linear(x, torch.zeros(64, 64, dtype=torch.float16))
    with pytest.raises(rb.InvalidArgument):
        rb.prompt_attention(h, h, h, i, 4)
    with pytest.raises(rb.InvalidArgument):
        rb.batch_tables(paged(), torch.zeros(2, dtype=torch.int32), 4)
    with pytest.raises(rb.InvalidArgument):
        rb.rope_append(paged(), h, h, h, i, i.long())
