"""Packed prompts: a batch of requests of different lengths, back to back in one set of rows.

``batch_tables`` turns request lengths into block tables and row maps on the GPU,
``rope_append`` rotates the packed q / k rows and scatters k / v into the paged cache by those
maps, ``prompt_attention`` attends whole packed prompts causally, and ``prompt_linear`` is the
projection of any number of rows with bias, activation and residual in its epilogue.
``Decoder.prefill_packed`` runs a model on them.  The four calls do not synchronise with the
device; ``prompt_status`` and ``append_status`` do.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib
from ._lib import PagedKV, call
from .tensor_ops import dtype_code

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "swiglu": 4}


_fns: dict = {}


def _call(device: torch.device, name: str, *args) -> None:
    """The C call on the current stream of ``device``, with that device current.  (A packed
    layer makes several calls a layer and token: what wraps them is kept to microseconds.)"""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.load(), name)
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _on(device: torch.device, *ts) -> None:
    """Every given tensor lives on ``device``, a CUDA device: a host or foreign-device pointer
    must never reach a kernel."""
    if device.type != "cuda":
        raise _lib.InvalidArgument(f"tensors must live on a CUDA device, got one on {device}")
    index = device.index
    for t in ts:
        if t is not None and t.get_device() != index:  # (-1 on the host)
            raise _lib.InvalidArgument(f"tensors must live on {device}, got one on {t.device}")


def prompt_status() -> int:
    """Reads and clears the wait status of ``prompt_attention`` and ``prompt_linear`` on the
    current device (synchronises): 0, or the TMLLM_TIMEOUT code."""
    st = C.c_int32()
    call("tmllm_prompt_status", C.byref(st))
    return st.value


def append_status() -> int:
    """Reads and clears the status of ``rope_append`` on the current device (synchronises): 0, or
    ``PositionOutOfRange.status`` when a row with a position past the rotation tables was appended,
    unrotated, since the last read."""
    st = C.c_int32()
    call("tmllm_append_status", C.byref(st))
    return st.value


class BatchTables(NamedTuple):
    """Row maps of a packed batch (``batch_tables``), all on the device."""

    q_start: torch.Tensor    # int32 [num_seqs + 1]: first row of each request
    positions: torch.Tensor  # int32 [rows]: position in its sequence, -1 for padding
    row_seq: torch.Tensor    # int32 [rows]: its request, -1 for padding
    slots: torch.Tensor      # int64 [rows]: block * block_size + offset, -1 without a block
    info: torch.Tensor       # int32 [4]: next free-list index, rows, refused, rows dropped

    @classmethod
    def empty(cls, num_seqs: int, rows: int, device=None) -> "BatchTables":
        """Buffers for ``batch_tables(..., out=)``."""
        i32 = dict(dtype=torch.int32, device=device or "cuda")
        return cls(torch.empty(num_seqs + 1, **i32), torch.empty(rows, **i32),
                   torch.empty(rows, **i32),
                   torch.empty(rows, dtype=torch.int64, device=device or "cuda"),
                   torch.empty(4, **i32))


def _int32(t: torch.Tensor, numel: int | None, what: str) -> None:
    if t.dtype != torch.int32:
        raise _lib.UnsupportedDType(f"{what} must be int32, got {t.dtype}")
    if not t.is_contiguous():
        raise _lib.NonContiguousTensor(f"{what} must be contiguous")
    if numel is not None and t.numel() != numel:
        raise _lib.InvalidShape(f"{what} must have {numel} entries, got {t.numel()}")


def _stride(t: torch.Tensor, rows: int, heads: int, d: int, what: str) -> int:
    """Row stride of a [rows, heads, D] tensor with packed heads (a view into a wider fused
    projection is fine); 0 (packed) for one row, whose stride means nothing."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != heads or shape[2] != d:
        raise _lib.ModelFormat(f"{what} must be [rows, {heads}, {d}], got {list(shape)}")
    if shape[0] != rows:
        raise _lib.ShapeMismatch(f"{what} must have {rows} rows", left=shape, right=[rows, heads, d])
    if stride[2] != 1 and d > 1 or stride[1] != d and heads > 1:
        raise _lib.NonContiguousTensor(f"{what} heads must be packed rows of {d} elements")
    if rows <= 1:
        return 0
    if stride[0] < heads * d:  # rows over one another (an expanded tensor)
        raise _lib.NonContiguousTensor(f"{what} rows overlap: stride {stride[0]}")
    return stride[0]


def _wide(what: str):
    """The refusal of sizes that the C call takes in 32 bits: ctypes would take the low bits of
    larger ones.  (The callers test several sizes at once, or-ed together.)"""
    return _lib.InvalidShape(f"{what} must fit 31 bits")


def batch_tables(kv: PagedKV, new_lens: torch.Tensor, rows: int, *,
                 free_blocks: torch.Tensor | None = None,
                 free_start: torch.Tensor | None = None,
                 out: BatchTables | None = None) -> BatchTables:
    """Block tables and slot maps from request lengths (``tmllm_batch_tables``): request s
    brings ``new_lens[s]`` tokens behind its ``seq_lens[s]`` cached ones.

    ``free_blocks`` int32: ids handed out in request order, beginning at ``free_start``
    (int32 [1], default 0), and written into ``kv``'s block table; None when every block is
    already there (a ``PagedKvCache`` view after ``reserve``: a cache hands out its own blocks, and
    a list for its table is refused).  ``rows`` is the capacity of
    the row maps; the rest of them is -1.  Requests that do not fit are refused (their rows
    get -1, ``info[2]`` counts them)."""
    dev = new_lens.device
    _on(dev, new_lens, free_blocks, free_start, *(out or ()))
    n = kv.num_seqs
    _int32(new_lens, n, "new_lens")
    if free_blocks is not None:
        _int32(free_blocks, None, "free_blocks")
        num_free = free_blocks.numel()
        if num_free >> 31:
            raise _wide("the number of free blocks")
    if free_start is not None:
        if free_blocks is None:
            raise _lib.InvalidArgument("free_start needs free_blocks")
        _int32(free_start, 1, "free_start")
    if rows < 0:
        raise _lib.InvalidShape(f"rows must not be negative, got {rows}")
    if out is None:
        out = BatchTables.empty(n, rows, dev)
    else:
        _int32(out.q_start, n + 1, "q_start")
        _int32(out.positions, rows, "positions")
        _int32(out.row_seq, rows, "row_seq")
        _int32(out.info, 4, "info")
        if out.slots.dtype != torch.int64 or out.slots.numel() != rows or not \
                out.slots.is_contiguous():
            raise _lib.InvalidArgument("slots must be a contiguous int64 tensor of rows entries")
    # an empty free list is not "no list": any non-null pointer stands for it (never read)
    _call(dev, "tmllm_batch_tables", C.byref(kv), new_lens.data_ptr(),
          (free_blocks.data_ptr() or new_lens.data_ptr()) if free_blocks is not None else None,
          num_free if free_blocks is not None else 0,
          free_start.data_ptr() if free_start is not None else None, rows,
          out.q_start.data_ptr(), out.positions.data_ptr(), out.row_seq.data_ptr(),
          out.slots.data_ptr(), out.info.data_ptr())
    return out


def rope_append(kv: PagedKV, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                positions: torch.Tensor, slots: torch.Tensor, *, rope=None,
                q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """RoPE of packed rows and their scatter into the paged cache (``tmllm_rope_append``).

    q [rows, Hq, D], k, v [rows, Hkv, D] in the cache dtype (views into a fused projection are
    read in place); ``positions`` int32 [rows] and ``slots`` int64 [rows] from
    ``batch_tables``; ``rope`` the (cos, sin) F32 tables, or None for no rotation (a row whose
    position is past the tables is not rotated, and ``append_status`` tells).  Rotated
    queries go to ``q_out`` (default: a new tensor, zeros in padding rows; ``q`` itself for in
    place), rotated keys and values to the cache, and the keys to ``k_out`` too when given.
    Returns (q_out, k_out)."""
    dev = q.device
    cos, sin = rope if rope is not None else (None, None)
    _on(dev, q, k, v, positions, slots, cos, sin, q_out, k_out)
    if q.dim() != 3:
        raise _lib.ModelFormat(f"q must be [rows, Hq, D], got {list(q.shape)}")
    rows, hq, d = q.shape
    hkv = kv.num_kv_heads
    if hq >> 31:
        raise _wide("the number of heads")
    if d != kv.head_dim:
        raise _lib.ModelFormat(f"the cache holds heads of {kv.head_dim}, got {d}")
    dtype = q.dtype
    if dtype_code(dtype) != kv.dtype or k.dtype != dtype or v.dtype != dtype or (
            q_out is not None and q_out.dtype != dtype) or (
            k_out is not None and k_out.dtype != dtype):
        raise _lib.UnsupportedDType("q, k, v and the cache must have one dtype")
    qs, ks = _stride(q, rows, hq, d, "q"), _stride(k, rows, hkv, d, "k")
    if _stride(v, rows, hkv, d, "v") != ks:
        raise _lib.NonContiguousTensor("k and v must have the same row stride")
    _int32(positions, rows, "positions")
    if slots.dtype != torch.int64 or slots.numel() != rows or not slots.is_contiguous():
        raise _lib.InvalidArgument("slots must be a contiguous int64 tensor of rows entries")
    if q_out is None:
        q_out = torch.zeros((rows, hq, d), dtype=dtype, device=dev)
    qos = _stride(q_out, rows, hq, d, "q_out")
    kos = _stride(k_out, rows, hkv, d, "k_out") if k_out is not None else 0
    if rope is not None:
        if cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise _lib.UnsupportedDType("RoPE requires F32 cos/sin tables")
        shape = cos.shape
        if len(shape) != 2 or shape != sin.shape or shape[1] * 2 != d or not (
                cos.is_contiguous() and sin.is_contiguous()):
            raise _lib.InvalidShape("RoPE cos/sin tables must be contiguous [positions, D/2]")
        rope_len = shape[0]
        if rope_len >> 31:
            raise _wide("the rows of the RoPE tables")
    if rows == 0:
        return q_out, k_out
    _call(dev, "tmllm_rope_append", C.byref(kv), q.data_ptr(), k.data_ptr(), v.data_ptr(), rows,
          hq, qs, ks, positions.data_ptr(), slots.data_ptr(),
          cos.data_ptr() if cos is not None else None, sin.data_ptr() if sin is not None else None,
          rope_len if cos is not None else 0, q_out.data_ptr(),
          qos, k_out.data_ptr() if k_out is not None else None, kos)
    return q_out, k_out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_start: torch.Tensor,
                     max_rows: int, *, scale: float = 0.0, out: torch.Tensor | None = None,
                     out_dtype: torch.dtype | None = None, lse: torch.Tensor | None = None,
                     want_lse: bool = False):
    """Causal attention over whole packed prompts (``tmllm_prompt_attention``).

    q [rows, Hq, D], k, v [rows, Hkv, D] (row-strided views allowed, k and v with one row
    stride); ``q_start`` int32
    [num_seqs + 1] first rows on the device; ``max_rows`` the longest sequence or about that (it
    sizes the launch; results do not depend on it, but 0 does nothing).  Row i of a sequence
    attends its rows 0 .. i.  Returns out [rows, Hq, D] in ``out_dtype`` (q's, or
    F32), and lse [rows, Hq] F32 with ``want_lse`` or ``lse``; rows of no sequence are left as
    they are (zeros in new tensors)."""
    dev = q.device
    _on(dev, q, k, v, q_start, out, lse)
    if q.dim() != 3 or k.dim() != 3:
        raise _lib.ModelFormat(f"q, k and v must be [rows, heads, D], got {list(q.shape)} and "
                               f"{list(k.shape)}")
    rows, hq, d = q.shape
    hkv = k.shape[1]
    dt = dtype_code(q.dtype)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise _lib.UnsupportedDType(f"prompt attention dtype mismatch: {q.dtype}, {k.dtype}, "
                                    f"{v.dtype}")
    qs, ks = _stride(q, rows, hq, d, "q"), _stride(k, rows, hkv, d, "k")
    if _stride(v, rows, hkv, d, "v") != ks:
        raise _lib.NonContiguousTensor("k and v must have the same row stride")
    _int32(q_start, None, "q_start")
    if q_start.numel() < 2:
        raise _lib.InvalidShape("q_start must have num_seqs + 1 entries")
    if (q_start.numel() | hq | hkv | d | rows) >> 31:
        raise _wide("the numbers of sequences, heads and rows")
    if max_rows < 0:
        raise _lib.InvalidShape(f"max_rows must not be negative, got {max_rows}")
    if out is None:
        out = torch.zeros((rows, hq, d), dtype=out_dtype or q.dtype, device=dev)
    if out.dtype not in (q.dtype, torch.float32) or out.shape != q.shape or not (
            out.is_contiguous()):
        raise _lib.InvalidArgument("out must be a contiguous [rows, Hq, D] tensor in q's dtype or "
                                   "F32")
    if lse is None and want_lse:
        lse = torch.zeros((rows, hq), dtype=torch.float32, device=dev)
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (rows, hq)
                            or not lse.is_contiguous()):
        raise _lib.InvalidArgument("lse must be a contiguous F32 [rows, Hq] tensor")
    _call(dev, "tmllm_prompt_attention", dt, q.data_ptr(), qs, k.data_ptr(), v.data_ptr(), ks,
          q_start.data_ptr(), q_start.numel() - 1, rows, min(max_rows, rows), hq, hkv, d, scale,
          out.data_ptr(), int(out.dtype == torch.float32),
          lse.data_ptr() if lse is not None else None)
    return (out, lse) if lse is not None else out


def prompt_linear(x: torch.Tensor, w: torch.Tensor, *, bias: torch.Tensor | None = None,
                  activation: str = "none", residual: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """out = residual + act(x · w + bias) for F16 x [rows, k], w [k, n] and any number of rows
    (``tmllm_prompt_linear``), rounded once.  ``activation``: "none", "relu", "silu", "gelu" or
    "swiglu" (w = [gate | up] [k, 2n]: silu(gate) * up).  ``residual`` [rows, n] may be ``out``.
    k and n must be multiples of 8, and so must row strides."""
    dev = x.device
    _on(dev, x, w, bias, residual, out)
    if x.dim() != 2 or w.dim() != 2:
        raise _lib.ModelFormat(f"Linear expects rank-2 input, got {tuple(x.shape)}")
    try:
        act = ACTIVATIONS[activation]
    except KeyError:
        raise _lib.InvalidArgument(f"unknown activation {activation!r}") from None
    rows, k = x.shape
    if w.shape[0] != k:
        raise _lib.ModelFormat(f"Linear input feature mismatch: expected {w.shape[0]}, got {k}")
    wide = w.shape[1]
    if act == 4 and wide % 2:
        raise _lib.InvalidShape(f"swiglu needs gate and up columns, got {wide}")
    n = wide // 2 if act == 4 else wide
    if (rows | k | wide) >> 31:
        raise _wide("rows and columns")
    if x.dtype != torch.float16:
        raise _lib.UnsupportedDType(f"prompt_linear takes F16 tensors, got {x.dtype}")
    for t, what in ((w, "w"), (bias, "bias"), (residual, "residual"), (out, "out")):
        if t is None:
            continue
        if t.dtype != torch.float16:
            raise _lib.UnsupportedDType(f"prompt_linear takes F16 tensors, got {what} {t.dtype}")
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise _lib.NonContiguousTensor(f"{what} needs unit column stride")
    if x.stride(1) != 1 and k > 1:
        raise _lib.NonContiguousTensor("x needs unit column stride")
    if bias is not None and tuple(bias.shape) != (wide,):
        raise _lib.ShapeMismatch("bias must have one entry per column of w", left=bias.shape,
                                 right=[wide])
    for t, what in ((residual, "residual"), (out, "out")):
        if t is not None and tuple(t.shape) != (rows, n):
            raise _lib.ShapeMismatch(f"{what} must be [rows, n]", left=t.shape, right=[rows, n])
    if out is None:
        out = torch.empty((rows, n), dtype=x.dtype, device=dev)
    if rows == 0:
        return out
    one = rows == 1  # the row stride of a single row means nothing
    _call(dev, "tmllm_prompt_linear", x.data_ptr(), k if one else x.stride(0), w.data_ptr(),
          w.stride(0), bias.data_ptr() if bias is not None else None, act,
          residual.data_ptr() if residual is not None else None,
          0 if residual is None else n if one else residual.stride(0), out.data_ptr(),
          n if one else out.stride(0), rows, k, n)
    return out


def prompt_linear_form(rows: int, k: int, n: int, activation: str = "none", *,
                       sms: int = 0) -> tuple[int, int, int]:
    """Which kernel ``prompt_linear`` takes (``tmllm_prompt_linear_form``): accumulator columns of a
    tile, CTAs that share a tile, CTAs that share its K; on a GPU of ``sms`` multiprocessors (0: the
    current device's)."""
    if activation not in ACTIVATIONS:
        raise _lib.InvalidArgument(f"unknown activation {activation!r}")
    form = (C.c_int32 * 3)()
    call("tmllm_prompt_linear_form", rows, k, n, ACTIVATIONS[activation], sms, form)
    return tuple(form)
