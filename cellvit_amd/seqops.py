"""Sequence operators on torch tensors: a learned position bias by buckets, the attention that reads it, the norms around a block.

For models over the token rows this package hands out: tile tokens ``[B, L, ...]`` and packed cell-token rows with prefix offsets
(``postproc.pool_cell_tokens``).  Every function runs the HIP kernels of ``libcellvit_amd.so`` on the tensors' device and its current stream; there is
no CPU fallback.  Nothing synchronises; every call can be captured into a graph, but for those that autograd records.

``rel_bias``, ``rel_attention`` and ``block_norm`` are differentiable (once, backward; forward-mode tangents are refused) through torch's autograd;
``*_train`` / ``*_grad`` are the two halves by themselves, for programs that keep their own backward pass or capture it.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple, Optional, Tuple

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib

__all__ = ["rel_buckets", "rel_bias", "rel_bias_grad", "rel_attention", "rel_attention_train", "rel_attention_grad", "block_norm", "block_norm_train",
           "block_norm_grad"]

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_F32 = torch.float32
# The C structs as packed bytes: filling a ctypes structure field by field costs more than a short kernel.
_ATTN, _NORM = struct.Struct("@10if3i17q16Pq"), struct.Struct("@6i2f6q20Pq")
assert _ATTN.size == C.sizeof(_lib.cv_rel_attn) and _NORM.size == C.sizeof(_lib.cv_block_norm)


def _pack(layout: struct.Struct, *fields) -> bytes:
    try:
        return layout.pack(*fields)
    except struct.error as e:                                # a size beyond the C struct's 32 bits
        raise ValueError(f"a size or length is out of range ({e})") from None


def _plane_sizes(q_len: int, k_len: int) -> None:
    if not (0 <= q_len <= 1 << 22 and 0 <= k_len <= 1 << 22):
        raise ValueError(f"a bias plane has 0 to 2^22 rows and columns (got {q_len}, {k_len})")


def _dtype(t: torch.dtype) -> int:
    code = _DTYPES.get(t)
    if code is None:
        raise ValueError(f"dtype must be float16, bfloat16 or float32 (got {t})")
    return code


def _same_device(first: torch.Tensor, *rest: Optional[torch.Tensor]) -> int:
    """The device index that all of them share."""
    d = first.get_device()
    if d < 0:
        raise RuntimeError("cellvit_amd runs on the MI355X only (no CPU fallback)")
    for t in rest:
        if t is not None and t.get_device() != d:
            raise ValueError(f"tensors on {first.device} and {t.device}")
    return d


def _call(device: int, fn, *args) -> None:
    """fn(*args, stream) with the device current, on its current stream."""
    stream = torch._C._cuda_getCurrentRawStream(device)      # torch.cuda.current_stream(device).cuda_stream without the objects
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _no_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """Refuses tensors that carry a forward-mode derivative: the kernels know none and would drop it."""
    if _forward_ad._current_level < 0:                       # no level is open: nothing carries one
        return
    for t in tensors:
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the sequence operators have no forward-mode derivatives")


def _differentiable(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd is to record the call.  Not inside a graph capture: torch adds a leaf's gradients on the stream where the leaf was first
    used, and a captured backward pass that meets an eager graph's addition on another stream ends the process."""
    _no_tangents(*tensors)
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)):
        return False
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("autograd inside a graph capture: capture the *_train / *_grad halves, or call under torch.no_grad()")
    return True


def _f32(t: Optional[torch.Tensor], shape: Tuple[int, ...], name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype is not _F32 or t.shape != shape:
        raise ValueError(f"{name} must be float32 {list(shape)} (got {t.dtype} {list(t.shape)})")
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


# ---------------------------------------------------------------------------------------------------------------------------------------
# bucket map and bias plane
# ---------------------------------------------------------------------------------------------------------------------------------------
def rel_buckets(num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True, device="cuda") -> torch.Tensor:
    """Bucket of every offset (key - query position) -max_distance .. max_distance, int32 [2 max_distance + 1]: half of a direction's buckets hold one
    distance each, the others are spaced by the logarithm up to ``max_distance``; offsets beyond belong to the last bucket.  Any other
    int32 tensor of odd length serves the operators as well; offsets outside it take its ends."""
    m = torch.empty(2 * max_distance + 1 if max_distance >= 0 else 0, dtype=torch.int32)
    _lib.check(_lib.load().cv_rel_buckets_host(num_buckets, max_distance, int(bidirectional), m.data_ptr()))
    return m.to(device)


def _check_map(buckets: torch.Tensor) -> int:
    if buckets.dtype != torch.int32 or buckets.dim() != 1 or buckets.numel() % 2 != 1 or not buckets.is_contiguous():
        raise ValueError("buckets must be a contiguous int32 vector of odd length (rel_buckets)")
    return buckets.numel() // 2


def _check_table(table: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    if table.dtype not in (torch.float32, dtype) or table.dim() != 2:
        raise ValueError(f"table must be [num_buckets, heads] of float32 or {dtype} (got {table.dtype} {list(table.shape)})")
    return table if table.is_contiguous() else table.contiguous()


def _rel_bias(table, buckets, q_len, k_len, dtype, out):
    span = _check_map(buckets)
    _plane_sizes(q_len, k_len)
    dtype = out.dtype if out is not None and dtype is None else dtype or table.dtype
    table = _check_table(table, dtype)
    nb, heads = table.shape
    if out is None:
        out = torch.empty((heads, q_len, k_len), dtype=dtype, device=table.device)
    elif tuple(out.shape) != (heads, q_len, k_len) or not out.is_contiguous() or out.dtype != dtype:
        raise ValueError(f"out must be contiguous [{heads}, {q_len}, {k_len}]")
    code = _dtype(out.dtype)
    _call(_same_device(table, buckets, out), _lib.load().cv_op_rel_bias, code, _dtype(table.dtype), table.data_ptr(), buckets.data_ptr(), nb, span, heads, q_len, k_len, out.data_ptr())
    return out


class _RelBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, buckets, q_len, k_len, dtype):
        ctx.save_for_backward(buckets)
        ctx.num_buckets, ctx.dtype = table.shape[0], table.dtype
        return _rel_bias(table, buckets, q_len, k_len, dtype, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dbias):
        return rel_bias_grad(dbias, ctx.saved_tensors[0], ctx.num_buckets, dtype=ctx.dtype), None, None, None, None


def rel_bias(table: torch.Tensor, buckets: torch.Tensor, q_len: int, k_len: int, *, dtype: Optional[torch.dtype] = None,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[heads, q_len, k_len]`` plane of ``table`` [num_buckets, heads]: row i stands at position i + k_len - q_len.  The plane has the table's
    dtype unless ``dtype`` or ``out`` says otherwise; the table is float32 or of the plane's dtype."""
    if _differentiable(table):
        if out is not None:
            raise ValueError("out= is not differentiable: call under torch.no_grad()")
        return _RelBias.apply(table, buckets, q_len, k_len, dtype)
    return _rel_bias(table, buckets, q_len, k_len, dtype, out)


def rel_bias_grad(dbias: torch.Tensor, buckets: torch.Tensor, num_buckets: int, *, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Gradient of the table, [num_buckets, heads] of ``dtype`` (float32 or dbias' own), from ``dbias`` [heads, q_len, k_len] or, where a batch
    shares the plane, [batch, heads, q_len, k_len]."""
    _no_tangents(dbias)
    span = _check_map(buckets)
    if dbias.dim() not in (3, 4):
        raise ValueError("dbias must be [heads, q_len, k_len] or [batch, heads, q_len, k_len]")
    code = _dtype(dbias.dtype)
    if dtype not in (torch.float32, dbias.dtype):
        raise ValueError(f"the table's gradient is float32 or {dbias.dtype} (got {dtype})")
    device = _same_device(dbias, buckets)
    dbias = dbias.contiguous()
    batch = dbias.shape[0] if dbias.dim() == 4 else 1
    heads, q_len, k_len = dbias.shape[-3:]
    _plane_sizes(q_len, k_len)
    if not 1 <= num_buckets <= 256 or batch > 0x7fffffff:
        raise ValueError(f"1 to 256 buckets and less than 2^31 planes (got {num_buckets}, {batch})")
    lib = _lib.load()
    need = lib.cv_op_rel_bias_grad_ws(num_buckets, heads, q_len, k_len)
    if need < 0:
        raise ValueError(f"bad sizes: num_buckets {num_buckets}, plane [{heads}, {q_len}, {k_len}]")
    ws = torch.empty(need, dtype=torch.uint8, device=dbias.device)
    dtable = torch.empty((num_buckets, heads), dtype=dtype, device=dbias.device)
    _call(device, lib.cv_op_rel_bias_grad, code, _dtype(dtype), dbias.data_ptr(), buckets.data_ptr(), num_buckets, span, batch, heads, q_len, k_len,
          dtable.data_ptr(), ws.data_ptr(), need)
    return dtable


# ---------------------------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------------------------
class RelAttentionSaved(NamedTuple):
    """What ``rel_attention_train`` hands to ``rel_attention_grad``."""
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    table: Optional[torch.Tensor]
    buckets: Optional[torch.Tensor]
    q_offsets: Optional[torch.Tensor]
    k_offsets: Optional[torch.Tensor]
    out: torch.Tensor
    lse: torch.Tensor
    out_lo: Optional[torch.Tensor]
    scale: float
    causal: bool
    max_q: int
    max_k: int


def _rows(t: torch.Tensor, step: int) -> Tuple[torch.Tensor, Tuple[int, int, int]]:
    """[S, L, H, D] or packed [T, H, D] with its (sequence, row, head) strides, an axis of one element counting 0: the tensor itself where the kernels can
    read it (unit stride within a head, steps of 16 bytes = `step` elements elsewhere), else a contiguous copy."""
    shape = t.shape
    if t.is_contiguous() and not t.data_ptr() & 15:
        head = shape[-1]
        row = shape[-2] * head
        return t, ((shape[1] * row, row, head) if len(shape) == 4 else (0, row, head))
    strides = t.stride()
    s = [st if n > 1 else 0 for n, st in zip(shape, strides)]
    if s[-1] != 1 or t.data_ptr() & 15 or any(x % step for x in s[:-1]):     # s[-1] is 0 in an expanded gradient (out.sum().backward())
        t = t.clone(memory_format=torch.contiguous_format)
        s = [st if n > 1 else 0 for n, st in zip(shape, t.stride())]
    return t, ((s[0], s[1], s[2]) if len(s) == 4 else (0, s[0], s[1]))


def _offsets(off: Optional[torch.Tensor], shape, most: Optional[int], name: str):
    """(offsets or None, sequences, longest length) of dense [S, L, H, D] or packed [T, H, D] rows."""
    if off is None:
        if len(shape) != 4:
            raise ValueError(f"{name} must be [sequences, length, heads, head_dim], or packed [rows, heads, head_dim] with offsets")
        if most is not None and most != shape[1]:
            raise ValueError(f"{name} has length {shape[1]}, not {most}")
        return None, shape[0], shape[1]
    if len(shape) != 3:
        raise ValueError(f"packed {name} must be [rows, heads, head_dim]")
    if off.dim() != 1 or off.numel() < 1 or off.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"offsets of {name} must be an integer vector [sequences + 1]")
    if most is None:
        raise ValueError(f"packed {name} needs the longest length (max_q / max_k)")
    if shape[0] > 0x7fffffff:
        raise NotImplementedError(f"packed {name} has more than 2^31 - 1 rows: offsets are int32")
    return off.to(torch.int32).contiguous(), off.numel() - 1, int(most)


class _Attn(NamedTuple):
    """One checked call: tensors as the kernels read them, and the fields of the C struct up to the strides of v, and of its pointers up to the map."""
    device: int
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    table: Optional[torch.Tensor]
    buckets: Optional[torch.Tensor]
    q_offsets: Optional[torch.Tensor]
    k_offsets: Optional[torch.Tensor]
    scale: float
    causal: bool
    max_q: int
    max_k: int
    n_seq: int
    head: tuple
    tail: tuple


def _attn_setup(q, k, v, table, buckets, scale, causal, q_offsets, k_offsets, max_q, max_k, zero_rest) -> _Attn:
    dt, qs, ks = q.dtype, q.shape, k.shape
    code = _dtype(dt)
    if k.dtype is not dt or v.dtype is not dt:
        raise ValueError("q, k and v must have one dtype")
    if (table is None) != (buckets is None):
        raise ValueError("table and buckets belong together")
    q_offsets, n_seq, max_q = _offsets(q_offsets, qs, max_q, "q")
    k_offsets, n_k, max_k = _offsets(k_offsets, ks, max_k, "k")
    dim = qs[-1]
    if n_seq != n_k or ks != v.shape or ks[-1] != dim:
        raise ValueError(f"q {list(qs)}, k {list(ks)} and v {list(v.shape)} do not fit together")
    heads, kv_heads = qs[-2], ks[-2]
    if kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads over {kv_heads} key heads")
    nb = span = tcode = 0
    if table is not None:
        span, table = _check_map(buckets), _check_table(table, dt)
        nb, tcode = table.shape[0], _DTYPES[table.dtype]
        if table.shape[1] != heads:
            raise ValueError(f"the table has {table.shape[1]} heads, q has {heads}")
    device = _same_device(q, k, v, table, buckets, q_offsets, k_offsets)
    step = 4 if code == _lib.DTYPE_F32 else 8
    (q, sq), (k, sk), (v, sv) = _rows(q, step), _rows(k, step), _rows(v, step)
    scale = dim ** -0.5 if scale is None else float(scale)
    head = (code, n_seq, heads, kv_heads, dim, max_q, max_k, 1 if causal else 0, nb, span, scale, tcode, zero_rest, 1, qs[0], ks[0], *sq, *sk, *sv)
    tail = (q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(q_offsets), _ptr(k_offsets), _ptr(table), _ptr(buckets))
    return _Attn(device, q, k, v, table, buckets, q_offsets, k_offsets, scale, bool(causal), max_q, max_k, n_seq, head, tail)


def _attn_call(c: _Attn, grad: int, strides: tuple, ptrs: tuple) -> None:
    """The C call, with its workspace (which lives until the call returns; the allocator orders its reuse on the stream)."""
    lib = _lib.load()
    a = _pack(_ATTN, *c.head, *strides, *c.tail, *ptrs, 0, 0)
    need = lib.cv_op_rel_attention_ws(a, grad)
    if need < 0:
        _lib.check(-need)
    if need > 0:
        ws = torch.empty(need, dtype=torch.uint8, device=c.q.device)
        a = _ATTN.pack(*c.head, *strides, *c.tail, *ptrs, ws.data_ptr(), need)
    _call(c.device, lib.cv_op_rel_attention_grad if grad else lib.cv_op_rel_attention, a)


def _attn_forward(c: _Attn, out, train):
    q = c.q
    if out is None:                                          # zero_rest: the kernels zero the rows that no sequence owns
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    so = _rows(out, 1)[1]
    lse = torch.empty(q.shape[:-1], dtype=_F32, device=q.device) if train else None
    lo = torch.empty(q.shape, dtype=_F32, device=q.device) if train and q.dtype is not _F32 else None
    _attn_call(c, 0, (*so, 0, 0, 0), (out.data_ptr(), _ptr(lse), _ptr(lo), 0, 0, 0, 0, 0))
    return out, lse, lo


class _RelAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, buckets, scale, causal, q_offsets, k_offsets, max_q, max_k):
        out, saved = rel_attention_train(q, k, v, table, buckets, scale=scale, causal=causal, q_offsets=q_offsets, k_offsets=k_offsets, max_q=max_q,
                                         max_k=max_k)
        ctx.save_for_backward(*saved[:10])
        ctx.rest = saved[10:]
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        saved = RelAttentionSaved(*ctx.saved_tensors, *ctx.rest)
        dq, dk, dv, dtable = rel_attention_grad(saved, dout, table_grad=ctx.needs_input_grad[3])
        return dq, dk, dv, dtable, None, None, None, None, None, None, None


def rel_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None, *,
                  scale: Optional[float] = None, causal: bool = False, q_offsets: Optional[torch.Tensor] = None,
                  k_offsets: Optional[torch.Tensor] = None, max_q: Optional[int] = None, max_k: Optional[int] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T + bias) v with the bucketed bias of ``rel_bias`` inside the softmax (no bias without a table, which is float32 or of
    q's dtype).

    q [S, Lq, heads, D], k and v [S, Lk, kv_heads, D] of one dtype (any strides; heads a multiple of kv_heads), or packed rows [T, heads, D] with int32
    ``q_offsets`` / ``k_offsets`` [S + 1] and the longest lengths ``max_q`` / ``max_k``.  Query i of a sequence stands at position
    i + Lk - Lq; ``causal`` hides later keys.  ``scale`` (1e-6 to 1e6) defaults to D ** -0.5.  A row that sees no key gets zeros.  Rows outside every
    sequence may hold anything, and are left as they were in ``out`` (zeros without it; it overlaps no input); keys and values inside one must be finite,
    hidden ones too.  A table entry of -inf hides its keys; finite ones act as if held to +-1.6e7 / log2(e), beyond which fp32 would lose the scores
    beside them: two mask levels below that (-1e8, -1e9) are one.  Strides: rows up to 16 MiB apart, the heads that share a key head up to 1 GiB."""
    if _differentiable(q, k, v, table):
        if out is not None:
            raise ValueError("out= is not differentiable: call under torch.no_grad()")
        return _RelAttention.apply(q, k, v, table, buckets, scale, causal, q_offsets, k_offsets, max_q, max_k)
    c = _attn_setup(q, k, v, table, buckets, scale, causal, q_offsets, k_offsets, max_q, max_k, 1 if out is None else 0)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or _rows(out, 16 // out.element_size())[0] is not out
                            or any(st == 0 and n > 1 for n, st in zip(out.shape, out.stride()))):
        raise ValueError("out must have q's shape, dtype and device, unit stride within a head, steps of 16 bytes and an element of its own for each value")
    return _attn_forward(c, out, False)[0]


def rel_attention_train(q, k, v, table=None, buckets=None, *, scale=None, causal=False, q_offsets=None, k_offsets=None, max_q=None, max_k=None
                        ) -> Tuple[torch.Tensor, RelAttentionSaved]:
    """``rel_attention`` that also returns what its backward pass reads (the inputs are kept, not copied)."""
    _no_tangents(q, k, v, table)
    c = _attn_setup(q, k, v, table, buckets, scale, causal, q_offsets, k_offsets, max_q, max_k, 1)
    out, lse, lo = _attn_forward(c, None, True)
    return out, RelAttentionSaved(*c[1:8], out, lse, lo, *c[8:12])


def rel_attention_grad(saved: RelAttentionSaved, dout: torch.Tensor, *, table_grad: bool = True
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(dq, dk, dv, dtable) of ``rel_attention``, each of its input's dtype; dtable None without a table or with ``table_grad`` false."""
    s = saved
    _no_tangents(s.q, s.k, s.v, s.table, dout)
    if dout.shape != s.out.shape or dout.dtype != s.out.dtype:
        raise ValueError(f"dout must be {s.out.dtype} {list(s.out.shape)}")
    if s.out_lo is not None and (s.out_lo.dtype is not _F32 or s.out_lo.shape != s.out.shape or not s.out_lo.is_contiguous()):
        raise ValueError("saved.out_lo must be contiguous float32 of out's shape, as rel_attention_train returns it")
    c = _attn_setup(s.q, s.k, s.v, s.table, s.buckets, s.scale, s.causal, s.q_offsets, s.k_offsets, s.max_q, s.max_k, 1)
    _same_device(s.q, dout)
    dout, sd = _rows(dout, 16 // dout.element_size())
    flat = torch.contiguous_format
    dq, dk, dv = (torch.empty_like(t, memory_format=flat) for t in (s.q, s.k, s.k))
    dtable = torch.empty_like(s.table, memory_format=flat) if s.table is not None and table_grad else None
    _attn_call(c, 1, (*_rows(s.out, 1)[1], *sd),
               (s.out.data_ptr(), s.lse.data_ptr(), _ptr(s.out_lo), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dtable)))
    return dq, dk, dv, dtable


# ---------------------------------------------------------------------------------------------------------------------------------------
# norms around a block
# ---------------------------------------------------------------------------------------------------------------------------------------
_KINDS = {"layer": 0, "rms": 1}


class BlockNormSaved(NamedTuple):
    """What ``block_norm_train`` hands to ``block_norm_grad``."""
    y: torch.Tensor
    x_out: torch.Tensor
    stats: torch.Tensor
    post: Optional[tuple]
    pre: Optional[tuple]
    gate: Optional[torch.Tensor]
    rows_per_gate: int
    alpha: float
    kind: str
    eps: float


def _pair(p, C_: int, name: str):
    if p is None:
        return None
    w, b = p if isinstance(p, (tuple, list)) else (p, None)
    return _f32(w, (C_,), name + " weight"), _f32(b, (C_,), name + " bias")


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """[rows, C] with unit stride and rows that do not overlap (an expanded gradient's do)."""
    t = t.reshape(-1, t.shape[-1])
    return t if (t.shape[1] == 1 or t.stride(1) == 1) and (t.shape[0] < 2 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _row(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else (t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _norm_setup(x, y, post, pre, gate, rows_per_gate, kind):
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'layer' or 'rms' (got {kind!r})")
    shape = y.shape
    if x.dtype is not _F32 or x.shape != shape or len(shape) < 1:
        raise ValueError(f"x must be float32 of y's shape (got {x.dtype} {list(x.shape)}, y {list(shape)})")
    width = shape[-1]
    if not 1 <= width <= 8192:
        raise NotImplementedError(f"1 to 8192 columns (got {width})")
    m = y.numel() // width
    post, pre = _pair(post, width, "post"), _pair(pre, width, "pre")
    per = m if rows_per_gate is None else int(rows_per_gate)
    if rows_per_gate is not None and per < 1:
        raise ValueError("rows_per_gate must be positive")
    per = max(min(per, m), 1)                                # more rows to a group than there are: one group
    if gate is not None:
        groups = max(1, -(-m // per))
        if gate.dtype is not _F32 or gate.numel() != groups * width or gate.shape[-1] != width:
            raise ValueError(f"gate must be float32 [{groups}, {width}] (got {gate.dtype} {list(gate.shape)})")
        gate = gate.contiguous()
    device = _same_device(y, x, gate, *(post or ()), *(pre or ()))
    return device, m, width, post, pre, gate, per


def _block_norm(x, y, post, pre, gate, rows_per_gate, alpha, kind, eps, train):
    code = _dtype(y.dtype)
    device, m, width, post, pre, gate, per = _norm_setup(x, y, post, pre, gate, rows_per_gate, kind)
    shape, dev = y.shape, y.device
    if len(shape) != 2 or x.stride() != (width, 1) or y.stride() != (width, 1):
        x, y = _rows_of(x), _rows_of(y)
    x_out = torch.empty_like(x, memory_format=torch.contiguous_format)
    z = torch.empty_like(y, memory_format=torch.contiguous_format) if pre is not None else None
    stats = torch.empty((m, 4), dtype=_F32, device=dev) if train else None
    pw, pb = post or (None, None)
    nw, nb = pre or (None, None)
    alpha, eps = float(alpha), float(eps)
    a = _pack(_NORM, code, _KINDS[kind], 0 if post is None else 1, m, width, per, alpha, eps, _row(x), _row(y), width, width, 0, 0, x.data_ptr(), y.data_ptr(),
                   _ptr(pw), _ptr(pb), _ptr(gate), _ptr(nw), _ptr(nb), x_out.data_ptr(), _ptr(z), _ptr(stats), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _call(device, _lib.load().cv_op_block_norm, a)
    saved = BlockNormSaved(y, x_out, stats, post, pre, gate, per, alpha, kind, eps) if train else None
    if len(shape) != 2:
        return x_out.view(shape), None if z is None else z.view(shape), saved
    return x_out, z, saved


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_w, post_b, pre_w, pre_b, gate, has_post, has_pre, rows_per_gate, alpha, kind, eps):
        x_out, z, s = _block_norm(x, y, (post_w, post_b) if has_post else None, (pre_w, pre_b) if has_pre else None, gate, rows_per_gate, alpha, kind, eps,
                                  True)
        ctx.save_for_backward(s.y, s.x_out, s.stats, *(s.post or (None, None)), *(s.pre or (None, None)), s.gate)
        ctx.has = has_post, has_pre
        ctx.rest = s[6:]
        ctx.shape, ctx.gate_shape = y.shape, None if gate is None else gate.shape
        ctx.set_materialize_grads(False)
        return x_out, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dx_out, dz):
        y, x_out, stats, post_w, post_b, pre_w, pre_b, gate = ctx.saved_tensors
        s = BlockNormSaved(y, x_out, stats, (post_w, post_b) if ctx.has[0] else None, (pre_w, pre_b) if ctx.has[1] else None, gate, *ctx.rest)
        g = block_norm_grad(s, dx_out, dz)
        dgate = None if gate is None else g["gate"].view(ctx.gate_shape)
        return (g["dx"].view(ctx.shape), g["dy"].view(ctx.shape), g["post_w"], g["post_b"], g["pre_w"], g["pre_b"], dgate) + (None,) * 6


def block_norm(x: torch.Tensor, y: torch.Tensor, *, post=None, pre=None, gate: Optional[torch.Tensor] = None, rows_per_gate: Optional[int] = None,
               alpha: float = 1.0, kind: str = "layer", eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(x_out, z):  x_out = alpha x + gate * N_post(y),  z = N_pre(x_out).

    x float32 [..., C] (the residual stream), y [..., C] (the block's output; z has its dtype).  ``post`` / ``pre``: (weight, bias) float32 [C] of the
    norm after the block and of the one before the next, each may be None inside; None alone: no such norm (z is then None).  ``gate``
    float32 [C], or [groups, C] with ``rows_per_gate`` rows (flattened) to a group.  ``kind``: "layer" or "rms"."""
    pw, pb = (post if isinstance(post, (tuple, list)) else (post, None))
    nw, nb = (pre if isinstance(pre, (tuple, list)) else (pre, None))
    if _differentiable(x, y, pw, pb, nw, nb, gate):
        return _BlockNorm.apply(x, y, pw, pb, nw, nb, gate, post is not None, pre is not None, rows_per_gate, alpha, kind, eps)
    return _block_norm(x, y, post, pre, gate, rows_per_gate, alpha, kind, eps, False)[:2]


def block_norm_train(x, y, *, post=None, pre=None, gate=None, rows_per_gate=None, alpha=1.0, kind="layer", eps=1e-6):
    """``block_norm`` that also returns what its backward pass reads (y is kept, not copied)."""
    _no_tangents(x, y, gate, *(post if isinstance(post, (tuple, list)) else (post,)), *(pre if isinstance(pre, (tuple, list)) else (pre,)))
    return _block_norm(x, y, post, pre, gate, rows_per_gate, alpha, kind, eps, True)


def block_norm_grad(saved: BlockNormSaved, dx_out: Optional[torch.Tensor], dz: Optional[torch.Tensor]) -> dict:
    """Gradients {dx, dy, post_w, post_b, gate, pre_w, pre_b} from those of x_out and z (either may be None); weights and gate float32, None where the
    forward had none.  dx and dy are [rows, C]."""
    s = saved
    _no_tangents(s.y, s.x_out, s.gate, *(s.post or ()), *(s.pre or ()), dx_out, dz)
    m, width = s.y.shape
    dev = s.y.device
    if dz is not None:
        if s.pre is None or dz.dtype != s.y.dtype or dz.numel() != m * width:
            raise ValueError("dz does not fit the forward's z")
        dz = _rows_of(dz)
    if dx_out is not None:
        if dx_out.dtype != torch.float32 or dx_out.numel() != m * width:
            raise ValueError("dx_out must be float32 of x_out's shape")
        dx_out = _rows_of(dx_out)
    device = _same_device(s.y, dx_out, dz)
    pw, pb = s.post or (None, None)
    nw, nb = s.pre or (None, None)
    dx = torch.empty_like(s.x_out, memory_format=torch.contiguous_format)
    dy = torch.empty_like(s.y, memory_format=torch.contiguous_format)
    grads = [None if t is None else torch.empty(width, dtype=_F32, device=dev) for t in (pw, pb, nw, nb)]
    dgate = None if s.gate is None else (torch.empty_like(s.gate) if m else torch.zeros_like(s.gate))
    args = (_dtype(s.y.dtype), _KINDS[s.kind], 0 if s.post is None else 1, m, width, s.rows_per_gate, s.alpha, s.eps, 0, _row(s.y), width, 0, _row(dx_out),
            _row(dz), 0, s.y.data_ptr(), _ptr(pw), _ptr(pb), _ptr(s.gate), _ptr(nw), _ptr(nb), s.x_out.data_ptr(), 0, s.stats.data_ptr(), _ptr(dx_out),
            _ptr(dz), dx.data_ptr(), dy.data_ptr(), _ptr(grads[0]), _ptr(grads[1]), _ptr(dgate), _ptr(grads[2]), _ptr(grads[3]))
    lib = _lib.load()
    need = lib.cv_op_block_norm_grad_ws(_pack(_NORM, *args, 0, 0))
    if need < 0:
        _lib.check(_lib.CV_ERR_INVALID)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    _call(device, lib.cv_op_block_norm_grad, _NORM.pack(*args, ws.data_ptr(), ws.numel()))
    return {"dx": dx, "dy": dy, "post_w": grads[0], "post_b": grads[1], "gate": dgate, "pre_w": grads[2], "pre_b": grads[3]}
