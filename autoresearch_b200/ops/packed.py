"""Causal attention over packed sequences of different lengths, with grouped heads (csrc/attn_packed_sm100.cu).

A packed batch is one [rows, heads, dim] tensor in which sequence i holds the rows ``cu_seqlens[i] .. cu_seqlens[i + 1]``;
a query sees the keys of its own sequence at most ``window`` positions back:

    o_i = sum_j softmax_j(scale * q_i . k_j) v_j,    i - window <= j <= i, same sequence

``PackedSequences`` holds the tile lists of one packing; every layer of a model uses the same one in both directions::

    seqs = PackedSequences(cu_seqlens, rows, n_head, n_kv_head)
    out = packed_attention(q, k, v, seqs, window=256)            # differentiable in q, k, v
"""
from __future__ import annotations

import math
import operator
import struct
from typing import Optional

import torch

from . import kernels as K

_ARGS = struct.Struct("=31qd")          # ArbPacked of csrc/api.h: 12 pointers, 7 sizes, 12 strides, the scale
MAX_ROWS = 1 << 30
MIN_SCALE = 2.0 ** -64                  # in fp32 neither it nor its reciprocal nears the ends of the range (a score that is not seen
                                        # is -inf times the scale: NaN for a scale that has become 0)
L2_SPAN_BYTES = 48 << 20                # keys and values whose tiles run together (126 MB of L2; attn_common.cuh)


def check_bounds(bounds, rows: int) -> None:
    """Raises unless ``bounds`` (host values, or a tensor on the host) ascend from at least 0 to at most ``rows``."""
    if torch.is_tensor(bounds):
        fine = 0 <= int(bounds[0]) and int(bounds[-1]) <= rows and bool((bounds[1:] >= bounds[:-1]).all())
    else:
        last = 0
        for b in bounds:
            if not last <= b <= rows:
                break
            last = b
        else:
            return
        fine = False
    if not fine:
        raise ValueError(f"sequence bounds must ascend within [0, {rows}]: got {list(bounds[:16])}")


def _to_device(bounds, device: torch.device) -> torch.Tensor:
    """A copy of host bounds (a list or a tensor) on ``device``, made in the order of its current stream and without waiting for what runs
    there: they travel through pinned memory of their own, which the allocator gives away again behind the copy only."""
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("under graph capture cu_seqlens must be a CUDA tensor: every replay would read the host's memory again")
        if torch.is_tensor(bounds):
            pinned = torch.empty(bounds.shape, dtype=torch.int32, device="cpu", pin_memory=True)
            pinned.copy_(bounds)
        else:
            pinned = torch.tensor(bounds, dtype=torch.int32, device="cpu", pin_memory=True)
        return pinned.to(device, non_blocking=True)


def document_bounds(ids: torch.Tensor, bos: int) -> torch.Tensor:
    """Bounds (int32, on the device of ``ids``) of the documents of a batch [B, T] of rows, flattened: one begins at every row and
    at every token ``bos``.  For ids on a GPU their number is read back."""
    B, T = ids.shape
    starts = ids == bos
    starts[:, 0] = True
    at = starts.reshape(-1).nonzero().reshape(-1).to(torch.int32)
    return torch.cat([at, torch.tensor([B * T], dtype=torch.int32, device=ids.device)])


class PackedSequences:
    """Which tiles the sequences of a packed batch have.

    ``cu_seqlens``: n + 1 ascending row numbers, an int32 CUDA tensor, or host values (a list, a CPU tensor), which are checked
    and copied here, without waiting for the device (under graph capture: a CUDA tensor only).  Bounds that only the device
    knows are not read back: where they descend or leave the rows they are moved inside,
    and ``kernels.check_err_flag()`` reports it.  Empty sequences are allowed.  Rows of no sequence (before the first bound
    and behind the last) get zero outputs and gradients, whatever their inputs hold.

    Made on the current stream; another stream has to wait for it, as for any tensor.  Under graph capture the lists are made
    again with every replay, from what ``cu_seqlens`` holds then."""

    def __init__(self, cu_seqlens, rows: int, n_head: int, n_kv_head: Optional[int] = None, device=None):
        n_kv_head = n_head if n_kv_head is None else n_kv_head
        if n_head <= 0 or n_kv_head <= 0 or n_head % n_kv_head or n_head // n_kv_head > 128:
            raise ValueError(f"{n_head} query heads do not form groups of at most 128 on {n_kv_head} key heads")
        if not 0 <= rows <= MAX_ROWS:
            raise ValueError(f"rows must lie in [0, {MAX_ROWS}], got {rows}")
        if not (torch.is_tensor(cu_seqlens) and cu_seqlens.is_cuda):
            if torch.is_tensor(cu_seqlens) and (cu_seqlens.dim() != 1 or cu_seqlens.dtype not in (torch.int32, torch.int64)):
                raise TypeError("cu_seqlens must be a 1-D tensor of integers")
            if not torch.is_tensor(cu_seqlens):
                cu_seqlens = [operator.index(b) for b in cu_seqlens]
            elif cu_seqlens.numel() <= 256:                    # a short list is looked through faster than three tensor operations start
                cu_seqlens = cu_seqlens.tolist()
            if not len(cu_seqlens):
                raise ValueError("cu_seqlens needs at least one bound")
            check_bounds(cu_seqlens, rows)
            device = torch.device(device if device is not None else "cuda")
            if device.type != "cuda":
                raise ValueError(f"the sequences must be packed on a CUDA device, not {device}")
            cu_seqlens = _to_device(cu_seqlens, device)
        elif cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype is not torch.int32:
            raise TypeError("cu_seqlens must be a 1-D int32 tensor of at least one element")
        self.cu_seqlens = cu_seqlens.contiguous()
        self.rows, self.n_head, self.n_kv_head = rows, n_head, n_kv_head
        self.n_seq = cu_seqlens.numel() - 1
        self.group = n_head // n_kv_head
        # bounds of the tile counts: every sequence and the rows before and behind them end in one tile that is not full
        self.cap_q = rows // (128 // self.group) + self.n_seq + 2
        self.cap_k = rows // 128 + self.n_seq + 2
        self.device = cu_seqlens.device
        self._err = K.err_flag(self.device)
        if (self.cap_q + self.cap_k) * n_kv_head >= 1 << 31:
            raise ValueError("too many tiles for one launch")
        items = 4 * (self.cap_q + self.cap_k)
        self.items = torch.empty(items + 4 * (self.n_seq + 3), dtype=torch.int32, device=self.device)
        self._err_ptr = self._err.data_ptr()
        with K.on_device(self.device):
            self._stream = K._stream()
            if rows:
                span = max(128, L2_SPAN_BYTES // (512 * min(n_kv_head, 8)))
                K._check(K.lib().arb_packed_plan(self.cu_seqlens.data_ptr(), self.n_seq, rows, self.group, span, self.items.data_ptr(),
                                                 self.cap_q, self.cap_k, self.items.data_ptr() + 4 * items,
                                                 self._err_ptr, self._stream), "packed_plan")


def _layout(t: torch.Tensor):
    """(tensor, row stride, head stride): ``t`` itself where the kernels can read it - unit inner stride, the others positive
    multiples of 8 elements, 16-byte aligned - else a dense copy.  The stride of a dimension of size 1 is never used and
    may be anything; it is given as that of dense storage."""
    s0, s1, s2 = t.stride()
    n0, n1, d = t.shape
    if n1 == 1:
        s1 = d
    if n0 == 1:
        s0 = n1 * d
    if s2 == 1 and s0 > 0 and s1 > 0 and not (s0 | s1) & 7 and not t.data_ptr() & 15:
        return t, s0, s1
    return t.clone(memory_format=torch.contiguous_format), n1 * d, d


def _forward(q, k, v, strides, seqs, window, scale, keep):
    """(O, kept).  ``strides``: row and head stride of q, k and v.  ``kept``, for the backward pass, is one buffer (each tensor that
    autograd keeps costs microseconds): where ``keep``, what O's rounding left over (a byte an element), then lse [rows, H] (fp32)."""
    rows, H, d = q.shape
    out = q.new_empty((rows, H, d))
    rest = rows * H * d if keep else 0
    kept = q.new_empty(rest + rows * H * 4, dtype=torch.int8)
    if rows:
        at = kept.data_ptr()
        _launch("arb_packed_attn_fwd", _ARGS.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), at if keep else 0, at + rest, 0, 0, 0, 0, 0,
            seqs.items.data_ptr(), rows, seqs.n_kv_head, seqs.group, d, window, seqs.cap_q, seqs.cap_k,
            *strides, H * d, 0, 0, 0, 0, 0, scale), seqs)
    return out, kept


def _launch(entry, args, seqs):
    with K.on_device(seqs.device):
        stream = K._stream()
        if stream != seqs._stream:       # the lists' memory is the other stream's: not given away before this one is done with it
            seqs.items.record_stream(torch.cuda.current_stream())
        K._check(getattr(K.lib(), entry)(args, seqs._err_ptr, stream), entry)


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


def _backward(q, k, v, strides, out, kept, d_out, grads, grad_rows, seqs, window, scale):
    """Writes ``grads`` (dq, dk, dv), whose rows are ``grad_rows`` apart and whose heads are dense.  All that the forward call read
    or wrote comes in as autograd kept it: hooks on saved tensors (checkpointing, offloading) hand back others than the call had."""
    rows, H, d = q.shape
    if not rows:
        return
    for t in (q, k, v, out, kept):
        if t.device != seqs.device:
            raise ValueError(f"a saved tensor came back on {t.device}, the sequences are on {seqs.device}")
    d_out, do_row, do_head = _layout(d_out)
    out, kept = _dense(out), _dense(kept)
    at = kept.data_ptr()
    delta = q.new_empty(rows * H + 2, dtype=torch.float32)
    _launch("arb_packed_attn_bwd", _ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), at, at + rows * H * d, d_out.data_ptr(), delta.data_ptr(),
        *[g.data_ptr() for g in grads], seqs.items.data_ptr(), rows, seqs.n_kv_head, seqs.group, d, window, seqs.cap_q, seqs.cap_k,
        *strides, H * d, do_row, do_head, *grad_rows, scale), seqs)
    K.count_launch()                     # the row sums of dO o O and the gradient grid


def _first_order_only():
    if torch.is_grad_enabled():
        raise RuntimeError("packed attention has no second derivative (create_graph=True)")


class PackedAttentionFn(torch.autograd.Function):
    """q [rows, H, d], k and v [rows, KV, d] -> [rows, H, d]."""

    @staticmethod
    def forward(ctx, q, k, v, seqs, window, scale, keep):
        (q, q0, q1), (k, k0, k1), (v, v0, v1) = _layout(q), _layout(k), _layout(v)
        out, kept = _forward(q, k, v, (q0, q1, k0, k1, v0, v1), seqs, window, scale, keep)
        if keep:
            ctx.save_for_backward(q, k, v, out, kept)
            ctx.call = (seqs, window, scale)
        return out

    @staticmethod
    def backward(ctx, d_out):
        _first_order_only()
        q, k, v, out, kept = ctx.saved_tensors
        (q, q0, q1), (k, k0, k1), (v, v0, v1) = _layout(q), _layout(k), _layout(v)
        grads = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        row, kv_row = q.shape[1] * q.shape[2], k.shape[1] * k.shape[2]
        _backward(q, k, v, (q0, q1, k0, k1, v0, v1), out, kept, d_out, grads, (row, kv_row, kv_row), *ctx.call)
        return (*grads, None, None, None, None)


class PackedQKVAttentionFn(torch.autograd.Function):
    """The same on the packed projection output [rows, (H + 2 KV) d]; its gradient is written in place of three tensors."""

    @staticmethod
    def forward(ctx, qkv, seqs, window, scale, d, keep):
        out, kept = _forward(*_blocks(qkv, seqs, d), (qkv.shape[1], d) * 3, seqs, window, scale, keep)
        out = out.view(qkv.shape[0], seqs.n_head * d)
        if keep:
            ctx.save_for_backward(qkv, out, kept)
            ctx.call = (seqs, window, scale)
        return out

    @staticmethod
    def backward(ctx, d_out):
        _first_order_only()
        qkv, out, kept = ctx.saved_tensors
        seqs = ctx.call[0]
        qkv, d = _dense(qkv), out.shape[1] // seqs.n_head
        d_qkv, ld = qkv.new_empty(qkv.shape), qkv.shape[1]
        _backward(*_blocks(qkv, seqs, d), (ld, d) * 3, out, kept, d_out.view(-1, seqs.n_head, d), _blocks(d_qkv, seqs, d), (ld,) * 3,
                  *ctx.call)
        return d_qkv, None, None, None, None, None


def _blocks(qkv, seqs, d):
    H, KV = seqs.n_head, seqs.n_kv_head
    t = qkv.view(qkv.shape[0], H + 2 * KV, d)
    return t[:, :H], t[:, H:H + KV], t[:, H + KV:]


def _common(device, rows, d, seqs, window, scale):
    if not isinstance(seqs, PackedSequences):
        raise TypeError("seqs must be a PackedSequences")
    if d not in (64, 128):
        raise ValueError(f"the kernels have head dimensions 64 and 128, not {d}")
    if seqs.rows != rows or seqs.device != device:
        raise ValueError(f"the sequences are packed in {seqs.rows} rows on {seqs.device}, the tensors have {rows} on {device}")
    if window is None:
        window = rows
    if window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    if scale is not None and not MIN_SCALE <= scale <= 1.0 / MIN_SCALE:
        raise ValueError(f"scale must be positive and lie in [{MIN_SCALE}, {1.0 / MIN_SCALE}], got {scale}")
    return min(int(window), rows), 1.0 / math.sqrt(d) if scale is None else float(scale)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seqs: PackedSequences, window: Optional[int] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """Attention of packed sequences: q [rows, H, d], k and v [rows, KV, d], bf16, d = 64 or 128, any strides -> [rows, H, d].

    Query head h reads key head h // (H / KV).  ``window``: how many positions back a query sees (None: all); ``scale``
    (positive, 2^-64 to 2^64) defaults to 1 / sqrt(d).  The inputs of a sequence reach no other sequence's outputs or gradients, not even as NaN.
    Within a sequence every row has to be finite: a weight of zero does not silence a NaN in a later key's value.  Scores are
    fp32 and have to stay below 2^30 in magnitude (their rounding, 2^-24 of the score, is a relative error of the weights)."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        K._bf16(t, name)
        if t.dim() != 3:
            raise ValueError(f"{name} must be [rows, heads, dim], got {tuple(t.shape)}")
    rows, H, d = q.shape
    window, scale = _common(q.device, rows, d, seqs, window, scale)
    if H != seqs.n_head or k.shape != (rows, seqs.n_kv_head, d) or v.shape != k.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit {seqs.n_head} heads on "
                         f"{seqs.n_kv_head} key heads")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on one device")
    keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return PackedAttentionFn.apply(q, k, v, seqs, window, scale, keep)


def packed_qkv_attention(qkv: torch.Tensor, seqs: PackedSequences, window: Optional[int] = None, scale: Optional[float] = None,
                         head_dim: int = 128) -> torch.Tensor:
    """The same on the contiguous packed projection output [rows, (H + 2 KV) head_dim] -> [rows, H head_dim]."""
    K._bf16(qkv, "qkv")
    if qkv.dim() != 2 or not qkv.is_contiguous() or qkv.data_ptr() & 15:
        raise ValueError("qkv must be 2-D, contiguous and 16-byte aligned")
    rows = qkv.shape[0]
    window, scale = _common(qkv.device, rows, head_dim, seqs, window, scale)
    if qkv.shape[1] != (seqs.n_head + 2 * seqs.n_kv_head) * head_dim:
        raise ValueError(f"qkv has {qkv.shape[1]} columns for {seqs.n_head} + 2 x {seqs.n_kv_head} heads of {head_dim}")
    return PackedQKVAttentionFn.apply(qkv, seqs, window, scale, head_dim, torch.is_grad_enabled() and qkv.requires_grad)
