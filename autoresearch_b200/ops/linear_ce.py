"""Cross entropy of a linear head over a vocabulary of any size, without its logits in memory (csrc/gemm_sm100.cu).

    s = softcap tanh(x w^T / softcap)         (softcap 0: s = x w^T)
    loss[n] = log sum_v exp s[n, v] - s[n, target[n]]

The forward product hands out the maximum and the exponential sum of every row and tile of 256 ids, which one small kernel
joins; no logit is written.  The backward pass multiplies again, a piece of the vocabulary at a time: the epilogue turns a
piece of logits into d = g[n] (softmax(s) - [v = target]) ds/dx in bf16, which the two gradient products dx += d w and
dw = d^T x read.  What is kept between the passes is one fp32 number per row.

Scratch: the forward pass takes 8 bytes per row and tile of 256 ids (N V / 32 bytes: 67 MB for 16384 x 131072, a 64th of bf16 logits); the
backward pass a piece, at most ``PIECE_BYTES`` or, where there are so many rows that a single tile takes more, 512 bytes a row, and
fp32 sums of dx where the vocabulary has several pieces or the sum has several parts (up to four).

Logits are fp32 sums of the tensor cores, which cut every partial sum (of 16 columns) to 24 bits instead of rounding it: a loss is off
by about 2e-7 of itself at 256 columns and 1.2e-6 at 2048.

Beside ``LMHeadCEFn`` (ops/sm100.py), which keeps whole rows of logits for a chunk of tokens and makes the gradients in its
forward pass, this form returns per-token losses with any later weighting, and keeps no logits.
"""
from __future__ import annotations

import functools
import struct

import torch

from . import kernels as K

_ARGS = struct.Struct("=9q9qd")         # ArbLinearCE of csrc/api.h: 9 pointers, 9 sizes, the soft cap
PIECE_BYTES = 1 << 29                   # bf16 gradient of a piece of logits; never less than one tile of every row
TILE = 256
MAX_SOFTCAP = 100.0                     # a capped logit is off by up to 2^-22 of the cap
MIN_SOFTCAP = 2.0 ** -64                # its reciprocal is a normal fp32 number, and the cap is not taken for none


def piece_columns(rows: int, vocab: int) -> int:
    """Ids per piece of the backward pass: whole tiles, pieces of about the same size."""
    most = max(TILE, PIECE_BYTES // (2 * max(rows, 1)) // TILE * TILE)
    pieces = -(-vocab // most)
    return -(-(-(-vocab // pieces)) // TILE) * TILE if pieces > 1 else vocab


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where the copy engine can read its rows, else a contiguous copy."""
    if t.stride(1) == 1 and (t.shape[0] == 1 or (t.stride(0) >= t.shape[1] and not t.stride(0) & 7)) and not t.data_ptr() & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


@functools.lru_cache(maxsize=256)
def _backward_plan(rows: int, dim: int, vocab: int):
    """(ids per piece, row stride of its gradient, fp32 slabs of dx, kernels without those of dx and dw)."""
    cols = piece_columns(rows, vocab)
    parts = K.lib().arb_linear_ce_parts(rows, dim, vocab) if cols == vocab else 1
    return cols, -(-cols // 8) * 8, parts if cols < vocab or parts > 1 else 0, -(-vocab // cols)


class LinearCEFn(torch.autograd.Function):
    """Per-row losses [N] fp32.  A weight with a ``main_grad`` takes its gradient up there, as in the other products."""

    @staticmethod
    def forward(ctx, x, w, targets, softcap, keep):
        N, D = x.shape
        V = w.shape[0]
        loss = x.new_empty(N, dtype=torch.float32)
        lse = x.new_empty(N, dtype=torch.float32)
        xr, wr = _rows(x), _rows(w)
        if N:
            with K.on_device(x.device):
                if K.pending_pulls:
                    K.flush_pending_pulls()
                tiles = -(-V // TILE)
                scratch = x.new_empty((2 * tiles + 1) * N, dtype=torch.float32)
                part = scratch.data_ptr()
                args = _ARGS.pack(xr.data_ptr(), wr.data_ptr(), targets.data_ptr(), part, part + 8 * tiles * N, lse.data_ptr(),
                                  loss.data_ptr(), 0, 0, N, V, D, V, 0, int(targets.dtype is torch.int64), _ld(xr), _ld(wr), 0, softcap)
                K._check(K.lib().arb_linear_ce_fwd(args, K.err_flag(x.device).data_ptr(), K._stream()), "linear_ce_fwd")
                K.count_launch()                                     # the product and the join
        if keep:
            ctx.save_for_backward(xr, wr, targets, lse)
            ctx.parameter = w if w.is_leaf else None                 # hooks on saved tensors hand back others, without its main gradient
            ctx.softcap = softcap
        return loss

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():
            raise RuntimeError("linear cross entropy has no second derivative (create_graph=True)")
        x, w, targets, lse = ctx.saved_tensors
        with K.on_device(g.device):
            return (*_gradients(x, w, ctx.parameter, targets, lse, g.contiguous(), ctx.softcap, *ctx.needs_input_grad[:2]), None, None, None)


def _gradients(x, w, parameter, targets, lse, g, softcap, need_x, need_w):
    """(dx, dw); dw is None where the main gradient of the parameter has taken it up.  All that the forward call read or wrote comes
    in as autograd kept it: hooks on saved tensors (checkpointing, offloading) hand back others than the call had."""
    N, D = x.shape
    V = w.shape[0]
    main = getattr(w if parameter is None else parameter, "main_grad", None) if need_w else None
    if main is not None and (main.dtype is not torch.float32 or main.shape != w.shape or main.device != w.device or main.stride(1) != 1
                             or main.stride(0) % 4 or main.data_ptr() & 15):
        raise ValueError(f"main_grad of a {tuple(w.shape)} weight must be fp32 of that shape with unit inner stride and 16-byte aligned rows")
    if not N:
        return (torch.zeros_like(x) if need_x else None), (torch.zeros_like(w) if need_w and main is None else None)
    for t in (x, w, targets, lse):
        if t.device != g.device:
            raise ValueError(f"a saved tensor came back on {t.device}, the gradient is on {g.device}")
    if K.pending_pulls:
        K.flush_pending_pulls()
    xr, wr, targets, lse = _rows(x), _rows(w), targets.contiguous(), lse.contiguous()
    cols, ldd, slabs, pieces = _backward_plan(N, D, V)
    d = x.new_empty(N * ldd)
    dx = x.new_empty((N, D)) if need_x else None
    dw = w.new_empty((V, D)) if need_w and main is None else None
    # several pieces meet in fp32, in the order of the vocabulary; a single one may be summed in parts
    acc = x.new_empty((slabs, N, D), dtype=torch.float32) if need_x and slabs else None
    args = _ARGS.pack(xr.data_ptr(), wr.data_ptr(), targets.data_ptr(), 0, 0, lse.data_ptr(), 0, g.data_ptr(), d.data_ptr(),
                      N, V, D, V, 0, int(targets.dtype is torch.int64), _ld(xr), _ld(wr), ldd, softcap)
    K._check(K.lib().arb_linear_ce_bwd(args, cols, dx.data_ptr() if need_x else 0, acc.data_ptr() if acc is not None else 0,
                                       dw.data_ptr() if dw is not None else 0, main.data_ptr() if main is not None else 0,
                                       main.stride(0) if main is not None else 0, K.err_flag(x.device).data_ptr(), K._stream()), "linear_ce_bwd")
    K.count_launch(pieces * (1 + need_x + need_w) - 1 + (acc is not None))
    return dx, dw


def linear_cross_entropy(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, softcap: float = 0.0) -> torch.Tensor:
    """Per-token losses [N] (fp32) of the head ``w`` [V, D] on ``x`` [N, D], both bf16, D a multiple of 8; differentiable in both.

    ``targets`` [N], int32 or int64: a value outside of [0, V) marks a token that does not count (loss 0, no gradient).
    ``softcap`` > 0 (2^-64 to 100): the logits are softcap * tanh(. / softcap).  Every row of ``x`` has to be finite, those that do not count
    too: the gradient of ``w`` sums over all of them."""
    K._bf16(x, "x")
    K._bf16(w, "w")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"x must be [N, D] and w [V, D], got {tuple(x.shape)} and {tuple(w.shape)}")
    N, D = x.shape
    if D < 8 or D % 8 or w.shape[0] < 1:
        raise ValueError(f"D must be a positive multiple of 8 and w not empty, got {tuple(w.shape)}")
    if targets.dtype not in (torch.int32, torch.int64) or targets.shape != (N,):
        raise ValueError(f"targets must be int32 or int64 [{N}], got {targets.dtype} {tuple(targets.shape)}")
    if w.device != x.device or targets.device != x.device:
        raise ValueError("x, w and targets must be on one device")
    if softcap != 0 and not MIN_SOFTCAP <= softcap <= MAX_SOFTCAP:
        raise ValueError(f"softcap must be 0 or lie in [{MIN_SOFTCAP}, {MAX_SOFTCAP}], got {softcap}")
    keep = torch.is_grad_enabled() and (x.requires_grad or w.requires_grad)
    return LinearCEFn.apply(x, w, targets.contiguous(), float(softcap), keep)
