"""Softmax cross entropy of a linear head without the logits, differentiable (``nk_linear_xent_fwd`` / ``_bwd``).

Stands beside :func:`~nerf_kinematics_amd.render.mse_loss`: the loss of a field that answers with one of many
labels instead of a colour.
"""
from __future__ import annotations

import torch

from . import lib as _lib
from .scan import _given, _layout, _like, _no_tangents, _once, _ptr, _unpacked, _whole


def _options(layout, ignore_index, reduction, piece) -> "_lib.NkXentOpts":
    (N, D), (V, _), (sh, _), (sw, _), dt, _ = layout
    # a dimension of one row has any stride
    return _lib.NkXentOpts(N, D, V, sh if N > 1 else D, sw if V > 1 else D, ignore_index, _lib.DTYPES[dt], reduction, piece)


def _opts(hidden, weight, *more) -> "_lib.NkXentOpts":
    return _options(_layout(hidden, weight), *more)


def _workspace(L, o, hidden, weight, backward):
    n = _lib.check(L.nk_linear_xent_workspace_bytes(o, hidden.data_ptr(), weight.data_ptr(), backward))
    return torch.empty(n, dtype=torch.uint8, device=hidden.device), n         # torch's blocks are 512-byte aligned


_FAR = 1 << 22          # bytes between rows that the library takes
_TOKENS32 = 1 << 20     # and tokens of a backward pass in float32


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with unit stride along its rows, which neither overlap nor lie further apart than the library takes (a copy where they do)."""
    return t if t.stride(1) == 1 and t.shape[1] <= t.stride(0) <= _FAR // t.element_size() and not t.is_neg() else _whole(t)


def _forward(hidden, weight, target, o, reduction):
    L = _lib.load()
    N, dev = o.N, hidden.device
    ws, n = _workspace(L, o, hidden, weight, 0)
    if reduction:       # the losses of the tokens, which nobody asked for, lie behind lse
        lse, out = torch.empty(2 * N, dtype=torch.float32, device=dev), torch.empty((), dtype=torch.float32, device=dev)
        loss, reduced = lse.data_ptr() + 4 * N, out.data_ptr()
    else:
        lse, out = torch.empty(N, dtype=torch.float32, device=dev), torch.empty(N, dtype=torch.float32, device=dev)
        loss, reduced = out.data_ptr(), None
    _lib.launch(dev, L.nk_linear_xent_fwd, o, hidden.data_ptr(), weight.data_ptr(), target.data_ptr(), loss, lse.data_ptr(), reduced,
                ws.data_ptr(), n)
    return out, lse


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction, piece):
        ctx.layout = _layout(hidden, weight)
        ctx.opts = o = _options(ctx.layout, ignore_index, reduction, piece)
        loss, lse = _forward(hidden, weight, target, o, reduction)
        ctx.save_for_backward(hidden, weight, target, lse)
        return loss

    @staticmethod
    @_once
    def backward(ctx, d_loss):
        saved = ctx.saved_tensors
        hidden, weight, layout = _unpacked(ctx, _rows, saved, d_loss)
        o = ctx.opts
        if layout is not ctx.layout:
            o = _options(layout, o.ignore_index, o.reduction, o.piece)
        target = _given(saved[2], torch.int64, o.N, hidden)
        lse = _given(saved[3], torch.float32, 2 * o.N if o.reduction else o.N, hidden)
        dev = hidden.device
        want_h, want_w = ctx.needs_input_grad[:2]
        d_hidden = _like(hidden) if want_h else None
        if hidden.shape[0] == 0:
            return d_hidden, torch.zeros_like(weight) if want_w else None, None, None, None, None
        d_weight = _like(weight) if want_w else None
        d_loss = _whole(d_loss)
        L = _lib.load()
        ws, n = _workspace(L, o, hidden, weight, 1)
        _lib.launch(dev, L.nk_linear_xent_bwd, o, hidden.data_ptr(), weight.data_ptr(), target.data_ptr(), lse.data_ptr(),
                    d_loss.data_ptr(), _ptr(d_hidden), _ptr(d_weight), ws.data_ptr(), n)
        return d_hidden, d_weight, None, None, None, None


def _call(hidden, weight, target, ignore_index, reduction, piece):
    """The operator on checked arguments."""
    hidden, weight, target = _rows(hidden), _rows(weight), target.contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(hidden, weight, target, ignore_index, reduction, piece)
    return _forward(hidden, weight, target, _opts(hidden, weight, ignore_index, reduction, piece), reduction)[0]


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", piece: int = 0) -> torch.Tensor:
    """``cross_entropy(hidden @ weight.T, target)`` as float32, without holding the logits.

    ``hidden`` [N, D] and ``weight`` [V, D] share a dtype (float32, bfloat16 or float16); ``target`` [N] is int64.
    Tokens whose target is ``ignore_index`` have loss 0 and no gradient, whatever their row of ``hidden``
    holds; any other target outside 0..V-1 makes its loss and the gradients NaN.  ``reduction`` is "mean" (over the
    tokens that are not ignored; 0 without any), "sum" or "none" ([N] losses).

    Differentiable in ``hidden`` and ``weight`` (first order, reverse mode).  The backward pass walks the vocabulary in pieces
    of ``piece`` rows (default: as many as keep a piece's scratch near 256 MB, 2048 at least) and rounds the logit gradients once to
    the operands' dtype between its products (float16: those below 2^-38 of the largest finite ``|d_loss|`` vanish); sums are
    float32.

    A call takes D up to 2^20, V up to 2^26 and N up to 2^24 (float32 with gradients: 2^20).  Rows of any layout are taken; those that
    overlap, are strided inside or lie more than 2^22 bytes apart are copied.
    """
    if reduction not in _lib.REDUCTIONS:
        raise ValueError(f"reduction={reduction!r}: expected one of {sorted(_lib.REDUCTIONS)}")
    if not isinstance(hidden, torch.Tensor) or hidden.dim() != 2 or hidden.dtype not in _lib.DTYPES or hidden.shape[1] < 1:
        raise ValueError("hidden: expected a [N, D] tensor of float32, bfloat16 or float16")
    N, D = hidden.shape
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.dtype != hidden.dtype or weight.numel() == 0 or weight.shape[1] != D:
        raise ValueError(f"weight: expected a [V, {D}] tensor of {hidden.dtype}")
    if not isinstance(target, torch.Tensor) or target.dtype != torch.int64 or target.shape != (N,):
        raise ValueError(f"target: expected an int64 tensor of shape {(N,)}")
    if piece < 0:
        raise ValueError(f"piece={piece} (>= 0)")
    _no_tangents(hidden, weight)
    if N > _TOKENS32 and hidden.dtype == torch.float32 and torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        raise ValueError(f"hidden: float32 gradients of up to {_TOKENS32} tokens a call, got {N}")
    dev = hidden.device
    if dev.type != "cuda":
        raise ValueError("hidden: expected a GPU tensor (there is no CPU implementation)")
    if weight.device != dev or target.device != dev:
        raise ValueError(f"weight, target: expected tensors on {dev}")
    return _call(hidden, weight, target, int(ignore_index), _lib.REDUCTIONS[reduction], int(piece))
