"""Gated linear recurrence along a long axis, differentiable (``nk_gated_scan_fwd`` / ``_bwd``).

Stands beside :func:`~nerf_kinematics_amd.render.raw2outputs`: alpha compositing along a ray is the
recurrence with ``a = 1 - alpha``, ``x = alpha * colour``, walked from the far sample to the near one with one
gate for all channels; here the channels, the length and the gates are free.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward_ad

from . import lib as _lib


_KEEP = 32              # the forward pass of a training step keeps the state in front of every 32nd step


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` [B, T, n] with unit stride along n and no negative strides (a copy where it has neither)."""
    sb, st, sc = t.stride()
    return t if (sc == 1 or t.shape[2] == 1) and sb >= 0 and st >= 0 and not t.is_neg() else _whole(t)


def _whole(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """`t` contiguous, with its values in memory as they are (torch negates the imaginary part of a conjugate lazily)."""
    if t is None:
        return None
    t = t.contiguous()
    return t.resolve_neg() if t.is_neg() else t


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _like(t: torch.Tensor) -> torch.Tensor:
    """An empty contiguous tensor of `t`'s shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _no_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """Refuses forward-mode tangents: a call that autograd does not see would drop them, and their absence reads as zero."""
    if _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("forward-mode derivatives are not available here (first-order gradients by backward() are)")


def _layout(p: torch.Tensor, q: torch.Tensor) -> tuple:
    return p.shape, q.shape, p.stride(), q.stride(), p.dtype, q.dtype


def _unpacked(ctx, rows, saved, like: torch.Tensor) -> tuple:
    """The first two saved tensors and their layout.  Saved-tensor hooks may hand them back in another layout (copies of strided
    ones come back dense), so it is read from these and not kept from the forward pass; a hook that changes more than that is
    refused, as far as memory is concerned."""
    p, q = saved[0], saved[1]
    layout = _layout(p, q)
    if layout == ctx.layout:
        layout = ctx.layout
    else:
        if layout[:2] + layout[4:] != ctx.layout[:2] + ctx.layout[4:]:
            _refuse_hook()
        p, q = rows(p), rows(q)
        layout = _layout(p, q)
    if not p.get_device() == q.get_device() == like.get_device():
        _refuse_hook()
    return p, q, layout


def _refuse_hook() -> None:
    raise RuntimeError("a saved-tensor hook returned a tensor of another dtype, shape or device than it was given")


def _given(t: torch.Tensor, dtype: torch.dtype, numel: int, like: torch.Tensor) -> torch.Tensor:
    """Another saved tensor, contiguous."""
    if t.dtype is not dtype or t.numel() != numel or t.get_device() != like.get_device():
        _refuse_hook()
    return t.contiguous()


def _once(backward):
    """once_differentiable, whose context manager a backward pass without create_graph does not need."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def call(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return call


def _opts(layout, g, lengths, reverse) -> "_lib.NkScanOpts":
    (_, _, J), (B, T, C), (ab, at, _), (xb, xt, _), dt_a, dt_x = layout
    gb, gt, _ = (0, 0, 0) if g is None else g.stride()
    return _lib.NkScanOpts(B, T, C, J, _lib.DTYPES[dt_x], _lib.DTYPES[dt_a], reverse, 0, ab, at, xb, xt, gb, gt, _ptr(lengths))


def _workspace(L, o, backward, dev):
    n = L.nk_gated_scan_workspace_bytes(o, backward)
    if n == 0:
        return None, 0
    return torch.empty(_lib.check(n), dtype=torch.uint8, device=dev), n         # torch's blocks are 512-byte aligned


def _forward(a, x, layout, h0, lengths, reverse, training):
    L = _lib.load()
    B, T, C = layout[1]
    dev = x.device
    if B == 0 or T == 0:        # no step: the state passes through
        return x.new_empty(B, T, C), (h0.clone() if h0 is not None else torch.zeros(B, C, dtype=torch.float32, device=dev)), None
    h = _like(x)
    last = torch.empty_like(h0) if h0 is not None else torch.empty((B, C), dtype=torch.float32, device=dev)
    o = _opts(layout, None, lengths, reverse)
    states = torch.empty(B * (-(-T // _KEEP)) * C, dtype=torch.float32, device=dev) if training else None
    ws, n = _workspace(L, o, 0, dev)
    _lib.launch(dev, L.nk_gated_scan_fwd, o, a.data_ptr(), x.data_ptr(), _ptr(h0), h.data_ptr(), last.data_ptr(), _ptr(states), _ptr(ws), n)
    return h, last, states


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, x, h0, lengths, reverse):
        # the kept states serve the gates' gradient alone
        ctx.layout = _layout(a, x)
        h, last, states = _forward(a, x, ctx.layout, h0, lengths, reverse, ctx.needs_input_grad[0])
        ctx.save_for_backward(a, x, h0, lengths, states)
        ctx.reverse = reverse
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @_once
    def backward(ctx, d_h, d_last):
        want_a, want_x, want_0 = ctx.needs_input_grad[:3]
        if d_h is None and d_last is None:
            return None, None, None, None, None
        saved = ctx.saved_tensors
        a, x, layout = _unpacked(ctx, _rows, saved, d_h if d_h is not None else d_last)
        B, T, C = layout[1]
        h0, lengths, states = saved[2:]
        if h0 is not None:
            h0 = _given(h0, torch.float32, B * C, x)
        if lengths is not None:
            lengths = _given(lengths, torch.int32, B, x)
        if states is not None:
            states = _given(states, torch.float32, B * -(-T // _KEEP) * C, x)
        dev = x.device
        d_last = _whole(d_last)
        if B == 0 or T == 0:
            z = lambda t, want: torch.zeros_like(t) if want else None
            d_0 = None
            if want_0:
                d_0 = d_last.clone() if d_last is not None else torch.zeros_like(h0)
            return z(a, want_a), z(x, want_x), d_0, None, None
        L = _lib.load()
        g = _rows(d_h) if d_h is not None else None
        o = _opts(layout, g, lengths, ctx.reverse)
        d_a = _like(a) if want_a else None
        d_x = _like(x) if want_x else None
        d_0 = torch.empty_like(h0) if want_0 else None
        ws, n = _workspace(L, o, 1, dev)
        _lib.launch(dev, L.nk_gated_scan_bwd, o, a.data_ptr(), x.data_ptr(), _ptr(states), _ptr(h0), _ptr(g), _ptr(d_last),
                    _ptr(d_a), _ptr(d_x), _ptr(d_0), _ptr(ws), n)
        return d_a, d_x, d_0, None, None


def _call(a, x, h0, lengths, reverse):
    """The operator on checked arguments."""
    a, x, h0 = _rows(a), _rows(x), _whole(h0)
    if torch.is_grad_enabled() and (a.requires_grad or x.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(a, x, h0, lengths, reverse)
    return _forward(a, x, _layout(a, x), h0, lengths, reverse, False)[:2]


def gated_scan(a: torch.Tensor, x: torch.Tensor, h0: Optional[torch.Tensor] = None, *, lengths: Optional[torch.Tensor] = None,
               reverse: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h_t = a_t * h_(t-1) + x_t`` along axis 1 of ``x`` [B, T, C]; returns ``(h, h_last)``.

    ``a`` is [B, T, J] with J dividing C: gate j serves the C / J consecutive channels from ``j * C / J`` on (J = 1:
    one gate per step; J = C: one per channel), of ``x``'s dtype or float32.  ``x`` and ``h`` are float32,
    bfloat16 or float16; the state is float32: ``h0`` [B, C] (default zero) and ``h_last`` [B, C].  ``reverse`` walks
    from the last step to the first.  ``lengths`` [B] int32 cuts sequence b short: rows behind it are not read and
    ``h`` and all gradients are zero there; values outside 0..T are clamped.

    Differentiable in ``a``, ``x`` and ``h0`` (first order, reverse mode), through both results.  For one step at a time pass T = 1
    and the last state as ``h0``.  A training call also keeps the float32 state in front of every 32nd step.
    """
    if not isinstance(x, torch.Tensor) or x.dtype not in _lib.DTYPES or x.dim() != 3:
        raise ValueError("x: expected a [B, T, C] tensor of float32, bfloat16 or float16")
    B, T, C = x.shape
    if not isinstance(a, torch.Tensor) or a.dim() != 3 or a.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"a: expected a [{B}, {T}, J] tensor of {x.dtype} or float32")
    Ba, Ta, J = a.shape
    if Ba != B or Ta != T:
        raise ValueError(f"a: expected a [{B}, {T}, J] tensor of {x.dtype} or float32")
    if C < 1 or J < 1 or C % J:
        raise ValueError(f"a: {J} gates for {C} channels (a divisor of them)")
    _no_tangents(a, x, h0)
    reverse = bool(reverse)
    dev = x.device
    if dev.type != "cuda":
        raise ValueError("x: expected a GPU tensor (there is no CPU implementation)")
    if a.device != dev:
        raise ValueError(f"a: expected a tensor on {dev}")
    if h0 is not None:
        if h0.dtype != torch.float32 or h0.shape != (B, C) or h0.device != dev:
            raise ValueError(f"h0: expected a float32 tensor of shape {(B, C)} on {dev}")
    if lengths is not None:
        if lengths.dtype != torch.int32 or lengths.shape != (B,) or lengths.device != dev:
            raise ValueError(f"lengths: expected an int32 tensor of shape {(B,)} on {dev}")
        lengths = lengths.contiguous()
    return _call(a, x, h0, lengths, int(reverse))
