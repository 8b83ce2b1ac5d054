"""AdamW over many tensors in one launch (``nk_adamw_step``), with 32-bit or 8-bit moments.

Stands beside :func:`~nerf_kinematics_amd.render.adam_step` (Adam on flat fp32 buffers, the optimiser of
the reference's checkpoints).  ``adamw_step`` updates lists of tensors once; :class:`AdamW` keeps the
moments of a list of parameters and the launch table a program reuses.  Everything runs on the current
torch stream of the tensors' GPU; bad shapes, types or overlaps of parameters, masters and moments raise ``ValueError`` before any
launch (that gradients share no memory with what a step writes is the caller's to see to).

8-bit moments: blocks of 256 consecutive elements of a tensor share a power-of-two fp32 scale; an element
is ``code * scale`` with an OCP e4m3 code (first moment) or e5m2 code (second moment).
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import List, Optional, Sequence, Tuple

import torch
from torch.autograd.graph import increment_version as _increment_version

from . import lib as _lib

BLOCK = 256                       # elements that share a scale in an 8-bit moment
MOMENT_DTYPES = {32: (torch.float32, torch.float32), 8: (torch.float8_e4m3fn, torch.float8_e5m2)}
_TENSOR_WORDS = C.sizeof(_lib.NkAdamwTensor) // 8
_address, _numel, _get_device, _is_contiguous = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous
_dtype = operator.attrgetter("dtype")


def _check_list(name: str, tensors: Sequence[torch.Tensor], numels: Sequence[int], dtype: torch.dtype, device, spans: list) -> List[int]:
    """Checks a list against the parameters' element counts; returns the addresses, adds the extents to `spans`."""
    if len(tensors) != len(numels):
        raise ValueError(f"{name}: {len(tensors)} tensors for {len(numels)} parameters")
    size, out = dtype.itemsize, []
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
            raise ValueError(f"{name}[{i}]: expected a {dtype} tensor on {device}")
        if t.numel() != numels[i]:
            raise ValueError(f"{name}[{i}]: {t.numel()} elements, expected {numels[i]}")
        if not t.is_contiguous():
            raise ValueError(f"{name}[{i}]: must be contiguous")
        if t.is_neg():          # its memory holds the opposite sign
            raise ValueError(f"{name}[{i}]: is negated lazily (an imaginary part of a conjugate): resolve_neg() it")
        at = t.data_ptr()
        out.append(at)
        if numels[i]:
            if at == 0:
                raise ValueError(f"{name}[{i}]: has no storage")
            spans.append((at, at + numels[i] * size))
    return out


def _check_disjoint(spans: list) -> None:
    spans.sort()
    end = 0
    for a, b in spans:
        if a < end:
            raise ValueError("parameters, masters and moments must not overlap in memory (the same tensor twice?)")
        end = b


def adamw_state(params: Sequence[torch.Tensor], state_bits: int = 32):
    """Zero moments for ``params``: ``(exp_avgs, exp_avg_sqs, scales)``; ``scales`` is None for 32-bit moments
    and a list of ``(scale_m, scale_v)`` pairs, one value per block of 256 elements, for 8-bit ones."""
    if state_bits not in MOMENT_DTYPES:
        raise ValueError(f"state_bits={state_bits}: 32 or 8")
    dm, dv = MOMENT_DTYPES[state_bits]
    m = [torch.zeros(p.numel(), dtype=dm, device=p.device) for p in params]
    v = [torch.zeros(p.numel(), dtype=dv, device=p.device) for p in params]
    if state_bits == 32:
        return m, v, None
    mk = lambda p: torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
    return m, v, [(mk(p), mk(p)) for p in params]


def decode_moment(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp32 values of an 8-bit moment (a host-side helper for checkpoints)."""
    n = codes.numel()
    return codes.reshape(-1).float() * scale.repeat_interleave(BLOCK)[:n]


def encode_moment(values: torch.Tensor, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of fp32 values, rounded to nearest (a host-side helper for checkpoints); values
    that ``decode_moment`` gave come back as the same values."""
    top = {torch.float8_e4m3fn: 8, torch.float8_e5m2: 15}[dtype]
    n = values.numel()
    b = torch.nn.functional.pad(values.reshape(-1).float(), (0, -n % BLOCK)).view(-1, BLOCK)
    frac, e = torch.frexp(b.abs().amax(1, keepdim=True))
    e = torch.where(frac == 0, torch.full_like(e, -100), e - (frac == 0.5).to(e.dtype) - top).clamp_min(-100)
    pow2 = lambda k: ((k.to(torch.int32) + 127) << 23).view(torch.float32)      # exact, which torch.ldexp is not on every device
    scaled = b * pow2(-e)
    codes = scaled.to(dtype)
    if dtype == torch.float8_e5m2:       # a second moment stays positive
        least = torch.full_like(scaled, 2.0 ** -16).to(dtype)
        codes = torch.where((scaled > 0) & (codes.float() == 0), least.view(torch.uint8), codes.view(torch.uint8)).view(dtype)
    return codes.reshape(-1)[:n].clone(), pow2(e[:, 0])


class AdamW:
    """torch.optim.AdamW's update for a list of parameters, updated in place by one launch per 56 tensors.

    ``params``: contiguous GPU tensors of one dtype (fp32, bf16 or fp16) on one device.  ``masters``: fp32
    copies that the step updates instead, the parameters then receive them rounded; low-precision
    parameters without masters lose updates below half their last place.  ``state_bits``: 32 or 8.
    ``state``: moments to continue from, as ``adamw_state`` lays them out (their dtype decides the format); they
    stay the optimiser's, load into them with ``copy_``.  Parameters and masters may move (``p.data = ...``), and ``lr``, ``betas``,
    ``eps`` and ``weight_decay`` may be assigned: a step takes them as they are then."""

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, masters: Optional[Sequence[torch.Tensor]] = None,
                 state=None, seed: int = 0):
        self._L = _lib.load()
        params = list(params)
        if not params:
            raise ValueError("AdamW: no parameters")
        dt, dev = params[0].dtype, params[0].device
        if dt not in _lib.DTYPES:
            raise ValueError(f"AdamW: parameters of dtype {dt} (float32, bfloat16 or float16)")
        if dev.type != "cuda":
            raise ValueError("AdamW: expected GPU tensors (there is no CPU implementation)")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0):
            raise ValueError(f"AdamW: betas={tuple(betas)} in [0, 1), eps={eps} >= 0 wanted")
        if state is None:
            state = adamw_state(params, state_bits)
        m, v, scales = state
        if not m or m[0].dtype not in (torch.float32, torch.float8_e4m3fn):
            raise ValueError("AdamW: moments are float32 or float8_e4m3fn / float8_e5m2")
        state_bits = 32 if m[0].dtype == torch.float32 else 8
        if state_bits == 8 and scales is None:
            raise ValueError("AdamW: 8-bit moments need one (scale_m, scale_v) pair per parameter")
        if state_bits == 32 and scales is not None:
            raise ValueError("AdamW: scales belong to 8-bit moments")
        self.params, self.masters = tuple(params), None if masters is None else tuple(masters)
        self.exp_avgs, self.exp_avg_sqs, self.scales = tuple(m), tuple(v), None if scales is None else tuple(tuple(s) for s in scales)
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), (float(betas[0]), float(betas[1])), float(eps), float(weight_decay)
        self.state_bits, self.seed, self.steps = state_bits, int(seed), 0
        self.device, self._dtype = dev, dt
        self._numels, self._indices = [p.numel() for p in params], [dev.index] * len(params)
        self._single = [i for i, n in enumerate(self._numels) if n == 1]       # alone can be contiguous and an imaginary part of a conjugate
        self._owned = self.params + (self.masters or ())
        self._held = [t.detach() for t in (*m, *v, *(s for pair in scales or () for s in pair))]       # the table's moments, whatever becomes of `state`
        self._bind()
        self._opts = _lib.NkAdamwOpts()
        self._opts.param_dtype, self._opts.state_bits = _lib.DTYPES[dt], state_bits

    def _bind(self) -> None:
        """Checks every tensor and lays down the launch table."""
        numels, dev, spans, n = self._numels, self.device, [], len(self.params)
        none = [0] * n
        at_p = _check_list("params", self.params, numels, self._dtype, dev, spans)
        at_w = none if self.masters is None else _check_list("masters", self.masters, numels, torch.float32, dev, spans)
        dm, dv = MOMENT_DTYPES[self.state_bits]
        at_m = _check_list("exp_avgs", self._held[:len(self.exp_avgs)], numels, dm, dev, spans)
        at_v = _check_list("exp_avg_sqs", self._held[len(self.exp_avgs):len(self.exp_avgs) + len(self.exp_avg_sqs)], numels, dv, dev, spans)
        at_sm = at_sv = none
        if self.state_bits == 8:
            blocks = [-(-k // BLOCK) for k in numels]
            scales = self._held[len(self.exp_avgs) + len(self.exp_avg_sqs):]
            at_sm = _check_list("scale_m", scales[0::2], blocks, torch.float32, dev, spans)
            at_sv = _check_list("scale_v", scales[1::2], blocks, torch.float32, dev, spans)
        _check_disjoint(spans)
        self._at = at_p + (at_w if self.masters is not None else [])
        # nk_adamw_tensor, word by word: param, grad (filled in by step), exp_avg, exp_avg_sq, master, scales, n
        self._words = (C.c_int64 * (_TENSOR_WORDS * n))(*[w for row in zip(at_p, none, at_m, at_v, at_w, at_sm, at_sv, numels) for w in row])
        self._table = C.cast(self._words, C.POINTER(_lib.NkAdamwTensor))

    def _check_grads(self, grads) -> List[int]:
        """Addresses of the gradients, after their checks (whole lists at a time: a step is called with hundreds)."""
        n, numels, dev = len(self.params), self._numels, self.device
        try:
            same = len(grads) == n and list(map(_numel, grads)) == numels and list(map(_get_device, grads)) == self._indices and all(map(_is_contiguous, grads))
        except TypeError:           # not a tensor
            raise ValueError(f"grads: {len(grads)} entries for {n} parameters, one tensor each wanted") from None
        if len(grads) != n:
            raise ValueError(f"grads: {len(grads)} tensors for {n} parameters")
        gd = grads[0].dtype
        if gd != torch.float32 and gd != self._dtype:
            raise ValueError(f"grads: dtype {gd} (float32 or the parameters' {self._dtype})")
        if not same or list(map(_dtype, grads)) != [gd] * n:
            for i, (g, k) in enumerate(zip(grads, numels)):
                if g.dtype != gd or g.numel() != k or g.device != dev or not g.is_contiguous():
                    raise ValueError(f"grads[{i}]: expected {k} contiguous {gd} values on {dev}")
        return list(map(_address, grads))

    def step(self, grads: Optional[Sequence[torch.Tensor]] = None, *, lr: Optional[float] = None, step: Optional[int] = None,
             grad_scale: float = 1.0, seed: Optional[int] = None, step_state: Optional[int] = None) -> None:
        """One update.  ``grads``: one contiguous tensor per parameter, all fp32 or all of the parameters' dtype
        (default: the parameters' ``.grad``, which must exist); they share no memory with what the step writes.  ``step`` (from 1; default: one more than the
        last) sets the bias corrections, ``seed`` the stochastic rounding of 8-bit moments (default: the
        optimiser's, moved on by the step).  ``step_state``: device address of an ``nk_step_state`` to read the
        step-dependent scalars from when the kernel runs (graph replay)."""
        n = len(self.params)
        if list(map(_address, self._owned)) != self._at:        # a parameter moved
            self._bind()
        if grads is None:
            grads = [p.grad for p in self.params]
            if any(g is None for g in grads):
                raise ValueError("AdamW.step: a parameter has no .grad")
        self._words[1::_TENSOR_WORDS] = self._check_grads(grads)
        if any(grads[i].is_neg() for i in self._single):        # the memory of such a view holds the opposite sign
            grads = [g.resolve_neg() for g in grads]
            self._words[1::_TENSOR_WORDS] = list(map(_address, grads))
        gd = grads[0].dtype
        step = self.steps + 1 if step is None else int(step)
        if step < 1:
            raise ValueError(f"step={step}: from 1")
        o = self._opts
        o.grad_dtype, o.step, o.lr, o.weight_decay = _lib.DTYPES[gd], step, self.lr if lr is None else float(lr), self.weight_decay
        (o.beta1, o.beta2), o.eps, o.grad_scale = self.betas, self.eps, float(grad_scale)
        o.seed = (self.seed + 0x9E3779B1 * step if seed is None else int(seed)) & 0xFFFFFFFF
        o.state = step_state
        _lib.launch(self.device, self._L.nk_adamw_step, self._table, n, o)
        self.steps = step
        _increment_version(self._owned)         # autograd refuses to use what it saved of them before


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], step: int, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, *, scales=None, masters: Optional[Sequence[torch.Tensor]] = None,
               grad_scale: float = 1.0, seed: int = 0) -> None:
    """One AdamW update of ``params`` in place (see :class:`AdamW` for the arguments)."""
    AdamW(params, lr, betas, eps, weight_decay, masters=masters, state=(exp_avgs, exp_avg_sqs, scales)).step(
        grads, step=step, grad_scale=grad_scale, seed=seed)
