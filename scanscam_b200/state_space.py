"""Selective state-space operators: the scan whose gates, inputs and read-out depend on the token,
and the short causal convolution in front of it, for prompts and for single tokens.

``scan_selective`` is ``scan`` with ``gate = exp(dt * A)`` and ``value = dt * B * x`` for every one of
``S`` states of a channel, read out through ``C``: done with ``scan`` the gates, values and states
would be ``[N, C, S, T]`` tensors, ``S`` times what goes in and out.  Here they stay in registers.

Layouts are the package's: ``[N, C, T]`` with time last, dense or as the ``[N, C, T]`` view of dense
``[N, T, C]`` (channels last), or any slice of a larger tensor; outputs and gradients have the
layout (channels adjacent or steps adjacent) of the operand they belong to, but a packed convolution gives channels last.
Fastest are operands of one layout whose rows start on 16 bytes; others are fetched element by element.  float32, bfloat16 and
float16 tensors are taken; the arithmetic, the states and all sums are float32.

A batch holds one sequence per row, of all ``T`` steps or of the first ``lengths[n]``; or it is one
row of packed sequences, sequence ``s`` at steps ``offsets[s] .. offsets[s+1]``.  ``lengths`` and
``offsets`` are int32 tensors on the device and are not read on the host.  Steps that belong to no
sequence give zero, whatever lies there.  These operators are additions: the reference has no counterpart.
"""
from __future__ import annotations

from typing import Any, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.jit import is_tracing

from . import cuda

Out = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _recorded() -> bool:
    """Whether a call has to go through its autograd function although no gradient is asked for: a trace would keep
    the allocation of the outputs alone, and a forward-mode derivative, which the functions refuse, would be dropped."""
    return is_tracing() or forward_ad._current_level >= 0


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _refuse_grad(name: str, *tensors: Optional[torch.Tensor]) -> None:
    if _wants_grad(*tensors):
        raise RuntimeError(f"scanscam_b200.{name} updates its state in place and has no gradient; call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"scanscam_b200.{name} has no forward-mode derivative")


def _silu(activation: Optional[str]) -> bool:
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    return activation == "silu"


class ScanSelective(torch.autograd.Function):
    """``(out, state)`` of :func:`scan_selective`, ``B`` and ``C`` as ``[N, G, S, T]``."""

    @staticmethod
    def forward(ctx: Any, x, dt, A, B, C, D, z, dt_bias, state, lengths, offsets, dt_softplus):
        out, state_out, checkpoints = cuda._ext().selective_forward(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, lengths,
                                                                    offsets, any(ctx.needs_input_grad))
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, state, lengths, offsets, checkpoints)
        ctx.dt_softplus = dt_softplus
        ctx.set_materialize_grads(False)
        return out, state_out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad_out, grad_state):
        x, dt, A, B, C, D, z, dt_bias, state, lengths, offsets, checkpoints = ctx.saved_tensors
        if grad_out is None:
            if grad_state is None:
                return (None,) * 12
            grad_out = torch.zeros_like(x)
        grads = cuda._ext().selective_backward(x, dt, A, B, C, D, z, dt_bias, ctx.dt_softplus, state, lengths, offsets, checkpoints,
                                               grad_out, _dense(grad_state))
        return (*grads, None, None, None)


def scan_selective(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   dt_softplus: bool = False, state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   offsets: Optional[torch.Tensor] = None, return_state: bool = False) -> Out:
    """Selective scan: ``h_t = exp(dt_t A) h_{t-1} + dt_t B_t x_t``, ``y_t = C_t . h_t + D x_t``, times ``silu(z_t)``.

    :param x: ``[N, C, T]`` CUDA tensor
    :param dt: like ``x``: the step sizes, before ``dt_bias`` is added and, with ``dt_softplus``, before the softplus
    :param A: ``[C, S]`` float32, 1 to 256 states; negative entries decay (``exp(dt A)`` over 8 steps and more is formed as a product)
    :param B: ``[N, S, T]``, or ``[N, G, S, T]`` for ``G`` groups of ``C / G`` adjacent channels, in the dtype of ``x``
    :param C: like ``B``
    :param D: ``[C]`` float32, or None
    :param z: like ``x``: the gate's logits, or None for no gate
    :param dt_bias: ``[C]`` float32, or None
    :param state: ``[sequences, C, S]`` float32 state before the first step, or None for zero
    :param lengths: ``[N]`` int32 steps of each row, or None for all
    :param offsets: ``[sequences + 1]`` int32 bounds of packed sequences (``N`` is 1), or None
    :param return_state: also return the float32 state behind each sequence's last step
    :return: ``[N, C, T]``, and the state if asked for; differentiable (once) in every tensor but ``lengths`` and ``offsets``
    """
    if B.dim() == 3:
        B = B.unsqueeze(1)
    if C.dim() == 3:
        C = C.unsqueeze(1)
    A, D, dt_bias, state, lengths, offsets = map(_dense, (A, D, dt_bias, state, lengths, offsets))
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias, state) or _recorded():
        out, state_out = ScanSelective.apply(x, dt, A, B, C, D, z, dt_bias, state, lengths, offsets, dt_softplus)
    else:
        out, state_out, _ = cuda._ext().selective_forward(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, lengths, offsets, False)
    return (out, state_out) if return_state else out


class ScanSelectiveStep(torch.autograd.Function):
    """:func:`scan_selective_step` for traces; no gradient."""

    @staticmethod
    def forward(ctx: Any, x, dt, A, B, C, state, D, z, dt_bias, dt_softplus, slots):
        return cuda._ext().selective_step(x, dt, A, B, C, state, D, z, dt_bias, dt_softplus, slots)


def scan_selective_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor, *,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                        dt_softplus: bool = False, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step of :func:`scan_selective` for each of ``M`` tokens; ``state`` is updated in place.

    :param x: ``[M, C]`` CUDA tensor; ``dt`` and ``z`` like it
    :param B: ``[M, S]`` or ``[M, G, S]``; ``C`` like it
    :param state: ``[pool, C, S]`` float32, contiguous
    :param slots: ``[M]`` int32: the row of ``state`` each token works on, or None for its own number
        (``pool`` is then ``M``).  A slot outside the pool marks an idle entry: its output is zero and
        no state changes.  Entries with the same slot are consecutive tokens of it, in batch order.
    :return: ``[M, C]``; carries no gradient (a call that would need one is refused)
    """
    _refuse_grad("scan_selective_step", x, dt, A, B, C, state, D, z, dt_bias)
    step = ScanSelectiveStep.apply if is_tracing() else cuda._ext().selective_step
    return step(x, dt, _dense(A), B, C, state, _dense(D), z, _dense(dt_bias), dt_softplus, _dense(slots))


class ShortConv(torch.autograd.Function):
    """``(out, window)`` of :func:`short_conv`."""

    @staticmethod
    def forward(ctx: Any, x, weight, bias, state, lengths, offsets, silu):
        out, state_out = cuda._ext().short_conv_forward(x, weight, bias, silu, state, lengths, offsets)
        ctx.save_for_backward(x, weight, bias, state, lengths, offsets)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return out, state_out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad_out, grad_state):
        x, weight, bias, state, lengths, offsets = ctx.saved_tensors
        if grad_out is None:
            if grad_state is None:
                return (None,) * 7
            grad_out = torch.zeros_like(x)
        if offsets is not None and grad_out.stride(1) != 1:
            grad_out = grad_out.mT.contiguous().mT
        grads = cuda._ext().short_conv_backward(x, weight, bias, ctx.silu, state, lengths, offsets, grad_out, _dense(grad_state))
        return (*grads, None, None, None)


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
               state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
               offsets: Optional[torch.Tensor] = None, return_state: bool = False) -> Out:
    """Causal convolution of each channel with its own ``W`` taps: ``act(bias + sum_j weight[:, j] x_{t-W+1+j})``.

    :param x: ``[N, C, T]`` CUDA tensor
    :param weight: ``[C, W]`` with ``W`` of 2, 3 or 4, the last tap on the current step; in the dtype of ``x``, or float32
    :param bias: ``[C]`` in the dtype of ``weight``, or None
    :param activation: None or ``"silu"``
    :param state: ``[sequences, C, W-1]`` in the dtype of ``x``: the inputs before the first step, oldest first, or None for zeros
    :param lengths: ``[N]`` int32 steps of each row, or None for all
    :param offsets: ``[sequences + 1]`` int32 bounds of packed sequences (``N`` is 1), or None; packed
        sequences are computed channels last, other layouts are copied
    :param return_state: also return the window behind each sequence's last step
    :return: ``[N, C, T]``, and the window if asked for; differentiable (once) in ``x``, ``weight``, ``bias`` and ``state``
    """
    silu = _silu(activation)
    weight, bias, state, lengths, offsets = map(_dense, (weight, bias, state, lengths, offsets))
    if offsets is not None and x.dim() == 3 and x.stride(1) != 1:
        x = x.mT.contiguous().mT
    if _wants_grad(x, weight, bias, state) or _recorded():
        out, state_out = ShortConv.apply(x, weight, bias, state, lengths, offsets, silu)
    else:
        out, state_out = cuda._ext().short_conv_forward(x, weight, bias, silu, state, lengths, offsets)
    return (out, state_out) if return_state else out


class ShortConvStep(torch.autograd.Function):
    """:func:`short_conv_step` for traces; no gradient."""

    @staticmethod
    def forward(ctx: Any, x, state, weight, bias, silu, slots):
        return cuda._ext().short_conv_step(x, state, weight, bias, silu, slots)


def short_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                    activation: Optional[str] = None, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step of :func:`short_conv` for each of ``M`` tokens; ``state`` is updated in place.

    :param x: ``[M, C]`` CUDA tensor
    :param state: ``[pool, C, W-1]`` in the dtype of ``x``, contiguous: the last inputs, oldest first
    :param slots: as for :func:`scan_selective_step`
    :return: ``[M, C]``; carries no gradient (a call that would need one is refused)
    """
    silu = _silu(activation)
    _refuse_grad("short_conv_step", x, state, weight, bias)
    step = ShortConvStep.apply if is_tracing() else cuda._ext().short_conv_step
    return step(x, state, _dense(weight), _dense(bias), silu, _dense(slots))
