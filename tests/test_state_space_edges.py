"""State-space operators without a GPU: calls that no gradient is asked of, and sizes of one."""
import ctypes
import types

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import scanscam_b200
from scanscam_b200 import _native, cuda


# ---- forward-mode derivatives and traces ------------------------------------------------------------
def fill(t: torch.Tensor, value: float) -> None:
    """Writes as a kernel does, where neither autograd nor a trace sees it."""
    at = (ctypes.c_float * t.numel()).from_address(t.data_ptr())
    at[:] = [value] * t.numel()


@pytest.fixture
def stand_in(monkeypatch):
    """An extension whose functions allocate, and fill with the sum of x, as the kernels would: no GPU is needed to
    see what autograd and traces make of a call."""
    calls = []

    def made(x, *shapes):
        calls.append(x)
        total = sum((ctypes.c_float * x.numel()).from_address(x.data_ptr()))
        outs = tuple(torch.empty(s) for s in shapes)
        for out in outs:
            fill(out, total)
        return outs

    ext = types.SimpleNamespace(
        selective_forward=lambda x, dt, A, *rest: (*made(x, x.shape, (x.shape[0], *A.shape)), torch.empty(0)),
        selective_step=lambda x, dt, A, B, C, state, *rest: made(x, x.shape)[0],
        short_conv_forward=lambda x, w, *rest: made(x, x.shape, (x.shape[0], x.shape[1], w.shape[1] - 1)),
        short_conv_step=lambda x, state, *rest: made(x, x.shape)[0])
    monkeypatch.setattr(cuda, "_ext", lambda: ext)
    return calls


def call(name, x):
    A, w = -torch.ones(6, 4), torch.ones(6, 4)
    if name == "scan_selective":
        return scanscam_b200.scan_selective(x, torch.ones(2, 6, 5), A, torch.ones(2, 4, 5), torch.ones(2, 4, 5))
    if name == "short_conv":
        return scanscam_b200.short_conv(x, w)
    if name == "scan_selective_step":
        return scanscam_b200.scan_selective_step(x, torch.ones(2, 6), A, torch.ones(2, 4), torch.ones(2, 4), torch.zeros(2, 6, 4))
    return scanscam_b200.short_conv_step(x, torch.zeros(2, 6, 3), w)


NAMES = ["scan_selective", "scan_selective_step", "short_conv", "short_conv_step"]


def operand(name, value=1.0):
    return torch.full((2, 6) if name.endswith("step") else (2, 6, 5), value)


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_derivatives_are_refused(stand_in, name):
    """They are not built: the call says so, as `scan` does, instead of giving a result without a tangent."""
    x = operand(name)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            call(name, forward_ad.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(NotImplementedError):
            call(name, forward_ad.make_dual(x, torch.ones_like(x)))
        assert forward_ad.unpack_dual(call(name, x)).tangent is None  # nothing to carry


@pytest.mark.parametrize("name", ["scan_selective_step", "short_conv_step"])
def test_a_refused_step_leaves_its_state(stand_in, name):
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(operand(name), torch.ones(2, 6))
        with pytest.raises(NotImplementedError):
            call(name, dual)
        # the same where the tangent comes with another operand
        with pytest.raises(NotImplementedError):
            scanscam_b200.short_conv_step(operand(name), torch.zeros(2, 6, 3), forward_ad.make_dual(torch.ones(6, 4), torch.ones(6, 4)))
    assert not stand_in  # no kernel ran


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad_mode", [True, False])
def test_a_trace_makes_the_call(stand_in, name, grad_mode):
    """A trace of the call gives the values of its own inputs, not memory that was never written."""
    with torch.set_grad_enabled(grad_mode):
        traced = torch.jit.trace(lambda x: call(name, x), (operand(name),))
        before = len(stand_in)
        other = operand(name, 3.0)
        out = traced(other)
    assert len(stand_in) == before + 1
    assert torch.equal(out, torch.full_like(other, float(other.sum())))


@pytest.mark.parametrize("name", NAMES)
def test_ordinary_calls(stand_in, name):
    for mode in (torch.no_grad, torch.enable_grad, torch.inference_mode):
        with mode():
            x = operand(name)
            assert torch.equal(call(name, x), torch.full_like(x, float(x.sum())))


# ---- one channel ----------------------------------------------------------------------------------------
def test_one_packed_channel_lies_either_way(native):
    """The stride of an axis of one channel says nothing: no layout of it is refused."""
    conv = _native.ShortConv(dtype=_native.F32, batch=1, channels=1, steps=10, width=4, sequences=2, offsets=0x1000,
                             x=_native.View(0x1000, (ctypes.c_int64 * 4)(10, 10, 1, 0)))
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_BAD_ARG
    assert b"weight is NULL" in native.ssb_last_error()
    conv.weight = 0x1000
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_BAD_ARG
    assert b"out is NULL" in native.ssb_last_error()
    grads = _native.ShortConvGrads(gout=conv.x, gx=conv.x)
    assert native.ssb_short_conv_bwd(ctypes.byref(conv), ctypes.byref(grads), None, 0, None) == _native.ERR_BAD_ARG
    assert b"gweight is NULL" in native.ssb_last_error()
    conv.channels = 2
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_UNSUPPORTED
