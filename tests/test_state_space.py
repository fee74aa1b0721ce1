"""State-space operators without a GPU: the 64-bit definitions the GPU tests compare with, refusals,
and the C-ABI's host-side checks."""
import ctypes
import os
import re
import subprocess
import textwrap

import pytest
import torch

import _state_space as ref
import scanscam_b200
from scanscam_b200 import _native

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rand(*shape, seed=0, dtype=torch.float64):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape)), dtype=torch.float64).to(dtype)


# ---- the definitions --------------------------------------------------------------------------
@pytest.mark.parametrize("softplus,gated,offsets", [(True, True, None), (False, False, None), (True, False, [0, 3, 3, 9])])
def test_scan_definition_agrees_with_differences(softplus, gated, offsets):
    n, c, t, s, g = (1 if offsets else 2), 4, 9, 3, 2
    spans = ref.spans_of(n, t, offsets=offsets)
    ops = {"x": rand(n, c, t), "dt": rand(n, c, t, seed=1).abs() * 0.3, "A": -rand(c, s, seed=2).abs(), "B": rand(n, g, s, t, seed=3),
           "C": rand(n, g, s, t, seed=4), "D": rand(c, seed=5), "dt_bias": rand(c, seed=6), "state": rand(len(spans), c, s, seed=7)}
    if gated:
        ops["z"] = rand(n, c, t, seed=8)
    gout, gstate = rand(n, c, t, seed=9), rand(len(spans), c, s, seed=10)

    def loss(o):
        r = ref.scan_selective(**o, dt_softplus=softplus, spans=spans)
        return (r["out"][0] * gout).sum() + (r["state"][0] * gstate).sum()

    r = ref.scan_selective(**ops, dt_softplus=softplus, spans=spans, gout=gout, gstate=gstate)
    step = 1e-5
    for name, value in ops.items():
        way = rand(*value.shape, seed=11)
        up, down = ({**ops, name: value + sign * step * way} for sign in (1, -1))
        slope = (loss(up) - loss(down)) / (2 * step)
        # central differences: the third derivative's term, about 1e-10 here, and 1e-16 / 1e-5 of the loss
        assert abs(slope - (r["g" + name][0] * way).sum()) < 1e-7 * (1 + abs(slope)), name


@pytest.mark.parametrize("silu,width,offsets", [(True, 4, None), (False, 2, None), (True, 3, [0, 1, 1, 7])])
def test_convolution_definition_agrees_with_differences(silu, width, offsets):
    n, c, t = (1 if offsets else 2), 3, 7
    spans = ref.spans_of(n, t, offsets=offsets)
    ops = {"x": rand(n, c, t), "weight": rand(c, width, seed=1), "bias": rand(c, seed=2), "state": rand(len(spans), c, width - 1, seed=3)}
    gout, gstate = rand(n, c, t, seed=4), rand(len(spans), c, width - 1, seed=5)

    def loss(o):
        r = ref.short_conv(**o, silu=silu, spans=spans)
        return (r["out"][0] * gout).sum() + (r["state"][0] * gstate).sum()

    r = ref.short_conv(**ops, silu=silu, spans=spans, gout=gout, gstate=gstate)
    for name, value in ops.items():
        way = rand(*value.shape, seed=6)
        up, down = ({**ops, name: value + sign * 1e-5 * way} for sign in (1, -1))
        slope = (loss(up) - loss(down)) / 2e-5
        assert abs(slope - (r["g" + name][0] * way).sum()) < 1e-7 * (1 + abs(slope)), name


def test_a_planted_mistake_is_seen():
    """The comparison refuses a result that is off by a few steps of its type, and takes one that is off by half of one."""
    value = torch.tensor([1.0, -3.0, 0.25], dtype=torch.float64)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        ref.check(value * (1 + 0.49 * torch.finfo(dtype).eps), (value, value.abs()), dtype, 0, "half a step")
        with pytest.raises(AssertionError):
            ref.check(value * (1 + 3 * torch.finfo(dtype).eps), (value, value.abs()), dtype, 2, "three steps")
    with pytest.raises(AssertionError):
        ref.check(torch.tensor([float("nan")]), (value[:1], value[:1]), torch.float32, 0, "nan")


# ---- refusals -------------------------------------------------------------------------------------
def scan_args(**other):
    f = torch.float32
    a = {"x": rand(2, 6, 5, dtype=f), "dt": rand(2, 6, 5, dtype=f), "A": rand(6, 4, dtype=f), "B": rand(2, 4, 5, dtype=f), "C": rand(2, 4, 5, dtype=f)}
    return {**a, **other}


SCAN_REFUSALS = [
    (dict(), "no CPU path"),
    (dict(x=torch.zeros(6, 5)), "3-D"),
    (dict(dt=torch.zeros(2, 6, 4)), "dt must have the shape"),
    (dict(dt=torch.zeros(2, 6, 5).bfloat16()), "dt must have the same dtype"),
    (dict(A=torch.zeros(5, 4)), "A must be"),
    (dict(A=torch.zeros(6, 4).bfloat16()), "A must be float32"),
    (dict(A=torch.zeros(6, 257), B=torch.zeros(2, 257, 5), C=torch.zeros(2, 257, 5)), "1 to 256 states"),
    (dict(A=torch.zeros(6, 0), B=torch.zeros(2, 0, 5), C=torch.zeros(2, 0, 5)), "1 to 256 states"),
    (dict(B=torch.zeros(2, 3, 5)), "B must be"),
    (dict(B=torch.zeros(2, 4, 4, 5), C=torch.zeros(2, 4, 4, 5)), "do not divide"),
    (dict(C=torch.zeros(2, 2, 4, 5)), "C must have the shape"),
    (dict(C=torch.zeros(2, 4, 5).half()), "C must have the same dtype"),
    (dict(D=torch.zeros(5)), "D must have the shape"),
    (dict(D=torch.zeros(6).half()), "D must be float32"),
    (dict(dt_bias=torch.zeros(6, 1)), "dt_bias must have the shape"),
    (dict(z=torch.zeros(2, 5, 6)), "z must have the shape"),
    (dict(state=torch.zeros(1, 6, 4)), "state must have the shape"),
    (dict(state=torch.zeros(2, 6, 4).half()), "state must be float32"),
    (dict(lengths=torch.zeros(2)), "lengths must be int32"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "one entry per row"),
    (dict(offsets=torch.zeros(2, dtype=torch.int32)), "packed sequences"),
    (dict(offsets=torch.zeros(2, dtype=torch.int64)), "offsets must be int32"),
    (dict(x=torch.zeros(1, 6, 5), dt=torch.zeros(1, 6, 5), B=torch.zeros(1, 4, 5), C=torch.zeros(1, 4, 5), offsets=torch.zeros(1, dtype=torch.int32)),
     "at least one sequence"),
    (dict(lengths=torch.zeros(2, dtype=torch.int32), offsets=torch.zeros(2, dtype=torch.int32)), "exclude each other"),
]


@pytest.mark.parametrize("other,message", SCAN_REFUSALS)
def test_scan_refuses(other, message):
    a = scan_args(**other)
    with pytest.raises(RuntimeError, match=message):
        scanscam_b200.scan_selective(a.pop("x"), a.pop("dt"), a.pop("A"), a.pop("B"), a.pop("C"), **a)
    if "shape" not in message:  # the same words where a gradient is wanted
        a = scan_args(**other)
        x = a.pop("x").requires_grad_(True)
        with pytest.raises(RuntimeError, match=message):
            scanscam_b200.scan_selective(x, a.pop("dt"), a.pop("A"), a.pop("B"), a.pop("C"), **a)


def test_float64_is_refused_like_other_types():
    a = scan_args()
    with pytest.raises(NotImplementedError, match="not implemented for 'Double'"):
        scanscam_b200.scan_selective(a["x"].double(), a["dt"], a["A"], a["B"], a["C"])
    with pytest.raises(NotImplementedError, match="not implemented for 'Int'"):
        scanscam_b200.short_conv(torch.zeros(1, 2, 3, dtype=torch.int32), torch.zeros(2, 4))


STEP = dict(x=torch.zeros(3, 6), dt=torch.zeros(3, 6), A=torch.zeros(6, 4), B=torch.zeros(3, 4), C=torch.zeros(3, 4), state=torch.zeros(3, 6, 4))
STEP_REFUSALS = [
    (dict(), "no CPU path"),
    (dict(x=torch.zeros(6)), "2-D"),
    (dict(B=torch.zeros(2, 4)), "B must be"),
    (dict(state=torch.zeros(4, 6, 4)), "one row per row"),
    (dict(state=torch.zeros(3, 6, 5)), "state must have the shape"),
    (dict(state=torch.zeros(3, 4, 6).mT), "state must be contiguous"),
    (dict(state=torch.zeros(3, 6, 4).half()), "state must be float32"),
    (dict(slots=torch.zeros(3)), "slots must be int32"),
    (dict(slots=torch.zeros(2, dtype=torch.int32)), "slots must have one entry"),
    (dict(x=torch.zeros(3, 6, requires_grad=True)), "no_grad"),
]


@pytest.mark.parametrize("other,message", STEP_REFUSALS)
def test_scan_step_refuses(other, message):
    a = {**STEP, **other}
    with pytest.raises(RuntimeError, match=message):
        scanscam_b200.scan_selective_step(**a)


CONV_REFUSALS = [
    (dict(), "no CPU path"),
    (dict(x=torch.zeros(6, 5)), "3-D"),
    (dict(weight=torch.zeros(5, 4)), "weight must be"),
    (dict(weight=torch.zeros(6, 1)), "2, 3 or 4 taps"),
    (dict(weight=torch.zeros(6, 5)), "2, 3 or 4 taps"),
    (dict(weight=torch.zeros(6, 4).half()), "float32 or have the dtype of x"),
    (dict(bias=torch.zeros(5)), "bias must have the shape"),
    (dict(x=torch.zeros(2, 6, 5).half(), bias=torch.zeros(6).half()), "same dtype as weight"),
    (dict(state=torch.zeros(2, 6, 4)), "state must have the shape"),
    (dict(state=torch.zeros(2, 6, 3).half()), "state must have the same dtype"),
    (dict(offsets=torch.zeros(2, dtype=torch.int32)), "packed sequences"),
]


@pytest.mark.parametrize("other,message", CONV_REFUSALS)
def test_short_conv_refuses(other, message):
    a = {"x": torch.zeros(2, 6, 5), "weight": torch.zeros(6, 4), **other}
    with pytest.raises(RuntimeError, match=message):
        scanscam_b200.short_conv(**a)


def test_short_conv_activation_and_step_refusals():
    x, w = torch.zeros(2, 6, 5), torch.zeros(6, 4)
    with pytest.raises(ValueError, match="activation"):
        scanscam_b200.short_conv(x, w, activation="relu")
    with pytest.raises(ValueError, match="activation"):
        scanscam_b200.short_conv_step(x[:, :, 0], torch.zeros(2, 6, 3), w, activation="gelu")
    for other, message in [(dict(), "no CPU path"), (dict(state=torch.zeros(3, 6, 3)), "one row per row"),
                           (dict(state=torch.zeros(2, 6, 4)), "state must have the shape"),
                           (dict(slots=torch.zeros(1, dtype=torch.int32)), "slots must have one entry"),
                           (dict(weight=w.clone().requires_grad_(True)), "no_grad")]:
        a = {"x": x[:, :, 0], "state": torch.zeros(2, 6, 3), "weight": w, **other}
        with pytest.raises(RuntimeError, match=message):
            scanscam_b200.short_conv_step(**a)


# ---- the C-ABI --------------------------------------------------------------------------------------
STRUCTS = {"ssb_view_t": _native.View, "ssb_selective_t": _native.Selective, "ssb_selective_grads_t": _native.SelectiveGrads,
           "ssb_selective_step_t": _native.SelectiveStep, "ssb_short_conv_t": _native.ShortConv,
           "ssb_short_conv_grads_t": _native.ShortConvGrads, "ssb_short_conv_step_t": _native.ShortConvStep}


def test_structures_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{REPO}/include/scanscam_b200.h"', "int main(void) {"]
    for name, struct in STRUCTS.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {field}));' for field, _ in struct._fields_]
        lines.append('printf("\\n");')
    (tmp_path / "sizes.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", tmp_path / "sizes", tmp_path / "sizes.c"], check=True)
    for line in subprocess.run([tmp_path / "sizes"], capture_output=True, text=True, check=True).stdout.splitlines():
        name, size, *at = line.split()
        struct = STRUCTS[name]
        assert ctypes.sizeof(struct) == int(size), name
        assert [getattr(struct, f).offset for f, _ in struct._fields_] == [int(a) for a in at], name


def problem(**other):
    p = _native.Selective(dtype=_native.F32, batch=2, channels=6, steps=5, states=4, groups=1)
    for k, v in other.items():
        setattr(p, k, v)
    return p


def test_scan_arguments_are_checked_on_the_host(native):
    """These calls return before any CUDA call: fake addresses are not dereferenced."""
    call = lambda p: native.ssb_selective_fwd(ctypes.byref(p), None)  # noqa: E731
    good = _native.View(0x1000, (ctypes.c_int64 * 4)(30, 5, 1, 0))
    assert native.ssb_selective_fwd(None, None) == _native.ERR_BAD_ARG
    assert call(problem()) == _native.ERR_BAD_ARG and b"x is NULL" in native.ssb_last_error()
    assert call(problem(dtype=7)) == _native.ERR_BAD_ARG
    assert call(problem(steps=-1)) == _native.ERR_BAD_ARG
    assert call(problem(steps=2**40, channels=2**40)) == _native.ERR_BAD_ARG
    assert call(problem(states=0)) == _native.ERR_UNSUPPORTED
    assert call(problem(states=257)) == _native.ERR_UNSUPPORTED
    assert call(problem(groups=4)) == _native.ERR_BAD_ARG
    assert call(problem(offsets=0x1000)) == _native.ERR_BAD_ARG and b"batch of 1" in native.ssb_last_error()
    assert call(problem(batch=1, offsets=0x1000, lengths=0x1000)) == _native.ERR_BAD_ARG
    assert call(problem(batch=1, offsets=0x1000, sequences=0)) == _native.ERR_BAD_ARG
    assert call(problem(x=_native.View(0x1002, (ctypes.c_int64 * 4)(30, 5, 1, 0)))) == _native.ERR_ALIGNMENT
    full = dict(x=good, dt=good, B=good, C=good, A=0x1000)
    assert call(problem(**full)) == _native.ERR_BAD_ARG and b"out is NULL" in native.ssb_last_error()
    assert call(problem(**{**full, "A": None})) == _native.ERR_BAD_ARG
    assert call(problem(**full, out=good, state=0x1001)) == _native.ERR_ALIGNMENT
    # nothing to do
    assert call(problem(batch=0, **full)) == _native.OK
    assert call(problem(channels=0)) == _native.OK
    # backward
    g = _native.SelectiveGrads()
    back = lambda p, ws=None, size=0: native.ssb_selective_bwd(ctypes.byref(p), ctypes.byref(g), ws, size, None)  # noqa: E731
    assert back(problem(**full)) == _native.ERR_BAD_ARG
    g.gout = g.gx = g.gdt = g.gB = g.gC = good
    assert back(problem(**full)) == _native.ERR_BAD_ARG and b"checkpoints" in native.ssb_last_error()
    g.gA = 0x1000
    assert back(problem(**full, checkpoints=0x1000)) == _native.ERR_WORKSPACE
    assert back(problem(**full, checkpoints=0x1000), 0x1000, 8) == _native.ERR_WORKSPACE


def test_scan_scratch_sizes(native):
    size = lambda f, **o: getattr(native, f)(ctypes.byref(problem(**o)))  # noqa: E731
    for f in ("ssb_selective_checkpoint_bytes", "ssb_selective_bwd_workspace_bytes"):
        assert size(f, states=300) == 0
        assert size(f, batch=4, channels=2048, steps=2048, states=16) > 0
    # one state in 16 steps is kept, at most
    assert size("ssb_selective_checkpoint_bytes", batch=4, channels=2048, steps=2048, states=16) <= 4 * 128 * 2048 * 16 * 4


def test_step_and_convolution_arguments_are_checked_on_the_host(native):
    v = _native.View(0x1000, (ctypes.c_int64 * 4)(6, 1, 0, 0))
    step = _native.SelectiveStep(dtype=_native.BF16, entries=3, channels=6, states=4, groups=1, pool=2)
    assert native.ssb_selective_step(ctypes.byref(step), None) == _native.ERR_BAD_ARG  # fewer states than entries
    step.slots = 0x1000
    assert native.ssb_selective_step(ctypes.byref(step), None) == _native.ERR_BAD_ARG  # x is NULL
    step.entries = 0
    assert native.ssb_selective_step(ctypes.byref(step), None) == _native.OK
    conv = _native.ShortConv(dtype=_native.F16, batch=1, channels=6, steps=5, width=5)
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_UNSUPPORTED
    conv.width = 4
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_BAD_ARG
    conv.x = _native.View(0x1000, (ctypes.c_int64 * 4)(30, 5, 1, 0))
    conv.sequences, conv.offsets = 2, 0x1000
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_UNSUPPORTED  # packed rows, time adjacent
    assert native.ssb_short_conv_bwd_workspace_bytes(ctypes.byref(conv)) > 0
    one = _native.ShortConvStep(dtype=_native.F32, entries=2, channels=6, width=4, pool=2, x=v, out=v, weight=0x1002)
    assert native.ssb_short_conv_step(ctypes.byref(one), None) == _native.ERR_ALIGNMENT


def test_names_are_offered():
    for name in ("scan_selective", "scan_selective_step", "short_conv", "short_conv_step"):
        assert callable(getattr(scanscam_b200, name)) and name in scanscam_b200.__all__
    text = open(os.path.join(REPO, "include", "scanscam_b200.h")).read()
    assert set(STRUCTS) <= set(re.findall(r"}\s*(ssb_\w+_t);", text))
    assert textwrap.dedent(scanscam_b200.scan_selective.__doc__)
