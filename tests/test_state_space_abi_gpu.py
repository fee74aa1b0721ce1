"""The state-space entry points of the C-ABI through ctypes, with raw pointers, strides and workspaces, against
the definitions in 64 bits; and the same again on the checked build, which reports any index outside a tensor.
Tolerances: tests/test_state_space_gpu.py."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import _state_space as ref
from scanscam_b200 import _native

pytestmark = pytest.mark.gpu
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}


def randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def status(lib):
    detail = ctypes.c_int(0)
    _native.check(lib.ssb_device_status(ctypes.byref(detail)))


def like_layout(x):
    n, c, t = x.shape
    return torch.empty(n, t, c, dtype=x.dtype, device="cuda").mT if x.stride(1) == 1 else torch.empty(n, c, t, dtype=x.dtype, device="cuda")


# both layouts, each form of the backward (few channels; many; more than 32 states), odd sizes, packed sequences
CASES = [(torch.float32, "rows", 2, 37, 70, 10, 1, None), (torch.bfloat16, "cl", 1, 24, 131, 16, 2, [1, 1, 33, 33, 97, 130]),
         (torch.float16, "cl", 2, 21, 40, 64, 3, None), (torch.float32, "cl", 10, 501, 33, 16, 1, None), (torch.bfloat16, "rows", 10, 512, 48, 16, 2, None),
         (torch.float32, "cl", 1, 212, 100, 13, 1, [0, *range(2, 98, 4), 99]), (torch.bfloat16, "cl", 3, 800, 35, 32, 1, None), (torch.float32, "rows", 1, 9, 33, 200, 1, None)]


@pytest.mark.parametrize("dtype,layout,n,c,t,s,g,offsets", CASES, ids=[f"{i}" for i in range(len(CASES))])
def test_selective_scan(native, dtype, layout, n, c, t, s, g, offsets):
    def nct(seed):
        return randn(n, t, 2 * c, seed=seed, dtype=dtype)[:, :, c:].mT if layout == "cl" else randn(n, c, t, seed=seed, dtype=dtype)

    def proj(seed):
        return randn(n, t, g, s, seed=seed, dtype=dtype).permute(0, 2, 3, 1) if layout == "cl" else randn(n, g, s, t, seed=seed, dtype=dtype)

    spans = ref.spans_of(n, t, offsets=offsets)
    x, dt, z, gout, B, C = nct(1), nct(2), nct(3), nct(4), proj(5), proj(6)
    A, D, bias, state = -torch.exp(randn(c, s, seed=7)), randn(c, seed=8), randn(c, seed=9) - 3, randn(len(spans), c, s, seed=10)
    gstate_out, state_out = randn(len(spans), c, s, seed=11), torch.full((len(spans), c, s), float("nan"), device="cuda")
    cuts = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out = like_layout(x)
    v, st = _native.view, _native.stream_of(x)
    p = _native.Selective(dtype=DTYPES[dtype], softplus=1, batch=n, channels=c, steps=t, states=s, groups=g, sequences=len(spans),
                          offsets=_native.ptr(cuts), x=v(x), dt=v(dt), z=v(z), B=v(B), C=v(C), out=v(out), A=A.data_ptr(), D=D.data_ptr(),
                          dt_bias=bias.data_ptr(), state=state.data_ptr(), state_out=state_out.data_ptr())
    kept = torch.empty(native.ssb_selective_checkpoint_bytes(ctypes.byref(p)), dtype=torch.uint8, device="cuda")
    p.checkpoints = kept.data_ptr()
    _native.check(native.ssb_selective_fwd(ctypes.byref(p), st))
    status(native)
    got = {"out": out, "state": state_out, "gx": like_layout(x), "gdt": like_layout(x), "gz": like_layout(x), "gA": torch.empty_like(A),
           "gB": torch.empty_like(B), "gC": torch.empty_like(C), "gD": torch.empty_like(D), "gdt_bias": torch.empty_like(bias), "gstate": torch.empty_like(state)}
    q = _native.SelectiveGrads(gout=v(gout), gstate_out=gstate_out.data_ptr(), **{k: v(got[k]) for k in ("gx", "gdt", "gz", "gB", "gC")},
                               **{k: got[k].data_ptr() for k in ("gA", "gD", "gdt_bias", "gstate")})
    size = native.ssb_selective_bwd_workspace_bytes(ctypes.byref(p))
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert native.ssb_selective_bwd(ctypes.byref(p), ctypes.byref(q), work.data_ptr(), size - 1, st) == _native.ERR_WORKSPACE
    _native.check(native.ssb_selective_bwd(ctypes.byref(p), ctypes.byref(q), work.data_ptr(), size, st))
    status(native)
    want = ref.scan_selective(x, dt, A, B, C, D, z, bias, True, state, spans, gout, gstate_out)
    step = float((ref.softplus(dt.double() + bias.double()[:, None]).amax((0, 2))[:, None] * A.double().abs()).max())
    roundings = 6 * t + s + 12 * (20 + min(step, 90)) + 60 + c + n * t
    for k, val in got.items():
        ref.check(val, want[k], dtype if k in ("out", "gx", "gdt", "gz", "gB", "gC") else torch.float32, roundings, k)


@pytest.mark.parametrize("dtype,layout,n,c,t,w,offsets", [(torch.float32, "rows", 2, 37, 70, 3, None), (torch.bfloat16, "cl", 1, 36, 131, 4, [1, 1, 33, 33, 97, 130]),
                                                          (torch.float16, "cl", 3, 21, 40, 2, None), (torch.float32, "cl", 5, 260, 600, 4, None)])
def test_short_convolution(native, dtype, layout, n, c, t, w, offsets):
    def nct(seed):
        return randn(n, t, c, seed=seed, dtype=dtype).mT if layout == "cl" else randn(n, c, t, seed=seed, dtype=dtype)

    spans = ref.spans_of(n, t, offsets=offsets)
    x, gout, weight, bias = nct(1), nct(2), randn(c, w, seed=3), randn(c, seed=4)
    state, gstate_out = randn(len(spans), c, w - 1, seed=5, dtype=dtype), randn(len(spans), c, w - 1, seed=6, dtype=dtype)
    cuts = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    got = {"out": like_layout(x), "state": torch.empty_like(state), "gx": like_layout(x), "gweight": torch.empty_like(weight),
           "gbias": torch.empty_like(bias), "gstate": torch.empty_like(state)}
    v, st = _native.view, _native.stream_of(x)
    p = _native.ShortConv(dtype=DTYPES[dtype], silu=1, weight_f32=1, batch=n, channels=c, steps=t, width=w, sequences=len(spans), offsets=_native.ptr(cuts),
                          x=v(x), out=v(got["out"]), weight=weight.data_ptr(), bias=bias.data_ptr(), state=state.data_ptr(), state_out=got["state"].data_ptr())
    _native.check(native.ssb_short_conv_fwd(ctypes.byref(p), st))
    size = native.ssb_short_conv_bwd_workspace_bytes(ctypes.byref(p))
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    q = _native.ShortConvGrads(gout=v(gout), gx=v(got["gx"]), gstate_out=gstate_out.data_ptr(), gweight=got["gweight"].data_ptr(),
                               gbias=got["gbias"].data_ptr(), gstate=got["gstate"].data_ptr())
    _native.check(native.ssb_short_conv_bwd(ctypes.byref(p), ctypes.byref(q), work.data_ptr(), size, st))
    status(native)
    want = ref.short_conv(x, weight, bias, True, state, spans, gout, gstate_out)
    for k, val in got.items():
        ref.check(val, want[k], torch.float32 if k in ("gweight", "gbias") else dtype, 24 + n * t, k)


def test_single_tokens(native):
    m, pool, c, s, w = 5, 7, 44, 16, 4
    slots = torch.tensor([6, -1, 0, 6, 7], dtype=torch.int32, device="cuda")
    x, taps, window = randn(m, c, seed=1), randn(c, w, seed=2), randn(pool, c, w - 1, seed=3)
    held, out, v, st = window.clone(), torch.empty(m, c, device="cuda"), _native.view, _native.stream_of(x)
    p = _native.ShortConvStep(dtype=_native.F32, weight_f32=1, entries=m, channels=c, width=w, pool=pool, slots=slots.data_ptr(), x=v(x), out=v(out),
                              weight=taps.data_ptr(), state=window.data_ptr())
    _native.check(native.ssb_short_conv_step(ctypes.byref(p), st))
    for i, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pool:
            assert (out[i] == 0).all()
            continue
        seen = torch.cat([held[slot], x[i][:, None]], 1)
        value = (seen.double() * taps.double()).sum(1).cpu()
        ref.check(out[i], (value, (seen * taps).double().abs().sum(1).cpu()), torch.float32, 8, "out")
        held[slot] = seen[:, 1:]
    assert torch.equal(window, held)
    A, B, C, state = -torch.exp(randn(c, s, seed=4)), randn(m, 1, s, seed=5), randn(m, 1, s, seed=6), randn(pool, c, s, seed=7)
    dt, before = randn(m, c, seed=8).abs() * 0.1, state.clone()
    q = _native.SelectiveStep(dtype=_native.F32, entries=m, channels=c, states=s, groups=1, pool=pool, slots=slots.data_ptr(), x=v(x), dt=v(dt), B=v(B), C=v(C),
                              out=v(out), A=A.data_ptr(), state=state.data_ptr())
    _native.check(native.ssb_selective_step(ctypes.byref(q), st))
    status(native)
    h = before.double()
    for i, slot in enumerate(slots.tolist()):
        if 0 <= slot < pool:
            d, u = dt[i].double()[:, None], x[i].double()[:, None]
            h[slot] = torch.exp(d * A.double()) * h[slot] + d * u * B[i].double()
            value, size = (h[slot] * C[i].double()).sum(1), (h[slot] * C[i].double()).abs().sum(1)
            ref.check(out[i], (value.cpu(), 2 * size.cpu() + 1), torch.float32, 12 + s + 24, "out")
        else:
            assert (out[i] == 0).all()
    ref.check(state, (h.cpu(), h.abs().cpu() + 1), torch.float32, 36, "state")


def test_the_same_on_the_checked_build():
    from scanscam_b200 import build

    if os.environ.get("SCANSCAM_B200_LIB"):
        pytest.skip("another build of the library was selected for this session")
    checked = build.LIB_CHECKED
    if not os.path.exists(checked):
        checked = build.build_library(checked=True)
    env = dict(os.environ, SCANSCAM_B200_LIB=checked)
    out = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", os.path.abspath(__file__)], capture_output=True,
                         text=True, env=env, cwd=REPO, timeout=900)
    assert out.returncode == 0, out.stdout[-3000:] + out.stderr[-2000:]
