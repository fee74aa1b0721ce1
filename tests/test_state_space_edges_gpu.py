"""State-space operators on the GPU at the edges of what they take: step logits far from zero, long
sums, one channel, projections of one group, traces.
Definitions in 64 bits: tests/_state_space.py; tolerances: tests/test_state_space_gpu.py."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import _state_space as ref
import scanscam_b200 as sc
from scanscam_b200 import _native
from test_state_space_gpu import BF16, F16, F32, INF, check_conv, ints, make_conv, make_scan, randn, run_scan, scan_roundings

pytestmark = pytest.mark.gpu


# each form of the backward: few channels, more than 32 states, many channels
@pytest.mark.parametrize("n,c,s", [(1, 6, 4), (1, 10, 40), (10, 500, 16)])
@pytest.mark.parametrize("dtype,layout", [(F32, "rows"), (BF16, "cl"), (F16, "cl")])
def test_scan_far_step_logits(n, c, s, dtype, layout):
    """Logits that switch single steps off (every other channel's, so that sums over channels keep their size): the step
    size is zero, or e^-87 = 1.6e-38 where a form keeps the type's smallest normal number, and so is its slope."""
    t = 32
    o = make_scan(dtype, layout, n, c, t, s, bias=False, state=True, seed=31)
    o["dt_bias"] = torch.zeros(c, device="cuda")
    # 88.7 and 89 on either side of where e^-v leaves fp32
    far = torch.tensor([-86, -88, -88.7, -89, -95, -96.5, -99, -110, -500, -1000, -65504, -INF], device="cuda").to(dtype)
    at = torch.arange(len(far), device="cuda") * 2 + 3
    o["dt"] = o["dt"].clone()
    o["dt"][:, ::2, at] = far
    got, gout, gstate = run_scan(o, True)
    want = ref.scan_selective(**o, dt_softplus=True, spans=ref.spans_of(n, t), gout=gout, gstate=gstate)
    assert torch.isfinite(got["gdt"]).all()
    # the slope there, 1.6e-38 at most, times a gradient that is far below 1e6
    assert (got["gdt"][:, ::2, at[1:]].abs() <= 1.7e-32).all()
    got["gdt"] = got["gdt"].clone()
    for v in (got["gdt"], *want["gdt"]):
        v[:, ::2, at.to(v.device)] = 0
    base, channels, steps = scan_roundings({**o, "dt": o["dt"].clamp(min=-80)}, True)
    for k, v in got.items():
        kind = dtype if k in ("out", "gx", "gdt", "gz", "gB", "gC") else F32
        ref.check(v.reshape(want[k][0].shape), want[k], kind, base + channels + steps, k)


def test_scan_gradient_of_decays_over_many_steps():
    """8192 equal terms: added to one running sum each step rounds the same way, up to a quarter of 8192 roundings in all.

    Sums of 32 steps, and of those over 256 tiles, are within 32 + 256.  A term is dt a h dh with a = exp(-1 .. -2): a is
    off by 2.4 roundings and 12 of dt |A|, with a product and a sum 29 a step; h and dh are geometric sums with a ratio of at
    most 0.37, 46 each; three products: 125 with a's own.  In all 413, of which 8192 / 4 would be five times as much."""
    c, t, s = 4736, 8192, 16  # the form for many channels: c * s / 4 of at least 128 lanes an SM
    ones = torch.ones(1, c, t, device="cuda")
    A = -1 - torch.rand(c, s, generator=torch.Generator(device="cuda").manual_seed(32), device="cuda")
    B = torch.ones(1, s, t, device="cuda")
    A.requires_grad_(True)
    (got,) = torch.autograd.grad(sc.scan_selective(ones, ones, A, B, B), A, ones)
    some = slice(0, c, 148)  # a channel of every block of 32 and more
    part = ones[:, some]
    want = ref.scan_selective(part, part, A.detach()[some], B, B, spans=ref.spans_of(1, t), gout=part)
    ref.check(got[some], want["gA"], F32, 413, "gA")


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("states", [8, 16, 32])
def test_scan_form_for_many_channels_is_built(native, dtype, states):
    """Its kernels pass registers between warps and need the compiler to give them a certain number.  Where it did not, the
    other form does the work, slower: its checkpoints lie 32 steps apart at least, this one's 16."""
    n, c, t = 4, 5000, 100
    p = _native.Selective(dtype=getattr(_native, dtype), batch=n, channels=c, steps=t, states=states, groups=1)
    assert native.ssb_selective_checkpoint_bytes(ctypes.byref(p)) == n * -(-t // 16) * c * states * 4


# ---- one channel --------------------------------------------------------------------------------------
@pytest.mark.parametrize("offsets,t", [([0, 1, 1, 3, 40, 40, 300], 300), ([2, 7], 9), ([0, 1], 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["rows", "cl", "strided"])
def test_conv_packed_single_channel(offsets, t, dtype, layout):
    o = make_conv(dtype, layout, 1, 1, t, 4, state=True, count=len(offsets) - 1, seed=33)
    check_conv(o, True, ref.spans_of(1, t, offsets=offsets), offsets=ints(offsets))


@pytest.mark.parametrize("offsets", [None, [0, 5, 5, 64]])
def test_scan_single_channel(offsets):
    spans = ref.spans_of(1, 64, offsets=offsets)
    for layout in ("rows", "cl"):
        o = make_scan(F32, layout, 1, 1, 64, 16, state=True, count=len(spans), seed=34)
        got, gout, gstate = run_scan(o, True, offsets=None if offsets is None else ints(offsets))
        want = ref.scan_selective(**o, dt_softplus=True, spans=spans, gout=gout, gstate=gstate)
        for k, v in got.items():
            ref.check(v, want[k], F32, scan_roundings(o, True)[0] + 65, k)


# ---- projections of one group ---------------------------------------------------------------------------
@pytest.mark.parametrize("m,c,s", [(3, 40, 16), (64, 1024, 16), (5, 33, 7)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_step_two_dimensional_projections(m, c, s, dtype):
    """[M, S], dense or a slice at an odd place of a projection, is [M, 1, S]."""
    x, dt, A = randn(m, c, seed=1, dtype=dtype), randn(m, c, seed=2, dtype=dtype), -torch.exp(randn(c, s, seed=3))
    wide = randn(m, 3 * s, seed=4, dtype=dtype)
    for B, C in ((wide[:, :s].contiguous(), wide[:, s: 2 * s].contiguous()), (wide[:, 1: s + 1], wide[:, 2 * s:])):
        states = [randn(m, c, s, seed=5) for _ in range(2)]
        outs = [sc.scan_selective_step(x, dt, A, b, r, state, dt_softplus=True) for b, r, state in ((B, C, states[0]), (B[:, None], C[:, None], states[1]))]
        assert torch.equal(*outs) and torch.equal(*states)


# ---- traces and forward-mode derivatives ----------------------------------------------------------------
def test_traced_calls_and_tangents():
    o, v = make_scan(F32, "rows", 2, 6, 20, 4, seed=35), make_conv(F32, "rows", 2, 6, 20, 4, seed=36)
    pos, kw = [o[k] for k in ("dt", "A", "B", "C")], {k: o[k] for k in ("D", "z", "dt_bias")}
    states, windows = torch.zeros(2, 6, 4, device="cuda"), torch.zeros(2, 6, 3, device="cuda")
    calls = [(lambda x: sc.scan_selective(x, *pos, **kw, dt_softplus=True), o["x"]), (lambda x: sc.short_conv(x, v["weight"], v["bias"]), v["x"]),
             (lambda x: sc.scan_selective_step(x, o["dt"][..., 0], o["A"], o["B"][..., 0], o["C"][..., 0], states.zero_()), o["x"][..., 0]),
             (lambda x: sc.short_conv_step(x, windows.zero_(), v["weight"]), v["x"][..., 0])]
    with torch.no_grad():
        for call, x in calls:
            traced = torch.jit.trace(call, (torch.zeros_like(x),))
            assert torch.equal(traced(x), call(x))
            with forward_ad.dual_level(), pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(x, torch.ones_like(x)))


def test_traced_calls_have_gradients():
    """Traced without a gradient in sight, replayed with one: the call keeps what its backward needs."""
    o = make_scan(F32, "rows", 2, 6, 40, 4, seed=37)
    pos, gout = [o[k] for k in ("dt", "A", "B", "C")], randn(2, 6, 40, seed=38)
    v = make_conv(F32, "rows", 2, 6, 40, 4, seed=39)
    for call in (lambda x: sc.scan_selective(x, *pos, dt_softplus=True), lambda x: sc.short_conv(x, v["weight"], activation="silu")):
        with torch.no_grad():
            traced = torch.jit.trace(call, (torch.zeros_like(o["x"]),))
        x = o["x"].clone().requires_grad_(True)
        (got,), (want,) = (torch.autograd.grad(f(x), x, gout) for f in (traced, call))
        assert torch.equal(got, want)
