"""State-space operators on the GPU against their definitions in 64 bits (tests/_state_space.py).

Tolerances count roundings of 32 bits, relative to the size of what is added up.  Scan, T steps, S
states: a term of h_t passes at most T decays, each off by 2.4 roundings of the exponential (1.42e-7),
one of the product and one of the sum, some of them once more where runs of steps are composed: 6 T.
The exponents' errors, at most 12 roundings of dt |A| (softplus with its argument, two products), count
with the sum of the exponents that a term has passed: 12 (20 + the largest of one step), terms
beyond e^-20 being smaller than a rounding of the ones before.  The read-out adds S, the gradients of B and C a sum over
C channels, those of A, D and the bias a sum over N T steps; gates, slopes and the rest are within 60.
"""
import pytest
import torch

import _state_space as ref
import scanscam_b200 as sc

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_scan(dtype, layout, n, c, t, s, g=1, D=True, z=True, bias=True, softplus=True, state=False, count=None, seed=0, dt_scale=1.0):
    """Operands as a layer has them; channels last they are slices of wider projections."""
    count = n if count is None else count

    def nct(k):
        if layout == "cl":
            return randn(n, t, c, seed=seed + k, dtype=dtype).mT
        if layout == "slice":  # the second half of [N, T, 2C]
            return randn(n, t, 2 * c, seed=seed + k, dtype=dtype)[:, :, c:].mT
        if layout == "strided":  # neither channels nor steps adjacent
            return randn(n, c, t, 2, seed=seed + k, dtype=dtype)[..., 1]
        return randn(n, c, t, seed=seed + k, dtype=dtype)

    def proj(k):
        if layout in ("cl", "slice"):
            return randn(n, t, 2 * g * s, seed=seed + k, dtype=dtype)[:, :, g * s:].unflatten(2, (g, s)).permute(0, 2, 3, 1)
        return randn(n, g, s, t, seed=seed + k, dtype=dtype)

    o = {"x": nct(1), "dt": nct(2) if softplus else nct(2).abs() * 0.1, "A": -torch.exp(randn(c, s, seed=seed + 3)) * dt_scale, "B": proj(4), "C": proj(5)}
    if D:
        o["D"] = randn(c, seed=seed + 6)
    if z:
        o["z"] = nct(7)
    if bias:
        o["dt_bias"] = randn(c, seed=seed + 8) - 3 if softplus else randn(c, seed=seed + 8).abs() * 0.1
    if state:
        o["state"] = randn(count, c, s, seed=seed + 9)
    return o


def scan_roundings(o, softplus):
    n, c, t = o["x"].shape
    s = o["A"].shape[1]
    raw = o["dt"].detach().double() + (o["dt_bias"].detach().double()[:, None] if "dt_bias" in o else 0)
    dt = ref.softplus(raw) if softplus else raw
    a = o["A"].double()
    step = float((dt.abs().amax((0, 2))[:, None] * a.abs().where(a.isfinite(), torch.zeros_like(a))).max()) if dt.numel() else 0.0
    return 6 * t + s + 12 * (20 + min(step, 90)) + 60, c, n * t  # beyond e^-90 a decay is zero in 32 bits


def run_scan(o, softplus, back="both", seed=50, **more):
    """-> {name: tensor}: out, state and, unless back is None, the gradients."""
    o = {k: v.detach().requires_grad_(back is not None) for k, v in o.items()}
    pos = [o[k] for k in ("x", "dt", "A", "B", "C")]
    kw = {k: v for k, v in o.items() if k not in ("x", "dt", "A", "B", "C")}
    out, state = sc.scan_selective(*pos, **kw, dt_softplus=softplus, return_state=True, **more)
    r = {"out": out.detach(), "state": state.detach()}
    gout = gstate = None
    if back is not None:
        gout = randn(*out.shape, seed=seed, dtype=out.dtype) if back in ("both", "out") else None
        gstate = randn(*state.shape, seed=seed + 1) if back in ("both", "state") else None
        pairs = [(a, b) for a, b in ((out, gout), (state, gstate)) if b is not None]
        grads = torch.autograd.grad([a for a, _ in pairs], list(o.values()), [b for _, b in pairs])
        r |= {"g" + k: v for k, v in zip(o, grads)}
    return r, gout, gstate


def check_scan(o, softplus, spans, back="both", **more):
    got, gout, gstate = run_scan(o, softplus, back, **more)
    want = ref.scan_selective(**o, dt_softplus=softplus, spans=spans, gout=gout, gstate=gstate)
    base, channels, steps = scan_roundings(o, softplus)
    kind = {k: o["x"].dtype for k in ("out", "gx", "gdt", "gz", "gB", "gC")}
    extra = {"gB": channels, "gC": channels, "gA": steps, "gD": steps, "gdt_bias": steps}
    for k, v in got.items():
        ref.check(v.reshape(want[k][0].shape), want[k], kind.get(k, F32), base + extra.get(k, 0), k)
    assert got["out"].stride(1) == 1 or o["x"].stride(1) != 1  # the layout of x
    return got


# ---- selective scan, whole sequences ------------------------------------------------------------
SHAPES = [  # n, c, t, s, g: one and few steps, tiles of 32 to 256 steps and one more or less, odd channels, one to 256 states
    (1, 1, 1, 1, 1), (2, 3, 2, 5, 1), (1, 2, 7, 16, 1), (3, 17, 8, 4, 1), (1, 64, 9, 16, 1), (2, 34, 31, 7, 2), (1, 130, 33, 16, 1),
    (2, 24, 64, 33, 3), (1, 8, 65, 64, 1), (1, 16, 255, 16, 4), (1, 6, 257, 16, 1), (2, 5, 300, 11, 1), (1, 4, 40, 256, 1), (1, 20, 130, 40, 2),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype,layout", [(F32, "rows"), (BF16, "cl"), (F16, "slice"), (F32, "strided"), (BF16, "rows"), (F32, "cl")])
def test_scan_and_gradients(shape, dtype, layout):
    n, c, t, s, g = shape
    o = make_scan(dtype, layout, n, c, t, s, g, state=c % 2 == 0, seed=sum(shape))
    check_scan(o, True, ref.spans_of(n, t))


@pytest.mark.parametrize("missing", ["D", "z", "bias", "softplus", "all"])
@pytest.mark.parametrize("layout", ["rows", "cl"])
def test_scan_without_optional_operands(missing, layout):
    names = ("D", "z", "bias", "softplus") if missing == "all" else (missing,)
    have = {k: k not in names for k in ("D", "z", "bias", "softplus")}
    o = make_scan(F32, layout, 2, 10, 50, 16, seed=3, **have)
    check_scan(o, have["softplus"], ref.spans_of(2, 50))


@pytest.mark.parametrize("back", ["out", "state"])
def test_scan_gradients_of_one_result_alone(back):
    o = make_scan(BF16, "cl", 2, 18, 70, 16, state=True, seed=4)
    check_scan(o, True, ref.spans_of(2, 70), back=back)


@pytest.mark.parametrize("n,c,t", [(4, 600, 40), (2, 1300, 70), (9, 2050, 36)])
def test_scan_with_many_channels(n, c, t):
    """Enough channel blocks for each split of the warps between time and channels."""
    o = make_scan(BF16, "cl", n, c, t, 4, seed=5)
    check_scan(o, True, ref.spans_of(n, t))


# The forms that are chosen where channels and sequences abound: 8 states a lane in the forward (from 37 888 channels
# x sequences x eighths of the states up), lanes across states in the backward (from 18 944 x quarters, up to 32 states).
MANY = [("rows", F32, 10, 520, 33, 16, 2), ("cl", BF16, 10, 520, 70, 16, 1), ("slice", F16, 5, 1000, 40, 13, 1), ("cl", F32, 6, 800, 31, 16, 1),
        ("strided", BF16, 10, 501, 20, 16, 1), ("cl", BF16, 3, 802, 48, 32, 2), ("cl", F32, 12, 800, 17, 7, 1), ("rows", BF16, 40, 512, 64, 16, 1),
        ("cl", F16, 38, 513, 9, 16, 3), ("cl", BF16, 20, 500, 12, 32, 1), ("cl", F32, 5, 1000, 1, 16, 1), ("rows", F16, 12, 808, 40, 8, 1)]


@pytest.mark.parametrize("layout,dtype,n,c,t,s,g", MANY, ids=str)
def test_scan_with_many_channels_and_sequences(layout, dtype, n, c, t, s, g):
    o = make_scan(dtype, layout, n, c, t, s, g, state=True, seed=n + s)
    check_scan(o, True, ref.spans_of(n, t))


@pytest.mark.parametrize("missing", ["D", "z", "bias", "softplus", "all"])
def test_scan_with_many_channels_without_optional_operands(missing):
    names = ("D", "z", "bias", "softplus") if missing == "all" else (missing,)
    have = {k: k not in names for k in ("D", "z", "bias", "softplus")}
    o = make_scan(F32, "cl", 10, 500, 35, 16, seed=23, **have)
    check_scan(o, have["softplus"], ref.spans_of(10, 35))


@pytest.mark.parametrize("dtype,layout", [(F32, "cl"), (BF16, "cl"), (F16, "rows")])
def test_scan_packed_with_many_sequences(dtype, layout):
    """Empty ones, single steps, bounds at and off the runs of 16 and the tiles of 32 steps; steps that belong to none."""
    offsets = [2, 2, 3, 19, 35, 35, 67, 99, 100, 116, 133, 133, 150, 151, 152, 168, 200, 231, 264, 264, 265, 281, 290, 291, 300]
    t, count = 303, len(offsets) - 1
    o = make_scan(dtype, layout, 1, 212, t, 16, 2, state=True, count=count, seed=24)
    clean = {k: v.clone() for k, v in o.items()}
    for k in ("x", "dt", "z", "B", "C"):
        o[k] = o[k].clone()
        o[k][..., : offsets[0]] = NAN
        o[k][..., offsets[-1]:] = INF
    got, gout, gstate = run_scan(o, True, offsets=ints(offsets))
    want = ref.scan_selective(**clean, dt_softplus=True, spans=ref.spans_of(1, t, offsets=offsets), gout=gout, gstate=gstate)
    base, channels, steps = scan_roundings(clean, True)
    for k, v in got.items():
        ref.check(v, want[k], dtype if k in ("out", "gx", "gdt", "gz", "gB", "gC") else F32, base + channels + steps, k)


def test_scan_padded_batch_of_many_channels():
    lengths, t = [0, 1, 16, 17, 32, 33, 40, 47, 48, 50], 50
    o = make_scan(F32, "cl", 10, 500, t, 16, state=True, seed=25)
    clean = {k: v.clone() for k, v in o.items()}
    for k in ("x", "dt", "z", "B", "C"):
        o[k] = o[k].clone()
        for i, size in enumerate(lengths):
            o[k][i, ..., size:] = NAN if i % 2 else -INF
    got, gout, gstate = run_scan(o, True, lengths=ints(lengths))
    want = ref.scan_selective(**clean, dt_softplus=True, spans=ref.spans_of(10, t, lengths), gout=gout, gstate=gstate)
    base, channels, steps = scan_roundings(clean, True)
    for k, v in got.items():
        ref.check(v, want[k], F32, base + channels + steps, k)


def test_scan_of_many_channels_is_repeatable():
    o = make_scan(BF16, "cl", 10, 520, 150, 16, seed=26)
    first, _, _ = run_scan(o, True)
    for _ in range(3):
        again, _, _ = run_scan(o, True)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_scan_more_sequences_than_a_block_of_sums():
    """The CTAs of the backward take several sequences each."""
    o = make_scan(F32, "cl", 90, 260, 18, 16, state=True, seed=27)
    check_scan(o, True, ref.spans_of(90, 18))


@pytest.mark.parametrize("dtype,layout", [(F32, "cl"), (BF16, "cl"), (F32, "rows"), (F16, "rows")])
@pytest.mark.parametrize("offsets,t", [([0, 5, 5, 6, 70, 70, 135], 135), ([3, 3, 40, 41, 110], 120), ([0, 0], 9), ([0, 64, 128, 192], 192), ([7, 7, 7], 20)])
def test_scan_packed(dtype, layout, offsets, t):
    """Empty and single-step sequences, tile bounds, steps before the first and behind the last; what lies there is never used."""
    count = len(offsets) - 1
    o = make_scan(dtype, layout, 1, 14, t, 16, 2, state=True, count=count, seed=6)
    clean = {k: v.clone() for k, v in o.items()}
    for k in ("x", "dt", "z", "B", "C"):
        o[k] = o[k].clone()
        o[k][..., : offsets[0]] = NAN
        o[k][..., offsets[-1]:] = INF
    spans = ref.spans_of(1, t, offsets=offsets)
    got, gout, gstate = run_scan(o, True, offsets=ints(offsets))
    want = ref.scan_selective(**clean, dt_softplus=True, spans=spans, gout=gout, gstate=gstate)
    base, channels, steps = scan_roundings(clean, True)
    for k, v in got.items():
        ref.check(v, want[k], dtype if k in ("out", "gx", "gdt", "gz", "gB", "gC") else F32, base + channels + steps, k)
    for k in ("out", "gx", "gdt", "gz", "gB", "gC"):
        assert (got[k][..., : offsets[0]] == 0).all() and (got[k][..., offsets[-1]:] == 0).all(), k


@pytest.mark.parametrize("layout", ["rows", "cl"])
def test_scan_padded_batch(layout):
    lengths, t = [0, 1, 33, 64, 70], 70
    o = make_scan(F32, layout, 5, 12, t, 16, state=True, seed=7)
    clean = {k: v.clone() for k, v in o.items()}
    for k in ("x", "dt", "z", "B", "C"):
        o[k] = o[k].clone()
        for i, size in enumerate(lengths):
            o[k][i, ..., size:] = NAN if i % 2 else -INF
    got, gout, gstate = run_scan(o, True, lengths=ints(lengths))
    want = ref.scan_selective(**clean, dt_softplus=True, spans=ref.spans_of(5, t, lengths), gout=gout, gstate=gstate)
    base, channels, steps = scan_roundings(clean, True)
    for k, v in got.items():
        ref.check(v, want[k], F32, base + channels + steps, k)
    assert torch.equal(got["state"][0], o["state"][0])


def test_scan_sequences_do_not_see_one_another():
    """NaN in one packed sequence stays there."""
    o = make_scan(F32, "cl", 1, 16, 90, 16, seed=8)
    offsets = ints([0, 30, 60, 90])
    clean, _, _ = run_scan(o, True, offsets=offsets)
    o["x"][..., 30:60] = NAN
    got, _, _ = run_scan(o, True, offsets=offsets)
    for k in ("out", "gx", "gdt", "gz", "gB", "gC"):
        assert torch.equal(got[k][..., :30], clean[k][..., :30]) and torch.equal(got[k][..., 60:], clean[k][..., 60:]), k
    assert torch.equal(got["state"][[0, 2]], clean["state"][[0, 2]])


def test_scan_empty():
    for n, c, t in ((0, 8, 5), (2, 8, 0), (2, 0, 5)):
        o = make_scan(F32, "rows", n, c, t, 4, state=True, seed=9)
        got, _, _ = run_scan(o, True)
        assert got["out"].shape == (n, c, t) and torch.equal(got["state"], o["state"])
        assert all(got["g" + k].shape == v.shape for k, v in o.items())
        assert (got["gA"] == 0).all()


@pytest.mark.parametrize("layout", ["rows", "cl"])
def test_scan_extreme_decays(layout):
    """Steps of zero, decays of one, entries of A that forget at once (-inf, -1e30) and a positive one."""
    o = make_scan(F32, layout, 1, 8, 40, 6, softplus=False, bias=False, seed=10)
    o["dt"][..., ::3] = 0
    o["A"][:, 0] = 0
    o["A"][:, 1] = -1e30
    o["A"][:, 2] = 0.5
    check_scan(o, False, ref.spans_of(1, 40))
    o["A"][:, 1] = -INF
    o["dt"] = o["dt"].abs() + 0.01  # exp(0 * -inf) has no value
    got, _, _ = run_scan(o, False, back=None)
    o["A"][:, 1] = -1e30
    want, _, _ = run_scan(o, False, back=None)
    assert torch.equal(got["out"], want["out"])


@pytest.mark.parametrize("n,c,s", [(1, 10, 16), (10, 500, 16), (1, 6, 100)])
def test_scan_steps_of_zero_change_nothing(n, c, s):
    """exp(0 A) is 1 to the last bit: the state comes out as it went in, its gradient too."""
    o = make_scan(F32, "cl", n, c, 45, s, softplus=False, bias=False, state=True, seed=28)
    o["dt"] = torch.zeros_like(o["dt"])
    got, _, gstate = run_scan(o, False, back="state")
    assert torch.equal(got["state"], o["state"]) and torch.equal(got["gstate"], gstate)
    state = o["state"].clone()
    sc.scan_selective_step(*(o[k][..., 0] if k != "A" else o[k] for k in ("x", "dt", "A", "B", "C")), state)
    assert torch.equal(state, o["state"])


def test_scan_extreme_step_logits():
    """softplus far from zero on both sides, and gates that are shut or wide open."""
    o = make_scan(F32, "rows", 1, 6, 32, 4, bias=False, seed=11, dt_scale=1e-3)
    o["dt"][0, :, 0], o["dt"][0, :, 1], o["dt"][0, :, 2], o["dt"][0, :, 3] = -80, 80, -20, 30
    o["z"][0, :, 4], o["z"][0, :, 5], o["z"][0, :, 6] = -200, 200, 0
    check_scan(o, True, ref.spans_of(1, 32))


def test_scan_in_pieces_is_the_whole():
    """The state carried over a cut, its gradient too, for cuts anywhere in a tile."""
    o = make_scan(F32, "cl", 2, 20, 150, 16, seed=12)
    whole, gout, gstate = run_scan(o, True)
    for cut in (1, 64, 77, 149):
        leaves = {k: v.detach().requires_grad_(True) for k, v in o.items()}
        state, outs = None, []
        for a, b in ((0, cut), (cut, 150)):
            part = {k: v[..., a:b] if k in ("x", "dt", "z", "B", "C") else v for k, v in leaves.items()}
            pos = [part.pop(k) for k in ("x", "dt", "A", "B", "C")]
            out, state = sc.scan_selective(*pos, **part, dt_softplus=True, state=state, return_state=True)
            outs.append(out)
        grads = torch.autograd.grad([torch.cat(outs, 2), state], list(leaves.values()), [gout, gstate])
        want = ref.scan_selective(**o, dt_softplus=True, spans=ref.spans_of(2, 150), gout=gout, gstate=gstate)
        base, channels, steps = scan_roundings(o, True)
        ref.check(torch.cat(outs, 2), want["out"], F32, base, f"out cut at {cut}")
        ref.check(state, want["state"], F32, base, f"state cut at {cut}")
        for k, v in zip(leaves, grads):
            ref.check(v, want["g" + k], F32, base + channels + steps + 2, f"g{k} cut at {cut}")


def test_scan_broadcast_operands():
    """Expanded B, C (shared by the batch) and dt (shared by channels): gradients are summed over what shares them."""
    n, c, t, s = 3, 12, 40, 8
    o = make_scan(F32, "rows", n, c, t, s, seed=13)
    small = {"B": randn(1, 1, s, t, seed=90), "C": randn(1, 1, s, t, seed=91), "dt": randn(n, 1, t, seed=92)}
    leaves = {k: v.requires_grad_(True) for k, v in small.items()}
    wide = {**o, "B": leaves["B"].expand(n, 1, s, t), "C": leaves["C"].expand(n, 1, s, t), "dt": leaves["dt"].expand(n, c, t)}
    kw = {k: v for k, v in wide.items() if k not in ("x", "dt", "A", "B", "C")}
    out = sc.scan_selective(*(wide[k] for k in ("x", "dt", "A", "B", "C")), **kw, dt_softplus=True)
    gout = randn(n, c, t, seed=93)
    grads = torch.autograd.grad(out, list(leaves.values()), gout)
    want = ref.scan_selective(**wide, dt_softplus=True, spans=ref.spans_of(n, t), gout=gout)
    base, channels, steps = scan_roundings(wide, True)
    for (k, leaf), got in zip(leaves.items(), grads):
        axis = 1 if k == "dt" else 0
        ref.check(got, tuple(v.sum(axis, keepdim=True) for v in want["g" + k]), F32, base + channels + n, "g" + k)


def test_scan_three_dimensional_projections():
    o = make_scan(F32, "rows", 2, 6, 20, 4, seed=14)
    a = sc.scan_selective(o["x"], o["dt"], o["A"], o["B"], o["C"])
    b = sc.scan_selective(o["x"], o["dt"], o["A"], o["B"][:, 0], o["C"][:, 0])
    assert torch.equal(a, b)


def test_scan_long_sequence():
    """20 000 steps, few channels: slow decays remember thousands of steps."""
    n, c, t, s = 1, 4, 20000, 4
    o = make_scan(F32, "rows", n, c, t, s, seed=15, dt_scale=0.01)
    got, _, _ = run_scan(o, True, back=None)
    want = ref.scan_selective(**o, dt_softplus=True, spans=ref.spans_of(n, t))
    base, _, _ = scan_roundings(o, True)
    ref.check(got["out"], want["out"], F32, base, "out")
    ref.check(got["state"], want["state"], F32, base, "state")


def test_scan_beyond_32_bit_offsets():
    """More than 2^31 elements: the last steps equal those of the same operands cut out, carried state and all."""
    c, t, s, tail = 4096, 540000, 4, 100
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 40 GB")
    x = torch.empty(1, t, c, device="cuda", dtype=BF16).normal_(generator=gen(16)).mT
    B = randn(1, t, s, seed=17, dtype=BF16).mT
    A, bias = -torch.exp(randn(c, s, seed=18)), randn(c, seed=19) - 3
    kw = dict(dt_bias=bias, dt_softplus=True, return_state=True)
    out, state = sc.scan_selective(x, x, A, B, B, z=x, **kw)
    _, mid = sc.scan_selective(x[..., :-tail], x[..., :-tail], A, B[..., :-tail], B[..., :-tail], **kw)
    end, last = sc.scan_selective(x[..., -tail:], x[..., -tail:], A, B[..., -tail:], B[..., -tail:], z=x[..., -tail:], state=mid, **kw)
    # the two cut the last steps into tiles at other places: 6 roundings a step and one to bf16 apart
    off = (out[..., -tail:].float() - end.float()).abs()
    assert (off <= 2 * 2.0 ** -8 * end.float().abs() + 6 * tail * 2.0 ** -24 * 100).all()
    assert ((state - last).abs() <= 6 * tail * 2.0 ** -24 * (last.abs() + 10)).all()
    del out, state, end, x
    torch.cuda.empty_cache()


def test_scan_backward_is_repeatable():
    o = make_scan(BF16, "cl", 3, 300, 200, 16, seed=20)
    first, _, _ = run_scan(o, True)
    for _ in range(3):
        again, _, _ = run_scan(o, True)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_scan_second_derivative_is_refused():
    o = make_scan(F32, "rows", 1, 4, 8, 2, z=False, seed=21)
    x = o["x"].requires_grad_(True)
    out = sc.scan_selective(x, o["dt"], o["A"], o["B"], o["C"])
    (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---- short convolution -----------------------------------------------------------------------------
def make_conv(dtype, layout, n, c, t, w, bias=True, state=False, count=None, seed=0, weight_dtype=None):
    wd = weight_dtype or dtype
    x = {"cl": lambda: randn(n, t, c, seed=seed, dtype=dtype).mT, "slice": lambda: randn(n, t, 3 * c, seed=seed, dtype=dtype)[:, :, c: 2 * c].mT,
         "rows": lambda: randn(n, c, t, seed=seed, dtype=dtype), "strided": lambda: randn(n, c, t, 2, seed=seed, dtype=dtype)[..., 0]}[layout]()
    o = {"x": x, "weight": randn(c, w, seed=seed + 1, dtype=wd)}
    if bias:
        o["bias"] = randn(c, seed=seed + 2, dtype=wd)
    if state:
        o["state"] = randn(n if count is None else count, c, w - 1, seed=seed + 3, dtype=dtype)
    return o


def run_conv(o, silu, back="both", **more):
    o = {k: v.detach().requires_grad_(back is not None) for k, v in o.items()}
    out, state = sc.short_conv(**o, activation="silu" if silu else None, return_state=True, **more)
    r = {"out": out.detach(), "state": state.detach()}
    gout = gstate = None
    if back is not None:
        gout = randn(*out.shape, seed=60, dtype=out.dtype) if back in ("both", "out") else None
        gstate = randn(*state.shape, seed=61, dtype=out.dtype) if back in ("both", "state") else None
        pairs = [(a, b) for a, b in ((out, gout), (state, gstate)) if b is not None]
        r |= {"g" + k: v for k, v in zip(o, torch.autograd.grad([a for a, _ in pairs], list(o.values()), [b for _, b in pairs]))}
    return r, gout, gstate


def check_conv(o, silu, spans, back="both", clean=None, **more):
    """Roundings: W products and sums, 4 of the logistic with its argument (which counts with the sum's size), and what the
    gradients add: W, and a sum over N T steps for the taps."""
    got, gout, gstate = run_conv(o, silu, back, **more)
    want = ref.short_conv(**(clean or o), silu=silu, spans=spans, gout=gout, gstate=gstate)
    n, _, t = o["x"].shape
    for k, v in got.items():
        kind = o["weight"].dtype if k in ("gweight", "gbias") else o["x"].dtype
        ref.check(v, want[k], kind, 24 + (n * t if k in ("gweight", "gbias") else 0), k)
    return got


@pytest.mark.parametrize("n,c,t,w", [(1, 1, 1, 4), (2, 3, 2, 3), (1, 4, 3, 4), (3, 36, 8, 2), (1, 130, 31, 4), (2, 64, 33, 3), (1, 12, 255, 4),
                                     (2, 515, 65, 4), (1, 8, 1030, 3), (1, 260, 300, 2), (7, 2052, 600, 4), (60, 1028, 40, 3)])
@pytest.mark.parametrize("dtype,layout", [(F32, "rows"), (BF16, "cl"), (F16, "slice"), (F32, "strided"), (F32, "cl"), (BF16, "rows")])
def test_conv_and_gradients(n, c, t, w, dtype, layout):
    check_conv(make_conv(dtype, layout, n, c, t, w, state=t % 2 == 1, bias=c != 64, seed=n + c + t), t != 31, ref.spans_of(n, t))


@pytest.mark.parametrize("back", ["out", "state"])
@pytest.mark.parametrize("layout", ["rows", "cl"])
def test_conv_gradients_of_one_result_alone(back, layout):
    check_conv(make_conv(F32, layout, 2, 12, 2, 4, state=True, seed=1), True, ref.spans_of(2, 2), back=back)


def test_conv_float32_taps_on_16_bit_tensors():
    got = check_conv(make_conv(BF16, "cl", 2, 24, 40, 4, seed=2, weight_dtype=F32), True, ref.spans_of(2, 40))
    assert got["gweight"].dtype == F32 and got["gbias"].dtype == F32


@pytest.mark.parametrize("dtype,layout", [(F32, "cl"), (BF16, "slice"), (F32, "rows"), (F16, "strided")])
@pytest.mark.parametrize("offsets,t", [([0, 1, 1, 3, 40, 40, 300], 300), ([5, 5, 7, 33, 64], 80), ([0, 0], 9), ([9, 9, 9], 20), ([0, 32, 64, 256], 256)])
def test_conv_packed(dtype, layout, offsets, t):
    count = len(offsets) - 1
    o = make_conv(dtype, layout, 1, 20, t, 4, state=True, count=count, seed=3)
    clean = {k: v.clone() for k, v in o.items()}
    o["x"] = o["x"].clone()
    o["x"][..., : offsets[0]], o["x"][..., offsets[-1]:] = NAN, INF
    got = check_conv(o, True, ref.spans_of(1, t, offsets=offsets), clean=clean, offsets=ints(offsets))
    for k in ("out", "gx"):
        assert (got[k][..., : offsets[0]] == 0).all() and (got[k][..., offsets[-1]:] == 0).all()


def test_conv_many_packed_sequences():
    """More sequences than the search looks at in one round, some of them empty."""
    g = torch.Generator().manual_seed(4)
    cuts = torch.randint(0, 700, (1500,), generator=g).sort().values.tolist()
    offsets = [0, *cuts, 700]
    o = make_conv(F32, "cl", 1, 8, 700, 4, state=True, count=len(offsets) - 1, seed=4)
    check_conv(o, True, ref.spans_of(1, 700, offsets=offsets), offsets=ints(offsets))


@pytest.mark.parametrize("layout", ["rows", "cl"])
def test_conv_padded_batch(layout):
    lengths, t = [0, 1, 2, 33, 40], 40
    o = make_conv(F32, layout, 5, 12, t, 4, state=True, seed=5)
    clean = {k: v.clone() for k, v in o.items()}
    for i, size in enumerate(lengths):
        o["x"][i, :, size:] = NAN if i % 2 else INF
    check_conv(o, True, ref.spans_of(5, t, lengths), clean=clean, lengths=ints(lengths))


def test_conv_empty():
    for n, c, t in ((0, 8, 5), (2, 8, 0), (2, 0, 5)):
        for layout in ("rows", "cl"):
            o = make_conv(F32, layout, n, c, t, 4, state=True, seed=6)
            got, _, gstate = run_conv(o, True)
            assert got["out"].shape == (n, c, t) and torch.equal(got["state"], o["state"])
            assert (got["gweight"] == 0).all() and (got["gbias"] == 0).all()
            if t == 0:
                assert torch.equal(got["gstate"], gstate)


def test_conv_backward_is_repeatable():
    o = make_conv(BF16, "cl", 3, 300, 500, 4, seed=7)
    first, _, _ = run_conv(o, True)
    again, _, _ = run_conv(o, True)
    assert all(torch.equal(first[k], again[k]) for k in first)


# ---- single tokens -----------------------------------------------------------------------------------
def step_reference(x, dt, A, B, C, state, D, z, bias, softplus, slots):
    """Entry after entry in 64 bits: (out, state) as (value, size)."""
    x, dt, A, B, C, state = (v.double().cpu() for v in (x, dt, A, B, C, state))
    if B.dim() == 2:
        B, C = B[:, None], C[:, None]
    of = torch.arange(x.shape[1]) // (x.shape[1] // B.shape[1])
    out, out_m, state_m = torch.zeros_like(x), torch.zeros_like(x), state.abs()
    for m, s in enumerate(slots):
        if not 0 <= s < state.shape[0]:
            continue
        d = dt[m] + (bias.double().cpu() if bias is not None else 0)
        d = ref.softplus(d) if softplus else d
        a, u = torch.exp(d[:, None] * A), (d * x[m])[:, None] * B[m][of]
        state[s], state_m[s] = a * state[s] + u, a * state_m[s] + u.abs()
        y, ym = (state[s] * C[m][of]).sum(1), (state_m[s] * C[m][of].abs()).sum(1)
        if D is not None:
            y, ym = y + D.double().cpu() * x[m], ym + (D.double().cpu() * x[m]).abs()
        gate = ref._silu(z[m].double().cpu()) if z is not None else 1.0
        out[m], out_m[m] = y * gate, ym * abs(gate)
    return (out, out_m), (state, state_m)


@pytest.mark.parametrize("m,c,s,g,pool,slots", [
    (1, 1, 1, 1, 1, None), (1, 2048, 16, 1, 1, None), (3, 33, 7, 3, 3, None), (5, 64, 16, 2, 9, [8, -1, 0, 3, 9]), (4, 40, 64, 1, 6, [2, 2, 2, 2]),
    (6, 17, 256, 1, 4, [0, 3, 0, -5, 3, 1]), (2, 10, 33, 5, 2, [1, 0]), (300, 20, 4, 1, 40, [i * 7 % 43 for i in range(300)]), (0, 8, 4, 1, 3, []),
    (2, 8, 4, 1, 0, [0, -1]), (40, 1001, 16, 1, 40, None), (64, 520, 16, 2, 70, [(i * 11) % 71 - 1 for i in range(64)]), (300, 66, 64, 3, 300, None),
    (300, 130, 13, 1, 40, [i * 7 % 43 for i in range(300)])])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_step(m, c, s, g, pool, slots, dtype):
    o = {"x": randn(m, c, seed=1, dtype=dtype), "dt": randn(m, 2 * c, seed=2, dtype=dtype)[:, c:], "A": -torch.exp(randn(c, s, seed=3)),
         "B": randn(m, 2 * g * s, seed=4, dtype=dtype)[:, g * s:].unflatten(1, (g, s)), "C": randn(m, g, s, seed=5, dtype=dtype)}
    state, D, z, bias = randn(pool, c, s, seed=6), randn(c, seed=7), randn(m, c, seed=8, dtype=dtype), randn(c, seed=9) - 2
    which = list(range(m)) if slots is None else slots
    want, want_state = step_reference(**o, state=state, D=D, z=z, bias=bias, softplus=True, slots=which)
    out = sc.scan_selective_step(**o, state=state, D=D, z=z, dt_bias=bias, dt_softplus=True, slots=None if slots is None else ints(slots))
    # as for the scan, over the tokens of one slot: 6 each, S for the read-out, 12 per unit of dt |A|, 60 for the rest
    most = max([which.count(v) for v in set(which)], default=0)
    d = ref.softplus(o["dt"].double() + bias) if m else torch.zeros(1, c)
    roundings = 6 * most + s + 60 + 12 * float((d.amax(0)[:, None].cpu() * o["A"].abs().double().cpu()).max()) * max(most, 1)
    ref.check(out, want, dtype, roundings, "out")
    ref.check(state, want_state, F32, roundings, "state")
    touched = {v for v in which if 0 <= v < pool}
    rest = [v for v in range(pool) if v not in touched]
    assert torch.equal(state[rest], randn(pool, c, s, seed=6)[rest])


def test_scan_step_without_optional_operands():
    m, c, s = 3, 20, 5
    o = {"x": randn(m, c, seed=1), "dt": randn(m, c, seed=2).abs() * 0.1, "A": -torch.exp(randn(c, s, seed=3)), "B": randn(m, s, seed=4), "C": randn(m, s, seed=5)}
    state = randn(m, c, s, seed=6)
    want, want_state = step_reference(**o, state=state, D=None, z=None, bias=None, softplus=False, slots=range(m))
    ref.check(sc.scan_selective_step(**o, state=state), want, F32, s + 100, "out")
    ref.check(state, want_state, F32, s + 100, "state")


@pytest.mark.parametrize("m,c,w,pool,slots", [(1, 1, 4, 1, None), (1, 2048, 4, 1, None), (3, 33, 3, 3, None), (5, 64, 2, 9, [8, -1, 0, 3, 9]),
                                              (4, 40, 4, 6, [2, 2, 2, 2]), (6, 17, 4, 4, [0, 3, 0, -5, 3, 1]), (0, 8, 4, 3, []), (2, 8, 4, 0, [0, -1]),
                                              (300, 24, 4, 40, [i * 7 % 43 for i in range(300)])])
@pytest.mark.parametrize("dtype,weight", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("silu,bias", [(True, True), (False, False)])
def test_conv_step(m, c, w, pool, slots, dtype, weight, silu, bias):
    x, taps = randn(m, 2 * c, seed=1, dtype=dtype)[:, c:], randn(c, w, seed=2, dtype=weight)
    b, state = (randn(c, seed=3, dtype=weight) if bias else None), randn(pool, c, w - 1, seed=4, dtype=dtype)
    held, out, size = state.double().cpu(), torch.zeros(m, c, dtype=torch.float64), torch.zeros(m, c, dtype=torch.float64)
    for i, s in enumerate(range(m) if slots is None else slots):
        if 0 <= s < pool:
            seen = torch.cat([held[s], x[i].double().cpu()[:, None]], 1)
            v = (seen * taps.double().cpu()).sum(1) + (b.double().cpu() if bias else 0)
            out[i], size[i] = (ref._silu(v) if silu else v), 1.1 * ((seen * taps.double().cpu()).abs().sum(1) + (b.abs().double().cpu() if bias else 0))
            held[s] = seen[:, 1:]
    got = sc.short_conv_step(x, state, taps, b, activation="silu" if silu else None, slots=None if slots is None else ints(slots))
    ref.check(got, (out, size), dtype, 24, "out")
    assert torch.equal(state.double().cpu(), held)


def test_step_marks_its_state_as_written():
    state = torch.zeros(2, 8, 4, device="cuda")
    before = state._version
    sc.scan_selective_step(randn(2, 8, seed=1), randn(2, 8, seed=2), -torch.ones(8, 4, device="cuda"), randn(2, 4, seed=3), randn(2, 4, seed=4), state)
    assert state._version > before


# ---- as a layer uses them ------------------------------------------------------------------------------
class Layer:
    """Convolution and scan of one layer; dt, B and C come from the convolution's output through a small projection."""

    def __init__(self, c, s, w, dtype, seed):
        self.taps, self.bias = randn(c, w, seed=seed, dtype=dtype) / 2, randn(c, seed=seed + 1, dtype=dtype) / 2
        self.A, self.D, self.dt_bias = -torch.exp(randn(c, s, seed=seed + 2)), randn(c, seed=seed + 3), randn(c, seed=seed + 4) - 3
        self.proj = (randn(c + 2 * s, c, seed=seed + 5) / c ** 0.5).to(dtype)
        self.c, self.s = c, s

    def split(self, u):  # u [..., C] -> dt, B, C
        return (u @ self.proj.T).split([self.c, self.s, self.s], -1)

    def prompt(self, x, z, window=None, state=None, **seqs):
        u, window = sc.short_conv(x, self.taps, self.bias, activation="silu", state=window, return_state=True, **seqs)
        dt, B, C = (v.mT for v in self.split(u.mT))
        y, state = sc.scan_selective(u, dt, self.A, B, C, D=self.D, z=z, dt_bias=self.dt_bias, dt_softplus=True, state=state,
                                     return_state=True, **seqs)
        return y, window, state

    def token(self, x, z, windows, states, slots=None):
        u = sc.short_conv_step(x, windows, self.taps, self.bias, activation="silu", slots=slots)
        dt, B, C = self.split(u)
        return sc.scan_selective_step(u, dt, self.A, B, C, states, D=self.D, z=z, dt_bias=self.dt_bias, dt_softplus=True, slots=slots)


def test_prompts_then_tokens_are_the_whole_sequences():
    """Packed prompts fill a pool; tokens of all sequences follow, one batch at a time; a long run over each whole sequence agrees."""
    c, s, prompts, tokens = 24, 16, [1, 37, 64, 5], 6
    layer = Layer(c, s, 4, F32, 30)
    n = len(prompts)
    x = [randn(1, p + tokens, c, seed=40 + i).mT for i, p in enumerate(prompts)]
    z = [randn(1, p + tokens, c, seed=50 + i).mT for i, p in enumerate(prompts)]
    offsets = ints([0, *torch.tensor(prompts).cumsum(0).tolist()])
    with torch.no_grad():
        y, window, state = layer.prompt(torch.cat([v[..., :p] for v, p in zip(x, prompts)], 2), torch.cat([v[..., :p] for v, p in zip(z, prompts)], 2),
                                        offsets=offsets)
        windows, states = torch.zeros(9, c, 3, device="cuda"), torch.zeros(9, c, s, device="cuda")
        slots = ints([7, 2, 4, 0])
        windows[slots.long()], states[slots.long()] = window, state
        outs = [layer.token(torch.stack([v[0, :, p + k] for v, p in zip(x, prompts)]), torch.stack([v[0, :, p + k] for v, p in zip(z, prompts)]),
                            windows, states, slots) for k in range(tokens)]
        for i, p in enumerate(prompts):
            whole, window, state = layer.prompt(x[i], z[i])
            a, b = int(offsets[i]), int(offsets[i + 1])
            # both sides differ by roundings of 70 steps; the products of the projection feed them back: three decimal digits to spare
            for got, want in [(y[0, :, a:b], whole[0, :, :p]), (torch.stack([o[i] for o in outs], 1), whole[0, :, p:]), (states[slots[i].long()], state[0])]:
                assert ((got - want).abs() <= 1e-4 * (1 + want.abs().max())).all()
            assert torch.equal(windows[slots[i].long()], window[0])


def test_layer_gradients_against_differences():
    """The gradient of a whole layer along random directions, against central differences of its own output in 32 bits."""
    c, s, t = 12, 8, 40
    layer = Layer(c, s, 4, F32, 60)
    names = ["taps", "bias", "A", "D", "dt_bias", "proj"]
    x, z, way = randn(2, c, t, seed=61), randn(2, c, t, seed=62), randn(2, c, t, seed=63)
    base = {k: getattr(layer, k).clone() for k in names}

    def loss():
        return (layer.prompt(x, z)[0].double() * way).sum()

    for k in names:
        setattr(layer, k, base[k].clone().requires_grad_(True))
    grads = dict(zip(names, torch.autograd.grad(loss(), [getattr(layer, k) for k in names])))
    for i, k in enumerate(names):
        d = randn(*base[k].shape, seed=70 + i)
        step = 1e-2 / float(d.norm())
        with torch.no_grad():
            at = []
            for sign in (1, -1):
                for j in names:
                    setattr(layer, j, base[j] + sign * step * d if j == k else base[j])
                at.append(float(loss()))
        slope = (at[0] - at[1]) / (2 * step)
        # the loss is a sum of 960 terms of about 1, each off by some 1e-6 at most: 1e-4 / step in all; the step's own term
        # is 1e-4 of the third derivative: together 1 % of the gradient's size over the direction
        assert abs(slope - float((grads[k] * d).sum())) <= 0.02 * float(grads[k].norm() * d.norm()), k


# ---- streams, graphs, devices ----------------------------------------------------------------------------
def test_side_stream():
    o = make_scan(BF16, "cl", 2, 64, 100, 16, seed=80)
    v = make_conv(BF16, "cl", 2, 64, 100, 4, seed=81)
    want, _, _ = run_scan(o, True)
    want_conv, _, _ = run_conv(v, True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got, _, _ = run_scan(o, True)
        got_conv, _, _ = run_conv(v, True)
    stream.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want) and all(torch.equal(got_conv[k], want_conv[k]) for k in want_conv)


def test_captured_training_step_and_tokens():
    """Two graphs, each a layer's forward and backward on tensors of its own, replayed in turn; and a graph of tokens."""
    graphs = []
    for i in range(2):
        o = make_scan(BF16, "cl", 1, 48, 90 + 50 * i, 16, seed=82 + i)
        want, gout, _ = run_scan(o, True, back="out")
        static = {k: torch.zeros_like(v).requires_grad_(True) for k, v in o.items()}

        def step(static=static, gout=gout):
            kw = {k: v for k, v in static.items() if k not in ("x", "dt", "A", "B", "C")}
            out = sc.scan_selective(*(static[k] for k in ("x", "dt", "A", "B", "C")), **kw, dt_softplus=True)
            return [out, *torch.autograd.grad(out, list(static.values()), gout)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step()
        graphs.append((graph, static, o, result, want, gout))  # the graph reads gout where it lies
    for turn in range(2):
        for graph, static, o, result, want, _ in graphs:
            with torch.no_grad():
                for k in o:
                    static[k].copy_(o[k])
            graph.replay()
        torch.cuda.synchronize()
        for graph, static, o, result, want, _ in graphs:
            for k, v in zip(["out", *("g" + k for k in o)], result):
                assert torch.equal(v, want[k]), k
    layer = Layer(32, 16, 4, F32, 84)
    x, z = randn(3, 32, seed=85), randn(3, 32, seed=86)
    windows, states = torch.zeros(3, 32, 3, device="cuda"), torch.zeros(3, 32, 16, device="cuda")
    slots = ints([2, 0, -1])
    with torch.no_grad():
        layer.token(x, z, windows.clone(), states.clone(), slots)  # products are set up outside the capture
        eager_w, eager_s = windows.clone(), states.clone()
        eager = [layer.token(x, z, eager_w, eager_s, slots) for _ in range(3)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer.token(x, z, windows, states, slots)
        windows.zero_(), states.zero_()
        for k in range(3):
            graph.replay()
            assert torch.equal(out, eager[k])
    assert torch.equal(windows, eager_w) and torch.equal(states, eager_s)


def test_two_streams_at_once():
    """Calls on two streams share nothing."""
    cases = [make_scan(BF16, "cl", 2, 256, 300, 16, seed=87 + i) for i in range(2)]
    want = [run_scan(o, True)[0] for o in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(5):
        for i, (o, stream) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(stream):
                got[i] = run_scan(o, True)[0]
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(g[k], w[k]) for k in w)


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two devices")
def test_another_device_than_the_current():
    o = {k: v.to("cuda:1") for k, v in make_scan(F32, "rows", 1, 8, 20, 4, seed=89).items()}
    out = sc.scan_selective(*(o[k] for k in ("x", "dt", "A", "B", "C")))
    assert out.device == torch.device("cuda:1") and torch.isfinite(out).all()


def test_status_is_clean():
    import ctypes

    from scanscam_b200 import _native

    detail = ctypes.c_int(0)
    assert _native.load().ssb_device_status(ctypes.byref(detail)) == _native.OK, detail.value
