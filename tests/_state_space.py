"""The state-space operators' definitions in 64 bits, one step after the other, with the size of
what was added up: for every value `v` of a result there is `m >= |v|`, the same sum with every term
taken by its size.  A kernel in 32 bits may be off by a few roundings per term, so tolerances are
counts of roundings times `m` (see `tolerance`)."""
import torch

F8 = torch.float64


def spans_of(n, steps, lengths=None, offsets=None):
    """(row, first step, step behind the last) of each sequence."""
    if offsets is not None:
        return [(0, a, b) for a, b in zip(offsets, offsets[1:])]
    return [(i, 0, steps if lengths is None else lengths[i]) for i in range(n)]


def _d(t):
    return None if t is None else t.detach().double().cpu()


def _silu(v):
    return v * torch.sigmoid(v)


def _silu_slope(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def scan_selective(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, state=None, spans=None, gout=None, gstate=None):
    """-> {name: (value, size)} for out, state and, with gout or gstate, gx, gdt, gA, gB, gC, gD, gz, gdt_bias, gstate."""
    x, dt, A, B, C, D, z, dt_bias, state, gout, gstate = map(_d, (x, dt, A, B, C, D, z, dt_bias, state, gout, gstate))
    if B.dim() == 3:
        B, C = B[:, None], C[:, None]
    n, ch, steps = x.shape
    groups, s = B.shape[1], A.shape[1]
    of = torch.arange(ch) // (ch // groups)
    raw = dt + (dt_bias[:, None] if dt_bias is not None else 0)
    D0 = D if D is not None else torch.zeros(ch, dtype=F8)
    count = len(spans)
    grad = gout is not None or gstate is not None
    g0 = gout if gout is not None else torch.zeros_like(x)

    def zeros(*shape):
        return torch.zeros(*shape, dtype=F8)

    names = {"out": (n, ch, steps), "state": (count, ch, s)}
    if grad:
        names |= {"gx": (n, ch, steps), "gdt": (n, ch, steps), "gA": (ch, s), "gB": (n, groups, s, steps), "gC": (n, groups, s, steps),
                  "gD": (ch,), "gz": (n, ch, steps), "gdt_bias": (ch,), "gstate": (count, ch, s)}
    v = {k: zeros(*w) for k, w in names.items()}
    m = {k: zeros(*w) for k, w in names.items()}
    for q, (row, lo, hi) in enumerate(spans):
        h = state[q].clone() if state is not None else zeros(ch, s)
        hm = h.abs()
        kept = []
        xs, rs = x[row, :, lo:hi], raw[row, :, lo:hi]
        ds = softplus(rs) if dt_softplus else rs
        zs = z[row, :, lo:hi] if z is not None else None
        for t in range(hi - lo):
            b, c = B[row, of, :, lo + t], C[row, of, :, lo + t]
            d, u = ds[:, t, None], xs[:, t, None]
            a = torch.exp(d * A)
            kept.append((h, hm, a))
            h, hm = a * h + d * u * b, a * hm + (d * u * b).abs()
            y, ym = (h * c).sum(1) + D0 * xs[:, t], (hm * c.abs()).sum(1) + (D0 * xs[:, t]).abs()
            gate = _silu(zs[:, t]) if zs is not None else 1.0
            v["out"][row, :, lo + t], m["out"][row, :, lo + t] = y * gate, ym * abs(gate)
            if grad:
                if zs is not None:
                    v["gz"][row, :, lo + t] = g0[row, :, lo + t] * y * _silu_slope(zs[:, t])
                    m["gz"][row, :, lo + t] = (g0[row, :, lo + t]).abs() * ym * 1.1  # the slope is at most 1.1
                gy = g0[row, :, lo + t] * gate
                v["gC"][row, :, :, lo + t].index_add_(0, of, gy[:, None] * h)
                m["gC"][row, :, :, lo + t].index_add_(0, of, gy.abs()[:, None] * hm)
        v["state"][q], m["state"][q] = h, hm
        if not grad:
            continue
        r = gstate[q].clone() if gstate is not None else zeros(ch, s)
        rm = r.abs()
        for t in range(hi - lo - 1, -1, -1):
            b, c = B[row, of, :, lo + t], C[row, of, :, lo + t]
            d, u = ds[:, t, None], xs[:, t, None]
            gate = _silu(zs[:, t]) if zs is not None else 1.0
            gy = (g0[row, :, lo + t] * gate)[:, None]
            before, before_m, a = kept[t]
            dh, dhm = gy * c + r, (gy * c).abs() + rm
            v["gB"][row, :, :, lo + t].index_add_(0, of, dh * d * u)
            m["gB"][row, :, :, lo + t].index_add_(0, of, dhm * (d * u).abs())
            through, through_m = (dh * b).sum(1), (dhm * b.abs()).sum(1)
            w, wm = dh * a * before, dhm * a * before_m
            v["gA"] += w * d
            m["gA"] += wm * d.abs()
            gd = through * xs[:, t] + (w * A).sum(1)
            gdm = through_m * xs[:, t].abs() + (wm * A.abs()).sum(1)
            slope = torch.sigmoid(rs[:, t]) if dt_softplus else 1.0
            v["gdt"][row, :, lo + t], m["gdt"][row, :, lo + t] = gd * slope, gdm * slope
            v["gx"][row, :, lo + t] = through * ds[:, t] + D0 * gy[:, 0]
            m["gx"][row, :, lo + t] = through_m * ds[:, t].abs() + (D0 * gy[:, 0]).abs()
            v["gD"] += gy[:, 0] * xs[:, t]
            m["gD"] += (gy[:, 0] * xs[:, t]).abs()
            v["gdt_bias"] += gd * slope
            m["gdt_bias"] += gdm * slope
            r, rm = a * dh, a * dhm
        v["gstate"][q], m["gstate"][q] = r, rm
    return {k: (v[k], m[k]) for k in v}


def short_conv(x, weight, bias=None, silu=False, state=None, spans=None, gout=None, gstate=None):
    """-> {name: (value, size)} for out, state and, with gout or gstate, gx, gweight, gbias, gstate."""
    x, weight, bias, state, gout, gstate = map(_d, (x, weight, bias, state, gout, gstate))
    n, ch, steps = x.shape
    w = weight.shape[1]
    grad = gout is not None or gstate is not None
    shapes = {"out": x.shape, "state": (len(spans), ch, w - 1)}
    if grad:
        shapes |= {"gx": x.shape, "gweight": weight.shape, "gbias": (ch,), "gstate": (len(spans), ch, w - 1)}
    v = {k: torch.zeros(*s, dtype=F8) for k, s in shapes.items()}
    m = {k: torch.zeros(*s, dtype=F8) for k, s in shapes.items()}
    for q, (row, lo, hi) in enumerate(spans):
        before = state[q] if state is not None else torch.zeros(ch, w - 1, dtype=F8)
        seen = torch.cat([before, x[row, :, lo:hi]], 1)
        size = hi - lo
        v["state"][q] = seen[:, size:]
        m["state"][q] = seen[:, size:].abs()
        gseen = torch.zeros_like(seen)
        gseen_m = torch.zeros_like(seen)
        for t in range(size):
            win = seen[:, t: t + w]
            pre = (win * weight).sum(1) + (bias if bias is not None else 0)
            pre_m = (win * weight).abs().sum(1) + (bias.abs() if bias is not None else 0)
            v["out"][row, :, lo + t] = _silu(pre) if silu else pre
            m["out"][row, :, lo + t] = pre_m * 1.1 if silu else pre_m
            if grad and gout is not None:
                g = gout[row, :, lo + t]
                gv = g * (_silu_slope(pre) if silu else 1.0)
                gm = g.abs() * ((1.1 + 0.5 * pre_m) if silu else 1.0)  # the slope, and how far it moves with the sum (silu'' <= 0.5)
                gseen[:, t: t + w] += gv[:, None] * weight
                gseen_m[:, t: t + w] += gm[:, None] * weight.abs()
                v["gweight"] += gv[:, None] * win
                m["gweight"] += gm[:, None] * win.abs()
                v["gbias"] += gv
                m["gbias"] += gm
        if grad:
            if gstate is not None:
                gseen[:, size:] += gstate[q]
                gseen_m[:, size:] += gstate[q].abs()
            v["gx"][row, :, lo:hi], m["gx"][row, :, lo:hi] = gseen[:, w - 1:], gseen_m[:, w - 1:]
            v["gstate"][q], m["gstate"][q] = gseen[:, : w - 1], gseen_m[:, : w - 1]
    return {k: (v[k], m[k]) for k in v}


def tolerance(dtype, value, size, roundings):
    """One rounding to `dtype` (half a step of the value), and `roundings` of 32 bits of the size of what was added up;
    values below the type's normal range are off by half of its smallest step."""
    info = torch.finfo(dtype)
    tiny = info.tiny * info.eps  # the step below the normal range
    return info.eps / 2 * value.abs() + roundings * 2.0 ** -24 * (1 + info.eps) * size + tiny


def check(got, want, dtype, roundings, name):
    value, size = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), (name, "not finite")
    off = (got - value).abs() - tolerance(dtype, value, size, roundings)
    worst = off.argmax() if off.numel() else None
    assert off.numel() == 0 or off.max() <= 0, (
        f"{name}: {got.flatten()[worst].item()} for {value.flatten()[worst].item()} (size {size.flatten()[worst].item()}), "
        f"allowed {tolerance(dtype, value, size, roundings).flatten()[worst].item():.3g}")
