"""The state-space operators: cases, plain forms and definitions.

Four operators that follow one another in a layer whose sequence mixing is a selective scan:

``short_conv``           the short causal convolution in front of the scan, over whole prompts
``short_conv_step``      the same for single tokens, its window held in a pool of states
``scan_selective``       the scan with input-dependent steps and projections, over whole prompts
``scan_selective_step``  the same for single tokens, its state held in a pool

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits; with ``own``
true it makes the calls that a user of the framework makes.  ``exact`` computes the definitions in
64 bits, one time step after the other.

Tensors are laid out as the framework's are: ``[N, C, T]`` with time last, either dense that way
("rows") or as a view of dense ``[N, T, C]`` ("channels last"), where x and z, dt, B and C are
slices of the projections that make them, as in a layer.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one sequence: the smallest call there is, a matter of launches
        {"name": "conv_step_1", "op": "conv_step", "dtype": "bf16", "M": 1, "C": 2048, "W": 4, "pool": 0},
        # a full serving batch whose windows lie scattered in a pool, some entries of the batch idle
        {"name": "conv_step_256", "op": "conv_step", "dtype": "bf16", "M": 256, "C": 8192, "W": 4, "pool": 512},
        # packed prompts of different lengths, continued from earlier pieces
        {"name": "conv_prompts_packed", "op": "conv", "dtype": "bf16", "layout": "cl", "N": 1, "C": 4096, "T": 8192, "W": 4,
         "seqs": 13, "state": True, "train": False},
        # a training batch of a usual size
        {"name": "conv_train", "op": "conv", "dtype": "bf16", "layout": "cl", "N": 8, "C": 4096, "T": 2048, "W": 4,
         "seqs": 0, "state": False, "train": True},
        # odd channels and steps in the framework's rows layout, gradients through the carried window too
        {"name": "conv_train_odd_rows", "op": "conv", "dtype": "fp32", "layout": "rows", "N": 3, "C": 515, "T": 1001, "W": 3,
         "seqs": 0, "state": True, "train": True},
        # one token of one sequence
        {"name": "scan_step_1", "op": "scan_step", "dtype": "bf16", "M": 1, "C": 2048, "S": 16, "G": 1, "pool": 0},
        # a full serving batch on a pool of states, some entries idle
        {"name": "scan_step_256", "op": "scan_step", "dtype": "bf16", "M": 256, "C": 4096, "S": 16, "G": 1, "pool": 512},
        # a single long prompt: few channels, many steps
        {"name": "scan_prompt_long", "op": "scan", "dtype": "bf16", "layout": "cl", "N": 1, "C": 2048, "T": 8192, "S": 16, "G": 1,
         "seqs": 0, "state": False, "train": False},
        # packed prompts of different lengths, continued from earlier pieces
        {"name": "scan_prompts_packed", "op": "scan", "dtype": "bf16", "layout": "cl", "N": 1, "C": 4096, "T": 4096, "S": 16, "G": 1,
         "seqs": 13, "state": True, "train": False},
        # a training batch of a usual size
        {"name": "scan_train", "op": "scan", "dtype": "bf16", "layout": "cl", "N": 4, "C": 2048, "T": 2048, "S": 16, "G": 1,
         "seqs": 0, "state": False, "train": True},
        # odd channels, steps and states in the rows layout, channels in three groups, gradients through the carried state too
        {"name": "scan_train_odd_rows", "op": "scan", "dtype": "fp32", "layout": "rows", "N": 2, "C": 387, "T": 1001, "S": 10, "G": 3,
         "seqs": 0, "state": True, "train": True},
        # wide states, channels in groups, half precision
        {"name": "scan_train_wide", "op": "scan", "dtype": "fp16", "layout": "cl", "N": 2, "C": 1024, "T": 1024, "S": 64, "G": 4,
         "seqs": 0, "state": False, "train": True},
    ]


def draw(rng):
    def spread(lo, hi, step=1):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, v // step * step)

    op = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op.endswith("step"):
        M = spread(1, 256)
        c = {"op": op, "dtype": dtype, "M": M, "C": spread(256, 4096, rng.choice([1, 8, 64])), "pool": rng.choice([0, M, 2 * M])}
        if op == "conv_step":
            c["W"] = rng.randint(2, 4)
        else:
            c["G"] = rng.choice([1, 1, 2])
            c["C"] = max(c["G"], c["C"] // c["G"] * c["G"])
            c["S"] = rng.choice([7, 16, 16, 32])
        return c
    layout = rng.choice(["cl", "cl", "rows"])
    train = rng.random() < 0.5
    packed = layout == "cl" and rng.random() < 0.4
    N = 1 if packed else rng.randint(1, 8)
    step = rng.choice([1, 8, 64])
    c = {"op": op, "dtype": dtype, "layout": layout, "N": N}
    if op == "conv":
        c["C"] = spread(128, 4096, step)
        c["T"] = spread(1, min(8192, 33554432 // (N * c["C"])))
        c["W"] = rng.randint(2, 4)
    else:
        c["S"] = rng.choice([8, 11, 16, 16, 16, 32, 64])
        c["G"] = rng.choice([1, 1, 1, 2])
        c["C"] = max(c["G"], spread(128, 4096, step) // c["G"] * c["G"])
        c["T"] = spread(1, max(1, min(8192, 134217728 // (N * c["C"] * c["S"]))))
    c["seqs"] = min(c["T"], rng.randint(1, 24)) if packed else 0
    c["state"] = rng.random() < 0.5
    c["train"] = train
    return c


def work(case):
    """Every input read once, every output written once; a multiply, an add or an exponential counts as one operation."""
    e = 4 if case["dtype"] == "fp32" else 2
    C = case["C"]
    if case["op"] == "conv_step":
        M, W = case["M"], case["W"]
        return {"bytes": M * C * e * (2 + 2 * (W - 1)) + C * e * (W + 1), "flops": M * C * (2 * W + 4)}
    if case["op"] == "scan_step":
        M, S, G = case["M"], case["S"], case["G"]
        return {"bytes": M * C * (4 * e + 8 * S) + M * G * S * 2 * e + C * (4 * S + 8), "flops": M * C * (7 * S + 12)}
    N, T, train = case["N"], case["T"], case["train"]
    seqs = case["seqs"] or N
    if case["op"] == "conv":
        W = case["W"]
        held = seqs * C * (W - 1) * e * (2 if case["state"] else 1)
        fwd = {"bytes": 2 * N * C * T * e + C * (W + 1) * e + held, "flops": N * C * T * (2 * W + 4)}
        if not train:
            return fwd
        # backward: x and the upstream gradient in, the gradients of x, weight and bias out
        return {"bytes": fwd["bytes"] + 3 * N * C * T * e + 2 * C * (W + 1) * e, "flops": fwd["flops"] + N * C * T * (6 * W + 10)}
    S, G = case["S"], case["G"]
    held = seqs * C * S * 4 * (2 if case["state"] else 1)
    proj = 2 * N * T * G * S * e
    fwd = {"bytes": 4 * N * C * T * e + proj + C * (4 * S + 8) + held, "flops": N * C * T * (7 * S + 12)}
    if not train:
        return fwd
    # backward: x, dt, z and the upstream gradient in, three gradients of that size out; B and C in, their gradients out
    return {"bytes": fwd["bytes"] + 7 * N * C * T * e + 2 * proj + 2 * C * (4 * S + 8),
            "flops": fwd["flops"] + N * C * T * (20 * S + 30)}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _cuts(total, seqs, g):
    """Offsets of `seqs` sequences of random lengths, one at least, that fill `total` steps."""
    inner = torch.randperm(total - 1, generator=g)[: seqs - 1] + 1
    return torch.cat([torch.tensor([0]), inner.sort().values, torch.tensor([total])]).to(torch.int32)


def _slots(M, pool, g):
    """Places in the pool, each once; about one entry in sixteen idle (-1), as in a batch whose sequences have ended."""
    slots = torch.randperm(pool, generator=g)[:M].to(torch.int32)
    if M > 1:
        slots[torch.rand(M, generator=g) < 1 / 16] = -1
    return slots


def prepare(case, seed):
    dev, dt = "cuda", DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    C = case["C"]
    s = {"case": case}
    if case["op"] in ("conv", "conv_step"):
        W = case["W"]
        # taps as a depthwise convolution is initialised: uniform within 1 / sqrt(W)
        s["weight"] = ((2 * rand(C, W) - 1) / math.sqrt(W)).to(dt)
        s["bias"] = ((2 * rand(C) - 1) / math.sqrt(W)).to(dt)
        if case["op"] == "conv_step":
            P = case["pool"] or case["M"]
            s["x"] = randn(case["M"], C).to(dt)
            s["state"] = randn(P, C, W - 1).to(dt)
            s["slots"] = _slots(case["M"], P, h).to(dev) if case["pool"] else None
            return s
    else:
        S, G = case["S"], case["G"]
        # decays -1 ... -S with some spread, steps of 0.001 ... 0.1 through the softplus' inverse: the usual start of training
        s["A"] = -torch.arange(1, S + 1, device=dev).float() * torch.exp(0.2 * randn(C, S))
        step = torch.exp(rand(C) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["D"] = 1 + 0.1 * randn(C)
        if case["op"] == "scan_step":
            P = case["pool"] or case["M"]
            M = case["M"]
            s["x"], s["z"] = torch.nn.functional.silu(randn(M, C)).to(dt), randn(M, C).to(dt)
            s["dt"] = (0.5 * randn(M, C)).to(dt)
            s["B"], s["C"] = randn(M, G, S).to(dt), randn(M, G, S).to(dt)
            s["state"] = 0.3 * randn(P, C, S)
            s["slots"] = _slots(M, P, h).to(dev) if case["pool"] else None
            return s
    N, T, cl = case["N"], case["T"], case["layout"] == "cl"
    s["offsets"] = _cuts(T, case["seqs"], h).to(dev) if case["seqs"] else None
    held = case["seqs"] or N

    def leaf(t):
        return t.requires_grad_(True) if case["train"] else t

    if case["op"] == "conv":
        # channels last: the half of a projection that goes into the convolution
        s["x"] = leaf(randn(N, T, 2 * C).to(dt)[:, :, :C].mT if cl else randn(N, C, T).to(dt))
        s["state"] = leaf(randn(held, C, W - 1).to(dt)) if case["state"] else None
        s["weight"], s["bias"] = leaf(s["weight"]), leaf(s["bias"])
        s["grad"] = randn(N, T, C).to(dt).mT if cl else randn(N, C, T).to(dt)
        return s
    silu = torch.nn.functional.silu
    if cl:
        s["x"] = leaf(silu(randn(N, T, C)).to(dt).mT)
        s["z"] = leaf(randn(N, T, 2 * C).to(dt)[:, :, C:].mT)  # the other half of that projection
        s["dt"] = leaf((0.5 * randn(N, T, C)).to(dt).mT)
        proj = randn(N, T, 2 * G * S).to(dt)
        s["B"] = leaf(proj[:, :, : G * S].unflatten(2, (G, S)).permute(0, 2, 3, 1))
        s["C"] = leaf(proj[:, :, G * S:].unflatten(2, (G, S)).permute(0, 2, 3, 1))
        s["grad"] = randn(N, T, C).to(dt).mT
    else:
        s["x"], s["z"] = leaf(silu(randn(N, C, T)).to(dt)), leaf(randn(N, C, T).to(dt))
        s["dt"] = leaf((0.5 * randn(N, C, T)).to(dt))
        s["B"], s["C"] = leaf(randn(N, G, S, T).to(dt)), leaf(randn(N, G, S, T).to(dt))
        s["grad"] = randn(N, C, T).to(dt)
    for k in ("A", "D", "dt_bias"):
        leaf(s[k])
    s["state"] = leaf(0.3 * randn(held, C, S)) if case["state"] else None
    s["grad_state"] = randn(held, C, S)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if op == "conv_step":
        f = _own_conv_step if own else _plain_conv_step
        return {"out": f(s), "state": s["state"]}
    if op == "scan_step":
        f = _own_scan_step if own else _plain_scan_step
        return {"out": f(s), "state": s["state"]}
    if op == "conv":
        out, state = (_own_conv if own else _plain_conv)(s)
        if not s["case"]["train"]:
            return {"out": out, "state": state}
        wrt = {k: s[k] for k in ("x", "weight", "bias", "state") if s[k] is not None}
        grads = torch.autograd.grad(out, list(wrt.values()), s["grad"], materialize_grads=True)
        return {"out": out, "state": state, "grads": dict(zip(wrt, grads))}
    out, state = (_own_scan if own else _plain_scan)(s)
    if not s["case"]["train"]:
        return {"out": out, "state": state}
    wrt = {k: s[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state") if s[k] is not None}
    if s["case"]["state"]:  # a piece of a longer sequence: a gradient comes in from the piece behind it too
        grads = torch.autograd.grad([out, state], list(wrt.values()), [s["grad"], s["grad_state"]], materialize_grads=True)
    else:
        # a single step from nothing has no gradient for A
        grads = torch.autograd.grad(out, list(wrt.values()), s["grad"], materialize_grads=True)
    return {"out": out, "state": state, "grads": dict(zip(wrt, grads))}


# the framework's calls
def _own_conv_step(s):
    import scanscam_b200 as scanscam
    return scanscam.short_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu", slots=s["slots"])


def _own_scan_step(s):
    import scanscam_b200 as scanscam
    return scanscam.scan_selective_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                                        dt_bias=s["dt_bias"], dt_softplus=True, slots=s["slots"])


def _own_conv(s):
    import scanscam_b200 as scanscam
    return scanscam.short_conv(s["x"], s["weight"], s["bias"], activation="silu", state=s["state"], offsets=s["offsets"],
                               return_state=True)


def _own_scan(s):
    import scanscam_b200 as scanscam
    return scanscam.scan_selective(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                   dt_softplus=True, state=s["state"], offsets=s["offsets"], return_state=True)


# the plain forms
def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    # log(1 + e^v) without overflow, and without loss where e^v is small
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _plain_conv_step(s):
    x, state, W = s["x"], s["state"], s["case"]["W"]
    at = torch.arange(x.shape[0], device=x.device) if s["slots"] is None else s["slots"].long()
    live = at >= 0
    window = torch.cat([state[at.clamp(min=0)], x[:, :, None]], 2)  # [M, C, W]
    y = _silu((window.float() * s["weight"].float()).sum(2) + s["bias"].float())
    state[at[live]] = window[live][:, :, 1:]
    return (y * live[:, None]).to(x.dtype)


def _plain_scan_step(s):
    x, state, C = s["x"], s["state"], s["case"]["C"]
    at = torch.arange(x.shape[0], device=x.device) if s["slots"] is None else s["slots"].long()
    live = at >= 0
    u = x.float()
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    per = C // s["case"]["G"]
    B, Cm = (s[k].float().repeat_interleave(per, 1) for k in ("B", "C"))  # [M, C, S]
    h = torch.exp(dt[:, :, None] * s["A"]) * state[at.clamp(min=0)] + (dt * u)[:, :, None] * B
    y = ((h * Cm).sum(2) + s["D"] * u) * _silu(s["z"].float())
    state[at[live]] = h[live]
    return (y * live[:, None]).to(x.dtype)


def _starts(s):
    """For every step of [N, T]: the first step of its sequence, and which sequence it is."""
    N, T = s["case"]["N"], s["case"]["T"]
    t = torch.arange(T, device=s["x"].device)
    if s["offsets"] is None:
        return torch.zeros(N, T, dtype=torch.long, device=t.device), torch.arange(N, device=t.device)[:, None].expand(N, T)
    seq = torch.searchsorted(s["offsets"][1:].long(), t, right=True)
    return s["offsets"].long()[seq][None], seq[None]


def _last(s):
    """Place of the last step of each sequence in the flattened [N * T]."""
    N, T = s["case"]["N"], s["case"]["T"]
    if s["offsets"] is None:
        return torch.arange(1, N + 1, device=s["x"].device) * T - 1
    return s["offsets"][1:].long() - 1


def _plain_conv(s):
    x, W = s["x"].mT, s["case"]["W"]  # [N, T, C]
    N, T, C = x.shape
    dt = s["x"].dtype
    start, seq = _starts(s)
    held = s["state"] if s["state"] is not None else torch.zeros(s["case"]["seqs"] or N, C, W - 1, device=x.device, dtype=dt)
    t = torch.arange(T, device=x.device)[None]
    flat, row = x.reshape(N * T, C), torch.arange(N, device=x.device)[:, None] * T

    def back(j, t, start, seq, row):
        """The input j steps before step t of its sequence: from x, or from the window that came before."""
        far = (t - j < start)[..., None]
        return torch.where(far, held.mT[seq, (W - 1 + t - j - start).clamp(0, W - 2)], flat[(row + t - j).clamp(min=0)])

    w = s["weight"].float()
    y = sum(back(j, t, start, seq, row).float() * w[:, W - 1 - j] for j in range(W)) + s["bias"].float()
    last = _last(s)
    state = torch.stack([back(j, last % T, start.expand(N, T).reshape(-1)[last], seq.reshape(-1)[last], last // T * T)
                         for j in range(W - 2, -1, -1)], 2)
    return _silu(y).to(dt).mT, state


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1, from zero: pairs of steps are joined into one, half the length is solved, the rest filled in."""
    T = a.shape[1]
    if T == 1:
        return b
    a0, b0, a1, b1 = a[:, : T - 1: 2], b[:, : T - 1: 2], a[:, 1::2], b[:, 1::2]
    odd = _recurrence(a1 * a0, a1 * b0 + b1)
    even = torch.cat([b[:, :1], a[:, 2::2] * odd[:, : (T - 1) // 2] + b[:, 2::2]], 1)
    both = torch.stack([even[:, : T // 2], odd], 2).flatten(1, 2)
    return both if T % 2 == 0 else torch.cat([both, even[:, -1:]], 1)


def _plain_scan(s):
    u, z = s["x"].mT.float(), s["z"].mT.float()  # [N, T, C]
    N, T, C = u.shape
    per = C // s["case"]["G"]
    start, seq = _starts(s)
    dt = _softplus(s["dt"].mT.float() + s["dt_bias"])
    # in the inputs' type, widened where used: [N, T, G, 1, S] against [N, T, G, per, 1]
    B, Cm = (s[k].permute(0, 3, 1, 2).float()[:, :, :, None] for k in ("B", "C"))

    def grouped(v):
        return v.unflatten(2, (s["case"]["G"], per))[..., None]

    a = torch.exp(grouped(dt) * s["A"].unflatten(0, (-1, per)))  # [N, T, G, per, S]
    b = grouped(dt * u) * B
    first = (torch.arange(T, device=u.device)[None] == start)[:, :, None, None, None]
    if s["state"] is not None:
        b = b + torch.where(first, a * s["state"][seq].unflatten(2, (-1, per)), 0)
    h = _recurrence(torch.where(first, 0, a), b)
    y = (h * Cm).sum(4).flatten(2) + s["D"] * u
    state = h.flatten(0, 1)[_last(s)].flatten(1, 2)
    return (y * _silu(z)).to(s["x"].dtype).mT, state


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    with torch.no_grad():
        return {"conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan, "scan_step": _exact_scan_step}[case["op"]](s)


def _bounds(s):
    """(row of x, first step, step behind the last) of each sequence."""
    if s["offsets"] is None:
        return [(n, 0, s["case"]["T"]) for n in range(s["case"]["N"])]
    o = s["offsets"].tolist()
    return [(0, a, b) for a, b in zip(o, o[1:])]


def _exact_conv_step(s):
    x, w, W = s["x"].double(), s["weight"].double(), s["case"]["W"]
    state = s["state"].double()
    out = torch.zeros_like(x)
    for m, at in enumerate(s["slots"].tolist() if s["slots"] is not None else range(len(x))):
        if at >= 0:
            seen = torch.cat([state[at], x[m][:, None]], 1)
            v = s["bias"].double() + torch.einsum("cw,cw->c", seen, w)
            out[m] = v * torch.sigmoid(v)
            state[at] = seen[:, 1:]
    return {"out": out, "state": state}


def _exact_scan_step(s):
    x, state, case = s["x"].double(), s["state"].double(), s["case"]
    of = torch.arange(case["C"], device=x.device) // (case["C"] // case["G"])
    out = torch.zeros_like(x)
    for m, at in enumerate(s["slots"].tolist() if s["slots"] is not None else range(len(x))):
        if at >= 0:
            dt = torch.logaddexp(s["dt"][m].double() + s["dt_bias"].double(), torch.zeros((), device=x.device, dtype=torch.float64))
            state[at] = torch.exp(dt[:, None] * s["A"].double()) * state[at] + (dt * x[m])[:, None] * s["B"][m].double()[of]
            z = s["z"][m].double()
            out[m] = (torch.einsum("cs,cs->c", state[at], s["C"][m].double()[of]) + s["D"].double() * x[m]) * z * torch.sigmoid(z)
    return {"out": out, "state": state}


def _exact_conv(s):
    case, W = s["case"], s["case"]["W"]
    x, w = s["x"].double(), s["weight"].double()
    N, C, T = x.shape
    out, gx = torch.empty_like(x), torch.empty_like(x)
    gw, gb = torch.zeros_like(w), torch.zeros(C, device=x.device, dtype=torch.float64)
    states, gstates = [], []
    for i, (n, lo, hi) in enumerate(_bounds(s)):
        before = s["state"][i].double() if s["state"] is not None else torch.zeros(C, W - 1, device=x.device, dtype=torch.float64)
        seen = torch.cat([before, x[n, :, lo:hi]], 1)
        L = hi - lo
        v = s["bias"].double()[:, None] + sum(w[:, k: k + 1] * seen[:, k: k + L] for k in range(W))
        sg = torch.sigmoid(v)
        out[n, :, lo:hi] = v * sg
        states.append(seen[:, L:])
        if case["train"]:
            gv = s["grad"][n, :, lo:hi].double() * sg * (1 + v * (1 - sg))
            gseen = torch.zeros_like(seen)
            for k in range(W):
                gseen[:, k: k + L] += w[:, k: k + 1] * gv
                gw[:, k] += (seen[:, k: k + L] * gv).sum(1)
            gb += gv.sum(1)
            gx[n, :, lo:hi] = gseen[:, W - 1:]
            gstates.append(gseen[:, : W - 1])
    r = {"out": out, "state": torch.stack(states)}
    if case["train"]:
        r["grads"] = {"x": gx, "weight": gw, "bias": gb}
        if s["state"] is not None:
            r["grads"]["state"] = torch.stack(gstates)
    return r


def _exact_scan(s):
    """Step after step, then the same steps backwards with the adjoint of the state."""
    case = s["case"]
    N, T, S, G = case["N"], case["T"], case["S"], case["G"]
    Ch = case["C"]
    f8 = dict(device=s["x"].device, dtype=torch.float64)
    of = torch.arange(Ch, device=s["x"].device) // (Ch // G)
    A, D = s["A"].double(), s["D"].double()
    x, z = (s[k].double().permute(2, 0, 1).contiguous() for k in ("x", "z"))  # [T, N, C]
    v = s["dt"].double().permute(2, 0, 1) + s["dt_bias"].double()
    dt = torch.logaddexp(v, torch.zeros((), **f8))
    B, Cm = (s[k].double().permute(3, 0, 1, 2).contiguous() for k in ("B", "C"))  # [T, N, G, S]
    where = _bounds(s)
    opens = {(n, lo): i for i, (n, lo, hi) in enumerate(where)}
    closes = {(n, hi - 1): i for i, (n, lo, hi) in enumerate(where)}
    marks = {t for n, t in opens} | {t for n, t in closes}
    state = torch.zeros(len(where), Ch, S, **f8)
    y = torch.empty(T, N, Ch, **f8)
    h = torch.zeros(N, Ch, S, **f8)
    kept = torch.empty(T, N, Ch, S, **f8) if case["train"] else None  # the state before each step
    for t in range(T):
        if t in marks:
            for n in range(N):
                if (n, t) in opens:
                    h[n] = s["state"][opens[n, t]].double() if s["state"] is not None else 0
        if kept is not None:
            kept[t] = h
        h = torch.exp(dt[t][..., None] * A) * h + (dt[t] * x[t])[..., None] * B[t][:, of]
        y[t] = (h * Cm[t][:, of]).sum(2)
        if t in marks:
            for n in range(N):
                if (n, t) in closes:
                    state[closes[n, t]] = h[n]
    y += D * x
    sz = torch.sigmoid(z)
    r = {"out": (y * z * sz).permute(1, 2, 0), "state": state}
    if not case["train"]:
        return r
    go = s["grad"].double().permute(2, 0, 1)
    gy = go * z * sz
    gz = go * y * sz * (1 + z * (1 - sz))
    gx, gdt = D * gy, torch.zeros_like(dt)
    gA = torch.zeros_like(A)
    gB, gC = torch.zeros_like(B), torch.zeros_like(Cm)
    gstate = torch.zeros_like(state)
    gh = torch.zeros(N, Ch, S, **f8)
    for t in range(T - 1, -1, -1):
        if t in marks:
            for n in range(N):
                if (n, t) in closes:
                    gh[n] = s["grad_state"][closes[n, t]].double() if s["state"] is not None else 0
        gh = gh + gy[t][..., None] * Cm[t][:, of]
        decay = torch.exp(dt[t][..., None] * A)
        now = decay * kept[t] + (dt[t] * x[t])[..., None] * B[t][:, of]
        gC[t] = (gy[t][..., None] * now).unflatten(1, (G, -1)).sum(2)
        gB[t] = (gh * (dt[t] * x[t])[..., None]).unflatten(1, (G, -1)).sum(2)
        through = (gh * B[t][:, of]).sum(2)
        gx[t] += through * dt[t]
        by_decay = gh * kept[t] * decay
        gdt[t] = through * x[t] + (by_decay * A).sum(2)
        gA += (by_decay * dt[t][..., None]).sum(0)
        gh = gh * decay
        if t in marks:
            for n in range(N):
                if (n, t) in opens:
                    gstate[opens[n, t]] = gh[n]
    gv = gdt * torch.sigmoid(v)
    r["grads"] = {"x": gx.permute(1, 2, 0), "dt": gv.permute(1, 2, 0), "A": gA, "B": gB.permute(1, 2, 3, 0), "C": gC.permute(1, 2, 3, 0),
                  "D": (gy * x).sum((0, 1)), "z": gz.permute(1, 2, 0), "dt_bias": gv.sum((0, 1))}
    if s["state"] is not None:
        r["grads"]["state"] = gstate
    return r
