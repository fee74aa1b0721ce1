"""State-space operators on the GPU at the edges of what they take: step logits far from zero.
Definitions in 64 bits: tests/_state_space.py; tolerances: tests/test_state_space_gpu.py."""
import pytest
import torch

import _state_space as ref
import scanscam_b200 as sc
from test_state_space_gpu import BF16, F16, F32, INF, make_scan, run_scan, scan_roundings

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
