"""GPU: sizes at which the kernels behind the norms and the 8-bit activations go round their rings of rows several times: slots filled
again, phases that flip, ends in the middle of a step, CTAs that go from one gate row to the next."""

import pytest
import torch

from test_act8_gpu import kept_values
from test_sandwich_gpu import check, formulas, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(16391, 3584), (9001, 3616), (40000, 200), (5003, 37888)])
def test_lora_gradient_over_many_steps(cuda_lib, rows, cols):
    """More steps of 16 rows to a warp than its ring has slots, a remainder behind them; rows whose blocks are far apart in size (a step
    below 2^-24 or above 2^5 takes another branch), and empty ones."""
    from hackaton_b200 import act8_quantize, lora_grad_act8

    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, cols, device="cuda", generator=g)
    size = torch.exp2(torch.randint(-14, 13, (rows, 1), device="cuda", generator=g).float())
    size[torch.rand(rows, 1, device="cuda", generator=g) < 0.1] = 0
    x = (x * size).half()
    s = torch.randn(rows, 16, device="cuda", generator=g).half()
    kept = act8_quantize(x)
    got = lora_grad_act8(kept, s)
    s64 = s.double()
    for c in range(0, cols, 4096):      # (kept_values: 64 bits on the host)
        v = kept_values(x[:, c:c + 4096])[0].cuda()
        bound = rows * 2.0 ** -23 * (s64.abs().t() @ v.abs()) + 1e-45
        assert ((got[:, c:c + 4096].double() - s64.t() @ v).abs() <= bound).all(), c
    assert torch.equal(got, lora_grad_act8(kept, s))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden,gates", [(4100, 1536, 1), (4084, 3584, 4), (3000, 256, 3000), (6000, 64, 2000), (5000, 130, 5000),
                                               (2500, 1001, 5), (9000, 8, 3), (1500, 8192, 3), (3001, 4096, 0), (700, 5001, 1)])
def test_norms_over_many_rows(cuda_lib, dtype, rows, hidden, gates):
    t, d_stream, d_normed = inputs(rows, hidden, dtype, gates, rows + hidden)
    got = run(t, d_stream, d_normed, 0.75, 1e-6)
    want = formulas(t["residual"], t["delta"], t["post"], t["pre"], t["gate"], 0.75, 1e-6, d_stream, d_normed.to(dtype))
    for name, (value, mags) in want.items():
        check(name, got[name], value, mags, 64 + (rows if name in ("d_post", "d_pre", "d_gate") else 0))
    again = run(t, d_stream, d_normed, 0.75, 1e-6)
    assert all(torch.equal(got[k], again[k]) for k in got)
    cuda_lib.device_status()
