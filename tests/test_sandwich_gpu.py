"""GPU: the norms around a block with its gate and residual scale, both directions, against the formulas in 64 bits.

Bounds. In fp32 each operation is off by 2^-24 of its result, a sum over a row by its depth in additions: a thread's own
values (at most 16), five levels in the warp and five across warps, three sums at most: under 64 units. So every output is off by at
most 64 * 2^-24 of the magnitudes that meet in it (the same formula with absolute values), carried through the second norm;
sums over rows by one unit per row more. A 16-bit output adds one rounding, half of its type's eps of the value."""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def formulas(residual, delta, post, pre, gate, scale, eps, d_stream=None, d_normed=None):
    """Outputs and gradients in 64 bits, and for each the magnitudes that meet in it. gate: [gates, hidden] or None."""
    f = lambda t: t.detach().double()
    r, d, post, pre = f(residual), f(delta), f(post), f(pre)
    rows, hidden = r.shape
    g = torch.ones(1, hidden, dtype=torch.float64, device=r.device) if gate is None else f(gate)
    gr = g.repeat_interleave(rows // g.shape[0], dim=0)
    rd = 1 / (d.pow(2).mean(1, keepdim=True) + eps).sqrt()
    dh = d * rd
    s = scale * r + gr * dh * post
    s_mag = (scale * r).abs() + (gr * dh * post).abs()
    rs = 1 / (s.pow(2).mean(1, keepdim=True) + eps).sqrt()
    sh = s * rs
    sh_mag = s_mag * rs + sh.abs() * (s_mag * s.abs()).mean(1, keepdim=True) * rs * rs   # (through its own norm)
    out = {"stream": (s, s_mag), "normed": (sh * pre, sh_mag * pre.abs())}
    if d_normed is None:
        return out
    t, y = f(d_stream), f(d_normed)
    w = y * pre
    m1 = (w * sh).mean(1, keepdim=True)
    m1_mag = (w.abs() * sh_mag).mean(1, keepdim=True)
    ds = t + rs * (w - sh * m1)
    # (rs itself is off by sh_mag's share)
    ds_mag = t.abs() + rs * (w.abs() + 2 * sh_mag * m1_mag) + rs * w.abs() * (sh_mag * sh.abs()).mean(1, keepdim=True)
    q, q_mag = ds * gr * post, ds_mag * (gr * post).abs()
    out["d_residual"] = (scale * ds, abs(scale) * ds_mag)
    out["d_delta"] = (rd * (q - dh * (q * dh).mean(1, keepdim=True)),
                      rd * (q_mag + 3 * dh.abs() * (q_mag * dh.abs()).mean(1, keepdim=True)))
    out["d_post"] = ((ds * gr * dh).sum(0), (ds_mag * (gr * dh).abs()).sum(0))
    out["d_pre"] = ((y * sh).sum(0), (y.abs() * sh_mag).sum(0))
    if gate is not None:
        cut = (g.shape[0], rows // g.shape[0], hidden)
        out["d_gate"] = ((ds * dh * post).view(cut).sum(1), (ds_mag * (dh * post).abs()).view(cut).sum(1))
    return out


def check(name, got, want, mags, units):
    # (a value beyond the type's largest is an infinity once rounded: fp16's 65504 + 16 and more)
    top = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    beyond = want.abs() - units * U * mags >= top
    assert torch.equal(got[beyond].double(), want[beyond].sign() * float("inf")), name
    got, want, mags = got[~beyond], want[~beyond], mags[~beyond]
    off = (got.double() - want).abs()
    bound = units * U * mags + 1e-40
    if got.dtype != torch.float32:
        bound = bound + torch.finfo(got.dtype).eps / 2 * (want.abs() + bound) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    assert (off <= bound).all(), (name, float((off / bound).max()))


def inputs(rows, hidden, dtype, gates, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    channel = torch.where(torch.rand(hidden, device="cuda", generator=g) < 0.02, 30.0, 1.0)
    t = {"residual": n(rows, hidden) * 2 * channel, "delta": (n(rows, hidden) * 0.5 * channel).to(dtype),
         "post": 1 + 0.2 * n(hidden), "pre": 1 + 0.2 * n(hidden), "gate": 0.3 * n(gates, hidden) if gates else None}
    for v in t.values():
        if v is not None:
            v.requires_grad_()
    return t, n(rows, hidden), n(rows, hidden)


def run(t, d_stream, d_normed, scale, eps, out_dtype=None):
    from hackaton_b200 import sandwich_norm

    stream, normed = sandwich_norm(t["residual"], t["delta"], t["post"], t["pre"], eps, gate=t["gate"],
                                   residual_scale=scale, out_dtype=out_dtype)
    out = {"stream": stream, "normed": normed}
    names = [k for k, v in t.items() if v is not None]
    grads = torch.autograd.grad([stream, normed], [t[k] for k in names], [d_stream, d_normed.to(normed.dtype)])
    out.update({"d_" + k: g for k, g in zip(names, grads)})
    return {k: v.detach() for k, v in out.items()}     # (an eager graph that lives on keeps its leaves from a capture)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden,gates", [(1, 1, 0), (1, 7, 1), (3, 64, 1), (5, 130, 5), (12, 100, 4), (300, 1000, 3),
                                               (1031, 1536, 1), (64, 3584, 2), (7, 4096, 0), (9, 5000, 3), (6, 8192, 1),
                                               (4, 5001, 2), (3, 16384, 1), (2, 16383, 1)])
def test_matches_the_formulas(cuda_lib, dtype, rows, hidden, gates):
    t, d_stream, d_normed = inputs(rows, hidden, dtype, gates, rows + hidden)
    got = run(t, d_stream, d_normed, 0.75, 1e-6)
    want = formulas(t["residual"], t["delta"], t["post"], t["pre"], t["gate"], 0.75, 1e-6, d_stream, d_normed.to(dtype))
    for name, (value, mags) in want.items():
        assert got[name].dtype == (dtype if name in ("normed", "d_delta") else torch.float32)
        check(name, got[name], value, mags, 64 + (rows if name in ("d_post", "d_pre", "d_gate") else 0))
    again = run(t, d_stream, d_normed, 0.75, 1e-6)
    assert all(torch.equal(got[k], again[k]) for k in got)           # the same order of additions


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fp32_output(cuda_lib, dtype):
    t, d_stream, d_normed = inputs(33, 320, dtype, 1, 5)
    got = run(t, d_stream, d_normed, 1.0, 1e-5, torch.float32)
    want = formulas(t["residual"], t["delta"], t["post"], t["pre"], t["gate"], 1.0, 1e-5, d_stream, d_normed)
    assert got["normed"].dtype == torch.float32
    for name, (value, mags) in want.items():
        check(name, got[name], value, mags, 64 + 33)


def test_gradients_against_differences(cuda_lib):
    """The fp32 forward's own differences along a direction in each input: (L(x + h v) - L(x - h v)) / 2h is off by
    the third derivative (h^2) and by the forward's rounding (64 units of |L|'s terms over h)."""
    from hackaton_b200 import sandwich_norm

    t, d_stream, d_normed = inputs(6, 40, torch.float32, 3, 11)
    got = run(t, d_stream, d_normed, 0.5, 1e-6)

    def loss(**change):
        a = {k: change.get(k, v.detach()) for k, v in t.items()}
        s, y = sandwich_norm(a["residual"], a["delta"], a["post"], a["pre"], 1e-6, gate=a["gate"], residual_scale=0.5)
        return float((s.double() * d_stream.double()).sum() + (y.double() * d_normed.double()).sum())

    h = 2.0 ** -8
    terms = float(sum((got[k].detach().double() * d.double()).abs().sum() for k, d in (("stream", d_stream), ("normed", d_normed))))
    for name, v in t.items():
        step = torch.randn(v.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * v.detach().abs().clamp(min=0.1)
        by_difference = (loss(**{name: v.detach() + h * step}) - loss(**{name: v.detach() - h * step})) / (2 * h)
        by_gradient = float((got["d_" + name].double() * step.double()).sum())
        scale = float((got["d_" + name].double() * step.double()).abs().sum())
        assert abs(by_difference - by_gradient) <= 64 * U * terms / h + 40 * h * h * scale + 1e-3 * scale * h, name


def test_rows_of_zeros_and_cancelling_rows(cuda_lib):
    """A row of zeros divides by sqrt(eps) alone; a stream that cancels keeps the accuracy of its terms."""
    t, d_stream, d_normed = inputs(8, 256, torch.float16, 0, 2)
    with torch.no_grad():
        t["residual"][0] = 0
        t["delta"][0] = 0
        t["delta"][1] = 0
        t["residual"][2] = -(t["delta"][2].float() / t["delta"][2].float().pow(2).mean().sqrt() * t["post"])
    got = run(t, d_stream, d_normed, 1.0, 1e-6)
    want = formulas(t["residual"], t["delta"], t["post"], t["pre"], None, 1.0, 1e-6, d_stream, d_normed.half())
    assert not got["stream"][0].any() and not got["normed"][0].any()
    for name in ("stream", "d_residual", "d_delta"):
        keep = [i for i in range(8) if i != 2]
        check(name, got[name][keep], want[name][0][keep], want[name][1][keep], 64)
    check("stream", got["stream"], *want["stream"], 64)
    assert got["d_delta"][1:].isfinite().all()      # (row 0: 1 / sqrt(eps) twice, beyond fp16)


def test_nan_and_infinity_stay_in_their_rows(cuda_lib):
    t, d_stream, d_normed = inputs(16, 128, torch.float16, 0, 4)
    clean = run(t, d_stream, d_normed, 1.0, 1e-6)
    with torch.no_grad():
        t["delta"][3, 5] = float("nan")
        t["residual"][7, 1] = float("inf")
    got = run(t, d_stream, d_normed, 1.0, 1e-6)
    rows = [i for i in range(16) if i not in (3, 7)]
    for name in ("stream", "normed", "d_residual", "d_delta"):
        assert torch.equal(got[name][rows], clean[name][rows])
    assert got["normed"][3].isnan().all() and got["normed"][7].isnan().any() and got["d_pre"].isnan().any()


def test_layouts(cuda_lib):
    """Leading dimensions, a gate row per sequence, other strides, odd addresses, broadcast weights."""
    from hackaton_b200 import sandwich_norm

    t, *_ = inputs(24, 96, torch.float16, 4, 6)
    t = {k: v.detach() for k, v in t.items()}
    want = sandwich_norm(t["residual"], t["delta"], t["post"], t["pre"], 1e-6, gate=t["gate"])
    got = sandwich_norm(t["residual"].view(4, 6, 96), t["delta"].view(4, 6, 96), t["post"], t["pre"], 1e-6,
                        gate=t["gate"].view(4, 1, 96))
    assert all(torch.equal(w.view(4, 6, 96), g) for w, g in zip(want, got))
    got = sandwich_norm(t["residual"].t().contiguous().t(), t["delta"].t().contiguous().t(), t["post"], t["pre"], 1e-6,
                        gate=t["gate"].t().contiguous().t())
    assert all(torch.equal(w, g) for w, g in zip(want, got))
    odd = torch.zeros(24 * 96 + 1, device="cuda")[1:].view(24, 96)
    odd.copy_(t["residual"])
    half = torch.zeros(24 * 96 + 1, device="cuda", dtype=torch.float16)[1:].view(24, 96)
    half.copy_(t["delta"])
    got = sandwich_norm(odd, half, t["post"], t["pre"], 1e-6, gate=t["gate"])
    ref = formulas(t["residual"], t["delta"], t["post"], t["pre"], t["gate"], 1.0, 1e-6)
    check("stream", got[0], *ref["stream"], 64)
    check("normed", got[1], *ref["normed"], 64)
    one = torch.ones(1, device="cuda").expand(96)
    got = sandwich_norm(t["residual"], t["delta"], one, one, 1e-6)
    ref = formulas(t["residual"], t["delta"], one, one, None, 1.0, 1e-6)
    check("normed", got[1], *ref["normed"], 64)


def test_only_what_is_asked_for(cuda_lib):
    """Each input's gradient alone equals the one among all; without rows everything is empty or zero."""
    from hackaton_b200 import sandwich_norm

    t, d_stream, d_normed = inputs(40, 256, torch.bfloat16, 1, 8)
    every = run(t, d_stream, d_normed, 0.5, 1e-6)
    for name in t:
        part = {k: (v if k == name else v.detach()) for k, v in t.items()}
        s, y = sandwich_norm(part["residual"], part["delta"], part["post"], part["pre"], 1e-6, gate=part["gate"],
                             residual_scale=0.5)
        (g,) = torch.autograd.grad([s, y], [part[name]], [d_stream, d_normed.to(y.dtype)])
        assert torch.equal(g, every["d_" + name]), name
    s, y = sandwich_norm(t["residual"], t["delta"], t["post"], t["pre"], 1e-6, gate=t["gate"], residual_scale=0.5)
    (alone,) = torch.autograd.grad(y, [t["delta"]], d_normed.to(y.dtype))     # nothing reaches the stream itself
    want = formulas(t["residual"], t["delta"], t["post"], t["pre"], t["gate"], 0.5, 1e-6, torch.zeros_like(d_stream),
                    d_normed.to(y.dtype))
    check("d_delta", alone, *want["d_delta"], 64)
    empty = {k: (v.detach()[:0] if k in ("residual", "delta") else v.detach()).requires_grad_() for k, v in t.items()}
    s, y = sandwich_norm(empty["residual"], empty["delta"], empty["post"], empty["pre"], 1e-6, gate=empty["gate"])
    grads = torch.autograd.grad([s, y], list(empty.values()), [torch.zeros_like(s), torch.zeros_like(y)])
    assert all(g.shape == v.shape and not g.any() for g, v in zip(grads, empty.values()))


def test_streams_and_graphs(cuda_lib):
    t, d_stream, d_normed = inputs(70, 512, torch.float16, 2, 9)
    d16 = d_normed.half()
    want = run(t, d_stream, d16, 0.5, 1e-6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, d_stream, d16, 0.5, 1e-6)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want[k], got[k]) for k in want)
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(t, d_stream, d16, 0.5, 1e-6)
    other, *_ = inputs(70, 512, torch.float16, 2, 10)
    with torch.no_grad():
        for k in t:
            t[k].copy_(other[k])
    graph.replay()
    now = run(t, d_stream, d16, 0.5, 1e-6)
    assert all(torch.equal(out[k], now[k]) for k in now)
