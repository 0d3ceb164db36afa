"""GPU: activations kept in 8 bits and what reads them (the SwiGLU backward, the gradient of a LoRA pair's first
factor) against plain implementations in 64 bits.

Bounds. The kept values are exact: equal to the 64-bit form's. One rounding to fp16 is 2^-11 of the value, or 2^-25
below fp16's normal range. The SwiGLU backward's fp32 arithmetic: __expf is off by 2 + |1.173 x| units in the last
place (2^-23 of the value), a handful of other operations by one each; |x| <= 90 here, so 120 * 2^-23 of the terms'
magnitudes. Sums of n products in fp32, in any order: n * 2^-23 of the sum of their magnitudes (a unit per addition)."""

import numpy as np
import pytest
import torch

from tests.util import synthetic_weight

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def kept_values(x):
    """What 8 bits hold of x, in numpy's 64 bits: (values, steps as exponents)."""
    x = x.detach().double().cpu().numpy()
    rows, cols = x.shape
    blocks = -(-cols // 32)
    b = np.zeros((rows, blocks * 32))
    b[:, :cols] = x
    b = b.reshape(rows, blocks, 32)
    finite = np.isfinite(b).all(axis=2, keepdims=True)
    top = np.where(finite, np.abs(b).max(axis=2, keepdims=True), 1.0)
    _, e = np.frexp(top)                      # top = m 2^e, 1/2 <= m < 1
    e = np.maximum(np.where(top > 0, e - 7, -126), -126)
    q = np.clip(np.rint(np.where(finite, b, 0.0) * np.exp2(-e.astype(np.float64))), -127, 127)
    v = np.where(finite, q * np.exp2(e.astype(np.float64)), np.nan)
    return torch.from_numpy(v.reshape(rows, -1)[:, :cols]), np.where(finite, e, 128)[..., 0]


def activations(rows, cols, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp2(
        torch.randint(-12, 6, (rows, max(1, -(-cols // 32))), device="cuda", generator=g).float()
    ).repeat_interleave(32, dim=1)[:, :cols]
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 96), (129, 1000), (64, 4096), (1, 100003)])
def test_kept_values_are_exact(cuda_lib, dtype, rows, cols):
    from hackaton_b200 import act8_dequantize, act8_quantize

    x = activations(rows, cols, dtype, rows + cols)
    kept = act8_quantize(x)
    want, exps = kept_values(x)
    assert kept.codes.shape == (rows, -(-cols // 32) * 32) and kept.steps.shape == (rows, -(-cols // 32))
    assert np.array_equal(kept.steps.cpu().numpy().astype(np.int64), exps + 127)
    got = act8_dequantize(kept)
    assert got.dtype == dtype and got.shape == x.shape
    assert torch.equal(got.double().cpu(), want)
    assert not kept.codes[:, cols:].any()


def test_kept_values_at_the_edges(cuda_lib):
    """Zeros, the types' largest and smallest values, blocks with an infinity or a NaN, ties, the top half step."""
    from hackaton_b200 import act8_dequantize, act8_quantize

    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        info = torch.finfo(dtype)
        for cols in (32, 33):           # whole blocks, and the path for any width
            x = torch.zeros(9, cols, device="cuda", dtype=dtype)
            x[1, 3] = info.max
            x[2, 4] = info.tiny
            x[3, 5] = info.smallest_normal * info.eps      # the smallest subnormal
            x[4, 6] = float("inf")
            x[5, 7] = float("nan")
            x[6, :4] = torch.tensor([127.75, 63.5, -0.5, 1.5], dtype=dtype)
            x[7, :3] = torch.tensor([-info.max, 1.0, 2.0], dtype=dtype)
            x[8, 0] = -float("inf")
            x[8, 1] = float("nan")
            got = act8_dequantize(act8_quantize(x)).double().cpu()
            want, _ = kept_values(x)
            assert torch.equal(got.nan_to_num(7.25), want.nan_to_num(7.25)), (dtype, cols)
            assert got[4, :32].isnan().all() and got[5, :32].isnan().all()


def test_layouts_shapes_and_empties(cuda_lib):
    from hackaton_b200 import act8_dequantize, act8_quantize

    x = activations(48, 256, torch.float16, 3)
    want = act8_dequantize(act8_quantize(x))
    assert torch.equal(act8_dequantize(act8_quantize(x.reshape(4, 3, 4, 256))), want.reshape(4, 3, 4, 256))
    assert torch.equal(act8_dequantize(act8_quantize(x.t().contiguous().t())), want)                # other strides
    wide = torch.zeros(48, 300, device="cuda", dtype=torch.float16)
    wide[:, 5:261] = x
    assert torch.equal(act8_dequantize(act8_quantize(wide[:, 5:261])), want)
    odd = torch.zeros(48 * 256 + 1, device="cuda", dtype=torch.float16)[1:].view(48, 256)            # an odd address
    odd.copy_(x)
    assert torch.equal(act8_dequantize(act8_quantize(odd)), want)
    for shape in ((0, 64), (3, 0), (0,)):
        empty = torch.empty(shape, device="cuda", dtype=torch.float16)
        assert act8_dequantize(act8_quantize(empty)).shape == empty.shape


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (17, 96), (333, 1000), (64, 8960)])
def test_swiglu_from_8_bits(cuda_lib, rows, cols):
    from hackaton_b200 import silu_mul

    gate, up = activations(rows, cols, torch.float16, 1), activations(rows, cols, torch.float16, 2)
    gate = gate.clamp(-60, 60)
    d = activations(rows, cols, torch.float16, 4).clamp(-4, 4)
    gate.requires_grad_()
    up.requires_grad_()
    hidden = silu_mul(gate, up, keep8=True)
    assert torch.equal(hidden, silu_mul(gate.detach(), up.detach()))
    d_gate, d_up = torch.autograd.grad(hidden, [gate, up], d)
    g8, u8 = (kept_values(t)[0] for t in (gate, up))
    d64 = d.double().cpu()
    sig = torch.sigmoid(g8)
    arith = 120 * 2.0 ** -23
    for got, want, terms in ((d_gate, d64 * u8 * sig * (1 + g8 * (1 - sig)), (d64 * u8 * sig).abs() * (1 + g8.abs())),
                             (d_up, d64 * g8 * sig, (d64 * g8 * sig).abs())):
        off = (got.double().cpu() - want).abs()
        assert (off <= want.abs() * 2.0 ** -11 + 2.0 ** -25 + arith * terms).all()


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 64), (15, 33), (16, 32), (17, 1000), (128, 96), (810, 1536), (5000, 200)])
def test_lora_gradient_from_8_bits(cuda_lib, rows, cols):
    from hackaton_b200 import act8_quantize, lora_grad_act8

    x = activations(rows, cols, torch.float16, 5)
    s = activations(rows, 16, torch.float16, 6)
    kept = act8_quantize(x)
    got = lora_grad_act8(kept, s)
    v, s64 = kept_values(x)[0], s.double().cpu()
    bound = rows * 2.0 ** -23 * (s64.abs().t() @ v.abs()) + 1e-45
    assert got.dtype == torch.float32 and ((got.double().cpu() - s64.t() @ v).abs() <= bound).all()
    assert torch.equal(got, lora_grad_act8(kept, s))                 # the same order of additions


def test_lora_gradient_of_tiny_and_huge_values(cuda_lib):
    """Blocks at both ends of fp16 keep their share of the gradient; a NaN shows in its own columns only."""
    from hackaton_b200 import act8_quantize, lora_grad_act8

    x = torch.zeros(20, 96, device="cuda", dtype=torch.float16)
    x[:, :32] = 2.0 ** -24
    x[:, 32:64] = 60000.0
    s = torch.ones(20, 16, device="cuda", dtype=torch.float16)
    s[:, 3] = 2.0 ** -24
    got = lora_grad_act8(act8_quantize(x), s).double().cpu()
    v, s64 = kept_values(x)[0], s.double().cpu()
    assert ((got - s64.t() @ v).abs() <= 20 * 2.0 ** -23 * (s64.t() @ v.abs())).all() and (got[:, :64] != 0).all()
    x[7, 70] = float("inf")
    got = lora_grad_act8(act8_quantize(x), s)
    assert got[:, 64:].isnan().all() and got[:, :64].isfinite().all()


def test_lora_gradient_without_rows(cuda_lib):
    from hackaton_b200 import act8_quantize, lora_grad_act8

    kept = act8_quantize(torch.empty(0, 64, device="cuda", dtype=torch.float16))
    got = lora_grad_act8(kept, torch.empty(0, 16, device="cuda", dtype=torch.float16))
    assert got.shape == (16, 64) and not got.any()


def lora_parts(n, k, seed):
    packed, state = synthetic_weight(n, k, True, seed=seed, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = (torch.randn(16, k, device="cuda", generator=g) / k ** 0.5).requires_grad_()
    b = (torch.randn(n, 16, device="cuda", generator=g) * 0.1).requires_grad_()
    return packed, state, a, b


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_lora_linear_keeps_its_input_in_8_bits(cuda_lib, rows):
    """keep8 changes the gradient of A alone, to what the kept values give."""
    from hackaton_b200 import nf4_lora_linear

    packed, state, a, b = lora_parts(128, 256, 9)
    x = activations(rows, 256, torch.float16, 7).clamp(-8, 8).requires_grad_()
    dy = activations(rows, 128, torch.float16, 8).clamp(-1, 1)
    want = nf4_lora_linear(x, packed, None, state, a, b, 2.0)
    got = nf4_lora_linear(x, packed, None, state, a, b, 2.0, keep8=True)
    assert torch.equal(want, got)
    kept = [t.dtype for t in got.grad_fn.saved_tensors]
    assert kept.count(torch.int8) == 1 and kept.count(torch.uint8) == 1
    gw = torch.autograd.grad(want, [x, a, b], dy)
    gg = torch.autograd.grad(got, [x, a, b], dy)
    assert torch.equal(gw[0], gg[0])
    assert torch.allclose(gw[2], gg[2], rtol=1e-5, atol=1e-5)       # (atomic sums of the same products)
    # u = s dy B in fp16 as the framework forms it: the 64-bit product is off by fp16's half step and fp32's sums
    u = 2.0 * dy.double() @ b.detach().half().double()
    ua = 2.0 * dy.double().abs() @ b.detach().half().double().abs()
    v = kept_values(x)[0].cuda()
    bound = (u.abs() * 2.0 ** -11 + 2.0 ** -25 + 160 * 2.0 ** -23 * ua).t() @ v.abs() + rows * 2.0 ** -23 * ua.t() @ v.abs()
    assert ((gg[1].double() - u.t() @ v).abs() <= bound).all()
    # nothing but A reads the input: without its gradient it is not kept at all
    frozen = nf4_lora_linear(x, packed, None, state, a.detach(), b, 2.0, keep8=True)
    assert not any(t.dtype == torch.int8 or t.shape == x.shape for t in frozen.grad_fn.saved_tensors)
    assert torch.equal(torch.autograd.grad(frozen, [x], dy)[0], gw[0])


def test_lora_linear_with_a_branch_of_its_own(cuda_lib):
    """x_lora other than x (dropout): both gradients, with x_lora kept in 8 bits."""
    from hackaton_b200 import nf4_lora_linear

    packed, state, a, b = lora_parts(128, 256, 10)
    x = activations(33, 256, torch.float16, 7).clamp(-4, 4).requires_grad_()
    x_l = (x.detach() * (torch.rand(33, 256, device="cuda") < 0.9)).requires_grad_()
    dy = activations(33, 128, torch.float16, 8).clamp(-1, 1)
    want = torch.autograd.grad(nf4_lora_linear(x, packed, None, state, a, b, 2.0, x_lora=x_l), [x, x_l, a], dy)
    got = torch.autograd.grad(nf4_lora_linear(x, packed, None, state, a, b, 2.0, x_lora=x_l, keep8=True), [x, x_l, a], dy)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    assert (want[2] - got[2]).norm() <= 2.0 ** -6 * want[2].norm()   # 2^-7 of each block's largest value at most


def test_group_keeps_its_input_once(cuda_lib):
    from hackaton_b200 import Projection, nf4_linear_group

    parts = [lora_parts(n, 256, 20 + n) for n in (128, 64, 64)]
    projs = [Projection(p, s, None, a, b, 2.0) for p, s, a, b in parts[:2]] + [Projection(*parts[2][:2])]
    x = activations(50, 256, torch.float16, 7).clamp(-8, 8).requires_grad_()
    dys = [activations(50, n, torch.float16, n).clamp(-1, 1) for n in (128, 64, 64)]
    leaves = [x] + [t for p in parts[:2] for t in p[2:]]
    want_y = nf4_linear_group(x, projs)
    got_y = nf4_linear_group(x, projs, keep8=True)
    assert all(torch.equal(w, g) for w, g in zip(want_y, got_y))
    assert sum(t.dtype == torch.int8 for t in got_y[0].grad_fn.saved_tensors) == 1
    want, got = torch.autograd.grad(want_y, leaves, dys), torch.autograd.grad(got_y, leaves, dys)
    assert torch.equal(want[0], got[0])
    for i in (1, 3):     # A: 2^-7 of each block's largest value at most, far less in the mean
        assert (want[i] - got[i]).norm() <= 2.0 ** -6 * want[i].norm()
    for i in (2, 4):
        assert torch.allclose(want[i], got[i], rtol=1e-5, atol=1e-5)
    plain = nf4_linear_group(x, [Projection(*parts[2][:2])], keep8=True)     # no pair: nothing to keep
    assert torch.autograd.grad(plain, [x], [dys[2]])[0].shape == x.shape


@pytest.mark.parametrize("lora", [False, True])
@pytest.mark.parametrize("rows", [5, 300])
def test_mlp_keeps_gate_and_up_in_8_bits(cuda_lib, lora, rows):
    from hackaton_b200 import Projection, nf4_swiglu_mlp

    shapes = [(512, 128), (512, 128), (128, 512)]
    projs, pairs = [], []
    for i, (n, k) in enumerate(shapes):
        packed, state, a, b = lora_parts(n, k, 30 + i)
        pairs += [a, b] if lora else []
        projs.append(Projection(packed, state, None, a, b, 2.0) if lora else Projection(packed, state))
    x = activations(rows, 128, torch.float16, 7).clamp(-8, 8).requires_grad_()
    dy = activations(rows, 128, torch.float16, 8).clamp(-1, 1)
    want, got = nf4_swiglu_mlp(x, *projs), nf4_swiglu_mlp(x, *projs, keep8=True)
    if not lora:
        assert torch.equal(want, got)
        assert sum(t.dtype == torch.int8 for t in got.grad_fn.saved_tensors) == 2
    gw, gg = torch.autograd.grad(want, [x] + pairs, dy), torch.autograd.grad(got, [x] + pairs, dy)
    for w, g in zip(gw, gg):      # gate, up, inputs: 2^-7 of each block's largest at most, summed over many
        assert (w - g).float().norm() <= 2.0 ** -5 * w.float().norm()
    with torch.no_grad():
        assert torch.equal(nf4_swiglu_mlp(x, *projs, keep8=True), nf4_swiglu_mlp(x, *projs))


def test_streams_and_graphs(cuda_lib):
    """On a stream of its own, and captured: replays with new inputs give what a direct call gives."""
    from hackaton_b200 import act8_quantize, lora_grad_act8, silu_mul

    x, s = activations(300, 640, torch.float16, 5), activations(300, 16, torch.float16, 6)
    want = lora_grad_act8(act8_quantize(x), s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lora_grad_act8(act8_quantize(x), s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
    gate = torch.zeros(64, 320, device="cuda", dtype=torch.float16, requires_grad=True)
    up = torch.zeros_like(gate, requires_grad=True)
    d = torch.zeros_like(gate.detach())
    xs, ss = torch.zeros_like(x), torch.zeros_like(s)

    def step():
        hidden = silu_mul(gate, up, keep8=True)
        return (hidden.detach(), *torch.autograd.grad(hidden, [gate, up], d), lora_grad_act8(act8_quantize(xs), ss))

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        with torch.no_grad():
            gate.copy_(activations(64, 320, torch.float16, seed))
            up.copy_(activations(64, 320, torch.float16, seed + 10))
            d.copy_(activations(64, 320, torch.float16, seed + 20))
            xs.copy_(activations(300, 640, torch.float16, seed))
            ss.copy_(activations(300, 16, torch.float16, seed + 1))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
