"""GPU: the operators as a model's layer runs them: norms around the blocks with gate and residual scale, grouped and
single projections with LoRA and the SwiGLU block, their inputs kept in 8 bits, and the loss from the hidden states; against
the same formulas in 64 bits.

Bounds, in norm. On a way through the layer fp16 roundings of at most 2^-11 of a tensor meet: three outputs of norms, four of
projections, their four inner products with 16 ranks, the two products of the mixing, the hidden values of the block: 14, which
no step here makes more than twice as large: 28 * 2^-11 < 2^-6 for what the head reads. A logit is then off by at most
2^-6 |h| |w| (Cauchy and Schwarz), a loss by twice the largest of them. A gradient meets as many on its way back, multiplies values of the
forward off as above, and where a factor was kept in 8 bits 2^-7 of each block's largest value, less than 4 of its
root mean square here, with a mean of a quarter of that: 2^-6 + 2^-6 + 4 * 2^-9 * 2 < 2^-4."""

import pytest
import torch

from util import synthetic_weight

pytestmark = pytest.mark.gpu

HIDDEN, INNER, VOCAB, SCALE = 128, 320, 1003, 0.7


def model(seed=0):
    from hackaton_b200 import Projection

    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    m = {"projs": {}, "weights": {}, "leaves": []}
    shapes = dict(q=(HIDDEN, HIDDEN), k=(HIDDEN, HIDDEN), v=(HIDDEN, HIDDEN), o=(HIDDEN, HIDDEN),
                  gate=(INNER, HIDDEN), up=(INNER, HIDDEN), down=(HIDDEN, INNER))
    for i, (name, (rows, cols)) in enumerate(shapes.items()):
        packed, state = synthetic_weight(rows, cols, True, seed=seed + i, device="cuda")
        a = (n(16, cols) / cols ** 0.5).requires_grad_()
        b = (n(rows, 16) * 0.05).requires_grad_()
        m["projs"][name] = Projection(packed, state, None, a, b, 2.0)
        m["leaves"] += [a, b]
    for name in ("post1", "pre1", "post2", "pre2"):
        m[name] = (1 + 0.2 * n(HIDDEN)).requires_grad_()
        m["leaves"].append(m[name])
    m["gates"] = (0.5 * n(4, HIDDEN)).requires_grad_()        # a row per sequence
    m["head"] = (n(VOCAB, HIDDEN) / HIDDEN ** 0.5).half().requires_grad_()
    m["leaves"] += [m["gates"], m["head"]]
    return m


def layer(m, residual, x, targets, keep8):
    """residual: fp32 [4, T, HIDDEN]; x: fp16, its norm -> (rows that the head reads, losses)."""
    from hackaton_b200 import nf4_linear_group, nf4_lora_linear, nf4_swiglu_mlp, sandwich_norm, vocab_cross_entropy

    p = m["projs"]
    q, k, v = nf4_linear_group(x, [p["q"], p["k"], p["v"]], keep8=keep8)
    mixed = torch.tanh(q * k) + v
    o = nf4_lora_linear(mixed, p["o"].packed, None, p["o"].state, p["o"].lora_a, p["o"].lora_b, 2.0, keep8=keep8)
    stream, x = sandwich_norm(residual, o, m["post1"], m["pre1"], 1e-6, gate=m["gates"].unsqueeze(1), residual_scale=SCALE)
    delta = nf4_swiglu_mlp(x, p["gate"], p["up"], p["down"], keep8=keep8)
    _, x = sandwich_norm(stream, delta, m["post2"], m["pre2"], 1e-6, residual_scale=SCALE)
    return x, vocab_cross_entropy(x, m["head"], targets)[0]


def plain(m, residual, x, targets):
    """The same in 64 bits, on copies of the leaves in m's order."""
    from hackaton_b200 import dequantize_nf4

    leaves = [t.detach().double().requires_grad_() for t in m["leaves"]]
    pairs = {name: leaves[2 * i:2 * i + 2] for i, name in enumerate(m["projs"])}
    post1, pre1, post2, pre2, gates, head = leaves[-6:]

    def linear(name, t):
        a, b = pairs[name]
        w = dequantize_nf4(m["projs"][name].packed, m["projs"][name].state).double()
        return t @ w.t() + 2.0 * t @ a.t() @ b.t()

    norm = lambda t, w: t * (t.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    residual, x = residual.detach().double().requires_grad_(), x.detach().double().requires_grad_()
    mixed = torch.tanh(linear("q", x) * linear("k", x)) + linear("v", x)
    stream = SCALE * residual + gates.unsqueeze(1) * norm(linear("o", mixed), post1)
    t = norm(stream, pre1)
    hidden = torch.nn.functional.silu(linear("gate", t)) * linear("up", t)
    stream = SCALE * stream + norm(linear("down", hidden), post2)
    h = norm(stream, pre2)
    logits = h @ head.t()
    losses = torch.logsumexp(logits, -1) - logits.gather(-1, targets.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    return h, torch.where(targets >= 0, losses, torch.zeros_like(losses)), leaves + [residual, x]


def batch(tokens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    residual = torch.randn(4, tokens, HIDDEN, device="cuda", generator=g)
    x = (residual * (residual.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()).half()
    targets = torch.randint(0, VOCAB, (4, tokens), device="cuda", generator=g)
    targets[torch.rand(4, tokens, device="cuda", generator=g) < 0.3] = -100
    targets[1, :] = -100             # a sequence of which nothing is learnt
    targets[0, 0] = 5
    return residual.requires_grad_(), x.requires_grad_(), targets


def off(got, want):
    return float((got.detach().double() - want.detach()).norm() / want.detach().norm())


@pytest.mark.parametrize("tokens", [1, 37, 150])
@pytest.mark.parametrize("keep8", [False, True])
def test_layer_and_its_gradients(cuda_lib, tokens, keep8):
    m = model()
    residual, x, targets = batch(tokens, 1)
    h, losses = layer(m, residual, x, targets, keep8)
    h64, losses64, leaves64 = plain(m, residual, x, targets)
    assert off(h, h64) <= 2.0 ** -6
    reach = (h.detach().double() - h64.detach()).norm(dim=-1) * m["head"].detach().double().norm(dim=-1).max()
    assert ((losses.double() - losses64).abs() <= 2 * reach + 1e-4).all()
    assert torch.equal(losses[targets < 0], torch.zeros_like(losses[targets < 0]))
    grads = torch.autograd.grad(losses.sum() * 16, m["leaves"] + [residual, x])
    want = torch.autograd.grad(losses64.sum() * 16, leaves64)
    for i, (g, w) in enumerate(zip(grads, want)):
        assert off(g, w) <= 2.0 ** -4, i
    cuda_lib.device_status()


def test_what_the_backward_holds(cuda_lib):
    """With keep8 the layer's forward leaves less behind: 33 for 64 bytes per value of every kept 16-bit tensor."""
    m = model()
    residual, x, targets = batch(150, 1)
    held = []
    for keep8 in (False, True):
        kept = {}

        def pack(t):
            kept[t.untyped_storage().data_ptr()] = t.numel() * t.element_size()
            return t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            layer(m, residual, x, targets, keep8)
        held.append(sum(kept.values()))
    rows = 600
    # gate, up, the hidden values and the input of the block in 8 bits for certain
    assert held[0] - held[1] >= rows * (3 * INNER + HIDDEN) * 2 * 31 // 64


def test_single_tokens_without_gradients(cuda_lib):
    m = model()
    residual, x, targets = batch(1, 3)
    with torch.no_grad():
        h, losses = layer(m, residual, x, targets, True)
        h2, losses2 = layer(m, residual, x, targets, False)
    assert torch.equal(h, h2) and torch.equal(losses, losses2)
    h64, losses64, _ = plain(m, residual, x, targets)
    assert off(h, h64) <= 2.0 ** -6
    reach = (h.double() - h64.detach()).norm(dim=-1) * m["head"].detach().double().norm(dim=-1).max()
    assert ((losses.double() - losses64.detach()).abs() <= 2 * reach + 1e-4).all()


def test_a_captured_training_step(cuda_lib):
    """Forward and backward of the layer captured; replays on other batches give what direct calls give, but for the order
    in which the LoRA factors' kernels add (each sum of 600 products: 600 * 2^-23 of its terms at most)."""
    m = model()
    residual, x, targets = batch(150, 5)

    def step():
        h, losses = layer(m, residual, x, targets, True)
        return (h.detach(), losses.detach(), *torch.autograd.grad(losses.sum() * 16, m["leaves"] + [residual, x]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (6, 7):
        new = batch(150, seed)
        with torch.no_grad():
            for t, v in zip((residual, x, targets), new):
                t.copy_(v)
        graph.replay()
        for i, (o, w) in enumerate(zip(out, step())):
            assert off(o, w.double()) <= 2.0 ** -12, i
        assert torch.equal(out[0], step()[0]) and torch.equal(out[1], step()[1])
    cuda_lib.device_status()


def test_gradients_of_gradients_are_refused(cuda_lib):
    from hackaton_b200 import sandwich_norm, silu_mul, vocab_cross_entropy

    ones = torch.ones(64, device="cuda")
    x = torch.ones(4, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    calls = (lambda: silu_mul(x, x, keep8=True), lambda: sandwich_norm(x.detach().float(), x, ones, ones, 1e-6)[0],
             lambda: vocab_cross_entropy(x, x.detach(), torch.zeros(4, dtype=torch.int64, device="cuda"))[0])
    for call in calls:
        with pytest.raises(NotImplementedError, match="second derivative"):
            torch.autograd.grad(call().sum(), [x], create_graph=True)


def test_parts_of_kept_activations_that_do_not_fit(cuda_lib):
    from hackaton_b200 import act8_dequantize, act8_quantize, lora_grad_act8
    from hackaton_b200.act8 import Act8

    kept = act8_quantize(torch.ones(6, 64, device="cuda", dtype=torch.float16))
    s = torch.ones(6, 16, device="cuda", dtype=torch.float16)
    wrong = [(kept.codes[:5], kept.steps, (5, 64)), (kept.codes, kept.steps, (7, 64)), (kept.codes, kept.steps, (6, 65)),
             (kept.codes, kept.steps, (6, 32)), (kept.codes, kept.steps, ()), (kept.codes.view(torch.uint8), kept.steps, (6, 64)),
             (kept.codes.t().contiguous().t(), kept.steps, (6, 64)), (kept.codes, kept.steps.cpu(), (6, 64)),
             (kept.codes, kept.steps[:, :1], (6, 64))]
    for codes, steps, shape in wrong:
        with pytest.raises(ValueError):
            act8_dequantize(Act8(codes, steps, shape, torch.float16))
    for codes, steps, shape in wrong:
        if shape and shape[0] != 7:
            with pytest.raises(ValueError):
                lora_grad_act8(Act8(codes, steps, shape, torch.float16), s)
    with pytest.raises(TypeError):
        act8_dequantize(Act8(kept.codes, kept.steps, (6, 64), torch.float64))
