"""GPU: what the operators around a training step answer to calls beside the usual one."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from test_act8_gpu import activations, lora_parts

pytestmark = pytest.mark.gpu


def test_forward_mode_is_refused(cuda_lib):
    """A tangent is not dropped silently, with gradients on or off, whichever operand carries it."""
    from hackaton_b200 import act8_quantize, lora_grad_act8, sandwich_norm, silu_mul, vocab_cross_entropy

    x = activations(4, 64, torch.float16).clamp(-4, 4)
    s = activations(4, 16, torch.float16).clamp(-4, 4)
    ones, t = torch.ones(64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    kept = act8_quantize(x)
    calls = [lambda d: vocab_cross_entropy(d(x), x, t), lambda d: vocab_cross_entropy(x, d(x), t),
             lambda d: sandwich_norm(d(x.float()), x, ones, ones, 1e-6), lambda d: sandwich_norm(x.float(), d(x), ones, ones, 1e-6),
             lambda d: sandwich_norm(x.float(), x, d(ones), ones, 1e-6), lambda d: sandwich_norm(x.float(), x, ones, d(ones), 1e-6),
             lambda d: sandwich_norm(x.float(), x, ones, ones, 1e-6, gate=d(ones)),
             lambda d: silu_mul(d(x), x, keep8=True), lambda d: silu_mul(x, d(x.clone().requires_grad_()), keep8=True),
             lambda d: act8_quantize(d(x)), lambda d: lora_grad_act8(kept, d(s))]
    with fwad.dual_level():
        dual = lambda v: fwad.make_dual(v, torch.ones_like(v))
        for call in calls:
            call(lambda v: v)
            with pytest.raises(RuntimeError):        # (NotImplementedError is one)
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError):
                call(dual)


def test_outputs_can_be_changed_in_place(cuda_lib):
    from hackaton_b200 import sandwich_norm, silu_mul, vocab_cross_entropy

    g, u = (activations(6, 64, torch.float16, k).clamp(-4, 4).requires_grad_() for k in (1, 2))
    for shape in ((6, 64), (2, 3, 64)):
        want = torch.autograd.grad((silu_mul(g.view(shape), u.view(shape), keep8=True) * 2).sum(), [g, u])
        got = silu_mul(g.view(shape), u.view(shape), keep8=True)
        got.mul_(2)
        assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(got.sum(), [g, u])))
        w = torch.ones(5, 64, device="cuda", dtype=torch.float16)
        t = torch.arange(6, device="cuda").view(shape[:-1]) % 5
        mask = (t > 1).float()
        losses, lse = vocab_cross_entropy(g.view(*shape), w, t)
        want = torch.autograd.grad((losses * mask).sum() + (lse * 3).sum(), [g])[0]
        losses, lse = vocab_cross_entropy(g.view(*shape), w, t)
        losses.mul_(mask)
        lse *= 3
        assert torch.equal(want, torch.autograd.grad(losses.sum() + lse.sum(), [g])[0])
    ones = torch.ones(64, device="cuda")
    stream, normed = sandwich_norm(g.detach().float(), u, ones, ones, 1e-6)
    want = torch.autograd.grad((normed * 2).sum(), [u])[0]
    stream, normed = sandwich_norm(g.detach().float(), u, ones, ones, 1e-6)
    normed.mul_(2)
    assert torch.equal(want, torch.autograd.grad(normed.sum(), [u])[0])


def test_nothing_is_kept_without_gradients(cuda_lib, monkeypatch):
    """An evaluation pass with trainable factors does not quantise what no backward will read."""
    from hackaton_b200 import Projection, act8, group, lora, mlp, nf4_linear_group, nf4_lora_linear, nf4_swiglu_mlp

    packed, state, a, b = lora_parts(128, 256, 9)
    x = activations(40, 256, torch.float16, 7).clamp(-8, 8)
    gate, up, down = (Projection(*lora_parts(n, k, 30 + i)[:2]) for i, (n, k) in enumerate(((512, 256), (512, 256), (256, 512))))
    pair = Projection(packed, state, None, a, b, 2.0)
    calls = [lambda v: nf4_lora_linear(v, packed, None, state, a, b, 2.0, keep8=True), lambda v: nf4_linear_group(v, [pair], keep8=True)[0],
             lambda v: nf4_swiglu_mlp(v, gate, up, down, keep8=True)]
    want = [call(x.clone().requires_grad_()) for call in calls]
    quantised = []
    for module in (lora, group, mlp):
        monkeypatch.setattr(module, "act8_quantize", lambda t: quantised.append(t.shape) or act8.act8_quantize(t))
    for w, call in zip(want, calls):
        with torch.no_grad():
            assert torch.equal(w, call(x.clone().requires_grad_()))
        assert not quantised
    assert calls[0](x.clone().requires_grad_()).requires_grad and quantised


def test_checkpoints_and_saved_tensors_elsewhere(cuda_lib):
    """Run again for the backward, or with what is saved moved to the host meanwhile: the same gradients."""
    from torch.utils.checkpoint import checkpoint

    from hackaton_b200 import sandwich_norm, silu_mul, vocab_cross_entropy

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(40, 64, device="cuda", generator=g).half().requires_grad_()
    ones = torch.ones(64, device="cuda").requires_grad_()
    head = torch.randn(300, 64, device="cuda", generator=g).half().requires_grad_()
    t = torch.randint(0, 300, (40,), device="cuda", generator=g)

    def loss(x, ones, head):
        stream, y = sandwich_norm(x.float(), silu_mul(x, x, keep8=True), ones, ones, 1e-6)
        return vocab_cross_entropy(y, head, t)[0].sum() + stream.mean()

    leaves = [x, ones, head]
    want = torch.autograd.grad(loss(*leaves), leaves)
    again = torch.autograd.grad(checkpoint(loss, *leaves, use_reentrant=False), leaves)
    with torch.autograd.graph.save_on_cpu():
        moved = loss(*leaves)
    moved = torch.autograd.grad(moved, leaves)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, again, moved))
