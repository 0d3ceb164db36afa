"""Cases of the operators that make a fine-tuning step leaner: the loss from the hidden states in pieces of
the vocabulary, norms before and after a block with its gate and residual scale, and activations kept in
8 bits with their use in the backward pass.

Sizes are those of the networks that the package's tests and benchmark use (hidden 1536 / MLP 8960, hidden
3584 / MLP 18944, vocabulary 151,936), and ragged ones around them. `listed` names the fixed cases, `draw` makes
others from the same ranges, `prepare` builds what a program holds before the call, `run` is one pass (in plain
torch operations, or with `own` through the package), `exact` the same result in 64 bits, `work` the bytes and
operations that a pass cannot do without.
"""

import math

import torch

own = False

EPS = 1e-6
BLOCK = 32                  # values of a row that share a step
RANK = 16
IGNORE = -100
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LARGEST = 2048 * 151936 * 1536      # rows * vocabulary * features of the largest loss


def listed():
    return [
        # a few rows over a small odd vocabulary: all latency
        {"name": "loss_small_odd", "kind": "loss", "dtype": "fp16", "rows": 61, "vocab": 1003, "hidden": 128,
         "ignored": 0.25, "grad_head": True, "z": 0.0, "train": True},
        # log probabilities of an answer of 64 tokens under the larger network, nothing to differentiate
        {"name": "loss_score_large", "kind": "loss", "dtype": "fp16", "rows": 64, "vocab": 151936, "hidden": 3584,
         "ignored": 0.0, "grad_head": False, "z": 0.0, "train": False},
        # fine-tuning with a frozen head: four sequences of 512, all tokens but the first of each are trained on
        {"name": "loss_frozen_head", "kind": "loss", "dtype": "fp16", "rows": 2048, "vocab": 151936, "hidden": 1536,
         "ignored": 0.002, "grad_head": False, "z": 0.0, "train": True},
        # fine-tuning with the head trained too, in bf16, prompts masked out, the normaliser kept small: the largest call
        {"name": "loss_trained_head", "kind": "loss", "dtype": "bf16", "rows": 2048, "vocab": 151936, "hidden": 1536,
         "ignored": 0.4, "grad_head": True, "z": 1e-4, "train": True},
        # the norms around a block for three new tokens
        {"name": "norm_decode", "kind": "norm", "dtype": "fp16", "rows": 3, "hidden": 3584, "gates": 1, "scale": 1.0,
         "train": False},
        # a training batch of packed tokens, a gate per channel, all weights trained
        {"name": "norm_train", "kind": "norm", "dtype": "fp16", "rows": 16384, "hidden": 1536, "gates": 1,
         "scale": 0.5, "train": True},
        # a gate row per sequence (four sequences of 1021 tokens), bf16, the larger network
        {"name": "norm_train_gated", "kind": "norm", "dtype": "bf16", "rows": 4084, "hidden": 3584, "gates": 4,
         "scale": 1.0, "train": True},
        # the MLP product of a ragged batch, gate and up kept in 8 bits
        {"name": "swiglu_ragged", "kind": "swiglu", "dtype": "fp16", "rows": 333, "width": 1000},
        # the same for a training batch
        {"name": "swiglu_train", "kind": "swiglu", "dtype": "fp16", "rows": 4096, "width": 8960},
        # the input of a LoRA linear kept in 8 bits, read back, and the factor's gradient from it: a packed batch
        {"name": "kept_packed", "kind": "kept", "dtype": "fp16", "rows": 810, "width": 1536},
        # the same for a long batch
        {"name": "kept_train", "kind": "kept", "dtype": "fp16", "rows": 16384, "width": 3584},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "norm", "swiglu", "kept"])
    if kind == "loss":
        while True:
            rows, vocab = _log_uniform(rng, 1, 2500), _log_uniform(rng, 300, 160000)
            hidden = 8 * _log_uniform(rng, 8, 512)
            if rows * vocab * hidden <= LARGEST * 0.9:
                break
        train = rng.random() < 0.75
        return {"kind": kind, "dtype": rng.choice(["fp16", "bf16"]), "rows": rows, "vocab": vocab, "hidden": hidden,
                "ignored": rng.choice([0.0, 0.1, 0.5]), "grad_head": train and rng.random() < 0.5,
                "z": rng.choice([0.0, 1e-4]), "train": train}
    if kind == "norm":
        hidden = rng.choice([8 * _log_uniform(rng, 8, 1024), _log_uniform(rng, 60, 5000)])
        rows = _log_uniform(rng, 1, max(1, min(20000, 16384 * 1536 // hidden)))
        gates = rng.choice([0, 1, 1, rows, max(1, min(rows, 4))])
        if gates:
            rows = max(gates, rows // gates * gates)
        return {"kind": kind, "dtype": rng.choice(["fp16", "bf16", "fp32"]), "rows": rows, "hidden": hidden,
                "gates": gates, "scale": rng.choice([1.0, 0.5, 1.25]), "train": rng.random() < 0.75}
    width = rng.choice([8 * _log_uniform(rng, 8, 2500), _log_uniform(rng, 33, 9000)])
    rows = _log_uniform(rng, 1, max(1, min(20000, 4096 * 8960 // width)))
    return {"kind": kind, "dtype": "fp16", "rows": rows, "width": width}


# ---------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _with_outliers(g, rows, width, spread):
    """Activations as they are found: a few channels many times the others, each row with a size of its own."""
    x = _normal(g, rows, width) * spread * torch.exp(0.3 * _normal(g, rows, 1))
    channel = torch.rand(width, generator=g, device="cuda")
    return x * torch.where(channel < 0.01, 20.0, 1.0)


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    dtype = DTYPES[case["dtype"]]
    if kind == "loss":
        rows, vocab, width = case["rows"], case["vocab"], case["hidden"]
        weight = _normal(g, vocab, width) * (1.6 / math.sqrt(width))
        targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        # what a trained network gives its targets: from nothing to near certainty
        lift = 20.0 * torch.rand(rows, 1, generator=g, device="cuda")
        towards = weight[targets]
        hidden = _normal(g, rows, width) + lift * towards / (towards * towards).sum(dim=1, keepdim=True)
        skipped = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
        skipped[0] = False
        targets = torch.where(skipped, IGNORE, targets)
        # mixed precision in fp16 multiplies the loss so that small gradients stay normal numbers
        factor = (16384.0 if dtype == torch.float16 else 1.0) / float((targets >= 0).sum())
        return {"kind": kind, "case": case, "hidden": hidden.to(dtype).requires_grad_(case["train"]),
                "weight": weight.to(dtype).requires_grad_(case["grad_head"]), "targets": targets, "factor": factor}
    if kind == "norm":
        rows, width = case["rows"], case["hidden"]
        train = case["train"]
        state = {"kind": kind, "case": case,
                 "residual": _with_outliers(g, rows, width, 2.0).requires_grad_(train),
                 "delta": _with_outliers(g, rows, width, 0.5).to(dtype).requires_grad_(train),
                 "post": (1.0 + 0.2 * _normal(g, width)).requires_grad_(train),
                 "pre": (1.0 + 0.2 * _normal(g, width)).requires_grad_(train), "gate": None}
        if case["gates"]:
            state["gate"] = (0.3 * _normal(g, case["gates"], width)).requires_grad_(train)
        if train:
            state["d_stream"] = _normal(g, rows, width)
            state["d_normed"] = _normal(g, rows, width).to(dtype)
        return state
    rows, width = case["rows"], case["width"]
    if kind == "swiglu":
        return {"kind": kind, "case": case, "gate": _with_outliers(g, rows, width, 1.0).to(dtype).requires_grad_(),
                "up": _with_outliers(g, rows, width, 0.7).to(dtype).requires_grad_(),
                "d_hidden": _normal(g, rows, width).to(dtype)}
    return {"kind": kind, "case": case, "x": _with_outliers(g, rows, width, 1.0).to(dtype),
            "u": (_normal(g, rows, RANK) * 0.5).to(dtype)}


# ------------------------------------------------------------------------------------- the plain forms

def _kept_values(x):
    """What 8 bits hold of fp32 `x`: blocks of 32 values of a row, a power of two as their step."""
    rows, width = x.shape
    blocks = (width + BLOCK - 1) // BLOCK
    padded = torch.zeros(rows, blocks * BLOCK, dtype=x.dtype, device=x.device)
    padded[:, :width] = x
    b = padded.reshape(rows, blocks, BLOCK)
    top = b.abs().amax(dim=2, keepdim=True)
    _, exponent = torch.frexp(top)                      # top = m * 2^exponent, 0.5 <= m < 1
    step = (((exponent - 7).clamp(min=-126) + 127) << 23).view(torch.float32)
    q = (b / step).round().clamp(-127.0, 127.0)
    return (q * step).reshape(rows, blocks * BLOCK)[:, :width]


def _plain_loss(s):
    case = s["case"]
    hidden, weight, targets = s["hidden"].detach(), s["weight"].detach(), s["targets"]
    h, w = hidden.float(), weight.float()
    valid = targets >= 0
    logits = h @ w.t()
    top = logits.amax(dim=1, keepdim=True)
    lse = (logits - top).exp().sum(dim=1).log() + top[:, 0]
    at = targets.clamp(min=0)
    picked = torch.gather(logits, 1, at[:, None])[:, 0]
    losses = torch.where(valid, lse - picked, 0.0)
    out = {"losses": losses, "lse": torch.where(valid, lse, 0.0)}
    if not case["train"]:
        return out
    # loss = factor * (sum of losses + z * sum of lse^2)
    b = torch.where(valid, s["factor"], 0.0)
    c = torch.where(valid, 2.0 * case["z"] * s["factor"] * lse, 0.0)
    p = (logits - lse[:, None]).exp_()
    p *= (b + c)[:, None]
    p.scatter_add_(1, at[:, None], -b[:, None])
    out["d_hidden"] = (p @ w).to(hidden.dtype)
    if case["grad_head"]:
        out["d_weight"] = (p.t() @ h).to(weight.dtype)
    return out


def _gate_rows(gate, rows):
    """The gate row of each row, as a tensor that broadcasts."""
    return gate.repeat_interleave(rows // gate.shape[0], dim=0) if gate.shape[0] > 1 else gate


def _plain_norm(s):
    case = s["case"]
    rows = case["rows"]
    r, d = s["residual"].detach(), s["delta"].detach().float()
    post, pre = s["post"].detach(), s["pre"].detach()
    rstd_d = torch.rsqrt((d * d).mean(dim=1, keepdim=True) + EPS)
    dhat = d * rstd_d
    n = dhat * post
    gate = None if s["gate"] is None else _gate_rows(s["gate"].detach(), rows)
    stream = case["scale"] * r + (n if gate is None else gate * n)
    rstd_s = torch.rsqrt((stream * stream).mean(dim=1, keepdim=True) + EPS)
    shat = stream * rstd_s
    dtype = s["delta"].dtype
    out = {"stream": stream, "normed": (shat * pre).to(dtype)}
    if not case["train"]:
        return out
    dy = s["d_normed"].float()
    w = dy * pre
    ds = s["d_stream"] + rstd_s * (w - shat * (w * shat).mean(dim=1, keepdim=True))
    out["d_residual"] = case["scale"] * ds
    dn = ds if gate is None else ds * gate
    q = dn * post
    out["d_delta"] = (rstd_d * (q - dhat * (q * dhat).mean(dim=1, keepdim=True))).to(dtype)
    out["d_post"] = (dn * dhat).sum(dim=0)
    out["d_pre"] = (dy * shat).sum(dim=0)
    if gate is not None:
        out["d_gate"] = (ds * n).reshape(case["gates"], rows // case["gates"], case["hidden"]).sum(dim=1)
    return out


def _plain_swiglu(s):
    g, u, d = s["gate"].detach().float(), s["up"].detach().float(), s["d_hidden"].float()
    hidden = g / (1.0 + (-g).exp()) * u
    g8, u8 = _kept_values(g), _kept_values(u)
    sig = 1.0 / (1.0 + (-g8).exp())
    dtype = s["gate"].dtype
    return {"hidden": hidden.to(dtype), "d_gate": (d * u8 * sig * (1.0 + g8 * (1.0 - sig))).to(dtype),
            "d_up": (d * g8 * sig).to(dtype)}


def _plain_kept(s):
    kept = _kept_values(s["x"].float())
    return {"values": kept.to(s["x"].dtype), "grad": s["u"].float().t() @ kept}


_PLAIN = {"loss": _plain_loss, "norm": _plain_norm, "swiglu": _plain_swiglu, "kept": _plain_kept}


# ------------------------------------------------------------------------------- the package's operators

def _own_loss(s):
    import hackaton_b200

    case = s["case"]
    hidden, weight = s["hidden"], s["weight"]
    losses, lse = hackaton_b200.vocab_cross_entropy(hidden, weight, s["targets"])
    out = {"losses": losses.detach(), "lse": lse.detach()}
    if not case["train"]:
        return out
    loss = losses.sum() * s["factor"]
    if case["z"]:
        loss = loss + (case["z"] * s["factor"]) * (lse * lse).sum()
    if case["grad_head"]:
        out["d_hidden"], out["d_weight"] = torch.autograd.grad(loss, [hidden, weight])
    else:
        (out["d_hidden"],) = torch.autograd.grad(loss, [hidden])
    return out


def _own_norm(s):
    import hackaton_b200

    stream, normed = hackaton_b200.sandwich_norm(s["residual"], s["delta"], s["post"], s["pre"], EPS, gate=s["gate"],
                                                 residual_scale=s["case"]["scale"], out_dtype=s["delta"].dtype)
    out = {"stream": stream.detach(), "normed": normed.detach()}
    if not s["case"]["train"]:
        return out
    wanted = ["residual", "delta", "post", "pre"] + ([] if s["gate"] is None else ["gate"])
    grads = torch.autograd.grad([stream, normed], [s[name] for name in wanted], [s["d_stream"], s["d_normed"]])
    out.update({"d_" + name: grad for name, grad in zip(wanted, grads)})
    return out


def _own_swiglu(s):
    import hackaton_b200

    hidden = hackaton_b200.silu_mul(s["gate"], s["up"], keep8=True)
    d_gate, d_up = torch.autograd.grad(hidden, [s["gate"], s["up"]], s["d_hidden"])
    return {"hidden": hidden.detach(), "d_gate": d_gate, "d_up": d_up}


def _own_kept(s):
    import hackaton_b200

    kept = hackaton_b200.act8_quantize(s["x"])
    return {"values": hackaton_b200.act8_dequantize(kept), "grad": hackaton_b200.lora_grad_act8(kept, s["u"])}


_OWN = {"loss": _own_loss, "norm": _own_norm, "swiglu": _own_swiglu, "kept": _own_kept}


def run(state):
    if own:
        return _OWN[state["kind"]](state)
    return _PLAIN[state["kind"]](state)


# ------------------------------------------------------------------------------------------ in 64 bits

def _exact_kept(x):
    rows, width = x.shape
    blocks = -(-width // BLOCK)
    x = torch.nn.functional.pad(x.double(), (0, blocks * BLOCK - width)).view(rows, blocks, BLOCK)
    top = x.abs().max(dim=2, keepdim=True).values
    power = torch.where(top > 0, top, torch.ones_like(top)).log2().floor()
    power = torch.where(torch.exp2(power) > top, power - 1, power)         # (a rounded logarithm next to a power of two)
    power = torch.where(torch.exp2(power + 1) <= top, power + 1, power)
    step = ((power.long() - 6).clamp(min=-126) + 1023).bitwise_left_shift(52).view(torch.float64)
    q = torch.minimum(torch.maximum((x / step).round(), x.new_tensor(-127.0)), x.new_tensor(127.0))
    return (q * step).view(rows, blocks * BLOCK)[:, :width]


def _exact_loss(s):
    case = s["case"]
    h, w, targets = s["hidden"].detach().double(), s["weight"].detach().double(), s["targets"]
    valid = (targets >= 0).nonzero()[:, 0]
    rows = len(targets)
    t = targets[valid]
    logits = h[valid] @ w.t()
    lse_v = torch.logsumexp(logits, dim=1)
    losses, lse = h.new_zeros(rows), h.new_zeros(rows)
    losses[valid] = lse_v - logits[torch.arange(len(t), device=t.device), t]
    lse[valid] = lse_v
    out = {"losses": losses, "lse": lse}
    if not case["train"]:
        return out
    d = torch.softmax(logits, dim=1)
    del logits
    d *= (s["factor"] * (1.0 + 2.0 * case["z"] * lse_v))[:, None]
    d[torch.arange(len(t), device=t.device), t] -= s["factor"]
    d_hidden = torch.zeros_like(h)
    d_hidden[valid] = d @ w
    out["d_hidden"] = d_hidden
    if case["grad_head"]:
        out["d_weight"] = d.t() @ h[valid]
    return out


def _exact_norm(s):
    case = s["case"]
    rows, width = case["rows"], case["hidden"]
    groups = max(1, case["gates"])

    def rms(x):
        return ((x * x).sum(dim=-1, keepdim=True) / width + EPS).sqrt()

    def rms_back(x, upstream):     # gradient through x / rms(x)
        r = rms(x)
        return upstream / r - x * (upstream * x).sum(dim=-1, keepdim=True) / (width * r ** 3)

    cut = (groups, rows // groups, width)
    d, r = s["delta"].detach().double().view(cut), s["residual"].detach().double().view(cut)
    post, pre = s["post"].detach().double(), s["pre"].detach().double()
    gate = torch.ones(groups, 1, width, dtype=torch.float64, device=d.device)
    if s["gate"] is not None:
        gate = s["gate"].detach().double().view(groups, 1, width)
    dn = d / rms(d)
    stream = case["scale"] * r + gate * (dn * post)
    sn = stream / rms(stream)
    out = {"stream": stream.view(rows, width), "normed": (sn * pre).view(rows, width)}
    if not case["train"]:
        return out
    dy = s["d_normed"].double().view(cut)
    ds = s["d_stream"].double().view(cut) + rms_back(stream, dy * pre)
    out["d_residual"] = (ds * case["scale"]).view(rows, width)
    out["d_delta"] = rms_back(d, ds * gate * post).view(rows, width)
    out["d_post"] = (ds * gate * dn).sum(dim=(0, 1))
    out["d_pre"] = (dy * sn).sum(dim=(0, 1))
    if s["gate"] is not None:
        out["d_gate"] = (ds * dn * post).sum(dim=1)
    return out


def _exact_swiglu(s):
    g, u, d = s["gate"].detach().double(), s["up"].detach().double(), s["d_hidden"].double()
    g8, u8 = _exact_kept(g), _exact_kept(u)
    sig = torch.sigmoid(g8)
    return {"hidden": torch.sigmoid(g) * g * u, "d_gate": d * u8 * (sig + g8 * sig * (1.0 - sig)),
            "d_up": d * (g8 * sig)}


def _exact_kept_case(s):
    kept = _exact_kept(s["x"])
    return {"values": kept, "grad": s["u"].double().t() @ kept}


def exact(case, seed):
    state = prepare(case, seed)
    return {"loss": _exact_loss, "norm": _exact_norm, "swiglu": _exact_swiglu, "kept": _exact_kept_case}[case["kind"]](state)


# ----------------------------------------------------------------------------------------------- the work

def work(case):
    kind = case["kind"]
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
    rows = case["rows"]
    if kind == "loss":
        # rows that are ignored need neither reading nor products
        active = max(1.0, rows * (1.0 - case["ignored"]))
        vocab, width = case["vocab"], case["hidden"]
        product = 2.0 * active * vocab * width
        moved = (active + vocab) * width * size + rows * 16
        products = 1
        if case["train"]:
            moved += rows * width * size
            products += 1
        if case["grad_head"]:
            moved += vocab * width * size
            products += 1
        return {"bytes": moved, "flops": products * product}
    if kind == "norm":
        n = rows * case["hidden"]
        side = (2 + case["gates"]) * case["hidden"] * 4
        moved, flops = n * (8 + 2 * size) + side, 10 * n
        if case["train"]:
            moved += n * (8 + 2 * size) + side       # d_stream, d_normed; d_residual, d_delta
            flops += 24 * n
        return {"bytes": moved, "flops": flops}
    n = rows * case["width"]
    # (what is kept in 8 bits between the two directions is neither an input nor an output of a pass)
    if kind == "swiglu":
        return {"bytes": n * 6 * size, "flops": 25 * n}
    return {"bytes": 2 * n * size + rows * RANK * size + case["width"] * RANK * 4, "flops": (2 * RANK + 6) * n}
