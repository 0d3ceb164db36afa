"""GPU: cross-entropy from the hidden states in pieces of the vocabulary, both directions, against the formulas in 64 bits.

Bounds. A product of two 16-bit numbers is exact in fp32; a sum of n of them in the tensor cores is off by at most a unit
(2^-23) of the sum of magnitudes per addition: eta = K 2^-23 max_v sum |h w| for a row's logits. lse adds the base-2
arithmetic (four units of the largest |logit|) and sums whose chains are under 64 additions. The gradient of a logit is
off by 2 eta + that in relative terms, then rounded to 16 bits (half a step, and 2^-25 / 2^13 of the row's factor below
fp16's range); dH and dW are sums of V or R of those, rounded once more."""

import pytest
import torch

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -23


def make(rows, vocab, hidden, dtype, seed=0, spread=1.5, lift=True, ignored=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(vocab, hidden, device="cuda", generator=g) * (spread / hidden ** 0.5)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    h = torch.randn(rows, hidden, device="cuda", generator=g)
    if lift:
        a = 20 * torch.rand(rows, 1, device="cuda", generator=g)
        h = h + a * w[t] / (w[t] * w[t]).sum(1, keepdim=True).clamp(min=1e-3)
    if ignored:
        t = torch.where(torch.rand(rows, device="cuda", generator=g) < ignored, -100, t)
    return h.to(dtype), w.to(dtype), t


def exact(h, w, t, b=None, c=None, whole=False):
    """losses, lse, and from b = dL/d loss and c = dL/d lse the gradients, each with a bound on what the arithmetic may add (`whole`: dW without what the target's dl loses in 16 bits)."""
    valid = (t >= 0) & (t < w.shape[0])
    h64, w64 = torch.where(valid[:, None], h.double(), 0.0), w.double()
    hidden, half = h.shape[1], torch.finfo(h.dtype).eps / 2
    logits = h64 @ w64.t()
    mags = h64.abs() @ w64.abs().t()
    eta = hidden * UNIT * mags.max(1).values + (64 + 4 * logits.abs().max(1).values) * UNIT
    lse = torch.logsumexp(logits, 1)
    at = t.clamp(0, w.shape[0] - 1)
    z = lambda x: torch.where(valid, x, 0.0)
    out = {"lse": (z(lse), z(eta)), "losses": (z(lse - logits.gather(1, at[:, None])[:, 0]), z(2 * eta))}
    if b is None:
        return out
    b, c = z(b.double()), z(c.double())
    p = torch.softmax(logits, 1)
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    dl = (b + c)[:, None] * p - b[:, None] * hot
    size = (b + c).abs()[:, None] * p + (b.abs()[:, None] * (1 - p) + c.abs()[:, None] * p) * hot
    tiny = 2.0 ** -25 / 8192 if h.dtype == torch.float16 else 0.0
    off = size * (half + 3 * eta[:, None] + 8 * UNIT) + tiny * 2 * torch.maximum(b.abs(), c.abs())[:, None]
    dh, dw = dl @ w64, dl.t() @ h64
    sub = torch.finfo(h.dtype).smallest_normal * torch.finfo(h.dtype).eps / 2
    dh_off = off @ w64.abs() + w.shape[0] * UNIT * (size @ w64.abs())
    # (rows whose factor is far below the largest are scaled down before the sum over rows)
    top = torch.maximum(b.abs(), c.abs()).max() if len(t) else 0.0
    low = 2.0 ** -25 * 4 * top if h.dtype == torch.float16 else 0.0
    if whole:
        off = off - hot * size * half
    dw_off = off.t() @ h64.abs() + (len(t) + 1) * UNIT * (size.t() @ h64.abs()) + low * (size.t() / top.clamp(min=1e-30)).sum(1, keepdim=True)
    out["d_hidden"] = (dh, dh_off + half * (dh.abs() + dh_off) + sub)
    out["d_weight"] = (dw, dw_off + half * (dw.abs() + dw_off) + sub)
    return out


def check(got, want):
    for name, (value, bound) in want.items():
        off = (got[name].double() - value).abs()
        assert (off <= bound * 1.001 + 1e-30).all(), (name, float((off / (bound + 1e-30)).max()))


def run(h, w, t, b, c):
    from hackaton_b200 import vocab_cross_entropy

    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    losses, lse = vocab_cross_entropy(h, w, t)
    dh, dw = torch.autograd.grad([losses, lse], [h, w], [b, c])
    assert dh.dtype == h.dtype and dw.dtype == w.dtype
    return {"losses": losses.detach(), "lse": lse.detach(), "d_hidden": dh, "d_weight": dw}


def factors(rows, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b = torch.randn(rows, device="cuda", generator=g) * torch.exp2(torch.randint(-6, 3, (rows,), device="cuda", generator=g).float())
    return b, torch.randn(rows, device="cuda", generator=g) * 0.3


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,hidden", [(1, 300, 64), (3, 1, 8), (5, 2, 72), (61, 1003, 128), (256, 256, 64), (257, 257, 200),
                                               (300, 511, 1536), (700, 5000, 320), (17, 40007, 64)])
def test_matches_the_formulas(cuda_lib, dtype, rows, vocab, hidden):
    h, w, t = make(rows, vocab, hidden, dtype, rows + vocab)
    b, c = factors(rows)
    got = run(h, w, t, b, c)
    check(got, exact(h, w, t, b, c))
    again = run(h, w, t, b, c)
    assert all(torch.equal(got[k], again[k]) for k in got)
    cuda_lib.device_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_several_pieces_of_the_vocabulary(cuda_lib, dtype):
    """1000 rows: pieces of 32,768 words; the second one ends in the middle of a tile."""
    h, w, t = make(1000, 33007, 136, dtype, 3, ignored=0.3)
    t[5], t[6] = 33006, 32767
    b, c = factors(1000)
    check(run(h, w, t, b, c), exact(h, w, t, b, c))


def test_many_rows(cuda_lib):
    """More tiles of rows than a piece of the vocabulary has room for two tiles of words."""
    h, w, t = make(263_000, 600, 64, torch.bfloat16, 21, ignored=0.1)
    b, c = factors(263_000)
    check(run(h, w, t, b, c), exact(h, w, t, b, c))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_logits_that_outgrow_what_the_first_words_showed(cuda_lib, dtype):
    """Words far behind the first 2048 beat them, and the target, by up to 2^60, in both pieces, for some rows of some
    tiles: their references move, sums so far go along. (bf16 has room for most of it; 2^120 more for one row.)"""
    h, w, t = make(1000, 33007, 136, dtype, 21, spread=0.5, lift=False)
    t = t % 2048
    h[:, 0] = 0
    w[:, 0] = 0
    step = 2.0
    h[3, 0], h[200, 0], h[201, 0], h[700, 0], h[999, 0] = 1 * step, 4 * step, 8 * step, 20 * step, 45 * step
    w[5000, 0], w[20000, 0], w[30000, 0], w[33006, 0] = 0.5, 0.75, 1.0, 1.25
    b, c = factors(1000)
    got = run(h, w, t, b, c)
    check(got, exact(h, w, t, b, c))
    assert float(got["losses"][999]) > 60


@pytest.mark.parametrize("ignored", [0.0, 0.5, 0.97, 1.0])
@pytest.mark.parametrize("rows", [70, 600])
def test_ignored_rows(cuda_lib, rows, ignored):
    """They give zeros, and what they hold (NaN and infinities here) reaches nothing."""
    h, w, t = make(rows, 700, 96, torch.bfloat16, 4, ignored=ignored)
    if ignored == 1.0:
        t[:] = -1
    skip = t < 0
    clean = h.clone()
    h[skip] = float("nan")
    if rows > 10:
        h[:10][skip[:10]] = float("inf")
    b, c = factors(rows)
    b[skip] = float("nan")
    got = run(h, w, t, b, c)
    clean[skip] = 0
    check(got, exact(clean, w, t, torch.where(skip, 0.0, b), c))
    assert not got["losses"][skip].any() and not got["lse"][skip].any() and not got["d_hidden"][skip].any()


def test_target_beyond_the_vocabulary(cuda_lib):
    h, w, t = make(40, 500, 64, torch.float16, 5)
    t[7] = 500
    b, c = factors(40)
    got = run(h, w, t, b, c)
    with pytest.raises(Exception, match="200"):
        cuda_lib.device_status()
    check(got, exact(h, w, t, b, c))
    assert float(got["losses"][7]) == 0.0 and not got["d_hidden"][7].any()
    cuda_lib.device_status()


def test_only_what_is_asked_for(cuda_lib):
    from hackaton_b200 import vocab_cross_entropy

    h, w, t = make(130, 900, 128, torch.float16, 6, ignored=0.1)
    b, c = factors(130)
    every = run(h, w, t, b, c)
    want = exact(h, w, t, b, c)
    with torch.no_grad():
        losses, lse = vocab_cross_entropy(h, w, t)
    # (without the hidden states' gradient the sums are relative to maxima, not to references: other roundings in fp32,
    # each within the bound)
    check({"losses": losses, "lse": lse}, {k: want[k] for k in ("losses", "lse")})
    h1 = h.clone().requires_grad_()
    out = vocab_cross_entropy(h1, w, t)
    assert torch.equal(torch.autograd.grad(out, [h1], [b, c])[0], every["d_hidden"])
    w1 = w.clone().requires_grad_()
    out = vocab_cross_entropy(h, w1, t)
    check({"d_weight": torch.autograd.grad(out, [w1], [b, c])[0]}, {"d_weight": want["d_weight"]})
    # one output alone, a mean, and a number broadcast to all rows
    losses, lse = vocab_cross_entropy(h1, w, t)
    (d,) = torch.autograd.grad(losses.sum() / 64, [h1], retain_graph=True)
    want = exact(h, w, t, torch.full((130,), 1 / 64, device="cuda"), torch.zeros(130, device="cuda"))
    assert ((d.double() - want["d_hidden"][0]).abs() <= want["d_hidden"][1] * 1.001).all()
    (d,) = torch.autograd.grad((lse * lse).sum(), [h1])
    want = exact(h, w, t, torch.zeros(130, device="cuda"), 2 * lse.detach())
    assert ((d.double() - want["d_hidden"][0]).abs() <= want["d_hidden"][1] * 1.001).all()


def test_gradient_against_differences(cuda_lib):
    """(L(h + e v) - L(h - e v)) / 2e for steps that bf16 holds exactly: off by the rounding of L (eta) over e and by
    the third derivative, at most |v . w|^3 e^2."""
    from hackaton_b200 import vocab_cross_entropy

    h, w, t = make(6, 300, 64, torch.bfloat16, 8, lift=False)
    h = (h * 8).round() / 8               # multiples of 1/8 below 8: bf16 holds them and their neighbours at 1/32
    h = h.clamp(-3, 3)
    v = torch.randint(-1, 2, h.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(h.dtype)
    e = 1 / 32
    b = torch.ones(6, device="cuda")
    got = run(h, w, t, b, 0 * b)
    up, down = (vocab_cross_entropy((h.float() + s * e * v.float()).to(h.dtype), w, t)[0].double() for s in (1, -1))
    assert torch.equal((h.float() + e * v.float()).to(h.dtype).float(), h.float() + e * v.float())
    by_gradient = (got["d_hidden"].double() * v.double()).sum(1)
    want = exact(h, w, t, b, 0 * b)
    turn = (v.double() @ w.double().t()).abs().max(1).values
    bound = 2 * want["losses"][1] / e + (2 * turn) ** 3 * e * e + (want["d_hidden"][1] * v.double().abs()).sum(1)
    assert ((up - down) / (2 * e) - by_gradient).abs().le(bound).all()


def test_confident_rows_keep_their_digits(cuda_lib):
    """A target 15 above all others: the loss is 1e-5 and less, right to a relative bound, and so is its gradient."""
    g = torch.Generator(device="cuda").manual_seed(9)
    w = torch.zeros(512, 64, device="cuda")
    w[:, :8] = torch.randn(512, 8, device="cuda", generator=g) * 0.1
    w[:64, 8:] = 0
    h = torch.randn(32, 64, device="cuda", generator=g) * 0.5
    t = torch.arange(32, device="cuda")
    w[t, 16 + t] = 4.0
    h[:, 16:48] = 0
    h[t, 16 + t] = 6.0
    h, w = h.bfloat16(), w.bfloat16()
    b = torch.ones(32, device="cuda")
    got = run(h, w, t, b, 0 * b)
    want = exact(h, w, t, b, 0 * b)
    loss = want["losses"][0]
    assert (loss < 1e-6).all()
    assert ((got["losses"].double() - loss).abs() <= loss * 2 * want["losses"][1]).all()
    size = want["d_hidden"][0].abs().max(1).values
    assert ((got["d_hidden"].double() - want["d_hidden"][0]).abs().max(1).values <= size * 2.0 ** -7).all()


def test_large_logits(cuda_lib):
    """Logits of thousands: nothing overflows, the running maximum carries over pieces and tiles."""
    h, w, t = make(64, 2000, 64, torch.bfloat16, 10, lift=False)
    h = h * 400
    b, c = factors(64)
    got = run(h, w, t, b, c)
    want = exact(h, w, t, b, c)
    for name in ("losses", "lse"):
        assert ((got[name].double() - want[name][0]).abs() <= want[name][1] * 1.001).all()
    assert all(v.isfinite().all() for v in got.values())


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("vocab", [900, 5000])
def test_logits_of_millions(cuda_lib, vocab, sign):
    """References far from zero on either side, over a vocabulary that is asked for them as a whole and one that is not."""
    g = torch.Generator(device="cuda").manual_seed(23)
    h = sign * (100 + torch.rand(70, 512, device="cuda", generator=g)).half()
    w = (100 + 0.01 * torch.randint(0, 3, (vocab, 512), device="cuda", generator=g)).half()
    t = torch.randint(0, vocab, (70,), device="cuda", generator=g)
    b, c = factors(70)
    got = run(h, w, t, b, c)
    want = exact(h, w, t, b, c)
    for name in ("losses", "lse"):
        assert ((got[name].double() - want[name][0]).abs() <= want[name][1] * 1.001).all()
    assert all(v.isfinite().all() for v in got.values())


def test_nan_and_infinity_show(cuda_lib):
    h, w, t = make(300, 600, 64, torch.float16, 11)
    b, c = factors(300)
    clean = run(h, w, t, b, c)
    h[4, 3] = float("nan")
    h[280, 5] = float("inf")
    got = run(h, w, t, b, c)
    keep = [i for i in range(300) if i not in (4, 280)]
    for name in ("losses", "lse", "d_hidden"):
        assert torch.equal(got[name][keep], clean[name][keep]) and got[name][4].isnan().all()
        assert not got[name][280].isfinite().all()
    assert got["d_weight"].isnan().any()
    b[9] = float("inf")                       # what a loss scaler looks for
    h, w, t = make(300, 600, 64, torch.float16, 11)
    assert not run(h, w, t, b, c)["d_hidden"][9].isfinite().all()


def test_layouts(cuda_lib):
    """Leading dimensions, strides, odd addresses, a view of the weight; no rows at all."""
    from hackaton_b200 import vocab_cross_entropy

    h, w, t = make(60, 800, 72, torch.float16, 12, ignored=0.2)
    want = vocab_cross_entropy(h, w, t)
    got = vocab_cross_entropy(h.view(3, 20, 72), w, t.view(3, 20))
    assert all(torch.equal(a, b.view(60)) and b.shape == (3, 20) for a, b in zip(want, got))
    odd = torch.zeros(60 * 72 + 1, device="cuda", dtype=h.dtype)[1:].view(60, 72)
    odd.copy_(h)
    wide = torch.zeros(800, 75, device="cuda", dtype=h.dtype)
    wide[:, 1:73] = w
    pitch = torch.zeros(800, 96, device="cuda", dtype=h.dtype)
    pitch[:, 8:80] = w
    for hh, ww, tt in ((odd, w, t), (h.t().contiguous().t(), w, t), (h, wide[:, 1:73], t), (h, pitch[:, 8:80], t),
                       (h, w.t().contiguous().t(), t), (h, w, torch.stack([t, t], 1)[:, 0])):
        assert all(torch.equal(a, b) for a, b in zip(want, vocab_cross_entropy(hh, ww, tt)))
    one = vocab_cross_entropy(h[0], w, t[0].clamp(min=0))
    assert one[0].shape == ()
    b = torch.ones(60, device="cuda")
    wv = pitch[:, 8:80].detach().requires_grad_()
    (dw,) = torch.autograd.grad(vocab_cross_entropy(h, wv, t), [wv], [b, b])
    check({"d_weight": dw}, {"d_weight": exact(h, w, t, b, b)["d_weight"]})
    leaf = h[:0].detach().requires_grad_()
    wl = w.detach().requires_grad_()
    losses, _ = vocab_cross_entropy(leaf, wl, t[:0])
    gh, gw = torch.autograd.grad(losses.sum(), [leaf, wl])
    assert gh.shape == (0, 72) and not gw.any()


def test_streams_and_graphs(cuda_lib):
    """On another stream, two calls at once, and a captured training step replayed with other rows ignored."""
    from hackaton_b200 import vocab_cross_entropy

    h, w, t = make(300, 3000, 128, torch.float16, 13, ignored=0.3)
    h2, _, t2 = make(300, 3000, 128, torch.float16, 14, ignored=0.6)
    b, c = factors(300)
    want, want2 = run(h, w, t, b, c), run(h2, w, t2, b, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(h, w, t, b, c)
    got2 = run(h2, w, t2, b, c)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want[k], got[k]) and torch.equal(want2[k], got2[k]) for k in want)
    hs, ts = h.clone().requires_grad_(), t.clone()
    ws = w.clone().requires_grad_()

    def step():
        losses, lse = vocab_cross_entropy(hs, ws, ts)
        return (losses.detach(), *torch.autograd.grad([losses, lse], [hs, ws], [b, c]))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for hh, tt, ref in ((h2, t2, want2), (h, t, want)):
        with torch.no_grad():
            hs.copy_(hh)
            ts.copy_(tt)
        graph.replay()
        assert all(torch.equal(o, ref[k]) for o, k in zip(out, ("losses", "d_hidden", "d_weight")))
    cuda_lib.device_status()


def test_agrees_with_the_chunked_loss(cuda_lib):
    """The same loss and gradient as linear_cross_entropy, which rounds its logits to fp16 (half a step of up to 16: 2^-8)."""
    from hackaton_b200 import linear_cross_entropy, vocab_cross_entropy

    h, w, t = make(600, 5000, 256, torch.float16, 15, spread=1.0, lift=False, ignored=0.2)
    denom = (t >= 0).sum().float()
    h1, h2 = h.clone().requires_grad_(), h.clone().requires_grad_()
    loss, *_ = linear_cross_entropy(h1, w, t, denom)
    mine = vocab_cross_entropy(h2, w, t)[0].sum() / denom
    assert abs(float(loss) - float(mine)) <= 2.0 ** -8
    (loss * 1024).backward()
    (mine * 1024).backward()
    assert (h1.grad.float() - h2.grad.float()).norm() <= 2.0 ** -7 * h2.grad.float().norm()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,hidden", [(1, 1, 8), (1, 40007, 64), (16, 300, 128), (17, 5000, 72), (32, 257, 64), (33, 1003, 320),
                                               (64, 20000, 1536), (65, 1003, 128), (300, 5000, 64)])
def test_without_gradients(cuda_lib, dtype, rows, vocab, hidden):
    """Losses and logsumexps alone: up to 64 rows they come out of a product with the words on the long side."""
    from hackaton_b200 import vocab_cross_entropy

    h, w, t = make(rows, vocab, hidden, dtype, rows * 3 + vocab, ignored=0.2 if rows > 4 else 0.0)
    if rows > 20:
        t[3], t[9] = 0, vocab - 1
    with torch.no_grad():
        losses, lse = vocab_cross_entropy(h, w, t)
        check({"losses": losses, "lse": lse}, exact(h, w, t))
        again = vocab_cross_entropy(h, w, t)
    assert torch.equal(losses, again[0]) and torch.equal(lse, again[1])
    cuda_lib.device_status()


def test_without_gradients_and_nan(cuda_lib):
    from hackaton_b200 import vocab_cross_entropy

    h, w, t = make(40, 3000, 64, torch.float16, 31)
    clean = vocab_cross_entropy(h, w, t)
    h[5, 1] = float("nan")
    got = vocab_cross_entropy(h, w, t)
    keep = [i for i in range(40) if i != 5]
    assert all(torch.equal(g[keep], c[keep]) and g[5].isnan() for g, c in zip(got, clean))
    h[5, 1] = 0
    h[:, 0], w[:, 0] = 30000.0, 0.0
    w[2999, 0] = 1.0                      # one word far above the rest, in the last tile
    t[:] = torch.arange(40, device="cuda")
    with torch.no_grad():
        losses, lse = vocab_cross_entropy(h, w, t)
        check({"losses": losses, "lse": lse}, exact(h, w, t))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 300), (40, 900), (150, 300)])
def test_targets_rows_of_the_heads_gradient(cuda_lib, dtype, rows, vocab):
    """Up to four rows to a word: what their dl lose in 16 bits is not lost. Rows that want little (p of the target near zero)
    leave the target's as the largest by far, so that it would show."""
    h, w, _ = make(rows, vocab, 128, dtype, 22, spread=1.0, lift=False)
    t = (torch.arange(rows, device="cuda") % 60) * 5 + (torch.arange(rows, device="cuda") // 60)
    b, c = factors(rows)
    check(run(h, w, t, b, 0 * c), exact(h, w, t, b, 0 * c, whole=True))


@pytest.mark.parametrize("rows,grad", [(5, False), (70, False), (70, True)])
def test_long_rows_keep_their_digits(cuda_lib, rows, grad):
    """16,384 features of one sign: a sum of 1024 steps of 16 products only grows, and each step may cut off a unit of what it has
    reached, twice over (its products, the addition): in one chain 1024 units of the final value. In chains of 128 steps that is 2 * 65,
    and one for each of eight chains."""
    from hackaton_b200 import vocab_cross_entropy

    g = torch.Generator(device="cuda").manual_seed(3)
    h = (0.05 * torch.rand(rows, 16384, device="cuda", generator=g)).to(torch.bfloat16)
    w = (0.2 * torch.rand(700, 16384, device="cuda", generator=g)).to(torch.bfloat16)
    t = torch.randint(0, 700, (rows,), device="cuda", generator=g)
    logits = h.double() @ w.double().t()
    want = torch.logsumexp(logits, 1)
    top = logits.max(1).values
    lse = vocab_cross_entropy(h.requires_grad_(grad), w, t)[1].detach()
    assert ((lse.double() - want).abs() <= (138 * top + 64 + 4 * top) * UNIT).all()
