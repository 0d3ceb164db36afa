"""GPU: the hidden states' gradient of rows that are nearly certain of their target, where everything but the target is
far below it, and of the rows beside them.

Bound. The exponentials of the words other than the target are rounded to 16 bits: half a step of each, or half of
the smallest number of the type, which in fp16 is 2^-25 where the largest of them lies at least 2^3 above a row's
reference: 2^-28 of the largest. The rest is fp32 arithmetic as in test_vocab_loss_gpu.py (eta: a logit's error), and the output's own
rounding."""

import pytest
import torch

from test_vocab_loss_gpu import UNIT, check, exact, run

pytestmark = pytest.mark.gpu


def confident(gaps, vocab, dtype, late=False):
    """Row r: noise for logits, but its target's, `gaps[r]` above them by a coordinate of its own. All other words share a direction
    (coordinate 1), which the target's word has with the other sign, so that both parts of the gradient show in it. `late`: a word
    behind the first 2048 lies half way up for every row."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows, hidden = len(gaps), max(64, -(-(len(gaps) + 2) // 8) * 8)
    gap = torch.tensor([float(x) for x in gaps], device="cuda")
    own = 2 + torch.arange(rows, device="cuda")
    t = torch.arange(rows, device="cuda") * 7 % min(vocab, 2000)
    w = 0.05 * torch.randn(vocab, hidden, device="cuda", generator=g)
    w[:, 0] = 0
    w[:, 1] = 0.5
    w[t] = 0
    w[t, 1] = -0.5
    w[t, own] = 1.0
    h = 0.25 * torch.randn(rows, hidden, device="cuda", generator=g)
    h[:, 1] = 0
    h[torch.arange(rows, device="cuda"), own] = gap
    if late:
        w[vocab - 3, 2:] = 0.5
    return h.to(dtype), w.to(dtype), t


def bound_of(h, w, t, b):
    want = exact(h, w, t, b, 0 * b)
    h64, w64 = h.double(), w.double()
    half = torch.finfo(h.dtype).eps / 2
    logits = h64 @ w64.t()
    eta = h.shape[1] * UNIT * (h64.abs() @ w64.abs().t()).max(1).values + (64 + 4 * logits.abs().max(1).values) * UNIT
    p = torch.softmax(logits, 1)
    hot = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    others = p * (1 - hot)
    low = 2.0 ** -28 if h.dtype == torch.float16 else 0.0
    off = others * (half + 3 * eta[:, None] + 8 * UNIT) + low * others.max(1, keepdim=True).values * (1 - hot)
    size = others + hot * others.sum(1, keepdim=True)
    off = off + hot * others.sum(1, keepdim=True) * (3 * eta[:, None] + 64 * UNIT)
    off = b.double().abs()[:, None] * off @ w64.abs() + w.shape[0] * UNIT * (b.double().abs()[:, None] * size @ w64.abs())
    dh = b.double()[:, None] * (others @ w64 - others.sum(1, keepdim=True) * w64[t])
    assert (dh - want["d_hidden"][0]).abs().max() <= 1e-9 * b.abs().max()     # (that form cancels in 64 bits too)
    sub = torch.finfo(h.dtype).smallest_normal * torch.finfo(h.dtype).eps / 2
    return dh, off + half * (dh.abs() + off) + sub


GAPS = [1, 6, 9, 12, 15, 17, 18, 19, 20, 21, 23, 24, 25, 26, 28, 30, 35, 45, 60]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab,late", [(1500, False), (2048, False), (5000, False), (5000, True)])
def test_gradients_of_confident_rows(cuda_lib, dtype, vocab, late):
    """1500 and 2048 words are asked for the references as a whole, 5000 are not."""
    h, w, t = confident(GAPS * 3, vocab, dtype, late)
    b = torch.full((len(t),), 65536.0 if dtype == torch.float16 else 1.0, device="cuda")
    got = run(h, w, t, b, 0 * b)
    dh, bound = bound_of(h, w, t, b)
    far = (got["d_hidden"].double() - dh).abs() / (bound * 1.001)
    assert (far <= 1).all(), {GAPS[r % len(GAPS)]: float(far[r].max()) for r in range(len(GAPS))}
    check({k: got[k] for k in ("losses", "lse")}, {k: v for k, v in exact(h, w, t).items()})
    again = run(h, w, t, b, 0 * b)
    assert all(torch.equal(got[k], again[k]) for k in got)
    cuda_lib.device_status()


def test_rows_beside_a_confident_one_stay_as_they_are(cuda_lib):
    """Whether a row's tile is done again for another row's sake does not show in it."""
    h, w, t = confident([5, 8] * 300, 5000, torch.float16)
    b = torch.ones(600, device="cuda")
    plain = run(h, w, t, b, 0 * b)
    h[300] *= 6                    # from 5 to 30 above the others
    got = run(h, w, t, b, 0 * b)
    rest = [r for r in range(600) if r != 300]
    for name in ("losses", "lse", "d_hidden"):
        assert torch.equal(got[name][rest], plain[name][rest])
    assert not torch.equal(got["d_hidden"][300], plain["d_hidden"][300])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_nan_and_infinity_beside_confident_rows(cuda_lib, dtype):
    """Rows without a finite logit, or with infinite ones, over a vocabulary that is not asked for the references as a whole."""
    h, w, t = confident([5, 30] * 150, 5000, dtype)
    b = torch.ones(300, device="cuda")
    clean = run(h, w, t, b, 0 * b)
    h[4, 3], h[280, 1], h[281, 1] = float("nan"), float("inf"), -float("inf")
    got = run(h, w, t, b, 0 * b)
    rest = [r for r in range(300) if r not in (4, 280, 281)]
    for name in ("losses", "lse", "d_hidden"):
        assert torch.equal(got[name][rest], clean[name][rest])
        assert got[name][4].isnan().all()
    assert not got["losses"][280].isfinite() and not got["d_hidden"][280].isfinite().all()
    cuda_lib.device_status()


@pytest.mark.parametrize("gap", [14, 17, 18, 18.8, 20, 24, 30])
def test_many_words_far_below_one(cuda_lib, gap):
    """Beside a certain target one word, and 40,000 that are e^-12 of it each, a third of it together, in a direction of their own: they
    reach the gradient. (In norm: roundings that are 2^-12 of each term, and 40,000 times 2^-28 of the largest.)"""
    h, w, t = confident([gap] * 8, 40007, torch.float16)
    w[:, 2:] = 0
    w[t] = 0
    w[t, 1] = -0.5
    w[t, 2 + torch.arange(8, device="cuda")] = 1.0
    w[1900] = 0
    w[1900, 20] = 1.0
    h[:, 1], h[:, 20] = 0.055, 12.0      # (16.45 of fp16's smallest numbers where the one word is at 2^-2.7)
    h[torch.arange(8, device="cuda"), 2 + torch.arange(8, device="cuda")] = gap + 12.0
    b = torch.full((8,), 65536.0, device="cuda")
    got = run(h, w, t, b, 0 * b)["d_hidden"]
    dh, _ = bound_of(h, w, t, b)
    sub = 2.0 ** -25 * h.shape[1] ** 0.5
    assert ((got.double() - dh).norm(dim=1) <= dh.norm(dim=1) * (2.0 ** -11 + 2.0 ** -12.7) + sub).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gaps", [[2], [18], [22], [26], [30], [34], [18, 30], [2, 30], [60]])
@pytest.mark.parametrize("rows", [1, 20])
def test_head_gradients_of_confident_rows(cuda_lib, dtype, gaps, rows):
    """Where every row is nearly certain, what there is keeps its digits: a row's dl are rounded to half a step each, or in fp16 to 2^-25 / 2^13
    of twice the largest 1 - p of a target (times its factor); for the target's word what that loses is added in fp32."""
    h, w, t = confident((gaps * rows)[:max(rows, len(gaps))], 1500, dtype)
    b = torch.full((len(t),), 2.0 ** 20, device="cuda")
    got = run(h, w, t, b, 0 * b)["d_weight"]
    h64, w64 = h.double(), w.double()
    half = torch.finfo(dtype).eps / 2
    logits = h64 @ w64.t()
    eta = h.shape[1] * UNIT * (h64.abs() @ w64.abs().t()).max(1).values + (64 + 4 * logits.abs().max(1).values) * UNIT
    p = torch.softmax(logits, 1)
    hot = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    others = p * (1 - hot)
    rest = others.sum(1, keepdim=True)
    dl = b[:, None].double() * (others - hot * rest)
    floor = 2.0 ** -25 / 8192 * 2 * (b.double() * rest[:, 0]).max() if dtype == torch.float16 else 0.0
    off = dl.abs() * (half * (1 - hot) + 3 * eta[:, None] + 64 * UNIT) + floor * (1 - hot)
    dw = dl.t() @ h64
    bound = off.t() @ h64.abs() + (len(t) + 1) * UNIT * (dl.abs().t() @ h64.abs())
    sub = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    bound = bound + half * (dw.abs() + bound) + sub
    beyond = (dw.abs() + bound >= torch.finfo(dtype).max) & (got.double() == dw.sign() * float("inf"))      # (2^20 times a gap of 2)
    far = torch.where(beyond, 0.0, (got.double() - dw).abs() / bound)
    assert (far <= 1.001).all(), float(far.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tiles_done_again_repeat_themselves(cuda_lib, dtype):
    """Rows of several tiles meet a word behind the first 2048 that is far above those: whichever order the tiles are done again in."""
    h, w, t = confident([40, 3, 250, 9] * 300, 5000, dtype, late=True)
    b = torch.ones(1200, device="cuda")
    first = run(h, w, t, b, 0 * b)
    dh, bound = bound_of(h, w, t, b)
    assert ((first["d_hidden"].double() - dh).abs() <= bound * 1.001).all()
    for _ in range(8):
        again = run(h, w, t, b, 0 * b)
        assert all(torch.equal(first[k], again[k]) for k in first)
