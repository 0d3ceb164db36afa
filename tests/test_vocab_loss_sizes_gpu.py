"""GPU: the vocabulary loss where its sizes are large."""

import pytest
import torch

from test_vocab_loss_gpu import check, exact, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [4097, 32768, 32769, 33792, 66559, 1050001])
@pytest.mark.parametrize("ignored", [0.0, 0.4, 0.9999])
def test_rows_that_take_part_among_many(cuda_lib, rows, ignored):
    from hackaton_b200 import vocab_cross_entropy

    h, w, t = make(rows, 9, 8, torch.float16, rows, ignored=ignored)
    h[t < 0] = float("nan")
    check(dict(zip(("losses", "lse"), vocab_cross_entropy(h, w, t))), exact(h, w, t))
    if rows > 100_000:
        return
    b = torch.ones(rows, device="cuda")
    h.requires_grad_()
    losses, lse = vocab_cross_entropy(h, w, t)
    (d,) = torch.autograd.grad(losses.sum(), [h])
    want = exact(h.detach(), w, t, b, 0 * b)
    check({"losses": losses.detach(), "d_hidden": d}, {k: want[k] for k in ("losses", "d_hidden")})


def test_time_grows_with_the_rows(cuda_lib):
    """Four times the rows take about four times as long; twice that is allowed here."""
    from hackaton_b200 import vocab_cross_entropy

    def time(rows):
        h, w, t = make(rows, 8, 8, torch.float16)
        best = float("inf")
        for _ in range(6):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            vocab_cross_entropy(h, w, t)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        return best

    time(1 << 19)
    assert time(1 << 21) <= 8 * time(1 << 19)
