"""GPU: calls of the C ABI that are refused before anything is launched."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("off", [1, 2, 3])
def test_sandwich_norm_refuses_an_rstd_at_an_odd_address(cuda_lib, off):
    """Rows of it are read and written as 16 bytes; everything else may lie at any address of its type."""
    lib = cuda_lib.lib()
    rows, hidden = 3, 64
    r, w = torch.ones(rows, hidden, device="cuda"), torch.ones(hidden, device="cuda")
    d, y, s = r.half(), torch.zeros(rows, hidden, device="cuda", dtype=torch.float16), torch.zeros(rows, hidden, device="cuda")
    room = torch.full((4 * rows + 4,), 7.0, device="cuda")
    rstd = room[off:]
    rc = lib.nf4b200_sandwich_norm_fwd(r.data_ptr(), d.data_ptr(), 0, w.data_ptr(), w.data_ptr(), None, 0, s.data_ptr(), y.data_ptr(), 0,
                                       rstd.data_ptr(), rows, hidden, 1.0, 1e-6, None)
    assert rc == -1 and b"rstd" in lib.nf4b200_last_error()
    need = lib.nf4b200_sandwich_norm_workspace_bytes(rows, hidden, 0)
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    rc = lib.nf4b200_sandwich_norm_bwd(s.data_ptr(), d.data_ptr(), 0, w.data_ptr(), w.data_ptr(), None, 0, rstd.data_ptr(), None, y.data_ptr(),
                                       0, r.data_ptr(), None, None, None, None, rows, hidden, 1.0, ws.data_ptr(), need, None)
    assert rc == -1 and b"rstd" in lib.nf4b200_last_error()
    torch.cuda.synchronize()
    assert (room == 7).all() and not s.any() and not y.any()
