"""Row operators on the MI355X under the calls around them, and on values at the ends of the types' ranges."""
import pytest
import torch

import row_ops_util as R
from test_gpu_row_ops import BF16, F32, d, data, params

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def B():
    import bilinear_amd
    return bilinear_amd


# ---- values at the ends of the range ----------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,width", [(2, 12), (3, 64), (1025, 64), (1026, 12), (1027, 5), (1027, 200), (2, 20004)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_mean_times_rstd_past_the_largest_number(B, rows, width, dtype):
    """A last row of equal values v = 2^119 (2^112 in the longest rows).  Its sum stays below the largest number (200 v < 2^127,
    20004 v < 2^127) and is exact, so h - mean is 0 and rstd = eps^-1/2; mean rstd = 2^119 2^10 (2^112 2^20) passes 2^128, but
    no result holds that product: with t = dy w, dx = rstd (t - mean t), dw = 0, db = sum dy.  The other rows are ordinary."""
    eps = 2.0 ** -20 if width < 10000 else 2.0 ** -40
    x = data(rows, width, dtype, 1)
    x[-1] = 2.0 ** (119 if width < 10000 else 112)
    w, b = params(width, F32, 5)
    dy = data(rows, width, dtype, 2)
    x.requires_grad_()
    y = B.layer_norm(x, w, b, eps)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    for t in (y, dx, dw, db):
        assert torch.isfinite(t).all()
    D, Wt, Bi = d(dy), d(w), d(b)
    t, n = D[-1] * Wt, R.chain(width)
    rstd = eps ** -0.5
    want = rstd * (t - t.mean())
    e = rstd * ((n + 4) * R.U * t.abs().mean() + 6 * R.U * (t.abs() + t.mean().abs()))
    R.close(dx[-1], want, R.rounded(e, want, dtype), "dx")
    R.close(y[-1], Bi, R.rounded(torch.zeros_like(Bi), Bi, dtype), "y")
    X = d(x[:-1])
    _, e_hat, e_rstd = R.forward_bounds(X, Wt, Bi, eps, dtype)
    _, e_dw, e_db = R.backward_bounds(X, Wt, D[:-1], eps, e_hat, e_rstd)
    want = (D[:-1] * R.norm64(X, Wt, Bi, eps)[3]).sum(0)
    R.close(dw, want, R.rounded(e_dw, want, F32), "dw")
    R.close(db, D.sum(0), R.rounded(e_db + 400 * R.U * D[-1].abs(), D.sum(0), F32), "db")
