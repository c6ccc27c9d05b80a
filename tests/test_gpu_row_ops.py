"""Row operators on the MI355X against their definitions in 64 bits (row_ops_util.py, on the CPU): every type, widths on
both sides of each kernel variant's limits, odd widths and strides, empty inputs, values that poison a row."""
import ctypes

import numpy as np
import pytest
import torch

import row_ops_util as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# one column, inside one unit, on both sides of the lanes' and the variants' widths, wide rows; one row to a few thousand
SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 65), (70, 128), (4, 129), (64, 1024), (37, 333), (1, 512), (9, 513), (4, 2048),
         (3, 2049), (2, 4100), (2, 8192), (3, 8200), (2, 12001), (2, 16384), (2, 16385), (2, 20001), (1, 100003), (300000, 1), (70000, 3), (1030, 48), (2500, 96), (1500, 1000), (1100, 2056),
         # rows on both sides of the one-launch backward (1024), for each of the other's variants
         (1024, 40), (1025, 40), (1100, 5), (1025, 200), (1100, 400), (1030, 2048), (1025, 2500), (1027, 4100), (300, 9001)]


@pytest.fixture(scope="module")
def B():
    import bilinear_amd
    return bilinear_amd


def data(rows, width, dtype, seed, pad=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(rows, width + pad, generator=g) * (scale * (0.5 + torch.rand(width + pad, generator=g))) + shift
         + 0.3 * torch.randn(width + pad, generator=g)).to(dtype)
    return t.cuda()[:, pad // 2:pad // 2 + width]


def params(width, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return ((1 + 0.3 * torch.randn(width, generator=g)).to(dtype).cuda().requires_grad_(),
            (0.3 * torch.randn(width, generator=g)).to(dtype).cuda().requires_grad_())


def d(t):
    return None if t is None else t.detach().double().cpu()


def check_layer_norm(B, x, w, b, dy, eps=1e-5):
    x = x.detach().requires_grad_()
    y = B.layer_norm(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    wants = [t for t in (x, w, b) if t is not None]
    got = torch.autograd.grad(y, wants, dy)
    X, Wt, Bi, D = d(x).requires_grad_(), d(w), d(b), d(dy)
    for t in (Wt, Bi):
        if t is not None:
            t.requires_grad_()
    Y = R.norm64(X, Wt, Bi, eps)[0]
    want = torch.autograd.grad(Y, [t for t in (X, Wt, Bi) if t is not None], D)
    with torch.no_grad():
        e_y, e_hat, e_rstd = R.forward_bounds(X, Wt, Bi, eps, x.dtype)
        e_dx, e_dw, e_db = R.backward_bounds(X, Wt, D, eps, e_hat, e_rstd)
        R.close(y, Y, e_y, "y")
        R.close(got[0], want[0], R.rounded(e_dx, want[0], x.dtype), "dx")
        for g, v, e, t, what in zip(got[1:], want[1:], [e for e, t in ((e_dw, w), (e_db, b)) if t is not None],
                                    [t for t in (w, b) if t is not None], ("first parameter", "second parameter")):
            assert g.dtype == t.dtype
            R.close(g, v, R.rounded(e, v, t.dtype), what)
    with torch.no_grad():
        assert torch.equal(B.layer_norm(x, w, b, eps), y)          # without the saved moments: the same bits


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("dtype,ptype", [(F32, F32), (BF16, F32), (F16, F16)])
def test_layer_norm(B, rows, width, dtype, ptype):
    w, b = params(width, ptype, 5)
    check_layer_norm(B, data(rows, width, dtype, 1), w, b, data(rows, width, dtype, 2))


@pytest.mark.parametrize("dtype,ptype", [(BF16, BF16), (F16, F32)])
def test_layer_norm_other_parameter_types(B, dtype, ptype):
    w, b = params(515, ptype, 5)
    check_layer_norm(B, data(33, 515, dtype, 1), w, b, data(33, 515, dtype, 2))


@pytest.mark.parametrize("width", [40, 700, 5000])
def test_layer_norm_without_weight_or_bias(B, width):
    w, b = params(width, F32, 5)
    x, dy = data(21, width, BF16, 1), data(21, width, BF16, 2)
    check_layer_norm(B, x, None, None, dy)
    check_layer_norm(B, x, w, None, dy)
    check_layer_norm(B, x, None, b, dy)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_rows_far_from_zero_and_large_eps(B, dtype):
    """A mean of 50 standard deviations (the bound grows with it), and eps that outweighs the variance."""
    w, b = params(600, F32, 5)
    check_layer_norm(B, data(12, 600, dtype, 1, shift=50.0), w, b, data(12, 600, dtype, 2))
    check_layer_norm(B, data(12, 600, dtype, 1, scale=1e-3), w, b, data(12, 600, dtype, 2), eps=0.5)


def test_constant_rows_are_exactly_the_bias(B):
    for width in (8, 64, 1024, 4096, 16384):      # powers of two: the mean of equal values is that value exactly
        w, b = params(width, F32, 5)
        x = torch.full((3, width), 1234.5, device="cuda")
        assert torch.equal(B.layer_norm(x, w, b), b.expand(3, width))


@pytest.mark.parametrize("rows,width", [(3, 200), (700, 200), (3, 3000), (3, 9000)])
def test_a_poisoned_row_poisons_only_its_own_results(B, rows, width):
    w, b = params(width, F32, 5)
    x, dy = data(rows, width, F32, 1), data(rows, width, F32, 2)
    clean = B.layer_norm(x, w, b)
    bad = x.clone()
    bad[1, width // 2] = float("nan")
    bad[2, 3] = float("inf")
    bad.requires_grad_()
    y = B.layer_norm(bad, w, b)
    assert torch.isnan(y[1:3]).all() and torch.equal(y[:1], clean[:1]) and torch.equal(y[3:], clean[3:])
    dx, dw = torch.autograd.grad(y, (bad, w), dy)
    assert torch.isnan(dx[1:3]).all() and not torch.isnan(dx[:1]).any() and not torch.isnan(dx[3:]).any()
    assert torch.isnan(dw).all()


@pytest.mark.parametrize("pad", [1, 2, 8, 23])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_of_a_wider_tensor(B, dtype, pad):
    w, b = params(777, F32, 5)
    check_layer_norm(B, data(19, 777, dtype, 1, pad=pad), w, b, data(19, 777, dtype, 2, pad=pad + 1))


def test_other_layouts(B):
    """Leading axes, transposed inputs, repeated rows, an expanded gradient, one axis, no rows."""
    w, b = params(24, F32, 5)
    x = data(30, 24, F32, 1)
    y = B.layer_norm(x, w, b)
    assert torch.equal(B.layer_norm(x.view(2, 3, 5, 24), w, b), y.view(2, 3, 5, 24))
    assert torch.equal(B.layer_norm(x.t().contiguous().t(), w, b), y)
    assert torch.equal(B.layer_norm(x.view(5, 6, 24).transpose(0, 1), w, b), y.view(5, 6, 24).transpose(0, 1))
    assert torch.equal(B.layer_norm(x[4].expand(7, 24), w, b), y[4].expand(7, 24))
    assert torch.equal(B.layer_norm(x[4], w, b), y[4])
    x = x.requires_grad_()
    ones = torch.ones(30, 24, device="cuda")
    for dy in (torch.ones((), device="cuda").expand(30, 24), torch.ones(24, device="cuda").expand(30, 24)):
        for p, q in zip(torch.autograd.grad(B.layer_norm(x, w, b), (x, w, b), dy),
                        torch.autograd.grad(B.layer_norm(x, w, b), (x, w, b), ones)):
            assert torch.equal(p, q)
    e = torch.empty(0, 24, device="cuda", requires_grad=True)
    out = B.layer_norm(e, w, b)
    de, dw, db = torch.autograd.grad(out, (e, w, b), torch.empty(0, 24, device="cuda"))
    assert out.shape == de.shape == (0, 24) and not dw.any() and not db.any()


def test_only_the_gradients_that_are_wanted(B):
    x, dy = data(200, 500, BF16, 1), data(200, 500, BF16, 2)
    w, b = params(500, F32, 5)
    full = torch.autograd.grad(B.layer_norm(x.requires_grad_(), w, b), (x, w, b), dy)
    assert torch.equal(torch.autograd.grad(B.layer_norm(x, w.detach(), b.detach()), x, dy)[0], full[0])
    assert torch.equal(torch.autograd.grad(B.layer_norm(x.detach(), w, b.detach()), w, dy)[0], full[1])
    assert torch.equal(torch.autograd.grad(B.layer_norm(x.detach(), w.detach(), b), b, dy)[0], full[2])


def test_parameters_that_are_not_dense(B):
    w, b = params(2 * 300, F32, 5)
    x, dy = data(7, 300, F32, 1).requires_grad_(), data(7, 300, F32, 2)
    for p, q in ((w[::2], b[1::2]), (w.view(300, 2)[:, 1], b[:1].expand(300))):
        got = torch.autograd.grad(B.layer_norm(x, p, q), (x, w, b), dy)
        want = torch.autograd.grad(B.layer_norm(x, p.contiguous(), q.contiguous()), (x, w, b), dy)
        for u, v in zip(got, want):
            assert torch.equal(u, v)


def test_graphs_kept_freed_and_written_to(B):
    x, r, dy = data(20, 64, F32, 1).requires_grad_(), data(20, 64, F32, 2).requires_grad_(), data(20, 64, F32, 3)
    y, h = B.residual_norm(x, r, p=0.3, seed=1)
    once = torch.autograd.grad((y, h), (x, r), (dy, dy), retain_graph=True)
    for p, q in zip(once, torch.autograd.grad((y, h), (x, r), (dy, dy))):
        assert torch.equal(p, q)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad((y, h), (x, r), (dy, dy))
    y, h = B.residual_norm(x, r, p=0.3, seed=1)
    h.add_(1)                                 # what the backward reads: refused by its version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)
    z = B.layer_norm(x)
    z.mul_(2)                                 # nothing reads y: this stays a plain factor
    assert torch.equal(torch.autograd.grad(z, x, dy)[0], torch.autograd.grad(B.layer_norm(x), x, 2 * dy)[0])


def test_a_checkpointed_block_is_recomputed_with_its_mask(B):
    from torch.utils.checkpoint import checkpoint
    x, dy = data(40, 64, F32, 1).requires_grad_(), data(40, 64, F32, 2)
    norm, drop = B.ResidualNorm(64, p=0.4).cuda(), B.Dropout(0.4)
    block = lambda t: drop(norm(t, t)[0])     # noqa: E731
    torch.manual_seed(8)
    want = torch.autograd.grad(block(x), (x, norm.weight), dy)
    for reentrant in (False, True):
        torch.manual_seed(8)
        out = checkpoint(block, x, use_reentrant=reentrant)
        x.grad = norm.weight.grad = None
        out.backward(dy)
        assert torch.equal(x.grad, want[0]) and torch.equal(norm.weight.grad, want[1])


def test_a_second_thread_and_single_threaded_backward(B):
    import threading
    x, dy = data(500, 300, BF16, 1), data(500, 300, BF16, 2)
    w, b = params(300, F32, 5)

    def work():
        t = x.detach().requires_grad_()
        return torch.autograd.grad(B.layer_norm(t, w, b), (t, w, b), dy)

    want, got = work(), [None] * 4
    torch.cuda.synchronize()

    def run(i):
        got[i] = work()
        torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    with torch.autograd.set_multithreading_enabled(False):
        got.append(work())
    for g in got:
        for p, q in zip(g, want):
            assert torch.equal(p, q)


def test_lazily_negated_views_and_forward_mode(B):
    z = torch.view_as_complex(data(6, 80, F32, 1).view(6, 40, 2))
    x = z.conj().imag                        # a float view that is to be read negated
    assert x.is_neg()
    w, b = params(40, F32, 5)
    assert torch.equal(B.layer_norm(x, w, b), B.layer_norm(x.resolve_neg(), w, b))
    assert torch.equal(B.dropout(x, 0.5, seed=1), B.dropout(x.resolve_neg(), 0.5, seed=1))
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        dual = fwd.make_dual(data(3, 8, F32, 1), data(3, 8, F32, 2))
        with pytest.raises(NotImplementedError):
            B.layer_norm(dual)


def test_custom_operators_are_what_their_schemas_say(B):
    x, r = data(6, 40, BF16, 1).requires_grad_(), data(6, 40, F32, 2).requires_grad_()
    w, b = params(40, F32, 5)
    op = torch.ops.bilinear_hip
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(op.layer_norm.default, (x, w, b, 1e-5), test_utils=checks)
    torch.library.opcheck(op.row_dropout.default, (x, 0.3, 1, 2, 3, 4, None), test_utils=checks)
    torch.library.opcheck(op.residual_norm.default, (x, r, w, b, 1e-5, 0.3, 1, 2, 3, 4, None), test_utils=checks)


def test_double_backward_is_refused(B):
    x = data(3, 16, F32, 1).requires_grad_()
    g, = torch.autograd.grad(B.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_gradient_against_differences(B):
    """Central differences of the fp32 forward along one direction v, f = sum(y c): (f(x + s v) - f(x - s v)) / 2 s.  The
    truncation is about s^2 of the third derivative and the rounding W-fold sums of U |y c| / s: with s = 2^-7, values of
    order one and 60 columns both stay under 5e-3 of the sum of |terms|."""
    x, v, c = (data(4, 60, F32, k) for k in (1, 2, 3))
    w, b = params(60, F32, 5)
    s = 2.0 ** -7
    x = x.requires_grad_()
    grad, = torch.autograd.grad(B.layer_norm(x, w, b), x, c)
    with torch.no_grad():
        f = lambda t: (B.layer_norm(t, w, b).double() * c.double()).sum()   # noqa: E731
        slope = (f(x + s * v) - f(x - s * v)) / (2 * s)
    along = (grad.double() * v.double())
    assert abs(slope - along.sum()) <= 5e-3 * along.abs().sum()


# ---- dropout --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (64, 1024), (37, 333), (2, 4100), (1030, 48), (5, 20001), (2500, 96)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.999])
def test_dropout(B, rows, width, dtype, p):
    """fp32 multiplies once, narrower types multiply in fp32 and round once: equal to the definition bit for bit."""
    kw = dict(seed=(1 << 62) + 12345678901, step=(3 << 32) + 9, layer=1007, row_offset=(1 << 32) - 16)
    x, dy = data(rows, width, dtype, 1).requires_grad_(), data(rows, width, dtype, 2)
    f = R.factor(rows, width, p, **kw)
    y = B.dropout(x, p, **kw)
    dx, = torch.autograd.grad(y, x, dy)
    for got, src in ((y, x), (dx, dy)):
        want = torch.where(f > 0, (d(src) * f).float(), torch.zeros(())).to(dtype)
        assert torch.equal(got.detach().cpu(), want)


def test_dropout_rates_and_independence(B):
    """Kept share within 6 standard deviations; masks of another seed, step, layer and row differ."""
    n, p = 1 << 22, 0.3
    one = torch.ones(1 << 10, 1 << 12, device="cuda")
    keep = B.dropout(one, p, seed=11) != 0
    assert abs(keep.double().mean().item() - 0.7) < 6 * (0.21 / n) ** 0.5
    for kw in (dict(seed=12), dict(seed=11, step=1), dict(seed=11, layer=1), dict(seed=11, row_offset=1024), dict(seed=11, step=1 << 32)):
        other = B.dropout(one, p, **kw) != 0
        both = (keep & other).double().mean().item()
        assert abs(both - 0.49) < 6 * (0.49 * 0.51 / n) ** 0.5


def test_dropout_edges(B):
    x = data(5, 33, F32, 1)
    x[2, 2], x[3, 4] = float("nan"), float("inf")
    y = B.dropout(x, 0.0, seed=1)
    assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(x))
    assert not B.dropout(x, 1.0, seed=1).any()
    assert B.dropout(torch.empty(0, 7, device="cuda"), 0.5, seed=1).shape == (0, 7)


def test_mask_does_not_depend_on_how_rows_are_spread(B):
    x = data(96, 50, F32, 1)
    whole = B.dropout(x, 0.4, seed=3, step=2)
    parts = [B.dropout(x[i:i + 32], 0.4, seed=3, step=2, row_offset=i) for i in (0, 32, 64)]
    assert torch.equal(torch.cat(parts), whole)
    wide = data(96, 60, F32, 1)[:, 5:55]
    assert torch.equal(B.dropout(wide, 0.4, seed=3, step=2) != 0, whole != 0)


def test_modules_of_two_ranks_draw_the_parts_of_one_mask(B):
    x = data(96, 50, F32, 1)
    drop, norm = B.Dropout(0.4), B.ResidualNorm(50, p=0.4).cuda()

    def call(rows, offset):
        torch.manual_seed(5)                       # what every rank does
        drop.row_offset = norm.row_offset = offset
        return drop(x[rows]), norm(x[rows], x[rows])[1]
    whole, lower, upper = call(slice(None), 0), call(slice(0, 40), 0), call(slice(40, 96), 40)
    for w, a, b in zip(whole, lower, upper):
        assert torch.equal(torch.cat((a, b)), w)


# ---- residual norm --------------------------------------------------------------------------------------------------

def check_residual_norm(B, x, r, w, b, dy, dh, p, eps=1e-5):
    kw = dict(seed=77, step=5, layer=1001, row_offset=64)
    rows, width = x.shape
    x, r = x.detach().requires_grad_(), r.detach().requires_grad_()
    y, h = B.residual_norm(x, r, w, b, eps, p, **kw)
    assert y.dtype == x.dtype and h.dtype == r.dtype
    X, Rs, Wt, Bi = d(x), d(r), d(w), d(b)
    f = R.factor(rows, width, p, **kw) if R.threshold(p) else torch.ones(rows, width, dtype=torch.double)
    # the stream: one rounding to fp32 (a fused multiply-add), one to its type
    want_h = (Rs + X * f).float().to(r.dtype)
    R.close(h, Rs + X * f, R.U * (Rs + X * f).abs() + R.half_step(r.dtype) * (Rs + X * f).abs() * (1 + R.U) + R.tiny(r.dtype), "h")
    assert (h.detach().cpu() != want_h).double().mean() < 1e-4     # (64 -> 32 -> type rounds twice, once in a long while)
    H = d(h).requires_grad_()                                       # what the norm is taken of
    Wt.requires_grad_(), Bi.requires_grad_()
    Y = R.norm64(H, Wt, Bi, eps)[0]
    outs, grads = ([y, h], [dy, dh]) if dh is not None else ([y], [dy])
    got = torch.autograd.grad(outs, (x, r, w, b), grads)
    want = list(torch.autograd.grad(Y, (H, Wt, Bi), d(dy)))
    total = want[0] + (d(dh) if dh is not None else 0)
    with torch.no_grad():
        e_y, e_hat, e_rstd = R.forward_bounds(H, Wt, Bi, eps, x.dtype)
        e_dh, e_dw, e_db = R.backward_bounds(H, Wt, d(dy), eps, e_hat, e_rstd)
        e_dh = e_dh + R.U * total.abs()
        R.close(y, Y, e_y, "y")
        R.close(got[0], total * f, R.rounded(f * (e_dh + R.U * total.abs()), total * f, x.dtype), "dx")
        R.close(got[1], total, R.rounded(e_dh, total, r.dtype), "dresidual")
        R.close(got[2], want[1], R.rounded(e_dw, want[1], w.dtype), "dweight")
        R.close(got[3], want[2], R.rounded(e_db, want[2], b.dtype), "dbias")


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("dtype,rtype,p", [(F32, F32, 0.5), (BF16, F32, 0.1), (F16, F16, 0.25)])
def test_residual_norm(B, rows, width, dtype, rtype, p):
    w, b = params(width, F32, 5)
    check_residual_norm(B, data(rows, width, dtype, 1), data(rows, width, rtype, 2), w, b, data(rows, width, dtype, 3),
                        data(rows, width, rtype, 4), p)


@pytest.mark.parametrize("dtype,rtype,ptype", [(BF16, BF16, BF16), (F16, F32, F16), (BF16, F32, BF16)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_residual_norm_types_strides_and_no_stream_gradient(B, dtype, rtype, ptype, p):
    w, b = params(333, ptype, 5)
    check_residual_norm(B, data(40, 333, dtype, 1, pad=3), data(40, 333, rtype, 2, pad=9), w, b,
                        data(40, 333, dtype, 3, pad=1), data(40, 333, rtype, 4, pad=5), p)
    check_residual_norm(B, data(40, 333, dtype, 1), data(40, 333, rtype, 2), w, b, data(40, 333, dtype, 3), None, p)


def test_residual_norm_is_its_parts(B):
    """The fused pass against dropout, the sum and layer_norm called one after the other."""
    x, r = data(50, 700, BF16, 1), data(50, 700, F32, 2)
    w, b = params(700, F32, 5)
    kw = dict(seed=9, step=1, layer=4)
    with torch.no_grad():
        y, h = B.residual_norm(x, r, w, b, p=0.2, **kw)
        f = R.factor(50, 700, 0.2, **kw)
        assert torch.equal(h.cpu(), (d(r) + d(x) * f).float())
        assert torch.equal(B.dropout(x, 0.2, **kw).cpu() != 0, (d(x) * f) != 0)
        # y in bf16 from the same h: layer_norm of the fp32 stream, rounded to bf16
        assert torch.equal(y, B.layer_norm(h, w, b).to(BF16))


def test_residual_norm_gradients_of_one_output(B):
    x, r = data(20, 100, F32, 1).requires_grad_(), data(20, 100, F32, 2).requires_grad_()
    w, b = params(100, F32, 5)
    dh = data(20, 100, F32, 3)
    kw = dict(p=0.3, seed=1)
    _, h = B.residual_norm(x, r, w, b, **kw)
    dx, dr, dw = torch.autograd.grad(h, (x, r, w), dh)
    assert torch.equal(dr, dh) and torch.equal(dx, B.dropout(dh, 0.3, seed=1)) and not dw.any()
    y, h = B.residual_norm(x.detach(), r, w, b, **kw)          # the branch needs no gradient
    dr2, = torch.autograd.grad((y, h), r, (dh, dh))
    y, h = B.residual_norm(x, r.detach(), w, b, **kw)          # the stream needs none
    dx2, = torch.autograd.grad((y, h), x, (dh, dh))
    y, h = B.residual_norm(x, r, w, b, **kw)
    both = torch.autograd.grad((y, h), (x, r), (dh, dh))
    assert torch.equal(both[0], dx2) and torch.equal(both[1], dr2)


def test_what_is_dropped_does_not_reach_the_stream(B):
    x, r = data(6, 40, F32, 1), data(6, 40, F32, 2)
    f = R.factor(6, 40, 0.5, seed=4)
    x[f.cuda() == 0] = float("nan")
    y, h = B.residual_norm(x, r, p=0.5, seed=4)
    assert torch.isfinite(y).all() and torch.equal(h[f.cuda() == 0], r[f.cuda() == 0])


# ---- the calls around the operators -----------------------------------------------------------------------------------

def test_results_do_not_change_from_run_to_run(B):
    x, dy = data(3000, 1000, BF16, 1).requires_grad_(), data(3000, 1000, BF16, 2)
    w, b = params(1000, F32, 5)
    first = torch.autograd.grad(B.layer_norm(x, w, b), (x, w, b), dy)
    for _ in range(3):
        for p, q in zip(first, torch.autograd.grad(B.layer_norm(x, w, b), (x, w, b), dy)):
            assert torch.equal(p, q)


def test_nothing_is_written_behind_the_last_row(B, native):
    """The C entry points on buffers with a guarded tail (and work in place where the header allows it)."""
    from bilinear_amd import _native as N
    rows, width = 5, 37
    st = N.current_stream()
    x, dy = data(rows, width, BF16, 1).contiguous(), data(rows, width, BF16, 2).contiguous()
    guard = lambda n, t=BF16: torch.full((n + 64,), 7.0, dtype=t, device="cuda")   # noqa: E731
    y, h, dx, dr = (guard(rows * width) for _ in range(4))
    mean, rstd, dw, db = guard(rows, F32), guard(rows, F32), guard(width, F32), guard(width, F32)
    drop = N.RowDrop(0.5, 1, 2, 3, None, None, 4, 0)
    assert native.blh_residual_norm_forward(st, x.data_ptr(), width, dy.data_ptr(), width, None, None, 1e-5,
                                            ctypes.byref(drop), y.data_ptr(), h.data_ptr(), mean.data_ptr(),
                                            rstd.data_ptr(), rows, width, 1, 1, 0) == 0
    need = native.blh_row_norm_workspace_bytes(rows, width)
    ws = torch.full((need + 256,), 7, dtype=torch.uint8, device="cuda")
    assert native.blh_residual_norm_backward(st, dy.data_ptr(), width, x.data_ptr(), width, h.data_ptr(), width, None,
                                             mean.data_ptr(), rstd.data_ptr(), ctypes.byref(drop), dx.data_ptr(),
                                             dr.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need, rows, width,
                                             1, 1, 0) == 0
    for t, n in ((y, rows * width), (h, rows * width), (dx, rows * width), (dr, rows * width), (mean, rows), (rstd, rows),
                 (dw, width), (db, width)):
        assert (t[n:] == 7).all() and not (t[:n] == 7).all()
    assert (ws[need:] == 7).all()
    z = x.clone()
    assert native.blh_row_dropout(st, z.data_ptr(), width, z.data_ptr(), ctypes.byref(drop), rows, width, 1) == 0
    assert torch.equal(z, B.dropout(x, 0.5, seed=1, step=2, layer=4, row_offset=3))


def test_another_stream(B):
    x, dy = data(2000, 512, F32, 1).requires_grad_(), data(2000, 512, F32, 2)
    w, b = params(512, F32, 5)
    want = torch.autograd.grad(B.layer_norm(x, w, b), (x, w, b), dy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = torch.autograd.grad(B.layer_norm(x, w, b), (x, w, b), dy)
    side.synchronize()
    for p, q in zip(got, want):
        assert torch.equal(p, q)


def test_captured_step_replays_with_fresh_masks(B):
    """Forward and backward of the three operators in one graph; every replay against the eager call of that step, with the
    program's own work between the replays."""
    x, r = data(300, 200, BF16, 1).requires_grad_(), data(300, 200, F32, 2).requires_grad_()
    dy, dh = data(300, 200, BF16, 3), data(300, 200, F32, 4)
    w, b = params(200, F32, 5)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def work(**kw):
        y, h = B.residual_norm(x, r, w, b, 1e-5, 0.2, seed=5, layer=1, **kw)
        z = B.layer_norm(B.dropout(y, 0.3, seed=5, layer=2, **kw), w, b)
        return torch.autograd.grad((z, h), (x, r, w, b), (dy, dh)) + (z.detach(), h.detach())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(device_step=step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(device_step=step)
        step.add_(1)             # (after the backward was recorded: it reads the step its forward used)
    for n in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = work(step=n)
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(p, q), n
    assert step.item() == 4


def test_backward_reads_the_step_its_forward_used(B):
    x = data(30, 40, F32, 1).requires_grad_()
    step = torch.full((1,), 6, dtype=torch.int64, device="cuda")
    y = B.dropout(x, 0.5, seed=1, device_step=step)
    step.add_(10)
    dx, = torch.autograd.grad(y, x, torch.ones_like(x))
    assert torch.equal(dx != 0, B.dropout(torch.ones_like(x), 0.5, seed=1, step=6) != 0)


def test_capture_with_a_live_eager_graph_is_refused(B):
    """The refusal comes before anything is enqueued: the capture ends empty and the process goes on."""
    x = data(8, 16, F32, 1)
    w, b = params(16, F32, 5)
    eager = B.layer_norm(x, w, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="still part of an eager autograd graph"):
            B.layer_norm(x, w, b)
        with pytest.raises(RuntimeError, match="still part of an eager autograd graph"):
            torch.ops.bilinear_hip.layer_norm(x, w, b, 1e-5)
        with torch.no_grad():
            z = B.layer_norm(x, w, b)      # nothing to differentiate: nothing to refuse
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, eager)


def test_a_captured_backward_beside_a_live_graph_of_a_side_stream(B):
    """The usual warm-up: eager steps on a side stream whose outputs are still held when the capture begins."""
    x, dy = data(64, 128, F32, 1).requires_grad_(), data(64, 128, F32, 2)
    w, b = params(128, F32, 5)
    torch.autograd.graph.set_warn_on_accumulate_grad_stream_mismatch(False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = B.layer_norm(x, w, b)
        held.backward(dy)
    torch.cuda.current_stream().wait_stream(side)
    want = [t.grad.clone() for t in (x, w, b)]
    x.grad = w.grad = b.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        B.layer_norm(x, w, b).backward(dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for t, v in zip((x, w, b), want):
            assert torch.equal(t.grad, v)
            t.grad.zero_()
    assert torch.isfinite(held).all()
    torch.autograd.graph.set_warn_on_accumulate_grad_stream_mismatch(True)


def test_under_torch_compile(B):
    """The custom operators' autograd formulas: the compiled function equals the eager one (no code generator involved)."""
    x, r = data(40, 96, BF16, 1).requires_grad_(), data(40, 96, F32, 2).requires_grad_()
    w, b = params(96, F32, 5)
    dy, dh = data(40, 96, BF16, 3), data(40, 96, F32, 4)

    def f(x, r, w, b):
        y, h = B.residual_norm(x, r, w, b, 1e-5, 0.2, seed=5, step=7, layer=1)
        return B.layer_norm(B.dropout(y, 0.3, seed=5, step=7, layer=2), w, b), h

    want = f(x, r, w, b)
    want += torch.autograd.grad(want, (x, r, w, b), (dy, dh))
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(x, r, w, b)
    got += torch.autograd.grad(got, (x, r, w, b), (dy, dh))
    for p, q in zip(got, want):
        assert torch.equal(p, q)


def test_compiled_functions_of_one_output_and_compiled_modules(B):
    x, r = data(40, 96, F32, 1).requires_grad_(), data(40, 96, F32, 2).requires_grad_()
    dh = data(40, 96, F32, 4)
    f = lambda x, r: B.residual_norm(x, r, p=0.2, seed=5)[1]     # noqa: E731
    want = torch.autograd.grad(f(x, r), (x, r), dh)
    for p, q in zip(torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(x, r), (x, r), dh), want):
        assert torch.equal(p, q)
    net = torch.nn.Sequential(B.LayerNorm(96), B.Dropout(0.3)).cuda()
    step = torch.compile(net, backend="aot_eager")
    outs = []
    for compiled in (False, True):
        torch.manual_seed(21)
        outs.append([(step if compiled else net)(x) for _ in range(4)])
    for p, q in zip(*outs):
        assert torch.equal(p, q)
    assert not torch.equal(outs[0][0], outs[0][1])


def test_offsets_past_32_bits(B):
    """More than 2^32 elements: the last rows are those of the same rows on their own (bit for bit: rows do not meet)."""
    rows, width = (1 << 19) + 3, 8192
    w, b = params(width, F32, 5)
    block = data(1024, width, BF16, 1)
    x = torch.empty(rows, width, dtype=BF16, device="cuda")
    for i in range(0, rows, 1024):
        x[i:i + 1024] = block[:min(1024, rows - i)]
    x.requires_grad_()
    tail = x.detach()[-5:].clone().requires_grad_()
    y, small = B.layer_norm(x, w, b), B.layer_norm(tail, w, b)
    assert torch.equal(y[-5:], small)
    dx, = torch.autograd.grad(y, x, x.detach())
    assert torch.equal(dx[-5:], torch.autograd.grad(small, tail, tail.detach())[0])
    del y, dx
    y = B.dropout(x.detach(), 0.3, seed=3)
    assert torch.equal(y[-5:], B.dropout(tail.detach(), 0.3, seed=3, row_offset=rows - 5))
    del y
    y, h = B.residual_norm(x.detach(), x.detach(), p=0.3, seed=3)
    u, v = B.residual_norm(tail.detach(), tail.detach(), p=0.3, seed=3, row_offset=rows - 5)
    assert torch.equal(y[-5:], u) and torch.equal(h[-5:], v)


def test_the_custom_operators_refuse_what_the_functions_refuse(B):
    x = torch.zeros(2, 8, device="cuda")
    op = torch.ops.bilinear_hip
    with pytest.raises(RuntimeError):
        op.layer_norm(x, torch.zeros(9, device="cuda"), None, 1e-5)
    with pytest.raises(RuntimeError):
        op.layer_norm(x, torch.zeros(8), None, 1e-5)
    with pytest.raises(RuntimeError):
        op.layer_norm_backward(x, x, None, torch.zeros(1, device="cuda"), torch.zeros(2, device="cuda"), True, False, False, 0)
    with pytest.raises(RuntimeError):
        op.layer_norm_backward(x[:1], x, None, torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda"), True, False, False, 0)
    with pytest.raises(RuntimeError):
        B.residual_norm(x, x.cpu())
    with pytest.raises(RuntimeError):
        B.residual_norm(x, x.half())
    with pytest.raises(RuntimeError):
        B.layer_norm(x.double())
    with pytest.raises(ValueError):
        B.dropout(x, 1.5, seed=0)


def test_a_residual_network_of_the_operators_trains(B):
    """As they are used together: an encoder, residual blocks (norm, linear, dropout on the way back into the stream), a final
    norm and a decoder, one backward pass, against the same network in 64 bits on the masks its modules drew."""
    torch.manual_seed(4)
    width, rows, blocks, p = 96, 50, 3, 0.25

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.encode = torch.nn.Linear(32, width)
            self.drop = B.Dropout(p)
            self.first = B.LayerNorm(width)
            self.linears = torch.nn.ModuleList(torch.nn.Linear(width, width) for _ in range(blocks))
            self.norms = torch.nn.ModuleList(B.ResidualNorm(width, p=p) for _ in range(blocks))
            self.decode = torch.nn.Linear(width, 48)

        def forward(self, x):
            h = self.drop(self.encode(x))
            y = self.first(h)
            for lin, norm in zip(self.linears, self.norms):
                y, h = norm(torch.relu(lin(y)), h)
            return self.decode(y)

    net = Net().cuda()
    x, t = data(rows, 32, F32, 1), data(rows, 48, F32, 2)
    state = torch.get_rng_state()
    torch.nn.functional.mse_loss(net(x), t).backward()
    torch.set_rng_state(state)                # the numbers the modules drew, in the order of their calls
    masks = []
    for m in [net.drop, *net.norms]:
        kw = m._next_draws()
        assert kw.pop("device_step") is None
        masks.append(R.factor(rows, width, p, **kw))

    P = {k: v.detach().double().cpu().requires_grad_() for k, v in net.named_parameters()}
    h = (d(x) @ P["encode.weight"].t() + P["encode.bias"]) * masks[0]
    y = R.norm64(h, P["first.weight"], P["first.bias"], 1e-5)[0]
    for i in range(blocks):
        z = torch.relu(y @ P["linears.%d.weight" % i].t() + P["linears.%d.bias" % i])
        h = h + z * masks[i + 1]
        y = R.norm64(h, P["norms.%d.weight" % i], P["norms.%d.bias" % i], 1e-5)[0]
    ((y @ P["decode.weight"].t() + P["decode.bias"] - d(t)) ** 2).mean().backward()
    for k, v in net.named_parameters():
        # fp32 products of 96 terms through a dozen layers: 1e-4 of the tensor's norm is 800 half-steps of fp32
        assert (v.grad.double().cpu() - P[k].grad).norm() <= 1e-4 * P[k].grad.norm(), k
    first = net(x)
    assert not torch.equal(first, net(x))                 # another mask each call ...
    net.eval()
    assert torch.equal(net(x), net(x))                    # ... and none in eval mode
