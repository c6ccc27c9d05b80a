"""Row operators on the MI355X under the calls around them, and on values at the ends of the types' ranges."""
import pytest
import torch

import row_ops_util as R
from test_gpu_row_ops import BF16, F16, F32, d, data, params

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def B():
    import bilinear_amd
    return bilinear_amd


# ---- second derivatives ---------------------------------------------------------------------------------------------

def _first_outputs(B):
    op = torch.ops.bilinear_hip
    return {
        "layer_norm": lambda x, r, w, b: B.layer_norm(x, w, b),
        "residual_norm": lambda x, r, w, b: B.residual_norm(x, r, w, b, p=0.3, seed=1)[0],
        "residual_norm without dropout": lambda x, r, w, b: B.residual_norm(x, r, w, b)[0],
        "operator layer_norm": lambda x, r, w, b: op.layer_norm(x, w, b, 1e-5)[0],
        "operator residual_norm": lambda x, r, w, b: op.residual_norm(x, r, w, b, 1e-5, 0.3, 1, 0, 0, 0, None)[0],
    }


@pytest.mark.parametrize("name", ["layer_norm", "residual_norm", "residual_norm without dropout", "operator layer_norm",
                                  "operator residual_norm"])
def test_a_second_derivative_is_refused_beside_other_terms(B, name):
    """A gradient penalty in a loss that has other gradients: its share must not be dropped in silence."""
    x, r = data(3, 16, F32, 1).requires_grad_(), data(3, 16, F32, 2).requires_grad_()
    w, b = params(16, F32, 5)
    y = _first_outputs(B)[name](x, r, w, b)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="differentiate the backward pass"):
        (y.sum() + g.square().sum()).backward()


@pytest.mark.parametrize("name", ["layer_norm", "residual_norm", "residual_norm without dropout", "operator layer_norm",
                                  "operator residual_norm"])
def test_a_second_derivative_is_refused_towards_chosen_inputs(B, name):
    """torch.autograd.grad runs what leads to the inputs it is given, and functional.hessian takes what does not for zero."""
    def tensors():
        x, r = data(3, 16, F32, 1).requires_grad_(), data(3, 16, F32, 2).requires_grad_()
        return (x, r, *params(16, F32, 5))
    f = _first_outputs(B)[name]
    for of in (0, 2):                                       # of dx, of dweight
        for towards in (0, 2):
            args = tensors()
            y = f(*args)
            g, = torch.autograd.grad(y.square().sum(), args[of], create_graph=True)
            with pytest.raises(RuntimeError, match="differentiate the backward pass"):
                torch.autograd.grad(y.sum() + g.square().sum(), args[towards], allow_unused=True)
    x, r, w, b = tensors()
    with pytest.raises(RuntimeError, match="differentiate the backward pass"):
        torch.autograd.functional.hessian(lambda t: f(t, r, w, b).pow(3).sum(), x.detach())


def test_a_graph_of_gradients_that_depend_on_nothing_more_is_plain(B):
    x = data(3, 16, F32, 1)
    w, b = params(16, F32, 5)
    db, = torch.autograd.grad(B.layer_norm(x, w.detach(), b).sum(), b, create_graph=True)
    assert not db.requires_grad


def test_the_backward_operators_refuse_to_be_differentiated(B):
    op = torch.ops.bilinear_hip
    x, dy = data(3, 16, F32, 1), data(3, 16, F32, 2).requires_grad_()
    w = params(16, F32, 5)[0]
    with torch.no_grad():
        _, mean, rstd = op.layer_norm(x, w, None, 1e-5)
    dx = op.layer_norm_backward(dy, x, w, mean, rstd, True, True, True, 0)[0]
    with pytest.raises(RuntimeError, match="differentiate the backward pass"):
        (dx.sum() + dy.sum()).backward()
    dx = op.residual_norm_backward(dy, None, x, w, mean, rstd, 0.3, 1, 0, 0, 0, None, True, True, True, True, 0)[0]
    with pytest.raises(RuntimeError, match="differentiate the backward pass"):
        (dx.sum() + dy.sum()).backward()


def test_the_backward_operators_refuse_tangents(B):
    import torch.autograd.forward_ad as fwd
    x, w = data(3, 16, F32, 1), params(16, F32, 5)[0].detach()
    _, mean, rstd = torch.ops.bilinear_hip.layer_norm(x, w, None, 1e-5)
    with fwd.dual_level():
        dual = fwd.make_dual(data(3, 16, F32, 2), data(3, 16, F32, 3))
        with pytest.raises(NotImplementedError):
            torch.ops.bilinear_hip.layer_norm_backward(dual, x, w, mean, rstd, True, True, True, 0)


@pytest.mark.parametrize("operator", [False, True])
@pytest.mark.parametrize("device_step", [False, True])
def test_second_derivative_of_dropout(B, operator, device_step):
    """f: the factor of an element.  y = f x, g = d(sum y^3)/dx = 3 f^3 x^2, d(sum g^2 + sum y)/dx = 36 f^6 x^3 + f: some
    fifteen fp32 products, of half a step each."""
    x = data(20, 40, F32, 1).requires_grad_()
    step = torch.full((1,), 4, dtype=torch.int64, device="cuda") if device_step else None
    args = (0.3, 7, 1 if device_step else 5, 2, 3, step)
    y = torch.ops.bilinear_hip.row_dropout(x, *args)[0] if operator else B.dropout(x, *args)
    if device_step:
        step.add_(1)                     # the backward passes read the step that the forward used
    g, = torch.autograd.grad(y.pow(3).sum(), x, create_graph=True)
    got, = torch.autograd.grad(g.square().sum() + y.sum(), x)
    f = R.factor(20, 40, 0.3, seed=7, step=5, layer=2, row_offset=3)
    want = 36 * f ** 6 * d(x) ** 3 + f
    R.close(got, want, 24 * R.U * (36 * f ** 6 * d(x).abs() ** 3 + f) + R.tiny(F32), "second derivative")


@pytest.mark.parametrize("operator", [False, True])
def test_second_derivative_of_the_stream(B, operator):
    """h = r + f x, g = d(sum h^3)/dx = 3 f h^2, d(sum g^2)/dx = 36 f^3 h^3.  h is off by U |h|, the rest by some fifteen roundings
    more."""
    x, r = data(9, 40, F32, 1).requires_grad_(), data(9, 40, F32, 2).requires_grad_()
    w, b = params(40, F32, 5)
    h = (torch.ops.bilinear_hip.residual_norm(x, r, w, b, 1e-5, 0.3, 7, 0, 0, 0, None) if operator
         else B.residual_norm(x, r, w, b, p=0.3, seed=7))[1]
    g, = torch.autograd.grad(h.pow(3).sum(), x, create_graph=True)
    got, = torch.autograd.grad(g.square().sum(), x)
    f = R.factor(9, 40, 0.3, seed=7)
    want = 36 * f ** 3 * (d(r) + f * d(x)) ** 3
    R.close(got, want, 28 * R.U * want.abs() + R.tiny(F32), "second derivative")


# ---- tracers --------------------------------------------------------------------------------------------------------

def _functions(B):
    def norm(x, r, w, b):
        return B.layer_norm(x, w, b)

    def drop(x, r, w, b):
        return B.dropout(x, 0.3, 5, 7, 1)

    def residual(x, r, w, b):
        return B.residual_norm(x, r, w, b, 1e-5, 0.3, 5, 7, 1)
    return {"layer_norm": norm, "dropout": drop, "residual_norm": residual}


def _inputs(seed, grad=False):
    return tuple(t.requires_grad_(grad) for t in (data(6, 40, BF16, seed), data(6, 40, F32, seed + 1),
                                                   data(1, 40, F32, seed + 2)[0], data(1, 40, F32, seed + 3)[0]))


def _equal(got, want):
    got, want = (t if isinstance(t, (tuple, list)) else (t,) for t in (got, want))
    assert len(got) == len(want)
    for p, q in zip(got, want):
        assert torch.equal(p, q)


@pytest.mark.parametrize("name", ["layer_norm", "dropout", "residual_norm"])
@pytest.mark.parametrize("grad", [False, True])
def test_a_jit_trace_holds_the_operator(B, name, grad):
    f = _functions(B)[name]
    traced = torch.jit.trace(f, _inputs(1, grad))
    assert "bilinear_hip::" in str(traced.graph)
    for seed in (1, 10):
        args = _inputs(seed, grad)
        got, want = traced(*args), f(*args)
        _equal(got, want)
        if grad:
            (got, want) = ((t,) if torch.is_tensor(t) else t for t in (got, want))
            ones = [torch.ones_like(t) for t in want]
            wrt = args[:1] if name == "dropout" else args if name == "residual_norm" else (args[0], *args[2:])
            _equal(torch.autograd.grad(got, wrt, ones), torch.autograd.grad(want, wrt, ones))


@pytest.mark.parametrize("name", ["layer_norm", "dropout", "residual_norm"])
def test_make_fx_holds_the_operator_and_its_backward(B, name):
    from torch.fx.experimental.proxy_tensor import make_fx
    f = _functions(B)[name]
    _equal(make_fx(f)(*_inputs(1))(*_inputs(10)), f(*_inputs(10)))

    def step(x, r, w, b):
        x = x.detach().requires_grad_()
        out = f(x, r, w, b)
        out = out if torch.is_tensor(out) else out[0]
        return torch.autograd.grad(out, x, torch.ones_like(out))[0]
    graph = make_fx(step)(*_inputs(1))
    assert sum(str(n.target).startswith("bilinear_hip.") for n in graph.graph.nodes) == 2
    _equal(graph(*_inputs(10)), step(*_inputs(10)))


@pytest.mark.parametrize("name", ["layer_norm", "dropout", "residual_norm"])
def test_the_backward_of_an_eager_graph_under_make_fx(B, name):
    from torch.fx.experimental.proxy_tensor import make_fx
    args = _inputs(1, True)
    out = _functions(B)[name](*args)
    out = (out,) if torch.is_tensor(out) else out
    wrt = args[:1] if name == "dropout" else args if name == "residual_norm" else (args[0], *args[2:])
    back = lambda *dy: torch.autograd.grad(out, wrt, dy, retain_graph=True)    # noqa: E731
    one, two = ([data(6, 40, t.dtype, s + k) for k, t in enumerate(out)] for s in (20, 30))
    graph = make_fx(back)(*one)
    assert any(str(n.target).startswith("bilinear_hip.") for n in graph.graph.nodes)
    _equal(graph(*two), back(*two))


def test_a_dispatch_mode_sees_the_operators(B):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(str(func))
            return func(*args, **(kwargs or {}))
    names, args = [], _inputs(1, True)
    want = [f(*args) for f in _functions(B).values()]
    with Seen():
        got = [f(*args) for f in _functions(B).values()]
    for p, q in zip(got, want):
        _equal(p, q)
    assert [n for n in names if n.startswith("bilinear_hip.")] == [
        "bilinear_hip.layer_norm.default", "bilinear_hip.row_dropout.default", "bilinear_hip.residual_norm.default"]


def test_modules_that_drop_are_not_traced_with_one_mask(B):
    x = data(6, 40, F32, 1)
    for m, args in ((B.Dropout(0.3), (x,)), (B.ResidualNorm(40, p=0.3).cuda(), (x, x))):
        with pytest.raises(RuntimeError, match="every call would draw the same mask"):
            torch.jit.trace(m, args)
        traced = torch.jit.trace(m.eval(), args)
        _equal(traced(*args), m(*args))


# ---- captures -------------------------------------------------------------------------------------------------------

def test_captured_modules_draw_again_what_a_restored_generator_drew(B):
    """What a checkpointed block does: the CPU generator's state is restored and the block called again, in one capture."""
    x = data(60, 48, F32, 1)
    drop, norm = B.Dropout(0.4), B.ResidualNorm(48, p=0.4).cuda()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    drop.set_device_step(step)
    norm.set_device_step(step)

    def block():
        return drop(x), norm(x, x)[1]
    with torch.no_grad():
        B.dropout(x, 0.4, seed=1, device_step=step)           # (loads the library outside the capture)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            state = torch.get_rng_state()
            first = block()
            torch.set_rng_state(state)
            again = block()
            other = block()
            step.add_(1)
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        _equal(again, first)
        for p, q in zip(other, first):
            assert not torch.equal(p, q)
        seen.append([t.clone() for t in first])
    for i in (1, 2):
        for p, q in zip(seen[i], seen[0]):
            assert not torch.equal(p, q)


def test_a_checkpointed_block_in_a_captured_step(B):
    """Forward, recomputation and backward in one graph: with the gradient of sum y each kept element of dx is the scale, so dx
    shows the recomputed mask beside the forward's."""
    from torch.utils.checkpoint import checkpoint
    drop, x = B.Dropout(0.4), torch.ones(30, 48, device="cuda", requires_grad=True)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    drop.set_device_step(step)

    def work():
        state = torch.get_rng_state()
        y = checkpoint(lambda t: _restored(drop, t, state), x, use_reentrant=False, preserve_rng_state=False)
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]

    def _restored(m, t, state):
        torch.set_rng_state(state)
        return m(t).square() * 0.5                 # (reads its input in the backward: it has to be recomputed)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = work()
        step.add_(1)
    masks = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        masks.append(y != 0)
        assert torch.equal(dx != 0, masks[-1]) and masks[-1].any() and not masks[-1].all()
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])


def test_compiled_functions_in_torchs_own_graphs(B):
    """mode="reduce-overhead" captures the compiled calls; the step on the device moves on between them."""
    x, dy = data(40, 96, F32, 1).requires_grad_(), data(40, 96, F32, 2)
    w, b = params(96, F32, 5)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def f(x, w, b, step):
        return B.layer_norm(B.dropout(x, 0.3, 5, 7, 2, 0, step), w, b)
    compiled = torch.compile(f, mode="reduce-overhead", fullgraph=True)
    outs = []
    for n in range(5):
        torch.compiler.cudagraph_mark_step_begin()
        y = compiled(x, w, b, step)
        got = [y.detach().clone()] + [t.clone() for t in torch.autograd.grad(y, (x, w, b), dy)]
        del y
        z = f(x, w, b, step)
        for p, q in zip(got, [z.detach(), *torch.autograd.grad(z, (x, w, b), dy)]):
            assert torch.equal(p, q), n
        outs.append(got[0])
        step.add_(1)
    assert not torch.equal(outs[3], outs[4])


@pytest.mark.parametrize("p", [0.0, 1e-7, 0.3])
@pytest.mark.parametrize("rows", [0, 3])
def test_the_operators_return_the_step_they_used(B, p, rows):
    op = torch.ops.bilinear_hip
    x = torch.zeros(rows, 24, device="cuda")
    step = torch.full((1,), 11, dtype=torch.int64, device="cuda")
    junk = [torch.full((1,), 77, dtype=torch.int64, device="cuda") for _ in range(8)]      # what a fresh allocation may hold
    del junk
    assert op.row_dropout(x, p, 1, 5, 0, 0, step)[1].item() == 16
    assert op.residual_norm(x, x, None, None, 1e-5, p, 1, 5, 0, 0, step)[4].item() == 16


def test_a_view_of_a_leaf_of_a_live_eager_graph_is_refused_in_a_capture(B):
    x = data(8, 16, F32, 1)
    w = params(32, F32, 5)[0]
    eager = B.layer_norm(x, w[:16])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="still part of an eager autograd graph"):
            B.layer_norm(x, w[:16])
        with torch.no_grad():
            z = B.layer_norm(x, w[:16])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, eager)


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


@pytest.mark.parametrize("operator", [False, True])
@pytest.mark.parametrize("dtype,rtype,p", [(F32, F32, 0.0), (F32, F32, 0.3), (BF16, F32, 0.3), (BF16, BF16, 0.0), (F16, F32, 0.0)])
def test_the_stream_alone_carries_its_gradient_past_a_row_without_statistics(B, operator, dtype, rtype, p):
    """Only h goes on: dresidual = dh and dx = dropout(dh), whatever the norm of that row would have been."""
    x, r, dh = data(5, 40, dtype, 1), data(5, 40, rtype, 2), data(5, 40, rtype, 3)
    x[1, 4], r[2, 5], r[3, 6] = float("inf"), float("nan"), float("-inf")
    x.requires_grad_(), r.requires_grad_()
    w, b = params(40, F32, 5)
    if operator:
        h = torch.ops.bilinear_hip.residual_norm(x, r, w, b, 1e-5, p, 9, 0, 0, 0, None)[1]
    else:
        h = B.residual_norm(x, r, w, b, p=p, seed=9)[1]
    dx, dr, dw, db = torch.autograd.grad(h, (x, r, w, b), dh)
    f = R.factor(5, 40, p, seed=9) if p else torch.ones(5, 40, dtype=torch.double)
    assert torch.equal(dr, dh)
    assert torch.equal(dx.cpu(), (d(dh) * f).float().to(dtype))
    assert dw.dtype == db.dtype == F32 and not dw.any() and not db.any()


def test_tensors_whose_storage_is_gone_are_refused(B):
    """(A parameter that a sharding library has freed is not a parameter that was left out.)"""
    x = data(4, 16, F32, 1).contiguous()
    gone = torch.ones(16, device="cuda")
    gone.untyped_storage().resize_(0)
    for call in (lambda: B.layer_norm(x, gone), lambda: B.layer_norm(x, None, gone), lambda: B.residual_norm(x, x, gone),
                 lambda: torch.ops.bilinear_hip.layer_norm(x, gone, None, 1e-5)):
        with pytest.raises(RuntimeError, match="no storage"):
            call()


def test_wrappers_of_function_transforms_are_refused(B):
    """None of them is taken for a parameter that was left out."""
    x, w = data(4, 16, F32, 1).contiguous(), params(16, F32, 5)[0].detach()
    for call in (lambda: torch.func.functionalize(lambda t: B.layer_norm(x, t))(w),
                 lambda: torch.func.functionalize(lambda t: B.residual_norm(x, x, None, t)[0])(w),
                 lambda: torch.func.grad(lambda t: B.layer_norm(x, t).sum())(w),
                 lambda: torch.vmap(lambda t: B.layer_norm(x, t))(w.expand(2, 16)),
                 lambda: torch.func.jvp(lambda t: B.layer_norm(x, t), (w,), (w,))):
        with pytest.raises(RuntimeError):
            call()
