"""Row operators without a GPU: the generator of the oracle, argument checks of the C ABI and of the Python surface, the
operators' shape functions, the modules' bookkeeping."""
import copy
import ctypes
import pickle

import numpy as np
import pytest
import torch

import bilinear_amd as B
import row_ops_util as R
from bilinear_amd import _native as N
from bilinear_amd import row_ops


def test_oracle_generator_known_answers():
    """Philox4x32-10's published vectors (Random123's known-answer file)."""
    zero = R.philox4x32_10([0, 0, 0, 0], (0, 0))
    assert [int(v) for v in zero] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = R.philox4x32_10([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF))
    assert [int(v) for v in ones] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_oracle_gradient_against_differences():
    """The oracle's gradients (double automatic differentiation) against central differences."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 11, generator=g, dtype=torch.double, requires_grad=True)
    w = torch.randn(11, generator=g, dtype=torch.double, requires_grad=True)
    b = torch.randn(11, generator=g, dtype=torch.double, requires_grad=True)
    f = R.factor(3, 11, 0.3, seed=5)
    assert torch.autograd.gradcheck(lambda x, w, b: R.norm64(x * f + x.flip(0), w, b, 1e-5)[0], (x, w, b))


def _buf(n=4096):
    return (ctypes.c_char * n)()


def _drop(p=0.1, seed=1, step=0, row_offset=0, layer=0):
    return ctypes.byref(N.RowDrop(p, seed, step, row_offset, None, None, layer, 0))


def test_c_abi_refuses_bad_arguments(native):
    """Refused on the host before anything is launched (no device here: a launch would fail with BLH_ERR_HIP)."""
    b = _buf()
    at = ctypes.addressof(b)
    at += -at % 16
    drop = native.blh_row_dropout
    assert drop(None, at, 8, at, None, 2, 8, 0) == -1
    assert drop(None, at, 8, at, _drop(), 2, 8, 3) == -1                       # type
    assert drop(None, at, -1, at, _drop(), 2, 8, 0) == -1                      # stride
    assert drop(None, at, 8, at, _drop(), -1, 8, 0) == -1
    assert drop(None, at, 8, at, _drop(), 2, 0, 0) == -1
    assert drop(None, at, 8, at, _drop(), 2, (1 << 24) + 1, 0) == -2
    assert drop(None, at, 8, at, _drop(), (1 << 43) + 1, 8, 0) == -2
    assert drop(None, at, 8, at, _drop(row_offset=(1 << 43) - 1), 2, 8, 0) == -2
    assert drop(None, at, 8, at, _drop(row_offset=-1), 2, 8, 0) == -1
    assert drop(None, at, 8, at, _drop(layer=-1), 2, 8, 0) == -1
    for p in (-0.1, 1.1, float("nan")):
        assert drop(None, at, 8, at, _drop(p=p), 2, 8, 0) == -1
    assert drop(None, None, 8, at, _drop(), 2, 8, 0) == -1
    assert drop(None, at + 2, 8, at, _drop(), 2, 8, 0) == -1                   # fp32 off its alignment
    assert drop(None, at + 1, 8, at, _drop(), 2, 8, 1) == -1
    assert drop(None, None, 8, None, _drop(), 0, 8, 0) == 0                    # no rows: nothing to do
    fwd = native.blh_layer_norm_forward
    assert fwd(None, at, 8, None, None, -1e-5, at, None, None, 2, 8, 0, 0) == -1
    assert fwd(None, at, 8, None, None, float("nan"), at, None, None, 2, 8, 0, 0) == -1
    assert fwd(None, at, 8, None, None, 1e-5, at, at, None, 2, 8, 0, 0) == -1  # mean without rstd
    assert fwd(None, at, 8, None, None, 1e-5, at, None, None, 2, 8, 0, 1) == -1    # bf16 weights on fp32 rows
    assert fwd(None, at, 8, at + 2, None, 1e-5, at, None, None, 2, 8, 1, 0) == -1  # fp32 weight off its alignment
    assert fwd(None, None, 8, None, None, 1e-5, None, None, None, 0, 8, 0, 0) == 0
    assert native.blh_row_norm_workspace_bytes(-1, 8) == -1
    assert native.blh_row_norm_workspace_bytes(4, 0) == -1
    assert native.blh_row_norm_workspace_bytes(4, 1 << 25) == -2
    need = native.blh_row_norm_workspace_bytes(64, 1024)
    assert need >= 256
    bwd = native.blh_layer_norm_backward
    assert bwd(None, at, 8, at, 8, None, at, at, at, at, at, None, 0, 2, 8, 0, 0) == -1     # no workspace
    assert bwd(None, at, 8, at, 8, None, at, at, at, at, at, at, 16, 2, 8, 0, 0) == -4
    assert bwd(None, at, 8, at, 8, None, at, at, at, at, at, at + 4, 1 << 20, 2, 8, 0, 0) == -1
    assert bwd(None, None, 8, at, 8, None, at, at, at, None, None, None, 0, 2, 8, 0, 0) == -1
    rf = native.blh_residual_norm_forward
    assert rf(None, at, 8, at, 8, None, None, 1e-5, None, at, at, None, None, 2, 8, 0, 1, 0) == -1   # bf16 stream, fp32 rows
    assert rf(None, at, 8, at, 8, None, None, 1e-5, None, at, at, None, None, 2, 8, 1, 2, 0) == -1
    assert rf(None, at, 8, None, 8, None, None, 1e-5, None, at, at, None, None, 2, 8, 0, 0, 0) == -1
    assert rf(None, at, 8, at, 8, None, None, 1e-5, _drop(p=2.0), at, at, None, None, 2, 8, 0, 0, 0) == -1
    rb = native.blh_residual_norm_backward
    assert rb(None, at, 8, None, -1, at, 8, None, at, at, None, at, at, None, None, None, 0, 2, 8, 0, 0, 0) == -1
    assert rb(None, at, 8, None, 0, at, 8, None, at, at, None, at, at, at, at, at, 16, 2, 8, 0, 0, 0) == -4


def test_python_surface_refuses_bad_arguments(monkeypatch):
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="only on a HIP device"):
        B.layer_norm(x)
    with pytest.raises(RuntimeError, match="only on a HIP device"):
        B.dropout(x, 0.5, seed=1)
    with pytest.raises(RuntimeError, match="only on a HIP device"):
        B.residual_norm(x, x)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.ops.bilinear_hip.layer_norm(x, None, None, 1e-5)

    class Hip:       # the checks behind the device's
        type = "cuda"
    fake = lambda shape, dtype=torch.float32: type("T", (), {   # noqa: E731
        "device": Hip, "dtype": dtype, "shape": torch.Size(shape), "dim": lambda s: len(shape),
        "numel": lambda s: int(np.prod(shape)), "requires_grad": False})()
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        row_ops._check_rows(fake((2, 8), torch.float64), "x")
    with pytest.raises(RuntimeError, match="at least one column"):
        row_ops._check_rows(fake((2, 0)), "x")
    with pytest.raises(RuntimeError, match="at least one column"):
        row_ops._check_rows(fake(()), "x")
    x = fake((2, 8), torch.bfloat16)
    with pytest.raises(RuntimeError, match="weight has shape"):
        row_ops._check_params(x, fake((9,)), None)
    with pytest.raises(RuntimeError, match="bias is torch.float16"):
        row_ops._check_params(x, None, fake((8,), torch.float16))
    with pytest.raises(RuntimeError, match="one type for both"):
        row_ops._check_params(x, fake((8,)), fake((8,), torch.bfloat16))
    with pytest.raises(RuntimeError, match="residual has shape"):
        row_ops._check_like(fake((2, 9)), x, "residual", (torch.float32,))
    with pytest.raises(RuntimeError, match="residual is torch.float16"):
        row_ops._check_like(fake((2, 8), torch.float16), x, "residual", (torch.bfloat16, torch.float32))
    good = dict(p=0.5, seed=1, step=0, layer=0, row_offset=0, device_step=None, x=x)
    row_ops._check_draws(**good)
    for bad in (dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(seed=-1), dict(seed=1 << 63), dict(step=-1),
                dict(step=1 << 63), dict(layer=-1), dict(layer=1 << 31), dict(row_offset=-1), dict(row_offset=1 << 43)):
        with pytest.raises(ValueError):
            row_ops._check_draws(**{**good, **bad})
    with pytest.raises(RuntimeError, match="one int64"):
        row_ops._check_draws(**{**good, "device_step": torch.zeros(1)})
    with pytest.raises(ValueError):
        row_ops._check_eps(-1.0)


def test_rows_are_read_in_place_where_they_can_be():
    wide = torch.zeros(6, 20)
    for t, ld in ((torch.zeros(4, 8), 8), (wide[:, 3:11], 20), (wide[::2, :8], 40), (torch.zeros(1, 8).expand(5, 8), 0),
                  (torch.zeros(2, 3, 20)[..., 4:12], 20), (torch.zeros(8), 8), (torch.zeros(0, 8), 8)):
        v, got = row_ops._rows(t)
        assert v.data_ptr() == t.data_ptr() and got == ld
    for t in (torch.zeros(8, 4).t(), torch.zeros(4, 16)[:, ::2], torch.zeros(2, 3, 8).transpose(0, 1), torch.zeros(()).expand(4, 8)):
        v, got = row_ops._rows(t)
        assert v.is_contiguous() and v.shape == t.shape and got == t.shape[-1]


def test_operators_trace_through_their_fake_implementations():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 5, 48, device="cuda", dtype=torch.bfloat16)
        r = torch.empty(3, 5, 48, device="cuda")
        w = torch.empty(48, device="cuda")
        op = torch.ops.bilinear_hip
        y, mean, rstd = op.layer_norm(x, w, w, 1e-5)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == rstd.shape == (15,)
        dx, dw, db = op.layer_norm_backward(y, x, w, mean, rstd, True, True, False, 0)
        assert dx.shape == x.shape and dw.shape == (48,) and dw.dtype == torch.float32 and db.shape == (0,)
        y, used = op.row_dropout(x, 0.1, 1, 2, 3, 4, None)
        assert y.shape == x.shape and used.shape == (0,)
        step = torch.zeros(1, dtype=torch.int64, device="cuda")
        y, h, mean, rstd, used = op.residual_norm(x, r, w, None, 1e-5, 0.1, 1, 2, 3, 4, step)
        assert y.dtype == x.dtype and h.dtype == r.dtype and used.shape == (1,)
        dx, dr, dw, db = op.residual_norm_backward(y, None, h, w, mean, rstd, 0.1, 1, 2, 3, 4, used, True, True, True, True, 0)
        assert dx.dtype == x.dtype and dr.dtype == r.dtype and dw.shape == db.shape == (48,)


def test_modules_mirror_torch_and_never_share_a_mask():
    ref = torch.nn.LayerNorm(16, eps=1e-3)
    for m in (B.LayerNorm(16, eps=1e-3), B.ResidualNorm(16, p=0.2, eps=1e-3)):
        assert list(m.state_dict()) == list(ref.state_dict()) and m.eps == ref.eps
        m.load_state_dict(ref.state_dict())
    assert B.LayerNorm(16, bias=False).bias is None and B.LayerNorm(16, elementwise_affine=False).weight is None
    with pytest.raises(RuntimeError):
        B.LayerNorm((4, 4))
    with pytest.raises(RuntimeError):
        B.Dropout(0.5, inplace=True)
    with pytest.raises(ValueError):
        B.Dropout(1.5)
    with pytest.raises(ValueError):
        B.ResidualNorm(16, p=-0.5)
    a, b = B.Dropout(0.1), B.Dropout(0.1)
    c, d = copy.deepcopy(a), pickle.loads(pickle.dumps(a))
    assert len({m._layer for m in (a, b, c, d)}) == 4
    stage = B.heavy_linear(4, 4)
    assert stage._stage_id not in {m._layer for m in (a, b, c, d)}
    first, second = a._next_draws(), a._next_draws()
    assert first["seed"] == second["seed"] == torch.initial_seed() & ((1 << 63) - 1)
    assert second["step"] == first["step"] + 1
    assert a.eval()(torch.ones(3)) is not None and torch.equal(B.Dropout(0.0)(torch.ones(3)), torch.ones(3))


def test_dropout_in_a_capture_needs_a_step_on_the_device(monkeypatch):
    monkeypatch.setattr(row_ops, "_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    m = B.Dropout(0.1)
    with pytest.raises(RuntimeError, match="every replay would draw the same mask"):
        m._next_draws()
    with pytest.raises(RuntimeError):
        m.set_device_step(torch.zeros(2, dtype=torch.int64))
    m.set_device_step(torch.zeros(1, dtype=torch.int64))
    first, second = m._next_draws(), m._next_draws()
    assert first["device_step"] is m._device_step and first["step"] != second["step"] and first["step"] >= 1 << 32


def test_leaves_of_a_live_eager_graph_are_refused_in_a_capture():
    """row_ops._apply marks the accumulators of an eager graph on the default stream; a capture that meets a marked one is
    refused (here with a plain function on the CPU in the operator's place)."""
    leaf = torch.nn.Parameter(torch.ones(4))
    out = leaf * 2
    out.grad_fn.next_functions[0][0].metadata[row_ops._EAGER] = True
    with pytest.raises(RuntimeError, match="still part of an eager autograd graph"):
        row_ops._refuse_eager_leaves((None, leaf))
    del out
    row_ops._refuse_eager_leaves((None, leaf, torch.ones(4)))       # the graph is gone: nothing to refuse
