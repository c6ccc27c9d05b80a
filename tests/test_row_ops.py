"""Row operators without a GPU: the generator of the oracle, argument checks of the C ABI and of the Python surface, the
operators' shape functions, the modules' bookkeeping."""
import copy
import ctypes
import pickle

import pytest
import torch

import bilinear_amd as B
import row_ops_util as R
from bilinear_amd import _native as N


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
    same = N.RowDrop(0.1, 1, 0, 0, at, at, 0, 0)                               # the step read is the step written
    assert drop(None, at, 8, at, ctypes.byref(same), 2, 8, 0) == -1
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
    assert native.blh_row_norm_workspace_bytes(0, 1024) == 0 and native.blh_row_norm_workspace_bytes(5000, 1024) > 0
    bwd = native.blh_layer_norm_backward
    assert bwd(None, at, 8, at, 8, None, at, at, at, at, at, None, 0, 5000, 8, 0, 0) == -1     # no workspace
    assert bwd(None, at, 8, at, 8, None, at, at, at, at, at, at, 16, 5000, 8, 0, 0) == -4
    assert bwd(None, at, 8, at, 8, None, at, at, at, at, at, at + 4, 1 << 20, 5000, 8, 0, 0) == -1
    assert bwd(None, None, 8, at, 8, None, at, at, at, None, None, None, 0, 2, 8, 0, 0) == -1
    rf = native.blh_residual_norm_forward
    assert rf(None, at, 8, at, 8, None, None, 1e-5, None, at, at, None, None, 2, 8, 0, 1, 0) == -1   # bf16 stream, fp32 rows
    assert rf(None, at, 8, at, 8, None, None, 1e-5, None, at, at, None, None, 2, 8, 1, 2, 0) == -1
    assert rf(None, at, 8, None, 8, None, None, 1e-5, None, at, at, None, None, 2, 8, 0, 0, 0) == -1
    assert rf(None, at, 8, at, 8, None, None, 1e-5, _drop(p=2.0), at, at, None, None, 2, 8, 0, 0, 0) == -1
    rb = native.blh_residual_norm_backward
    assert rb(None, at, 8, None, -1, at, 8, None, at, at, None, at, at, None, None, None, 0, 2, 8, 0, 0, 0) == -1
    assert rb(None, at, 8, None, 0, at, 8, None, at, at, None, at, at, at, at, at, 16, 5000, 8, 0, 0, 0) == -4


def test_python_surface_refuses_bad_arguments():
    """The checks in front of the native calls, on tensors without storage where they need a HIP device's."""
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="only on a HIP device"):
        B.layer_norm(x)
    with pytest.raises(RuntimeError, match="only on a HIP device"):
        B.dropout(x, 0.5, seed=1)
    with pytest.raises(RuntimeError, match="only on a HIP device"):
        B.residual_norm(x, x)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.ops.bilinear_hip.layer_norm(x, None, None, 1e-5)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(shape, dtype=dtype, device="cuda")
        x = t(2, 8)
        f32 = dict(dtype=torch.float32)
        for call, what in (
                (lambda: B.layer_norm(t(2, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
                (lambda: B.layer_norm(t(2, 0)), "at least one column"),
                (lambda: B.layer_norm(t()), "at least one column"),
                (lambda: B.layer_norm(x, t(9, **f32)), "weight has shape"),
                (lambda: B.layer_norm(x, t(1, 8, **f32)), "weight has shape"),
                (lambda: B.layer_norm(x, None, t(8, dtype=torch.float16)), "bias is Half"),
                (lambda: B.layer_norm(x, t(8, **f32), t(8)), "one type for both"),
                (lambda: B.layer_norm(x, torch.empty(8)), "weight is on 'cpu'"),
                (lambda: B.residual_norm(x, t(2, 9)), "residual has shape"),
                (lambda: B.residual_norm(x, t(2, 8, dtype=torch.float16)), "residual is Half"),
                (lambda: B.residual_norm(t(2, 8, **f32), x), "residual is BFloat16"),
                (lambda: B.residual_norm(x, torch.empty(2, 8)), "residual is on 'cpu'"),
                (lambda: B.dropout(x, 0.5, seed=1, device_step=t(1, **f32)), "one int64"),
                (lambda: B.dropout(x, 0.5, seed=1, device_step=t(2, dtype=torch.int64)), "one int64"),
                (lambda: B.dropout(x, 0.5, seed=1, device_step=torch.empty(1, dtype=torch.int64)), "one int64")):
            with pytest.raises(RuntimeError, match=what):
                call()
        for bad in (dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(seed=-1), dict(step=-1), dict(layer=-1),
                    dict(layer=1 << 31), dict(row_offset=-1), dict(row_offset=1 << 43)):
            with pytest.raises(ValueError):
                B.dropout(x, **{"p": 0.5, "seed": 1, **bad})
            with pytest.raises(ValueError):
                B.residual_norm(x, x, **{"p": 0.5, "seed": 1, **bad})
        for eps in (-1.0, float("nan")):
            with pytest.raises(ValueError):
                B.layer_norm(x, eps=eps)
        for bad in (dict(seed=1 << 63), dict(step=1 << 63)):
            with pytest.raises((TypeError, ValueError)):
                B.dropout(x, **{"p": 0.5, "seed": 1, **bad})


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
    torch.manual_seed(11)
    first, second = a._next_draws(), a._next_draws()
    assert first["seed"] == second["seed"] and first["step"] != second["step"]
    torch.manual_seed(11)
    assert a._next_draws() == first and b._next_draws()["layer"] != first["layer"]
    assert torch.equal(B.Dropout(0.0)(torch.ones(3)), torch.ones(3)) and torch.equal(a.eval()(torch.ones(3)), torch.ones(3))


def test_dropout_in_a_capture_needs_a_step_on_the_device(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    m = B.Dropout(0.1)
    with pytest.raises(RuntimeError, match="every replay would draw the same mask"):
        m._next_draws()
    with pytest.raises(RuntimeError):
        m.set_device_step(torch.zeros(2, dtype=torch.int64))
    m.set_device_step(torch.zeros(1, dtype=torch.int64))
    first, second = m._next_draws(), m._next_draws()
    assert first["device_step"] is m._device_step and first["step"] != second["step"] and first["step"] >= 1 << 32
