"""Operators on rows: ``layer_norm``, ``dropout`` with a mask that is never stored, and ``residual_norm``
(``h = residual + dropout(x)``, ``y = layer_norm(h)``), forward and backward, on libbilinear_hip.so's
``blh_layer_norm_*``, ``blh_row_dropout`` and ``blh_residual_norm_*``.

They are the counterparts of a stage's BatchNorm1d and Dropout(0.5) (/root/reference/model/bilinear.py:7-13) that need no
batch and no stored mask.  Three surfaces, as for the lifter:

    y = bilinear_amd.layer_norm(x, weight, bias)                      # functions, differentiable
    y = bilinear_amd.dropout(x, 0.1, seed=7, step=3, layer=0)
    y, h = bilinear_amd.residual_norm(x, h, weight, bias, p=0.1, seed=7, step=3, layer=1)
    bilinear_amd.LayerNorm(1024), .Dropout(0.1), .ResidualNorm(1024, p=0.1)     # modules
    torch.ops.bilinear_hip.{layer_norm, row_dropout, residual_norm, ...}        # custom operators (torch.compile)

The last axis is the row.  Types: x float32 / bfloat16 / float16; weight and bias float32 or x's type; the residual
stream (``residual``, ``h``) float32 or x's type.  Rows of a wider tensor (last axis dense) are read in place.  Tensors
must live on a HIP device: there is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch
import torch.nn as nn

from . import _native as N
from .ops import _LIB

__all__ = ["layer_norm", "dropout", "residual_norm", "LayerNorm", "Dropout", "ResidualNorm"]

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # blh_dtype
_LIMIT63 = 1 << 63


# ---- checks ---------------------------------------------------------------------------------------------------------

def _check_rows(t, what):
    if t.device.type != "cuda":
        raise RuntimeError("bilinear_amd row operators run only on a HIP device (MI355X); %s is on '%s' and there is no "
                           "CPU/ATen fallback." % (what, t.device))
    if t.dtype not in _CODES:
        raise RuntimeError("%s must be float32, bfloat16 or float16, got %s" % (what, t.dtype))
    if t.dim() < 1 or t.shape[-1] < 1:
        raise RuntimeError("%s needs a last axis of at least one column, got shape %s" % (what, tuple(t.shape)))


def _check_like(t, x, what, dtypes):
    if t.device != x.device:
        raise RuntimeError("%s is on '%s' where '%s' is expected" % (what, t.device, x.device))
    if t.shape != x.shape:
        raise RuntimeError("%s has shape %s where %s is expected" % (what, tuple(t.shape), tuple(x.shape)))
    if t.dtype not in dtypes:
        raise RuntimeError("%s is %s where %s is expected" % (what, t.dtype, " or ".join(str(d) for d in dtypes)))


def _check_params(x, weight, bias):
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.device != x.device:
            raise RuntimeError("%s is on '%s' where '%s' is expected" % (what, t.device, x.device))
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise RuntimeError("%s has shape %s where (%d,) is expected" % (what, tuple(t.shape), x.shape[-1]))
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise RuntimeError("%s is %s where float32 or %s is expected" % (what, t.dtype, x.dtype))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight is %s and bias %s: one type for both is expected" % (weight.dtype, bias.dtype))


def _check_eps(eps):
    if not eps >= 0.0:
        raise ValueError("eps must not be negative, got %r" % (eps,))


def _check_draws(p, seed, step, layer, row_offset, device_step, x):
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout probability has to be between 0 and 1, got %r" % (p,))
    for v, what in ((seed, "seed"), (step, "step")):
        if not 0 <= v < _LIMIT63:
            raise ValueError("%s must be in [0, 2^63), got %r" % (what, v))
    if not 0 <= layer < 1 << 31:
        raise ValueError("layer must be in [0, 2^31), got %r" % (layer,))
    if not 0 <= row_offset < 1 << 43:
        raise ValueError("row_offset must be in [0, 2^43), got %r" % (row_offset,))
    if device_step is not None and (device_step.dtype != torch.int64 or device_step.numel() != 1
                                    or device_step.device != x.device):
        raise RuntimeError("device_step must be one int64 on '%s'" % (x.device,))


# ---- native calls (tensors are checked; impls of the custom operators) -----------------------------------------------

def _rows(t):
    """(tensor to read, elements between its rows): rows are read in place where the last axis is dense and the leading
    axes collapse to one, else from a dense copy."""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, width
    if t.stride(-1) == 1 or width == 1:
        if t.dim() == 2:
            return t, t.stride(0)
        try:
            v = t.view(-1, width)
            return v, v.stride(0)
        except RuntimeError:
            pass
    return t.contiguous(), width


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _launch(name, x, *args):
    """One entry point on the current stream of x's device (which need not be the current device)."""
    index = x.get_device()
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _launch(name, x, *args)
    status = getattr(N.lib(), name)(torch._C._cuda_getCurrentRawStream(index), *args)
    if status:
        N.check(status, name)


def _drop(p, seed, step, layer, row_offset, device_step, used):
    return ctypes.byref(N.RowDrop(p, seed, step, row_offset, _ptr(device_step), _ptr(used), layer, 0))


def _param_code(x, weight, bias):
    t = weight if weight is not None else bias
    return 0 if t is None else _CODES[t.dtype]


def _workspace(x, rows, width):
    need = N.lib().blh_row_norm_workspace_bytes(rows, width)
    if need < 0:
        N.check(int(need), "blh_row_norm_workspace_bytes")
    return torch.empty(need, dtype=torch.uint8, device=x.device), need


def _layer_norm(x, weight, bias, eps, save=True):
    width = x.shape[-1]
    rows = x.numel() // width
    src, ld = _rows(x)
    weight, bias = _dense(weight), _dense(bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows) if save else (2, 0), dtype=torch.float32, device=x.device)
    mean, rstd = stats.unbind(0)
    _launch("blh_layer_norm_forward", x, src.data_ptr(), ld, _ptr(weight), _ptr(bias), eps, y.data_ptr(),
            mean.data_ptr() if save else None, rstd.data_ptr() if save else None, rows, width, _CODES[x.dtype],
            _param_code(x, weight, bias))
    return y, mean, rstd


def _grads_of_params(x, width, need_weight, need_bias, code):
    dtype = torch.float32 if code == 0 else x.dtype
    dw = torch.empty(width if need_weight else 0, dtype=dtype, device=x.device)
    db = torch.empty(width if need_bias else 0, dtype=dtype, device=x.device)
    return dw, db


def _layer_norm_backward(dy, x, weight, mean, rstd, need_x, need_weight, need_bias, param_code):
    width = x.shape[-1]
    rows = x.numel() // width
    (dy_, lddy), (x_, ldx) = _rows(dy), _rows(x)
    weight = _dense(weight)
    dx = torch.empty(x.shape if need_x else (0,), dtype=x.dtype, device=x.device)
    dw, db = _grads_of_params(x, width, need_weight, need_bias, param_code)
    ws, size = _workspace(x, rows, width) if need_weight or need_bias else (None, 0)
    _launch("blh_layer_norm_backward", x, dy_.data_ptr(), lddy, x_.data_ptr(), ldx, _ptr(weight), mean.data_ptr(),
            rstd.data_ptr(), dx.data_ptr() if need_x else None, dw.data_ptr() if need_weight else None,
            db.data_ptr() if need_bias else None, _ptr(ws), size, rows, width, _CODES[x.dtype], param_code)
    return dx, dw, db


def _row_dropout(x, p, seed, step, layer, row_offset, device_step):
    width = x.shape[-1]
    src, ld = _rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    used = torch.empty(0 if device_step is None else 1, dtype=torch.int64, device=x.device)
    _launch("blh_row_dropout", x, src.data_ptr(), ld, y.data_ptr(),
            _drop(p, seed, step, layer, row_offset, device_step, None if device_step is None else used),
            x.numel() // width, width, _CODES[x.dtype])
    return y, used


def _residual_norm(x, residual, weight, bias, eps, p, seed, step, layer, row_offset, device_step, save=True):
    width = x.shape[-1]
    rows = x.numel() // width
    (src, ldx), (res, ldr) = _rows(x), _rows(residual)
    weight, bias = _dense(weight), _dense(bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    stats = torch.empty((2, rows) if save else (2, 0), dtype=torch.float32, device=x.device)
    mean, rstd = stats.unbind(0)
    used = torch.empty(0 if device_step is None else 1, dtype=torch.int64, device=x.device)
    drop = _drop(p, seed, step, layer, row_offset, device_step, None if device_step is None else used) if p else None
    _launch("blh_residual_norm_forward", x, src.data_ptr(), ldx, res.data_ptr(), ldr, _ptr(weight), _ptr(bias), eps, drop,
            y.data_ptr(), h.data_ptr(), mean.data_ptr() if save else None, rstd.data_ptr() if save else None, rows, width,
            _CODES[x.dtype], _CODES[residual.dtype], _param_code(x, weight, bias))
    return y, h, mean, rstd, used


def _residual_norm_backward(dy, dh, h, weight, mean, rstd, p, seed, step, layer, row_offset, device_step, need_x,
                            need_residual, need_weight, need_bias, param_code):
    width = h.shape[-1]
    rows = h.numel() // width
    (dy_, lddy), (h_, ldh) = _rows(dy), _rows(h)
    dh_, lddh = (None, 0) if dh is None else _rows(dh)
    weight = _dense(weight)
    dx = torch.empty(h.shape if need_x else (0,), dtype=dy.dtype, device=h.device)
    dres = torch.empty(h.shape if need_residual else (0,), dtype=h.dtype, device=h.device)
    dw, db = _grads_of_params(dy, width, need_weight, need_bias, param_code)
    ws, size = _workspace(h, rows, width) if need_weight or need_bias else (None, 0)
    drop = _drop(p, seed, step, layer, row_offset, device_step, None) if p else None
    _launch("blh_residual_norm_backward", h, dy_.data_ptr(), lddy, _ptr(dh_), lddh, h_.data_ptr(), ldh, _ptr(weight),
            mean.data_ptr(), rstd.data_ptr(), drop, dx.data_ptr() if need_x else None,
            dres.data_ptr() if need_residual else None, dw.data_ptr() if need_weight else None,
            db.data_ptr() if need_bias else None, _ptr(ws), size, rows, width, _CODES[dy.dtype], _CODES[h.dtype],
            param_code)
    return dx, dres, dw, db


# ---- custom operators -----------------------------------------------------------------------------------------------
# All functional.  Outputs that were not asked for come back empty.

_DRAWS = "float p, SymInt seed, SymInt step, SymInt layer, SymInt row_offset, Tensor? device_step"
_LIB.define("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor)")
_LIB.define("layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor mean, Tensor rstd, bool need_x, "
            "bool need_weight, bool need_bias, int param_code) -> (Tensor, Tensor, Tensor)")
_LIB.define("row_dropout(Tensor x, %s) -> (Tensor, Tensor)" % _DRAWS)
_LIB.define("residual_norm(Tensor x, Tensor residual, Tensor? weight, Tensor? bias, float eps, %s) "
            "-> (Tensor, Tensor, Tensor, Tensor, Tensor)" % _DRAWS)
_LIB.define("residual_norm_backward(Tensor dy, Tensor? dh, Tensor h, Tensor? weight, Tensor mean, Tensor rstd, %s, "
            "bool need_x, bool need_residual, bool need_weight, bool need_bias, int param_code) "
            "-> (Tensor, Tensor, Tensor, Tensor)" % _DRAWS)


def _op_layer_norm(x, weight, bias, eps):
    _check_rows(x, "x")
    _check_params(x, weight, bias)
    _check_eps(eps)
    return _layer_norm(x, weight, bias, eps)


def _check_stats(x, mean, rstd):
    rows = x.numel() // x.shape[-1]
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous() or t.device != x.device:
            raise RuntimeError("%s must be %d dense float32 values on '%s'" % (what, rows, x.device))


def _check_param_code(x, code):
    if code not in (0, _CODES[x.dtype]):
        raise RuntimeError("param_code must be 0 (float32) or %d (%s)" % (_CODES[x.dtype], x.dtype))


def _op_layer_norm_backward(dy, x, weight, mean, rstd, need_x, need_weight, need_bias, param_code):
    _check_rows(x, "x")
    _check_like(dy, x, "dy", (x.dtype,))
    _check_params(x, weight, None)
    _check_stats(x, mean, rstd)
    _check_param_code(x, param_code)
    if weight is not None and _CODES[weight.dtype] != param_code:
        raise RuntimeError("param_code is not the weight's type")
    return _layer_norm_backward(dy, x, weight, mean, rstd, need_x, need_weight, need_bias, param_code)


def _op_row_dropout(x, p, seed, step, layer, row_offset, device_step):
    _check_rows(x, "x")
    _check_draws(p, seed, step, layer, row_offset, device_step, x)
    return _row_dropout(x, p, seed, step, layer, row_offset, device_step)


def _op_residual_norm(x, residual, weight, bias, eps, p, seed, step, layer, row_offset, device_step):
    _check_rows(x, "x")
    _check_like(residual, x, "residual", (x.dtype, torch.float32))
    _check_params(x, weight, bias)
    _check_eps(eps)
    _check_draws(p, seed, step, layer, row_offset, device_step, x)
    return _residual_norm(x, residual, weight, bias, eps, p, seed, step, layer, row_offset, device_step)


def _op_residual_norm_backward(dy, dh, h, weight, mean, rstd, p, seed, step, layer, row_offset, device_step, need_x,
                               need_residual, need_weight, need_bias, param_code):
    _check_rows(dy, "dy")
    _check_like(h, dy, "h", (dy.dtype, torch.float32))
    if dh is not None:
        _check_like(dh, dy, "dh", (h.dtype,))
    _check_params(dy, weight, None)
    _check_stats(h, mean, rstd)
    _check_param_code(dy, param_code)
    if weight is not None and _CODES[weight.dtype] != param_code:
        raise RuntimeError("param_code is not the weight's type")
    _check_draws(p, seed, step, layer, row_offset, device_step, dy)
    return _residual_norm_backward(dy, dh, h, weight, mean, rstd, p, seed, step, layer, row_offset, device_step, need_x,
                                   need_residual, need_weight, need_bias, param_code)


for _name, _impl in (("layer_norm", _op_layer_norm), ("layer_norm_backward", _op_layer_norm_backward),
                     ("row_dropout", _op_row_dropout), ("residual_norm", _op_residual_norm),
                     ("residual_norm_backward", _op_residual_norm_backward)):
    _LIB.impl(_name, _impl, "CUDA")


def _new(x, shape, dtype=None):
    return x.new_empty(shape, dtype=dtype or x.dtype)


def _row_count(x):
    rows = 1
    for n in x.shape[:-1]:
        rows = rows * n
    return rows


def _fake_stats(x):
    return _new(x, (_row_count(x),), torch.float32), _new(x, (_row_count(x),), torch.float32)


def _fake_params(x, need_weight, need_bias, code):
    dtype = torch.float32 if code == 0 else x.dtype
    return (_new(x, (x.shape[-1] if need_weight else 0,), dtype), _new(x, (x.shape[-1] if need_bias else 0,), dtype))


torch.library.register_fake("bilinear_hip::layer_norm", lambda x, weight, bias, eps: (
    _new(x, x.shape),) + _fake_stats(x), lib=_LIB)
torch.library.register_fake("bilinear_hip::layer_norm_backward", lambda dy, x, weight, mean, rstd, nx, nw, nb, code: (
    _new(x, x.shape if nx else (0,)),) + _fake_params(x, nw, nb, code), lib=_LIB)
torch.library.register_fake("bilinear_hip::row_dropout", lambda x, p, seed, step, layer, row_offset, device_step: (
    _new(x, x.shape), _new(x, (0 if device_step is None else 1,), torch.int64)), lib=_LIB)
torch.library.register_fake(
    "bilinear_hip::residual_norm",
    lambda x, residual, weight, bias, eps, p, seed, step, layer, row_offset, device_step: (
        _new(x, x.shape), _new(residual, x.shape)) + _fake_stats(x) + (
        _new(x, (0 if device_step is None else 1,), torch.int64),), lib=_LIB)
torch.library.register_fake(
    "bilinear_hip::residual_norm_backward",
    lambda dy, dh, h, weight, mean, rstd, p, seed, step, layer, row_offset, device_step, nx, nr, nw, nb, code: (
        _new(dy, h.shape if nx else (0,)), _new(h, h.shape if nr else (0,))) + _fake_params(dy, nw, nb, code), lib=_LIB)


def _pick(needed, grads):
    return tuple(g if n else None for n, g in zip(needed, grads))


def _ln_setup(ctx, inputs, output):
    x, weight, bias, _ = inputs
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.code = _param_code(x, weight, bias)


def _ln_formula(ctx, dy, dmean, drstd):
    x, weight, mean, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad[:3]
    return _pick(need, torch.ops.bilinear_hip.layer_norm_backward(dy, x, weight, mean, rstd, *need, ctx.code)) + (None,)


def _drop_setup(ctx, inputs, output):
    _, p, seed, step, layer, row_offset, device_step = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(*(() if device_step is None else (output[1],)))
    ctx.draws = (p, seed, step if device_step is None else 0, layer, row_offset)


def _drop_formula(ctx, dy, dused):
    used = ctx.saved_tensors[0] if ctx.saved_tensors else None
    return (torch.ops.bilinear_hip.row_dropout(dy, *ctx.draws, used)[0],) + (None,) * 6


def _res_setup(ctx, inputs, output):
    x, residual, weight, bias, _, p, seed, step, layer, row_offset, device_step = inputs
    ctx.mark_non_differentiable(*output[2:])
    ctx.save_for_backward(output[1], weight, output[2], output[3], None if device_step is None else output[4])
    ctx.draws = (p, seed, step if device_step is None else 0, layer, row_offset)
    ctx.code = _param_code(x, weight, bias)


def _res_formula(ctx, dy, dh, *unused):
    h, weight, mean, rstd, used = ctx.saved_tensors
    need = ctx.needs_input_grad[:4]
    return _pick(need, torch.ops.bilinear_hip.residual_norm_backward(
        dy, dh, h, weight, mean, rstd, *ctx.draws, used, *need, ctx.code)) + (None,) * 7


torch.library.register_autograd("bilinear_hip::layer_norm", _ln_formula, setup_context=_ln_setup, lib=_LIB)
torch.library.register_autograd("bilinear_hip::row_dropout", _drop_formula, setup_context=_drop_setup, lib=_LIB)
torch.library.register_autograd("bilinear_hip::residual_norm", _res_formula, setup_context=_res_setup, lib=_LIB)


# ---- eager autograd bridges (the same native calls without the operator dispatch) ------------------------------------

_once = torch.autograd.function.once_differentiable


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _layer_norm(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.code = _param_code(x, weight, bias)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        return _pick(need, _layer_norm_backward(dy, x, weight, mean, rstd, *need, ctx.code)) + (None,)


class _DropoutFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, step, layer, row_offset, device_step):
        y, used = _row_dropout(x, p, seed, step, layer, row_offset, device_step)
        ctx.used = None if device_step is None else used
        ctx.draws = (p, seed, step if device_step is None else 0, layer, row_offset)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        return (_row_dropout(dy, *ctx.draws, ctx.used)[0],) + (None,) * 6


class _ResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, seed, step, layer, row_offset, device_step):
        y, h, mean, rstd, used = _residual_norm(x, residual, weight, bias, eps, p, seed, step, layer, row_offset,
                                                device_step)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, weight, mean, rstd)
        ctx.used = None if device_step is None else used
        ctx.draws = (p, seed, step if device_step is None else 0, layer, row_offset)
        ctx.code, ctx.dtype = _param_code(x, weight, bias), x.dtype
        return y, h

    @staticmethod
    @_once
    def backward(ctx, dy, dh):
        h, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[:4]
        if dy is None and dh is None:
            return (None,) * 11
        if dy is None:               # only the stream went on: the norm's share is zero
            dy = torch.zeros(h.shape, dtype=ctx.dtype, device=h.device)
        # without dropout and with one type both branches of the sum get the same gradient: it is written once
        same = need[0] and need[1] and h.dtype == ctx.dtype and int(ctx.draws[0] * 65536.0 + 0.5) == 0
        dx, dres, dw, db = _residual_norm_backward(dy, dh, h, weight, mean, rstd, *ctx.draws, ctx.used,
                                                   need[0] and not same, *need[1:], ctx.code)
        return _pick(need, (dres if same else dx, dres, dw, db)) + (None,) * 7


# A leaf's gradient accumulator belongs to the stream it was made on.  One that an eager graph on the DEFAULT stream still
# holds cannot take part in a stream capture (the default stream cannot be captured: the capture would break inside the
# autograd engine, where the error ends the process), so such calls are refused while a graph is being captured.
_EAGER = "bilinear_hip_default_stream"


def _capturing():
    return torch._C._cuda_isCurrentStreamCapturing()


def _refuse_eager_leaves(tensors):
    for t in tensors:
        if t is not None and t.requires_grad and t.is_leaf:
            if torch.autograd.graph.get_gradient_edge(t).node.metadata.get(_EAGER):
                raise RuntimeError(
                    "bilinear_amd: a tensor that needs a gradient in this stream capture is still part of an eager autograd "
                    "graph recorded on the default stream.  Drop that graph (its outputs and losses) before the capture, or "
                    "run the eager steps on a side stream (torch.cuda.stream).")


def _apply(function, leaves, *args):
    if _capturing():
        _refuse_eager_leaves(leaves)
        return function.apply(*args)
    out = function.apply(*args)
    first = out[0] if type(out) is tuple else out
    if first.grad_fn is not None and not torch._C._cuda_getCurrentRawStream(first.get_device()):
        for node, _ in first.grad_fn.next_functions:
            if node is not None and hasattr(node, "variable"):
                node.metadata[_EAGER] = True
    return out


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- functions ------------------------------------------------------------------------------------------------------

def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis (biased variance); weight / bias: ``[width]``
    or None.  The result has x's type and shape."""
    if torch.compiler.is_compiling():
        return torch.ops.bilinear_hip.layer_norm(x, weight, bias, eps)[0]
    _check_rows(x, "x")
    _check_params(x, weight, bias)
    _check_eps(eps)
    if _wants_grad(x, weight, bias):
        return _apply(_LayerNormFunction, (x, weight, bias), x, weight, bias, eps)
    return _layer_norm(x, weight, bias, eps, save=False)[0]


def dropout(x, p, seed, step=0, layer=0, row_offset=0, device_step=None):
    """Drop elements of ``x`` with probability ``p`` (rounded to a multiple of 2^-16) and scale the others so that the
    expectation stays; what is dropped is zero whatever it held.  The mask depends on (seed, step, layer, global row,
    column) alone — ``row_offset`` is the global index of the first row, so a batch split over devices draws the mask of
    the whole one — and is drawn again in the backward pass instead of being stored.  ``device_step``: an int64 tensor
    that is added to ``step`` when the kernel runs: a captured graph that advances it draws another mask each replay."""
    if torch.compiler.is_compiling():
        return torch.ops.bilinear_hip.row_dropout(x, p, seed, step, layer, row_offset, device_step)[0]
    _check_rows(x, "x")
    _check_draws(p, seed, step, layer, row_offset, device_step, x)
    if _wants_grad(x):
        return _apply(_DropoutFunction, (x,), x, p, seed, step, layer, row_offset, device_step)
    return _row_dropout(x, p, seed, step, layer, row_offset, device_step)[0]


def residual_norm(x, residual, weight=None, bias=None, eps=1e-5, p=0.0, seed=0, step=0, layer=0, row_offset=0,
                  device_step=None):
    """``h = residual + dropout(x)`` and ``y = layer_norm(h)`` in one pass; returns ``(y, h)``: y in x's type, h — the
    residual stream, rounded to its type before it is normalised — in residual's (x's or float32).  The draws are those
    of ``dropout``; ``p=0`` draws none."""
    if torch.compiler.is_compiling():
        return torch.ops.bilinear_hip.residual_norm(x, residual, weight, bias, eps, p, seed, step, layer, row_offset,
                                                    device_step)[:2]
    _check_rows(x, "x")
    _check_like(residual, x, "residual", (x.dtype, torch.float32))
    _check_params(x, weight, bias)
    _check_eps(eps)
    _check_draws(p, seed, step, layer, row_offset, device_step, x)
    if _wants_grad(x, residual, weight, bias):
        return _apply(_ResidualNormFunction, (x, residual, weight, bias), x, residual, weight, bias, eps, p, seed, step,
                      layer, row_offset, device_step)
    return _residual_norm(x, residual, weight, bias, eps, p, seed, step, layer, row_offset, device_step, save=False)[:2]


# ---- modules --------------------------------------------------------------------------------------------------------

class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last axis on the native kernels: the same constructor, parameters and state_dict."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise RuntimeError("bilinear_amd.LayerNorm normalises the last axis only")

    def forward(self, x):
        if x.dim() < 1 or x.shape[-1] != self.normalized_shape[0]:
            raise RuntimeError("expected rows of %d columns, got shape %s" % (self.normalized_shape[0], tuple(x.shape)))
        return layer_norm(x, self.weight, self.bias, self.eps)


class _Draws:
    """The seed, the step count and the stream id of a module that drops.  As for a stand-alone stage the seed is torch's
    at the first call, the id is unique in the process (a copy gets its own) and the step counts calls; none is part of the
    state_dict.  In a captured graph a step counted on the host would be frozen: give the module an int64 device tensor
    (``set_device_step``) that the graph advances between replays."""

    _device_step = None

    def _init_draws(self):
        from .model.bilinear import _HeavyLinear
        self._layer = _HeavyLinear._next_stage_id[0]
        _HeavyLinear._next_stage_id[0] += 1
        self._seed, self._step, self._captured = None, 0, 0

    def __setstate__(self, state):
        super().__setstate__(state)
        step, seed = self._step, self._seed
        self._init_draws()
        self._step, self._seed, self._device_step = step, seed, None

    def set_device_step(self, tensor):
        if tensor is not None and (tensor.dtype != torch.int64 or tensor.numel() != 1):
            raise RuntimeError("the device step is one int64")
        self._device_step = tensor

    @torch.compiler.disable
    def _next_draws(self):
        if self._seed is None:
            self._seed = int(torch.initial_seed()) & (_LIMIT63 - 1)
        if torch.cuda.is_available() and _capturing():
            if self._device_step is None:
                raise RuntimeError("bilinear_amd: dropout in a stream capture needs a step on the device "
                                   "(set_device_step): every replay would draw the same mask")
            # calls of one captured step differ in the upper half of the step, replays in the device's count
            self._captured += 1
            return {"seed": self._seed, "step": self._captured << 32, "layer": self._layer, "device_step": self._device_step}
        self._step += 1
        return {"seed": self._seed, "step": self._step - 1, "layer": self._layer}


class Dropout(_Draws, nn.Dropout):
    """``nn.Dropout`` with the regenerated mask of ``dropout``."""

    def __init__(self, p=0.5, inplace=False):
        super().__init__(p, inplace)
        if inplace:
            raise RuntimeError("bilinear_amd.Dropout does not work in place")
        self._init_draws()

    def forward(self, x):
        if not self.training or self.p == 0.0:
            return x
        return dropout(x, self.p, **self._next_draws())


class ResidualNorm(_Draws, nn.LayerNorm):
    """``y, h = module(x, residual)``: ``h = residual + dropout(x, p)``, ``y = layer_norm(h)`` (``residual_norm``).
    Parameters and state_dict are those of ``nn.LayerNorm``; eval mode drops nothing."""

    def __init__(self, width, p=0.0, eps=1e-5, **kwargs):
        super().__init__(width, eps, **kwargs)
        if len(self.normalized_shape) != 1:
            raise RuntimeError("bilinear_amd.ResidualNorm normalises the last axis only")
        if not 0.0 <= p <= 1.0:
            raise ValueError("dropout probability has to be between 0 and 1, got %r" % (p,))
        self.p = p
        self._init_draws()

    def extra_repr(self):
        return super().extra_repr() + ", p=%s" % self.p

    def forward(self, x, residual):
        if x.dim() < 1 or x.shape[-1] != self.normalized_shape[0]:
            raise RuntimeError("expected rows of %d columns, got shape %s" % (self.normalized_shape[0], tuple(x.shape)))
        draws = self._next_draws() if self.training and self.p else {}
        return residual_norm(x, residual, self.weight, self.bias, self.eps, self.p if draws else 0.0, **draws)
