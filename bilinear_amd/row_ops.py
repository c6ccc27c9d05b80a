"""Operators on rows: ``layer_norm``, ``dropout`` with a mask that is never stored, and ``residual_norm``
(``h = residual + dropout(x)``, ``y = layer_norm(h)``), forward and backward, on libbilinear_hip.so's
``blh_layer_norm_*``, ``blh_row_dropout`` and ``blh_residual_norm_*``.

They are the counterparts of a stage's BatchNorm1d and Dropout(0.5) (/root/reference/model/bilinear.py:7-13) that need no
batch and no stored mask.  Three surfaces, as for the lifter:

    y = bilinear_amd.layer_norm(x, weight, bias)                      # functions, differentiable
    y = bilinear_amd.dropout(x, 0.1, seed=7, step=3, layer=0)
    y, h = bilinear_amd.residual_norm(x, h, weight, bias, p=0.1, seed=7, step=3, layer=1)
    bilinear_amd.LayerNorm(1024), .Dropout(0.1), .ResidualNorm(1024, p=0.1)     # modules
    torch.ops.bilinear_hip.{layer_norm, row_dropout, residual_norm, ...}        # custom operators (torch.compile, tracers)

The functions go to the library directly.  Under a tracer (torch.jit.trace, make_fx), a dispatch mode, or with tensor
subclasses, they call the custom operators, which these can see.

Second derivatives: those of dropout; a backward pass through the norms' gradients is refused.

The last axis is the row.  Types: x float32 / bfloat16 / float16; weight and bias float32 or x's type; the residual
stream (``residual``, ``h``) float32 or x's type.  Rows of a wider tensor (last axis dense) are read in place.  Tensors
must live on a HIP device: there is no CPU path.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import torch
import torch.nn as nn

from . import _native as N
from .ops import _LIB

__all__ = ["layer_norm", "dropout", "residual_norm", "LayerNorm", "Dropout", "ResidualNorm"]

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # blh_dtype
_BINDING = os.path.join(os.path.dirname(N.LIB_PATH), "_rows.so")
_rows = None


def _native():
    """The PyTorch side of the operators (csrc/torch_rows.cpp: argument checks, allocation, autograd nodes), loaded once.
    There is no other implementation: a missing library raises."""
    global _rows
    if _rows is None:
        N.lib()                       # libbilinear_hip.so against the HIP runtime torch has loaded
        if not os.path.exists(_BINDING):
            raise RuntimeError("bilinear_amd: %s not found. Build it with `python -c 'import __graft_entry__ as g; "
                               "g.build()'` or `make -C bilinear_amd/csrc`. There is no fallback path." % _BINDING)
        loader = importlib.machinery.ExtensionFileLoader("_rows", _BINDING)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_rows", loader))
        loader.exec_module(module)
        _rows = module
    return _rows


def _param_code(x, weight, bias):
    t = weight if weight is not None else bias
    return 0 if t is None else _CODES[t.dtype]


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


for _name in ("layer_norm", "layer_norm_backward", "row_dropout", "residual_norm", "residual_norm_backward"):
    _LIB.impl(_name, lambda *args, _name="op_" + _name: getattr(_native(), _name)(*args), "CUDA")


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


def _capturing(x):
    """Whether the current stream of x's device, where the kernels go, is being captured."""
    if not torch.cuda.is_available():
        return False
    if x is None or x.device.index is None or x.device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(x.device):
        return torch.cuda.is_current_stream_capturing()


def _refuse_eager_leaves(inputs):
    """In a stream capture: what the functions refuse (csrc/torch_rows.cpp), for calls of the operators themselves."""
    if not torch.compiler.is_compiling() and _capturing(inputs[0]):
        _native().refuse_eager_leaves([t for t in inputs if isinstance(t, torch.Tensor)])


def _ln_setup(ctx, inputs, output):
    _refuse_eager_leaves(inputs)
    x, weight, bias, _ = inputs
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.code = _param_code(x, weight, bias)


def _ln_formula(ctx, dy, dmean, drstd):
    x, weight, mean, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad[:3]
    return _pick(need, torch.ops.bilinear_hip.layer_norm_backward(dy, x, weight, mean, rstd, *need, ctx.code)) + (None,)


def _drop_setup(ctx, inputs, output):
    _refuse_eager_leaves(inputs)
    _, p, seed, step, layer, row_offset, device_step = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(*(() if device_step is None else (output[1],)))
    ctx.draws = (p, seed, step if device_step is None else 0, layer, row_offset)


def _drop_formula(ctx, dy, dused):
    used = ctx.saved_tensors[0] if ctx.saved_tensors else None
    return (torch.ops.bilinear_hip.row_dropout(dy, *ctx.draws, used)[0],) + (None,) * 6


def _res_setup(ctx, inputs, output):
    _refuse_eager_leaves(inputs)
    x, residual, weight, bias, _, p, seed, step, layer, row_offset, device_step = inputs
    ctx.mark_non_differentiable(*output[2:])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(output[1], weight, output[2], output[3], None if device_step is None else output[4])
    ctx.draws = (p, seed, step if device_step is None else 0, layer, row_offset)
    ctx.code, ctx.dtype = _param_code(x, weight, bias), x.dtype


def _res_formula(ctx, dy, dh, *unused):
    h, weight, mean, rstd, used = ctx.saved_tensors
    need = ctx.needs_input_grad[:4]
    if dy is None:
        if dh is None:
            return (None,) * 11
        # only the stream went on: the sum's gradients, whatever the rows' statistics are
        dx = torch.ops.bilinear_hip.row_dropout(dh, *ctx.draws, used)[0] if int(ctx.draws[0] * 65536 + 0.5) else dh
        zeros = dh.new_zeros(dh.shape[-1], dtype=torch.float32 if ctx.code == 0 else ctx.dtype)
        return _pick(need, (dx.to(ctx.dtype), dh, zeros, zeros.clone())) + (None,) * 7
    return _pick(need, torch.ops.bilinear_hip.residual_norm_backward(
        dy, dh, h, weight, mean, rstd, *ctx.draws, used, *need, ctx.code)) + (None,) * 7


torch.library.register_autograd("bilinear_hip::layer_norm", _ln_formula, setup_context=_ln_setup, lib=_LIB)
torch.library.register_autograd("bilinear_hip::row_dropout", _drop_formula, setup_context=_drop_setup, lib=_LIB)
torch.library.register_autograd("bilinear_hip::residual_norm", _res_formula, setup_context=_res_setup, lib=_LIB)


# ---- functions ------------------------------------------------------------------------------------------------------

def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis (biased variance); weight / bias: ``[width]``
    or None.  The result has x's type and shape."""
    if torch.compiler.is_compiling():
        return torch.ops.bilinear_hip.layer_norm(x, weight, bias, eps)[0]
    return (_rows or _native()).layer_norm(x, weight, bias, eps)


def dropout(x, p, seed, step=0, layer=0, row_offset=0, device_step=None):
    """Drop elements of ``x`` with probability ``p`` (rounded to a multiple of 2^-16) and scale the others so that the
    expectation stays; what is dropped is zero whatever it held.  The mask depends on (seed, step, layer, global row,
    column) alone — ``row_offset`` is the global index of the first row, so a batch split over devices draws the mask of
    the whole one — and is drawn again in the backward pass instead of being stored.  One word of the generator's key is
    ``seed ^ (step >> 32)``: let steps that count stay below 2^32 where several seeds are in use.  ``device_step``: an
    int64 tensor that is added to ``step`` when the kernel runs: a captured graph that advances it draws another mask each
    replay."""
    if torch.compiler.is_compiling():
        return torch.ops.bilinear_hip.row_dropout(x, p, seed, step, layer, row_offset, device_step)[0]
    return (_rows or _native()).dropout(x, p, seed, step, layer, row_offset, device_step)


def residual_norm(x, residual, weight=None, bias=None, eps=1e-5, p=0.0, seed=0, step=0, layer=0, row_offset=0,
                  device_step=None):
    """``h = residual + dropout(x)`` and ``y = layer_norm(h)`` in one pass; returns ``(y, h)``: y in x's type, h — the
    residual stream, rounded to its type before it is normalised — in residual's (x's or float32).  The draws are those
    of ``dropout``; ``p=0`` draws none."""
    if torch.compiler.is_compiling():
        return torch.ops.bilinear_hip.residual_norm(x, residual, weight, bias, eps, p, seed, step, layer, row_offset,
                                                    device_step)[:2]
    return (_rows or _native()).residual_norm(x, residual, weight, bias, eps, p, seed, step, layer, row_offset, device_step)


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
    """The draws of a module that drops: torch's seed at the first call, a stream id that is unique in the process (a copy
    gets its own, as every stand-alone stage does) and, as the step, a number from torch's CPU generator — so
    ``torch.manual_seed`` repeats the masks, a saved generator state continues them and a checkpointed block (which
    restores that state) is recomputed with the mask it had, in a captured graph as well.  There the number is frozen: give
    the module an int64 device tensor (``set_device_step``), which is added to it and which the graph advances between
    replays.  ``row_offset``: the global index of this process's first row, so that ranks with one seed draw the parts of
    one mask."""

    _device_step = None
    row_offset = 0

    def _init_draws(self):
        from .model.bilinear import _HeavyLinear
        self._layer = _HeavyLinear._next_stage_id[0]
        _HeavyLinear._next_stage_id[0] += 1
        self._seed = None

    def __setstate__(self, state):
        super().__setstate__(state)
        seed = self._seed
        self._init_draws()
        self._seed, self._device_step = seed, None

    def set_device_step(self, tensor):
        if tensor is not None and (tensor.dtype != torch.int64 or tensor.numel() != 1):
            raise RuntimeError("the device step is one int64")
        self._device_step = tensor

    def _next_draws(self, x=None):
        if self._seed is None:
            self._seed = int(torch.initial_seed()) & ((1 << 63) - 1)
        if torch.jit.is_tracing():
            raise RuntimeError("bilinear_amd: dropout in a trace: every call would draw the same mask.  Trace the module in "
                               "eval mode, or the function `dropout` with a device_step")
        step, device_step = int(torch.empty((), dtype=torch.int64).random_()), None
        if _capturing(x):
            device_step = self._device_step
            if device_step is None:
                raise RuntimeError("bilinear_amd: dropout in a stream capture needs a step on the device "
                                   "(set_device_step): every replay would draw the same mask")
        return {"seed": self._seed, "step": step, "layer": self._layer, "row_offset": self.row_offset,
                "device_step": device_step}


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
        return dropout(x, self.p, **self._next_draws(x))


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
        draws = self._next_draws(x) if self.training and self.p else {}
        return residual_norm(x, residual, self.weight, self.bias, self.eps, self.p if draws else 0.0, **draws)
