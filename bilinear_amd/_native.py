"""ctypes binding of libbilinear_hip.so (the C ABI declared in include/bilinear_hip.h).

This is the stub a maintainer of the reference would add to
``model/bilinear.py`` to route ``BilinearUnit`` through the MI355X kernels (see
INTEGRATION.md).  There is NO fallback: if the library is missing or a call
fails, a ``RuntimeError`` is raised — results never silently come from another
code path.
"""
from __future__ import annotations

import ctypes
import os
from ctypes import (POINTER, Structure, c_char_p, c_double, c_float, c_int, c_int32, c_int64,
                    c_uint64, c_void_p)

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libbilinear_hip.so")

OK = 0


class ModelDesc(Structure):
    _fields_ = [("num_blocks", c_int32), ("width", c_int32),
                ("in_features", c_int32), ("out_features", c_int32), ("gemm_dtype", c_int32)]


class Dropout(Structure):
    _fields_ = [("keep_mask", c_void_p), ("seed", c_uint64), ("step", c_uint64),
                ("row_offset", c_int64), ("layer_base", c_int32), ("reserved", c_int32)]


class AdamHyper(Structure):
    _fields_ = [("lr", c_double), ("beta1", c_double), ("beta2", c_double), ("eps", c_double),
                ("max_norm", c_double), ("step", c_int32), ("reserved", c_int32)]


class StepState(Structure):
    _fields_ = [("lr", c_double), ("beta1", c_double), ("beta2", c_double), ("eps", c_double),
                ("max_norm", c_double), ("rng_step", c_uint64), ("step", c_int32), ("reserved", c_int32),
                ("step_size", c_float), ("bc2_sqrt", c_float)]


class RowDrop(Structure):
    _fields_ = [("p", c_double), ("seed", c_uint64), ("step", c_uint64), ("row_offset", c_int64),
                ("step_dev", c_void_p), ("step_used", c_void_p), ("layer", c_int32), ("reserved", c_int32)]


GradReadyFn = ctypes.CFUNCTYPE(None, c_void_p, c_int64, c_int64)
SyncFn = ctypes.CFUNCTYPE(None, c_void_p, c_void_p, c_int64, c_int32)

# name -> (restype, argtypes); mirrors include/bilinear_hip.h one to one
_SIGNATURES = {
    "blh_status_string": (c_char_p, [c_int]),
    "blh_last_hip_error": (c_int, []),
    "blh_abi_version": (c_int, []),
    "blh_context_create": (c_int, [POINTER(c_void_p)]),
    "blh_context_destroy": (c_int, [c_void_p]),
    "blh_context_set_option": (c_int, [c_void_p, c_int32, c_int32]),
    "blh_context_get_option": (c_int, [c_void_p, c_int32]),
    "blh_context_side_stream": (c_void_p, [c_void_p]),
    "blh_num_heavy": (c_int32, [POINTER(ModelDesc)]),
    "blh_param_arena_floats": (c_int64, [POINTER(ModelDesc)]),
    "blh_num_param_tensors": (c_int32, [POINTER(ModelDesc)]),
    "blh_param_tensor_info": (c_int, [POINTER(ModelDesc), c_int32, c_char_p, c_int32,
                                      POINTER(c_int64), POINTER(c_int64), POINTER(c_int64)]),
    "blh_bn_running_floats": (c_int64, [POINTER(ModelDesc)]),
    "blh_workspace_bytes": (c_int64, [POINTER(ModelDesc), c_int64]),
    "blh_forward_train": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, c_void_p,
                                  c_void_p, POINTER(Dropout), c_float, c_void_p, c_int64,
                                  c_void_p, c_int64]),
    "blh_clip_adam_step_bf16": (c_int, [c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_void_p, c_void_p,
                                        c_int64, POINTER(AdamHyper), c_void_p, c_int64, c_void_p]),
    "blh_refresh_param_shadow": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, c_int64,
                                         c_int64]),
    "blh_forward_train_loss": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, c_void_p,
                                       c_void_p, c_void_p, POINTER(Dropout), c_float, c_void_p, c_int64,
                                       c_void_p, c_void_p, c_int64]),
    "blh_forward_train_loss_sync": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p,
                                            c_void_p, c_void_p, c_void_p, POINTER(Dropout), c_float,
                                            c_void_p, c_int64, c_void_p, c_void_p, c_int64, c_int64,
                                            SyncFn, c_void_p]),
    "blh_forward_eval": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, c_void_p,
                                 c_void_p, c_int64, c_void_p, c_int64]),
    "blh_mse_loss_grad": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_double,
                                  c_float, c_void_p, c_void_p, c_void_p, c_int64]),
    "blh_backward": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, POINTER(Dropout),
                             c_void_p, c_int64, c_void_p, c_void_p, c_int64, GradReadyFn,
                             c_void_p]),
    "blh_forward_train_sync": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, c_void_p,
                                       c_void_p, POINTER(Dropout), c_float, c_void_p, c_int64,
                                       c_void_p, c_int64, c_int64, SyncFn, c_void_p]),
    "blh_backward_sync": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p,
                                  POINTER(Dropout), c_void_p, c_int64, c_void_p, c_void_p, c_int64,
                                  GradReadyFn, c_void_p, c_int64, SyncFn, c_void_p]),
    "blh_clip_grad_norm": (c_int, [c_void_p, c_void_p, c_int64, c_float, c_void_p, c_int64,
                                   c_void_p]),
    "blh_clip_adam_step": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64,
                                   POINTER(AdamHyper), c_void_p, c_int64, c_void_p]),
    "blh_train_step": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, c_void_p,
                               c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                               POINTER(Dropout), c_float, POINTER(AdamHyper), c_void_p, c_int64,
                               c_void_p, c_void_p, c_void_p, c_int64]),
    "blh_heavy_workspace_bytes": (c_int64, [c_int64, c_int32, c_int32]),
    "blh_heavy_forward": (c_int, [c_void_p] * 10 + [POINTER(Dropout), c_float, c_int32, c_int32,
                                                   c_void_p, c_int64, c_void_p, c_int64, c_int32,
                                                   c_int32]),
    "blh_heavy_backward": (c_int, [c_void_p] * 6 + [POINTER(Dropout), c_int32, c_void_p, c_int64,
                                                    c_void_p, c_void_p, c_void_p, c_void_p,
                                                    c_void_p, c_int64, c_int32, c_int32]),
    "blh_mpjpe": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int32,
                          c_void_p, c_void_p, c_int32, c_void_p, c_void_p]),
    "blh_step_state_advance": (c_int, [c_void_p, c_void_p]),
    "blh_context_set_step_state": (c_int, [c_void_p, c_void_p]),
    "blh_clip_adam_step_captured": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64,
                                            c_void_p, c_void_p, c_int64, c_void_p]),
    "blh_gemm_bf16s_tile": (c_int32, [c_int64, c_int64, c_int64, c_int32, c_int32, c_int32, c_int32]),
    "blh_gemm_bf16s_force_tile": (c_int, [c_int32]),
    "blh_side_stream_renew": (c_int, []),
    "blh_side_stream_generation": (c_int32, []),
    "blh_tune_streams": (c_int, [c_void_p, c_int32, POINTER(c_float)]),
    "blh_wgrad_plan_bf16s": (c_int, [c_int64, c_int64, c_int32, POINTER(c_int32), POINTER(c_int32)]),
    "blh_gemm_bf16s_tile_cols": (c_int32, [c_int64, c_int64, c_int64, c_int32, c_int32, c_int32, c_int32]),
    "blh_train_step_captured": (c_int, [c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, c_void_p,
                                        c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                        POINTER(Dropout), c_float, c_void_p, c_void_p, c_int64,
                                        c_void_p, c_void_p, c_void_p, c_int64]),
    "blh_gemm_f32": (c_int, [c_void_p, c_void_p, c_int64, c_int32, c_void_p, c_int64, c_int32,
                             c_void_p, c_int64, c_int64, c_int64, c_int64, c_int32, c_void_p,
                             c_void_p, c_int64]),
    "blh_gemm_bf16x3": (c_int, [c_void_p, c_void_p, c_int64, c_int32, c_void_p, c_int64, c_int32,
                                c_void_p, c_int64, c_int64, c_int64, c_int64, c_int32, c_void_p,
                                c_void_p, c_int64]),
    "blh_gemm_fp16x2_workspace_bytes": (c_int64, []),
    "blh_gemm_fp16x2": (c_int, [c_void_p, c_void_p, c_int64, c_int32, c_void_p, c_int64, c_int32,
                                c_void_p, c_int64, c_int64, c_int64, c_int64, c_int32, c_void_p,
                                c_void_p, c_int64, c_void_p, c_int32]),
    "blh_sum_slabs": (c_int, [c_void_p, c_void_p, c_int64, c_int32, c_void_p]),
    "blh_skinny_workspace_bytes": (c_int64, [c_int64, c_int32, c_int32, c_int32]),
    "blh_skinny_encode_fwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                      POINTER(c_int32), c_int64, c_int32, c_int32]),
    "blh_skinny_decode_fwd_mse": (c_int, [c_void_p] * 9 + [c_int64, c_int64, c_int32, c_int32]),
    "blh_skinny_decode_fused": (c_int, [c_void_p] * 10 + [c_int64, c_int64, c_int32, c_int32]),
    "blh_skinny_decode_fused_bf16_workspace_bytes": (c_int64, [c_int64, c_int32, c_int32]),
    "blh_skinny_decode_fused_bf16": (c_int, [c_void_p] * 10 + [c_int64, c_int64, c_int32, c_int32]),
    "blh_skinny_encode_fused_fwd": (c_int, [c_void_p] * 9 + [c_float] + [c_void_p] * 5 + [c_int64, c_int32, c_int32]),
    "blh_skinny_encode_fused_bwd": (c_int, [c_void_p] * 12 + [c_int64, c_int32, c_int32]),
    "blh_skinny_encode_fused_fwd_bf16": (c_int, [c_void_p] * 9 + [c_float] + [c_void_p] * 5 + [c_int64, c_int32, c_int32]),
    "blh_skinny_encode_fused_bwd_bf16": (c_int, [c_void_p] * 12 + [c_int64, c_int32, c_int32]),
    "blh_skinny_decode_bwd": (c_int, [c_void_p] * 7 + [c_int64, c_int64, c_int32, c_int32]),
    "blh_skinny_encode_wgrad": (c_int, [c_void_p] * 5 + [c_int64, c_int64, c_int32, c_int32]),
    "blh_gemm_bf16s": (c_int, [c_void_p, c_void_p, c_int64, c_int32, c_void_p, c_int64, c_int32,
                               c_void_p, c_int64, c_int32, c_int64, c_int64, c_int64, c_int32,
                               c_void_p, c_void_p, c_int64, c_void_p]),
    "blh_gemm_bf16s_batched": (c_int, [c_void_p, c_void_p, c_int64, c_int32, c_int64, c_void_p, c_int64, c_int32,
                                       c_int64, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int64, c_int32,
                                       c_int32]),
    "blh_cast_f32_to_bf16": (c_int, [c_void_p, c_void_p, c_void_p, c_int64]),
    "blh_cast_bf16_to_f32": (c_int, [c_void_p, c_void_p, c_void_p, c_int64]),
    "blh_linear_fwd_stats": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                     c_int64, c_int64, c_int64]),
    "blh_dropout_mask": (c_int, [c_void_p, POINTER(Dropout), c_int32, c_int64, c_int32, c_void_p]),
    # operators on rows (csrc/row_norm.hip, row_dropout.hip)
    "blh_row_dropout": (c_int, [c_void_p, c_void_p, c_int64, c_void_p, POINTER(RowDrop), c_int64, c_int64, c_int32]),
    "blh_layer_norm_forward": (c_int, [c_void_p, c_void_p, c_int64, c_void_p, c_void_p, c_double, c_void_p, c_void_p,
                                       c_void_p, c_int64, c_int64, c_int32, c_int32]),
    "blh_row_norm_workspace_bytes": (c_int64, [c_int64, c_int64]),
    "blh_layer_norm_backward": (c_int, [c_void_p, c_void_p, c_int64, c_void_p, c_int64] + [c_void_p] * 7
                                + [c_int64, c_int64, c_int64, c_int32, c_int32]),
    "blh_residual_norm_forward": (c_int, [c_void_p, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_void_p, c_double,
                                          POINTER(RowDrop), c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                                          c_int32, c_int32, c_int32]),
    "blh_residual_norm_backward": (c_int, [c_void_p, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_void_p,
                                           c_void_p, c_void_p, POINTER(RowDrop)] + [c_void_p] * 5
                                   + [c_int64, c_int64, c_int64, c_int32, c_int32, c_int32]),
    # collectives issued by the library (opt-in data-parallel path, csrc/comm.hip)
    "blh_rccl_version": (c_int, []),
    "blh_rccl_unique_id": (c_int, [c_void_p, c_int64]),
    "blh_comm_create": (c_int, [POINTER(c_void_p), c_void_p, c_int64, c_int32, c_int32]),
    "blh_comm_destroy": (c_int, [c_void_p]),
    "blh_comm_info": (c_int, [c_void_p, POINTER(c_int32), POINTER(c_int32), POINTER(c_int32), POINTER(c_int64)]),
    "blh_comm_stream": (c_void_p, [c_void_p]),
    "blh_comm_set_bf16_buffer": (c_int, [c_void_p, c_void_p, c_int64]),
    "blh_comm_all_reduce": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int32, c_int32]),
    "blh_comm_broadcast": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int32]),
    "blh_comm_last_error": (c_char_p, []),
    "blh_train_step_dp": (c_int, [c_void_p, c_void_p, POINTER(ModelDesc), c_void_p, c_void_p, c_void_p, c_void_p,
                                  c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, POINTER(Dropout), c_float,
                                  POINTER(AdamHyper), c_void_p, c_void_p, c_int64, c_void_p, c_void_p, c_void_p,
                                  c_int64, c_int64, SyncFn, c_void_p, c_int32]),
}

_lib = None


def lib():
    """Load (once) and return the library.  torch is imported first so that the
    library's ``libamdhip64.so.7`` dependency resolves to the HIP runtime already
    loaded by PyTorch (same soname): streams and device pointers are then shared."""
    global _lib
    if _lib is not None:
        return _lib
    import torch  # noqa: F401  (loads torch's HIP runtime before ours is resolved)
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            "bilinear_amd: native library %s not found. Build it with "
            "`python -c 'import __graft_entry__ as g; g.build()'` or "
            "`make -C bilinear_amd/csrc`. There is no fallback path." % LIB_PATH)
    try:
        handle = ctypes.CDLL(LIB_PATH, mode=ctypes.RTLD_LOCAL)
    except OSError as exc:
        raise RuntimeError("bilinear_amd: cannot load %s: %s" % (LIB_PATH, exc)) from exc
    for name, (restype, argtypes) in _SIGNATURES.items():
        try:
            fn = getattr(handle, name)
        except AttributeError as exc:
            raise RuntimeError("bilinear_amd: %s does not export %s" % (LIB_PATH, name)) from exc
        fn.restype = restype
        fn.argtypes = argtypes
    _lib = handle
    return _lib


OPT_TWO_STREAM = 0
OPT_LATE_FORK = 2
OPT_PERSISTENT_SHADOW = 3
OPT_SMALL_STEP = 4
OPT_BUCKET_FLOATS = 6     # blh_backward merges ready ranges into buckets of at least this many elements
OPT_DEV_KNOBS = 5         # bit mask of developer A/B switches (csrc/step.h: blh::KNOB_*), latched from BLH_* at context creation


class Context:
    """Owner of one ``blh_context`` (include/bilinear_hip.h): the library's side stream, events
    and option flags on ONE device.  Created with that device current; destroyed with the object."""

    def __init__(self, device):
        import torch
        self.device = torch.device(device)
        handle = c_void_p()
        with torch.cuda.device(self.device):
            check(lib().blh_context_create(ctypes.byref(handle)), "blh_context_create")
        self.handle = handle

    def set_option(self, option, value):
        check(lib().blh_context_set_option(self.handle, int(option), int(value)), "blh_context_set_option")

    def get_option(self, option):
        return int(lib().blh_context_get_option(self.handle, int(option)))

    def side_stream(self):
        return lib().blh_context_side_stream(self.handle)

    def __del__(self):
        try:
            if self.handle and _lib is not None:
                _lib.blh_context_destroy(self.handle)
                self.handle = None
        except Exception:   # noqa: BLE001  (interpreter shutdown)
            pass


DP_TAIL_ON_COMM_STREAM = 1     # blh_train_step_dp flags (include/bilinear_hip.h)
DP_BF16_BUCKETS = 2
UNIQUE_ID_BYTES = 128


class Comm:
    """Owner of one ``blh_comm`` (include/bilinear_hip.h): an RCCL communicator the LIBRARY drives, with its own
    collective stream, on the current device.  ``unique_id``: the 128 bytes rank 0 got from ``rccl_unique_id()``.
    Creating it is a collective call (every rank of the communicator)."""

    def __init__(self, device, unique_id, world, rank):
        import torch
        self.device = torch.device(device)
        if len(unique_id) != UNIQUE_ID_BYTES:
            raise ValueError("an RCCL unique id has %d bytes" % UNIQUE_ID_BYTES)
        handle = c_void_p()
        buf = ctypes.create_string_buffer(bytes(unique_id), UNIQUE_ID_BYTES)
        with torch.cuda.device(self.device):
            check(lib().blh_comm_create(ctypes.byref(handle), buf, UNIQUE_ID_BYTES, int(world), int(rank)),
                  "blh_comm_create")
        self.handle = handle
        self.world, self.rank = int(world), int(rank)

    def info(self):
        w, r, v, n = c_int32(), c_int32(), c_int32(), c_int64()
        check(lib().blh_comm_info(self.handle, ctypes.byref(w), ctypes.byref(r), ctypes.byref(v), ctypes.byref(n)),
              "blh_comm_info")
        return {"world": w.value, "rank": r.value, "rccl_version": v.value, "collectives_issued": n.value}

    def all_reduce(self, tensor, average=False):
        """In place, on torch's current stream."""
        import torch
        dt = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2}[tensor.dtype]
        if not tensor.is_contiguous():
            raise RuntimeError("all_reduce needs a contiguous tensor")
        check(lib().blh_comm_all_reduce(self.handle, current_stream(), ptr(tensor), tensor.numel(), dt,
                                        1 if average else 0), "blh_comm_all_reduce")

    def broadcast(self, tensor, root=0):
        if not tensor.is_contiguous():
            raise RuntimeError("broadcast needs a contiguous tensor")
        check(lib().blh_comm_broadcast(self.handle, current_stream(), ptr(tensor),
                                       tensor.numel() * tensor.element_size(), int(root)), "blh_comm_broadcast")

    def destroy(self):
        if self.handle and _lib is not None:
            h, self.handle = self.handle, None
            check(_lib.blh_comm_destroy(h), "blh_comm_destroy")

    def __del__(self):
        try:
            if self.handle and _lib is not None:
                _lib.blh_comm_destroy(self.handle)
                self.handle = None
        except Exception:   # noqa: BLE001  (interpreter shutdown)
            pass


def rccl_unique_id():
    buf = ctypes.create_string_buffer(UNIQUE_ID_BYTES)
    check(lib().blh_rccl_unique_id(buf, UNIQUE_ID_BYTES), "blh_rccl_unique_id")
    return bytes(buf.raw)


_contexts = {}


def default_context(device):
    """One shared context per device for callers that own no engine (stand-alone stages)."""
    import torch
    dev = torch.device(device)
    key = (dev.type, dev.index if dev.index is not None else torch.cuda.current_device())
    if key not in _contexts:
        _contexts[key] = Context(torch.device("cuda", key[1]))
    return _contexts[key]


def exported_names():
    return sorted(_SIGNATURES)


def check(status, what):
    """Raise RuntimeError for a non-OK blh_status (the reference relies on
    PyTorch raising RuntimeError on shape/device errors; so do we)."""
    if status != OK:
        l = lib()
        msg = l.blh_status_string(int(status)).decode()
        if status == -3:
            msg += " (hipError_t %d)" % l.blh_last_hip_error()
        if status == -5:
            msg += ": " + l.blh_comm_last_error().decode()
        raise RuntimeError("bilinear_amd: %s failed: %s" % (what, msg))


def current_stream():
    """hipStream_t of torch's current stream on the current device, as a c_void_p.  Through the raw accessor
    (no torch.cuda.Stream object, no device-index parsing: ~1 us instead of ~5 us per call — the drop-in step at
    the reference's batch of 64 is host-bound and asks three times per step)."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is None:
        return c_void_p(torch.cuda.current_stream().cuda_stream)
    return c_void_p(raw(torch._C._cuda_getDevice()))


def ptr(t):
    """Device pointer of a torch tensor (None -> NULL)."""
    return None if t is None else c_void_p(t.data_ptr())
