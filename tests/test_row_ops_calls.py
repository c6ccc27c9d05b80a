"""Row operators without a GPU under the calls around them: tracers, shape propagation, the modules' draws."""
import os
import subprocess
import sys
import types

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import bilinear_amd as B


def _shapes(*tensors):
    return [(tuple(t.shape), t.dtype, t.device.type) for t in tensors]


def test_functions_propagate_shapes_under_a_fake_mode():
    with FakeTensorMode():
        x, r = torch.empty(3, 5, 48, dtype=torch.bfloat16, device="cuda"), torch.empty(3, 5, 48, device="cuda")
        w = torch.empty(48, device="cuda")
        step = torch.zeros(1, dtype=torch.int64, device="cuda")
        assert _shapes(B.layer_norm(x, w, w)) == _shapes(x)
        assert _shapes(B.dropout(x, 0.3, seed=1, device_step=step)) == _shapes(x)
        assert _shapes(*B.residual_norm(x, r, w, None, p=0.3, seed=1)) == _shapes(x, r)
        with pytest.raises(RuntimeError, match="weight has shape"):         # the checks come first
            B.layer_norm(x, torch.empty(47, device="cuda"))
    assert _shapes(B.layer_norm(x, w, w)) == _shapes(x)                     # fake tensors outside their mode


@pytest.mark.parametrize("name,call", [
    ("layer_norm", lambda x: B.layer_norm(x)),
    ("row_dropout", lambda x: B.dropout(x, 0.3, seed=1)),
    ("residual_norm", lambda x: B.residual_norm(x, x, p=0.3, seed=1))])
def test_make_fx_records_the_custom_operators(name, call):
    with FakeTensorMode():
        x = torch.empty(2, 8, device="cuda")
        graph = make_fx(call)(x)
    targets = [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]
    assert "bilinear_hip.%s.default" % name in targets and not any("empty" in t for t in targets)


def test_a_module_that_drops_is_not_traced_with_one_mask():
    with pytest.raises(RuntimeError, match="every call would draw the same mask"):
        torch.jit.trace(B.Dropout(0.3), torch.ones(3))
    with pytest.raises(RuntimeError, match="every call would draw the same mask"):
        torch.jit.trace(B.ResidualNorm(3, p=0.3), (torch.ones(3), torch.ones(3)))
    torch.jit.trace(B.Dropout(0.3).eval(), torch.ones(3))


def test_a_restored_generator_repeats_the_draws_in_a_capture(monkeypatch):
    """(A checkpointed block, called again in the capture of its backward pass, restores the CPU generator's state.)"""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    for m in (B.Dropout(0.1), B.ResidualNorm(8, p=0.1)):
        m.set_device_step(torch.zeros(1, dtype=torch.int64))
        state = torch.get_rng_state()
        first, second = m._next_draws(), m._next_draws()
        torch.set_rng_state(state)
        again = m._next_draws()
        assert again["device_step"] is first["device_step"] is m._device_step
        assert again["step"] == first["step"] and second["step"] != first["step"]


def test_seeds_that_differ_do_not_share_masks_in_a_capture(monkeypatch):
    """The generator's key holds seed ^ (step >> 32) in one word: steps that counted calls in those bits gave modules of two seeds
    (ranks that seed by their index) one another's masks."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    keys = set()
    for seed in range(8):
        torch.manual_seed(seed)
        m = B.Dropout(0.1)
        m.set_device_step(torch.zeros(1, dtype=torch.int64))
        for _ in range(8):
            d = m._next_draws()
            keys.add(((d["seed"] & 0xFFFFFFFF) ^ (d["step"] >> 32), d["seed"] >> 32))
    assert len(keys) == 64


def test_the_capture_that_counts_is_that_of_the_inputs_device(monkeypatch):
    """(Stands in for two devices: the stream of device 1 is captured, device 0 is the current one.)"""
    current = [0]

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == 1)
    m = B.Dropout(0.1)
    m.set_device_step(torch.zeros(1, dtype=torch.int64))
    there, here = (types.SimpleNamespace(device=torch.device("cuda", i)) for i in (1, 0))
    assert m._next_draws(there)["device_step"] is m._device_step and m._next_draws(here)["device_step"] is None
    assert current == [0]


def test_the_c_library_builds_without_pytorch():
    csrc = os.path.join(os.path.dirname(B.__file__), "csrc")

    def commands(*args):
        return subprocess.run(["make", "-n", "-B", "-C", csrc, "all", *args], capture_output=True, text=True, check=True).stdout
    with_torch, without = commands("PYTHON=" + sys.executable), commands("PYTHON=false")
    assert "libbilinear_hip.so" in without and "torch_rows" not in without and "torch_rows" in with_torch
