"""Cases that measure bilinear_amd's row operators: ``layer_norm``, ``dropout`` and ``residual_norm``.

``own = False``: the operators in plain form, elementary torch operations in 32 bits (the Philox draws in 64-bit
integers, the sum of the residual stream in 64 bits because it is rounded to the stream's type).  ``own = True``: the
framework's calls.  All inputs come from ``prepare``; ``exact`` is the definition in 64 bits, written apart.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
LARGEST = 16384 * 2048      # elements of the largest listed case


def _case(name, op, mode, rows, width, dtype, params="fp32", stream=None, p=0.0, pad=0):
    """op: layer_norm | dropout | residual_norm; mode: infer (forward alone) | train (forward and backward);
    dtype: of x and y; params: of weight and bias; stream: of the residual stream; pad: columns between the rows' ends
    (the input is a slice of a wider tensor)."""
    c = {"op": op, "mode": mode, "rows": rows, "width": width, "dtype": dtype, "params": params,
         "stream": stream or dtype, "p": p, "pad": pad}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one pose in eval mode: a single row of the hidden width, where latency is all there is
        _case("norm, one row", "layer_norm", "infer", 1, 1024, "fp32"),
        # an evaluation batch of the bf16-storage network
        _case("norm, eval batch", "layer_norm", "infer", 16384, 1024, "bf16"),
        # the batch of 64 that the training scripts default to
        _case("norm, batch of 64", "layer_norm", "train", 64, 1024, "fp32"),
        # the headline benchmark's batch and width
        _case("norm, 4096 rows", "layer_norm", "train", 4096, 1024, "fp32"),
        # the largest benchmark shape per GPU: bf16 storage, fp32 master weights
        _case("norm, 16384 rows of 2048", "layer_norm", "train", 16384, 2048, "bf16"),
        # a loader's last batch, an odd width, and rows that are a slice of a wider tensor
        _case("norm, odd and strided", "layer_norm", "train", 1237, 1001, "fp16", params="fp16", pad=23),
        # dropout of a small batch's activations
        _case("dropout, batch of 64", "dropout", "train", 64, 1024, "fp32", p=0.5),
        # dropout of the largest activation tensor
        _case("dropout, 16384 rows of 2048", "dropout", "train", 16384, 2048, "bf16", p=0.1),
        # an odd width, rows that start off every alignment
        _case("dropout, odd", "dropout", "train", 4097, 333, "fp16", p=0.25),
        # serving: the residual stream of one row, no dropout
        _case("residual norm, one row", "residual_norm", "infer", 1, 2048, "bf16", params="bf16"),
        # the headline batch with an fp32 residual stream
        _case("residual norm, 4096 rows", "residual_norm", "train", 4096, 1024, "fp32", p=0.5),
        # the largest shape: bf16 branch on an fp32 residual stream
        _case("residual norm, 16384 rows", "residual_norm", "train", 16384, 2048, "bf16", stream="fp32", p=0.1),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "dropout", "residual_norm"])
    while True:
        rows, width = _log_int(rng, 1, 65536), _log_int(rng, 8, 8192)
        if rows * -(-width // 8) * 8 <= LARGEST:
            break
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    return _case(None, op, rng.choice(["infer", "train", "train"]) if op != "dropout" else "train", rows, width, dtype,
                 params=rng.choice(["fp32", dtype]), stream=rng.choice(["fp32", dtype]),
                 p=round(rng.uniform(0.02, 0.6), 3) if op != "layer_norm" else 0.0, pad=rng.choice([0, 0, 8, rng.randint(1, 40)]))


def work(case):
    """Every input once, every output once (forward and backward together where the case trains)."""
    n, w = case["rows"] * case["width"], case["width"]
    e, s, q = BYTES[case["dtype"]], BYTES[case["stream"]], BYTES[case["params"]]
    train = case["mode"] == "train"
    if case["op"] == "dropout":
        return {"bytes": 4 * e * n, "flops": 2 * n}
    if case["op"] == "layer_norm":
        return {"bytes": (4 if train else 2) * e * n + (4 if train else 2) * q * w, "flops": (22 if train else 8) * n}
    return {"bytes": (4 if train else 2) * (e + s) * n + (4 if train else 2) * q * w, "flops": (26 if train else 10) * n}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rows, width, pad = case["rows"], case["width"], case["pad"]
    dtype, stream, params = DTYPES[case["dtype"]], DTYPES[case["stream"]], DTYPES[case["params"]]
    train = case["mode"] == "train"

    def rand(kind, scale=1.0, offset=None):
        t = torch.randn(rows, width + pad, device=dev, generator=g) * scale
        return (t if offset is None else t + offset).to(kind)[:, :width]

    # activations: columns of different scale around different means
    spread = 0.5 + torch.rand(width + pad, device=dev, generator=g)
    centre = 0.5 * torch.randn(width + pad, device=dev, generator=g)
    s = {"case": case, "x": rand(dtype, spread, centre).requires_grad_(train), "dy": rand(dtype)}
    if case["op"] != "dropout":
        s["weight"] = (1 + 0.2 * torch.randn(width, device=dev, generator=g)).to(params).requires_grad_(train)
        s["bias"] = (0.2 * torch.randn(width, device=dev, generator=g)).to(params).requires_grad_(train)
    if case["op"] == "residual_norm":
        s["residual"] = rand(stream, spread, centre).requires_grad_(train)
        s["dh"] = rand(stream)
    # what the counter-based generator draws from
    s["draws"] = {"seed": (0x9E3779B97F4A7C15 ^ (seed * 0x2545F4914F6CDD1D)) & ((1 << 63) - 1), "step": (seed << 20) + 7,
                  "layer": 1000 + seed % 1000, "row_offset": 32 * (seed % 100)}
    return s


# ---- the framework's calls ----------------------------------------------------------------------------------------

def _run_own(s):
    import bilinear_amd as B
    case, x, train = s["case"], s["x"], s["case"]["mode"] == "train"
    if case["op"] == "dropout":
        y = B.dropout(x, case["p"], **s["draws"])
        return (y.detach(),) + torch.autograd.grad(y, (x,), s["dy"])
    if case["op"] == "layer_norm":
        y = B.layer_norm(x, s["weight"], s["bias"], EPS)
        if not train:
            return (y,)
        return (y.detach(),) + torch.autograd.grad(y, (x, s["weight"], s["bias"]), s["dy"])
    y, h = B.residual_norm(x, s["residual"], s["weight"], s["bias"], EPS, case["p"], **s["draws"])
    if not train:
        return y, h
    return (y.detach(), h.detach()) + torch.autograd.grad((y, h), (x, s["residual"], s["weight"], s["bias"]), (s["dy"], s["dh"]))


# ---- the plain form -----------------------------------------------------------------------------------------------

def _mul_hi_lo(a, m):
    """High and low 32 bits of a * m for 32-bit values in 64-bit integers (the products stay below 2^49)."""
    low, high = a * (m & 0xFFFF), a * (m >> 16)
    return (high + (low >> 16)) >> 16, (low + (high << 16)) & 0xFFFFFFFF


def _keep(rows, width, p, seed, step, layer, row_offset, device):
    """[rows, width] truth values: the 16-bit draw of Philox4x32-10 (Salmon et al., SC'11) reaches the threshold."""
    row = torch.arange(row_offset, row_offset + rows, device=device, dtype=torch.int64)[:, None]
    block = torch.arange((width + 7) // 8, device=device, dtype=torch.int64)[None, :]
    c0, c1 = row & 0xFFFFFFFF, block | ((row >> 32) << 21)
    c2, c3 = torch.full_like(c1, layer | 0x80000000), torch.full_like(c1, step & 0xFFFFFFFF)
    k0, k1 = (seed ^ (step >> 32)) & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        (h0, l0), (h1, l1) = _mul_hi_lo(c0, 0xD2511F53), _mul_hi_lo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack((c0, c1, c2, c3), -1)
    draws = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, -1)[:, :width]
    return draws >= _threshold(p)


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _scale(p):
    t = _threshold(p)
    return float(np.float32(65536.0 / (65536 - t))) if t < 65536 else 0.0


def _norm(h, weight, bias):
    mean = h.mean(-1, keepdim=True)
    rstd = 1 / ((h - mean).square().mean(-1, keepdim=True) + EPS).sqrt()
    hat = (h - mean) * rstd
    return hat * weight.float() + bias.float(), hat, rstd


def _norm_back(dy, hat, rstd, weight):
    t = dy * weight.float()
    dx = rstd * (t - t.mean(-1, keepdim=True) - hat * (t * hat).mean(-1, keepdim=True))
    return dx, (dy * hat).sum(0), dy.sum(0)


@torch.no_grad()
def _run_plain(s):
    case, x, train = s["case"], s["x"], s["case"]["mode"] == "train"
    dtype = x.dtype
    keep, scale = None, 1.0
    if _threshold(case["p"]):
        keep, scale = _keep(case["rows"], case["width"], case["p"], device=x.device, **s["draws"]), _scale(case["p"])

    def drop(v):
        return v if keep is None else torch.where(keep, v * scale, torch.zeros_like(v))

    if case["op"] == "dropout":
        return drop(x.float()).to(dtype), drop(s["dy"].float()).to(dtype)
    weight, bias = s["weight"], s["bias"]
    if case["op"] == "layer_norm":
        y, hat, rstd = _norm(x.float(), weight, bias)
        if not train:
            return (y.to(dtype),)
        dx, dg, db = _norm_back(s["dy"].float(), hat, rstd, weight)
        return y.to(dtype), dx.to(dtype), dg.to(weight.dtype), db.to(bias.dtype)
    stream = s["residual"].dtype
    h = (s["residual"].double() + drop(x.double())).to(stream)      # the residual stream is kept in its own type
    y, hat, rstd = _norm(h.float(), weight, bias)
    if not train:
        return y.to(dtype), h
    dh, dg, db = _norm_back(s["dy"].float(), hat, rstd, weight)
    dh = dh + s["dh"].float()
    return y.to(dtype), h, drop(dh).to(dtype), dh.to(stream), dg.to(weight.dtype), db.to(bias.dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------

def _philox_numpy(rows, width, seed, step, layer, row_offset):
    """The 16-bit draws, [rows, width] uint16, from 64-bit unsigned products."""
    u = np.uint64
    mask = u(0xFFFFFFFF)
    blocks = -(-width // 8)
    row = np.repeat(np.arange(row_offset, row_offset + rows, dtype=u), blocks)
    ctr = [row & mask, np.tile(np.arange(blocks, dtype=u), rows) | ((row >> u(32)) << u(21)),
           np.full(rows * blocks, 0x80000000 | layer, u), np.full(rows * blocks, step & 0xFFFFFFFF, u)]
    key = [(seed & 0xFFFFFFFF) ^ (step >> 32), seed >> 32]
    for n in range(10):
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        k0, k1 = u((key[0] + n * 0x9E3779B9) & 0xFFFFFFFF), u((key[1] + n * 0xBB67AE85) & 0xFFFFFFFF)
        ctr = [(b >> u(32)) ^ ctr[1] ^ k0, b & mask, (a >> u(32)) ^ ctr[3] ^ k1, a & mask]
    out = np.empty((rows, blocks, 8), np.uint16)
    for e in range(8):
        out[:, :, e] = ((ctr[e // 2] >> u(16 * (e % 2))) & u(0xFFFF)).astype(np.uint16).reshape(rows, blocks)
    return out.reshape(rows, blocks * 8)[:, :width]


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    x, dy = s["x"].double(), s["dy"].double()
    rows, width = x.shape
    t = math.floor(case["p"] * 65536 + 0.5)
    factor = 1.0
    if t > 0:
        u = torch.from_numpy(_philox_numpy(rows, width, **s["draws"]).astype(np.int32)).to(x.device)
        factor = (u >= t).double() * (float(np.float32(65536 / (65536 - t))) if t < 65536 else 0.0)
    if case["op"] == "dropout":
        return x * factor, dy * factor
    w, b = s["weight"].double(), s["bias"].double()
    if case["op"] == "residual_norm":
        total = s["residual"].double() + x * factor
        h = total.to(s["residual"].dtype).double()      # the stream's own type, before it is normalised
    else:
        total = h = x
    var, mean = torch.var_mean(h, dim=1, correction=0, keepdim=True)
    sigma = torch.sqrt(var + EPS)
    hat = (h - mean) / sigma
    y = torch.addcmul(b, hat, w)
    forward = (y,) if case["op"] == "layer_norm" else (y, total)
    if case["mode"] != "train":
        return forward
    v = dy * w
    along = (v * hat).sum(1, keepdim=True) / width
    dh = (v - v.sum(1, keepdim=True) / width - along * hat) / sigma
    weights = (torch.einsum("ij,ij->j", dy, hat), dy.sum(0))
    if case["op"] == "layer_norm":
        return forward + (dh,) + weights
    dh = dh + s["dh"].double()
    return forward + (dh * factor, dh) + weights
