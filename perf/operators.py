"""Measured cases of the microscaled 4-bit (MXFP4) operators: quantise, read back, product, training step.

A row is cut into blocks of 32 values.  A block holds one power-of-two scale 2^(s - 127), s = max(E - 2, 0) with E the
biased fp32 exponent field of the block's largest magnitude, and 32 codes of 4 bits (sign, 2 exponent bits, 1 mantissa
bit: 0 .5 1 1.5 2 3 4 6), each the nearest to x / scale, ties to even, saturated at 6.  Packed rows: 64 bytes of codes
and 4 of scales for every 128 values, low nibble first, zeros behind the row's end.

    roundtrip   dequantize(quantize(x))
    read        dequantize(packed)
    product     y = post * f(pre * (Q(x) W^T + b)) with a packed W
    train       the same with a float W that is quantised in the call, and the gradients straight through Q:
                dz = dy * dy/dz, dx = dz W^, dW = dz^T x^, db = sum of dz
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token's hidden state, as a serving loop quantises it before several products: latency only
        {"name": "roundtrip token", "op": "roundtrip", "m": 1, "k": 4096, "pad": 0, "dtype": "bf16"},
        # a column slice of a wider activation matrix, a width that ends inside a block
        {"name": "roundtrip ragged", "op": "roundtrip", "m": 1031, "k": 1000, "pad": 24, "dtype": "fp16"},
        # hidden activations of 1024 rays x 256 samples, width 256: the layer-wise path of a training batch
        {"name": "roundtrip samples", "op": "roundtrip", "m": 262144, "k": 256, "pad": 0, "dtype": "fp32"},
        # one hidden layer's weights read back for export
        {"name": "read hidden layer", "op": "read", "m": 256, "k": 256, "dtype": "fp32"},
        # a wide layer's weights read back
        {"name": "read wide layer", "op": "read", "m": 8192, "k": 8192, "dtype": "bf16"},
        # one token through a dense layer: bound by the weights' bytes
        {"name": "product token", "op": "product", "m": 1, "k": 4096, "n": 4096, "dtype": "bf16", "act": "none", "bias": False},
        # a few tokens in flight, sizes that fill no tile
        {"name": "product few ragged", "op": "product", "m": 13, "k": 8000, "n": 2050, "dtype": "fp16", "act": "none", "bias": True},
        # one hidden layer of a NeRF over 1024 rays x 256 samples
        {"name": "product samples", "op": "product", "m": 262144, "k": 256, "n": 256, "dtype": "fp32", "act": "relu", "bias": True},
        # a prompt through a wide dense layer: bound by the matrix pipe
        {"name": "product prompt", "op": "product", "m": 4096, "k": 8192, "n": 8192, "dtype": "bf16", "act": "none", "bias": False},
        # training step of a layer that reads features and encoding together (256 + 63 -> 257), odd batch
        {"name": "train ragged", "op": "train", "m": 6000, "k": 319, "n": 257, "dtype": "fp32", "act": "sin", "bias": True},
        # training step of one hidden sine layer over 1024 rays x 256 samples
        {"name": "train samples", "op": "train", "m": 262144, "k": 256, "n": 256, "dtype": "fp32", "act": "sin", "bias": True},
        # training step of a wide dense layer over a batch of tokens
        {"name": "train tokens", "op": "train", "m": 4096, "k": 4096, "n": 4096, "dtype": "bf16", "act": "none", "bias": True},
    ]


def _log(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi], odd ones among them; half of the time a multiple of 32."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 64:
        v -= v % 32
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["roundtrip", "read", "product", "product", "train"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    while True:
        m, k, n = _log(rng, 1, 262144), _log(rng, 32, 8192), _log(rng, 16, 8192)
        if op == "train" and m < 64:
            continue
        if m * (k + n) <= 262144 * 512 and m * k * n <= 4096 ** 3:
            break
    if op == "roundtrip":
        return {"op": op, "m": m, "k": k, "pad": rng.choice([0, 8, 24]), "dtype": dtype}
    if op == "read":
        return {"op": op, "m": n, "k": k, "dtype": dtype}
    # In 32 bits a ReLU's decision at z ~ 0 is the rounding's, so its gradient is compared in 16 bits only.
    acts = ["none", "sin", "sigmoid"] if op == "train" and dtype == "fp32" else ["none", "relu", "sin", "sigmoid"]
    return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": rng.choice(acts), "bias": op == "train" or rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    m, k = case["m"], case["k"]

    def rand(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = {"case": dict(case), "dtype": dt}
    if case["op"] == "read":
        s["codes"], s["scales"] = _pack(*_quantise(rand(m, k) / math.sqrt(k)))
        return s
    # activations: Gaussian with a spread of channel magnitudes, as hidden states have
    x = rand(m, k + case.get("pad", 0)) * torch.exp(0.5 * rand(k + case.get("pad", 0)))
    s["x"] = x.to(dt)[:, :k]
    if case["op"] == "roundtrip":
        return s
    w = rand(case["n"], k) / math.sqrt(k)
    s["b"] = (0.1 * rand(case["n"])).to(dt) if case["bias"] else None
    if case["op"] == "product":
        s["codes"], s["scales"] = _pack(*_quantise(w))
        return s
    s["w"] = w.to(dt)
    s["dy"] = rand(m, case["n"]).to(dt)
    s["leaves"] = [t.requires_grad_(True) for t in (s["x"], s["w"], s["b"])]
    return s


# ---------------------------------------------------------------------------------------------- plain form
def _quantise(x):
    """Codes [m, k'] (0..15) and scale bytes [m, k'/32] of the rows, k' = k rounded up to 128."""
    m, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % 128)).view(m, -1, 32)
    amax = x.abs().amax(dim=-1)
    byte = torch.clamp(((amax.view(torch.int32) >> 23) & 255) - 2, min=0)
    v = torch.ldexp(x, (127 - byte).unsqueeze(-1))
    a = v.abs()
    q = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), (torch.round(a / 2) * 2).clamp(max=6)))
    # the level's index: 0 .5 1 1.5 2 -> twice the value, 3 4 -> value + 2, 6 -> 7
    code = torch.where(q <= 2, 2 * q, torch.where(q <= 4, q + 2, torch.full_like(q, 7))).to(torch.uint8)
    return (code + 8 * torch.signbit(v).to(torch.uint8)).view(m, -1), byte.to(torch.uint8)


def _pack(codes, byte):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), byte.contiguous()


def _values(codes, byte, k):
    """The fp32 values of codes [m, k'] and scale bytes."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    v = levels[codes.long()].view(codes.shape[0], -1, 32)
    return torch.ldexp(v, (byte.to(torch.int32) - 127).unsqueeze(-1)).view(codes.shape[0], -1)[:, :k]


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], dim=-1).view(packed.shape[0], -1)


def _activation(act, z):
    """f(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    if act == "sin":
        return torch.sin(z), torch.cos(z)
    y = 1 / (1 + torch.exp(-z))
    return y, y * (1 - y)


def _plain(s):
    c, dt = s["case"], s["dtype"]
    if c["op"] == "roundtrip":
        return {"values": _values(*_quantise(s["x"]), c["k"]).to(dt)}
    if c["op"] == "read":
        return {"values": _values(_unpack(s["codes"]), s["scales"], c["k"]).to(dt)}
    xq = _values(*_quantise(s["x"].detach()), c["k"])
    if c["op"] == "product":
        wq = _values(_unpack(s["codes"]), s["scales"], c["k"])
    else:
        wq = _values(*_quantise(s["w"].detach()), c["k"])
    z = xq @ wq.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y, slope = _activation(c["act"], z)
    if c["op"] == "product":
        return {"y": y.to(dt)}
    dz = s["dy"].float() * slope
    return {"y": y.to(dt), "dx": (dz @ wq).to(dt), "dw": (dz.t() @ xq).to(dt), "db": dz.sum(dim=0).to(dt)}


def _framework(s):
    path = os.path.join(ROOT, "nerf-pytorch_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from nerf import mx
    c = s["case"]
    if c["op"] == "roundtrip":
        return {"values": mx.dequantize(mx.quantize(s["x"]), s["dtype"])}
    if c["op"] == "read":
        return {"values": mx.dequantize(mx.MXTensor(s["codes"], s["scales"], c["k"]), s["dtype"])}
    act = mx.ACTIVATIONS[c["act"]]
    if c["op"] == "product":
        with torch.no_grad():
            return {"y": mx.linear(s["x"], mx.MXTensor(s["codes"], s["scales"], c["k"]), s["b"], act)}
    y = mx.linear(s["x"], s["w"], s["b"], act)
    dx, dw, db = torch.autograd.grad(y, s["leaves"], s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def run(state):
    return _framework(state) if own else _plain(state)


def work(case):
    m, k, size = case["m"], case["k"], SIZE[case["dtype"]]
    packed = (k / 2 + k / 32)
    if case["op"] == "roundtrip":
        return {"bytes": m * (2 * k * size + packed), "flops": 3 * m * k}
    if case["op"] == "read":
        return {"bytes": m * (k * size + packed), "flops": m * k}
    n = case["n"]
    if case["op"] == "product":
        return {"bytes": (m * k + m * n + (n if case["bias"] else 0)) * size + n * packed, "flops": 2 * m * n * k}
    return {"bytes": (2 * m * k + 2 * m * n + 2 * n * k + 2 * n) * size, "flops": 6 * m * n * k}


# --------------------------------------------------------------------------------------- 64-bit definition
def _exact_rows(x):
    """The values that the rows' nearest codes stand for, in 64 bits: the code is the number of borders passed."""
    m, k = x.shape
    x = torch.cat([x.double(), x.new_zeros((m, -k % 32), dtype=torch.float64)], dim=1).reshape(m, -1, 32)
    top = x.abs().max(dim=-1, keepdim=True).values
    exponent = torch.clamp(torch.frexp(top).exponent - 1, min=-126)
    scale = torch.pow(torch.full_like(top, 2.0), torch.clamp(exponent - 2, min=-127).double())
    a = x.abs() / scale
    index = (a > 0.25).long() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    return (torch.sign(x) * levels[index] * scale).reshape(m, -1)[:, :k]


def _exact_packed(codes, scales, k):
    nibbles = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.int64, device=codes.device)
    nibbles[:, 0::2], nibbles[:, 1::2] = codes % 16, codes // 16
    exponent, mantissa = (nibbles // 2) % 4, (nibbles % 2).double()
    size = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * torch.pow(2.0, (exponent - 1).double()))
    size = torch.where(nibbles >= 8, -size, size)
    return (size * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, dim=1))[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    op, k = case["op"], case["k"]
    if op == "roundtrip":
        return {"values": _exact_rows(s["x"])}
    if op == "read":
        return {"values": _exact_packed(s["codes"], s["scales"], k)}
    with torch.no_grad():
        xq = _exact_rows(s["x"])
        wq = _exact_packed(s["codes"], s["scales"], k) if op == "product" else _exact_rows(s["w"])
        z = torch.mm(xq, wq.t().contiguous())
        if s["b"] is not None:
            z += s["b"].double()
        if case["act"] == "relu":
            y, slope = z * (z > 0), (z > 0).double()
        elif case["act"] == "sin":
            y, slope = z.sin(), z.cos()
        elif case["act"] == "sigmoid":
            y = torch.special.expit(z)
            slope = torch.special.expit(-z) * y
        else:
            y, slope = z, 1.0
        if op == "product":
            return {"y": y}
        dz = s["dy"].double() * slope
        return {"y": y, "dx": torch.mm(dz, wq), "dw": torch.mm(dz.t().contiguous(), xq), "db": dz.sum(0)}
