"""Cases of the block-scaled ("MX") matrix operators: what a user's program has in hand, one pass through an
operator in its plain form and through the framework, and the same in 64 bits.

A block-scaled matrix holds blocks of 32 consecutive values along one axis: codes of 4 bits (E2M1: 0, 0.5, 1, 1.5,
2, 3, 4, 6 and a sign) or 8 bits (integers, a unit being 1/64) and one power of two per block (a byte, 127 = 1).
A line is what runs along the blocked axis.  Codes: (lines, 16 or 32 bytes a block), element 2i of a line in the low
half of byte i.  Scales: (lines, blocks rounded up to a multiple of 8)."""
import math

import numpy as np
import torch

own = False

BLOCK = 32
# activation functions and their derivatives at z, by name
ACTS = ("relu", "sig", "tanh", "silu", "gelu")


# ---- cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a minibatch of 128 in front of a dense layer of 4096 inputs: the smallest conversion a training step makes
        {"name": "quant-batch", "op": "quant", "rows": 4096, "cols": 128, "axis": 0, "fmt": "fp4", "dtype": "f16", "sr": False},
        # a large weight matrix after its update, converted for the next step with stochastic rounding
        {"name": "quant-weights", "op": "quant", "rows": 16384, "cols": 8192, "axis": 1, "fmt": "fp4", "dtype": "f16", "sr": True},
        # the classifier layer (1000 outputs of 4096 inputs) for a minibatch of 128
        {"name": "dot-classifier", "op": "dot", "m": 1000, "n": 128, "k": 4096, "out": "f16", "relu": True},
        # ragged in every extent, 32-bit result
        {"name": "dot-ragged", "op": "dot", "m": 1111, "n": 777, "k": 2500, "out": "f32", "relu": False},
        # a training product that fills the chip
        {"name": "dot-square", "op": "dot", "m": 8192, "n": 8192, "k": 8192, "out": "f16", "relu": False},
        # one token through a 4-bit layer: latency
        {"name": "serve-token", "op": "serve", "m": 4096, "n": 1, "k": 4096, "out": "f16", "relu": True},
        # sixteen streams through the widest dense layer of the benchmark networks (25088 inputs)
        {"name": "serve-streams", "op": "serve", "m": 4096, "n": 16, "k": 25088, "out": "f16", "relu": True},
        # a prompt of 1000 tokens through a 4-bit layer
        {"name": "serve-prompt", "op": "serve", "m": 4096, "n": 1000, "k": 9216, "out": "f16", "relu": False},
        # activations of a minibatch and their checkpoint
        {"name": "act-batch", "op": "act", "rows": 4096, "cols": 128, "f": "silu", "back": False, "dtype": "f16"},
        # the error through the activations of a wide layer, from the checkpoint
        {"name": "act-back-wide", "op": "act", "rows": 16384, "cols": 8192, "f": "gelu", "back": True, "dtype": "f16"},
        # weight gradient of a dense layer (9216 inputs) for a minibatch of 128, 32-bit result
        {"name": "grad-batch", "op": "grad", "m": 4096, "n": 9216, "k": 128, "out": "f32"},
        # weight gradient over a long batch of tokens
        {"name": "grad-tokens", "op": "grad", "m": 4096, "n": 8192, "k": 8000, "out": "f16"},
    ]


def _between(rng, lo, hi):
    """a whole number, even over the logarithm; half of them rounded to a multiple of 16"""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v > 32 and rng.random() < 0.5:
        v -= v % 16
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("quant", "dot", "serve", "act", "grad"))
    if op in ("quant", "act"):
        rows, cols = _between(rng, 32, 16384), _between(rng, 32, 8192)
        dtype = rng.choice(("f16", "f16", "f32"))
        if dtype == "f32":
            rows = max(32, rows // 2)
        if op == "quant":
            return {"op": op, "rows": rows, "cols": cols, "axis": rng.randrange(2), "fmt": rng.choice(("fp4", "fp4", "int8")),
                    "dtype": dtype, "sr": rng.random() < 0.5}
        return {"op": op, "rows": rows, "cols": cols, "f": rng.choice(ACTS), "back": rng.random() < 0.5, "dtype": dtype}
    out = rng.choice(("f16", "f16", "f32"))
    if op == "dot":
        return {"op": op, "m": _between(rng, 64, 8192), "n": _between(rng, 16, 8192), "k": _between(rng, 64, 8192), "out": out,
                "relu": rng.random() < 0.3}
    if op == "serve":
        return {"op": op, "m": _between(rng, 256, 8192), "n": _between(rng, 1, 1024), "k": _between(rng, 256, 25088), "out": out,
                "relu": rng.random() < 0.3}
    return {"op": op, "m": _between(rng, 128, 4096), "n": _between(rng, 128, 9216), "k": _between(rng, 32, 8192), "out": out}


def _blocks(depth):
    return -(-depth // BLOCK)


def _mx_bytes(lines, depth, fmt):
    return lines * _blocks(depth) * ((16 if fmt == "fp4" else 32) + 1)


def work(case):
    op = case["op"]
    if op in ("quant", "act"):
        size = 2 if case["dtype"] == "f16" else 4
        n = case["rows"] * case["cols"]
        if op == "quant":
            lines, depth = (case["rows"], case["cols"]) if case["axis"] == 1 else (case["cols"], case["rows"])
            # in, codes and scales out, and the values they stand for
            return {"bytes": 2 * n * size + _mx_bytes(lines, depth, case["fmt"]), "flops": 0}
        saved = _mx_bytes(case["rows"], case["cols"], "int8")
        # forward: in, out, the checkpoint, and the values it stands for; backward: the checkpoint, error in, error out
        return {"bytes": (2 if case["back"] else 3) * n * size + saved, "flops": 0}
    m, n, k = case["m"], case["n"], case["k"]
    out = m * n * (2 if case["out"] == "f16" else 4)
    if op == "dot":
        b = _mx_bytes(m, k, "fp4") + _mx_bytes(n, k, "fp4")
    elif op == "serve":
        b = _mx_bytes(m, k, "fp4") + 2 * n * k
    else:
        b = 2 * m * k + _mx_bytes(n, k, "int8")
    return {"bytes": b + out, "flops": 2 * m * n * k}


# ---- plain form ---------------------------------------------------------------------------------------------------

def _torch_dtype(name):
    return torch.float16 if name == "f16" else torch.float32


def _fmix(h):
    h ^= h >> 16
    h = (h * 0x85EBCA6B) & 0xFFFFFFFF
    h ^= h >> 13
    h = (h * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _rand16(seed, stream, count, device):
    """16 random bits for each of `count` elements: elements 2i and 2i + 1 take the halves of word i of the framework's
    counter-based stream (high half first)"""
    ka = (_fmix(seed ^ 0x9E3779B9) + stream * 0x85EBCA77) & 0xFFFFFFFF
    kb = _fmix((stream + 0xC2B2AE3D) & 0xFFFFFFFF) ^ seed
    x = (torch.arange((count + 1) // 2, dtype=torch.int64, device=device) + ka) & 0xFFFFFFFF
    x ^= x >> 16
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x ^= kb
    x ^= x >> 15
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    x ^= x >> 16
    return torch.stack((x >> 16, x & 0xFFFF), dim=1).reshape(-1)[:count]


def _plain_codes(x, fmt, rand=None):
    """(lines, depth) -> signed codes (lines, blocks, 32) and exponents (lines, blocks) of value = grid(code) * 2^e"""
    lines, depth = x.shape
    nb = _blocks(depth)
    t = torch.zeros((lines, nb * BLOCK), dtype=torch.float32, device=x.device)
    t[:, :depth] = x
    t = t.view(lines, nb, BLOCK)
    amax = t.abs().amax(dim=2)
    e = torch.frexp(amax).exponent.to(torch.int32) - 1 - (2 if fmt == "fp4" else 6)
    e = torch.where(amax > 0, e, torch.full_like(e, -126))
    e = e.clamp(min=-126)
    if fmt == "fp4" and rand is not None:
        e = torch.where(torch.ldexp(amax, -e) > 6, e + 1, e)
    a = torch.ldexp(t.abs(), -e[:, :, None])
    if rand is not None:
        r = torch.zeros((lines, nb * BLOCK), dtype=torch.int64, device=x.device)
        r[:, :depth] = rand.view(lines, depth)
        r = r.view(lines, nb, BLOCK)
    if fmt == "fp4":
        below2, below4 = a < 2, a < 4
        offset = torch.where(below2, 0, torch.where(below4, 2, 4))
        if rand is None:
            unit = torch.where(below2, 0.5, torch.where(below4, 1.0, 2.0))
            code = torch.round(a / unit).to(torch.int64) + offset
        else:
            bits = torch.where(below2, 14, torch.where(below4, 15, 16))
            code = (((a * 32768.0).to(torch.int64) + (r >> (16 - bits))) >> bits) + offset
        code = code.clamp(max=7)
    else:
        code = torch.round(a).to(torch.int64) if rand is None else ((a * 65536.0).to(torch.int64) + r) >> 16
        code = code.clamp(max=127)
    return torch.where(t < 0, -code, code), e


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _plain_values(code, e, fmt, depth):
    if fmt == "fp4":
        grid = torch.tensor(_GRID, dtype=torch.float32, device=code.device)
        v = torch.where(code < 0, -grid[code.abs()], grid[code.abs()])
    else:
        v = code.to(torch.float32)
    return torch.ldexp(v, e[:, :, None]).reshape(code.shape[0], -1)[:, :depth]


def _pack(x, fmt):
    """a matrix in hand as codes and scales, lines first (nearest rounding)"""
    code, e = _plain_codes(x, fmt)
    lines, nb = e.shape
    if fmt == "fp4":
        nibble = torch.where(code < 0, 8 - code, code).reshape(lines, -1)
        codes = (nibble[:, 0::2] | (nibble[:, 1::2] << 4)).to(torch.uint8)
        byte = e + 127
    else:
        codes = code.to(torch.int8).view(torch.uint8).reshape(lines, -1)
        byte = e + 6 + 127
    scales = torch.zeros((lines, -(-nb // 8) * 8), dtype=torch.uint8, device=x.device)
    scales[:, :nb] = byte.to(torch.uint8)
    return codes.contiguous(), scales


def _unpack(codes, scales, fmt, depth):
    """the 32-bit values of codes and scales, (lines, depth)"""
    lines, nb = codes.shape[0], _blocks(depth)
    s = scales[:, :nb].to(torch.int32) - 127
    if fmt == "fp4":
        low, high = (codes & 15).to(torch.int64), (codes >> 4).to(torch.int64)
        q = torch.stack((low, high), dim=2).view(lines, nb, BLOCK)
        return _plain_values(torch.where(q >= 8, 8 - q, q), s, fmt, depth)
    return _plain_values(codes.view(torch.int8).view(lines, nb, BLOCK).to(torch.int64), s - 6, fmt, depth)


def _act(f, z):
    if f == "relu":
        return z.clamp(min=0)
    if f == "tanh":
        return torch.tanh(z)
    if f == "gelu":
        return 0.5 * z * torch.special.erfc(z * -math.sqrt(0.5))
    s = 1 / (1 + torch.exp(-z))
    return s if f == "sig" else z * s


def _act_slope(f, z):
    if f == "relu":
        return (z > 0).to(z.dtype)
    if f == "tanh":
        return 1 - torch.tanh(z) ** 2
    if f == "gelu":
        return 0.5 * torch.special.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 - s) if f == "sig" else s * (1 + z * (1 - s))


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quant":
        x = s["x"].float() if case["axis"] == 1 else s["x"].float().T
        rand = _rand16(s["seed"], s["stream"], x.numel(), x.device) if case["sr"] else None
        code, e = _plain_codes(x, case["fmt"], rand)
        v = _plain_values(code, e, case["fmt"], x.shape[1])
        return (v if case["axis"] == 1 else v.T).to(s["x"].dtype).contiguous()
    if op == "act":
        if case["back"]:
            z = _unpack(s["codes"], s["scales"], "int8", case["cols"])
            return (s["err"].float() * _act_slope(case["f"], z)).to(s["err"].dtype)
        z = s["z"].float()
        code, e = _plain_codes(z, "int8")
        return {"y": _act(case["f"], z).to(s["z"].dtype), "saved": _plain_values(code, e, "int8", case["cols"]).to(s["z"].dtype)}
    out = _torch_dtype(case["out"])
    if op == "dot":
        c = _unpack(s["a_codes"], s["a_scales"], "fp4", case["k"]) @ _unpack(s["b_codes"], s["b_scales"], "fp4", case["k"]).T
    elif op == "serve":
        c = _unpack(s["a_codes"], s["a_scales"], "fp4", case["k"]) @ s["x"].float()
    else:
        c = s["err"].float() @ _unpack(s["b_codes"], s["b_scales"], "int8", case["k"]).T
    if case.get("relu"):
        c = c.clamp(min=0)
    return c.to(out)


# ---- a user's program ----------------------------------------------------------------------------------------------

def _normal(shape, seed, scale, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _batch(shape, seed):
    """rectified activations of differing strength per feature, as (features, minibatch)"""
    x = _normal(shape, seed, 1.0, torch.float32) * torch.exp(_normal((shape[0], 1), seed + 1, 0.7, torch.float32))
    return x.clamp(min=0).to(torch.float16)


def prepare(case, seed):
    op = case["op"]
    base = 16 * int(seed)
    s = {"case": case, "seed": (int(seed) * 2654435761 + 97) & 0x7FFFFFFF, "stream": 1 + int(seed) % 1000}
    if op == "quant":
        dt = _torch_dtype(case["dtype"])
        s["x"] = _normal((case["rows"], case["cols"]), base, 0.05, dt)
        s["values"] = torch.empty_like(s["x"])
        lines, depth = (case["rows"], case["cols"]) if case["axis"] == 1 else (case["cols"], case["rows"])
        nb = _blocks(depth)
        s["codes"] = torch.empty((lines, nb * (16 if case["fmt"] == "fp4" else 32)), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty((lines, -(-nb // 8) * 8), dtype=torch.uint8, device="cuda")
    elif op == "act":
        dt = _torch_dtype(case["dtype"])
        z = _normal((case["rows"], case["cols"]), base, 1.5, dt)
        if case["back"]:
            s["codes"], s["scales"] = _pack(z.float(), "int8")
            s["err"] = _normal(tuple(z.shape), base + 1, 0.1, dt)
            s["out"] = torch.empty_like(z)
        else:
            nb = _blocks(case["cols"])
            s["z"], s["y"], s["values"] = z, torch.empty_like(z), torch.empty_like(z)
            s["codes"] = torch.empty((case["rows"], nb * 32), dtype=torch.uint8, device="cuda")
            s["scales"] = torch.empty((case["rows"], -(-nb // 8) * 8), dtype=torch.uint8, device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["c"] = torch.empty((m, n), dtype=_torch_dtype(case["out"]), device="cuda")
        if op == "grad":
            s["err"] = _normal((m, k), base, 0.1, torch.float16)
            s["b_codes"], s["b_scales"] = _pack(_batch((n, k), base + 1).float(), "int8")
        else:
            s["a_codes"], s["a_scales"] = _pack(_normal((m, k), base, 0.05, torch.float32), "fp4")
            x = _batch((k, n), base + 1)
            if op == "serve":
                s["x"] = x
            else:
                s["b_codes"], s["b_scales"] = _pack(x.T.float(), "fp4")
    if own:
        s["own"] = _handles(s)
    return s


def _handles(s):
    """the framework's tensors over the memory in hand, which a program of the framework holds from the start"""
    from nervanagpu_amd import GPUTensor, MXTensor, NervanaGPU
    case = s["case"]
    ng = NervanaGPU(seed=s["seed"])
    np_dtype = {torch.float16: np.float16, torch.float32: np.float32, torch.uint8: np.uint8}

    def dense(t):
        return GPUTensor(ng, tuple(t.shape), np_dtype[t.dtype], gpudata=t.data_ptr())

    def mx(shape, fmt, axis, codes, scales, rounding=0):
        return MXTensor(ng, shape, fmt, axis, codes=dense(codes), scales=dense(scales), rounding=rounding)

    h = {"ng": ng}
    for key in ("x", "values", "z", "y", "err", "out", "c"):
        if key in s:
            h[key] = dense(s[key])
    if case["op"] == "quant":
        h["q"] = mx((case["rows"], case["cols"]), case["fmt"], case["axis"], s["codes"], s["scales"], int(case["sr"]))
    elif case["op"] == "act":
        h["saved"] = mx((case["rows"], case["cols"]), "int8", 1, s["codes"], s["scales"])
    elif case["op"] == "grad":
        # the checkpoint of the layer's input (inputs, tokens), blocks along the tokens; the product takes its transpose
        h["b"] = mx((case["n"], case["k"]), "int8", 1, s["b_codes"], s["b_scales"]).T
    else:
        h["a"] = mx((case["m"], case["k"]), "fp4", 1, s["a_codes"], s["a_scales"])
        h["b"] = h["x"] if case["op"] == "serve" else mx((case["k"], case["n"]), "fp4", 0, s["b_codes"], s["b_scales"])
    return h


def run(s):
    if not own:
        return _run_plain(s)
    case, h = s["case"], s["own"]
    ng, op = h["ng"], case["op"]
    if op == "quant":
        ng.rng_counter = s["stream"] - 1
        ng.mx_quantize(h["x"], h["q"])
        ng.mx_dequantize(h["q"], h["values"])
        return s["values"]
    if op == "act":
        if case["back"]:
            ng.bprop_act(case["f"], h["saved"], h["err"], h["out"])
            return s["out"]
        ng.fprop_act(case["f"], h["z"], h["y"], saved=h["saved"])
        ng.mx_dequantize(h["saved"], h["values"])
        return {"y": s["y"], "saved": s["values"]}
    if op == "grad":
        ng.mx_dot(h["err"], h["b"], h["c"])
    else:
        ng.mx_dot(h["a"], h["b"], h["c"], relu=case["relu"])
    return s["c"]


# ---- 64 bits ---------------------------------------------------------------------------------------------------------

def _exact_round(x, fmt, rand=None):
    """block-scaled values of (lines, depth) in 64 bits, by the table of what a code can stand for"""
    lines, depth = x.shape
    pad = -depth % BLOCK
    t = torch.nn.functional.pad(x.double(), (0, pad)).reshape(-1, BLOCK)
    top = t.abs().max(dim=1, keepdim=True).values
    log = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    log = torch.where(torch.exp2(log) > top, log - 1, log)
    log = torch.where(torch.exp2(log + 1) <= top, log + 1, log)
    scale = torch.exp2(log - (2 if fmt == "fp4" else 6))
    if fmt == "fp4" and rand is not None:
        scale = torch.where(top > 6 * scale, 2 * scale, scale)
    a = t.abs() / scale
    if rand is not None:
        r = torch.nn.functional.pad(rand.reshape(lines, depth), (0, pad)).reshape(-1, BLOCK).double()
    if fmt == "fp4":
        if rand is None:
            # borders between neighbours; a value on one goes to the neighbour with the even code
            q = torch.zeros_like(a)
            for border, up, value in ((0.25, False, 0.5), (0.75, True, 1.0), (1.25, False, 1.5), (1.75, True, 2.0),
                                      (2.5, False, 3.0), (3.5, True, 4.0), (5.0, False, 6.0)):
                q = torch.where((a >= border) if up else (a > border), torch.full_like(a, value), q)
        else:
            unit = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
            steps = 32768 * unit
            share = torch.floor(r * steps / 65536) / steps
            q = torch.floor(torch.floor(a * 32768) / steps + share) * unit
        q = q.clamp(max=6)
    else:
        q = (torch.round(a) if rand is None else torch.floor(torch.floor(a * 65536) / 65536 + r / 65536)).clamp(max=127)
    return (torch.sign(t) * q * scale).reshape(lines, -1)[:, :depth]


def _exact_words(seed, stream, count):
    """the random halves of elements 0 .. count-1, in numpy's 32-bit arithmetic"""
    def mix(h):
        h = np.uint32(h)
        h ^= h >> np.uint32(16)
        h = np.uint32(h * np.uint32(0x85EBCA6B))
        h ^= h >> np.uint32(13)
        h = np.uint32(h * np.uint32(0xC2B2AE35))
        return np.uint32(h ^ (h >> np.uint32(16)))
    with np.errstate(over="ignore"):
        first = np.uint32(mix(seed ^ 0x9E3779B9) + np.uint32(stream) * np.uint32(0x85EBCA77))
        second = np.uint32(mix((stream + 0xC2B2AE3D) & 0xFFFFFFFF) ^ np.uint32(seed))
        x = np.arange((count + 1) // 2, dtype=np.uint32)
        x += first
        x ^= x >> np.uint32(16)
        x *= np.uint32(0x7FEB352D)
        x ^= second
        x ^= x >> np.uint32(15)
        x *= np.uint32(0x846CA68B)
        x ^= x >> np.uint32(16)
    halves = np.empty((x.size, 2), dtype=np.int32)
    halves[:, 0], halves[:, 1] = x >> np.uint32(16), x & np.uint32(0xFFFF)
    return torch.from_numpy(halves.reshape(-1)[:count]).cuda()


def _exact_values(codes, scales, fmt, depth):
    """64-bit values from the fields of codes and scales"""
    nb = _blocks(depth)
    scale = torch.exp2(scales[:, :nb].double() - 127).repeat_interleave(BLOCK, dim=1)
    if fmt == "fp4":
        nibbles = torch.empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.uint8, device=codes.device)
        nibbles[:, 0::2], nibbles[:, 1::2] = codes % 16, codes // 16
        exponent, half = ((nibbles // 2) % 4).double(), (nibbles % 2).double() * 0.5
        v = torch.where(exponent == 0, half, (1 + half) * torch.exp2(exponent - 1)) * (1 - 2 * (nibbles // 8).double())
    else:
        v = codes.double()
        v = torch.where(v >= 128, v - 256, v) / 64
    return (v * scale)[:, :depth]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        x = s["x"] if case["axis"] == 1 else s["x"].T
        rand = _exact_words(s["seed"], s["stream"], x.numel()) if case["sr"] else None
        v = _exact_round(x, case["fmt"], rand)
        return v if case["axis"] == 1 else v.T.contiguous()
    if op == "act":
        f = case["f"]
        z = _exact_values(s["codes"], s["scales"], "int8", case["cols"]) if case["back"] else s["z"].double()
        normal = torch.special.ndtr(z)
        logistic = torch.sigmoid(z)
        if not case["back"]:
            y = {"relu": lambda: torch.relu(z), "sig": lambda: logistic, "tanh": lambda: torch.tanh(z),
                 "silu": lambda: z * logistic, "gelu": lambda: z * normal}[f]()
            return {"y": y, "saved": _exact_round(s["z"], "int8")}
        density = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        slope = {"relu": lambda: torch.where(z > 0, 1.0, 0.0).double(), "sig": lambda: logistic * torch.sigmoid(-z),
                 "tanh": lambda: 1 / torch.cosh(z) ** 2, "silu": lambda: logistic + z * logistic * torch.sigmoid(-z),
                 "gelu": lambda: normal + z * density}[f]()
        return s["err"].double() * slope
    if op == "grad":
        c = s["err"].double() @ _exact_values(s["b_codes"], s["b_scales"], "int8", case["k"]).T.contiguous()
    else:
        a = _exact_values(s["a_codes"], s["a_scales"], "fp4", case["k"])
        b = s["x"].double() if op == "serve" else _exact_values(s["b_codes"], s["b_scales"], "fp4", case["k"]).T.contiguous()
        c = a @ b
    return torch.relu(c) if case.get("relu") else c
