"""Cases that measure the microscaled operators (8- and 4-bit blocks with shared scales) and the layers around them.

The path is the linear layer of a language model in microscaled formats: values are quantised in blocks along the
contracted dimension ("mxfp8": e4m3 codes, one power-of-two scale per 32; "mxfp4": e2m1 codes, one power-of-two scale
per 32; "nvfp4": e2m1 codes, one e4m3 scale per 16 and one fp32 scale per tensor), the tensor cores multiply the
blocks, and the layers between two products (root-mean-square norm with the residual's addition, SiLU gate) write
their outputs in the format that the next product reads. `run` computes each in its plain form (fp32 torch) or, where
`own` is true, through `cs464_b200.micro`; `exact` restates the definitions in 64 bits.
"""
import math

import torch

own = False

BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
# The largest finite magnitude of each element type, its exponent, and the fp32 mantissa bits of that magnitude.
ELEM = {"mxfp8": (448.0, 8, 0x600000), "mxfp4": (6.0, 2, 0x400000)}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the magnitudes of e2m1, in the order of their codes


def listed():
    return [
        # a layer's down projection weights (4096 x 14336), brought to 4 bits when a checkpoint is loaded, read back
        {"name": "quantize weights nvfp4", "op": "quantize", "rows": 4096, "cols": 14336, "format": "nvfp4",
         "dtype": "bf16", "transposed": False},
        # one decoding step's activations: the call's latency counts
        {"name": "quantize 16 tokens mxfp8", "op": "quantize", "rows": 16, "cols": 4096, "format": "mxfp8",
         "dtype": "bf16", "transposed": False},
        # a gradient seen through its transpose, as the weight gradient's product reads it; an odd number of tokens
        {"name": "quantize transposed mxfp8", "op": "quantize", "rows": 4096, "cols": 2047, "format": "mxfp8",
         "dtype": "bf16", "transposed": True},
        # the gate and up projection for one token: the weights' bytes bound it
        {"name": "product 1 token nvfp4", "op": "product", "M": 1, "N": 28672, "K": 4096, "format": "nvfp4",
         "dtype": "bf16"},
        # the down projection for a batch of 128 tokens
        {"name": "product 128 tokens mxfp4", "op": "product", "M": 128, "N": 4096, "K": 14336, "format": "mxfp4",
         "dtype": "fp16"},
        # the gate and up projection of a prefill of 8192 tokens: the tensor cores bound it
        {"name": "product prefill nvfp4", "op": "product", "M": 8192, "N": 28672, "K": 4096, "format": "nvfp4",
         "dtype": "bf16"},
        # a training step's query, key and value projection: forward and both gradients, every product in 8 bits
        {"name": "linear training mxfp8", "op": "linear", "M": 2048, "N": 6144, "K": 4096, "format": "mxfp8",
         "dtype": "bf16"},
        # the norm in front of a layer, for one token
        {"name": "norm 1 token mxfp8", "op": "norm", "rows": 1, "cols": 4096, "format": "mxfp8", "dtype": "bf16",
         "residual": True, "backward": False},
        # the same for a prefill of 8192 tokens
        {"name": "norm prefill mxfp8", "op": "norm", "rows": 8192, "cols": 4096, "format": "mxfp8", "dtype": "bf16",
         "residual": True, "backward": False},
        # the norm's gradient in a training step, with the gradient that arrives along the residual
        {"name": "norm backward", "op": "norm", "rows": 8192, "cols": 4096, "format": "none", "dtype": "bf16",
         "residual": True, "backward": True},
        # the gate between the two products of the feed-forward block, an odd number of tokens
        {"name": "gate 2047 tokens mxfp8", "op": "gate", "rows": 2047, "cols": 14336, "format": "mxfp8",
         "dtype": "bf16", "backward": False},
        # its gradient
        {"name": "gate backward", "op": "gate", "rows": 2048, "cols": 14336, "format": "none", "dtype": "fp16",
         "backward": True},
    ]


def _size(rng, lo, hi):
    """A size whose logarithm is uniform over [lo, hi]; three in four are multiples of 8 where they can be."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.75 and n >= 8:
        n -= n % 8
    return min(hi, max(lo, n))


def draw(rng):
    op = rng.choice(("quantize", "product", "product", "linear", "norm", "norm", "gate", "gate"))
    fmt = rng.choice(("mxfp8", "mxfp4", "nvfp4"))
    half = rng.choice(("bf16", "bf16", "fp16"))
    if op == "quantize":
        cols = _size(rng, 1, 28672)
        return {"op": op, "rows": _size(rng, 1, min(16384, (1 << 25) // cols)), "cols": cols, "format": fmt,
                "dtype": rng.choice(("bf16", "fp16", "fp32")), "transposed": rng.random() < 0.4}
    if op == "product":
        n, k = _size(rng, 16, 28672), _size(rng, 32, 14336)
        return {"op": op, "M": _size(rng, 1, max(1, min(8192, (1 << 39) // (n * k)))), "N": n, "K": k, "format": fmt,
                "dtype": half}
    if op == "linear":
        return {"op": op, "M": _size(rng, 1, 2048), "N": _size(rng, 16, 6144), "K": _size(rng, 32, 4096),
                "format": fmt, "dtype": half}
    backward = rng.random() < 0.35
    fmt = "none" if backward or rng.random() < 0.2 else fmt
    if op == "norm":
        cols = _size(rng, 16, 16384)
        return {"op": op, "rows": _size(rng, 1, min(16384, (1 << 25) // cols)), "cols": cols, "format": fmt,
                "dtype": half, "residual": rng.random() < 0.7, "backward": backward}
    cols = _size(rng, 16, 28672)
    return {"op": op, "rows": _size(rng, 1, min(16384, (1 << 24) // cols)), "cols": cols, "format": fmt,
            "dtype": half, "backward": backward}


# ---------------------------------------------------------------- the plain forms' parts
def _round_e2m1(v):
    """`v` rounded to the nearest e2m1 value, ties to the even code, magnitudes over 6 to 6."""
    a = v.abs()
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float())
    q = q + (a > 2.5).float() + (a >= 3.5).float() + 2.0 * (a > 5.0).float()
    return torch.copysign(q, v)


def _blocks(x, size):
    """x [R, C] as [R, ceil(C / size), size], the last block filled up with zeros."""
    r, c = x.shape
    n = -(-c // size)
    if n * size != c:
        x = torch.cat([x, x.new_zeros(r, n * size - c)], 1)
    return x.reshape(r, n, size)


def _tensor_scale(x):
    """nvfp4's scale of a whole tensor: the smallest power of two, from 2^-100 up, at which the largest magnitude is at
    most the largest code times the largest block scale, 6 * 448 = 2688 = 1.3125 * 2^11."""
    bits = x.abs().amax().view(torch.int32)
    e = ((bits >> 23) - 11 + ((bits & 0x7FFFFF) > 0x280000)).clamp(min=27)
    return (e << 23).view(torch.float32).reshape(1)


def _quantize(x, fmt, scale=None):
    """Code values [R, B, size], block scale values [R, B] and, for the power-of-two scales, their bytes, of x in fp32."""
    b = _blocks(x, BLOCK[fmt])
    amax = b.abs().amax(2)
    if fmt == "nvfp4":
        s = (amax / (6.0 * scale)).clamp(max=448.0).to(torch.float8_e4m3fn).float()
        unit = torch.where(s > 0, s * scale, torch.full_like(s, math.inf))  # a block whose scale is zero is zero
        return _round_e2m1(b / unit[:, :, None]), s, None
    _, emax, mant = ELEM[fmt]
    bits = amax.view(torch.int32)
    byte = ((bits >> 23) - emax + ((bits & 0x7FFFFF) > mant)).clamp(min=0)
    v = b * ((254 - byte) << 23).view(torch.float32)[:, :, None]
    s = torch.where(byte > 0, (byte << 23).view(torch.float32), torch.full_like(amax, 2.0 ** -127))
    return (v.to(torch.float8_e4m3fn).float() if fmt == "mxfp8" else _round_e2m1(v)), s, byte


def _values(x, fmt, scale=None):
    """The values [R, C] that x has once quantised, in fp32."""
    q, s, _ = _quantize(x, fmt, scale)
    v = (q * s[:, :, None]).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return v if scale is None else v * scale


def _tiles(table):
    """Scales [R, B] in the order the tensor cores read: tiles of 128 rows and 4 blocks, row 32 i + j of a tile at
    [j, i]; what is added to whole tiles is zero."""
    r, n = table.shape
    full = table.new_zeros(-(-r // 128) * 128, -(-n // 4) * 4)
    full[:r, :n] = table
    return full.view(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4)


def _stored(x, fmt):
    """x as a program keeps it once quantised: codes (bytes, rows of whole 32 elements), scales in tile order, and
    nvfp4's tensor scale."""
    scale = _tensor_scale(x) if fmt == "nvfp4" else None
    q, s, byte = _quantize(x, fmt, scale)
    q = _blocks(q.reshape(x.shape[0], -1), 32).reshape(x.shape[0], -1)
    if fmt == "mxfp8":
        codes = q.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = q.abs()
        n = sum((a >= g).to(torch.uint8) for g in GRID[1:]) + 8 * (q < 0).to(torch.uint8)
        codes = n[:, 0::2] + 16 * n[:, 1::2]
    table = s.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "nvfp4" else byte.to(torch.uint8)
    return codes.contiguous(), _tiles(table).permute(0, 3, 2, 1, 4).contiguous().view(-1, -(-s.shape[1] // 4), 512), scale


def _read(codes, scales, scale, rows, cols, fmt):
    """The values [rows, cols] of stored codes and scales, in fp32."""
    if fmt == "mxfp8":
        q = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
        q = table[torch.stack([codes & 15, codes >> 4], 2).reshape(rows, -1).int()]
    n = -(-cols // BLOCK[fmt])
    t = scales.view(-1, scales.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:rows, :n]
    if fmt == "nvfp4":
        s = t.contiguous().view(torch.float8_e4m3fn).float()
    else:
        b = t.int()
        s = torch.where(b > 0, (b << 23).view(torch.float32), torch.full_like(b, 2.0 ** -127, dtype=torch.float32))
    v = (_blocks(q[:, :cols], BLOCK[fmt]) * s[:, :, None]).reshape(rows, -1)[:, :cols]
    return v if scale is None else v * scale


def _coded(y, fmt, scale, dtype):
    """What a layer that writes a format gives back: 8 bits as code and scale values, 4 bits as the values of both."""
    if fmt == "none":
        return y.to(dtype)
    if fmt == "mxfp8":
        q, _, byte = _quantize(y, fmt)
        q = q.reshape(y.shape[0], -1)[:, :y.shape[1]]
        return q.to(torch.float8_e4m3fn), _tiles(byte.to(torch.uint8)).view(torch.float8_e8m0fnu)
    return _values(y, fmt, scale).to(dtype)


def _own_coded(y, fmt, dtype):
    """The same of the framework's answer."""
    if fmt == "none":
        return y
    if fmt == "mxfp8":
        return y.code_values(), y.scale_tiles()
    return y.dequantize(dtype)


# ---------------------------------------------------------------- the measured interface
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=DTYPES[case["dtype"]]):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    op, fmt = case["op"], case["format"]
    st = {"case": case, "dtype": DTYPES[case["dtype"]]}
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        # values of an activation or a weight: normal, rows of differing size
        x = normal(c, r) if case["transposed"] else normal(r, c)
        x = x * torch.exp2(torch.randint(-6, 3, (x.shape[0], 1), generator=g, device="cuda")).to(x.dtype)
        st["x"] = x.t() if case["transposed"] else x
    elif op == "product":
        m, n, k = case["M"], case["N"], case["K"]
        st["a"] = _stored(normal(m, k, dtype=torch.float32), fmt)
        st["b"] = _stored(normal(n, k, std=0.02, dtype=torch.float32), fmt)
    elif op == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        st["x"] = normal(m, k).requires_grad_()
        st["w"] = normal(n, k, std=0.02).requires_grad_()
        st["dy"] = normal(m, n, std=0.01)
    elif op == "norm":
        r, c = case["rows"], case["cols"]
        st["x"] = normal(r, c)
        st["w"] = (1.0 + normal(c, std=0.1).float()).to(st["dtype"])
        st["res"] = normal(r, c, std=2.0) if case["residual"] else None
        st["dy"] = normal(r, c, std=0.01) if case["backward"] else None
        # what calibration found: the largest of the norm's outputs, with room above it
        st["scale"] = torch.full((1,), 8.0 / 2688.0, device="cuda")
    else:
        r, c = case["rows"], case["cols"]
        st["x"] = normal(r, 2 * c)
        st["dy"] = normal(r, c, std=0.01) if case["backward"] else None
        st["scale"] = torch.full((1,), 16.0 / 2688.0, device="cuda")
    return st


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    from cs464_b200 import micro
    case, dtype = st["case"], st["dtype"]
    op, fmt = case["op"], case["format"]
    if op == "quantize":
        return micro.quantize(st["x"], fmt).dequantize(dtype)
    if op == "product":
        a = micro.MicroTensor(*st["a"][:2], (case["M"], case["K"]), fmt, st["a"][2])
        b = micro.MicroTensor(*st["b"][:2], (case["N"], case["K"]), fmt, st["b"][2])
        return micro.micro_matmul(a, b, dtype=dtype)
    if op == "linear":
        y = micro.micro_linear(st["x"], st["w"], fmt)
        return (y.detach(), *torch.autograd.grad(y, (st["x"], st["w"]), st["dy"]))
    if case["backward"]:
        if op == "norm":
            return micro.rms_norm_backward(st["dy"], st["x"], st["w"], EPS, dh=st["res"])
        return micro.silu_mul_backward(st["dy"], st["x"])
    kw = {} if fmt == "none" else {"format": fmt}
    if fmt == "nvfp4":
        kw["scale"] = st["scale"]
    if op == "norm":
        y, h = micro.rms_norm(st["x"], st["w"], residual=st["res"], eps=EPS, **kw)
        return _own_coded(y, fmt, dtype), (h if case["residual"] else None)
    return _own_coded(micro.silu_mul(st["x"], **kw), fmt, dtype)


def _run_plain(st):
    case, dtype = st["case"], st["dtype"]
    op, fmt = case["op"], case["format"]
    if op == "quantize":
        x = st["x"].float()
        return _values(x, fmt, _tensor_scale(x) if fmt == "nvfp4" else None).to(dtype)
    if op == "product":
        a = _read(*st["a"], case["M"], case["K"], fmt)
        b = _read(*st["b"], case["N"], case["K"], fmt)
        return (a @ b.t()).to(dtype)
    if op == "linear":
        def q(x):
            return _values(x, fmt, _tensor_scale(x) if fmt == "nvfp4" else None)
        x, w, dy = st["x"].detach().float(), st["w"].detach().float(), st["dy"].float()
        # each product's operands are quantised along the dimension that it sums over
        return ((q(x) @ q(w).t()).to(dtype), (q(dy) @ q(w.t()).t()).to(dtype), (q(dy.t()) @ q(x.t()).t()).to(dtype))
    if op == "norm":
        x, w = st["x"].float(), st["w"].float()
        if case["backward"]:
            dy = st["dy"].float()
            rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
            n, gr = x * rstd, dy * w
            dx = rstd * (gr - n * (gr * n).mean(1, keepdim=True))
            if st["res"] is not None:  # the gradient that arrives at the sum along the residual
                dx = dx + st["res"].float()
            return dx.to(dtype), (dy * n).sum(0).to(dtype)
        h = x if st["res"] is None else x + st["res"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * w
        return _coded(y, fmt, st["scale"] if fmt == "nvfp4" else None, dtype), (h.to(dtype) if case["residual"] else None)
    gate, up = st["x"].float().chunk(2, 1)
    sig = 1.0 / (1.0 + torch.exp(-gate))
    if case["backward"]:
        dy = st["dy"].float()
        return torch.cat([dy * up * sig * (1.0 + gate * (1.0 - sig)), dy * gate * sig], 1).to(dtype)
    return _coded(gate * sig * up, fmt, st["scale"] if fmt == "nvfp4" else None, dtype)


def _coded_bytes(rows, cols, fmt, size):
    """Bytes of a [rows, cols] tensor in a format (`size` bytes an element without one)."""
    if fmt == "none":
        return rows * cols * size
    return rows * cols * (1 if fmt == "mxfp8" else 0.5) + rows * -(-cols // BLOCK[fmt])


def work(case):
    op, fmt = case["op"], case["format"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        # read x, write and read the codes and scales, write the values; 4 operations an element
        return {"bytes": 2 * r * c * size + 2 * _coded_bytes(r, c, fmt, size), "flops": 4 * r * c}
    if op == "product":
        m, n, k = case["M"], case["N"], case["K"]
        return {"bytes": _coded_bytes(m, k, fmt, 2) + _coded_bytes(n, k, fmt, 2) + 2 * m * n, "flops": 2 * m * n * k}
    if op == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        # x, w and dy are read, y, dx and dw written
        return {"bytes": 2 * (2 * m * k + 2 * n * k + 2 * m * n), "flops": 6 * m * n * k}
    r, c = case["rows"], case["cols"]
    if op == "norm" and case["backward"]:
        return {"bytes": (3 + case["residual"]) * r * c * 2 + 4 * c, "flops": 12 * r * c}
    if op == "norm":
        return {"bytes": (1 + 2 * case["residual"]) * r * c * 2 + 2 * c + _coded_bytes(r, c, fmt, 2), "flops": 8 * r * c}
    if case["backward"]:
        return {"bytes": 5 * r * c * 2, "flops": 16 * r * c}
    return {"bytes": 2 * r * c * 2 + _coded_bytes(r, c, fmt, 2), "flops": 10 * r * c}


# ---------------------------------------------------------------- the definitions in 64 bits
def _near(v, mantissa, lowest, top):
    """v at the nearest value with `mantissa` fraction bits, exponents from `lowest` up and magnitudes up to `top`."""
    e = torch.frexp(v.abs().clamp(min=2.0 ** lowest))[1] - 1
    step = torch.exp2((e - mantissa).double())
    return (torch.round(v / step) * step).clamp(-top, top)


def _exact_blocks(x, fmt, scale=None):
    """(code values [R, C], scale values [R, B]) in 64 bits."""
    size = BLOCK[fmt]
    r, c = x.shape
    n = (c + size - 1) // size
    p = torch.nn.functional.pad(x, (0, n * size - c)).unflatten(1, (n, size))
    big = p.abs().max(2).values
    if fmt == "nvfp4":
        s = _near(big / 6.0 / scale, 3, -6, 448.0)
        unit = s * scale
    else:
        # the smallest power of two at which the block's largest magnitude does not pass the element type's
        m, e = torch.frexp(big / (448.0 if fmt == "mxfp8" else 6.0))
        s = torch.exp2((e - (m == 0.5).int()).clamp(min=-127).double())
        s = torch.where(big > 0, s, torch.full_like(s, 2.0 ** -127))
        unit = s
    v = torch.where(unit[..., None] > 0, p / unit[..., None], torch.zeros_like(p))
    q = _near(v, 3, -6, 448.0) if fmt == "mxfp8" else _near(v, 1, 0, 6.0)
    return q.flatten(1)[:, :c], s


def _exact_values(x, fmt, scale=None):
    if fmt == "nvfp4" and scale is None:
        scale = max(2.0 ** math.ceil(math.log2(max(float(x.abs().max()), 2.0 ** -120) / 2688.0)), 2.0 ** -100)
    q, s = _exact_blocks(x, fmt, scale)
    return q * s.repeat_interleave(BLOCK[fmt], 1)[:, :x.shape[1]] * (scale if fmt == "nvfp4" else 1.0)


def _exact_coded(y, fmt, scale):
    if fmt == "none":
        return y
    if fmt != "mxfp8":
        return _exact_values(y, fmt, scale)
    q, s = _exact_blocks(y, fmt)
    r, n = s.shape
    full = torch.full(((r + 127) // 128 * 128, (n + 3) // 4 * 4), 2.0 ** -127, dtype=torch.float64, device=y.device)
    full[:r, :n] = s
    return q, full.unflatten(1, (-1, 4)).unflatten(0, (-1, 4, 32))


def _exact_stored(stored, rows, cols, fmt):
    """The values of a stored operand: code by code and scale by scale, in 64 bits."""
    codes, scales, scale = stored
    if fmt == "mxfp8":
        c = codes.long()
        e, m = (c >> 3) & 15, (c & 7).double()
        q = torch.where(e > 0, (1.0 + m / 8.0) * torch.exp2(e.double() - 7.0), m / 512.0) * (1.0 - 2.0 * (c >> 7))
    else:
        c = torch.stack([codes % 16, codes // 16], -1).flatten(1).long()
        e, m = (c >> 1) & 3, (c & 1).double()
        q = torch.where(e > 0, (1.0 + m / 2.0) * torch.exp2(e.double() - 1.0), m / 2.0) * (1.0 - 2.0 * (c >> 3))
    r = torch.arange(rows, device=codes.device)[:, None]
    b = torch.arange((cols + BLOCK[fmt] - 1) // BLOCK[fmt], device=codes.device)[None, :]
    at = ((r // 128) * scales.shape[1] + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4
    t = scales.flatten()[at].long()
    if fmt == "nvfp4":
        e, m = (t >> 3) & 15, (t & 7).double()
        s = torch.where(e > 0, (1.0 + m / 8.0) * torch.exp2(e.double() - 7.0), m / 512.0) * scale.double()
    else:
        s = torch.exp2(t.double() - 127.0)
    return q[:, :cols] * s.repeat_interleave(BLOCK[fmt], 1)[:, :cols]


def exact(case, seed):
    st = prepare(case, seed)
    op, fmt = case["op"], case["format"]
    if op == "quantize":
        return _exact_values(st["x"].double(), fmt)
    if op == "product":
        return _exact_stored(st["a"], case["M"], case["K"], fmt) @ _exact_stored(st["b"], case["N"], case["K"], fmt).T
    if op == "linear":
        x, w, dy = (st[k].detach().double() for k in ("x", "w", "dy"))

        def v(t):
            return _exact_values(t, fmt)
        return v(x) @ v(w).T, v(dy) @ v(w.T).T, v(dy.T) @ v(x.T).T
    scale = float(st["scale"])
    x = st["x"].double()
    if op == "norm":
        w = st["w"].double()
        if case["backward"]:
            dy = st["dy"].double()
            var = x.square().mean(1, keepdim=True) + EPS
            dx = dy * w / var.sqrt() - x * (dy * w * x).mean(1, keepdim=True) / var ** 1.5
            return dx + (0.0 if st["res"] is None else st["res"].double()), (dy * x / var.sqrt()).sum(0)
        h = x + (0.0 if st["res"] is None else st["res"].double())
        y = h * w / (h.square().mean(1, keepdim=True) + EPS).sqrt()
        return _exact_coded(y, fmt, scale), (h if case["residual"] else None)
    c = case["cols"]
    gate, up = x[:, :c], x[:, c:]
    sig = torch.sigmoid(gate)
    if case["backward"]:
        dy = st["dy"].double()
        return torch.cat([dy * up * (sig + gate * sig * (1.0 - sig)), dy * gate * sig], 1)
    return _exact_coded(gate * sig * up, fmt, scale)
