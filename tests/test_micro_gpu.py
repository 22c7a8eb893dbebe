"""The microscaled operators on a B200 against 64-bit references (oracle/micro.py for the formats, formulas here for the
layers). Quantisation is compared bit for bit; where values are computed, each tolerance is derived beside it."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cs464_b200 import micro
from cs464_b200.suites import LLAMA_LAYERS, WEIGHT_STD
from oracle import micro as om

pytestmark = pytest.mark.gpu

FORMATS = tuple(micro.FORMATS)
HALF = (torch.float16, torch.bfloat16)
ALL = (*HALF, torch.float32)


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def normal(*shape, dtype=torch.bfloat16, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * std).to(dtype).cuda()


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def stored(q: micro.MicroTensor):
    """(codes, scale bytes) of a MicroTensor; everything outside them must be zero."""
    c, s, zero = om.unpack(q.codes.cpu().numpy(), q.scales.cpu().numpy(), *q.shape, q.format)
    assert zero, "bytes outside the tensor's codes and scales are not zero"
    return c, s


def check_quantized(q: micro.MicroTensor, x: np.ndarray):
    g = None if q.scale is None else float(q.scale)
    c, s = stored(q)
    rc, rs = om.quantize(x, q.format, g)
    assert np.array_equal(s, rs), (s != rs).sum()
    assert np.array_equal(c, rc), ((c != rc).sum(), c[c != rc][:4], rc[c != rc][:4])


# ---------------------------------------------------------------- quantise and dequantise
SHAPES = [(1, 1), (1, 31), (3, 33), (1, 4096), (16, 128), (33, 96), (127, 257), (128, 128), (129, 1000), (300, 64), (257, 4)]


def views(rows, cols, dtype, seed):
    """The same values through different strides and alignments."""
    x = normal(rows, cols, dtype=dtype, seed=seed) * torch.exp2(
        torch.arange(cols, device="cuda") % 7 - 3).to(dtype)
    yield "contiguous", x
    yield "transposed", x.t().contiguous().t()
    wide = torch.zeros(rows, cols + 3, dtype=dtype, device="cuda")
    wide[:, 1:cols + 1] = x
    yield "odd rows", wide[:, 1:cols + 1]
    tall = torch.zeros(cols, rows + 3, dtype=dtype, device="cuda")
    tall[:, 1:rows + 1] = x.t()
    yield "odd columns", tall[:, 1:rows + 1].t()
    step = torch.zeros(2 * rows, 3 * cols, dtype=dtype, device="cuda")
    step[::2, ::3] = x
    yield "steps", step[::2, ::3]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_bit_for_bit(fmt, dtype):
    for i, (rows, cols) in enumerate(SHAPES):
        for name, x in views(rows, cols, dtype, i):
            q = micro.quantize(x, fmt)
            if fmt == "nvfp4":
                assert float(q.scale) == om.tensor_scale(f64(x)), name
            check_quantized(q, f64(x))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_special_values(fmt, dtype):
    """Infinities, NaN, both zeros, the type's extremes and subnormals, ties, blocks of zeros: alone in a block and among
    ordinary values, by rows and through a transpose."""
    info = torch.finfo(dtype)
    special = [float("inf"), -float("inf"), float("nan"), 0.0, -0.0, info.max, info.min, info.tiny, info.tiny / 8,
               info.smallest_normal * 1.5, 6.0, 448.0, 0.25, 2.5, 5.0]
    x = torch.zeros(len(special) * 3, 96, dtype=dtype)
    for i, v in enumerate(special):
        x[3 * i, 5] = v                      # alone in its block of zeros
        x[3 * i + 1, :] = 1.0
        x[3 * i + 1, 40] = v                 # among ones; the other blocks of the row keep theirs
        x[3 * i + 2, :] = v                  # the whole row
    x = x.cuda()
    with np.errstate(all="ignore"):
        for t in (x, x.t().contiguous().t(), x.t()):
            q = micro.quantize(t, fmt)
            check_quantized(q, f64(t))
            d = q.dequantize(torch.float32)
            c, s = om.quantize(f64(t), fmt, None if q.scale is None else float(q.scale))
            v = om.values(c, s, fmt, None if q.scale is None else float(q.scale))
            assert np.array_equal(np.isnan(f64(d)), np.isnan(v))


def test_nvfp4_given_scale_and_saturation():
    x = normal(65, 160, dtype=torch.float32, seed=3)
    for g in (2.0 ** -9, 0.25, 1.0 / 448, 3.3e-4, 100.0):
        q = micro.quantize(x, "nvfp4", scale=torch.full((1,), g, device="cuda"))
        g32 = float(np.float32(g))
        c, s = stored(q)
        rc, rs = om.quantize(f64(x), "nvfp4", g32)
        # a scale that is no power of two makes unit = block scale * g round in fp32: a value within an fp32 half step
        # (relative 2^-24, twice) of the border between two codes may fall on its other side. Count those borders.
        v = np.abs(f64(x)).reshape(65, -1, 16) / (om.E4M3[rs] * g32)[..., None]
        with np.errstate(invalid="ignore"):
            near = (np.abs(v[..., None] / np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0]) - 1) < 2.0 ** -22).any(-1)
        assert np.array_equal(s, rs) and ((c != rc) <= near.reshape(c.shape)).all()
    top = micro.quantize(torch.full((1, 16), 1e6, device="cuda"), "nvfp4", scale=torch.ones(1, device="cuda"))
    assert (f64(top.dequantize(torch.float32)) == 2688.0).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("fmt", FORMATS)
def test_dequantize(fmt, dtype):
    for rows, cols in SHAPES:
        x = normal(rows, cols, dtype=torch.float32, seed=rows)
        q = micro.quantize(x, fmt)
        g = None if q.scale is None else float(q.scale)
        v = om.values(*om.quantize(f64(x), fmt, g), fmt, g)
        # code * scale has at most 6 significant bits and the tensor scale is a power of two: fp32 holds it, bf16 too;
        # fp16 also where it is in range, which |x| < 8 is but for scales below its subnormals' step, 2^-24
        want = torch.from_numpy(v).to(dtype)
        out = q.dequantize(dtype).cpu()
        assert torch.equal(out, want), (rows, cols)
        place = torch.full((rows + 1, 2 * cols + 1), 7.0, dtype=dtype, device="cuda")
        micro.dequantize(q, out=place[:rows, 1::2])
        assert torch.equal(place[:rows, 1::2].cpu(), want)
        assert (place[rows:] == 7).all() and (place[:, 0::2] == 7).all()  # what is not q's stays as it was


# ---------------------------------------------------------------- products
@pytest.mark.parametrize("dtype", ALL)
def test_nvfp4_saturates_whatever_the_quotient(dtype):
    """Values whose quotient by the given scale leaves fp32's range (a mask's lowest value, say) saturate like others past
    2688 times it; the rest of their block is what the definition gives. Powers of two, so that nothing rounds but the
    codes."""
    info = torch.finfo(dtype)
    for g in (2.0 ** -100, 2.0 ** -58, 2.0 ** -20, 2.0 ** -3, 1.0):
        x = normal(70, 200, dtype=dtype, seed=5, std=min(700.0 * g, 100.0))
        x[:, 3] = info.min
        x[1::2, 77] = info.max
        x[2, 100:120] = info.min
        for t in (x, x.t().contiguous().t(), x[:, :199]):
            q = micro.quantize(t, "nvfp4", scale=torch.full((1,), g, device="cuda"))
            check_quantized(q, f64(t))


def random_operand(rows, cols, fmt, seed, std=1.0):
    q = micro.quantize(normal(rows, cols, dtype=torch.float32, seed=seed, std=std), fmt)
    g = None if q.scale is None else float(q.scale)
    return q, om.values(*stored(q), fmt, g)


def check_product(c: torch.Tensor, a: np.ndarray, b: np.ndarray):
    """|c - ref| <= half a step of the output's type + the accumulation's error. One MMA adds the exact products of its K
    step (32 or 64 columns) to an fp32 accumulator; a rounding or truncation there loses at most 2^-22 of the largest
    partial sum, itself at most S = sum |a| |b|. ceil(K / 32) steps, up to 8 sums across K splits, one scaling."""
    ref = a @ b.T
    bound = half_step(c.dtype) * np.abs(ref) + (-(-a.shape[1] // 32) + 9) * 2.0 ** -22 * (np.abs(a) @ np.abs(b).T)
    bound += 2.0 ** -25 if c.dtype == torch.float16 else 0  # half of fp16's smallest subnormal
    err = np.abs(f64(c) - ref)
    assert np.isfinite(f64(c)).all() and (err <= bound).all(), (err - bound).max()


PRODUCTS = [(1, 1, 1), (1, 128, 256), (1, 1000, 4096), (7, 130, 96), (16, 4096, 33), (17, 257, 500), (33, 96, 1031),
            (64, 512, 2048), (65, 127, 64), (128, 384, 640), (129, 129, 129), (200, 1024, 300), (300, 264, 1500),
            (5, 8, 14336), (512, 640, 256), (1024, 768, 320), (1000, 1111, 777),
            (513, 2050, 9300), (510, 2431, 7001)]  # the last two: K split over two and three CTA pairs of a cluster


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("fmt", FORMATS)
def test_product(fmt, dtype):
    for i, (m, n, k) in enumerate(PRODUCTS):
        qa, a = random_operand(m, k, fmt, 2 * i)
        qb, b = random_operand(n, k, fmt, 2 * i + 1, std=0.05)
        check_product(micro.micro_matmul(qa, qb, dtype=dtype), a, b)
    micro.check_status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_product_every_k(fmt):
    """K from one column over the ends of blocks, scale tiles, MMA steps and stages: codes past K do not exist, and what
    lies in the ring's shared memory there is left from earlier stages."""
    for k in [*range(1, 70, 7), 95, 97, 127, 128, 129, 191, 193, 255, 256, 257, 320, 383, 385, 511, 513, 1023, 1025]:
        qa, a = random_operand(40, k, fmt, k)
        qb, b = random_operand(70, k, fmt, k + 1)
        check_product(micro.micro_matmul(qa, qb), a, b)


@pytest.mark.parametrize("layer", list(LLAMA_LAYERS))
def test_product_llama_layers(layer):
    """The layers' projections at decode and prefill sizes, 512 of the output columns checked in 64 bits."""
    k, n = LLAMA_LAYERS[layer]
    for fmt in FORMATS:
        qb = micro.quantize(normal(n, k, dtype=torch.float32, std=WEIGHT_STD), fmt)
        at = torch.randperm(n, generator=torch.Generator().manual_seed(1))[:512].cuda()
        b = qb.dequantize(torch.float32)[at].double()
        for m in (1, 16, 128, 2048):
            qa = micro.quantize(normal(m, k, dtype=torch.float32, seed=m), fmt)
            a = qa.dequantize(torch.float32).double()
            c = micro.micro_matmul(qa, qb)[:, at].double()
            ref, s = a @ b.T, a.abs() @ b.abs().T
            bound = half_step(torch.bfloat16) * ref.abs() + (-(-k // 32) + 9) * 2.0 ** -22 * s  # as in check_product
            assert ((c - ref).abs() <= bound).all(), (layer, fmt, m)
    micro.check_status()


@pytest.mark.parametrize("shape", [(5, 130, 96), (130, 130, 96), (300, 264, 1500), (513, 2050, 9300)])
def test_product_of_large_and_small_tensor_scales(shape):
    """Tensor scales whose product leaves fp32's range while results do not: tiny operands, and huge ones with zero rows
    and columns (0, where 0 times an infinity would be NaN)."""
    M, N, K = shape
    a, b = normal(M, K, dtype=torch.float32, seed=1), normal(N, K, dtype=torch.float32, seed=2)
    for sa, sb in ((2.0 ** -70, 2.0 ** -60), (2.0 ** 90, 2.0 ** -90), (2.0 ** -20, 2.0 ** 110)):
        qa, qb = micro.quantize(a * sa, "nvfp4"), micro.quantize(b * sb, "nvfp4")
        va, vb = (om.values(*stored(q), "nvfp4", float(q.scale)) for q in (qa, qb))
        c = micro.micro_matmul(qa, qb)
        ref, size = va @ vb.T, np.abs(va) @ np.abs(vb).T
        # as check_product, one scaling more; bf16's smallest subnormal is 2^-133
        bound = half_step(c.dtype) * np.abs(ref) + (-(-K // 32) + 10) * 2.0 ** -22 * size + 2.0 ** -134
        assert (np.abs(f64(c) - ref) <= bound).all(), (sa, sb)
    a[M // 2:], b[N // 2:] = 0, 0
    c = f64(micro.micro_matmul(micro.quantize(a * 2.0 ** 90, "nvfp4"), micro.quantize(b * 2.0 ** 90, "nvfp4")))
    assert (c[M // 2:] == 0).all() and (c[:, N // 2:] == 0).all() and np.isinf(c[:M // 2, :N // 2]).any()


def test_product_of_nan_blocks_stays_in_its_rows():
    """A NaN scale makes its own row (or column) of the product NaN and nothing else, in every format."""
    for fmt in FORMATS:
        x, w = normal(40, 256, dtype=torch.float32), normal(300, 256, dtype=torch.float32, seed=1)
        x[7, 200] = float("inf")
        w[299, 3] = float("nan")
        qa = micro.quantize(x, fmt)
        qb = micro.quantize(w, fmt)
        c = f64(micro.micro_matmul(qa, qb))
        bad = np.zeros((40, 300), bool)
        bad[7], bad[:, 299] = True, True
        assert np.array_equal(np.isnan(c), bad), fmt


def test_product_output_views_and_empty():
    for fmt in FORMATS:
        qa, a = random_operand(37, 200, fmt, 1)
        qb, b = random_operand(61, 200, fmt, 2)
        for start, width in ((0, 64), (8, 72), (1, 63), (3, 70)):  # aligned and odd rows
            big = torch.full((40, width + start), 5.0, dtype=torch.bfloat16, device="cuda")
            out = big[:37, start:start + 61]
            assert micro.micro_matmul(qa, qb, out=out) is out
            check_product(out, a, b)
            assert (big[37:] == 5).all() and (big[:, :start] == 5).all() and (big[:, start + 61:] == 5).all()
        one = torch.empty(1, 61, dtype=torch.float16, device="cuda").as_strided((1, 61), (7, 1))
        qa1, a1 = random_operand(1, 200, fmt, 3)
        check_product(micro.micro_matmul(qa1, qb, out=one), a1, b)
        no_k = [micro.quantize(torch.empty(n, 0, device="cuda"), fmt) for n in (5, 6)]
        assert (micro.micro_matmul(*no_k) == 0).all()
        none = micro.quantize(torch.empty(0, 200, device="cuda"), fmt)
        assert micro.micro_matmul(none, qb).shape == (0, 61) and micro.micro_matmul(qa, none).shape == (37, 0)


def test_product_repeats_bit_for_bit_and_runner():
    for fmt in FORMATS:
        for m, n, k in ((1, 4096, 4096), (130, 1000, 2000), (1024, 2048, 512)):
            qa, _ = random_operand(m, k, fmt, 1)
            qb, _ = random_operand(n, k, fmt, 2)
            first = micro.micro_matmul(qa, qb)
            run = micro.MicroMatmul().make_runner(qa, qb)
            for _ in range(3):
                assert torch.equal(run(), first)
            run.raise_on_status()


def test_product_refusals():
    x = normal(4, 64)
    q8, q4, qn = (micro.quantize(x, f) for f in FORMATS)
    with pytest.raises(ValueError, match="one format"):
        micro.micro_matmul(q8, q4)
    with pytest.raises(ValueError, match="must agree"):
        micro.micro_matmul(q8, micro.quantize(normal(4, 32), "mxfp8"))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        micro.micro_matmul(q8, q8, dtype=torch.float32)
    for out in (torch.empty(4, 5, dtype=torch.bfloat16, device="cuda"),
                torch.empty(4, 4, dtype=torch.bfloat16, device="cuda").t(),
                torch.empty(1, 4, dtype=torch.bfloat16, device="cuda").expand(4, 4)):
        with pytest.raises(ValueError, match="out must be"):
            micro.micro_matmul(q8, q8, out=out)
    with pytest.raises(TypeError, match="out must be"):
        micro.micro_matmul(q8, q8, out=torch.empty(4, 4, device="cuda"))
    with pytest.raises(ValueError, match="codes of a"):
        micro.MicroTensor(q8.codes[:, :32], q8.scales, (4, 64), "mxfp8")
    with pytest.raises(ValueError, match="codes of a"):
        micro.MicroTensor(q8.codes[:, 1:], q8.scales, (4, 33), "mxfp8")
    with pytest.raises(ValueError, match="scales of a"):
        micro.MicroTensor(q8.codes, q8.scales[:-1], (4, 64), "mxfp8")
    with pytest.raises(ValueError, match="no tensor scale"):
        micro.MicroTensor(q8.codes, q8.scales, (4, 64), "mxfp8", torch.ones(1, device="cuda"))
    with pytest.raises(ValueError, match="scale must be"):
        micro.MicroTensor(qn.codes, qn.scales, (4, 64), "nvfp4")
    with pytest.raises(ValueError, match="scale must be"):
        micro.quantize(x, "nvfp4", scale=torch.ones(1))
    with pytest.raises(ValueError, match="no tensor scale"):
        micro.quantize(x, "mxfp4", scale=torch.ones(1, device="cuda"))
    with pytest.raises(TypeError, match="x must be"):
        micro.quantize(x.double(), "mxfp8")
    with pytest.raises(ValueError, match="a matrix"):
        micro.quantize(x[0], "mxfp8")
    with pytest.raises(TypeError, match="packed"):
        q4.code_values()


# ---------------------------------------------------------------- norm
def norm64(x, w, eps, res=None):
    h = x if res is None else x + res
    return h * w / np.sqrt((h * h).mean(1, keepdims=True) + eps), h


def norm_tolerance(y, dtype):
    """Half a step of the output's type, and in fp32 the sum of squares (pairwise over threads: a few tens of roundings of
    2^-24), a reciprocal root of two ulps and three products: below 2^-18 in all."""
    return (half_step(dtype) + 2.0 ** -18) * np.abs(y) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -130)


NORMS = [(1, 1), (1, 4096), (2, 7), (5, 64), (3, 1000), (130, 129), (600, 72), (33, 2048), (700, 520), (4, 8200), (2, 16384),
         (3, 16392), (2, 40001)]


@pytest.mark.parametrize("dtype", HALF)
def test_norm_values(dtype):
    for i, (rows, cols) in enumerate(NORMS):
        x, r = normal(rows, cols, dtype=dtype, seed=i), normal(rows, cols, dtype=dtype, seed=i + 50, std=2.0)
        w = normal(cols, dtype=dtype, seed=i + 99)
        for res in (None, r):
            y, h = micro.rms_norm(x, w, residual=res, eps=1e-5)
            ry, rh = norm64(f64(x), f64(w), 1e-5, None if res is None else f64(res))
            assert (np.abs(f64(y) - ry) <= norm_tolerance(ry, dtype)).all(), (rows, cols)
            # the sum of two values of the type in fp32 (half an ulp of fp32 at most), then rounded
            assert (np.abs(f64(h) - rh) <= (half_step(dtype) + 2.0 ** -24) * np.abs(rh)).all()
            assert h is x if res is None else True


def check_coded(q: micro.MicroTensor, y: np.ndarray, slack: float):
    """q holds y, known to the kernel up to a relative error `slack`: every value is within half a step of its code
    (relative to the block scale that q uses) plus that error, and every block scale is the definition's or, where the
    largest magnitude lies within `slack` of the border between two, its neighbour."""
    fmt = q.format
    g = None if q.scale is None else float(q.scale)
    c, s = stored(q)
    _, rs = om.quantize(y, fmt, g)
    lo = om.quantize(y * (1 - slack), fmt, g)[1].astype(int)
    hi = om.quantize(y * (1 + slack), fmt, g)[1].astype(int)
    assert ((s >= lo) & (s <= hi)).all()
    assert (s != rs).mean() < 0.01
    v = om.values(c, s, fmt, g)
    with np.errstate(divide="ignore"):
        unit = np.repeat(om.E4M3[s] * g if fmt == "nvfp4" else 2.0 ** (s.astype(int) - 127.0), om.BLOCK[fmt], 1)[:, :y.shape[1]]
    u = np.abs(y) / np.where(unit > 0, unit, np.inf)
    if fmt == "mxfp8":
        step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(u, 2.0 ** -6))), -6) - 3)
        top = 448.0
    else:
        step = np.where(u < 2, 0.5, np.where(u < 4, 1.0, 2.0))
        top = 6.0
    tol = (step / 2 + 2 * slack * u + np.maximum(u - top, 0)) * unit
    zero = unit == 0  # an nvfp4 block whose scale rounds to zero is zero
    assert (np.abs(v - y)[~zero] <= tol[~zero] * (1 + 1e-9)).all() and (v[zero] == 0).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("fmt", FORMATS)
def test_norm_coded(fmt, dtype):
    for i, (rows, cols) in enumerate(NORMS):
        x, r = normal(rows, cols, dtype=dtype, seed=i), normal(rows, cols, dtype=dtype, seed=i + 50)
        w = normal(cols, dtype=dtype, seed=i + 99)
        scale = torch.full((1,), 0.01, device="cuda") if fmt == "nvfp4" else None
        for res in (None, r):
            q, h = micro.rms_norm(x, w, residual=res, format=fmt, scale=scale)
            ry, rh = norm64(f64(x), f64(w), 1e-5, None if res is None else f64(res))
            check_coded(q, ry, 2.0 ** -18)
            assert (np.abs(f64(h) - rh) <= (half_step(dtype) + 2.0 ** -24) * np.abs(rh)).all()


def test_norm_of_strided_and_special_rows():
    """Views of every kind, rows of zeros, infinities and NaN; a row that is not finite leaves the others alone."""
    base = normal(40, 300, seed=3)
    w = normal(256, seed=4)
    for x in (base[:33, 4:260], base[:33, 40:296], normal(256, 33, seed=5).t(), normal(1, 256, seed=6).expand(33, 256),
              normal(66, 512, seed=7)[::2, ::2]):
        ry, _ = norm64(f64(x), f64(w), 1e-5)
        assert (np.abs(f64(micro.rms_norm(x, w)[0]) - ry) <= norm_tolerance(ry, torch.bfloat16)).all()
        check_coded(micro.rms_norm(x, w, format="mxfp8")[0], ry, 2.0 ** -18)
        ry, _ = norm64(f64(x), f64(w), 1e-5, f64(base[:33, 7:263]))
        y, _ = micro.rms_norm(x, w, residual=base[:33, 7:263])
        assert (np.abs(f64(y) - ry) <= norm_tolerance(ry, torch.bfloat16)).all()
    x = normal(6, 256, seed=8)
    x[1] = 0
    x[2, 3], x[4, 5] = float("inf"), float("nan")
    y = micro.rms_norm(x, w)[0]
    d = micro.rms_norm(x, w, format="mxfp8")[0].dequantize()
    good = [0, 1, 3, 5]
    ry, _ = norm64(f64(x)[good], f64(w), 1e-5)
    assert (np.abs(f64(y)[good] - ry) <= norm_tolerance(ry, torch.bfloat16)).all()
    assert np.isfinite(f64(d)[good]).all() and (f64(y)[1] == 0).all() and (f64(d)[1] == 0).all()
    assert np.isnan(f64(y)[4]).all() and np.isnan(f64(y)[2, 3]) and np.isnan(f64(d)[4]).all()
    assert micro.rms_norm(x[:0], w)[0].shape == (0, 256)
    y3, h3 = micro.rms_norm(x[good].view(2, 2, 256), w, residual=x[good].view(2, 2, 256))
    assert y3.shape == h3.shape == (2, 2, 256)


def norm_grad64(dy, h, w, eps, dh=None):
    n = h.shape[1]
    r = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    dot = (dy * w * h).sum(1, keepdims=True)
    dx = r * dy * w - h * r ** 3 * dot / n
    return dx + (0 if dh is None else dh), (dy * h * r).sum(0), r


@pytest.mark.parametrize("dtype", HALF)
def test_norm_backward(dtype):
    for i, (rows, cols) in enumerate(NORMS + [(3000, 64), (1500, 1024)]):
        dy, h = normal(rows, cols, dtype=dtype, seed=i), normal(rows, cols, dtype=dtype, seed=i + 20)
        w, dh = normal(cols, dtype=dtype, seed=i + 40), normal(rows, cols, dtype=dtype, seed=i + 60)
        for extra in (None, dh):
            dx, dw = micro.rms_norm_backward(dy, h, w, 1e-5, dh=extra)
            a, b, c = f64(dy), f64(h), f64(w)
            rx, rw, r = norm_grad64(a, b, c, 1e-5, None if extra is None else f64(extra))
            # dx: half a step of the type, and fp32 errors below 2^-18 of the terms' magnitudes (as in norm_tolerance;
            # the mean's against the sum of its terms' magnitudes)
            mag = np.abs(a * c) * r + np.abs(b) * r ** 3 * np.abs(a * b * c).mean(1, keepdims=True)
            tiny = 2.0 ** -25 if dtype == torch.float16 else 0
            assert (np.abs(f64(dx) - rx) <= half_step(dtype) * np.abs(rx) + 2.0 ** -18 * (mag + np.abs(rx)) + tiny).all(), (rows, cols)
            # dw: a sum over the rows in fp32, at most rows additions of 2^-24 each of the terms' sum
            tol = half_step(dtype) * np.abs(rw) + (2.0 ** -18 + rows * 2.0 ** -24) * np.abs(a * b * r).sum(0) + tiny
            assert (np.abs(f64(dw) - rw) <= tol).all(), (rows, cols)
            again = micro.rms_norm_backward(dy, h, w, 1e-5, dh=extra)
            assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("size", [1e-9, 1e9, 1e13, 1e15, 1e16])
def test_norm_backward_of_large_and_small_rows(size):
    """Rows whose 1 / norm cubed leaves fp32's range; the squares' sum does not (64 columns of up to 5e16: below 2e35).
    Bounds as in test_norm_backward. dweight's terms are of the size of dy."""
    dy, w = normal(33, 64, seed=1), normal(64, seed=2)
    h = (normal(33, 64, dtype=torch.float32, seed=3) * size).bfloat16()
    dx, dw = micro.rms_norm_backward(dy, h, w, 1e-5)
    a, b, c = f64(dy), f64(h), f64(w)
    rx, rw, r = norm_grad64(a, b, c, 1e-5)
    mag = np.abs(a * c) * r + np.abs(b) * r ** 3 * np.abs(a * b * c).mean(1, keepdims=True)
    assert (np.abs(f64(dx) - rx) <= half_step(torch.bfloat16) * np.abs(rx) + 2.0 ** -18 * (mag + np.abs(rx))).all()
    tol = half_step(torch.bfloat16) * np.abs(rw) + (2.0 ** -18 + 33 * 2.0 ** -24) * np.abs(a * b * r).sum(0)
    assert (np.abs(f64(dw) - rw) <= tol).all()


def test_norm_gradient_formula_against_differences():
    """The formula the gradients are tested against, by central differences of the 64-bit forward pass."""
    rng = np.random.default_rng(0)
    x, w, dy, dh = rng.normal(size=(3, 9)), rng.normal(size=9), rng.normal(size=(3, 9)), rng.normal(size=(3, 9))
    dx, dw, _ = norm_grad64(dy, x, w, 1e-5, dh)
    loss = lambda x, w: (norm64(x, w, 1e-5)[0] * dy).sum() + (x * dh).sum()  # noqa: E731
    e = 1e-6
    for i in np.ndindex(x.shape):
        d = np.zeros_like(x)
        d[i] = e
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * e) - dx[i]) < 1e-7
    for i in range(9):
        d = np.zeros(9)
        d[i] = e
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * e) - dw[i]) < 1e-7


def test_norm_autograd_with_shared_and_broadcast_inputs():
    """Gradients through autograd: strided and expanded upstream gradients, either output unused, x used twice."""
    x0, r0, w0 = normal(20, 72, seed=1), normal(20, 72, seed=2), normal(72, seed=3)
    for use in ("both", "y", "h", "same"):
        x, r, w = (t.clone().requires_grad_() for t in (x0, r0, w0))
        y, h = micro.rms_norm(x, w, residual=x if use == "same" else r)
        gy, gh = normal(72, 20, seed=4).t(), normal(20, 1, seed=5).expand(20, 72)
        loss = (y * gy).sum() if use != "h" else 0
        loss = loss + ((h * gh).sum() if use != "y" else 0)
        loss.backward()
        hr = f64(h)
        rx, rw, _ = norm_grad64(f64(gy) * (use != "h"), hr, f64(w0), 1e-5, f64(gh) * (use != "y"))
        tol = half_step(torch.bfloat16) * np.abs(rx) + 2.0 ** -16 * (np.abs(rx).max() + 1)
        if use == "same":  # two contributions of dx, added in bf16
            assert (np.abs(f64(x.grad) - 2 * rx) <= 4 * tol).all()
        else:
            assert (np.abs(f64(x.grad) - rx) <= tol).all() and torch.equal(x.grad, r.grad)
        if use == "h":
            assert w.grad is None or (w.grad == 0).all()
        else:
            assert (np.abs(f64(w.grad) - rw) <= half_step(torch.bfloat16) * np.abs(rw) + 1e-3).all()
    x = x0.clone().requires_grad_()
    y, h = micro.rms_norm(x, w0)
    assert h is x
    (g,) = torch.autograd.grad(y.sum(), x)
    rx, _, _ = norm_grad64(np.ones((20, 72)), f64(x0), f64(w0), 1e-5)
    assert (np.abs(f64(g) - rx) <= half_step(torch.bfloat16) * np.abs(rx) + 2.0 ** -16 * (np.abs(rx).max() + 1)).all()
    with pytest.raises(ValueError, match="no gradient"):
        micro.rms_norm(x, w0, format="mxfp8")
    with torch.no_grad():
        micro.rms_norm(x, w0, format="mxfp8")


def test_layer_refusals():
    x, w = normal(4, 64), normal(64)
    with pytest.raises(ValueError, match="weight must be"):
        micro.rms_norm(x, w[:63])
    with pytest.raises(TypeError, match="weight must be bfloat16"):
        micro.rms_norm(x, w.half())
    with pytest.raises(TypeError, match="x must be"):
        micro.rms_norm(x.float(), w.float())
    with pytest.raises(ValueError, match="residual is"):
        micro.rms_norm(x, w, residual=x[:3])
    with pytest.raises(ValueError, match="nvfp4 needs"):
        micro.rms_norm(x, w, format="nvfp4")
    with pytest.raises(ValueError, match="no tensor scale"):
        micro.rms_norm(x, w, format="mxfp8", scale=torch.ones(1, device="cuda"))
    with pytest.raises(ValueError, match="scale belongs"):
        micro.rms_norm(x, w, scale=torch.ones(1, device="cuda"))
    with pytest.raises(ValueError, match="one shape"):
        micro.rms_norm_backward(x[:3], x, w)
    with pytest.raises(ValueError, match=r"\[gate \| up\]"):
        micro.silu_mul(x[:, :63])
    with pytest.raises(ValueError, match="dy is"):
        micro.silu_mul_backward(x, x)
    with pytest.raises(ValueError, match="x must be"):
        micro.micro_linear(x, normal(8, 63))
    with pytest.raises(TypeError, match="w must be bfloat16"):
        micro.micro_linear(x, normal(8, 64).half())


# ---------------------------------------------------------------- gate
def gate64(x):
    c = x.shape[1] // 2
    g, u = x[:, :c], x[:, c:]
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u


def gate_grad64(dy, x):
    c = x.shape[1] // 2
    g, u = x[:, :c], x[:, c:]
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-g))
    return np.concatenate([dy * u * s * (1 + g * (1 - s)), dy * g * s], 1)


GATES = [(1, 1), (1, 14336), (3, 5), (2, 31), (130, 33), (64, 128), (129, 1000), (40, 1096), (2047, 72)]


@pytest.mark.parametrize("dtype", HALF)
def test_gate(dtype):
    """The fast exponential errs by at most 2 + 1.173 |gate| ulps (25 of 2^-23 for the |gate| < 20 here, below 2^-18.3),
    the division by 2 ulps, two products and a sum by half an ulp each: below 2^-18 in all."""
    for i, (rows, cols) in enumerate(GATES):
        wide = normal(rows, 2 * cols + 5, dtype=dtype, seed=i, std=4.0)
        for x in (wide[:, :2 * cols], wide[:, 5:], wide.contiguous()[:, 1:2 * cols + 1], wide[:, :2 * cols].t().contiguous().t(),
                  wide[:, :2 * cols].contiguous()):
            ry = gate64(f64(x))
            tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -130
            y = micro.silu_mul(x)
            assert (np.abs(f64(y) - ry) <= (half_step(dtype) + 2.0 ** -18) * np.abs(ry) + tiny).all(), (rows, cols)
            for fmt in FORMATS:
                q = micro.silu_mul(x, format=fmt, scale=torch.full((1,), 0.05, device="cuda") if fmt == "nvfp4" else None)
                check_coded(q, ry, 2.0 ** -18)
            dy = normal(rows, cols, dtype=dtype, seed=i + 30)
            a, b = f64(dy), f64(x)
            rg = gate_grad64(a, b)
            # 1 + g (1 - s) cancels near g = -1.28: its error is against the terms' magnitudes
            c = cols
            s = 1 / (1 + np.exp(-b[:, :c]))
            mag = np.concatenate([np.abs(a * b[:, c:]) * s * (1 + np.abs(b[:, :c]) * (1 - s)), np.abs(rg[:, c:])], 1)
            got = f64(micro.silu_mul_backward(dy, x))
            assert (np.abs(got - rg) <= half_step(dtype) * np.abs(rg) + 2.0 ** -18 * mag + tiny).all(), (rows, cols)


def test_gate_extremes():
    big = torch.finfo(torch.bfloat16).max
    g = torch.tensor([[0.0, -0.0, 100.0, -100.0, 1e4, -1e4, big, -big, 89.0, -89.0, -88.0, 30.0]], dtype=torch.bfloat16, device="cuda")
    x = torch.cat([g, torch.ones_like(g)], 1)
    y = f64(micro.silu_mul(x))
    assert (np.abs(y - gate64(f64(x))) <= (half_step(torch.bfloat16) + 2.0 ** -15) * np.abs(gate64(f64(x))) + 1e-35).all()
    d = f64(micro.silu_mul_backward(torch.ones_like(g), x))
    assert np.isfinite(d).all() and d[0, 2] == 1.0 and d[0, 3] == 0.0 and d[0, 6] == 1.0 and abs(d[0, 7]) == 0.0
    assert micro.silu_mul(x[:0]).shape == (0, 12) and micro.silu_mul(x.view(1, 1, 24)).shape == (1, 1, 12)


def test_gate_of_very_negative_gates():
    """Gates down to -88, where the sigmoid (6e-39 and up) is among fp32's subnormals, against large values: the
    exponential errs by 2 + 1.173 * 88 ulps, of at most 2^-149 / 6e-39 < 2^-21.9 of the value: below 2^-15 in all."""
    g = torch.linspace(-88.0, -60.0, 113).bfloat16().cuda().expand(3, -1)
    x = torch.cat([g, torch.full_like(g, 1e30)], 1)
    ref = gate64(f64(x))
    assert (np.abs(f64(micro.silu_mul(x)) - ref) <= (half_step(torch.bfloat16) + 2.0 ** -15) * np.abs(ref)).all()


def test_gate_gradient_formula_against_differences():
    rng = np.random.default_rng(0)
    x, dy, e = rng.normal(size=(2, 12)) * 2, rng.normal(size=(2, 6)), 1e-6
    grad = gate_grad64(dy, x)
    for i in np.ndindex(x.shape):
        d = np.zeros_like(x)
        d[i] = e
        assert abs(((gate64(x + d) - gate64(x - d)) * dy).sum() / (2 * e) - grad[i]) < 1e-7
    t = torch.from_numpy(x).bfloat16().cuda().requires_grad_()
    (g,) = torch.autograd.grad(micro.silu_mul(t), t, torch.from_numpy(dy).bfloat16().cuda())
    r = gate_grad64(f64(torch.from_numpy(dy).bfloat16()), f64(t))
    assert (np.abs(f64(g) - r) <= 2.0 ** -8 * np.abs(r) + 1e-4).all()


# ---------------------------------------------------------------- runs of them together
def q64(x: np.ndarray, fmt: str) -> np.ndarray:
    g = om.tensor_scale(x) if fmt == "nvfp4" else None
    return om.values(*om.quantize(x, fmt, g), fmt, g)


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_training(fmt):
    """Forward and both gradients: each product of exactly known quantised operands, within check_product's bound."""
    for m, n, k in ((1, 40, 64), (33, 130, 100), (200, 72, 257)):
        x, w = normal(m, k, seed=1).requires_grad_(), normal(n, k, seed=2, std=0.05).requires_grad_()
        dy = normal(n, m, seed=3).t()
        y = micro.micro_linear(x, w, fmt)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        a, b, d = f64(x), f64(w), f64(dy)
        check_product(y.detach(), q64(a, fmt), q64(b, fmt))
        check_product(dx, q64(d, fmt), q64(b.T, fmt))
        check_product(dw, q64(d.T, fmt), q64(a.T, fmt))
    x3 = normal(2, 3, 64, seed=4).requires_grad_()
    w = normal(8, 64, seed=5)
    y = micro.micro_linear(x3, w, fmt)
    assert y.shape == (2, 3, 8)
    y.sum().backward()  # an expanded gradient
    check_product(x3.grad.view(6, 64), q64(np.ones((6, 8)), fmt), q64(f64(w).T, fmt))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_mlp(fmt, tokens):
    """Norm, product, gate and product in a row. Every stage is checked on what the stage before really gave, within its
    own tolerance, so that nothing accumulates into a loose bound; the whole is the same as its parts."""
    hidden, ff = 256, 352
    x, r, nw = normal(tokens, hidden, seed=1), normal(tokens, hidden, seed=2), normal(hidden, seed=3)
    gu = micro.quantize(normal(2 * ff, hidden, seed=4, std=0.05), fmt)
    down = micro.quantize(normal(hidden, ff, seed=5, std=0.05), fmt)
    scales = (torch.full((1,), 0.01, device="cuda"), torch.full((1,), 0.01, device="cuda")) if fmt == "nvfp4" else None
    y, h = micro.micro_mlp(x, r, nw, gu, down, scales=scales)
    s = scales or (None, None)
    n, h2 = micro.rms_norm(x, nw, residual=r, format=fmt, scale=s[0])
    check_coded(n, norm64(f64(x), f64(nw), 1e-5, f64(r))[0], 2.0 ** -18)
    p = micro.micro_matmul(n, gu)

    def v(q):
        return om.values(*stored(q), fmt, None if q.scale is None else float(q.scale))
    check_product(p, v(n), v(gu))
    g = micro.silu_mul(p, format=fmt, scale=s[1])
    check_coded(g, gate64(f64(p)), 2.0 ** -18)
    check_product(y, v(g), v(down))
    assert torch.equal(y, micro.micro_matmul(g, down)) and torch.equal(h, h2)
    micro.check_status()


def test_capture_replay_and_streams():
    """A training step and an inference block captured into two graphs that are replayed at once on two streams, with new
    inputs, between eager steps on the same leaves. (torch refuses the capture of any operator's backward pass while an
    eager autograd graph of the same leaves is alive: theirs is gone before the capture begins.)"""
    fmt = "mxfp8"
    x, w = normal(130, 256, seed=1).requires_grad_(), normal(96, 256, seed=2).requires_grad_()
    dy, nw = normal(130, 96, seed=3), normal(96, seed=4)
    torch.autograd.grad(micro.micro_linear(x, w, fmt), (x, w), dy)

    def step():
        y = micro.micro_linear(x, w, fmt)
        n, _ = micro.rms_norm(y, nw)
        return (n.detach(), *torch.autograd.grad(n, (x, w), dy))

    def block():
        q, h = micro.rms_norm(dy, nw, residual=dy, format="nvfp4", scale=scale)
        return q.dequantize(), h, micro.micro_matmul(q, qw), micro.quantize(dy, "nvfp4").dequantize()

    scale = torch.full((1,), 0.01, device="cuda")
    qw = micro.quantize(normal(64, 96, seed=5), "nvfp4")
    graphs = []
    for f in (step, block):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out, f))
    torch.autograd.grad(micro.micro_linear(x, w, fmt), (x, w), dy)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in (10, 11):
        with torch.no_grad():
            x.copy_(normal(130, 256, seed=seed))
            dy.copy_(normal(130, 96, seed=seed + 1))
        torch.cuda.synchronize()
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, out, f in graphs:
            for a, b in zip(out, f()):
                assert torch.equal(a, b)
    micro.check_status()


def test_product_as_a_threads_first_call():
    """Threads that have not used CUDA yet (autograd's, a server's workers) build tensor maps too."""
    import threading
    (qa, a), (qb, b) = random_operand(40, 300, "nvfp4", 1), random_operand(70, 300, "nvfp4", 2)
    micro.micro_matmul(qa, qb)
    got = []

    def work():
        got.append(micro.micro_matmul(qa, qb))
        got.append(micro.MicroMatmul().make_runner(qa, qb)())
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(got) == 6
    for c in got:
        check_product(c, a, b)


def test_two_products_at_once():
    """Products on two streams at the same time, K split over clusters in both."""
    ops = [(random_operand(m, 4096, fmt, i), random_operand(1000, 4096, fmt, i + 9)) for i, (m, fmt) in
           enumerate(((1, "nvfp4"), (100, "mxfp8")))]
    want = [micro.micro_matmul(a[0], b[0]) for a, b in ops]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    got = [[], []]
    for _ in range(50):
        for i, ((a, b), s) in enumerate(zip(ops, streams)):
            with torch.cuda.stream(s):
                got[i].append(micro.micro_matmul(a[0], b[0]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, t) for t in g)
    micro.check_status()


def test_compare_times_the_formats():
    """compare.py's --micro: the product and the quantisation of a row-major problem in the callers' timing protocol."""
    from cs464_b200.compare import _time_micro
    from cs464_b200.gate import make_inputs
    a, b = make_inputs(64, 384, 512)
    for fmt in FORMATS:
        row = _time_micro(fmt, a, b)
        assert set(row) == {f"{fmt}_us", f"{fmt}_quantize_us"} and all(0 < v < 1e4 for v in row.values())


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_tensors_of_another_device_than_the_current_one():
    x = normal(40, 256).to("cuda:1")
    w = normal(96, 256, seed=1).to("cuda:1")
    with torch.cuda.device(0):
        c = micro.micro_matmul(micro.quantize(x, "nvfp4"), micro.quantize(w, "nvfp4"))
        y, _ = micro.rms_norm(x, w[0])
    with torch.cuda.device(1):
        assert torch.equal(c, micro.micro_matmul(micro.quantize(x, "nvfp4"), micro.quantize(w, "nvfp4")))
        assert torch.equal(y, micro.rms_norm(x, w[0])[0])
    with pytest.raises(ValueError, match="is on cuda:0"):
        micro.rms_norm(x, normal(256))


def test_offsets_past_32_bits():
    """Rows that lie more than 2^31 values into their buffers (6 GB at most here): first and last rows against the same
    rows quantised alone."""
    rows, cols = 70000, 32768
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:2], x[-3:] = normal(2, cols, seed=1), normal(3, cols, seed=2)
    x[2:-3] = 1.0
    q = micro.quantize(x, "mxfp4")
    ends = torch.cat([x[:2], x[-3:]])
    want = micro.quantize(ends, "mxfp4").dequantize()
    d = q.dequantize()
    assert torch.equal(torch.cat([d[:2], d[-3:]]), want) and bool((d[2:-3] == 1).all())
    del d
    qa, a = random_operand(1, cols, "mxfp4", 3)
    c = micro.micro_matmul(qa, q)
    check_product(torch.cat([c[:, :2], c[:, -3:]], 1), a, f64(want))
    c = micro.micro_matmul(q, qa)  # the long side as rows
    check_product(torch.cat([c[:2], c[-3:]]), f64(want), a)


# ---------------------------------------------------------------- derivatives and views that torch keeps lazily
def test_forward_mode_derivatives_are_refused():
    """A dual tensor has no requires_grad: the layers must not take it for a constant, whose tangent is zero."""
    from torch.autograd import forward_ad
    x, w, v, t = normal(4, 64), normal(64, seed=1), normal(8, 64, seed=2), normal(4, 64, seed=3)
    plain = micro.rms_norm(x, w, residual=t)[0], micro.silu_mul(x)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, t)
        dw = forward_ad.make_dual(w, t[0])
        calls = (lambda **kw: micro.rms_norm(d, w, **kw), lambda **kw: micro.rms_norm(x, dw, **kw),
                 lambda **kw: micro.rms_norm(x, w, residual=d, **kw), lambda **kw: micro.silu_mul(d, **kw))
        for call in (*calls, lambda: micro.micro_linear(d, v)):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        for call in calls:
            with pytest.raises(ValueError, match="no gradient"):
                call(format="mxfp8")
        assert torch.equal(micro.rms_norm(x, w, residual=t)[0], plain[0]) and torch.equal(micro.silu_mul(x), plain[1])
    for f in (lambda a: micro.rms_norm(a, w)[0], micro.silu_mul, lambda a: micro.micro_linear(a, v)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (x,), (t,))


def negated(rows, cols, dtype, seed):
    """A tensor whose values torch stores negated, with its flag set: the imaginary part of a conjugate."""
    z = torch.complex(*(normal(rows, cols, dtype=torch.float32, seed=s) for s in (seed, seed + 1)))
    if dtype == torch.float16:
        z = z.to(torch.complex32)
    v = z.conj().imag
    assert v.is_neg() and v.dtype == dtype
    return v


def test_lazily_negated_tensors_keep_their_sign():
    """The kernels read storage: values that torch would negate on the way have to be negated before."""
    v = negated(40, 64, torch.float32, 1)
    for fmt in FORMATS:
        check_quantized(micro.quantize(v, fmt), f64(v))
        check_quantized(micro.quantize(v.t(), fmt), f64(v.t()))
    half = torch.float16
    x, r, w, dy, dh = negated(40, 64, half, 2), negated(40, 64, half, 4), negated(1, 64, half, 6)[0], \
        negated(40, 64, half, 8), negated(40, 64, half, 10)
    plain = [t.resolve_neg() for t in (x, r, w, dy, dh)]
    for got, want in ((micro.rms_norm(x, w, residual=r), micro.rms_norm(plain[0], plain[2], residual=plain[1])),
                      (micro.rms_norm(x, w), micro.rms_norm(plain[0], plain[2])),
                      (micro.rms_norm_backward(dy, x, w, dh=dh), micro.rms_norm_backward(plain[3], plain[0], plain[2], dh=plain[4])),
                      ((micro.silu_mul(x),), (micro.silu_mul(plain[0]),)),
                      ((micro.silu_mul_backward(dy[:, :32], x),), (micro.silu_mul_backward(plain[3][:, :32], plain[0]),)),
                      ((micro.micro_linear(x, r),), (micro.micro_linear(plain[0], plain[1]),)),
                      ((micro.rms_norm(x, w, format="mxfp8")[0].dequantize(half),), (micro.rms_norm(plain[0], plain[2], format="mxfp8")[0].dequantize(half),)),
                      ((micro.silu_mul(x.view(4, 10, 64)),), (micro.silu_mul(plain[0]).view(4, 10, 32),)),
                      (micro.rms_norm(x[:, :1], w[:1]), micro.rms_norm(plain[0][:, :1], plain[2][:1]))):
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    # autograd hands such gradients down, the imaginary part of a complex gradient for one
    leaves = [t.clone().requires_grad_() for t in (plain[0], plain[1])]
    y = micro.micro_linear(*leaves)
    n = micro.rms_norm(leaves[0], plain[2])[0]
    for out, d in ((y, negated(40, 40, half, 12)), (n, dy), (micro.silu_mul(leaves[0]), dy[:, :32])):
        for a, b in zip(*(torch.autograd.grad(out, leaves, g, retain_graph=True, allow_unused=True) for g in (d, d.resolve_neg()))):
            assert (a is None and b is None) or torch.equal(a, b)
    q = micro.quantize(v, "mxfp8")
    with pytest.raises(ValueError, match="negated"):
        micro.dequantize(q, out=negated(40, 64, torch.float32, 14))
    with pytest.raises(ValueError, match="negated"):
        micro.micro_matmul(q, micro.quantize(v[:1], "mxfp8"), out=negated(40, 1, half, 16))
    with pytest.raises(ValueError, match="scale must be"):
        micro.quantize(v, "nvfp4", scale=negated(1, 1, torch.float32, 18)[0])


@pytest.mark.parametrize("g", [2.0 ** -100, (1 + 3 * 2.0 ** -23) * 2.0 ** -100, (1 + 14 * 2.0 ** -23) * 2.0 ** -100, 1.9 * 2.0 ** -100, 1.37 * 2.0 ** -96, 1.6 * 2.0 ** -61, 1.2e-18, 1.1e-7, 3.3e-4, 0.05,
                               1.0 / 448, 1.0, 7.7, 1e20, 1.99 * 2.0 ** 116, 2.0 ** 117])
def test_nvfp4_codes_next_to_every_border(g):
    """What include/b2g_micro.h defines for any scale: 6 g and u = block scale * g as fp32 values, quotients as fp32
    divisions give them, then rounding to the codes. numpy's division is the reference; block maxima lie at and next to the
    borders between block scales, values at and one fp32 step to either side of the borders between codes times u."""
    rng = np.random.default_rng(int(np.float32(g).view(np.uint32)))
    one = np.float32(1)
    g = np.float32(g)
    six = np.float32(6) * g

    def step(v, k):  # k fp32 steps up, for positive v
        return (v.view(np.uint32).astype(np.int64) + k).astype(np.uint32).view(np.float32)
    rows, blocks = 2048, 20
    mids = (om.E4M3[1:] + om.E4M3[:-1]) / 2
    # block maxima: random, and around the middle between two block scales
    with np.errstate(over="ignore"):
        top = np.where(rng.random((rows, blocks)) < 0.5, np.exp(rng.uniform(np.log(0.002), np.log(450.0), (rows, blocks))),
                       rng.choice(mids[:-1], (rows, blocks))).astype(np.float32) * six
        top = np.minimum(top, np.float32(3e38))
        top = step(top, rng.integers(-1, 2, top.shape))
        quotient = np.minimum(top, np.float32(448) * six) / six
    s = om._nearest(quotient.astype(np.float64), om.E4M3)
    u = om.E4M3[s].astype(np.float32) * g
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    x = step(np.minimum(rng.choice(border, (rows, blocks, 16)) * np.maximum(u, 0.5 * g * om.E4M3[1].astype(np.float32))[..., None], top[..., None]),
             rng.integers(-1, 2, (rows, blocks, 16)))
    x = np.minimum(x, top[..., None])
    x[..., 5] = top
    x *= rng.choice([-one, one], x.shape)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        q = np.where(s[..., None] > 0, x / u[..., None], np.float32(0))
    code = om._nearest(np.abs(q).astype(np.float64), om.E2M1) | (np.signbit(x).astype(int) << 3)
    x, code = x.reshape(rows, -1), code.reshape(rows, -1)
    t = torch.from_numpy(x).cuda()
    scale = torch.full((1,), float(g), device="cuda")
    for v in (t, t.t().contiguous().t()):
        c, sb = stored(micro.quantize(v, "nvfp4", scale=scale))
        assert np.array_equal(sb, s), (sb != s).sum()
        assert np.array_equal(c, code), ((c != code).sum(), x[c != code][:3], u.min())


@pytest.mark.parametrize("dtype", HALF)
def test_gate_gradient_of_large_and_small_factors(dtype):
    """Factors whose partial products leave fp32's range where the gradient does not: upstream gradients and ups from tiny
    to a mask's lowest value, gates from -100 up. Bound as in test_gate (the exponential errs by up to 2 + 1.173 * 100 ulps,
    below 2^-15 in all) and as much of a step of fp32's subnormals as the sigmoid is above them; half a step of the type's
    own subnormals. Past the type's largest value the gradient is infinite."""
    top = torch.finfo(dtype).max
    sizes = [1e-30, 1e-10, 1.0, 1e10, 1e20, 1e30, top] if dtype == torch.bfloat16 else [1e-4, 1.0, 300.0, top]
    g = torch.tensor([-100.0, -95.0, -88.0, -70.0, -60.0, -20.0, -3.0, -1.25, 0.0, 0.5, 2.375, 20.0, 100.0])
    g, u, d = (t.reshape(1, -1) for t in torch.meshgrid(g, torch.tensor([s * f for s in sizes for f in (1, -1)]), torch.tensor(sizes), indexing="ij"))
    x, dy = torch.cat([g, u], 1).to(dtype).cuda(), d.to(dtype).cuda()
    a, b = f64(dy), f64(x)
    n = a.shape[1]
    g, u = b[:, :n], b[:, n:]
    s = 1 / (1 + np.exp(-g))
    terms = [a * u * s * (1 + np.abs(g) * (1 - s)), a * g * s]
    ref = [a * u * s * (1 + g * (1 - s)), a * g * s]
    got = f64(micro.silu_mul_backward(dy, x))
    for y, r, t in zip((got[:, :n], got[:, n:]), ref, terms):
        bound = half_step(dtype) * np.abs(r) + (2.0 ** -15 + 2.0 ** -147 / s) * np.abs(t) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
        out = np.abs(r) > 1.01 * top
        near = np.abs(r) + bound > 0.99 * top  # may round to the largest value or to an infinity
        assert (np.isinf(y[out]) & (np.sign(y[out]) == np.sign(r[out]))).all()
        assert (np.abs(y - r)[~near] <= bound[~near]).all() and not np.isnan(y).any()


# ---------------------------------------------------------------- both families on one stream
def test_products_and_gemms_in_turn():
    """Products and fp16 GEMMs follow one another as programmatic dependents, each with tensor memory of its own (half of it
    or all, one or two CTAs to an SM), back to back and from a graph: everything is what each gives alone."""
    from cs464_b200.gate import make_inputs
    from cs464_b200.matmul import B200Matmul, MatmulConfig
    runs = []
    for cfg in (MatmulConfig(128, 256, 64, num_stages=2, PERSISTENT=0), MatmulConfig(128, 64, 64, num_stages=4, PERSISTENT=0),
                MatmulConfig(256, 256, 64, num_stages=4, CLUSTER=2), MatmulConfig(16, 128, 128, num_stages=4, SPLIT_K=4)):
        m = 16 if cfg.BLOCK_M == 16 else 512
        runs.append(B200Matmul(cfg).make_runner(*make_inputs(m, 9600, 512)))
    for fmt, m, n, k in (("mxfp8", 128, 9600, 512), ("nvfp4", 16, 19200, 256), ("mxfp4", 1, 4096, 4096), ("nvfp4", 512, 9600, 512)):
        runs.append(micro.MicroMatmul().make_runner(random_operand(m, k, fmt, 1)[0], random_operand(n, k, fmt, 2)[0]))
    want = []
    for r in runs:
        want.append(r().clone())
        torch.cuda.synchronize()
    order = torch.randint(len(runs), (400,), generator=torch.Generator().manual_seed(0)).tolist()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in order:
            runs[i]()

    def eager():
        for i in order:
            runs[i]()
    for go in (eager, graph.replay):
        for r in runs:
            r.c.zero_()
        go()
        torch.cuda.synchronize()
        for r, w in zip(runs, want):
            r.raise_on_status()
            assert torch.equal(r.c, w)


# ---------------------------------------------------------------- bounded waits that run out
TIMEOUTS = {0x101, 0x102, 0x103}


def test_expired_wait_reports_status_and_stores_nothing():
    """A product whose epilogue waits tens of microseconds for its tile, its waits limited to one: some wait runs out, the
    kernel ends, C stays as it was, the status word says so, and the next products are right."""
    (qa, a), (qb, b) = random_operand(128, 16384, "mxfp8", 1), random_operand(12800, 16384, "mxfp8", 2)
    run = micro.MicroMatmul(wait_limit_us=1).make_runner(qa, qb)
    for _ in range(2):  # cleared, the same runner gives up again rather than hanging
        run.c.fill_(7.0)
        run()
        torch.cuda.synchronize()
        assert run.device_status() in TIMEOUTS
        assert bool((run.c == 7).all())
        with pytest.raises(RuntimeError, match="status 0x10"):
            run.raise_on_status()
        run.status.zero_()
    ok = micro.MicroMatmul().make_runner(qa, qb)
    c = ok()
    ok.raise_on_status()
    check_product(c, a, b)


@pytest.mark.parametrize("k", [1, 128, 384, 1500])
@pytest.mark.parametrize("fmt", FORMATS)
def test_expired_waits_of_short_products(fmt, k):
    """Few K blocks: all copies are under way before any role gives up, and land before the CTA ends. Launches that gave up
    are followed at once by products whose ring lies in the same shared memory; a launch that made it stored its result."""
    (qa, a), (qb, b) = random_operand(128, k, fmt, 1), random_operand(12800, k, fmt, 2)
    run, ok = micro.MicroMatmul(wait_limit_us=1).make_runner(qa, qb), micro.MicroMatmul().make_runner(qa, qb)
    want = ok().clone()
    check_product(want, a, b)
    for _ in range(20):
        run()
        assert torch.equal(ok(), want)
    assert run.device_status() in TIMEOUTS | {0}
    ok.raise_on_status()


def test_wait_limit_is_refused_for_pairs_and_splits():
    from cs464_b200 import _abi
    (qa, _), (qb, _), (qc, _) = (random_operand(m, 512, "mxfp8", m) for m in (300, 400, 16))
    for a in (qa, qc):  # pairs; splits of a cluster
        with pytest.raises(_abi.Unsupported, match="wait_limit_single_cta_only"):
            micro.MicroMatmul(wait_limit_us=10).make_runner(a, qb)
        micro.MicroMatmul().make_runner(a, qb)()
    with pytest.raises(_abi.B2GError, match="wait_limit_us"):
        micro.MicroMatmul(wait_limit_us=-1).make_runner(qa, qb)
    micro.check_status()


FAR = 540_000_000  # five rows this many values apart reach past 2^31 values


def test_far_rows_of_every_input():
    """Views whose last rows lie past 2^31 values (a buffer of 4.3 GB): every operator's inputs, by rows and through
    transposes, aligned and not, against contiguous copies."""
    for shift in (0, 1):
        step = FAR + shift
        base = torch.empty(4 * step + 2048, dtype=torch.bfloat16, device="cuda")
        def far(cols, seed, at):
            v = base.as_strided((5, cols), (step, 1), at)
            v.copy_(normal(5, cols, seed=seed))
            return v, v.clone()
        (x, cx), (r, cr) = far(520, 1, 0), far(520, 2, 520)
        (d, cd), w = far(260, 3, 1040 + 8 * shift), normal(520, seed=4)
        for fmt in FORMATS:
            for a, b in ((x, cx), (x.t(), cx.t())):
                p, q = micro.quantize(a, fmt), micro.quantize(b, fmt)
                assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
                assert torch.equal(p.scale, q.scale) if fmt == "nvfp4" else True
        for a, b in ((micro.rms_norm(x, w, residual=r), micro.rms_norm(cx, w, residual=cr)),
                     (micro.rms_norm_backward(r, x, w, dh=x), micro.rms_norm_backward(cr, cx, w, dh=cx)),
                     ((micro.silu_mul(x), micro.silu_mul_backward(d, x)), (micro.silu_mul(cx), micro.silu_mul_backward(cd, cx)))):
            assert all(torch.equal(s, t) for s, t in zip(a, b))
        q = micro.quantize(cx, "nvfp4")
        micro.dequantize(q, out=x)
        assert torch.equal(x, q.dequantize())


@pytest.mark.parametrize("ldc", [8, 1])
def test_far_rows_of_products(ldc):
    """C with its last rows past 2^31 values, of few rows (single CTAs), of many (pairs), and of few pairs' tiles with a
    long K (splits); nothing else of the buffer is written."""
    base = torch.zeros(2 ** 31 + 2 ** 25, dtype=torch.bfloat16, device="cuda")
    for m, n, k in ((100, 264, 300), (300, 264, 300), (510, 200, 9000), (130, 5000, 96), (513, 2050, 9300)):
        step = (2 ** 31 // (m - 1) // 8 + 1) * 8 + (1 if ldc == 1 else 0)
        out = base.as_strided((m, n), (step, 1))
        (qa, a), (qb, b) = random_operand(m, k, "nvfp4", 1), random_operand(n, k, "nvfp4", 2, std=0.05)
        micro.micro_matmul(qa, qb, out=out)
        check_product(out, a, b)
        out.zero_()
        assert not base.any()
    micro.check_status()


def test_outputs_past_32_bits():
    """Codes past 2^31 bytes and outputs past 2^31 values that the operators allocate themselves (up to 40 GB here): first
    and last rows against the same rows alone."""
    rows, cols = 70000, 32768
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:2], x[-3:] = normal(2, cols, seed=1), normal(3, cols, seed=2)
    w = normal(cols, seed=3)

    def ends(t):
        return torch.cat([t[:2], t[-3:]])
    few = ends(x)
    q = micro.quantize(x, "mxfp8")
    assert torch.equal(ends(q.codes), micro.quantize(few, "mxfp8").codes)
    want = f64(micro.quantize(few, "mxfp8").dequantize())
    d = q.dequantize()
    assert torch.equal(ends(d), micro.quantize(few, "mxfp8").dequantize()) and bool((d[2:-3] == 1).all())
    del d
    for m in (1, 200):  # single CTAs, pairs
        qa, a = random_operand(m, cols, "mxfp8", 4)
        check_product(ends(micro.micro_matmul(qa, q).t()), want, a)
        check_product(ends(micro.micro_matmul(q, qa)), want, a)
    del q
    y, h = micro.rms_norm(x, w, residual=x)
    fy, fh = micro.rms_norm(few, w, residual=few)
    assert torch.equal(ends(h), fh) and torch.equal(ends(y), fy) and torch.equal(y[2], y[-4])
    del y, h
    n, fn = micro.rms_norm(x, w, format="mxfp8")[0], micro.rms_norm(few, w, format="mxfp8")[0]
    assert torch.equal(ends(n.codes), fn.codes)
    del n
    dx, _ = micro.rms_norm_backward(x, x, w)
    assert torch.equal(ends(dx), micro.rms_norm_backward(few, few, w)[0])
    del dx
    dx = micro.silu_mul_backward(x[:, :cols // 2], x)
    assert torch.equal(ends(dx), micro.silu_mul_backward(few[:, :cols // 2], few))
    del dx
    wide = x[:, None, :].expand(rows, 2, cols).reshape(rows, 2 * cols)
    y = micro.silu_mul(wide)
    assert torch.equal(ends(y), micro.silu_mul(ends(wide)))
    assert torch.equal(ends(micro.silu_mul(wide, format="mxfp8").codes), micro.silu_mul(ends(wide), format="mxfp8").codes)
    micro.check_status()


# ---------------------------------------------------------------- calls that the documentation allows
@pytest.mark.parametrize("fmt", FORMATS)
def test_wrapped_codes_in_wider_rows(fmt):
    """MicroTensors made of another program's bytes: rows further apart than they have to be, anything between them,
    scales inside a larger buffer."""
    for m, n, k in ((5, 130, 100), (300, 264, 1100), (16, 4096, 1500)):
        wrapped, values = [], []
        for rows, seed in ((m, 1), (n, 2)):
            q, v = random_operand(rows, k, fmt, seed)
            pitch = q.codes.shape[1]
            wide = torch.full((rows, pitch + 96), 0x7F, dtype=torch.uint8, device="cuda")
            used = k if fmt == "mxfp8" else (k + 1) // 2
            wide[:, :used] = q.codes[:, :used]
            buf = torch.full((q.scales.numel() + 48,), 0xFF, dtype=torch.uint8, device="cuda")
            buf[16:-32] = q.scales
            w = micro.MicroTensor(wide[:, :pitch], buf[16:-32], (rows, k), fmt, q.scale)
            assert torch.equal(w.dequantize(torch.float32), q.dequantize(torch.float32))
            assert torch.equal(w.scale_tiles().view(torch.uint8), q.scale_tiles().view(torch.uint8))
            if fmt == "mxfp8":
                assert torch.equal(w.code_values().view(torch.uint8), q.code_values().view(torch.uint8))
            wrapped.append(w)
            values.append(v)
        check_product(micro.micro_matmul(*wrapped), *values)
        check_product(micro.MicroMatmul().make_runner(*wrapped)(), *values)
    micro.check_status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_broadcast_inputs(fmt):
    """Inputs whose rows or columns are one and the same in memory."""
    row, col = normal(1, 200, seed=1), normal(200, 1, seed=2)
    for x in (row.expand(70, 200), col.expand(200, 70), col.expand(200, 70).t(), row.t().expand(200, 70).t(), row[:, :1].expand(70, 200)):
        check_quantized(micro.quantize(x, fmt), f64(x))
    x = row.expand(70, 200)
    assert torch.equal(micro.silu_mul(x), micro.silu_mul(x.contiguous()))
    assert torch.equal(micro.silu_mul_backward(col[:100].t().expand(70, 100), x), micro.silu_mul_backward(col[:100].t().repeat(70, 1), x.contiguous()))
    for got, want in ((micro.rms_norm_backward(x, x, row[0], dh=x), micro.rms_norm_backward(*[x.contiguous()] * 2, row[0], dh=x.contiguous())),
                      (micro.rms_norm(x, row[0, :1].expand(200), residual=x), micro.rms_norm(x.contiguous(), row[0, :1].repeat(200), residual=x.contiguous()))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("fmt", FORMATS)
def test_mlp_of_odd_sizes_and_no_tokens(fmt, dtype):
    hidden, ff = 200, 136
    r = normal(2, 3, hidden, dtype=dtype, seed=1)
    nw = normal(hidden, dtype=dtype, seed=3)
    gu, down = micro.quantize(normal(2 * ff, hidden, seed=4, std=0.05), fmt), micro.quantize(normal(hidden, ff, seed=5, std=0.05), fmt)
    scales = (torch.full((1,), 0.01, device="cuda"),) * 2 if fmt == "nvfp4" else None
    y, h = micro.micro_mlp(r, None, nw, gu, down, scales=scales)
    assert y.shape == h.shape == (2, 3, hidden) and h is r and y.dtype == dtype
    flat, _ = micro.micro_mlp(r.view(6, hidden), None, nw, gu, down, scales=scales)
    assert torch.equal(y.view(6, hidden), flat)
    for i in range(6):  # a token's result does not depend on its company beyond the order of K splits, which tiles share
        one, _ = micro.micro_mlp(r.view(6, hidden)[i:i + 1], None, nw, gu, down, scales=scales)
        assert torch.equal(one[0], flat[i])
    y, h = micro.micro_mlp(r[:0], r[:0], nw, gu, down, scales=scales)
    assert y.shape == h.shape == (0, 3, hidden)
    x = normal(0, hidden, dtype=dtype).requires_grad_()
    w = nw.clone().requires_grad_()
    n, _ = micro.rms_norm(x, w)
    n.sum().backward()
    assert x.grad.shape == x.shape and (w.grad == 0).all()
    a, b = normal(0, 64, dtype=dtype).requires_grad_(), normal(40, 64, dtype=dtype).requires_grad_()
    micro.micro_linear(a, b, fmt).sum().backward()
    assert a.grad.shape == a.shape and (b.grad == 0).all()
    micro.check_status()
