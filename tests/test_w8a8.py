"""The 8-bit serving operators (``pi05_pytorch_fast_b200.w8a8``) against plain
implementations in 64 bits, and their refusals.

Tolerances are derived from the arithmetic that the operators promise: fp32
inside, exact int32 sums, one rounding to the output's type.  u(dtype) is the
unit roundoff 2^-p of that rounding."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from pi05_pytorch_fast_b200 import _native as nat
from pi05_pytorch_fast_b200 import prefix_lm as plm
from pi05_pytorch_fast_b200 import snapflow as sf
from pi05_pytorch_fast_b200 import w8a8

DEV = "cuda:0"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38, torch.float32: 1e-38}  # half a step of the subnormals


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def on_gpu(t):
    return None if t is None else t.to(DEV)


def within(got, want, tol):
    """|got - want| <= tol elementwise, got on any device, NaN nowhere."""
    err = (got.detach().cpu().double() - want).abs()
    assert torch.isfinite(err).all()
    over = err - tol
    assert (over <= 0).all(), f"worst {err[over > 0].max():.3g}, {int((over > 0).sum())} of {err.numel()} too far"


def check_rows(codes, scale, y, tol_y):
    """codes x scale is y to within half a step of its row and what y itself may be off."""
    amax = y.abs().amax(-1)
    off = tol_y.amax(-1)
    within(scale, amax / 127, off / 127 + 2.0 ** -22 * amax / 127)
    assert int(codes.abs().max()) <= 127
    step = (amax / 127 + off / 127)[..., None]
    within(codes.cpu().double() * scale.cpu().double()[..., None], y, 0.5 * step * (1 + 2.0 ** -10) + tol_y + off[..., None])


# ------------------------------------------------------------------ norm
NORM_CASES = [
    # batch, tokens, h, dtype, delta, gate, gain and shift for each observation
    (1, 1, 2048, torch.float16, True, False, False),
    (8, 50, 1024, torch.bfloat16, True, True, True),
    (3, 5, 1152, torch.bfloat16, False, False, True),
    (2, 3, 1, torch.float32, True, False, False),
    (2, 7, 97, torch.float16, True, True, True),
    (1, 9, 1155, torch.bfloat16, True, True, False),
    (2, 2, 8192, torch.float16, True, False, False),
    (1, 2, 16385, torch.float16, True, False, True),
    (2, 1, 33000, torch.bfloat16, True, True, True),
    (5, 3, 264, torch.float32, True, True, True),
]


def norm_inputs(b, t, h, dtype, delta, gate, per_obs, seed=0):
    g = gen(seed)
    x = (randn(g, b, t, h) * torch.exp(0.6 * randn(g, h))).to(dtype)
    d = (randn(g, b, t, h) * 2).to(dtype) if delta else None
    ga = randn(g, b, h).to(dtype) if gate else None
    gain = (1 + 0.1 * randn(g, *((b, h) if per_obs else (h,)))).float()
    shift = (0.1 * randn(g, b, h)).float() if per_obs else None
    return x, d, ga, gain, shift


def norm64(x, delta, gate, gain, shift, eps):
    """(total, y, how far y may be off) in 64 bits."""
    def wide(p):
        return p.double() if p.dim() == 1 else p.double()[:, None]

    z, mag = x.double(), x.double().abs()
    if delta is not None:
        d = delta.double() * (1 if gate is None else wide(gate))
        z, mag = z + d, mag + d.abs()
    rstd = (z.square().mean(-1, keepdim=True) + eps).rsqrt()
    y = z * rstd * wide(gain)
    tol = 2.0 ** -17 * y.abs() + 2.0 ** -21 * mag * rstd * wide(gain).abs()
    if shift is not None:
        y, tol = y + wide(shift), tol + 2.0 ** -17 * wide(shift).abs()
    return z, y, tol, mag


@pytest.mark.gpu
@pytest.mark.parametrize("case", NORM_CASES)
def test_rms_norm_quant(case):
    x, d, ga, gain, shift = norm_inputs(*case)
    z, y, tol, mag = norm64(x, d, ga, gain, shift, 1e-6)
    xg = on_gpu(x)
    codes, scale, total = w8a8.rms_norm_quant(xg, on_gpu(gain), 1e-6, delta=on_gpu(d), gate=on_gpu(ga), shift=on_gpu(shift))
    if d is None:
        assert total is xg
    else:
        u = U[x.dtype]
        within(total, z, u * z.abs() + 2.0 ** -22 * mag + TINY[x.dtype])
    assert codes.dtype == torch.int8 and codes.shape == x.shape and scale.shape == x.shape[:-1]
    assert codes.stride(-1) == 1 and (x.shape[1] == 1 or codes.stride(-2) % 16 == 0)
    check_rows(codes, scale, y, tol)


MANY_ROW_CASES = [
    # more rows than CTAs of the kernel for them: a CTA takes several, of more than one observation
    (1001, 5, 64, torch.float16, True, True, True),
    (2003, 3, 512, torch.bfloat16, True, True, True),
    (31, 129, 2048, torch.float16, True, False, True),
    (9, 555, 1152, torch.bfloat16, False, False, True),
    (7, 100, 24576, torch.bfloat16, True, True, True),
    (5, 601, 328, torch.float32, True, True, False),
    (3, 701, 1026, torch.float16, True, True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", MANY_ROW_CASES)
def test_rms_norm_quant_many_rows(case):
    x, d, ga, gain, shift = norm_inputs(*case, seed=1)
    z, y, tol, mag = norm64(x, d, ga, gain, shift, 1e-6)
    codes, scale, total = w8a8.rms_norm_quant(on_gpu(x), on_gpu(gain), 1e-6, delta=on_gpu(d), gate=on_gpu(ga), shift=on_gpu(shift))
    if d is not None:
        within(total, z, U[x.dtype] * z.abs() + 2.0 ** -22 * mag + TINY[x.dtype])
    check_rows(codes, scale, y, tol)
    again = w8a8.rms_norm_quant(on_gpu(x), on_gpu(gain), 1e-6, delta=on_gpu(d), gate=on_gpu(ga), shift=on_gpu(shift))
    assert torch.equal(codes, again[0]) and torch.equal(scale, again[1])


@pytest.mark.gpu
def test_rms_norm_quant_takes_strided_and_misaligned_rows():
    g = gen(3)
    big = on_gpu(randn(g, 6, 4, 2 * 520 + 3).half())
    gain = on_gpu(1 + 0.1 * randn(g, 512).float())
    for lo in (0, 1, 8, 523):  # aligned or not; the row stride is odd
        x, d = big[:, :2, lo:lo + 512], big[:, 2:, lo:lo + 512]
        got = w8a8.rms_norm_quant(x, gain, delta=d)
        want = w8a8.rms_norm_quant(x.contiguous(), gain, delta=d.contiguous())
        _, y, tol, _ = norm64(x.cpu(), d.cpu(), None, gain.cpu(), None, 1e-6)
        check_rows(got[0], got[1], y, tol)
        assert torch.equal(got[2], want[2])


@pytest.mark.gpu
def test_rows_that_are_zero_tiny_or_not_finite():
    x = torch.zeros(6, 256)
    x[1] = 1e-41                       # scale far below the smallest normal number
    x[2, 3], x[3, 4], x[4, 5] = math.inf, math.nan, -math.inf
    x[5] = torch.linspace(-1, 1, 256)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        codes, scale = w8a8.quantize(x.to(dtype).to(DEV))
        codes, scale = codes.cpu(), scale.cpu()
        assert scale[0] == 0 and not codes[0].any()
        if dtype == torch.float32:
            assert scale[1] > 0 and (codes[1].abs() <= 127).all()
        assert not torch.isfinite(scale[2:5]).any() and not codes[2:5].any()
        assert not torch.isfinite(w8a8.dequantize(codes.to(DEV), scale.to(DEV), torch.float32)[2:5]).any()
        check_rows(codes[5:], scale[5:], x[5:].to(dtype).double(), torch.zeros(1, 256, dtype=torch.float64))
    # the norm of a zero row is its shift
    shift = on_gpu(torch.linspace(-2, 2, 256)[None])
    codes, scale, _ = w8a8.rms_norm_quant(torch.zeros(1, 3, 256, device=DEV), torch.ones(1, 256, device=DEV), shift=shift)
    check_rows(codes, scale, shift.cpu().double().expand(1, 3, 256), torch.full((1, 3, 256), 1e-6, dtype=torch.float64))


# ------------------------------------------------------------- quantise
def gelu64(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,h", [(1, 1), (1, 16), (3, 17), (5, 2048), (2, 4096), (7, 4304), (2, 16384), (1, 16388), (1, 40000)])
@pytest.mark.parametrize("geglu", [False, True])
def test_quantize(m, h, dtype, geglu):
    g = gen(m * 100003 + h)
    both = (3 * randn(g, m, 2 * h)).to(dtype)
    x, up = both[:, :h], both[:, h:]  # halves of one product: strided rows
    v = x.double()
    tol = torch.zeros_like(v)
    if geglu:
        v = gelu64(v) * up.double()
        # u = 2 sqrt(2/pi)(x + 0.044715 x^3) is off by 2^-21 |u|, which exp turns into a relative
        # error of that size wherever exp(-u) is not negligible next to 1 (|u| < 88)
        u = 1.6 * (x.double().abs() + 0.044715 * x.double().abs() ** 3).clamp(max=88)
        tol = v.abs() * (2.0 ** -20 + 2.0 ** -20 * u) + 1e-37 * up.double().abs()
    big = on_gpu(both)
    codes, scale = w8a8.quantize(big[:, :h], up=big[:, h:] if geglu else None)
    check_rows(codes, scale, v, tol)
    back = w8a8.dequantize(codes, scale, dtype)
    assert back.is_contiguous() and back.dtype == dtype
    exact = codes.cpu().double() * scale.cpu().double()[:, None]
    within(back, exact, (U[dtype] + 2.0 ** -23) * exact.abs() + TINY[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,h", [(5005, 64), (6007, 512), (4003, 2048), (601, 24576), (2003, 2394)])
def test_quantize_many_rows(m, h, dtype):
    """More rows than CTAs: each row as if it were alone, plain and of the GeGLU."""
    g = gen(m)
    both = (2 * randn(g, m, 2 * h)).to(dtype)
    big = on_gpu(both)
    codes, scale = w8a8.quantize(big[:, :h])
    want_codes, want_scale = codes_plain(both[:, :h])
    assert torch.equal(codes.cpu(), want_codes) and torch.equal(scale.cpu(), want_scale)
    x, up = both[:, :h].double(), both[:, h:].double()
    u = 1.6 * (x.abs() + 0.044715 * x.abs() ** 3).clamp(max=88)  # as in test_quantize
    v = gelu64(x) * up
    check_rows(*w8a8.quantize(big[:, :h], up=big[:, h:]), v, v.abs() * (2.0 ** -20 + 2.0 ** -20 * u) + 1e-37 * up.abs())


def codes_plain(x):
    """(codes, scale) in the fp32 steps that the operator defines."""
    x = x.float()
    scale = x.abs().amax(-1) * (torch.tensor(1.0) / 127)
    return (x / scale[:, None]).round().clamp(-127, 127).to(torch.int8), scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h", [17, 18, 20, 64, 2048, 2050])
def test_quantize_codes_at_ties(h, dtype):
    """Rows of every mantissa of the largest element (of 1,024 in fp32), with
    elements at its half, quarter and other multiples, and (fp32) at and next
    to every tie: the codes of the division, bit for bit."""
    g = gen(h)
    rows = 128 if dtype == torch.bfloat16 else 1024
    top = (1 + torch.arange(rows) / rows) * 2.0 ** torch.randint(-8, 9, (rows,), generator=g)
    x = (2 * torch.rand(rows, h, generator=g) - 1) * top[:, None]
    share = torch.tensor([1, -0.5, 0.5, 0.25, -0.75, 0.125, 0.375])
    x[:, :7] = top[:, None] * share
    if dtype == torch.float32:
        tie = (torch.randint(0, 127, (rows, h - 7), generator=g) + 0.5) * codes_plain(x)[1][:, None]
        beside = torch.randint(-1, 2, tie.shape, generator=g, dtype=torch.int32)
        tie = (tie.view(torch.int32) + beside).view(torch.float32) * (2 * torch.randint(0, 2, tie.shape, generator=g) - 1)
        x[:, 7:] = torch.where(tie.abs() <= top[:, None], tie, x[:, 7:])
    x = x.to(dtype)
    want_codes, want_scale = codes_plain(x)
    for n in (rows, 5):  # many rows and few take different kernels
        codes, scale = w8a8.quantize(on_gpu(x[:n].contiguous()))
        assert torch.equal(scale.cpu(), want_scale[:n])
        assert torch.equal(codes.cpu(), want_codes[:n])


# --------------------------------------------------------------- linear
LINEAR_CASES = [
    # m, n, k, dtype, bias
    (1, 1, 1, torch.float32, True),
    (1, 2560, 2048, torch.float16, False),
    (2, 130, 64, torch.bfloat16, True),
    (7, 33, 97, torch.float16, True),
    (16, 256, 4096, torch.bfloat16, False),
    (17, 1000, 1155, torch.float16, False),
    (50, 1024, 4096, torch.bfloat16, True),
    (65, 129, 2064, torch.float32, False),
    (129, 257, 272, torch.float16, True),
    (400, 1024, 1024, torch.bfloat16, False),
    (512, 1152, 4304, torch.bfloat16, True),
    (600, 520, 130, torch.float16, False),
    (1000, 999, 144, torch.bfloat16, True),
    (1111, 2048, 528, torch.float16, False),
    (300, 130, 16384, torch.float16, False),
    (3, 70, 131071, torch.float32, False),
]


def codes_rows(g, m, k, low=-127):
    ld = (k + 15) // 16 * 16
    return torch.randint(low, 128, (m, ld), generator=g, dtype=torch.int8)[:, :k]


def linear64(a, sa, w, sw, bias):
    acc = a.double() @ w.double().T  # exact: below 2^53
    prod = acc * sa.double()[:, None] * sw.double()
    return (prod if bias is None else prod + bias.double()), prod.abs() + (0 if bias is None else bias.double().abs())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,dtype,bias", LINEAR_CASES)
def test_linear(m, n, k, dtype, bias):
    g = gen(m + n + k)
    a, w = codes_rows(g, m, k), codes_rows(g, n, k, low=-128)
    sa, sw = (torch.rand(m, generator=g) * 0.02 + 0.001), (torch.rand(n, generator=g) * 0.002 + 0.0001)
    bi = randn(g, n).to(dtype) if bias else None
    want, mag = linear64(a, sa, w, sw, bi)
    pad = torch.full((2, max(m, n), (k + 15) // 16 * 16), 77, dtype=torch.int8, device=DEV)  # the pad is not read as K
    ag, wg = pad[0, :m, :k], pad[1, :n, :k]
    ag.copy_(a), wg.copy_(w)
    y = w8a8.linear(ag, on_gpu(sa), w8a8.Int8Weight(wg, on_gpu(sw)), bias=on_gpu(bi), dtype=dtype)
    assert y.shape == (m, n) and y.dtype == dtype and y.is_contiguous()
    within(y, want, U[dtype] * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -22 * mag + TINY[dtype])
    # the same call gives the same bits
    assert torch.equal(y, w8a8.linear(ag, on_gpu(sa), w8a8.Int8Weight(wg, on_gpu(sw)), bias=on_gpu(bi), dtype=dtype))
    assert nat.device_error() == 0


# shapes of the kernels for many tokens and many channels: rows of y at multiples of 16 bytes (TMA stores), of 8, 4 and 2;
# token counts that end inside a tile; several tiles a pair of CTAs and less than one
LARGE_LINEAR_CASES = [
    (4097, 4096, 400, torch.float16, True),
    (3003, 3004, 144, torch.float16, True),
    (3003, 3002, 272, torch.bfloat16, False),
    (3003, 3001, 130, torch.float16, True),
    (3003, 3000, 400, torch.float32, True),
    (3003, 3002, 144, torch.float32, False),
    (3003, 3001, 144, torch.float32, True),
    (9000, 1029, 528, torch.bfloat16, True),
    (1600, 2048, 2064, torch.float16, False),
    (3, 5001, 160, torch.float16, True),
    (16, 4999, 130, torch.bfloat16, False),
    (8, 4737, 64, torch.float32, True),
    (2, 130, 4100, torch.bfloat16, True),
    (11, 257, 4097, torch.float16, True),
    (20, 64, 1024, torch.float16, True),
    (40, 257, 2064, torch.bfloat16, True),
]


def test_linear_cases_reach_every_kernel():
    plans = [nat.gemm8_plan(m, n, k) for m, n, k, _, _ in LINEAR_CASES + LARGE_LINEAR_CASES]
    assert {p["kernel"] for p in plans} == {"few", "few_wide", "few_deep", "tile", "pair"}
    assert {p["split"] for p in plans if p["kernel"] == "tile"} == {1, 2, 4, 8}
    assert {p["tok_tile"] for p in plans if p["kernel"].startswith("few")} == {8, 16}
    pairs = [(n * torch.finfo(t).bits // 8 % 16, t) for (m, n, k, t, _), p in
             zip(LARGE_LINEAR_CASES, plans[len(LINEAR_CASES):]) if p["kernel"] == "pair"]
    assert {r for r, t in pairs if t != torch.float32} >= {0, 2, 4, 8} and {r for r, t in pairs if t == torch.float32} >= {0, 4, 8}
    for args in ((0, 8, 8), (4, 0, 8), (4, 8, 131072)):
        with pytest.raises(nat.W4A4Error, match="plan query"):
            nat.gemm8_plan(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,dtype,bias", LARGE_LINEAR_CASES)
def test_linear_large(m, n, k, dtype, bias):
    g = gen(m + n + k)
    a, w = on_gpu(codes_rows(g, m, k)), on_gpu(codes_rows(g, n, k, low=-128))
    sa, sw = (torch.rand(m, generator=g) * 0.02 + 0.001), (torch.rand(n, generator=g) * 0.002 + 0.0001)
    sa[m // 2] = 0
    bi = on_gpu(randn(g, n).to(dtype)) if bias else None
    want, mag = linear64(a, on_gpu(sa), w, on_gpu(sw), bi)
    weight = w8a8.Int8Weight(w, on_gpu(sw))
    y = w8a8.linear(a, on_gpu(sa), weight, bias=bi, dtype=dtype)
    err = (y.double() - want).abs()
    tol = U[dtype] * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -22 * mag + TINY[dtype]
    assert torch.isfinite(err).all() and (err <= tol).all(), f"{int((err > tol).sum())} of {err.numel()} too far"
    assert torch.equal(y, w8a8.linear(a, on_gpu(sa), weight, bias=bi, dtype=dtype))
    assert nat.device_error() == 0


@pytest.mark.gpu
def test_linear_takes_leading_dimensions_and_unaligned_rows():
    g = gen(5)
    x = on_gpu(randn(g, 2, 3, 5, 96).bfloat16())
    weight = w8a8.pack_weight(on_gpu(randn(g, 40, 96).float()))
    codes, scale = w8a8.quantize(x)
    y = w8a8.linear(codes, scale, weight)
    assert y.shape == (2, 3, 5, 40)
    flat = w8a8.linear(codes.view(30, 96), scale.view(30), weight)
    assert torch.equal(y.view(30, 40), flat)
    # rows at odd strides and from odd bases are laid out for the call
    odd = torch.empty(31, 97, dtype=torch.int8, device=DEV)[1:, 1:]
    odd.copy_(codes.view(30, 96))
    assert torch.equal(w8a8.linear(odd, scale.view(30), weight), flat)
    one = torch.empty(97, dtype=torch.int8, device=DEV)[1:]
    one.copy_(codes.view(30, 96)[7])
    assert torch.equal(w8a8.linear(one, scale.view(30)[7:8].clone(), weight), flat[7])
    assert w8a8.linear(codes.view(30, 96)[:0], scale.view(30)[:0], weight).shape == (0, 40)


@pytest.mark.gpu
def test_linear_rows_that_are_not_finite_stay_apart():
    g = gen(6)
    x = randn(g, 5, 128).float()
    x[2, 7] = math.nan
    x[3] = 0
    weight = w8a8.pack_weight(on_gpu(randn(g, 24, 128).float()))
    codes, scale = w8a8.quantize(x.to(DEV))
    y = w8a8.linear(codes, scale, weight, dtype=torch.float32).cpu()
    assert y[2].isnan().all() and (y[3] == 0).all() and torch.isfinite(y[[0, 1, 4]]).all()


@pytest.mark.gpu
def test_linear_in_eight_bits_is_near_the_float_product():
    """pack_weight + quantize + linear against the product of the values
    themselves: each operand is off by at most half a step, uniformly, so the
    sum over K is off by about sqrt(K / 12) of a step product."""
    g = gen(8)
    m, n, k = 33, 48, 1024
    x, w = randn(g, m, k).float(), randn(g, n, k).float()
    codes, scale = w8a8.quantize(on_gpu(x))
    weight = w8a8.pack_weight(on_gpu(w))
    y = w8a8.linear(codes, scale, weight, dtype=torch.float32).cpu().double()
    want = x.double() @ w.double().T
    sx, sw = x.abs().amax(1).double()[:, None] / 127, w.abs().amax(1).double()[None] / 127
    sigma = ((sx ** 2 * w.double().square().sum(1)[None] + sw ** 2 * x.double().square().sum(1)[:, None]) / 12).sqrt()
    assert ((y - want).abs() < 6 * sigma).all()


# ---------------------------------------------------------------- cache
def cache_state(g, b, cap, h, w):
    codes = torch.randint(-127, 128, (2, b, cap, h, w), generator=g, dtype=torch.int8)
    scale = torch.rand(2, b, h, cap // 16, generator=g) * 0.02 + 0.01
    return codes, scale


def append_plain(codes, scale, x, start, valid):
    """One of keys and values, sequence by sequence and block by block, in the
    fp32 steps the operator defines (numpy-exact): returns new (codes, scale)."""
    codes, scale = codes.clone(), scale.clone()
    b, cap, heads, _ = codes.shape
    inv127 = torch.tensor(1.0) / 127
    lengths = []
    for i in range(b):
        s0 = int(start[i])
        if s0 < 0 or s0 > cap:
            lengths.append(min(max(s0, 0), cap))
            continue
        new = x[i] if valid is None else x[i][valid[i].bool()]
        new = new[: cap - s0].float()
        end = s0 + len(new)
        lengths.append(end)
        for j in range(s0 // 16, -(-end // 16)):
            lo, hi = max(16 * j, s0), min(16 * j + 16, end)
            if hi <= lo:
                continue
            for h in range(heads):
                part = new[lo - s0:hi - s0, h]
                now = part.abs().max() * inv127
                if lo > 16 * j:
                    was = scale[i, h, j]
                    now = torch.maximum(now, was)
                    ratio = was / now if now > 0 else torch.tensor(0.0)
                    old = codes[i, 16 * j:lo, h].float() * ratio
                    codes[i, 16 * j:lo, h] = torch.where(torch.isfinite(now), old.round(), 0.0).to(torch.int8)
                scale[i, h, j] = now
                fresh = (part / now).round().clamp(-127, 127) if now > 0 and torch.isfinite(now) else part * 0
                codes[i, lo:hi, h] = torch.nan_to_num(fresh).to(torch.int8)
    return codes, scale, torch.tensor(lengths, dtype=torch.int32)


APPEND_CASES = [
    # heads, width, capacity, starts, tokens, share valid, dtype
    (1, 256, 1024, (676, 0, 15, 16, 1023), 1, None, torch.bfloat16),
    (1, 256, 832, (0, 0), 776, 0.8, torch.float16),
    (2, 64, 96, (0, 5, 31, 64), 17, None, torch.float16),
    (4, 128, 64, (3, 17), 40, 0.5, torch.bfloat16),
    (1, 64, 48, (1, 2, 3), 45, 0.0, torch.bfloat16),
    (8, 64, 1312, (7,), 1300, 0.97, torch.float16),
    (1, 128, 16, (0, 16, 9), 7, None, torch.float16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,width,cap,starts,tokens,share,dtype", APPEND_CASES)
def test_kv_append(heads, width, cap, starts, tokens, share, dtype):
    g = gen(cap + tokens)
    b = len(starts)
    codes, scale = cache_state(g, b, cap, heads, width)
    k = (randn(g, b, tokens, heads, width) * torch.exp(randn(g, b, tokens, 1, 1))).to(dtype)
    v = randn(g, b, tokens, heads, width).to(dtype)
    valid = None if share is None else torch.rand(b, tokens, generator=g) < share
    start = torch.tensor(starts, dtype=torch.int32)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    nat.device_error(clear=True)
    lengths = w8a8.kv_append(cache, on_gpu(k), on_gpu(v), on_gpu(start), valid=on_gpu(valid))
    want = [append_plain(codes[i], scale[i], x, start, valid) for i, x in enumerate((k, v))]
    count = torch.full((b,), tokens) if valid is None else valid.sum(1)
    over = bool((start + count > cap).any())
    assert nat.device_error(clear=True) == (nat.ERR_CACHE_FULL if over else 0)
    assert torch.equal(lengths.cpu(), want[0][2])
    for got_c, got_s, (wc, ws, _) in ((cache.keys, cache.key_scale, want[0]), (cache.values, cache.value_scale, want[1])):
        assert torch.equal(got_s.cpu(), ws)
        assert torch.equal(got_c.cpu(), wc)
    # the same tokens to the same slots again change nothing
    before = [t.clone() for t in cache]
    assert torch.equal(w8a8.kv_append(cache, on_gpu(k), on_gpu(v), on_gpu(start), valid=on_gpu(valid)), lengths)
    assert all(torch.equal(x, y) for x, y in zip(before, cache))
    nat.device_error(clear=True)
    # and the values that the cache stands for
    for dt in (torch.float32, dtype):
        for got, (wc, ws, wl) in zip(w8a8.kv_values(cache, lengths, dt), want):
            full = wc.double() * ws.double().repeat_interleave(16, 2).transpose(1, 2)[..., None]
            full[torch.arange(cap) >= wl[:, None]] = 0
            within(got, full, (U[dt] + 2.0 ** -23) * full.abs() + TINY[dt])


@pytest.mark.gpu
def test_kv_append_token_by_token_follows_the_plain_form():
    g = gen(77)
    x = randn(g, 1, 40, 2, 64).bfloat16() * (1 + torch.arange(40).bfloat16())[None, :, None, None]  # the scale keeps growing
    cache = w8a8.KVCache8.allocate(1, 40, 2, 64, DEV)
    assert cache.keys.shape[1] == 48
    codes, scale = cache.keys.cpu(), cache.key_scale.cpu()
    lengths = torch.zeros(1, dtype=torch.int32, device=DEV)
    for t in range(40):
        codes, scale, _ = append_plain(codes, scale, x[:, t:t + 1], lengths.cpu(), None)
        lengths = w8a8.kv_append(cache, on_gpu(x[:, t:t + 1]), on_gpu(-x[:, t:t + 1]), lengths)
    assert int(lengths) == 40
    assert torch.equal(cache.keys.cpu(), codes) and torch.equal(cache.key_scale.cpu(), scale)
    assert torch.equal(cache.values.cpu(), -codes)


@pytest.mark.gpu
def test_kv_append_strided_inputs_and_bad_starts():
    g = gen(78)
    b, t, heads, width, cap = 3, 9, 2, 64, 64
    qkv = on_gpu(randn(g, b, t, 4 * heads * width + 3).half())
    rows = qkv[..., 1:].as_strided((b, t, 2 * heads, width), (qkv.stride(0), qkv.stride(1), width, 1))
    k, v = rows[:, :, :heads], rows[:, :, heads:]  # odd strides, odd base
    start = torch.tensor([5, -1, cap + 1], dtype=torch.int32, device=DEV)
    a, c = (w8a8.KVCache8.allocate(b, cap, heads, width, DEV) for _ in range(2))
    nat.device_error(clear=True)
    la = w8a8.kv_append(a, k, v, start)
    lc = w8a8.kv_append(c, k.contiguous(), v.contiguous(), start)
    assert nat.device_error(clear=True) == nat.ERR_CACHE_FULL
    assert la.tolist() == [14, 0, cap] and torch.equal(la, lc)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    assert a.keys[0].any() and not a.keys[1:].any() and not a.key_scale[1:].any()
    # no tokens: nothing but the lengths
    none = w8a8.kv_append(a, k[:, :0], v[:, :0], torch.tensor([5, 0, cap], dtype=torch.int32, device=DEV))
    assert none.tolist() == [5, 0, cap] and all(torch.equal(x, y) for x, y in zip(a, c))
    # transposed [b, heads, t, width] inputs
    lt = w8a8.kv_append(c, k.transpose(1, 2).contiguous().transpose(1, 2), v, start.clamp(0, 5))
    w8a8.kv_append(a, k, v, start.clamp(0, 5))
    assert lt.tolist() == [14, 9, 14] and all(torch.equal(x, y) for x, y in zip(a, c))


@pytest.mark.gpu
def test_kv_append_values_that_are_not_finite():
    b, heads, width = 1, 2, 64
    cache = w8a8.KVCache8.allocate(b, 48, heads, width, DEV)
    k = torch.ones(b, 33, heads, width, dtype=torch.float16, device=DEV)
    k[0, 18, 1, 3] = math.inf
    v = torch.ones_like(k)
    v[0, 2, 0, 5] = math.nan
    lengths = w8a8.kv_append(cache, k, v, torch.zeros(1, dtype=torch.int32, device=DEV))
    keys, values = w8a8.kv_values(cache, lengths, torch.float32)
    bad = torch.zeros(1, 48, heads, dtype=torch.bool, device=DEV)
    bad[0, 16:32, 1] = True
    assert torch.equal(~torch.isfinite(keys).all(-1), bad)
    bad[:] = False
    bad[0, :16, 0] = True
    assert torch.equal(~torch.isfinite(values).all(-1), bad)


# ------------------------------------------------------------ attention
ATTEND_CASES = [
    # q heads, heads, width, capacity, lengths, tokens, causal, dtype
    (8, 1, 256, 784, (776,), 1, False, torch.bfloat16),
    (8, 1, 256, 688, (678, 640, 50, 1), 50, False, torch.bfloat16),
    (1, 1, 64, 16, (1, 0, 16), 1, False, torch.float16),
    (4, 4, 128, 64, (33, 64, 7), 1, True, torch.float16),
    (16, 2, 128, 4112, (4101, 1027, 16, 15, 0), 1, True, torch.float16),
    (6, 2, 64, 160, (160, 131, 17), 17, True, torch.bfloat16),
    (5, 1, 256, 224, (211, 100), 13, True, torch.float16),
    (8, 1, 256, 1040, (1033, 700), 129, True, torch.bfloat16),
    (8, 8, 64, 512, (505, 64), 64, True, torch.float16),
    (2, 1, 64, 96, (20, 3, 0), 33, True, torch.float16),  # more queries than tokens: rows that see nothing
    (40, 1, 128, 304, (300,), 3, False, torch.bfloat16),
    (8, 1, 256, 20000, (19991,), 2, True, torch.float16),
    (32, 4, 64, 2048, (2048, 2000), 4, True, torch.bfloat16),
]


def attention64(q, codes, scale, lengths, causal, softmax_scale):
    """(out, sum P |v|, largest |score|, keys seen, largest |v|) in 64 bits."""
    b, t, qh, w = q.shape
    cap, heads = codes.shape[2:4]
    kv = codes.double() * scale.double().repeat_interleave(16, 3).transpose(2, 3)[..., None]
    k, v = (x.repeat_interleave(qh // heads, 2) for x in kv)
    limit = lengths.long()[:, None].expand(b, t)
    if causal:
        limit = limit - t + 1 + torch.arange(t)
    sees = torch.arange(cap) < limit[..., None]
    s = torch.einsum("bthw,bchw->bhtc", q.double(), k) * softmax_scale
    s = s.masked_fill(~sees[:, None], -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1))
    out = torch.einsum("bhtc,bchw->bthw", p, v)
    mag = torch.einsum("bhtc,bchw->bthw", p, v.abs())
    top = torch.where(torch.isfinite(s), s.abs(), 0.0).amax(-1).permute(0, 2, 1)[..., None]
    return out, mag, top, cap, v.abs().max()


def attention_tol(dtype, out, mag, top, n, vmax):
    # the scores are fp32 sums of `width` products (relative error 2^-20 of the largest), exp's argument
    # carries that error, P is rounded to 11 bits (and to 2^-25 of the row's largest), and l likewise
    return U[dtype] * out.abs() + (2.0 ** -10 + 2.0 ** -18 * (1 + top)) * mag + n * 2.0 ** -25 * vmax + TINY[dtype]


def attention_inputs(qh, heads, width, cap, lengths, tokens, dtype, seed):
    g = gen(seed)
    b = len(lengths)
    codes, scale = cache_state(g, b, cap, heads, width)
    q = (randn(g, b, tokens, qh, width) * torch.exp(0.5 * randn(g, b, tokens, qh, 1))).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32)
    return q, codes, scale, n


@pytest.mark.gpu
@pytest.mark.parametrize("qh,heads,width,cap,lengths,tokens,causal,dtype", ATTEND_CASES)
def test_kv_attention(qh, heads, width, cap, lengths, tokens, causal, dtype):
    q, codes, scale, n = attention_inputs(qh, heads, width, cap, lengths, tokens, dtype, cap + tokens)
    want = attention64(q, codes, scale, n, causal, width ** -0.5)
    # what lies past the length is never seen: scales there are NaN
    past = torch.arange(cap // 16) * 16 >= n[:, None]
    dirty = scale.masked_fill(past[None, :, None], math.nan)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(dirty.to(DEV)))
    out = w8a8.kv_attention(on_gpu(q), cache, on_gpu(n), causal=causal)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    within(out, want[0], attention_tol(dtype, *want))
    limit = n.long()[:, None].expand(len(lengths), tokens)
    if causal:
        limit = limit - tokens + 1 + torch.arange(tokens)
    assert not out.cpu()[limit <= 0].any()  # exactly zero where nothing is seen
    assert torch.equal(out, w8a8.kv_attention(on_gpu(q), cache, on_gpu(n), causal=causal))
    assert nat.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 20, 140])
def test_kv_attention_over_wide_ranges(tokens):
    """Scales of the blocks and magnitudes of the queries over many orders, and
    scores that differ by hundreds."""
    q, codes, scale, n = attention_inputs(8, 2, 128, 640, (633, 320), tokens, torch.bfloat16, 9)
    g = gen(10)
    scale[1] *= torch.exp(6 * torch.randn(scale[1].shape, generator=g))
    q = q * torch.exp(3 * randn(g, 2, tokens, 8, 1)).bfloat16()
    want = attention64(q, codes, scale, n, True, 0.1)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    out = w8a8.kv_attention(on_gpu(q), cache, on_gpu(n), causal=True, softmax_scale=0.1)
    within(out, want[0], attention_tol(torch.bfloat16, *want))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128, 256])
def test_kv_attention_rescales_at_every_tile(width):
    """Many rows over up to 20 tiles of 64 keys whose scores grow by about 18
    bits a tile, so that each tile rescales what the one before it has just
    accumulated, sequences of every number of tiles among them.  Enough CTAs
    that none shares its keys with another; the same bits every time."""
    b, tokens, group, cap = 80, 66, 2, 1280
    g = gen(width)
    codes, scale = cache_state(g, b, cap, 1, width)
    codes[0, ..., 0] = 127
    scale[0] = (0.01 + 0.4 * (torch.arange(cap // 16) // 4)).float()
    q = 0.02 * randn(g, b, tokens, group, width)
    q[..., 0] = 4
    q = q.bfloat16()
    n = torch.tensor([16 * (i + 1) - i % 16 for i in range(b)], dtype=torch.int32)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    qg, ng = on_gpu(q), on_gpu(n)
    out = w8a8.kv_attention(qg, cache, ng, softmax_scale=1 / 16)
    for _ in range(20):
        assert torch.equal(w8a8.kv_attention(qg, cache, ng, softmax_scale=1 / 16), out)
    want = attention64(q, codes, scale, n, False, 1 / 16)
    within(out, want[0], attention_tol(torch.bfloat16, *want))
    assert nat.device_error() == 0


def attention64_rows(q, codes, scale, lengths, causal, softmax_scale):
    """(out, how far it may be off) in 64 bits, by each row's own terms alone:
    the scores' error as in attention_tol, 11 bits of each weight P vs, and for
    weights below fp16's normal numbers half a step of 2^-24 where the row's
    largest weight counts at least 2^-4: n 2^-21 of it, times 127."""
    b, t, qh, w = q.shape
    cap, heads = codes.shape[2:4]
    steps = scale.double().repeat_interleave(16, 3).transpose(2, 3)
    k, v = ((codes.double() * steps[..., None])[i].repeat_interleave(qh // heads, 2) for i in range(2))
    limit = lengths.long()[:, None].expand(b, t)
    if causal:
        limit = limit - t + 1 + torch.arange(t)
    sees = (torch.arange(cap) < limit[..., None])[:, None]
    v = torch.where((torch.arange(cap) < lengths.long()[:, None])[..., None, None], v, 0.0)
    s = torch.einsum("bthw,bchw->bhtc", q.double(), torch.nan_to_num(k)) * softmax_scale
    top = torch.where(sees, s.abs(), 0.0).amax(-1).permute(0, 2, 1)[..., None]
    p = torch.nan_to_num(torch.softmax(s.masked_fill(~sees, -math.inf), -1))
    own = torch.where(sees, p * torch.nan_to_num(steps[1].repeat_interleave(qh // heads, 2).transpose(1, 2))[:, :, None], 0.0)
    v = torch.nan_to_num(v)
    out, mag = (torch.einsum("bhtc,bchw->bthw", p, x) for x in (v, v.abs()))
    largest = own.amax(-1).permute(0, 2, 1)[..., None]
    u = U[q.dtype]
    return out, u * out.abs() + (2.0 ** -10 + 2.0 ** -18 * (1 + top)) * mag + cap * 127 * 2.0 ** -21 * largest + TINY[q.dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [0, 10, 14, 20, 40])
@pytest.mark.parametrize("tokens,width", [(1, 64), (1, 128), (1, 256), (4, 128), (140, 64), (140, 128), (140, 256)])
def test_kv_attention_value_scales_far_apart(tokens, width, gap):
    """Blocks whose value scale is 2^gap times the others' and whose keys get
    next to no weight: what they add to a row is below 2^-20 of it."""
    g = gen(gap + tokens)
    b, heads, group, cap = 2, 2, 4, 640
    codes, scale = cache_state(g, b, cap, heads, width)
    loud = torch.zeros(cap // 16, dtype=torch.bool)
    loud[[0, 3, 4, 17, 38]] = True
    codes[0, ..., 0] = torch.where(loud.repeat_interleave(16), -127, 127).to(torch.int8)[None, :, None]
    scale[0] = 0.02
    scale[1] = torch.where(loud, scale[1] * 2.0 ** gap, scale[1])
    q = 0.3 * randn(g, b, tokens, heads * group, width)
    q[..., 0] = 8
    n = torch.tensor([633, 320], dtype=torch.int32)
    q = q.bfloat16()
    shift = (gap + 24) * math.log(2) / (8 * 2 * 127 * 0.02)  # loud keys' scores lie gap + 24 bits below the others'
    want, tol = attention64_rows(q, codes, scale, n, False, shift)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    out = w8a8.kv_attention(on_gpu(q), cache, on_gpu(n), softmax_scale=shift)
    within(out, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [14, 20, 40, math.nan, math.inf])
@pytest.mark.parametrize("tokens,width", [(4, 64), (4, 256), (5, 128), (140, 64), (140, 128), (140, 256)])
def test_kv_attention_value_scales_that_a_row_does_not_see(tokens, width, gap):
    """Causal: the blocks of the last tokens have value scales 2^gap times the
    others', or ones that are not finite.  Rows before them are what they are
    without, and rows that see them are right or not finite."""
    g = gen(tokens)
    b, heads, group, cap = 2, 1, 2, 320
    codes, scale = cache_state(g, b, cap, heads, width)
    q = randn(g, b, tokens, heads * group, width).bfloat16()
    n = torch.tensor([305, 161], dtype=torch.int32)  # the last token begins a block
    first = (n.long() - 1) // 16 * 16 if tokens < 100 else (n.long() - 70) // 16 * 16
    factor = 2.0 ** gap if math.isfinite(gap) else gap
    for i in range(b):
        scale[1, i, :, first[i] // 16:] *= factor
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    out = w8a8.kv_attention(on_gpu(q), cache, on_gpu(n), causal=True)
    want, tol = attention64_rows(q, codes, scale, n, True, width ** -0.5)
    sees = n.long()[:, None] - tokens + 1 + torch.arange(tokens) > first[:, None]
    assert sees.any(1).all() and (~sees).any(1).all()
    within(out.cpu()[~sees], want[~sees], tol[~sees])
    if math.isfinite(factor):
        within(out, want, tol)
    else:
        assert not torch.isfinite(out.cpu()[sees]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,width", [(1, 64), (1, 128), (1, 256), (140, 64), (140, 128), (140, 256)])
def test_kv_attention_values_of_zero_that_get_nearly_all_weight(tokens, width):
    """Blocks of zero values whose scores lie 60 bits above the others': the
    result is the others' share, 2^-60 of their values."""
    g = gen(width + tokens)
    b, heads, group, cap = 1, 1, 8, 208
    codes, scale = cache_state(g, b, cap, heads, width)
    zero = torch.zeros(cap // 16, dtype=torch.bool)
    zero[[1, 6]] = True
    codes[0, ..., 0] = torch.where(zero.repeat_interleave(16), 127, -127).to(torch.int8)[None, :, None]
    scale[0] = 0.02
    scale[1, ..., zero] = 0
    q = 0.3 * randn(g, b, tokens, heads * group, width)
    q[..., 0] = 8
    q = q.bfloat16()
    n = torch.tensor([200], dtype=torch.int32)
    s = 60 * math.log(2) / (8 * 2 * 127 * 0.02)
    want, tol = attention64_rows(q, codes, scale, n, False, s)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    within(w8a8.kv_attention(on_gpu(q), cache, on_gpu(n), softmax_scale=s), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 140])
@pytest.mark.parametrize("size", [1e-30, 1e-36, 1e30])
def test_kv_attention_value_scales_of_any_size(tokens, size):
    g = gen(tokens)
    codes, scale = cache_state(g, 1, 320, 1, 128)
    scale[1] *= size * 100
    q = randn(g, 1, tokens, 2, 128).bfloat16()
    n = torch.tensor([311], dtype=torch.int32)
    want, tol = attention64_rows(q, codes, scale, n, False, 128 ** -0.5)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    within(w8a8.kv_attention(on_gpu(q), cache, on_gpu(n)), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 70])
def test_kv_attention_strides_and_sentinel_lengths(tokens):
    q, codes, scale, n = attention_inputs(4, 2, 64, 96, (96, 50), tokens, torch.float16, 21)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    qg, ng = on_gpu(q), on_gpu(n)
    out = w8a8.kv_attention(qg, cache, ng)
    # queries [b, heads, tokens, width] seen as [b, tokens, heads, width], from an odd base, reversed rows
    assert torch.equal(w8a8.kv_attention(qg.transpose(1, 2).contiguous().transpose(1, 2), cache, ng), out)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(qg)
    assert torch.equal(w8a8.kv_attention(odd, cache, ng), out)
    # a cache of two layers with heads outside tokens
    big = torch.empty(2, 2, 2, 96, 64, dtype=torch.int8, device=DEV)
    views = [big[i].transpose(1, 2) for i in range(2)]
    for view, c in zip(views, codes):
        view.copy_(c.to(DEV))
    assert torch.equal(w8a8.kv_attention(qg, w8a8.KVCache8(*views, *cache[2:]), ng), out)
    # lengths above the capacity count as the capacity, below zero as none
    ends = torch.tensor([1000, -3], dtype=torch.int32, device=DEV)
    got = w8a8.kv_attention(qg, cache, ends)
    assert torch.equal(got[:1], w8a8.kv_attention(qg, cache, torch.tensor([96, 0], dtype=torch.int32, device=DEV))[:1])
    assert not got[1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 30])
def test_kv_attention_passes_32_bit_offsets(tokens):
    """A cache whose last sequence begins past 2^32 bytes."""
    b, cap, heads, width = 3, 64, 1, 256
    far = (1 << 31) + 4096
    q, codes, scale, n = attention_inputs(2, heads, width, cap, (64, 63, 49), tokens, torch.bfloat16, 30)
    pool = torch.empty(2 * far + cap * width, dtype=torch.int8, device=DEV)
    keys = pool.as_strided((b, cap, heads, width), (far, width, width, 1))
    values = pool[cap * width:2 * far].new_empty(2 * far + cap * width).as_strided((b, cap, heads, width), (far, width, width, 1))
    keys.copy_(codes[0].to(DEV)), values.copy_(codes[1].to(DEV))
    cache = w8a8.KVCache8(keys, values, *(scale.to(DEV)))
    out = w8a8.kv_attention(on_gpu(q), cache, on_gpu(n))
    dense = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    assert torch.equal(out, w8a8.kv_attention(on_gpu(q), dense, on_gpu(n)))
    new = on_gpu(randn(gen(1), b, 3, heads, width).bfloat16())
    start = torch.tensor([3, 40, 61], dtype=torch.int32, device=DEV)
    w8a8.kv_append(cache, new, new, start)
    w8a8.kv_append(dense, new, new, start)
    assert torch.equal(cache.keys, dense.keys) and torch.equal(cache.value_scale, dense.value_scale)


@pytest.mark.gpu
def test_operators_follow_the_current_stream():
    """On a stream of its own, behind work that is still running there."""
    g = gen(40)
    x = on_gpu(randn(g, 64, 2048).bfloat16())
    gain = torch.ones(2048, device=DEV)
    weight = w8a8.pack_weight(on_gpu(randn(g, 256, 2048).bfloat16()))
    want = w8a8.linear(*w8a8.rms_norm_quant(x, gain)[:2], weight)
    q, codes, scale, n = attention_inputs(8, 1, 256, 4096, (4096,), 1, torch.bfloat16, 41)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    qg, ng = on_gpu(q), on_gpu(n)
    want_a = w8a8.kv_attention(qg, cache, ng)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late_x, late_q = torch.zeros_like(x), torch.zeros_like(qg)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=DEV)
        for _ in range(20):
            big = big @ big * 1e-3
        late_x.copy_(x), late_q.copy_(qg)
        got = w8a8.linear(*w8a8.rms_norm_quant(late_x, gain)[:2], weight)
        got_a = w8a8.kv_attention(late_q, cache, ng)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got_a, want_a)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [nat.GEMM_CTA_PAIR, nat.GEMM_SPLIT_K, nat.GEMM_NO_SPLIT])
def test_operators_beside_four_bit_products(variant):
    """Few-token 4-bit products (CTA pairs, split K) and 8-bit kernels with
    tensor memory: one after the other in a stream, and on two streams."""
    from pi05_pytorch_fast_b200 import w4a4

    g = gen(70)
    x = on_gpu(randn(g, 9, 2048).half())
    packed = w4a4.pack_linear_weight(randn(g, 2048, 2048).float(), device=DEV)
    x8 = on_gpu(randn(g, 40, 2048).half())
    weight = w8a8.pack_weight(on_gpu(randn(g, 512, 2048).half()))
    codes8, scale8 = w8a8.quantize(x8)
    q, codes, scale, n = attention_inputs(8, 1, 64, 1024, (1024,) * 4, 20, torch.bfloat16, 71)
    cache = w8a8.KVCache8(*(codes.to(DEV)), *(scale.to(DEV)))
    qg, ng = on_gpu(q), on_gpu(n)

    def four():
        return w4a4.int4_gemm(x, packed)

    def eight():
        return w8a8.linear(codes8, scale8, weight), w8a8.kv_attention(qg, cache, ng)

    try:
        nat.set_gemm_variant(variant)
        want4, want8 = four(), eight()
        for _ in range(50):
            got4, got8 = four(), eight()
        assert torch.equal(got4, want4) and all(torch.equal(a, b) for a, b in zip(got8, want8))
        torch.cuda.synchronize()
        streams = torch.cuda.Stream(), torch.cuda.Stream()
        for _ in range(50):
            with torch.cuda.stream(streams[0]):
                got4 = four()
            with torch.cuda.stream(streams[1]):
                got8 = eight()
        torch.cuda.synchronize()
        assert torch.equal(got4, want4) and all(torch.equal(a, b) for a, b in zip(got8, want8))
        assert nat.device_error() == 0
    finally:
        nat.set_gemm_variant(nat.GEMM_SINGLE_CTA)


@pytest.mark.gpu
def test_operators_in_a_cuda_graph():
    g = gen(50)
    x = on_gpu(randn(g, 8, 1, 512).bfloat16())
    gain = torch.ones(512, device=DEV)
    weight = w8a8.pack_weight(on_gpu(randn(g, 3 * 128, 512).bfloat16()))
    cache = w8a8.KVCache8.allocate(8, 64, 1, 128, DEV)
    start = torch.arange(8, dtype=torch.int32, device=DEV) * 6

    def step():
        codes, scale, _ = w8a8.rms_norm_quant(x, gain)
        q, k, v = w8a8.linear(codes, scale, weight).view(8, 1, 3, 128).split(1, 2)
        lengths = w8a8.kv_append(cache, k, v, start)
        return w8a8.kv_attention(q, cache, lengths, causal=True)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        x.copy_(on_gpu(randn(gen(seed), 8, 1, 512).bfloat16()))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step())


# ------------------------------------------------------------- refusals
def test_ops_refuse_cpu_tensors():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    codes, scale = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    cache = w8a8.KVCache8.allocate(1, 16, 1, 64, "cpu")
    n = torch.zeros(1, dtype=torch.int32)
    kv = torch.zeros(1, 1, 1, 64, dtype=torch.float16)
    for call in (lambda: w8a8.rms_norm_quant(x, torch.ones(64)), lambda: w8a8.quantize(x), lambda: w8a8.pack_weight(x),
                 lambda: w8a8.dequantize(codes, scale), lambda: w8a8.linear(codes, scale, w8a8.Int8Weight(codes, scale)),
                 lambda: w8a8.kv_append(cache, kv, kv, n), lambda: w8a8.kv_values(cache, n),
                 lambda: w8a8.kv_attention(kv, cache, n)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_fakes_give_shapes_and_strides():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 3, 97, dtype=torch.bfloat16, device="cuda")
        codes, scale, total = torch.ops.pi05_w8a8.rms_norm_quant(x, torch.empty(97, device="cuda"), 1e-6, x)
        assert codes.shape == x.shape and codes.stride() == (336, 112, 1) and codes.dtype == torch.int8
        assert scale.shape == (2, 3) and total.shape == x.shape and total.dtype == x.dtype
        y = torch.ops.pi05_w8a8.linear(codes, scale, torch.empty(5, 97, dtype=torch.int8, device="cuda"),
                                       torch.empty(5, device="cuda"), None, torch.float16)
        assert y.shape == (2, 3, 5) and y.dtype == torch.float16
        cache = w8a8.KVCache8.allocate(2, 20, 1, 64, "cuda")
        n = torch.empty(2, dtype=torch.int32, device="cuda")
        q = torch.empty(2, 7, 4, 64, dtype=torch.float16, device="cuda")
        assert torch.ops.pi05_w8a8.kv_append(*cache, q[:, :, :1], q[:, :, :1], n).shape == (2,)
        assert torch.ops.pi05_w8a8.kv_attention(q, *cache, n, False, 1.0).shape == q.shape
        assert torch.ops.pi05_w8a8.kv_values(*cache, n, torch.bfloat16)[1].shape == (2, 32, 1, 64)


def test_c_abi_argument_checks_without_gpu():
    lib = nat.lib()
    fake = 0x10000  # never dereferenced: every check comes first

    def message(status, code):
        assert status == code
        return nat.last_error()

    bad = nat.W4A4_ERR_INVALID
    norm = [fake, 64, None, 0, None, 0, fake, 0, None, 0, 1e-6, nat.BF16, 4, 1, 64, None, fake, 64, fake, None]

    def with_(args, **at):
        args = list(args)
        for i, v in at.items():
            args[int(i[1:])] = v
        return args

    assert "row stride" in message(lib.w4a4_rms_norm_quant8(*with_(norm, _1=63)), bad)
    assert "null" in message(lib.w4a4_rms_norm_quant8(*with_(norm, _6=None)), bad)
    assert "gate needs a delta" in message(lib.w4a4_rms_norm_quant8(*with_(norm, _4=fake)), bad)
    assert "rows_per_batch" in message(lib.w4a4_rms_norm_quant8(*with_(norm, _13=0)), bad)
    assert "dtype" in message(lib.w4a4_rms_norm_quant8(*with_(norm, _11=7)), bad)
    assert lib.w4a4_rms_norm_quant8(*with_(norm, _12=0)) == 0
    quant = [fake, 64, None, 0, nat.F16, 4, 64, fake, 64, fake, None]
    assert "shape" in message(lib.w4a4_quant8(*with_(quant, _6=0)), bad)
    assert "null" in message(lib.w4a4_quant8(*with_(quant, _9=None)), bad)
    assert "row stride" in message(lib.w4a4_quant8(*with_(quant, _2=fake, _3=8)), bad)
    assert "row stride" in message(lib.w4a4_dequant8(fake, 63, fake, nat.F16, 4, 64, fake, None), bad)
    gemm = [fake, 64, fake, fake, 64, fake, None, nat.F16, 4, 8, 64, fake, None]
    assert "shape" in message(lib.w4a4_gemm8(*with_(gemm, _9=0)), bad)
    assert "16 bytes" in message(lib.w4a4_gemm8(*with_(gemm, _1=72)), bad)
    assert "16 bytes" in message(lib.w4a4_gemm8(*with_(gemm, _3=fake + 8)), bad)
    assert "row stride" in message(lib.w4a4_gemm8(*with_(gemm, _4=48)), bad)
    assert "131072" in message(lib.w4a4_gemm8(*with_(gemm, _10=131072, _1=131072, _4=131072)), nat.W4A4_ERR_UNSUPPORTED)
    assert lib.w4a4_gemm8(*with_(gemm, _8=0)) == 0
    strides = (ctypes.c_int64 * 3)(64 * 32, 64, 64)
    att = [fake, strides, fake, fake, fake, fake, strides, 32, fake, nat.F16, 1, 1, 4, 2, 64, 0, 1.0, fake, None, 0, None]
    assert "query heads" in message(lib.w4a4_attention8(*with_(att, _12=3)), bad)
    assert "capacity" in message(lib.w4a4_attention8(*with_(att, _7=33)), bad)
    assert "width" in message(lib.w4a4_attention8(*with_(att, _14=72)), nat.W4A4_ERR_UNSUPPORTED)
    assert "dtype" in message(lib.w4a4_attention8(*with_(att, _9=nat.F32)), bad)
    odd = (ctypes.c_int64 * 3)(64 * 32, 72, 64)
    assert "16 bytes" in message(lib.w4a4_attention8(*with_(att, _6=odd)), bad)
    assert lib.w4a4_attention8(*with_(att, _11=0)) == 0
    app = [fake, fake, fake, fake, strides, 32, fake, strides, fake, strides, nat.F16, None, 0, fake, fake, 1, 1, 2, 64, None]
    assert "null" in message(lib.w4a4_kv8_append(*with_(app, _13=None)), bad)
    assert "token count" in message(lib.w4a4_kv8_append(*with_(app, _16=-1)), bad)
    assert "null" in message(lib.w4a4_kv8_values(fake, fake, fake, fake, strides, 32, None, nat.F16, 1, 2, 64, fake, fake, None), bad)


@pytest.mark.gpu
def test_ops_refuse_bad_arguments():
    x = torch.zeros(2, 3, 64, dtype=torch.bfloat16, device=DEV)
    ones = torch.ones(64, device=DEV)

    def refuses(match, call):
        with pytest.raises(RuntimeError, match=match):
            call()

    refuses("float16, bfloat16 or float32", lambda: w8a8.quantize(x.double()))
    refuses("non-empty last dimension", lambda: w8a8.quantize(x[..., :0]))
    refuses("gain must be", lambda: w8a8.rms_norm_quant(x, ones[:63]))
    refuses("gain must be", lambda: w8a8.rms_norm_quant(x, ones.expand(3, 64)))
    refuses("gain must be", lambda: w8a8.rms_norm_quant(x, ones.bfloat16()))
    refuses("gate needs a delta", lambda: w8a8.rms_norm_quant(x, ones, gate=x[:, 0]))
    refuses("delta must have", lambda: w8a8.rms_norm_quant(x, ones, delta=x.half()))
    refuses("shift is on cpu", lambda: w8a8.rms_norm_quant(x, ones, shift=torch.ones(64)))
    refuses("up must have", lambda: w8a8.quantize(x, up=x[:1]))
    codes, scale = w8a8.quantize(x)
    weight = w8a8.pack_weight(torch.ones(8, 64, device=DEV))
    refuses("weight must be", lambda: w8a8.linear(codes[..., :32], scale, weight))
    refuses("codes must be int8", lambda: w8a8.linear(x, scale, weight))
    refuses("scale must be", lambda: w8a8.linear(codes, scale[:1], weight))
    refuses("bias must be", lambda: w8a8.linear(codes, scale, weight, bias=torch.ones(8, device=DEV)))
    refuses("dtype must be", lambda: w8a8.linear(codes, scale, weight, dtype=torch.float64))
    refuses("pack_weight expects", lambda: w8a8.pack_weight(ones))
    cache = w8a8.KVCache8.allocate(2, 32, 2, 64, DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    kv = torch.zeros(2, 1, 2, 64, dtype=torch.float16, device=DEV)
    refuses("new keys must be", lambda: w8a8.kv_append(cache, kv[:, :, :1], kv, n))
    refuses("new values must have", lambda: w8a8.kv_append(cache, kv, kv[:1], n))
    refuses("new keys must be float16 or bfloat16", lambda: w8a8.kv_append(cache, kv.float(), kv.float(), n))
    refuses("start must be", lambda: w8a8.kv_append(cache, kv, kv, n.long()))
    refuses("valid must be", lambda: w8a8.kv_append(cache, kv, kv, n, valid=torch.ones(2, 2, device=DEV)))
    refuses("q must be", lambda: w8a8.kv_attention(kv[:, :, :1], cache, n))
    refuses("q must be float16 or bfloat16", lambda: w8a8.kv_attention(kv.float(), cache, n))
    refuses("lengths must be", lambda: w8a8.kv_attention(kv, cache, n[:1]))
    refuses("laid out like the keys", lambda: w8a8.kv_values(cache._replace(values=cache.values[:, :16]), n))
    refuses("multiple of 16", lambda: w8a8.kv_values(cache._replace(keys=cache.keys[:, :20], values=cache.values[:, :20]), n))
    refuses("cache scales must be", lambda: w8a8.kv_values(cache._replace(key_scale=cache.key_scale[..., :1]), n))
    wide = w8a8.KVCache8.allocate(2, 32, 2, 72, DEV)
    refuses("64, 128 or 256", lambda: w8a8.kv_values(wide, n))



@pytest.mark.gpu
def test_ops_refuse_inputs_that_want_a_gradient():
    x = torch.ones(1, 1, 1, 64, dtype=torch.float16, device=DEV)
    wants = x.clone().requires_grad_()
    ones = torch.ones(64, device=DEV)
    cache, n = w8a8.KVCache8.allocate(1, 16, 1, 64, DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    calls = (lambda t: w8a8.quantize(t), lambda t: w8a8.quantize(x, up=t), lambda t: w8a8.rms_norm_quant(t, ones),
             lambda t: w8a8.rms_norm_quant(x, ones, delta=t), lambda t: w8a8.kv_append(cache, t, x, n),
             lambda t: w8a8.kv_append(cache, x, t, n), lambda t: w8a8.kv_attention(t, cache, n))
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call(wants)
        with torch.no_grad():
            call(wants)
        call(wants.detach())
    assert w8a8.pack_weight(torch.nn.Parameter(torch.ones(8, 64, device=DEV))).codes.shape == (8, 64)


def _float_inputs():
    """Every floating-point input of every op: (name, a value, the call with it in that place)."""
    g = gen(60)
    x = on_gpu(randn(g, 2, 1, 64).half())
    gain, shift, gate = torch.ones(64, device=DEV), torch.zeros(2, 64, device=DEV), torch.ones(2, 64, device=DEV).half()
    codes, scale = w8a8.quantize(x)
    weight = w8a8.pack_weight(on_gpu(randn(g, 8, 64).half()))
    bias = torch.zeros(8, dtype=torch.float16, device=DEV)
    cache, n = w8a8.KVCache8.allocate(1, 16, 1, 64, DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    kv = on_gpu(randn(g, 1, 1, 1, 64).half())
    f16 = dict(dtype=torch.float16)
    norm = lambda **k: w8a8.rms_norm_quant(**{**dict(x=x, gain=gain, delta=x, gate=gate, shift=shift), **k})  # noqa: E731
    put = lambda t, i: cache._replace(**{("key_scale", "value_scale")[i]: t})  # noqa: E731
    return [
        ("x", x, lambda t: norm(x=t)), ("gain", gain, lambda t: norm(gain=t)), ("delta", x, lambda t: norm(delta=t)),
        ("gate", gate, lambda t: norm(gate=t)), ("shift", shift, lambda t: norm(shift=t)),
        ("x", x, lambda t: w8a8.quantize(t)), ("up", x, lambda t: w8a8.quantize(x, up=t)),
        ("scale", scale, lambda t: w8a8.dequantize(codes, t)),
        ("scale", scale, lambda t: w8a8.linear(codes, t, weight, **f16)),
        ("weight_scale", weight.scale, lambda t: w8a8.linear(codes, scale, weight._replace(scale=t), **f16)),
        ("bias", bias, lambda t: w8a8.linear(codes, scale, weight, bias=t, **f16)),
        ("new keys", kv, lambda t: w8a8.kv_append(cache, t, kv, n)), ("new values", kv, lambda t: w8a8.kv_append(cache, kv, t, n)),
        ("q", kv, lambda t: w8a8.kv_attention(t, cache, n)),
        *[("cache scale", cache.key_scale, lambda t, i=i, op=op: op(put(t, i))) for i in (0, 1) for op in (
            lambda c: w8a8.kv_append(c, kv, kv, n), lambda c: w8a8.kv_values(c, n), lambda c: w8a8.kv_attention(kv, c, n))],
    ]


@pytest.mark.gpu
def test_ops_refuse_a_gradient_of_any_input():
    for name, value, call in _float_inputs():
        wants = value.clone().requires_grad_()
        with pytest.raises(RuntimeError, match=name + " requires one"):
            call(wants)
        with torch.no_grad():
            call(wants)
        call(wants.detach())


@pytest.mark.gpu
def test_ops_refuse_forward_mode_tangents():
    import torch.autograd.forward_ad as fwd

    for name, value, call in _float_inputs():
        with fwd.dual_level():
            dual = fwd.make_dual(value.clone(), torch.ones_like(value))
            with pytest.raises(RuntimeError, match=name + " carries a forward-mode tangent"):
                call(dual)
            call(fwd.unpack_dual(dual).primal)


# --- the operators together: the SnapFlow action expert in 8 bits -----------


def _expert(layers=2, seed=3):
    """A bf16 expert of the published width, an 8-bit one of its weights, and
    inputs of two observations with different prefix lengths (40 slots)."""
    dev = torch.device("cuda:0")
    cfg = sf.SnapFlowConfig(expert_layers=layers)
    torch.manual_seed(seed)
    with torch.device(dev):
        expert = sf.ActionExpert(cfg)
    for p in expert.parameters():
        if p.dim() >= 2:
            torch.nn.init.normal_(p, std=0.02)
    expert = expert.bfloat16().eval()
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    pad = torch.zeros(2, 40, dtype=torch.bool, device=dev)
    pad[0, :33] = True
    pad[1, 5:40:3] = True
    kv = [[torch.randn(2, 40, 256, device=dev, generator=g).half() for _ in range(layers)] for _ in range(2)]
    x_t = torch.randn(2, cfg.chunk, cfg.action_dim, device=dev, generator=g).bfloat16()
    return expert, (x_t, torch.ones(2, device=dev), torch.ones(2, device=dev), pad, *kv)


@pytest.mark.gpu
def test_snapflow_expert_in_8_bits_against_fp64():
    """Relative error of the velocity.  A rounding to 127 steps of a row's
    largest value, r times the row's RMS, has a relative error r / (127
    sqrt(12)): 0.8 % for normal rows of 1,024 to 2,048 (r = 3.5), and at most
    2.3 % for the GeGLU product (r = 10).  Along the attention branch: norm
    codes and weights 1.1 %, keys and values 0.8 %, codes and weights of the
    output product 1.1 %, together under 2 %; along the MLP: 1.1 % on each
    factor, 2.3 % on their product, 0.8 % weights, together under 3 %.  The
    branches of two layers are summed, so their relative error is no more than
    one's plus what a layer passes on from the one before it (under 3 % again):
    6 %, and 1 % for bf16."""
    expert, inputs = _expert()
    expert8 = sf.ActionExpert8(expert)
    expert64 = sf.ActionExpert(expert.cfg).to("cuda:0").double()
    expert64.load_state_dict(expert.state_dict())
    with torch.no_grad():
        v = expert8(*inputs)
        ref = expert64(inputs[0].double(), *inputs[1:])
    assert v.shape == ref.shape and v.dtype == torch.bfloat16
    rel = (v.double() - ref).norm() / ref.norm()
    assert rel < 0.07, float(rel)


@pytest.mark.gpu
def test_snapflow_expert_in_8_bits_masked_prefix_and_reuse():
    """What stands in masked prefix slots does not matter, neither does what an
    earlier call left in the cache; a call of another batch in between neither."""
    expert, inputs = _expert(layers=1)
    expert8 = sf.ActionExpert8(expert)
    x_t, t, target, pad, keys, values = inputs
    with torch.no_grad():
        v = expert8(*inputs)
        other = expert8(x_t[:1], t[:1], target[:1], ~pad[:1], [k[:1] for k in keys], [k[:1] * 7 for k in values])
        junk = [[torch.where(pad[..., None], k, torch.tensor(bad, dtype=k.dtype, device=k.device)) for k in kv]
                for kv, bad in ((keys, math.nan), (values, math.inf))]
        expert8(x_t * 5, t, target, ~pad, [k * 9 for k in keys], [k * 9 for k in values])
        again = expert8(x_t, t, target, pad, *junk)
    assert torch.equal(v, again) and torch.isfinite(other).all()


@pytest.mark.gpu
def test_snapflow_expert_in_8_bits_in_a_graph():
    expert, inputs = _expert(layers=1)
    expert8 = sf.ActionExpert8(expert)
    with torch.no_grad():
        eager = expert8(*inputs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = expert8(*inputs)
        graph.replay()
    assert torch.equal(out, eager)


@pytest.mark.gpu
def test_snapflow_expert_in_8_bits_first_called_under_capture():
    """A shape's first call recorded in a graph, an eager call before the graph
    has run once, and the graph then: each as the call alone."""
    expert, inputs = _expert(layers=1)
    expert8 = sf.ActionExpert8(expert)
    alone = sf.ActionExpert8(expert)
    x_t, t, target, pad, keys, values = inputs
    with torch.no_grad():
        want = alone(*inputs)
        expert8(x_t[:1], t[:1], target[:1], pad[:1], [k[:1] for k in keys], [v[:1] for v in values])  # libraries' set-up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = expert8(*inputs)
        eager = expert8(*inputs)
        assert torch.equal(eager, want)
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_snapflow_expert_in_8_bits_on_two_streams():
    """Calls of one expert that run at the same time do not meet."""
    expert, inputs = _expert()
    expert8 = sf.ActionExpert8(expert)
    x_t, t, target, pad, keys, values = inputs
    other = (x_t.flip(0) * 3, t, target, ~pad, [k * 2 for k in keys], [v.flip(0) for v in values])
    with torch.no_grad():
        want = [expert8(*inputs), expert8(*other)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        got = ([], [])
        for _ in range(20):
            for i, args in enumerate((inputs, other)):
                with torch.cuda.stream(streams[i]):
                    got[i].append(expert8(*args))
        torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(v, w) for v in g)


@pytest.mark.gpu
def test_snapflow_expert_in_8_bits_keeps_nothing():
    expert, inputs = _expert(layers=1)
    expert8 = sf.ActionExpert8(expert)
    x_t, t, target, pad, keys, values = inputs

    def call(n, b):
        with torch.no_grad():
            expert8(x_t[:b], t[:b], target[:b], pad[:b, :n], [k[:b, :n] for k in keys], [v[:b, :n] for v in values])

    call(40, 2), call(40, 1)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for n in (8, 24, 33):
        call(n, 1)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


@pytest.mark.gpu
def test_snapflow_policy_with_the_expert_in_8_bits():
    """The whole step, eager and as a graph, and its velocity next to that of
    the bf16 policy of the same weights: two layers, so at most 6 % for the 8
    bits (see above) and 1 % for bf16 on either side."""
    dev = torch.device("cuda:0")
    lm_cfg = plm.PrefixLMConfig(layers=2)
    cfg = sf.SnapFlowConfig(vision_layers=1, expert_layers=2, vocab=512, lm=lm_cfg)
    lm = plm.W4A4PrefixLM.random(lm_cfg, dev, seed=5)
    policy8 = sf.SnapFlowPolicy(cfg, lm, dev, seed=6, expert_bits=8)
    obs = sf.synthetic_observation(cfg, 2, seed=7, device=dev)
    eager = policy8.sample_actions(*obs)
    graphed = sf.GraphedSnapFlow(policy8, 2)
    assert torch.equal(graphed.run(*obs), eager)
    x_t = obs[3].bfloat16().double()
    v8 = x_t - eager.double()
    v16 = x_t - sf.SnapFlowPolicy(cfg, lm, dev, seed=6).sample_actions(*obs).double()
    rel = (v8 - v16).norm() / v16.norm()
    assert rel < 0.08, float(rel)


def test_snapflow_expert_in_8_bits_refusals():
    cfg = sf.SnapFlowConfig(expert_layers=1, expert_hidden=32, expert_intermediate=32, head_dim=64)
    with pytest.raises(ValueError, match="bf16 expert on a CUDA device"):
        sf.ActionExpert8(sf.ActionExpert(cfg))
    with pytest.raises(ValueError, match="expert_bits is 8 or 16"):
        sf.SnapFlowPolicy(cfg, None, "cpu", expert_bits=4)
