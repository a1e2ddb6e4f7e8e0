"""rms_norm and matvec against their definitions in 64 bits."""
import copy
import ctypes
import math
import pickle

import numpy as np
import pytest
import torch

import oracle
import ptwm_b200
from ptwm_b200 import Projection, ScaledActivations, ScaledWeight, matvec, rms_norm
from _data import mixed_model, specs_mxfp4, specs_nvfp4, spec_norm

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64)
F32 = 2.0 ** -24  # half a step of fp32


@pytest.fixture(autouse=True)
def _cuda(cuda_device):
    torch.cuda.set_device(cuda_device)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):  # half the smallest step there is
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


# ---- rms_norm ----------------------------------------------------------------------------------------
def _norm64(x, weight, eps, residual):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    h64 = h.double()
    rms = (h64.square().mean(-1, keepdim=True) + eps).sqrt()
    return h, h64 / rms * weight.double()


def _norm_slack(cols):
    """Relative error of y before its rounding: a sum of positive terms in which a term goes through at most cols / 32 + 16
    additions (half of that after the root), the mean, the root (2 steps) and two products."""
    return ((cols / 32 + 16) / 2 + 8) * F32


def _inputs(rows, cols, dtype, seed, residual=True, weight_dtype=None):
    g = _gen(seed)
    x = (torch.randn(rows, cols, generator=g, device="cuda") * 3).to(dtype)
    res = (torch.randn(rows, cols, generator=g, device="cuda") * 2).to(dtype) if residual else None
    w = (1 + 0.1 * torch.randn(cols, generator=g, device="cuda")).to(weight_dtype or dtype)
    return x, res, w


ROWS_COLS = [(1, 1), (3, 7), (1, 32), (5, 96), (2, 1000), (17, 1024), (1, 4096), (333, 4095), (7, 8200), (2, 10501), (3, 16384), (2, 40000), (1200, 64), (1203, 128), (301, 32), (999, 256), (500, 1024), (4, 8224), (3, 16416), (2, 24992)]


@pytest.mark.parametrize("rows, cols", ROWS_COLS)
@pytest.mark.parametrize("dtype, weight_dtype", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32"), ("fp32", "bf16")])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_plain(rows, cols, dtype, weight_dtype, residual):
    x, res, w = _inputs(rows, cols, DT[dtype], rows + cols, residual, DT[weight_dtype])
    got = rms_norm(x, w, 1e-5, residual=res)
    y, h = got if residual else (got, None)
    want_h, want = _norm64(x, w, 1e-5, res)
    if residual:
        assert torch.equal(h, want_h)
    assert y.dtype == x.dtype and y.shape == x.shape
    tol = (_half_step(x.dtype) + _norm_slack(cols)) * want.abs() + _floor(x.dtype)
    assert bool(((y.double() - want).abs() <= tol).all())


def _check_8(values, scales, want, rel, step):
    """E4M3 values times scales against want: half a step of E4M3, relative 2^-4 or, below its normal numbers, 2^-10 of the scale."""
    back = values.double() * scales
    tol = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * scales) * (1 + 2.0 ** -10) + rel * want.abs()
    assert bool(((back - want).abs() <= tol).all())


@pytest.mark.parametrize("rows, cols", ROWS_COLS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_norm_row_scales(rows, cols, dtype):
    x, res, w = _inputs(rows, cols, DT[dtype], 2 * rows + cols)
    y, h = rms_norm(x, w, 1e-5, residual=res, quant="row")
    want_h, want = _norm64(x, w, 1e-5, res)
    assert torch.equal(h, want_h) and y.quant == "row" and y.shape == x.shape
    s = want.abs().amax(-1) / 448
    assert bool(((y.scales.double() - s).abs() <= (_norm_slack(cols) + 2 * F32) * s).all())
    _check_8(y.values, y.scales.double()[:, None], want, 2 * _norm_slack(cols), None)


@pytest.mark.parametrize("rows, cols", [rc for rc in ROWS_COLS if rc[1] % 32 == 0])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_norm_block_scales(rows, cols, dtype):
    x, res, w = _inputs(rows, cols, DT[dtype], 3 * rows + cols)
    w = w * torch.where(torch.arange(cols, device="cuda") % 3 == 0, 2.0 ** -9, 1.0).to(w.dtype)
    y, h = rms_norm(x, w, 1e-5, residual=res, quant="block")
    want_h, want = _norm64(x, w, 1e-5, res)
    assert torch.equal(h, want_h) and y.quant == "block" and y.scales.shape == (rows, cols // 32)
    most = want.reshape(rows, -1, 32).abs().amax(-1)
    slack = _norm_slack(cols)
    lo, hi = (torch.ceil(torch.log2(most * f / 448)).clamp(-127, 127) + 127 for f in (1 - slack, 1 + slack))
    e = y.scales.view(torch.uint8).double()
    assert bool(((e >= lo) & (e <= hi)).all())
    _check_8(y.values, torch.exp2(e - 127).repeat_interleave(32, 1), want, 2 * slack, None)


@pytest.mark.parametrize("quant", [None, "row", "block"])
def test_norm_of_zeros_infinities_and_nan(quant):
    cols = 4096
    x = torch.randn(6, cols, generator=_gen(1), device="cuda").to(torch.bfloat16)
    x[1] = 0
    x[2, 77] = math.inf
    x[3, 4095] = math.nan
    x[4] = 1e-30
    w = torch.ones(cols, device="cuda", dtype=torch.bfloat16)
    got = rms_norm(x, w, 0.0 if quant is None else 1e-6, quant=quant)
    if quant is None:
        y = got.double()
        assert bool(torch.isnan(y[1]).all())  # 0 / 0: no eps
        assert bool(torch.isnan(y[3]).all()) and math.isnan(y[2, 77]) and bool((y[2, :77] == 0).all())
    else:
        s = got.scales.view(torch.uint8).int() if quant == "block" else got.scales
        v = got.values.float()
        assert bool((v[1] == 0).all()) and bool((s[1] == 0).all())
        if quant == "row":
            assert bool(torch.isnan(s[2:4]).all()) and bool(torch.isnan(v[2:4]).all())
        else:
            assert s[2, 77 // 32] == 255 and bool(torch.isnan(v[2, 64:96]).all()) and bool((v[2, :64] == 0).all())
            assert bool((s[3] == 255).all()) and bool(torch.isnan(v[3]).all())
        assert bool((v[4] > 0).all())
    plain = rms_norm(x[5:], w, 1e-6, quant=quant)  # a row does not know its neighbours
    again = rms_norm(x, w, 1e-6, quant=quant)
    if quant is None:
        assert torch.equal(plain[0], again[5])
    else:
        assert torch.equal(plain.values.view(torch.uint8)[0], again.values.view(torch.uint8)[5])


@pytest.mark.parametrize("rows, cols", [(1, 5), (40, 1), (37, 9), (21, 17), (9, 513), (700, 333), (5, 4095), (3, 8190), (2, 8191), (5, 16367), (2, 16383), (3, 20003)])
@pytest.mark.parametrize("dtype, weight_dtype", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp32"), ("fp32", "fp32"), ("fp32", "fp16")])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("quant", [None, "row"])
def test_norm_rows_that_share_pieces_with_their_neighbours(rows, cols, dtype, weight_dtype, residual, quant):
    """Rows of a length that no 16 bytes divide; every second one, and all that lies around them, is NaN."""
    dt = DT[dtype]
    x, res, w = _inputs(rows, cols, dt, rows * 7 + cols, residual, DT[weight_dtype])
    front = 48  # values, whole pieces
    held = []
    for t in (x, res):
        if t is None:
            held.append(None)
            continue
        wide = torch.full((front + 2 * rows * cols + 64,), math.nan, dtype=dt, device="cuda")
        inside = wide[front:front + 2 * rows * cols].view(2 * rows, cols)
        inside[::2] = t
        held.append(inside)
    got = rms_norm(held[0], w, 1e-5, residual=held[1], quant=quant)
    y, h = got if residual else (got, None)
    want_h, want = _norm64(x, w, 1e-5, res)
    if residual:
        assert torch.equal(h[::2], want_h) and bool(torch.isnan(h[1::2]).all())
    if quant is None:
        assert bool(torch.isnan(y[1::2]).all())
        tol = (_half_step(dt) + _norm_slack(cols)) * want.abs() + _floor(dt)
        assert bool(((y[::2].double() - want).abs() <= tol).all())
    else:
        assert bool(torch.isnan(y.scales[1::2]).all()) and bool(torch.isnan(y.values[1::2].float()).all())
        s = want.abs().amax(-1) / 448
        assert bool(((y.scales[::2].double() - s).abs() <= (_norm_slack(cols) + 2 * F32) * s).all())
        _check_8(y.values[::2], y.scales[::2].double()[:, None], want, 2 * _norm_slack(cols), None)


def test_norm_strides_offsets_and_empty_rows():
    base = torch.randn(9, 517, generator=_gen(2), device="cuda").to(torch.bfloat16)
    w = torch.randn(1030, generator=_gen(3), device="cuda").to(torch.bfloat16)
    for x, weight in [(base[:, 1:513], w[3:515]), (base.t(), w[1:10]), (base[::2, ::2], w[::3][:259]), (base[1:].reshape(2, 4, 517), w[:517]), (base.flatten()[1:4097].view(4, 1024), w[5:1029])]:
        y = rms_norm(x, weight, 1e-5)
        _, want = _norm64(x, weight, 1e-5, None)
        assert y.shape == x.shape
        assert bool(((y.double() - want).abs() <= (_half_step(x.dtype) + _norm_slack(x.shape[-1])) * want.abs()).all())
    for quant in (None, "row", "block"):
        y, h = rms_norm(base[:0, :512], w[:512], residual=base[:0, :512], quant=quant)
        assert y.shape == (0, 512) and h.shape == (0, 512)


@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (5, 96), (1, 4096), (700, 1000), (333, 4095), (2, 10501), (3, 16384), (2, 40000), (1000, 333), (600, 4097), (297, 8191), (299, 16367), (900, 5), (310, 8200), (3, 16384), (300, 10001), (299, 12289)])
@pytest.mark.parametrize("dtype, weight_dtype", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_gradient(rows, cols, dtype, weight_dtype, residual):
    x, res, w = _inputs(rows, cols, DT[dtype], rows * 5 + cols, residual, DT[weight_dtype])
    leaves = [t.requires_grad_() for t in (x, w, res) if t is not None]
    g = _gen(9)
    dy = torch.randn(rows, cols, generator=g, device="cuda").to(x.dtype)
    dh = torch.randn(rows, cols, generator=g, device="cuda").to(x.dtype)
    got = rms_norm(x, w, 1e-5, residual=res)
    grads = torch.autograd.grad(got, leaves, (dy, dh) if residual else dy)
    h = (x.float() + res.float()).to(x.dtype).double().detach() if residual else x.double().detach()
    r = (h.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    gw = dy.double() * w.double().detach()
    parts = [r * gw, h * r ** 3 * (gw * h).mean(-1, keepdim=True)] + ([dh.double()] if residual else [])
    want = parts[0] - parts[1] + (parts[2] if residual else 0)
    # fp32 errors of each part: the dot product's go with the sum of its magnitudes; then one rounding
    size = parts[0].abs() + (h * r ** 3).abs() * (gw * h).abs().mean(-1, keepdim=True) + want.abs()
    tol = _half_step(x.dtype) * want.abs() + 4 * _norm_slack(cols) * size + _floor(x.dtype)
    assert bool(((grads[0].double() - want).abs() <= tol).all())
    if residual:
        assert torch.equal(grads[2], grads[0])
    terms = dy.double() * h * r
    tol = _half_step(w.dtype) * terms.sum(0).abs() + ((rows + 16) * F32 + 2 * _norm_slack(cols)) * terms.abs().sum(0) + _floor(w.dtype)
    assert grads[1].dtype == w.dtype and bool(((grads[1].double() - terms.sum(0)).abs() <= tol).all())


def test_norm_gradient_against_differences():
    x, res, w = _inputs(3, 40, torch.float32, 4)
    c1, c2 = (torch.randn(3, 40, generator=_gen(s), device="cuda") for s in (5, 6))

    def loss64(x, res, w):
        h = x.double() + res.double()
        y = h * (h.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w.double()
        return ((y * c1.double()).sum() + (h * c2.double()).sum()).item()

    for t in (x, res, w):
        t.requires_grad_()
    y, h = rms_norm(x, w, 1e-5, residual=res)
    ((y * c1).sum() + (h * c2).sum()).backward()
    step = 2.0 ** -8
    for t in (x, res, w):
        flat, grad = t.detach().clone().flatten(), t.grad.flatten()
        for i in range(0, flat.numel(), 7):
            args = []
            for sign in (1, -1):
                moved = flat.double().clone()
                moved[i] += sign * step
                args.append([moved.view(t.shape) if o is t else o.detach().double() for o in (x, res, w)])
            slope = (loss64(*args[0]) - loss64(*args[1])) / (2 * step)
            # third derivatives of order one: an error of some step^2
            assert abs(slope - grad[i].item()) <= 8 * step ** 2 * (1 + abs(slope))


def test_norm_gradient_of_one_output_and_of_some_inputs():
    x, res, w = _inputs(4, 64, torch.float32, 8)
    x.requires_grad_()
    y, h = rms_norm(x, w, residual=res)
    assert torch.equal(torch.autograd.grad(h.sum(), x)[0], torch.ones_like(x))
    y, h = rms_norm(x, w, residual=res)
    only, = torch.autograd.grad(y.sum(), x)
    w.requires_grad_()
    y, h = rms_norm(x.detach(), w, residual=res)
    dw, = torch.autograd.grad(y.sum(), w)
    y, h = rms_norm(x, w, residual=res)
    a, b = torch.autograd.grad(y.sum(), (x, w))
    assert torch.equal(a, only) and torch.equal(b, dw)
    empty = torch.empty(0, 64, device="cuda", requires_grad=True)
    a, b = torch.autograd.grad(rms_norm(empty, w).sum(), (empty, w))
    assert a.shape == (0, 64) and bool((b == 0).all())
    with pytest.raises(ValueError, match="no gradient"):
        rms_norm(x, w, quant="row")
    with torch.no_grad():
        rms_norm(x, w, quant="row")


def test_second_derivatives_are_refused():
    x, res, w = _inputs(3, 64, torch.float32, 1)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="first derivatives"):
        torch.autograd.grad(rms_norm(x, w).square().sum(), x, create_graph=True)
    m = ScaledWeight(*_matrix(32, 64, "mxfp4", 1))
    with pytest.raises(RuntimeError, match="first derivatives"):
        torch.autograd.grad(matvec(x, m).square().sum(), x, create_graph=True)


# ---- matvec ------------------------------------------------------------------------------------------
def _weight64(values, scales, top):
    codes = torch.stack((values & 15, values >> 4), -1).reshape(values.shape[0], -1)
    w = E2M1.to(values.device)[codes.long()]
    group = w.shape[1] // scales.shape[1]
    s = torch.exp2(scales.double() - 127) if scales.dtype == torch.uint8 else scales.double()
    if scales.dtype == torch.uint8:
        s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return w * s.repeat_interleave(group, 1) * (1.0 if top is None else top.double().item())


def _matrix(n, k, kind, seed, lo=-3, hi=3):
    """Any codes; scales are powers of two between 2^lo and 2^hi."""
    g = _gen(seed)
    values = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    if kind == "mxfp4":
        return values, torch.randint(127 + lo, 128 + hi, (n, k // 32), generator=g, device="cuda", dtype=torch.uint8), None
    return values, torch.exp2(torch.randint(lo, hi + 1, (n, k // 16), generator=g, device="cuda").float()).to(torch.float8_e4m3fn), torch.tensor([0.25], device="cuda")


SIZES = [(1, 32), (3, 64), (16, 32), (33, 96), (64, 512), (130, 1024), (127, 2080), (200, 4096), (129, 14336), (1000, 288)]
TOKENS = [1, 2, 7, 8, 9, 16, 33, 64, 100, 129, 300]


def _integers(tokens, k, dtype, seed):
    return torch.randint(-2, 3, (tokens, k), generator=_gen(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("n, k", SIZES)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_matvec_of_whole_numbers_is_exact(n, k, tokens, kind, dtype):
    # products are multiples of 1/16 (1/64 with the global scale) below 2^7; sums of 14336 of them fit 24 bits, whatever their order
    k = k + 16 if kind == "nvfp4" and k % 64 == 32 else k  # rows that end inside a pair of groups
    w = _matrix(n, k, kind, n + k)
    x = _integers(tokens, k, DT[dtype], tokens)
    want = (x.double() @ _weight64(*w).T)
    y = matvec(x, ScaledWeight(*w), out_dtype=torch.float32)
    assert y.shape == (tokens, n) and torch.equal(y.double(), want)
    y = matvec(x, ScaledWeight(*w))
    assert torch.equal(y, want.float().to(x.dtype))


@pytest.mark.parametrize("n, k", SIZES)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("quant", ["row", "block"])
def test_matvec_of_8_bit_whole_numbers_is_exact(n, k, tokens, kind, quant):
    w = _matrix(n, k, kind, n + k)
    x = _integers(tokens, k, torch.float8_e4m3fn, tokens + 1)
    g = _gen(11)
    if quant == "row":
        scales = torch.exp2(torch.randint(-2, 3, (tokens,), generator=g, device="cuda").float())
        x64 = x.double() * scales.double()[:, None]
    else:
        scales = torch.randint(126, 129, (tokens, k // 32), generator=g, device="cuda", dtype=torch.uint8)
        x64 = x.double() * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    want = x64 @ _weight64(*w).T
    y = matvec(ScaledActivations(x, scales), ScaledWeight(*w), out_dtype=torch.float32)
    assert torch.equal(y.double(), want)
    assert torch.equal(matvec(ScaledActivations(x, scales), ScaledWeight(*w)), want.float().to(torch.bfloat16))


def _check_product(y, x64, w64, dtype):
    """One rounding, and a fp32 sum: each of its terms goes through at most k additions, which tensor cores round towards zero
    (twice half a step); 8 more for products, parts of x and scales."""
    want = x64 @ w64.T
    tol = _half_step(dtype) * want.abs() + (w64.shape[1] + 8) * 2 * F32 * (x64.abs() @ w64.abs().T) + _floor(dtype)
    assert bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("tokens", [1, 5, 8, 40, 200])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_matvec_of_normal_values(kind, tokens, dtype):
    specs = (specs_mxfp4 if kind == "mxfp4" else specs_nvfp4)("w", 300, 1056, 3)
    values, scales = (torch.frombuffer(bytearray(s.raw), dtype=torch.uint8).cuda().reshape(300, -1) for s in specs[:2])
    top = torch.frombuffer(bytearray(specs[2].raw), dtype=torch.float32).cuda() if kind == "nvfp4" else None
    scales = scales.view(torch.float8_e4m3fn) if kind == "nvfp4" else scales
    x = (torch.randn(tokens, 1056, generator=_gen(tokens), device="cuda") * 10).to(DT[dtype])
    w64 = _weight64(values, scales, top)
    _check_product(matvec(x, ScaledWeight(values, scales, top)), x.double(), w64, x.dtype)
    # sums that nearly cancel keep their small part: fp32 output against the same bound
    _check_product(matvec(x, ScaledWeight(values, scales, top), out_dtype=torch.float32), x.double(), w64, torch.float32)
    for quant in ("row", "block"):
        y = rms_norm(x, torch.ones(1056, device="cuda"), quant=quant)
        s = y.scales.double()[:, None] if quant == "row" else torch.exp2(y.scales.view(torch.uint8).double() - 127).repeat_interleave(32, 1)
        _check_product(matvec(y, ScaledWeight(values, scales, top), out_dtype=torch.float32), y.values.double() * s, w64, torch.float32)


@pytest.mark.parametrize("tokens", [1, 6, 30, 150])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_matvec_far_apart_magnitudes(tokens, dtype):
    """Tokens and groups of very different size: each is held against its own row, not against the largest."""
    n, k = 70, 512
    values, scales, _ = _matrix(n, k, "mxfp4", 5, -60, 20)
    span = 12 if dtype == "fp16" else 60
    x = torch.randn(tokens, k, generator=_gen(6), device="cuda") * torch.exp2(torch.randint(-span, span // 2, (tokens, 1), generator=_gen(7), device="cuda").float())
    x = x.to(DT[dtype])
    y = matvec(x, ScaledWeight(values, scales), out_dtype=torch.float32)
    _check_product(y, x.double(), _weight64(values, scales, None), torch.float32)


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("tokens", [1, 3, 16, 40])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_matvec_small_values_beside_large_ones(kind, tokens, dtype):
    """What a token holds beside a far larger value is not lost: rows whose weight is zero there are held to their own terms."""
    n, k = 48, 2048
    values, scales, top = _matrix(n, k, kind, 12)
    values[::2, 300] = 0  # columns 600 and 601
    w = ScaledWeight(values, scales, top)
    w64 = _weight64(values, scales, top)
    for power in (20, 30, 36, 45, 70, 120):
        x = torch.randn(tokens, k, generator=_gen(power), device="cuda").to(DT[dtype])
        x[:, 600] = 2.0 ** power
        x[tokens // 2, 601] = 2.0 ** (power // 2)
        x[:, 1000:1010] *= 2.0 ** -20
        _check_product(matvec(x, w, out_dtype=torch.float32), x.double(), w64, torch.float32)


@pytest.mark.parametrize("tokens", [1, 4, 20, 140])
def test_matvec_extreme_scales(tokens):
    """E8M0 from 2^-127 to 2^127, NaN scales, E4M3 subnormals and its largest, infinities and NaN in x."""
    n, k = 40, 256
    g = _gen(8)
    values = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.full((n, k // 32), 127, device="cuda", dtype=torch.uint8)
    scales[0], scales[1], scales[2, 3], scales[3] = 0, 240, 255, 9
    x = torch.randint(-2, 3, (tokens, k), generator=g, device="cuda").float()
    w64 = _weight64(values, scales, None)
    for dtype in (torch.float32, torch.bfloat16):
        y = matvec(x.to(dtype), ScaledWeight(values, scales), out_dtype=torch.float32)
        want = (x.double() @ w64.T).float()
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.nan_to_num(y)[:, 1:], torch.nan_to_num(want)[:, 1:])
        # row 0 is made of terms around the smallest normal number, where a unit may take what is below for zero
        assert bool(((y - want)[:, 0].abs() <= k * 2.0 ** -126).all())
    nv = torch.tensor([2.0 ** -9, 3 * 2.0 ** -9, 448.0, 2.0 ** -6], device="cuda").to(torch.float8_e4m3fn).repeat(n, k // 64)
    y = matvec(x, ScaledWeight(values, nv))
    _check_product(y, x.double(), _weight64(values, nv, None), torch.float32)
    nv = nv.clone()
    nv.view(torch.uint8)[5, 2] = 0x7F
    assert bool(torch.isnan(matvec(x, ScaledWeight(values, nv))[:, 5]).all())
    # an infinity meets no zero in row 4: everything there is infinite with the code's sign; a NaN makes its token's sums NaN
    values[4] = 0x22
    ok = ScaledWeight(values, torch.full_like(scales, 127))
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        z = x.to(dtype).clone()
        z[tokens - 1, 9] = -math.inf
        z[tokens - 1, 10] = 60000.0
        y = matvec(z, ok)
        assert y[tokens - 1, 4] == -math.inf and (tokens == 1 or bool(torch.isfinite(y[:-1]).all()))
        z[tokens - 1, 200] = math.nan
        y = matvec(z, ok)
        assert bool(torch.isnan(y[tokens - 1]).all()) and (tokens == 1 or bool(torch.isfinite(y[:-1]).all()))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 3, 24, 200])
def test_matvec_largest_and_smallest_tokens(dtype, tokens):
    """Tokens at the ends of their type's range, where parts or scaled copies of them could overflow or vanish."""
    n, k = 32, 128
    values, scales, _ = _matrix(n, k, "mxfp4", 4, -4, -4)
    most = torch.finfo(DT[dtype]).max
    for size in (most, 2.0 ** -126, 2.0 ** -120):
        x = torch.zeros(tokens, k, device="cuda", dtype=DT[dtype])
        x[:, 5] = size
        x[0, 70] = -size
        y = matvec(x, ScaledWeight(values, scales), out_dtype=torch.float32)
        want = x.double() @ _weight64(values, scales, None).T
        tol = 2.0 ** -20 * (x.double().abs() @ _weight64(values, scales, None).abs().T) + 2 * 2.0 ** -126  # what is below the normal numbers may count as zero
        assert bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("n, k", SIZES)
@pytest.mark.parametrize("tokens", [1, 7, 16, 65, 130, 300])
@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_matvec_gradient_of_whole_numbers_is_exact(n, k, tokens, kind, dtype):
    k = k + 16 if kind == "nvfp4" and k % 64 == 32 else k
    w = _matrix(n, k, kind, n + k)
    x = _integers(tokens, k, DT[dtype], 1).requires_grad_()
    dy = _integers(tokens, n, DT[dtype], 2)
    dx, = torch.autograd.grad(matvec(x, ScaledWeight(*w)), x, dy)
    want = dy.double() @ _weight64(*w)
    assert dx.shape == x.shape and dx.dtype == x.dtype and torch.equal(dx, want.float().to(x.dtype))


def test_matvec_gradient_against_differences_and_between_types():
    w = _matrix(48, 96, "nvfp4", 3)
    handle = ScaledWeight(*w)
    x = torch.randn(5, 96, generator=_gen(1), device="cuda").requires_grad_()
    c = torch.randn(5, 48, generator=_gen(2), device="cuda")
    (matvec(x, handle) * c).sum().backward()
    w64 = _weight64(*w)
    for i in range(0, 480, 17):  # linear: the difference of two sums is the slope, but for rounding
        m, k = divmod(i, 96)
        step = torch.zeros(5, 96, device="cuda")
        step[m, k] = 1.0
        slope = ((matvec((x + step).detach(), handle).double() - matvec((x - step).detach(), handle).double()) * c.double()).sum().item() / 2
        size = ((x.detach().abs() + 1).double() @ w64.abs().T * c.abs().double()).sum().item()
        assert abs(slope - x.grad[m, k].item()) <= 2 * 104 * 2 * F32 * size
    xb = x.detach().to(torch.bfloat16).requires_grad_()
    y = matvec(xb, handle, out_dtype=torch.float32)
    dx, = torch.autograd.grad(y, xb, c.to(torch.bfloat16).float())
    assert y.dtype == torch.float32 and dx.dtype == torch.bfloat16
    _check_product(dx, c.to(torch.bfloat16).double(), w64.T.contiguous(), torch.bfloat16)


def test_matvec_layouts_of_matrix_and_tokens():
    values, scales, _ = _matrix(96, 1024, "mxfp4", 3)
    x = _integers(6, 1024, torch.bfloat16, 3)
    want = matvec(x, ScaledWeight(values, scales))
    assert torch.equal(matvec(x, ScaledWeight(values.reshape(96, 32, 16), scales)), want)
    assert torch.equal(matvec(x, ScaledWeight(values, scales.view(torch.float8_e8m0fnu))), want)
    if hasattr(torch, "float4_e2m1fn_x2"):
        assert torch.equal(matvec(x, ScaledWeight(values.view(torch.float4_e2m1fn_x2), scales)), want)
    stack = torch.stack((torch.zeros_like(values), values)).reshape(2, 96, 32, 16)
    assert torch.equal(matvec(x, ScaledWeight(stack, torch.stack((scales, scales)), expert=1)), want)
    # views: rows with room behind them, every second row, transposed storage, an odd offset
    room = torch.zeros(96, 1024, dtype=torch.uint8, device="cuda")
    room[:, 16:528] = values
    assert torch.equal(matvec(x, ScaledWeight(room[:, 16:528], scales)), want)
    twice = values.repeat_interleave(2, 0)
    assert torch.equal(matvec(x, ScaledWeight(twice[::2], scales.repeat_interleave(2, 0)[1::2])), want)
    assert torch.equal(matvec(x, ScaledWeight(values.t().contiguous().t(), scales.t().contiguous().t())), want)
    odd = torch.zeros(96 * 512 + 1, dtype=torch.uint8, device="cuda")
    odd[1:] = values.flatten()
    assert torch.equal(matvec(x, ScaledWeight(odd[1:].view(96, 512), scales)), want)
    one = ScaledWeight(values[5:6], scales[5:6])
    assert torch.equal(matvec(x, one), want[:, 5:6])
    # tokens: strided, offset by one element, more dimensions, one vector, none
    assert torch.equal(matvec(x.t().contiguous().t(), ScaledWeight(values, scales)), want)
    flat = torch.zeros(6 * 1024 + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = x.flatten()
    assert torch.equal(matvec(flat[1:].view(6, 1024), ScaledWeight(values, scales)), want)
    assert torch.equal(matvec(x.view(2, 3, 1024), ScaledWeight(values, scales)), want.view(2, 3, 96))
    assert torch.equal(matvec(x[2], ScaledWeight(values, scales)), want[2])
    assert matvec(x[:0], ScaledWeight(values, scales)).shape == (0, 96)
    e = x[:0].clone().requires_grad_()
    assert torch.autograd.grad(matvec(e, ScaledWeight(values, scales)).sum(), e)[0].shape == (0, 1024)
    q = x.to(torch.float8_e4m3fn)
    both = torch.ones(6, 2, device="cuda")
    assert torch.equal(matvec(ScaledActivations(q.t().contiguous().t(), both[:, 0]), ScaledWeight(values, scales)), want)


@pytest.mark.parametrize("tokens", [1, 2, 5, 12, 40])
@pytest.mark.parametrize("quant", [None, "row", "block"])
@pytest.mark.parametrize("sizes", [[64], [16, 8], [300, 33, 7], [1, 2000, 16, 48], [20, 40, 60, 80, 100], [7000, 40]])
def test_projections_of_several_matrices(tokens, quant, sizes):
    """Whole numbers, so that every matrix of a projection gives what it gives alone."""
    k = 1056
    kinds = ["nvfp4", "mxfp4"] if len(sizes) in (3, 5) else ["mxfp4"]
    weights = [ScaledWeight(*_matrix(n, k, kinds[i % len(kinds)], i + n)) for i, n in enumerate(sizes)]
    x = torch.randint(0, 2, (tokens, k), generator=_gen(5), device="cuda").to(torch.bfloat16) * 2 - 1  # a root mean square of one
    p = Projection(torch.ones(k, device="cuda", dtype=torch.bfloat16), weights, eps=0.0, quant=quant)
    ys, h = p(x)
    assert torch.equal(h, x) and len(ys) == len(sizes)
    same = rms_norm(x, torch.ones(k, device="cuda", dtype=torch.bfloat16), 0.0, quant=quant)  # with row scales that is 448 times 1/448, as fp32 has it
    for y, w, n in zip(ys, weights, sizes):
        assert y.shape == (tokens, n) and torch.equal(y, matvec(same, w, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("quant", [None, "row", "block"])
@pytest.mark.parametrize("shape", [(512,), (3, 512), (2, 3, 512), (0, 512), (2, 0, 512)])
def test_projections_of_any_number_of_dimensions(shape, quant):
    w = ScaledWeight(*_matrix(256, 512, "mxfp4", 3))
    norm = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(*shape, generator=_gen(3), device="cuda").to(torch.bfloat16)
    (y,), h = Projection(norm, [w], quant=quant)(x, x)
    q, k = rms_norm(x, norm, residual=x, quant=quant)
    assert y.shape == (*shape[:-1], 256) and h.shape == x.shape and torch.equal(h, k)
    assert torch.equal(y, matvec(q, w))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("offset", [0, 1])
def test_values_that_are_not_finite_stay_in_their_token(dtype, offset):
    """Tokens that are laid out anew: the largest numbers, infinities and NaN, from a 16-byte boundary and from beside one."""
    values, scales, _ = _matrix(48, 256, "mxfp4", 5)
    values = values & 0x77 | 0x11   # no zero, no sign: an infinity stays one
    w = ScaledWeight(values, scales)
    dt = DT[dtype]
    flat = torch.zeros(40 * 256 + 1, dtype=dt, device="cuda")
    x = flat[offset:offset + 40 * 256].view(40, 256)
    x.copy_(torch.randn(40, 256, generator=_gen(6), device="cuda"))
    want = matvec(x, w, out_dtype=torch.float32)
    x[3, 7], x[4, 250], x[5, 0], x[6] = math.inf, math.nan, -math.inf, 0
    x[6, 9] = torch.finfo(dt).max
    got = matvec(x, w, out_dtype=torch.float32)
    keep = [i for i in range(40) if i not in (3, 4, 5, 6)]
    assert torch.equal(got[keep], want[keep])
    assert bool((got[3] == math.inf).all()) and bool(torch.isnan(got[4]).all()) and bool((got[5] == -math.inf).all())
    w64 = _weight64(values, scales, None)
    top = torch.finfo(dt).max * w64[:, 9]
    fits = top < torch.finfo(torch.float32).max   # one product, of parts whose sums are exact
    assert bool(((got[6].double() - top).abs() <= 2.0 ** -20 * top)[fits].all())


def test_a_token_does_not_depend_on_its_neighbours():
    """The same token gives the same bits beside others that hold infinities, as long as as many are asked for."""
    w = ScaledWeight(*_matrix(200, 2048, "nvfp4", 3))
    for tokens in (2, 8, 40, 200):
        x = torch.randn(tokens, 2048, generator=_gen(3), device="cuda").to(torch.bfloat16)
        a = matvec(x, w)
        assert torch.equal(a, matvec(x, w))
        z = x.clone()
        z[1:] = math.inf
        assert torch.equal(matvec(z, w)[0], a[0])


def test_refusals():
    values, scales, top = _matrix(64, 128, "nvfp4", 1)
    mx_values, mx_scales, _ = _matrix(64, 128, "mxfp4", 1)
    w = ScaledWeight(values, scales, top)
    x = torch.zeros(2, 128, device="cuda")
    for bad in [lambda: ScaledWeight(values.float(), scales), lambda: ScaledWeight(values, scales.float()), lambda: ScaledWeight(values, scales, top.double()),
                lambda: ScaledWeight(values, scales, torch.ones(2, device="cuda")), lambda: matvec(x.double(), w), lambda: matvec(x, w, out_dtype=torch.float64),
                lambda: rms_norm(x.double(), x[0]), lambda: ScaledActivations(x, x[:, 0]), lambda: ScaledActivations(x.to(torch.float8_e4m3fn), x[:, 0].half()),
                lambda: matvec(x, values)]:
        with pytest.raises(TypeError):
            bad()
    for bad in [lambda: ScaledWeight(values, scales[:, :-1]), lambda: ScaledWeight(values[:, :-4], scales), lambda: ScaledWeight(mx_values, mx_scales, top),
                lambda: ScaledWeight(values[None], scales[None]), lambda: ScaledWeight(values[:0], scales[:0]), lambda: ScaledWeight(values, scales, top.cpu()),
                lambda: matvec(x[:, :64], w), lambda: matvec(x.cpu(), w), lambda: rms_norm(x, x[0, :64]), lambda: rms_norm(x, x[0], quant="int8"),
                lambda: rms_norm(x[:, :40], x[0, :40], quant="block"), lambda: rms_norm(x, x[0], residual=x[:1]), lambda: rms_norm(x, x[0], residual=x.half()),
                lambda: rms_norm(x[:, :0], x[0, :0]), lambda: ScaledActivations(x.to(torch.float8_e4m3fn), x[:, :2]), lambda: ScaledActivations(x[:, :40].to(torch.float8_e4m3fn), mx_scales[:2, :1]),
                lambda: Projection(x[0, :64], [w]), lambda: Projection(x, [w]), lambda: Projection(x[0], [w], quant="int8")]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(IndexError):
        ScaledWeight(values[None], scales[None], expert=1)


# ---- streams, graphs, containers ------------------------------------------------------------------------
def test_streams_and_overlapping_calls():
    w = ScaledWeight(*_matrix(1024, 2048, "mxfp4", 3))
    streams = [torch.cuda.Stream() for _ in range(3)]
    xs = [_integers(t, 2048, torch.bfloat16, t) for t in (1, 16, 100)]
    want = [matvec(x, w) for x in xs]
    norm = torch.ones(2048, device="cuda")
    want_norm = [rms_norm(x, norm, quant="row").values.view(torch.uint8) for x in xs]
    torch.cuda.synchronize()
    got = []
    for turn in range(20):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append((matvec(x, w), rms_norm(x, norm, quant="row").values.view(torch.uint8)))
    torch.cuda.synchronize()
    for i, (y, q) in enumerate(got):
        assert torch.equal(y, want[i % 3]) and torch.equal(q, want_norm[i % 3])


@pytest.mark.parametrize("tokens", [1, 12, 130])
def test_captured_and_replayed(tokens):
    w = ScaledWeight(*_matrix(512, 1024, "nvfp4", 3))
    norm = torch.ones(1024, device="cuda", dtype=torch.bfloat16)
    p = Projection(norm, [w, w], quant="block")
    x = torch.randn(tokens, 1024, generator=_gen(1), device="cuda").to(torch.bfloat16)
    res = torch.randn(tokens, 1024, generator=_gen(2), device="cuda").to(torch.bfloat16)
    p(x, res)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same handles, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = p(x, res)
        graphs.append((g, out))
    for seed in (3, 4):
        x.copy_(torch.randn(tokens, 1024, generator=_gen(seed), device="cuda"))
        for g, _ in graphs:
            g.replay()
        (y1, y2), h = p(x, res)
        for _, ((z1, z2), k) in graphs:
            assert torch.equal(z1, y1) and torch.equal(z2, y2) and torch.equal(k, h)


def test_gradients_captured_and_replayed():
    w = ScaledWeight(*_matrix(256, 512, "mxfp4", 3))
    norm = torch.ones(512, device="cuda", requires_grad=True)
    x = torch.randn(40, 512, generator=_gen(1), device="cuda", requires_grad=True)
    res = torch.randn(40, 512, generator=_gen(2), device="cuda", requires_grad=True)
    dy = torch.randn(40, 256, generator=_gen(3), device="cuda")

    def step():
        (y,), h = Projection(norm, [w])(x, res)
        return torch.autograd.grad((y, h), (x, norm, res), (dy, torch.ones_like(h)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    with torch.no_grad():
        x.copy_(torch.randn(40, 512, generator=_gen(5), device="cuda"))
    g.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows, cols", [(5, 4096), (40, 517), (700, 9), (3, 16416), (3, 20003), (2, 10008)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_the_sum_may_be_written_over_an_input(rows, cols, dtype, place):
    x, res, w = _inputs(rows, cols, DT[dtype], rows + cols)
    y, h = rms_norm(x, w, 1e-5, residual=res)
    torch.cuda.synchronize()
    into, out = {"x": x, "residual": res}[place].clone(), torch.empty_like(x)
    ins = {"x": x, "residual": res, place: into}
    code = {"bf16": 6, "fp32": 1}[dtype]
    torch.cuda.synchronize()
    assert ptwm_b200._lib.lib().ptwm_b200_rms_norm(ins["x"].data_ptr(), ins["residual"].data_ptr(), w.data_ptr(), into.data_ptr(), out.data_ptr(), 0, rows, cols, code, code, 0, 1e-5, 0, 1) == 0
    torch.cuda.synchronize()
    assert torch.equal(into, h) and torch.equal(out, y)


def test_nothing_is_written_outside_the_results():
    w = ScaledWeight(*_matrix(100, 512, "mxfp4", 3))
    room = torch.full((1 << 22,), 7, dtype=torch.uint8, device="cuda")
    L, stream = ptwm_b200._lib.lib(), 1
    x = _integers(20, 512, torch.float32, 2)
    torch.cuda.synchronize()
    at = room.data_ptr() + 4096
    assert L.ptwm_b200_matvec(w._ref, x.data_ptr(), 0, at, 8, 1, 0, 1, 0, 0, 0, stream) == 0
    torch.cuda.synchronize()
    end = 4096 + 8 * 100 * 4
    assert bool((room[:4096] == 7).all()) and bool((room[end:] == 7).all())
    for call, cols, tokens in ((L.ptwm_b200_matvec, 100, 20), (L.ptwm_b200_matvec_grad, 512, 9)):  # any 9 x 100 numbers do as a gradient
        room.fill_(7)
        grad = int(call is L.ptwm_b200_matvec_grad)
        size = L.ptwm_b200_matvec_scratch_bytes(w._ref, x.data_ptr(), tokens, 1, grad)
        there = room.data_ptr() + (1 << 21)
        more = () if grad else (0,)
        types = (1,) if grad else (1, 0, 1)
        torch.cuda.synchronize()
        assert call(w._ref, x.data_ptr(), *more, at, tokens, *types, there, size - 1, 0, stream) == -2
        assert call(w._ref, x.data_ptr(), *more, at, tokens, *types, there + 8, size, 0, stream) == -1
        assert call(w._ref, x.data_ptr(), *more, at, tokens, *types, there, size, 0, stream) == 0
        torch.cuda.synchronize()
        end = 4096 + tokens * cols * 4
        assert bool((room[:4096] == 7).all()) and bool((room[end:1 << 21] == 7).all()) and bool((room[(1 << 21) + size:] == 7).all())
    room.fill_(7)
    torch.cuda.synchronize()
    wt = torch.ones(511, device="cuda")
    assert L.ptwm_b200_rms_norm(x.data_ptr(), 0, wt.data_ptr(), 0, at, room.data_ptr() + (1 << 20), 3, 511, 1, 1, 1, 1e-6, 0, stream) == 0
    torch.cuda.synchronize()
    assert bool((room[:4096] == 7).all()) and bool((room[4096 + 3 * 511:1 << 20] == 7).all()) and bool((room[(1 << 20) + 12:] == 7).all())


def test_no_wait_has_given_up():
    assert ptwm_b200._lib.lib().ptwm_b200_operator_status(0) == 0


def test_weights_straight_from_a_container(tmp_path):
    specs = mixed_model()
    specs += [spec_norm("blk.norm2.weight", 256, 21)]
    for spec in specs_nvfp4("blk.nv2", 160, 256, 22):
        specs.append(spec)
    blob = oracle.write_container(specs, chunk_size=4096, emit_crc=True, emit_hash=True, menu=(oracle.IDENTITY, oracle.HUFFMAN, oracle.RANS, oracle.O1SAC))
    path = tmp_path / "m.ptwm"
    path.write_bytes(blob)
    raw = {s.name: s for s in specs}
    handle = ptwm_b200.ContainerHandle(blob)
    state = ptwm_b200.load_file(path)
    index, opened = ptwm_b200.TensorIndex(path), ptwm_b200.SafeOpen(path)
    x = torch.randn(3, 256, generator=_gen(1), device="cuda").to(torch.bfloat16)
    for name, values, scales, top in (("blk.mx", "blk.mx_blocks", "blk.mx_scales", None), ("blk.nv", "blk.nv.weight", "blk.nv.weight_scale", "blk.nv.weight_scale_2")):
        v = torch.from_numpy(np.frombuffer(raw[values].raw, dtype=np.uint8).copy()).reshape(raw[values].shape)
        s = torch.from_numpy(np.frombuffer(raw[scales].raw, dtype=np.uint8).copy()).reshape(raw[scales].shape)
        g = None if top is None else torch.from_numpy(np.frombuffer(raw[top].raw, dtype=np.float32).copy())
        w64 = _weight64(v, s if top is None else s.view(torch.float8_e4m3fn), g).cuda()
        w = handle.scaled_weight(name)
        assert w.shape == (96, 256) and w.kind == ("mxfp4" if top is None else "nvfp4")
        y = matvec(x, w)
        _check_product(y, x.double(), w64, torch.bfloat16)
        for other in (ScaledWeight.from_state(state, name), index.get_scaled_weight(name), opened.get_scaled_weight(name)):
            assert torch.equal(matvec(x, other), y)
    with pytest.raises(KeyError):
        handle.scaled_weight("blk.q")
    # a norm and the two matrices behind it, as a block of a model runs them
    p = handle.projection("blk.norm2.weight", ["blk.nv", "blk.nv2"], eps=1e-5, quant="block")
    res = torch.randn(3, 256, generator=_gen(2), device="cuda").to(torch.bfloat16)
    (a, b), h = p(x, res)
    q, k = rms_norm(x, handle.decode("blk.norm2.weight"), 1e-5, residual=res, quant="block")
    assert torch.equal(h, k) and torch.equal(a, matvec(q, handle.scaled_weight("blk.nv"))) and torch.equal(b, matvec(q, handle.scaled_weight("blk.nv2")))
    assert a.shape == (3, 96) and b.shape == (3, 160) and a.dtype == torch.bfloat16
    with pytest.raises(KeyError):
        handle.projection("blk.none", ["blk.nv"])


def test_tensor_sizes_beyond_32_bits():
    """Offsets into x and y that pass 2^31 elements."""
    rows, cols = 262145, 8224
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn(cols, generator=_gen(1), device="cuda")
    w = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    y = rms_norm(x, w, quant="block")
    one = rms_norm(x[-1:], w, quant="block")
    assert torch.equal(y.values.view(torch.uint8)[-1], one.values.view(torch.uint8)[0]) and torch.equal(y.scales.view(torch.uint8)[-1], one.scales.view(torch.uint8)[0])
    m = ScaledWeight(*_matrix(16, cols, "mxfp4", 2))
    got = matvec(y, m)
    assert bool((got[:-200] == 0).all())
    want = matvec(one, m, out_dtype=torch.float32).double()
    assert bool(((got[-1].double() - want[0]).abs() <= 2.0 ** -7 * want[0].abs() + 1e-3 * want.abs().max()).all())


@pytest.mark.parametrize("rows, cols", [(5, 4096), (700, 256), (40, 8192), (3, 16384), (300, 4097), (9, 513), (3, 10001), (3, 16384 + 8), (2, 40000)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("power, eps", [(45, 1e-5), (55, 1e-5), (-45, 0.0), (-55, 0.0)])
@pytest.mark.parametrize("place", [0, 1])
def test_norm_gradient_of_very_large_and_small_rows(rows, cols, dtype, power, eps, place):
    """Rows whose squares fit fp32 where the third power of their root mean square, or of its inverse, does not.  place: in values, from
    a boundary of 16 bytes."""
    dt = DT[dtype]
    g = _gen(rows + cols + power)

    def placed(t):
        flat = torch.zeros(t.numel() + place, dtype=dt, device="cuda")
        flat[place:] = t.to(dt).flatten()
        return flat[place:].view(t.shape)

    x = placed(torch.randn(rows, cols, generator=g, device="cuda") * 2.0 ** power).requires_grad_()
    w = placed(1 + 0.1 * torch.randn(cols, generator=g, device="cuda")).requires_grad_()
    dy = placed(torch.randn(rows, cols, generator=g, device="cuda") + x.detach().float() * 2.0 ** -power)  # (a part along x: the second term counts)
    dx, dw = torch.autograd.grad(rms_norm(x, w, eps), (x, w), dy)
    h = x.detach().double()
    r = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    gw = dy.double() * w.detach().double()
    mean = (gw * h).mean(-1, keepdim=True)
    want = r * gw - h * r ** 3 * mean
    size = r * gw.abs() + (h * r ** 3).abs() * (gw * h).abs().mean(-1, keepdim=True)
    tol = _half_step(dt) * want.abs() + 4 * _norm_slack(cols) * size + _floor(dt)
    assert bool(((dx.double() - want).abs() <= tol).all())
    terms = dy.double() * h * r
    tol = _half_step(dt) * terms.sum(0).abs() + ((rows + 16) * F32 + 2 * _norm_slack(cols)) * terms.abs().sum(0) + _floor(dt)
    assert bool(((dw.double() - terms.sum(0)).abs() <= tol).all())


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("tokens", [1, 6, 40, 200])
@pytest.mark.parametrize("dtype, out", [("bf16", "fp32"), ("fp16", "fp32"), ("bf16", "fp16"), ("fp16", "bf16"), ("fp32", "bf16"), ("fp32", "fp16")])
def test_matvec_gradient_from_an_output_of_another_type(kind, tokens, dtype, out):
    """The gradient of an output is used as it comes: one rounding, into x's type, behind the sum."""
    n, k = 160, 96
    w = _matrix(n, k, kind, 21)
    x = torch.randn(tokens, k, generator=_gen(1), device="cuda").to(DT[dtype]).requires_grad_()
    dy = torch.randn(tokens, n, generator=_gen(2), device="cuda").to(DT[out])
    dx, = torch.autograd.grad(matvec(x, ScaledWeight(*w), out_dtype=DT[out]), x, dy)
    assert dx.dtype == x.dtype
    _check_product(dx, dy.double(), _weight64(*w).T.contiguous(), x.dtype)


@pytest.mark.parametrize("tokens", [1, 30, 150])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_matvec_gradient_of_fp32_outputs_keeps_small_differences_and_large_values(tokens, dtype):
    # one nonzero to a column, or two that nearly cancel: the products and their sums are exact, and fit x's type where dy would not
    n, k = 64, 64
    codes = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    codes[0, 0], codes[1, 0], codes[2, 33], codes[3, 32 + 31] = 2, 10, 2, 2  # 1, -1, 1, 1
    scales = torch.full((n, 2), 127, dtype=torch.uint8, device="cuda")
    scales[2, 1], scales[3, 1] = 117, 157  # 2^-10, 2^30
    w = ScaledWeight(codes[:, 0::2] | codes[:, 1::2] << 4, scales)
    x = torch.zeros(tokens, k, device="cuda", dtype=DT[dtype], requires_grad=True)
    dy = torch.zeros(tokens, n, device="cuda")
    dy[:, 0], dy[:, 1] = 1 + 2.0 ** -20, 1.0
    dy[:, 2] = 100352.0     # past fp16: 98 in dx
    dy[:, 3] = 5 * 2.0 ** -33  # below half its smallest step
    dx, = torch.autograd.grad(matvec(x, w, out_dtype=torch.float32), x, dy)
    want = torch.zeros(tokens, k, device="cuda")
    want[:, 0], want[:, 33], want[:, 63] = 2.0 ** -20, 98.0, 0.625
    assert torch.equal(dx.float(), want.to(DT[dtype]).float())


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_of_handles_multiply_by_their_own_matrix(kind, how):
    values, scales, top = _matrix(80, 544, kind, 13)
    room = torch.zeros(80, 640, dtype=torch.uint8, device="cuda")
    room[:, :272] = values
    x = _integers(5, 544, torch.bfloat16, 2)
    w = ScaledWeight(room[:, :272], scales, top)
    p = Projection(torch.ones(544, device="cuda", dtype=torch.bfloat16), [w, w], quant="block" if kind == "mxfp4" else None)
    want, pair = matvec(x, w), p(x)[0]
    c, q = how(w), how(p)
    if how is not copy.copy:
        room.fill_(0x11)
        assert not torch.equal(matvec(x, w), want)
    assert torch.equal(matvec(x, c), want)
    for y, z in zip(q(x)[0], pair):
        assert torch.equal(y, z)


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("tokens", [1, 2, 3, 16])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_matvec_tiny_tokens_far_below_others_against_large_scales(kind, tokens, dtype):
    """Tokens at the low end of their type whose smallest values are a part of their own: it is undone by a power of two that fp32 does not hold."""
    n, k = 32, 512
    codes = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    codes[:, 40], codes[1::2, 300] = 2, 2  # ones; the even rows do not see the large value
    packed = codes[:, 0::2] | codes[:, 1::2] << 4
    if kind == "mxfp4":
        scales, top, factor = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda"), None, 2.0 ** 120
        scales[0::2, 1] = 247
    else:
        scales, top, factor = torch.ones(n, k // 16, device="cuda").to(torch.float8_e4m3fn), torch.tensor([2.0 ** 100], device="cuda"), 2.0 ** 108
        scales[0::2, 2] = 256.0
    x = torch.zeros(tokens, k, device="cuda")
    for large, small in ((-104, -133), (-100, -126), (-88, -120), (-60, -118)):
        x[:, 300], x[:, 40] = 2.0 ** large, 2.0 ** small
        y = matvec(x.to(DT[dtype]), ScaledWeight(packed, scales, top), out_dtype=torch.float32)
        # one product in a row, by powers of two: exact unless it, before NVFP4's global scale, is below the normal numbers
        assert bool((y[:, 0::2] == 2.0 ** small * factor).all()), (large, small)


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("tokens", [1, 2, 3, 16])
def test_matvec_smallest_8_bit_tokens_against_large_scales(kind, tokens):
    """E4M3's smallest number on the smallest block scale, 2^-136, beside values that leave it to a second part: 2^-25 once the largest is 2^14."""
    n, k = 32, 512
    codes = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    codes[:, 40], codes[1::2, 300] = 2, 2
    packed = codes[:, 0::2] | codes[:, 1::2] << 4
    if kind == "mxfp4":
        scales, top, factor = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda"), None, 2.0 ** 120
        scales[0::2, 1] = 247
    else:
        scales, top, factor = torch.ones(n, k // 16, device="cuda").to(torch.float8_e4m3fn), torch.tensor([2.0 ** 100], device="cuda"), 2.0 ** 108
        scales[0::2, 2] = 256.0
    x = torch.zeros(tokens, k, device="cuda")
    x[:, 300], x[:, 40] = 1.0, 2.0 ** -9
    for large in range(-110, -84):
        blocks = torch.full((tokens, k // 32), 127 + large, dtype=torch.uint8, device="cuda")
        blocks[:, 1] = 0
        y = matvec(ScaledActivations(x.to(torch.float8_e4m3fn), blocks), ScaledWeight(packed, scales, top), out_dtype=torch.float32)
        assert bool((y[:, 0::2] == 2.0 ** -136 * factor).all()), large


@pytest.mark.filterwarnings("ignore::DeprecationWarning")  # torch.func's own
def test_forward_mode_derivatives_are_refused():
    """A dual tensor has no requires_grad; its tangent is not dropped."""
    from torch.autograd import forward_ad
    x, res, w = _inputs(3, 64, torch.float32, 1)
    m = ScaledWeight(*_matrix(32, 64, "mxfp4", 1))
    plain, product = rms_norm(x, w), matvec(x, m)
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, res, w)]
        for call in (lambda: rms_norm(dual[0], w), lambda: rms_norm(x, dual[2]), lambda: rms_norm(x, w, residual=dual[1]), lambda: rms_norm(dual[0], w, quant="row"), lambda: matvec(dual[0], m),
                     lambda: Projection(w, [m])(dual[0]), lambda: Projection(dual[2], [m])(x), lambda: matvec(ScaledActivations(x.to(torch.float8_e4m3fn), dual[0][:, 0]), m)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            matvec(dual[0], m)
        assert torch.equal(rms_norm(x, w), plain) and torch.equal(matvec(x, m), product)
        leaf = x.clone().requires_grad_()
        for y in (rms_norm(leaf, w), matvec(leaf, m)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: rms_norm(t, w), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: matvec(t, m), (x,), (torch.ones_like(x),))


def test_8_bit_tokens_whose_gradient_would_be_lost_are_refused():
    m = ScaledWeight(*_matrix(32, 64, "mxfp4", 1))
    x = torch.randn(3, 64, generator=_gen(1), device="cuda", requires_grad=True)
    scales = x.abs().amax(-1) / 448
    values = (x / scales[:, None]).to(torch.float8_e4m3fn)
    for tokens in (ScaledActivations(values.detach(), scales), ScaledActivations(values, scales.detach())):
        with pytest.raises(ValueError, match="no gradient"):
            matvec(tokens, m)
        with torch.no_grad():
            y = matvec(tokens, m)
        assert torch.equal(y, matvec(ScaledActivations(values.detach(), scales.detach()), m))


def test_a_call_with_too_little_scratch_writes_nothing():
    few, many = ScaledWeight(*_matrix(16, 8192, "mxfp4", 1)), ScaledWeight(*_matrix(14336, 8192, "mxfp4", 2))
    x = _integers(12, 8192, torch.float16, 3)
    ys = [torch.full((12, w.rows), 7.0, device="cuda", dtype=torch.float16) for w in (few, many)]
    refs, at = (ctypes.c_uint64 * 2)(few._ref, many._ref), (ctypes.c_uint64 * 2)(*[y.data_ptr() for y in ys])
    torch.cuda.synchronize()
    assert ptwm_b200._lib.lib().ptwm_b200_matvec_group(refs, at, 2, x.data_ptr(), 0, 12, 4, 0, 4, 0, 0, 0, 1) == -2
    torch.cuda.synchronize()
    assert all(bool((y == 7.0).all()) for y in ys)
    norm = torch.ones(8192, device="cuda", dtype=torch.float16)
    for y, w in zip(Projection(norm, [few, many])(x)[0], (few, many)):
        assert torch.equal(y, matvec(rms_norm(x, norm), w))


def test_the_status_from_python():
    for device in (None, 0, "cuda", "cuda:0", torch.device("cuda", 0)):
        assert ptwm_b200.operator_status(device) == 0
    with pytest.raises(ptwm_b200.PtwmError):
        ptwm_b200.operator_status(1000)


def _one_to_a_row(n, k, kind, seed, along_columns=False):
    """Ones, halves and fours, one to a row (and, where along_columns, rather one to a column): every sum has one product, which is exact."""
    g = _gen(seed)
    codes = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    picks = torch.tensor([1, 2, 6, 9, 10, 14], dtype=torch.uint8, device="cuda")
    if along_columns:
        codes[torch.randint(0, n, (k,), generator=g, device="cuda"), torch.arange(k, device="cuda")] = picks[torch.randint(0, 6, (k,), generator=g, device="cuda")]
    else:
        codes[torch.arange(n, device="cuda"), torch.randint(0, k, (n,), generator=g, device="cuda")] = picks[torch.randint(0, 6, (n,), generator=g, device="cuda")]
    _, scales, top = _matrix(n, k, kind, seed)
    return codes[:, 0::2] | codes[:, 1::2] << 4, scales, top


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("tokens", [1, 2, 7, 16, 33, 130, 300])
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_every_bit_of_a_token_counts(kind, tokens, dtype):
    """All significant bits of fp16 (11) and fp32 (24), which are several parts of fewer bits: each product and its sum are exact, but for fp32
    where tokens are few, whose two parts of eleven bits and a sign hold a value to 2^-23."""
    n, k = 200, 544
    x = (torch.randn(tokens, k, generator=_gen(4), device="cuda") * 3).to(DT[dtype])
    w = _one_to_a_row(n, k, kind, 5)
    want = x.double() @ _weight64(*w).T
    y = matvec(x, ScaledWeight(*w), out_dtype=torch.float32).double()
    if dtype == "fp32" and tokens <= 16:
        assert bool(((y - want).abs() <= (2.0 ** -23 + 2.0 ** -24) * want.abs()).all())  # and the sum of the two parts is rounded once
    else:
        assert torch.equal(y, want)
    w = _one_to_a_row(n, k, kind, 6, along_columns=True)
    dy = (torch.randn(tokens, n, generator=_gen(7), device="cuda") * 3).to(DT[dtype])
    dx, = torch.autograd.grad(matvec(x.requires_grad_(), ScaledWeight(*w)), x, dy)
    assert torch.equal(dx.double(), (dy.double() @ _weight64(*w)).to(dx.dtype).double())  # exact, but for what fp16 has below its normal numbers


@pytest.mark.parametrize("tokens", [24, 200])
@pytest.mark.parametrize("grad", [False, True])
def test_a_long_sum_in_fp32_does_not_lose_what_is_small(tokens, grad):
    """2^28 and then ones: sixteen of them, what an MMA adds, are half a step of the sum.  Sums of 256 are apart, so all but the first 255 ones
    count, and 256 are a multiple of the step; sums in one piece would lose all of them."""
    n = 14336
    codes = torch.full((128, n) if not grad else (n, 128), 0x22, dtype=torch.uint8, device="cuda")[:, ::2].contiguous()
    w = ScaledWeight(codes, torch.full((codes.shape[0], codes.shape[1] // 16), 127, dtype=torch.uint8, device="cuda"))
    v = torch.ones(tokens, n, device="cuda")
    v[:, 0] = 2.0 ** 28
    if grad:
        x = torch.zeros(tokens, 128, device="cuda", requires_grad=True)
        y, = torch.autograd.grad(matvec(x, w), x, v)
    else:
        y = matvec(v, w)
    assert bool(((y.double() - (2.0 ** 28 + n - 1)).abs() <= 255 + 16).all())  # and the last rounding: half a step of 32


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("tokens", [1, 3, 8, 16])
def test_a_long_sum_of_few_fp32_tokens_does_not_lose_what_is_small(tokens, kind):
    """As above: the sums of 256 columns are apart, and what the one with 2^28 in it loses is at most the ones in it."""
    n, k = 4096, 14336
    values = torch.full((n, k // 2), 0x22, dtype=torch.uint8, device="cuda")
    w = ScaledWeight(values, torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")) if kind == "mxfp4" else ScaledWeight(values, torch.ones(n, k // 16, device="cuda").to(torch.float8_e4m3fn))
    x = torch.ones(tokens, k, device="cuda")
    x[:, 0] = 2.0 ** 28
    assert bool(((matvec(x, w).double() - (2.0 ** 28 + k - 1)).abs() <= 255 + 16).all())


def test_a_call_that_failed_leaves_no_error_to_the_next():
    blob = oracle.write_container([spec_norm("n.weight", 4096, 3)], chunk_size=4096, menu=(oracle.RANS,))
    want = ptwm_b200.ContainerHandle(blob).decode("n.weight")
    L = ptwm_b200._lib.lib()
    for rc in (lambda: L.ptwm_b200_operator_status(1000), lambda: L.ptwm_b200_rms_norm(want.data_ptr(), 0, want.data_ptr(), 0, want.data_ptr(), 0, 1, 8, 1, 1, 0, 1e-6, 1000, 1)):
        assert rc() == -7 and "ordinal" in ptwm_b200._lib.last_error()
        assert torch.equal(ptwm_b200.ContainerHandle(blob).decode("n.weight"), want)
