"""Layer norm, dropout, residual addition with dropout and norm, and GELU against plain forms in 64 bits.

Tolerances count roundings.  eps_t = finfo(t).eps / 2 is the most by which one rounding to t is off, relative to the
value.  The arithmetic is fp32 and each output is rounded once to t, so an output v may be off by eps_t |v| for that
rounding, plus the fp32 part: a norm's row is a chain of fewer than ten fp32 operations on values of the order of
|h w| + |b| (h: normalised value) behind two sums of `width` terms.  A sum over n terms that are added in blocks
of at most L in sequence (threads' own, then a tree) is off by at most (L + log2 n) eps_32 times the sum of magnitudes; here
L <= 128 for rows, so every such mean is off by less than 200 eps_32 times the mean magnitude.  Where an output is
scaled by 1 / sigma, so is the error of the mean.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from conftest import ROOT  # noqa: F401

pytestmark = pytest.mark.gpu

E32 = torch.finfo(torch.float32).eps / 2
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def mask64(shape, rate, seed):
    """Which elements are kept, in Python's own integers by way of numpy's uint64."""
    n = int(np.prod(shape))
    with np.errstate(over="ignore"):
        z = np.uint64(seed % 2 ** 64) + np.arange((n + 1) // 2, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    draws = np.stack([z & np.uint64(0xFFFFFFFF), z >> np.uint64(32)], 1).reshape(-1)[:n]
    return torch.from_numpy((draws >= np.uint64(int(float(np.float32(rate)) * 2.0 ** 32))).reshape(shape))


def drop64(x, rate, seed):
    if rate == 0:
        return x
    return torch.where(mask64(x.shape, rate, seed).to(x.device), x / (1 - rate), torch.zeros((), dtype=x.dtype, device=x.device))


def norm64(v, w, b, eps):
    mu = v.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((v - mu) ** 2).mean(-1, keepdim=True) + eps)
    h = (v - mu) * r
    return h * w + b, h, r


def norm_grads64(g, h, r, w):
    a = g * w
    dv = r * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
    dims = tuple(range(g.dim() - 1))
    return dv, (g * h).sum(dims), g.sum(dims)


def check(got, want, t, scale, what, extra=0.0):
    """|got - want| <= half a step of t at want + 256 eps_32 * scale + extra; `scale` bounds the magnitudes that were added."""
    got, want = got.detach().double(), want.double()
    bound = half_step(t) * want.abs() * (1 + 1e-6) + 256 * E32 * scale + extra
    # below the smallest normal number a rounding is off by half of the smallest step
    bound = bound + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    off = (got - want).abs() - bound
    assert not torch.isnan(got).any(), what
    assert off.max().item() <= 0, f"{what}: {off.max().item():.3g} over the bound"


def inputs(shape, t, seed, device, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64) + mean
    return x.to(t).to(device)


def params(width, t, seed, device):
    g = torch.Generator().manual_seed(seed)
    w = 1 + 0.2 * torch.randn(width, generator=g, dtype=torch.float64)
    b = 0.1 * torch.randn(width, generator=g, dtype=torch.float64)
    return w.to(t).to(device), b.to(t).to(device)


def check_norm(y, v, w, b, eps, t, what):
    """v: what was normalised, in 64 bits."""
    want, h, r = norm64(v, w, b, eps)
    scale = (1 + h.abs() + v.abs().mean(-1, keepdim=True) * r) * w.abs() + b.abs()
    check(y, want, t, scale, what)
    return h, r


def check_norm_grads(got, g, h, r, w, t, pt, what, gs=None):
    dv, dw, db = norm_grads64(g, h, r, w)
    a = (g * w).abs()
    scale = r * (a + a.mean(-1, keepdim=True) + h.abs() * (a * h.abs()).mean(-1, keepdim=True)) * (2 + h.abs())
    if gs is not None:
        dv, scale = dv + gs, scale + gs.abs()
    check(got[0], dv, t, scale, what + " dx")
    dims = tuple(range(g.dim() - 1))
    # sums over the rows: a thread adds at most a few hundred terms, partial sums are added in blocks
    if got[1] is not None:
        check(got[1], dw, pt, 4 * (g.abs() * (h.abs() + 1)).sum(dims), what + " dw")
    if got[2] is not None:
        check(got[2], db, pt, 4 * g.abs().sum(dims), what + " db")
    return dv, scale


WIDTHS = [1, 2, 3, 7, 32, 40, 64, 100, 129, 197, 256, 768, 1000, 1001, 1283, 2048, 2050, 4096, 4104, 5120, 8192, 8193,
          8200, 16384, 16385, 40000, 70001]


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_layer_norm_forward_and_gradients(cuda, width, t):
    from mamtorch_b200.nn import functional as MF

    for rows in (1, 3, 37, 700) if width <= 8200 else (1, 5, 200):
        for pt in {t, torch.float32}:
            x = inputs((rows, width), t, 1, cuda).requires_grad_()
            w, b = (p.requires_grad_() for p in params(width, pt, 2, cuda))
            g = inputs((rows, width), t, 3, cuda, 0.0)
            y = MF.layer_norm(x, w, b, 1e-5)
            assert y.dtype == t and y.shape == x.shape
            what = f"{rows}x{width} {t} {pt}"
            x64, w64, b64 = x.detach().double(), w.detach().double(), b.detach().double()
            h, r = check_norm(y, x64, w64, b64, 1e-5, t, what)
            got = torch.autograd.grad(y, (x, w, b), g)
            assert got[1].dtype == pt and got[2].dtype == pt
            check_norm_grads(got, g.double(), h, r, w64, t, pt, what)
            with torch.no_grad():
                assert torch.equal(MF.layer_norm(x, w, b, 1e-5), y)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("width", [1, 5, 64, 129, 768, 1001, 4096, 4098, 8200, 20000])
@pytest.mark.parametrize("rate", [0.0, 0.1, 0.5])
def test_dropout_add_layer_norm(cuda, width, rate, t):
    from mamtorch_b200.nn import functional as MF

    for rows in (1, 4, 301):
        seed = 2 ** 61 + 17 * width + rows
        x, res = (inputs((rows, width), t, k, cuda).requires_grad_() for k in (1, 2))
        w, b = (p.requires_grad_() for p in params(width, t, 3, cuda))
        gy, gs = (inputs((rows, width), t, k, cuda, 0.0) for k in (4, 5))
        y, s = MF.dropout_add_layer_norm(x, res, w, b, 1e-6, rate, seed)
        what = f"{rows}x{width} {t} {rate}"
        s64 = res.detach().double() + drop64(x.detach().double(), rate, seed)
        # product and sum rounded to fp32, then to t
        check(s, s64, t, (s64 - res.detach().double()).abs() + res.detach().double().abs(), what + " s")
        v, w64, b64 = s.detach().double(), w.detach().double(), b.detach().double()
        h, r = check_norm(y, v, w64, b64, 1e-6, t, what)
        dx, dres, dw, db = torch.autograd.grad((y, s), (x, res, w, b), (gy, gs))
        dv, scale = check_norm_grads((dres, dw, db), gy.double(), h, r, w64, t, t, what, gs.double())
        check(dx, drop64(dv, rate, seed), t, 2 * scale, what + " dx")
        # the same as the two operators one after the other
        s2 = MF.dropout(x, rate, seed, residual=res)
        assert torch.equal(s2, s) and torch.equal(MF.layer_norm(s2, w, b, 1e-6), y)
        # either output alone
        y1, s1 = MF.dropout_add_layer_norm(x, res, w, b, 1e-6, rate, seed)
        only_s = torch.autograd.grad(s1, (x, res), gs)
        check(only_s[0], drop64(gs.double(), rate, seed), t, gs.double().abs() * 2, what + " dx of s alone")
        assert torch.equal(only_s[1], gs)
        y1, s1 = MF.dropout_add_layer_norm(x, res, w, b, 1e-6, rate, seed)
        only_y = torch.autograd.grad(y1, (res, w, b), gy)
        check_norm_grads(only_y, gy.double(), h, r, w64, t, t, what + " y alone")


SIZES = [(1,), (2,), (3, 5), (197, 768), (33, 129), (7, 2731), (3, 1, 511), (64, 4096)]


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("rate", [0.0, 0.1, 0.75])
@pytest.mark.parametrize("shape", SIZES)
def test_gelu(cuda, shape, rate, t):
    from mamtorch_b200.nn import functional as MF

    x = (3 * inputs(shape, t, 1, cuda, 0.0)).requires_grad_()
    g = inputs(shape, t, 2, cuda, 0.0)
    y = MF.gelu(x, rate, 99)
    x64, g64 = x.detach().double(), g.double()
    cdf = 0.5 * torch.erfc(-x64 / math.sqrt(2))
    # Phi is formed as (1 + erf) / 2, a sum of the order of one: its error is relative to one, not to Phi
    check(y, drop64(x64 * cdf, rate, 99), t, x64.abs() / (1 - rate), "y")
    slope = cdf + x64 * torch.exp(-x64 ** 2 / 2) / math.sqrt(2 * math.pi)
    (dx,) = torch.autograd.grad(y, x, g)
    # exp's argument x^2 / 2 is rounded: relative error x^2 eps in a term of size |x| exp(-x^2 / 2) <= 1
    check(dx, drop64(g64 * slope, rate, 99), t, 2 * g64.abs() / (1 - rate), "dx")
    with torch.no_grad():
        assert torch.equal(MF.gelu(x, rate, 99), y)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("rate", [0.0, 0.1, 0.75])
@pytest.mark.parametrize("shape", SIZES)
def test_dropout(cuda, shape, rate, t):
    from mamtorch_b200.nn import functional as MF

    x, res, g = (inputs(shape, t, k, cuda).requires_grad_() for k in (1, 2, 3))
    g = g.detach()
    keep = mask64(shape, rate, -5).to(cuda) if rate else torch.ones(shape, dtype=torch.bool, device=cuda)
    y = MF.dropout(x, rate, -5)
    check(y, drop64(x.detach().double(), rate, -5), t, x.detach().double().abs() / (1 - rate), "y")
    assert torch.equal(y != 0, keep & (x != 0))
    (dx,) = torch.autograd.grad(y, x, g)
    check(dx, drop64(g.double(), rate, -5), t, g.double().abs() / (1 - rate), "dx")
    z = MF.dropout(x, rate, -5, residual=res)
    dx2, dres = torch.autograd.grad(z, (x, res), g)
    check(z, res.detach().double() + drop64(x.detach().double(), rate, -5), t,
          res.detach().double().abs() + x.detach().double().abs() / (1 - rate), "z")
    assert torch.equal(dx2, dx) and torch.equal(dres, g)
