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
import warnings

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
    # Sums over the rows: in these tests a thread adds at most 40 in sequence, a CTA's groups at most 16 sums, the last kernel
    # 19 and then 8 partial rows: less than 96 additions behind one another, each off by eps_32 times at most the sum of
    # magnitudes; and h itself by 8 eps_32 (1 + |h|).  Small enough that a row left out would show.
    if got[1] is not None:
        check(got[1], dw, pt, 104 / 256 * (g.abs() * (h.abs() + 1)).sum(dims), what + " dw")
    if got[2] is not None:
        check(got[2], db, pt, 96 / 256 * g.abs().sum(dims), what + " db")
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


# rows enough that every group of threads walks many of them, in each of the forms that a width and a type lead to
MANY = [(20000, 136), (20000, 131), (20001, 96), (20001, 61), (30000, 24), (9001, 773), (9000, 776), (6000, 1024), (6001, 2048),
        (3001, 4096), (3001, 4100), (3001, 4099), (2600, 6144), (2600, 5120), (1500, 8192), (1500, 8191), (2500, 9000)]


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("shape", MANY)
@pytest.mark.parametrize("pitched", [False, True])
def test_many_rows(cuda, shape, t, pitched):
    from mamtorch_b200.nn import functional as MF

    rows, width = shape

    def make(seed, mean=0.5):
        g = torch.Generator(device=cuda).manual_seed(seed)
        v = (torch.randn(rows, width + (16 if pitched else 0), generator=g, device=cuda) + mean).to(t)
        # a slice that starts on a vector, so that its alignment is that of the width
        return (v[:, 8:8 + width] if pitched else v).detach().requires_grad_()

    x, res = make(1), make(2)
    w, b = (p.requires_grad_() for p in params(width, t, 3, cuda))
    gy, gs = make(4, 0.0).detach(), make(5, 0.0).detach()
    what = f"{shape} {t}"
    y = MF.layer_norm(x, w, b, 1e-5)
    x64, w64, b64 = x.detach().double(), w.detach().double(), b.detach().double()
    h, r = check_norm(y, x64, w64, b64, 1e-5, t, what)
    check_norm_grads(torch.autograd.grad(y, (x, w, b), gy), gy.double(), h, r, w64, t, t, what)
    y, s = MF.dropout_add_layer_norm(x, res, w, b, 1e-6, 0.2, 77)
    r64 = res.detach().double()
    s64 = r64 + drop64(x64, 0.2, 77)
    check(s, s64, t, (s64 - r64).abs() + r64.abs(), what + " s")
    h, r = check_norm(y, s.detach().double(), w64, b64, 1e-6, t, what + " add")
    dx, dres, dw, db = torch.autograd.grad((y, s), (x, res, w, b), (gy, gs))
    dv, scale = check_norm_grads((dres, dw, db), gy.double(), h, r, w64, t, t, what + " add", gs.double())
    check(dx, drop64(dv, 0.2, 77), t, 2 * scale, what + " add dx")
    MF.check_device_flag()      # no wait inside a kernel gave up


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


# ---------------------------------------------------------------- layouts

def views(shape, t, device, seed):
    """The same values in several layouts: contiguous, a column slice, a row step, transposed, off by one element."""
    base = inputs(shape, t, seed, device)
    rows, width = shape
    wide = torch.zeros(rows, width + 9, dtype=t, device=device)
    wide[:, 5:5 + width] = base
    tall = torch.zeros(2 * rows, width, dtype=t, device=device)
    tall[::2] = base
    flat = torch.zeros(rows * width + 1, dtype=t, device=device)
    flat[1:] = base.reshape(-1)
    return base, {"slice": wide[:, 5:5 + width], "step": tall[::2], "transposed": base.t().contiguous().t(),
                  "shifted": flat[1:].view(rows, width)}


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("width", [48, 131, 512, 2056, 9000])
def test_any_layout_gives_what_contiguous_tensors_give(cuda, width, t):
    from mamtorch_b200.nn import functional as MF

    shape = (37, width)
    x, xs = views(shape, t, cuda, 1)
    r, rs = views(shape, t, cuda, 2)
    g, gs = views(shape, t, cuda, 3)
    w, b = params(width, t, 4, cuda)

    def all_of(x, r, g):
        x, r = x.detach().requires_grad_(), r.detach().requires_grad_()
        out = []
        y = MF.layer_norm(x, w, b)
        out += [y, torch.autograd.grad(y, x, g)[0]]
        y, s = MF.dropout_add_layer_norm(x, r, w, b, 1e-5, 0.2, 7)
        out += [y, s, *torch.autograd.grad((y, s), (x, r), (g, g))]
        y = MF.gelu(x, 0.2, 7)
        out += [y, torch.autograd.grad(y, x, g)[0]]
        y = MF.dropout(x, 0.2, 7, residual=r)
        out += [y, *torch.autograd.grad(y, (x, r), g)]
        return out

    want = all_of(x, r, g)
    for name in xs:
        for k, (got, ref) in enumerate(zip(all_of(xs[name], rs[name], gs[name]), want)):
            # the order of a row's sums may differ between layouts: a last digit of fp32, then one rounding
            scale = ref.double().abs() + 1
            off = (got.double() - ref.double()).abs() / scale
            assert off.max().item() <= 64 * E32 + 2 * half_step(t), f"{name} output {k}"


def test_neighbours_of_a_slice_are_left_alone_and_results_do_not_depend_on_them(cuda):
    from mamtorch_b200.nn import functional as MF

    for width in (64, 67):
        w, b = params(width, torch.bfloat16, 1, cuda)
        x = inputs((50, width), torch.bfloat16, 2, cuda)
        outs = []
        for fill in (0.0, float("nan"), float("inf")):
            wide = torch.full((50, width + 7), fill, dtype=torch.bfloat16, device=cuda)
            wide[:, 3:3 + width] = x
            outs.append(MF.layer_norm(wide[:, 3:3 + width], w, b))
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_leading_dimensions_and_expanded_gradients(cuda):
    from mamtorch_b200.nn import functional as MF

    x = inputs((3, 5, 7, 96), torch.float32, 1, cuda).requires_grad_()
    w, b = (p.requires_grad_() for p in params(96, torch.float32, 2, cuda))
    y = MF.layer_norm(x, w, b)
    assert y.shape == x.shape
    assert torch.equal(y.view(-1, 96), MF.layer_norm(x.view(-1, 96), w, b))
    a = torch.autograd.grad(MF.layer_norm(x, w, b).sum(), (x, w, b))
    c = torch.autograd.grad(MF.layer_norm(x, w, b), (x, w, b), torch.ones_like(x))
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    a = torch.autograd.grad(MF.gelu(x).sum(), x)[0]
    assert torch.equal(a, torch.autograd.grad(MF.gelu(x), x, torch.ones_like(x))[0])
    # a broadcast input: its gradient is summed by autograd
    row = inputs((96,), torch.float32, 3, cuda).requires_grad_()
    z = MF.dropout(row.expand(11, 96), 0.5, 3)
    (d,) = torch.autograd.grad(z, row, torch.ones_like(z))
    want = mask64((11, 96), 0.5, 3).to(cuda).double().sum(0) * 2
    assert torch.equal(d.double(), want)
    # parameters that are slices
    big = torch.randn(200, device=cuda)
    assert torch.equal(MF.layer_norm(x, big[::2][:96], big[3:99]), MF.layer_norm(x, big[::2][:96].contiguous(), big[3:99].clone()))


# ---------------------------------------------------------------- special values

@pytest.mark.parametrize("t", DTYPES)
def test_what_is_dropped_leaves_nothing_behind(cuda, t):
    from mamtorch_b200.nn import functional as MF

    shape, seed = (6, 101), 12
    keep = mask64(shape, 0.5, seed).to(cuda)
    x = inputs(shape, t, 1, cuda)
    for bad in (float("inf"), float("-inf"), float("nan")):
        xb = torch.where(keep, x, torch.full_like(x, bad)).requires_grad_()
        xc = torch.where(keep, x, torch.zeros_like(x)).requires_grad_()
        g = inputs(shape, t, 2, cuda)
        gb = torch.where(keep, g, torch.full_like(g, bad))
        for f in (lambda v: MF.dropout(v, 0.5, seed), lambda v: MF.gelu(v, 0.5, seed)):
            y, want = f(xb), f(xc)
            assert torch.equal(y, want)
            assert torch.equal(torch.autograd.grad(y, xb, gb)[0], torch.autograd.grad(want, xc, g)[0])
        res = inputs(shape, t, 3, cuda)
        y, s = MF.dropout_add_layer_norm(xb, res, None, None, 1e-5, 0.5, seed)
        y2, s2 = MF.dropout_add_layer_norm(xc, res, None, None, 1e-5, 0.5, seed)
        assert torch.equal(y, y2) and torch.equal(s, s2)


@pytest.mark.parametrize("width", [33, 256, 3000, 20000])
def test_a_bad_row_stays_alone(cuda, width):
    from mamtorch_b200.nn import functional as MF

    x = inputs((40, width), torch.float32, 1, cuda)
    w, b = params(width, torch.float32, 2, cuda)
    g = inputs((40, width), torch.float32, 3, cuda)
    good = MF.layer_norm(x, w, b)
    for bad in (float("nan"), float("inf")):
        xb = x.clone()
        xb[17, width // 2] = bad
        xb.requires_grad_()
        y = MF.layer_norm(xb, w, b)
        rows = [i for i in range(40) if i != 17]
        assert torch.equal(y[rows], good[rows]) and torch.isnan(y[17]).all()
        (dx,) = torch.autograd.grad(y, xb, g)
        assert torch.isfinite(dx[rows]).all() and torch.isnan(dx[17]).all()


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("eps", [1e-12, 1e-5])
def test_rows_of_equal_values_come_out_as_the_bias(cuda, t, eps):
    from mamtorch_b200.nn import functional as MF

    for width in (1, 7, 96, 769, 1000, 4096, 5000, 12345):
        w, b = params(width, t, 2, cuda)
        x = torch.tensor([[0.1], [-3.3], [1e4], [7e-3]], device=cuda).to(t).expand(4, width).contiguous().requires_grad_()
        y = MF.layer_norm(x, w, b, eps)
        assert torch.equal(y, b.expand(4, width)), width
        g = inputs((4, width), t, 3, cuda)
        dx, = torch.autograd.grad(y, x, g)
        assert torch.isfinite(dx).all() or eps < 1e-10     # 1 / sqrt(eps) may leave fp16's range
    # a weight's gradient is exactly zero there
    x = torch.full((9, 640), 3.7, device=cuda).to(t)
    w = torch.ones(640, device=cuda, dtype=t, requires_grad=True)
    (dw,) = torch.autograd.grad(MF.layer_norm(x, w, None, eps), w, torch.ones_like(x))
    assert torch.count_nonzero(dw) == 0


def test_a_mean_far_from_zero_costs_the_digits_of_the_inputs_only(cuda):
    from mamtorch_b200.nn import functional as MF

    for width in (64, 768, 1001, 5120, 30000):
        x = inputs((50, width), torch.float32, 1, cuda, mean=4000.0).requires_grad_()
        g = inputs((50, width), torch.float32, 2, cuda, mean=0.0)
        y = MF.layer_norm(x)
        x64 = x.detach().double()
        want, h, r = norm64(x64, torch.ones((), device=cuda), torch.zeros((), device=cuda), 1e-5)
        # the mean is stored in fp32: half a step of 4000 is 1.3e-4 (2^-13), every value of h is off by r times that, and
        # what a few fp32 operations on h add
        bound = 2.0 ** -13 * r * 1.01 + 16 * E32 * (1 + h.abs())
        assert ((y.detach().double() - want).abs() <= bound).all()
        (dx,) = torch.autograd.grad(y, x, g)
        dv, _, _ = norm_grads64(g.double(), h, r, torch.ones((), device=cuda))
        # h enters the gradient times mean(g h), and in that mean: at most 2^-13 r (mean|g h| + |h| mean|g|) r
        m = (g.double() * h).abs().mean(1, keepdim=True) + h.abs() * g.double().abs().mean(1, keepdim=True)
        bound = 2.0 ** -13 * r * r * 1.01 * m + 256 * E32 * r * (g.double().abs() + m + 1)
        assert ((dx.double() - dv).abs() <= bound).all()


def test_gelu_at_the_ends_of_the_range(cuda):
    from mamtorch_b200.nn import functional as MF

    x = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 40.0, -40.0, 1e30, -1e30, 1e-30],
                     device=cuda, requires_grad=True)
    y = MF.gelu(x)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(x))
    assert y[0] == float("inf") and y[1] == 0 and torch.isnan(y[2]) and y[3] == 0 and y[4] == 0
    assert y[5] == 40 and y[6] == 0 and y[7] == torch.tensor(1e30) and y[8] == 0
    assert dx[0] == 1 and dx[1] == 0 and torch.isnan(dx[2]) and dx[5] == 1 and dx[6] == 0 and dx[7] == 1 and dx[8] == 0
    # Phi(0) = 1/2: six fp32 operations on values up to one half
    assert abs(dx[3].item() - 0.5) <= 8 * E32 and abs(dx[4].item() - 0.5) <= 8 * E32
    assert abs(y[9].item() - 5e-31) <= 16 * E32 * 5e-31


@pytest.mark.parametrize("t", DTYPES)
def test_empty_tensors(cuda, t):
    from mamtorch_b200.nn import functional as MF

    w, b = (p.requires_grad_() for p in params(12, t, 1, cuda))
    x = torch.empty(0, 12, dtype=t, device=cuda, requires_grad=True)
    y = MF.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(x))
    assert y.shape == (0, 12) and dx.shape == (0, 12) and torch.count_nonzero(dw) == 0 and torch.count_nonzero(db) == 0
    y, s = MF.dropout_add_layer_norm(x, x, w, b, 1e-5, 0.5, 1)
    assert y.shape == s.shape == (0, 12)
    for v in (x, torch.empty(3, 0, dtype=t, device=cuda)):
        assert MF.gelu(v, 0.5, 1).shape == v.shape and MF.dropout(v, 0.5, 1, residual=v).shape == v.shape
    with pytest.raises(RuntimeError):
        MF.layer_norm(torch.empty(3, 0, dtype=t, device=cuda))


# ---------------------------------------------------------------- masks

def test_masks_have_their_rate_and_follow_the_seed(cuda):
    from mamtorch_b200.nn import functional as MF

    n = 1 << 22
    x = torch.ones(n, device=cuda)
    for rate in (1e-4, 0.1, 0.5, 0.9):
        kept = (MF.dropout(x, rate, 123) != 0).double().mean().item()
        assert abs(kept - (1 - rate)) <= 6 * math.sqrt(rate * (1 - rate) / n)    # six standard deviations
    assert not torch.equal(MF.dropout(x, 0.5, 1), MF.dropout(x, 0.5, 2))
    torch.manual_seed(5)
    a = MF.dropout(x, 0.5)
    b = MF.dropout(x, 0.5)
    torch.manual_seed(5)
    assert torch.equal(a, MF.dropout(x, 0.5)) and not torch.equal(a, b)
    # the same elements in any shape
    assert torch.equal(MF.dropout(x.view(-1, 64), 0.5, 9).view(-1), MF.dropout(x, 0.5, 9))
    # small rates: the threshold is odd
    m = mask64((n,), 3.3e-4, 77).to(cuda)
    assert int(float(np.float32(3.3e-4)) * 2 ** 32) % 2 == 1 and torch.equal(MF.dropout(x, 3.3e-4, 77) != 0, m)


def test_a_seed_tensor_is_read_when_the_kernel_runs(cuda):
    from mamtorch_b200.nn import functional as MF

    x = inputs((33, 100), torch.float32, 1, cuda).requires_grad_()
    seed = torch.tensor([41], device=cuda)
    assert torch.equal(MF.dropout(x, 0.3, seed), MF.dropout(x, 0.3, 41))
    y = MF.gelu(x, 0.3, seed)
    assert torch.equal(y, MF.gelu(x, 0.3, 41))
    (a,) = torch.autograd.grad(y, x, torch.ones_like(y))
    (b,) = torch.autograd.grad(MF.gelu(x, 0.3, 41), x, torch.ones_like(y))
    assert torch.equal(a, b)
    for f in (lambda: MF.gelu(x, 0.3, seed), lambda: MF.dropout(x, 0.3, seed),
              lambda: MF.dropout_add_layer_norm(x, x, None, None, 1e-5, 0.3, seed)[0]):
        y = f()
        seed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


# ---------------------------------------------------------------- gradients against differences

@pytest.mark.parametrize("width", [5, 64, 200])
def test_gradients_against_differences_of_the_definition(cuda, width):
    """Along random directions: (f(x + d v) - f(x - d v)) / 2 d of the definition in 64 bits, whose error is of the order
    of d^2 = 1e-10 and 1e-16 / d = 1e-11; the operators' own gradients are fp32."""
    from mamtorch_b200.nn import functional as MF

    rows, d, rate, seed = 9, 1e-5, 0.25, 31
    gen = torch.Generator().manual_seed(width)
    draw = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).to(cuda).float()   # noqa: E731
    x, res, w, b = (v.requires_grad_() for v in (draw(rows, width), draw(rows, width), draw(width), draw(width)))
    cy, cs = draw(rows, width), draw(rows, width)

    def norm(x, w, b):
        return (norm64(x, w, b, 1e-5)[0] * cy.double()).sum()

    def add_norm(x, res, w, b):
        s = res + drop64(x, rate, seed)
        return (norm64(s, w, b, 1e-5)[0] * cy.double()).sum() + (s * cs.double()).sum()

    def gelu(x):
        return (drop64(x * 0.5 * torch.erfc(-x / math.sqrt(2)), rate, seed) * cy.double()).sum()

    y, s = MF.dropout_add_layer_norm(x, res, w, b, 1e-5, rate, seed)
    for f, args, grads in (
            (norm, (x, w, b), torch.autograd.grad(MF.layer_norm(x, w, b), (x, w, b), cy)),
            (add_norm, (x, res, w, b), torch.autograd.grad((y, s), (x, res, w, b), (cy, cs))),
            (gelu, (x,), torch.autograd.grad(MF.gelu(x, rate, seed), (x,), cy))):
        for k, (arg, grad) in enumerate(zip(args, grads)):
            v = draw(*arg.shape).double()
            at = [a.detach().double() for a in args]
            up, down = list(at), list(at)
            up[k], down[k] = at[k] + d * v, at[k] - d * v
            slope = ((f(*up) - f(*down)) / (2 * d)).item()
            got = (grad.double() * v).sum().item()
            # every element of the gradient is off by at most 256 eps_32 times what it sums, a few times its largest
            size = (v.abs().sum() * grad.double().abs().max()).item()
            assert abs(got - slope) <= 256 * E32 * size + 1e-8 * size, (f.__name__, k)


def test_second_derivatives_are_refused(cuda):
    from mamtorch_b200.nn import functional as MF

    x = inputs((4, 32), torch.float32, 1, cuda).requires_grad_()
    for f in (MF.layer_norm, MF.gelu, lambda v: MF.dropout(v, 0.5, 1), lambda v: MF.dropout_add_layer_norm(v, v)[0]):
        (g,) = torch.autograd.grad(f(x).square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()


# ---------------------------------------------------------------- refusals

def test_refusals(cuda):
    from mamtorch_b200.nn import functional as MF

    x = torch.randn(4, 32, device=cuda)
    w = torch.ones(32, device=cuda)
    for call in (lambda: MF.layer_norm(x.double()), lambda: MF.layer_norm(x.int()), lambda: MF.layer_norm(x, w[:31]),
                 lambda: MF.layer_norm(x, w.half()), lambda: MF.layer_norm(x.half(), w.bfloat16()),
                 lambda: MF.layer_norm(x.half(), w, w.half()), lambda: MF.layer_norm(x, w.cpu()),
                 lambda: MF.layer_norm(x, w, w.view(1, 32)), lambda: MF.layer_norm(x, w, w, -1e-5),
                 lambda: MF.layer_norm(x[0, 0]), lambda: MF.layer_norm(x, eps=float("nan")),
                 lambda: MF.dropout_add_layer_norm(x, x[:3]), lambda: MF.dropout_add_layer_norm(x, x.half()),
                 lambda: MF.dropout_add_layer_norm(x, x.cpu()), lambda: MF.dropout(x, 0.5, 1, residual=x[:, :31]),
                 lambda: MF.dropout(x, 0.5, torch.tensor([1])), lambda: MF.dropout(x, 0.5, torch.tensor([1, 2], device=cuda)),
                 lambda: MF.dropout(x, 0.5, torch.tensor([1.0], device=cuda)), lambda: MF.gelu(x.double()),
                 lambda: MF.gelu(x, 0.5, torch.tensor([1], device=cuda, dtype=torch.int32)),
                 lambda: torch.ops.mamtorch_b200.dropout_forward(x, None, 1.0, 1, None),
                 lambda: torch.ops.mamtorch_b200.layer_norm_forward(x, None, w, w, 1e-5, 0.5, 1, None, False),
                 lambda: torch.ops.mamtorch_b200.layer_norm_backward(x, None, x, torch.zeros(3, 2, device=cuda), w, 0.0, 0,
                                                                     None, True, True, True),
                 lambda: torch.ops.mamtorch_b200.gelu_backward(x[:2], x, 0.0, 0, None)):
        with pytest.raises(RuntimeError):
            call()
    for rate in (-0.1, 1.0, 1.5, float("nan")):
        with pytest.raises(ValueError):
            MF.dropout(x, rate, 1)


# ---------------------------------------------------------------- streams, graphs, order

def test_gradients_do_not_change_from_run_to_run(cuda):
    from mamtorch_b200.nn import functional as MF

    for shape, t in (((3001, 768), torch.float32), ((999, 4096), torch.bfloat16), ((777, 1283), torch.float16),
                     ((5000, 96), torch.float32), ((40, 9000), torch.float32)):
        x, r = (inputs(shape, t, k, cuda).requires_grad_() for k in (1, 2))
        w, b = (p.requires_grad_() for p in params(shape[1], t, 3, cuda))
        g = inputs(shape, t, 4, cuda)
        runs = []
        for _ in range(3):
            y, s = MF.dropout_add_layer_norm(x, r, w, b, 1e-5, 0.1, 5)
            runs.append(torch.autograd.grad((y, s), (x, r, w, b), (g, g)))
        for other in runs[1:]:
            assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


def test_on_a_stream_of_its_own_and_two_at_once(cuda):
    from mamtorch_b200.nn import functional as MF

    shape = (2000, 1024)
    xs = [inputs(shape, torch.bfloat16, k, cuda).requires_grad_() for k in range(4)]
    w, b = (p.requires_grad_() for p in params(1024, torch.bfloat16, 9, cuda))
    g = inputs(shape, torch.bfloat16, 8, cuda)

    def work(x):
        y, s = MF.dropout_add_layer_norm(MF.gelu(x, 0.1, 3), x, w, b, 1e-5, 0.1, 4)
        return [y, s, *torch.autograd.grad((y, s), (x, w, b), (g, g))]

    want = [work(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, st in zip(xs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([work(x) for _ in range(3)])
    torch.cuda.synchronize()
    for per, ref in zip(got, want):
        for run in per:
            assert all(torch.equal(p, q) for p, q in zip(run, ref))


def test_from_several_threads_at_once(cuda):
    """First calls of kernels with different amounts of shared memory, from threads of their own."""
    from concurrent.futures import ThreadPoolExecutor

    from mamtorch_b200.nn import functional as MF

    def work(k):
        width = (200, 1000, 2500, 4500, 7000, 8192)[k % 6]
        t = DTYPES[k % 3]
        x, r, g = (inputs((300, width), t, 10 * k + j, cuda) for j in range(3))
        x.requires_grad_()
        w, b = (p.requires_grad_() for p in params(width, t, k, cuda))
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            y, s = MF.dropout_add_layer_norm(MF.gelu(x, 0.1, k), r, w, b, 1e-5, 0.1, k)
            out = [y, s, *torch.autograd.grad((y, s), (x, w, b), (g, g))]
            torch.cuda.current_stream().synchronize()
        return out

    with ThreadPoolExecutor(6) as pool:
        at_once = list(pool.map(work, range(18)))
    for k, out in enumerate(at_once):
        assert all(torch.equal(p, q) for p, q in zip(out, work(k)))


def test_captured_steps_replay_with_new_seeds(cuda):
    from mamtorch_b200.nn import functional as MF

    shape = (300, 520)
    x, r = (inputs(shape, torch.float32, k, cuda).requires_grad_() for k in (1, 2))
    w, b = (p.requires_grad_() for p in params(520, torch.float32, 3, cuda))
    g = inputs(shape, torch.float32, 4, cuda)
    seed = torch.tensor([1000], device=cuda)

    def work(seed):
        y, s = MF.dropout_add_layer_norm(MF.gelu(x, 0.2, seed), MF.dropout(r, 0.2, seed), w, b, 1e-5, 0.2, seed)
        return [y, s, *torch.autograd.grad((y, s), (x, r, w, b), (g, g))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(seed)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):      # two graphs at hand at once: neither keeps anything in the other's memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, work(seed)))
    for k in range(3):
        seed.fill_(1000 + k)
        for graph, _ in graphs:
            graph.replay()
        want = work(1000 + k)
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")      # the graph stays empty
        with pytest.raises(RuntimeError, match="capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                MF.dropout(x, 0.5)


# ---------------------------------------------------------------- long tensors

def test_more_than_two_to_the_thirty_two_elements(cuda):
    """Offsets beyond 32 bits: the last rows of a tensor of 4.3e9 elements, the mask's counters among them."""
    from mamtorch_b200.nn import functional as MF

    if torch.cuda.get_device_properties(cuda).total_memory < 60e9:
        pytest.skip("needs 60 GB")
    width, rows, rate, seed = 4097, 1048600, 0.25, 17
    n = rows * width
    assert n > 2 ** 32
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=cuda)
    tail = inputs((3, width), torch.bfloat16, 1, cuda)
    x[-3:] = tail
    # the mask of the last three rows, from its own counters
    first = (n - 3 * width) // 2 * 2
    with np.errstate(over="ignore"):
        z = np.uint64(seed) + np.arange(first // 2, (n + 1) // 2, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    draws = np.stack([z & np.uint64(0xFFFFFFFF), z >> np.uint64(32)], 1).reshape(-1)
    keep = torch.from_numpy((draws >= np.uint64(2 ** 30))[n - 3 * width - first:][:3 * width].reshape(3, width)).to(cuda)
    want = torch.where(keep, tail.double() / 0.75, torch.zeros((), dtype=torch.float64, device=cuda))
    y = MF.dropout(x, rate, seed)
    check(y[-3:], want, torch.bfloat16, want.abs(), "dropout")
    del y
    y, s = MF.dropout_add_layer_norm(x, x, None, None, 1e-5, rate, seed)
    check(s[-3:], tail.double() + want, torch.bfloat16, tail.double().abs() + want.abs(), "s")
    one, zero = torch.ones((), device=cuda, dtype=torch.float64), torch.zeros((), device=cuda, dtype=torch.float64)
    check_norm(y[-3:], s[-3:].double(), one, zero, 1e-5, torch.bfloat16, "y")


# ---------------------------------------------------------------- the C ABI itself

def test_c_abi_without_torch_operators(cuda):
    from mamtorch_b200 import _lib

    L = _lib.lib()
    p = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())   # noqa: E731
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    rows, width = 77, 264
    x, r, gy, gs = (inputs((rows, width), torch.float32, k, cuda) for k in range(4))
    w, b = params(width, torch.float32, 5, cuda)
    y, s, ds, dx = (torch.empty_like(x) for _ in range(4))
    dw, db = torch.empty_like(w), torch.empty_like(b)
    stats = torch.empty(rows, 2, device=cuda)
    assert L.mam_layer_norm_fwd(p(x), width, p(r), width, p(w), p(b), 0, 1e-5, 0.1, 7, None, p(y), p(s), p(stats), rows,
                                width, 0, st) == 0
    nbytes = L.mam_layer_norm_bwd_workspace_bytes(rows, width)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=cuda)
    args = (p(gy), p(gs), p(s), width, p(stats), p(w), 0, 0.1, 7, None, p(ds), p(dx), p(dw), p(db), rows, width, 0)
    assert L.mam_layer_norm_bwd(*args, p(ws), nbytes, st) == 0
    h, rs = check_norm(y, s.double(), w.double(), b.double(), 1e-5, torch.float32, "y")
    dv, scale = check_norm_grads((ds, dw, db), gy.double(), h, rs, w.double(), torch.float32, torch.float32, "c", gs.double())
    check(dx, drop64(dv, 0.1, 7), torch.float32, 2 * scale, "dx")
    assert L.mam_layer_norm_bwd(*args, None, 0, st) == 3 and L.mam_layer_norm_bwd(*args, p(ws), nbytes - 1, st) == 3
    assert L.mam_layer_norm_bwd(*args, ctypes.c_void_p(ws.data_ptr() + 4), nbytes, st) == 3
    # a second gradient although nothing is dropped: the same
    none = (0.0, 7, None)
    assert L.mam_layer_norm_bwd(*args[:7], *none, p(ds), p(dx), p(dw), p(db), rows, width, 0, p(ws), nbytes, st) == 0
    assert torch.equal(ds, dx)
    # without the parameters' gradients no workspace is needed
    ds2 = torch.empty_like(ds)
    assert L.mam_layer_norm_bwd(*args[:10], p(ds2), p(dx), None, None, rows, width, 0, None, 0, st) == 0
    assert torch.equal(ds, ds2) and not torch.equal(ds, dx)
    assert L.mam_check_device_flag() == 0


# ---------------------------------------------------------------- the blocks that call them

def test_fused_block_matches_the_composed_one(cuda):
    import copy

    from mamtorch_b200.nn.vit import MAMMlpBlock

    torch.manual_seed(1)
    plain = MAMMlpBlock(64, 160).to(cuda)
    fused = MAMMlpBlock(64, 160, fused=True).to(cuda)
    fused.load_state_dict(copy.deepcopy(plain.state_dict()))
    x = inputs((2, 37, 64), torch.float32, 2, cuda)
    # the MAM layers select single products, so that inputs which differ in the last digit give outputs that differ as much
    a, b = plain(x), fused(x)
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
    drop = MAMMlpBlock(64, 160, fused=True, drop_rate=0.4).to(cuda)
    drop.load_state_dict(plain.state_dict())
    assert torch.equal(drop.eval()(x), b)
    drop.train()
    assert not torch.equal(drop(x), drop(x))
    with pytest.raises(ValueError):
        MAMMlpBlock(64, 160, drop_rate=0.1)


def test_stack_is_its_blocks_one_after_the_other(cuda):
    from mamtorch_b200.nn import functional as MF
    from mamtorch_b200.nn.vit import MAMMlpStack

    torch.manual_seed(3)
    stack = MAMMlpStack(3, 72, 96, drop_rate=0.2).to(cuda).train()
    x = inputs((4, 19, 72), torch.float32, 4, cuda).requires_grad_()
    torch.manual_seed(11)
    y = stack(x)
    # the same draws by hand
    torch.manual_seed(11)
    z = x
    for block in stack.blocks:
        z = block(z)
    z = MF.layer_norm(z, stack.norm.weight, stack.norm.bias, stack.norm.eps)
    assert torch.equal(y, z)
    g = inputs(y.shape, torch.float32, 5, cuda)
    names = [n for n, _ in stack.named_parameters()]
    ga = torch.autograd.grad(y, [x, *stack.parameters()], g)
    gb = torch.autograd.grad(z, [x, *stack.parameters()], g)
    for n, p, q in zip(["x", *names], ga, gb):
        # sums in another order (the residual's gradient is added inside the kernel), through three blocks
        assert torch.allclose(p, q, rtol=1e-4, atol=1e-4 * q.abs().max().item()), n


def test_captured_block_drops_anew_at_each_replay(cuda):
    from mamtorch_b200.nn.vit import GraphedStep, MAMMlpBlock

    torch.manual_seed(5)
    block = MAMMlpBlock(64, 128, fused=True, drop_rate=0.5).to(cuda)
    x, gy = inputs((4, 50, 64), torch.float32, 1, cuda), inputs((4, 50, 64), torch.float32, 2, cuda)
    step = GraphedStep(block, x, gy)
    outs = [step(x, gy).clone() for _ in range(3)]
    assert not torch.equal(outs[0], outs[1]) and not torch.equal(outs[1], outs[2])
    # where the last dropout dropped, the output is the input, in about half of the places
    for y in outs:
        share = (y == x).double().mean().item()
        assert abs(share - 0.5) < 6 * 0.5 / math.sqrt(x.numel())
    assert torch.isfinite(step.grad_input).all()


# ---------------------------------------------------------------- torch around them

def test_schemas_and_shape_functions(cuda):
    from torch.library import opcheck

    import mamtorch_b200  # noqa: F401

    ops = torch.ops.mamtorch_b200
    x, r = (inputs((6, 5, 40), torch.bfloat16, k, cuda) for k in (1, 2))
    w, b = params(40, torch.float32, 3, cuda)
    at = torch.tensor([5], device=cuda)
    stats = torch.rand(30, 2, device=cuda)
    for op, args in ((ops.layer_norm_forward, (x, None, w, b, 1e-5, 0.0, 0, None, True)),
                     (ops.layer_norm_forward, (x, r, None, None, 1e-5, 0.1, 3, at, False)),
                     (ops.layer_norm_backward, (x, r, x, stats, w, 0.1, 3, None, True, True, True)),
                     (ops.layer_norm_backward, (x, None, x, stats, w, 0.0, 0, None, True, False, True)),
                     (ops.dropout_forward, (x, r, 0.1, 3, at)), (ops.gelu_forward, (x, 0.1, 3, None)),
                     (ops.gelu_backward, (r, x, 0.1, 3, None))):
        opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


def test_traced_checkpointed_and_transformed_calls(cuda):
    import torch.utils.checkpoint as checkpoint

    from mamtorch_b200.nn import functional as MF

    x = inputs((16, 64), torch.float32, 1, cuda).requires_grad_()
    w, b = (p.requires_grad_() for p in params(64, torch.float32, 2, cuda))

    def f(x, w, b):
        y, s = MF.dropout_add_layer_norm(MF.gelu(x, 0.1, 3), x, w, b, 1e-5, 0.1, 7)
        return y * s

    want = f(x, w, b)
    grads = torch.autograd.grad(want.sum(), (x, w, b))
    got = torch.compile(f, backend="aot_eager")(x, w, b)
    assert torch.equal(got, want)
    for p, q in zip(torch.autograd.grad(got.sum(), (x, w, b)), grads):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-5 * q.abs().max().item())
    # a recomputed forward draws the same numbers, from the restored generator
    drop = lambda v: MF.dropout(MF.gelu(v, 0.3), 0.3)   # noqa: E731
    torch.manual_seed(1)
    y = checkpoint.checkpoint(drop, x, use_reentrant=False)
    (a,) = torch.autograd.grad(y.sum(), x)
    torch.manual_seed(1)
    z = drop(x)
    assert torch.equal(y, z) and torch.equal(a, torch.autograd.grad(z.sum(), x)[0])
    (a,) = torch.autograd.grad(MF.gelu(x).square().sum(), x)
    assert torch.equal(torch.func.grad(lambda v: MF.gelu(v).square().sum())(x.detach()), a)


def test_saved_tensors_are_guarded(cuda):
    from mamtorch_b200.nn import functional as MF

    x = inputs((16, 64), torch.float32, 1, cuda).requires_grad_()
    y, s = MF.dropout_add_layer_norm(x * 2, x)
    s.data  # reading is fine
    with torch.no_grad():
        s.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = MF.layer_norm(x)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
