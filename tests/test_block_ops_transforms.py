"""Layer norm, dropout and GELU under torch's transforms: what a second or a forward-mode derivative does, and first ones inside
transforms.  The kernels take no part: plain CPU kernels stand in for the inner operators, the autograd nodes and operator
registrations above them are the library's own."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

from mamtorch_b200.nn import functional as MF

F64 = torch.float64


def keep(x, rate, seed):
    gen = torch.Generator().manual_seed(seed % 2 ** 63)
    return torch.rand(x.shape, generator=gen, dtype=F64) >= rate


def drop(x, rate, seed):
    return x.clone() if rate == 0 else torch.where(keep(x, rate, seed), x / (1 - rate), torch.zeros((), dtype=x.dtype))


def normed(s, eps):
    mu = s.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((s - mu) ** 2).mean(-1, keepdim=True) + eps)
    return mu, r, (s - mu) * r


def norm_forward(x, residual, weight, bias, eps, rate, seed, seed_at, want_stats):
    s = x if residual is None else residual + drop(x, rate, seed)
    mu, r, h = normed(s, eps)
    y = h if weight is None else h * weight
    out = [y.clone() if bias is None else y + bias]
    if residual is not None:
        out.append(s)
    if want_stats:
        out.append(torch.cat((mu.reshape(-1, 1), r.reshape(-1, 1)), 1))
    return out


def norm_backward(gy, gsum, s, stats, weight, rate, seed, seed_at, params_f32, want_weight, want_bias):
    shape = (*s.shape[:-1], 1)
    mu, r = stats[:, 0].reshape(shape), stats[:, 1].reshape(shape)
    h, g = (s - mu) * r, torch.zeros_like(s) if gy is None else gy
    a = g if weight is None else g * weight
    ds = r * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
    ds = ds if gsum is None else ds + gsum
    dims = tuple(range(s.dim() - 1))
    return ([ds] + ([drop(ds, rate, seed)] if rate > 0 else []) + ([(g * h).sum(dims)] if want_weight else [])
            + ([g.sum(dims)] if want_bias else []))


def slope(x):
    return 0.5 * torch.erfc(-x / math.sqrt(2)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


@pytest.fixture
def cpu_kernels():
    with torch.library._scoped_library("mamtorch_b200", "IMPL") as lib:
        for name, f in (
                ("layer_norm_forward", norm_forward), ("layer_norm_backward", norm_backward),
                ("dropout_forward", lambda x, res, rate, seed, at: drop(x, rate, seed) + (0 if res is None else res)),
                ("gelu_forward", lambda x, rate, seed, at: drop(x * 0.5 * torch.erfc(-x / math.sqrt(2)), rate, seed)),
                ("gelu_backward", lambda g, x, rate, seed, at: drop(g * slope(x), rate, seed))):
            lib.impl(name, f, "CPU")
        yield


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


W, B, RES = rand(6, seed=1), rand(6, seed=2), rand(3, 6, seed=3)
# one argument each, the others held; with the plain form in torch operations
OPS = {
    "gelu": (MF.gelu, torch.nn.functional.gelu),
    "gelu with dropout": (lambda x: MF.gelu(x, 0.5, 3), lambda x: drop(torch.nn.functional.gelu(x), 0.5, 3)),
    "dropout": (lambda x: MF.dropout(x, 0.5, 3), lambda x: drop(x, 0.5, 3)),
    "dropout, residual": (lambda x: MF.dropout(x, 0.5, 3, residual=RES), lambda x: RES + drop(x, 0.5, 3)),
    "residual of dropout": (lambda x: MF.dropout(RES, 0.5, 3, residual=x), lambda x: x + drop(RES, 0.5, 3)),
    "layer_norm": (lambda x: MF.layer_norm(x, W, B), lambda x: torch.nn.functional.layer_norm(x, (6,), W, B)),
    "layer_norm, weight": (lambda w: MF.layer_norm(RES, w.sum(0), B), lambda w: torch.nn.functional.layer_norm(RES, (6,), w.sum(0), B)),
    "layer_norm, bias": (lambda b: MF.layer_norm(RES, W, b.sum(0)), lambda b: torch.nn.functional.layer_norm(RES, (6,), W, b.sum(0))),
    "dropout_add_layer_norm": (lambda x: sum(MF.dropout_add_layer_norm(x, RES, W, B, 1e-5, 0.5, 3)),
                               lambda x: (s := RES + drop(x, 0.5, 3)) + torch.nn.functional.layer_norm(s, (6,), W, B)),
    "residual of dropout_add_layer_norm": (lambda x: sum(MF.dropout_add_layer_norm(RES, x, W, B, 1e-5, 0.5, 3)),
                                           lambda x: (s := x + drop(RES, 0.5, 3)) + torch.nn.functional.layer_norm(s, (6,), W, B)),
}
# those whose second derivative is not zero
CURVED = [k for k in OPS if k not in ("dropout", "dropout, residual", "residual of dropout", "layer_norm, weight", "layer_norm, bias")]
X, V = rand(3, 6, seed=4), rand(3, 6, seed=5)
# doubles throughout: fewer than a hundred operations on values of the order of ten
CLOSE = dict(rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("name", OPS)
def test_first_derivatives(cpu_kernels, name):
    f, plain = OPS[name]
    x, z = X.clone().requires_grad_(), X.clone().requires_grad_()
    torch.testing.assert_close(f(x), plain(z), **CLOSE)
    (got,), (want,) = torch.autograd.grad(f(x), x, V), torch.autograd.grad(plain(z), z, V)
    torch.testing.assert_close(got, want, **CLOSE)
    scalar, plain_scalar = (lambda v, h=h: (h(v) * V).sum() for h in (f, plain))
    torch.testing.assert_close(torch.func.grad(scalar)(X), want, **CLOSE)
    torch.testing.assert_close(torch.func.vjp(f, X)[1](V)[0], want, **CLOSE)
    # of a leaf that eager autograd follows too
    torch.testing.assert_close(torch.func.grad(scalar)(x), want, **CLOSE)
    # a level of transforms that does not touch the operator's input: still its first derivative for the level below
    inner = torch.func.grad(lambda v: torch.func.grad(lambda c: (f(v) * c).sum())(torch.ones_like(V)).mul(V).sum())
    torch.testing.assert_close(inner(X), want, **CLOSE)


@pytest.mark.parametrize("name", OPS)
def test_forward_mode_is_refused(cpu_kernels, name):
    f, _ = OPS[name]
    refused = pytest.raises((RuntimeError, NotImplementedError), match="forward-mode")
    with refused:
        torch.func.jvp(f, (X,), (V,))
    with refused:
        torch.func.jacfwd(f)(X)
    for leaf in (False, True):
        with fw.dual_level(), refused:
            f(fw.make_dual(X.clone().requires_grad_(leaf), V))
    # a tangent that comes with the upstream gradient
    x = X.clone().requires_grad_()
    y = f(x)
    with fw.dual_level():
        g = fw.make_dual(V, torch.ones_like(V))
        if name == "residual of dropout":      # its gradient is the upstream gradient itself
            assert torch.equal(fw.unpack_dual(torch.autograd.grad(y, x, g)[0]).tangent, torch.ones_like(V))
        else:
            with refused:
                torch.autograd.grad(y, x, g)


def test_forward_mode_is_refused_below_no_grad_and_by_the_operators(cpu_kernels):
    ops = torch.ops.mamtorch_b200
    calls = (lambda x: ops.gelu(x, 0.0, 0, None), lambda x: ops.dropout(RES, x, 0.5, 1, None), lambda x: ops.layer_norm(x, W, B, 1e-5),
             lambda x: ops.gelu_forward(x, 0.0, 0, None), lambda x: ops.gelu_backward(V, x, 0.0, 0, None),
             lambda x: ops.dropout_forward(x, None, 0.5, 1, None), MF.gelu,
             lambda x: ops.layer_norm_forward(x, None, None, None, 1e-5, 0.0, 0, None, True))
    for call in calls:
        with fw.dual_level(), torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="forward-mode"):
            call(fw.make_dual(X, V))


@pytest.mark.parametrize("name", CURVED)
def test_second_derivatives_are_refused_in_transforms(cpu_kernels, name):
    f, plain = OPS[name]
    scalar, plain_scalar = (lambda v, h=h: (h(v) ** 2 * V).sum() for h in (f, plain))
    once = lambda h: (lambda v: (torch.func.grad(h)(v) * V).sum())      # noqa: E731
    assert torch.func.grad(once(plain_scalar))(X).abs().max() > 0.01
    refused = pytest.raises(RuntimeError, match="differentiable once|forward-mode")
    with refused:
        torch.func.grad(once(scalar))(X)
    with refused:
        torch.func.jvp(torch.func.grad(scalar), (X,), (V,))
    with refused:
        torch.func.hessian(scalar)(X)
    with refused:
        torch.autograd.functional.hessian(scalar, X)
    x = X.clone().requires_grad_()
    (g,) = torch.autograd.grad(scalar(x), x, create_graph=True)
    with refused:
        g.sum().backward()
    # the gradient of a transform, followed by eager autograd
    with refused:
        torch.func.grad(scalar)(x).sum().backward()


def test_inner_operators_have_no_derivative_of_their_own(cpu_kernels):
    ops = torch.ops.mamtorch_b200
    x = X.clone().requires_grad_()
    for out in (ops.gelu_forward(x, 0.0, 0, None), ops.dropout_forward(x, None, 0.5, 1, None), ops.gelu_backward(V, x, 0.0, 0, None),
                *ops.layer_norm_forward(x, None, None, None, 1e-5, 0.0, 0, None, True)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            out.sum().backward()


# ---------------------------------------------------------------- vmap

@pytest.mark.parametrize("name", [k for k in OPS if "drop" in k])
def test_vmap_of_a_dropout_is_refused(cpu_kernels, name):
    """One seed and the same element numbers: every sample would lose the same elements."""
    f, _ = OPS[name]
    xs = rand(4, 3, 6, seed=6)
    for g in (f, torch.func.grad(lambda v: (f(v) * V).sum()), lambda v: torch.func.vmap(f)(v.unsqueeze(0)),
              lambda v: torch.func.vjp(f, v)[1](V)[0]):
        with pytest.raises(RuntimeError, match="same elements in every sample"):
            torch.func.vmap(g)(xs)


@pytest.mark.parametrize("name", OPS)
def test_many_upstream_gradients_of_one_call(cpu_kernels, name):
    """Mapped over the gradients alone: the forward is one, and so is its mask."""
    f, plain = OPS[name]
    want = torch.func.jacrev(plain)(X)
    torch.testing.assert_close(torch.func.jacrev(f)(X), want, **CLOSE)
    torch.testing.assert_close(torch.func.vmap(torch.func.vjp(f, X)[1])(torch.eye(18, dtype=F64).view(18, 3, 6))[0].view_as(want), want,
                               **CLOSE)


def test_vmap_without_a_dropout_goes_sample_by_sample(cpu_kernels):
    xs, ws, bs = rand(4, 3, 6, seed=6), rand(4, 6, seed=7), rand(6, 4, seed=8)
    cases = {
        "gelu": (MF.gelu, (0,), (xs,)), "gelu, last": (MF.gelu, (1,), (xs.movedim(0, 1),)),
        "dropout": (lambda v: MF.dropout(v, 0.0), (0,), (xs,)), "residual": (lambda v: MF.dropout(RES, 0.0, residual=v), (0,), (xs,)),
        "layer_norm": (lambda v: MF.layer_norm(v, W, B), (0,), (xs,)), "weights": (lambda w, b: MF.layer_norm(RES, w, b), (0, 1), (ws, bs)),
        "add": (lambda v, w: MF.dropout_add_layer_norm(v, RES, w, B), (0, 0), (xs, ws)),
        "per-sample gradients": (torch.func.grad(lambda w, v: (MF.layer_norm(v, w, B) * V).sum()), (None, 0), (W, xs)),
        "gelu's": (torch.func.grad(lambda v: (MF.gelu(v) * V).sum()), (0,), (xs,)),
    }
    for name, (f, dims, args) in cases.items():
        got = torch.func.vmap(f, in_dims=dims)(*args)
        want = [f(*(a if d is None else a.select(d, i) for a, d in zip(args, dims))) for i in range(4)]
        for g, w in zip(got if isinstance(got, tuple) else (got,), zip(*want) if isinstance(want[0], tuple) else (want,)):
            torch.testing.assert_close(g, torch.stack(w), **CLOSE, msg=name)


def test_vmap_over_seeds_gives_each_sample_its_mask():
    """Seeds in a tensor: the kernels get one a sample."""
    seeds, x = torch.tensor([3, 4, 9]), rand(50, seed=1)
    with torch.library._scoped_library("mamtorch_b200", "IMPL") as lib:
        lib.impl("dropout_forward", lambda x, res, rate, seed, at: drop(x, rate, seed + int(at)), "CPU")
        got = torch.func.vmap(lambda s: MF.dropout(x, 0.5, s))(seeds)
    assert torch.equal(got, torch.stack([drop(x, 0.5, int(s)) for s in seeds]))


# ---------------------------------------------------------------- torch.compile

def test_compiled_calls_take_any_seed(cpu_kernels):
    """A seed is an argument of the compiled graph, not a constant of it: one graph for the first, one for all others."""
    from torch._dynamo.testing import CompileCounterWithBackend

    def step(x, seed):
        y, s = MF.dropout_add_layer_norm(MF.gelu(x, 0.25, seed), x, W, B, 1e-5, 0.5, seed + 1)
        return MF.dropout(y, 0.5, seed + 2, residual=s)

    torch._dynamo.reset()
    counter = CompileCounterWithBackend("aot_eager")
    compiled = torch.compile(step, backend=counter, fullgraph=True)
    for seed in (3, 4, 2 ** 61 + 5, 7, 11, 2 ** 62 - 9, 10 ** 9, 12, 13, 14, 15, 16):
        x, z = X.clone().requires_grad_(), X.clone().requires_grad_()
        got, want = compiled(x, seed), step(z, seed)
        assert torch.equal(got, want)
        torch.testing.assert_close(torch.autograd.grad(got, x, V), torch.autograd.grad(want, z, V), **CLOSE)
    assert counter.frame_count <= 2
    torch._dynamo.reset()


def test_compiled_calls_that_draw_their_seeds(cpu_kernels):
    """The draw from torch's CPU generator breaks the graph; what follows it is compiled once more, not for each number."""
    from torch._dynamo.testing import CompileCounterWithBackend

    torch._dynamo.reset()
    counter = CompileCounterWithBackend("aot_eager")
    step = lambda x: MF.gelu(MF.dropout(x, 0.5) * 2)     # noqa: E731
    compiled = torch.compile(step, backend=counter)
    for k in range(12):
        torch.manual_seed(k)
        got = compiled(X)
        torch.manual_seed(k)
        assert torch.equal(got, step(X))
    assert counter.frame_count <= 4
    torch._dynamo.reset()


def test_seeds_are_whole_64_bit_numbers(cpu_kernels):
    seen = []
    with torch.library._scoped_library("mamtorch_b200", "IMPL") as lib:
        lib.impl("dropout_forward", lambda x, res, rate, seed, at: seen.append(seed) or x.clone(), "CPU", allow_override=True)
        seeds = (0, -1, 2 ** 63 - 1, -2 ** 63, -2 ** 62 - 7, 2 ** 62 + 1)
        for seed in seeds:
            x = X.clone().requires_grad_()
            torch.autograd.grad(MF.dropout(x, 0.5, seed), x, V)
    assert [int(s) for s in seen] == [s for s in seeds for _ in range(2)]
    for seed in (2 ** 63, -2 ** 63 - 1):
        with pytest.raises((TypeError, RuntimeError, OverflowError)):
            MF.dropout(X, 0.5, seed)


def test_a_seed_drawn_for_a_cpu_tensor_asks_no_driver():
    for f in (lambda: MF.dropout(X, 0.5), lambda: MF.gelu(X, 0.5), lambda: MF.dropout_add_layer_norm(X, X, drop_rate=0.5)):
        with pytest.raises(NotImplementedError):
            f()
