"""Layer norm, dropout and GELU operators: first calls of a process, copies of modules, waits that run out, what GELU's form is
worth."""
import copy
import math
import os
import subprocess
import sys
import textwrap

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def fresh_process(code, *args):
    """Runs a program in a process of its own, from the repository's root; its output.  The process leaves without the
    interpreter's teardown, where torch's engine threads may abort it after backward passes from several threads (with
    torch's own operators too)."""
    env = dict(os.environ, PYTHONPATH=ROOT)
    code = textwrap.dedent(code) + "\nimport os, sys\nsys.stdout.flush()\nos._exit(0)\n"
    run = subprocess.run([sys.executable, "-c", code, *args], cwd=ROOT, env=env, capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    return run.stdout


def test_first_calls_from_several_threads(cuda):
    """Nothing of the library has run in the process yet: each thread may be the one that asks for a device's attributes, a
    kernel's shared memory or the flag's address.  Every width in every type, rows enough for the forward's ring."""
    out = fresh_process("""
        import threading
        from concurrent.futures import ThreadPoolExecutor
        import torch
        from mamtorch_b200.nn import functional as MF

        CASES = [(rows, width, t) for rows, width in ((300, 200), (2400, 1283), (300, 2500), (2400, 4096), (300, 7000), (64, 9000),
                                                      (2400, 1000), (300, 8192))
                 for t in (torch.float32, torch.bfloat16, torch.float16)]
        torch.cuda.init()
        start = threading.Barrier(8)

        def work(k, wait):
            rows, width, t = CASES[k]
            g = torch.Generator().manual_seed(k)
            x, r, gy = (torch.randn(rows, width, generator=g).to(t).cuda() for _ in range(3))
            x.requires_grad_()
            w, b = (torch.randn(width, generator=g).to(t).cuda().requires_grad_() for _ in range(2))
            torch.cuda.synchronize()
            if wait:
                start.wait(60)
            with torch.cuda.stream(torch.cuda.Stream()):
                y, s = MF.dropout_add_layer_norm(MF.gelu(x, 0.1, k), r, w, b, 1e-5, 0.1, k)
                z = MF.layer_norm(x, w, b)
                out = [y, s, z, *torch.autograd.grad((y, s, z), (x, w, b), (gy, gy, gy))]
                torch.cuda.current_stream().synchronize()
            return out

        with ThreadPoolExecutor(8) as pool:
            at_once = list(pool.map(lambda k: work(k, True), range(len(CASES))))
        for k, got in enumerate(at_once):
            for p, q in zip(got, work(k, False)):
                assert torch.equal(p, q), CASES[k]
        MF.check_device_flag()
        print("same")
    """)
    assert out.strip() == "same"


def test_copies_of_a_module_drop_their_own_elements_in_a_captured_graph(cuda):
    """In a capture the seeds come from a device counter, which a deep copy of the module copies."""
    from mamtorch_b200.nn.vit import MAMMlpBlock

    torch.manual_seed(0)
    block = MAMMlpBlock(64, 128, fused=True, drop_rate=0.5).to(cuda)
    twins = [block, copy.deepcopy(block), copy.deepcopy(block)]
    x = torch.randn(40, 64, device=cuda)
    with torch.no_grad():
        for twin in twins:
            twin(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [twin(x) for twin in twins]
            seeds = [twin.drop_args()[1] for twin in twins]
    seen = []
    for _ in range(3):
        graph.replay()
        # where the last dropout dropped, the output is the input
        masks = [y == x for y in outs]
        assert not any(torch.equal(masks[i], masks[j]) for i in range(3) for j in range(i))
        seen += [int(s) for s in seeds]
    assert len(set(seen)) == 9


@pytest.fixture
def late():
    """Whether a norm's first wait for a row counts as run out, for every group of threads and with its copies on their way."""
    from mamtorch_b200 import _lib

    L = _lib.lib()
    yield lambda on: _lib.check(L.mam_tune_set(6, int(on)), "mam_tune_set")
    _lib.check(L.mam_tune_set(6, 0), "mam_tune_set")
    L.mam_check_device_flag()


# rows through shared memory: by columns one or several rows at a time in a CTA, aligned and ragged; many rows a group, and few
RING_SHAPES = [(3000, 131), (3000, 1283), (2400, 8191), (3000, 136), (3000, 768), (20, 1024), (2400, 4096), (2500, 8192), (1, 200)]


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", RING_SHAPES)
def test_a_wait_that_runs_out_is_reported_and_leaves_the_device_usable(cuda, late, shape, t):
    from mamtorch_b200.nn import functional as MF

    rows, width = shape
    x, r, gy = (torch.randn(rows, width, device=cuda).to(t) for _ in range(3))
    x.requires_grad_()
    w, b = (torch.randn(width, device=cuda).to(t).requires_grad_() for _ in range(2))

    def forward():
        return [*MF.dropout_add_layer_norm(x, r, w, b, 1e-5, 0.1, 5), MF.layer_norm(x, w, b)]

    def grads(outs):
        return torch.autograd.grad(outs, (x, w, b), (gy, gy, gy))

    want = forward()
    want += grads(want)
    MF.check_device_flag()
    for _ in range(3):
        outs = forward()
        for call in (lambda: grads(outs), lambda: grads(forward())):     # noqa: B023
            late(True)
            with pytest.raises(RuntimeError, match="gave up"):
                call()       # a later call in it may find what an earlier one left
                MF.check_device_flag()
            late(False)
            torch.cuda.synchronize()
            try:
                MF.check_device_flag()
            except RuntimeError as e:      # a kernel that was launched before the report
                assert "gave up" in str(e)
        outs = forward()
        assert all(torch.equal(p, q) for p, q in zip([*outs, *grads(outs)], want))
        MF.check_device_flag()


def test_a_forward_whose_wait_runs_out_is_reported(cuda, late):
    from mamtorch_b200.nn import functional as MF

    # ragged rows, and wide 16-bit ones behind a residual: the forward's forms through shared memory
    for shape, t, add in (((3000, 1283), torch.bfloat16, False), ((3000, 201), torch.float32, True), ((2400, 4096), torch.float16, True)):
        x, r = (torch.randn(shape, device=cuda).to(t) for _ in range(2))
        call = (lambda: MF.dropout_add_layer_norm(x, r, drop_rate=0.1, drop_seed=5)) if add else (lambda: (MF.layer_norm(x),))   # noqa: B023
        want = call()
        late(True)
        call()
        with pytest.raises(RuntimeError, match="gave up"):
            MF.check_device_flag()
        late(False)
        assert all(torch.equal(p, q) for p, q in zip(call(), want))
        MF.check_device_flag()


def test_the_next_call_of_the_norm_reports_a_wait_that_ran_out(cuda, late):
    from mamtorch_b200.nn import functional as MF

    x = torch.randn(3000, 1283, device=cuda, requires_grad=True)     # ragged rows: the forward and the backward wait
    few = torch.randn(4, 64, device=cuda)                            # no form of these waits
    gy = torch.randn_like(x)
    want = MF.layer_norm(few)

    def left_behind(call):
        late(True)
        call()
        torch.cuda.synchronize()
        late(False)

    y = MF.layer_norm(x)
    for call in (lambda: MF.layer_norm(x.detach()), lambda: torch.autograd.grad(y, x, gy, retain_graph=True),
                 lambda: MF.dropout_add_layer_norm(x.detach(), x.detach(), drop_rate=0.1, drop_seed=1)):
        for report in (lambda: MF.layer_norm(few), lambda: MF.dropout_add_layer_norm(few, few),
                       lambda: torch.autograd.grad(y, x, gy, retain_graph=True), MF.check_device_flag, MF.poll_device_flag):
            left_behind(call)
            with pytest.raises(RuntimeError, match="gave up"):
                report()
            # once
            assert torch.equal(MF.layer_norm(few), want)
            MF.check_device_flag()
    # in a capture nothing is reported; what a replay leaves behind the next eager call finds
    graph = torch.cuda.CUDAGraph()
    left_behind(lambda: MF.layer_norm(x.detach()))
    with torch.cuda.graph(graph):
        z = MF.layer_norm(x.detach())
    with pytest.raises(RuntimeError, match="gave up"):
        MF.layer_norm(few)
    graph.replay()
    torch.cuda.synchronize()
    MF.check_device_flag()      # captured without the hook
    assert torch.equal(z, y)


def test_the_first_call_of_a_process_inside_a_capture(cuda):
    """The library's look-ups (attributes, shared memory, flag, pinned word) happen while a stream is being captured."""
    for backward in ("", "1"):
        out = fresh_process("""
            import sys
            import torch
            from mamtorch_b200.nn import functional as MF

            backward = bool(sys.argv[1])
            x = torch.randn(3000, 1280 if backward else 1283, device="cuda", requires_grad=backward)
            gy = torch.randn_like(x)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = [MF.layer_norm(x)]
                if backward:
                    out += torch.autograd.grad(out[0], x, gy)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.detach().clone() for t in out]
            y = MF.layer_norm(x)
            want = [y.detach(), *(torch.autograd.grad(y, x, gy) if backward else ())]
            assert all(torch.equal(p, q) for p, q in zip(got, want))
            MF.check_device_flag()
            print("same")
        """, backward)
        assert out.strip() == "same"


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1 << 22, (1 << 21) + 1])
def test_gelu_over_a_dense_grid(cuda, n, t):
    """The elementwise error of GELU and its slope on [-15, 15], in eps = 2^-24, half a step of fp32.

    fp32, a = |x| < 0.85: q = -Phi(-a) = a R - 1/2.  R's roundings are 1.36 eps of R (its last step one, the step before and a^2
    damped by the coefficients), a R / Phi(-a) is 2.15 at most (at 1), the coefficients are off by 0.1 eps, q rounds once, and so
    does its product with a: 2.15 * 1.36 + 0.6 + 2 = 5.6 eps relative.  The slope's sum a c e + 1/2 + q: a c e within 1.5 eps (e = ex2,
    two units in the last place, its argument twice rounded; a c), two additions, q within 1.36 eps a R + eps / 4: 3.6 eps.
    Elsewhere, and in 16-bit types everywhere, Phi(-a) = s(t) t e: t within 3 eps (sum, reciprocal), each step of s one eps of its
    value, e as above, two products, and the coefficients: a Phi(-a) within 3.2 eps, 3.4 in 16-bit types, the slope's sum within
    5.8 eps, 12 in 16-bit types.  Then one rounding to fp32 relative to the value, one to t, and the product with the upstream
    gradient, which is one."""
    from mamtorch_b200.nn import functional as MF

    eps, half = 2.0 ** -24, torch.finfo(t).eps / 2
    x = torch.linspace(-15, 15, n, device=cuda, dtype=torch.float64).to(t).requires_grad_()
    y = MF.gelu(x)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    z = x.detach().double()
    phi = 0.5 * torch.erfc(-z / math.sqrt(2))
    want, slope = z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps
    near = (z.abs() < 0.85) & (t == torch.float32)
    far_y, far_slope = (3.2, 5.8) if t == torch.float32 else (3.4, 12.0)
    rounded = 0.0 if t == torch.float32 else half
    bound = torch.where(near, 5.6 * eps * want.abs(), far_y * eps + eps * want.abs()) + rounded * want.abs() + tiny
    assert ((y.detach().double() - want).abs() - bound).max().item() <= 0
    bound = torch.where(near, 3.6 * eps, torch.full_like(slope, far_slope * eps)) + (eps + rounded) * slope.abs() + tiny
    assert ((dx.double() - slope).abs() - bound).max().item() <= 0
    if t == torch.float32:      # no less exact than the erff form that it stands for: 10 % for the grid's luck
        other = torch.nn.functional.gelu(x.detach()).double()
        middle = (z.abs() < 1) & (z != 0)
        rms = lambda v: ((v - want)[middle] / want[middle]).square().mean().sqrt().item()   # noqa: E731
        assert rms(y.detach().double()) <= 1.1 * rms(other)
        assert (y.detach().double() - want).abs().max() <= (other - want).abs().max()


def test_compiled_calls_take_any_seed(cuda):
    from torch._dynamo.testing import CompileCounterWithBackend

    from mamtorch_b200.nn import functional as MF

    w, b = torch.randn(72, device=cuda), torch.randn(72, device=cuda)
    gy = torch.randn(40, 72, device=cuda)

    def step(x, seed):
        y, s = MF.dropout_add_layer_norm(MF.gelu(x, 0.25, seed), x, w, b, 1e-5, 0.5, seed + 1)
        return MF.dropout(y, 0.5, seed + 2, residual=s)

    torch._dynamo.reset()
    counter = CompileCounterWithBackend("aot_eager")
    compiled = torch.compile(step, backend=counter, fullgraph=True)
    for seed in (3, 4, 2 ** 61 + 5, 7, 11, 2 ** 62 - 9, 12, 13, 14, 15, 16, 17):
        x = torch.randn(40, 72, device=cuda, requires_grad=True)
        got, want = compiled(x, seed), step(x, seed)
        assert torch.equal(got, want)
        # the same kernels on the same numbers; autograd may add x's three gradients in another order
        torch.testing.assert_close(torch.autograd.grad(got, x, gy), torch.autograd.grad(want, x, gy), rtol=1e-5, atol=1e-5)
    assert counter.frame_count <= 2
    # a drawn seed: a new one at each call, and none inside a capture, however the call was compiled
    drawn = torch.compile(lambda v: MF.dropout(v, 0.5), backend="aot_eager")
    x = torch.ones(4096, device=cuda)
    assert not torch.equal(drawn(x), drawn(x))
    with pytest.raises(RuntimeError, match="capture"), pytest.warns(UserWarning, match="empty"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            drawn(x)
    torch._dynamo.reset()


def test_a_compiled_module_in_a_captured_graph_drops_anew_at_each_replay(cuda):
    """Compiled outside of a capture first: that answer must not stay."""
    from mamtorch_b200.nn.vit import MAMMlpBlock

    torch._dynamo.reset()
    torch.manual_seed(0)
    block = MAMMlpBlock(64, 128, fused=True, drop_rate=0.5).to(cuda)
    compiled = torch.compile(block, backend="aot_eager")
    x = torch.randn(40, 64, device=cuda)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                compiled(x)
        torch.cuda.current_stream().wait_stream(side)
        assert not torch.equal(compiled(x), compiled(x))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = compiled(x)
        outs = []
        for _ in range(3):
            graph.replay()
            outs.append(y.clone())
    assert not torch.equal(outs[0], outs[1]) and not torch.equal(outs[1], outs[2])
    torch._dynamo.reset()
