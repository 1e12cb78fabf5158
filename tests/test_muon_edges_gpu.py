"""optim.orthogonalize and optim.Muon at the edges of what they take, against the same steps in float64."""
import math

import pytest
import torch

from cvnets_amd import optim

pytestmark = pytest.mark.gpu


def steps64(u, steps, coefficients, eps=1e-7):
    a, b, c = coefficients
    x = u.double().cpu()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if flip else x


def one_strong_direction(r, c, seed=0):
    """a singular value of nearly 1 after the division by the norm; the others follow 1e-3 and below"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.outer(torch.randn(r, generator=g, device="cuda"), torch.randn(c, generator=g, device="cuda"))
    return u + torch.randn(r, c, generator=g, device="cuda") * (1e-3 / math.sqrt(max(r, c)))


def growth(steps, coefficients):
    """(largest singular value after the steps, bound of the error) of the direction that starts at 1.

    A step's three products have errors of 2^-22 of the operands' norms (pairs of 11 bits, sums in float32), so the step adds at most
    3 * 2^-22 (|a| s + |b| s^3 + |c| s^5), and the steps behind it multiply what is there by at most |p'(s)| <= |a| + 3 |b| s^2 + 5 |c| s^4."""
    a, b, c = coefficients
    s, error = 1.0, 2.0 ** -23
    for _ in range(steps):
        error = error * (abs(a) + 3 * abs(b) * s ** 2 + 5 * abs(c) * s ** 4) + 3 * 2.0 ** -22 * (abs(a) * s + abs(b) * s ** 3 + abs(c) * s ** 5)
        s = abs(a * s + b * s ** 3 + c * s ** 5)
    return s, error


# (the largest singular value in front of each step; behind the last one it may be anything)
LARGE = [((5.0, -0.1, 0.0), 2), ((5.0, -0.1, 0.0), 3), ((2.0, 0.0, 0.0), 4), ((4.2, 0.0, 0.0), 2), ((3.5, -0.01, 0.0), 3), ((14.0, 0.5, 0.5), 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 640), (640, 1), (70, 100), (1030, 1100)])
@pytest.mark.parametrize("coefficients,steps", LARGE)
def test_singular_values_beyond_4(dtype, shape, coefficients, steps):
    """G = x x^T holds their squares, and P what the last step makes of them"""
    u = one_strong_direction(*shape).to(dtype)
    x, want = optim.orthogonalize(u, steps=steps, coefficients=coefficients), steps64(u, steps, coefficients)
    s, error = growth(steps, coefficients)
    got = x.detach().double().cpu()
    assert torch.isfinite(got).all()
    rounding = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    assert float((got - want).norm() / want.norm()) <= error / s + rounding


def test_two_captured_steps_side_by_side():
    """one optimizer, a graph for each half of its parameters, replayed on two streams at a time: the same weights as eager steps, to the bit"""
    def make():
        g = torch.Generator(device="cuda").manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda")) for s in ((600, 500), (500, 620), (640, 510), (512, 512))]
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g, device="cuda")
        return ps, optim.Muon(ps, lr=0.1)

    (ps, opt), (twins, eager) = make(), make()
    grads = [p.grad for p in ps]
    opt.step()
    eager.step()
    graphs = []
    for half in ((0, 1), (2, 3)):
        for i, p in enumerate(ps):
            p.grad = grads[i] if i in half else None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step(sync_hyperparameters=False)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for it in range(6):
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        eager.step()
        torch.cuda.synchronize()
        for p, q in zip(ps, twins):
            assert torch.equal(p, q), it
            assert torch.equal(opt.state[p]["momentum_buffer"], eager.state[q]["momentum_buffer"]), it


def test_a_capture_without_an_eager_step_is_refused():
    p = torch.nn.Parameter(torch.randn(20, 30, device="cuda"))
    p.grad = torch.randn(20, 30, device="cuda")
    opt, before = optim.Muon([p], lr=0.1), p.detach().clone()
    opt.sync_hyperparameters()
    for lr in (0.2, None):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(graph):
                opt.step()
        assert torch.equal(p, before)
        opt.step()
        before = p.detach().clone()
        opt.param_groups[0]["lr"] = lr or 0.1
    opt.sync_hyperparameters()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(p, before)


def rounded(coefficients):
    return tuple(torch.tensor(c, dtype=torch.float32).item() for c in coefficients)


FEW = [(1, 1), (1, 2500), (2, 7), (3, 50), (16, 33), (17, 300), (22, 22), (23, 1000), (33, 66000), (39, 41), (40, 40), (40, 2500), (5, 70001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", FEW)
def test_few_rows(dtype, shape):
    """up to 40 rows everything but the result is held in 64 bits: one rounding to the result's type (coefficients and eps are float32 numbers)"""
    coefficients, eps = rounded(optim.NS_COEFFICIENTS), rounded([1e-7])[0]
    for r, c in (shape, shape[::-1]):
        g = torch.Generator(device="cuda").manual_seed(r)
        u = (torch.randn(r, c, generator=g, device="cuda") * torch.logspace(0, -3, c, device="cuda")).to(dtype)
        for steps in (1, 5):
            got, want = optim.orthogonalize(u, steps=steps), steps64(u, steps, coefficients, eps)
            off = (got.double().cpu() - want).abs()
            assert bool((off <= want.abs() * (torch.finfo(dtype).eps / 2) + 1e-13).all()), float((off / want.abs().clamp(min=1e-30)).max())


@pytest.mark.parametrize("nesterov", [True, False])
def test_few_rows_among_others_and_in_the_optimizer(nesterov):
    """lists of few and many rows, each result that of its matrix alone; steps with momentum, rates and decay"""
    shapes = [(1, 300), (300, 2), (100, 130), (40, 700), (41, 60), (64, 7, 3, 3), (8, 1, 3, 3), (500, 33)]
    g = torch.Generator(device="cuda").manual_seed(7)
    mats = [torch.randn(s[0], math.prod(s[1:]), generator=g, device="cuda") for s in shapes]
    for x, u in zip(optim.orthogonalize(mats), mats):
        assert torch.equal(x, optim.orthogonalize(u))
    params = [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda") * 0.1) for s in shapes]
    opt = optim.Muon([{"params": params[::2], "lr": 0.05, "weight_decay": 0.1}, {"params": params[1::2]}], lr=0.01, momentum=0.9, nesterov=nesterov)
    want = [p.detach().double().cpu() for p in params]
    mom = [torch.zeros_like(w) for w in want]
    for _ in range(3):
        for i, p in enumerate(params):
            p.grad = torch.randn(p.shape, generator=g, device="cuda")
            g64 = p.grad.double().cpu()
            mom[i] = 0.9 * mom[i] + g64
            u = g64 + 0.9 * mom[i] if nesterov else mom[i]
            lr, wd = (0.05, 0.1) if i % 2 == 0 else (0.01, 0.0)
            x = steps64(u.reshape(p.shape[0], -1), 5, optim.NS_COEFFICIENTS)
            want[i] = want[i] * (1 - lr * wd) - lr * max(1.0, p.shape[0] / x.shape[1]) ** 0.5 * x.view(p.shape)
        opt.step()
    for p, w, m in zip(params, want, mom):
        assert float((p.detach().double().cpu() - w).norm() / w.norm()) <= 2.0 ** -17
        assert float((opt.state[p]["momentum_buffer"].double().cpu() - m).norm() / m.norm()) <= 2.0 ** -22


def test_few_rows_of_zeros_and_without_finite_values():
    z, bad, u = torch.zeros(7, 90, device="cuda"), torch.ones(30, 50, device="cuda"), torch.randn(9, 40, device="cuda")
    bad[3, 4] = float("inf")
    x = optim.orthogonalize([z, bad, u])
    assert torch.equal(x[0], z) and torch.isnan(x[1]).all() and torch.equal(x[2], optim.orthogonalize(u))
    for s in (1e-30, 1e25):  # squares outside float32
        want = steps64(u.double() * s, 5, rounded(optim.NS_COEFFICIENTS), 0.0)
        assert float(((optim.orthogonalize(u * s, eps=0.0).double().cpu() - want).norm() / want.norm())) <= 2.0 ** -22
