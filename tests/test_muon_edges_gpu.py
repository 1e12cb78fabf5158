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
