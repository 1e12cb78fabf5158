"""What the orthogonalised update takes and refuses, without a GPU."""
import copy
import ctypes
import gc
import weakref

import numpy as np
import pytest
import torch

from cvnets_amd import _lib, optim


def largest(steps, coefficients, points=200001):
    """the largest singular value in front of the steps 2 .. `steps`, from points of 0 .. 1"""
    a, b, c = coefficients
    top, most = 1.0, 1.0
    for _ in range(steps - 1):
        s = np.linspace(0.0, top, points)
        top = float(np.abs(a * s + b * s ** 3 + c * s ** 5).max())
        most = max(most, top)
    return most


CASES = [(5, optim.NS_COEFFICIENTS), (50, optim.NS_COEFFICIENTS), (12, (1.875, -1.25, 0.375)), (30, (1.5, -0.5, 0.0)), (2, (5.0, -0.1, 0.0)), (3, (5.0, -0.1, 0.0)),
         (4, (5.0, -0.1, 0.0)), (4, (2.0, 0.0, 0.0)), (6, (2.0, 0.0, 0.0)), (2, (14.0, 0.5, 0.5)), (3, (14.0, 0.5, 0.5)), (1, (0.0, 0.0, -15.0)), (9, (0.0, 0.0, 0.0)),
         (4, (-3.0, 2.0, 0.1)), (5, (3.0, -3.5, 0.9)), (6, (-1.0, -2.0, 4.0)), (3, (0.0, 3.0, -1.0)), (7, (4.0, -6.0, 3.0))]


@pytest.mark.parametrize("steps,coefficients", CASES)
def test_coefficients_that_let_singular_values_grow_are_refused(steps, coefficients):
    bounded = largest(steps, coefficients) <= 15.0
    assert bool(_lib.load().cvh_ns_bounded(steps, *coefficients)) == bounded
    u = torch.zeros(4, 6)
    with pytest.raises(RuntimeError if bounded else ValueError):  # (bounded: the next refusal is that of a CPU tensor)
        optim.orthogonalize(u, steps=steps, coefficients=coefficients)
    p = torch.nn.Parameter(u)
    if bounded:
        optim.Muon([p], ns_steps=steps, ns_coefficients=coefficients)
    else:
        with pytest.raises(ValueError, match="grow beyond"):
            optim.Muon([p], ns_steps=steps, ns_coefficients=coefficients)
        m = (_lib.NsMatrix * 1)(_lib.NsMatrix(src=256, dst=256, momentum=256, param=256, rows=4, cols=6))
        assert _lib.load().cvh_orthogonalize(0, ctypes.byref(m), 1, steps, *coefficients, 1e-7, 256, None) == -2
        assert _lib.load().cvh_muon_step(ctypes.byref(m), 1, steps, *coefficients, 1e-7, 0.9, 1, 256, 256, None) == -2


def test_both_sides_of_the_bound_are_among_the_cases():
    assert {largest(*c) <= 15.0 for c in CASES} == {True, False}


@pytest.fixture
def launches(monkeypatch):
    """steps on CPU tensors up to the launch: the arguments that the kernels would get"""
    seen = []
    monkeypatch.setattr(optim.ops, "_check_dev", lambda t: None)
    monkeypatch.setattr(optim.ops, "call_on", lambda dev, name, *args: seen.append((name, *args)))
    return seen


def tensor_at(address):
    return next(t for t in gc.get_objects() if isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.numel() and t.data_ptr() == address)


def with_gradient(*shape):
    p = torch.nn.Parameter(torch.ones(shape))
    p.grad = torch.ones(shape)
    return p


def test_the_rates_of_a_group_that_was_added_are_handed_over(launches):
    """a step without synchronisation behind add_param_group: the kernels read the new group's row of the table, so there has to be one"""
    opt = optim.Muon([with_gradient(4, 6)], lr=0.5)
    opt.step()
    opt.add_param_group({"params": [with_gradient(6, 4)], "lr": 0.25, "weight_decay": 0.125})
    opt.step(sync_hyperparameters=False)
    table, rates = launches[-1][1]._obj, tensor_at(launches[-1][-2])
    assert sorted(table[i].group for i in range(2)) == [0, 1]
    assert rates[:2].tolist() == [[0.5, 0.0], [0.25, 0.125]]


def test_a_captured_step_keeps_its_table_of_rates(launches):
    """what a capture holds is the table's address: the table stays, and follows sync_hyperparameters(), after groups were added"""
    opt = optim.Muon([with_gradient(4, 6)], lr=0.5)
    opt.step()
    address = launches[-1][-2]
    held = weakref.ref(tensor_at(address))
    opt.add_param_group({"params": [with_gradient(6, 4)], "lr": 0.25})
    opt.step()
    gc.collect()
    assert held() is not None
    opt.param_groups[0]["lr"], opt.param_groups[0]["weight_decay"] = 0.125, 0.0625
    opt.sync_hyperparameters()
    assert tensor_at(address)[0].tolist() == [0.125, 0.0625]
    assert tensor_at(launches[-1][-2]).tolist() == [[0.125, 0.0625], [0.25, 0.0]]


def test_the_table_of_rates_is_on_the_parameters_device(launches):
    p = with_gradient(4, 6)
    opt = optim.Muon([p], lr=0.5)
    opt.step()
    with torch.no_grad():
        moved = torch.nn.Parameter(torch.ones(4, 6, device="meta"))
        moved.grad = torch.ones(4, 6, device="meta")
    opt.param_groups[0]["params"][0] = moved  # (what a module's .to(device) leaves behind where it replaces its parameters)
    opt.step(sync_hyperparameters=False)
    assert opt._rates[-1][0].device == moved.device


def test_a_transposed_square_parameter_or_momentum_is_refused(launches):
    """the same address and shape, another matrix"""
    p = with_gradient(4, 4)
    opt = optim.Muon([p], lr=0.5)
    opt.step()
    p.data = p.data.t()
    with pytest.raises(RuntimeError, match="another matrix"):
        opt.step()
    p.data = p.data.t()
    opt.step()
    opt.state[p]["momentum_buffer"] = torch.arange(16.0).view(4, 4).t()  # (a state that somebody else wrote: laid out again, the same values)
    opt.step()
    assert opt.state[p]["momentum_buffer"].is_contiguous() and torch.equal(opt.state[p]["momentum_buffer"], torch.arange(16.0).view(4, 4).t())
    opt.state[p]["momentum_buffer"] = opt.state[p]["momentum_buffer"].t()  # the same address
    want = opt.state[p]["momentum_buffer"].clone()
    opt.step()
    assert opt.state[p]["momentum_buffer"].is_contiguous() and torch.equal(opt.state[p]["momentum_buffer"], want)
    assert launches[-1][1]._obj[0].momentum == opt.state[p]["momentum_buffer"].data_ptr()


def test_a_loaded_state_goes_into_the_momentum_that_a_captured_step_holds(launches):
    p, q = with_gradient(4, 6), with_gradient(3, 5)
    opt = optim.Muon([p, q], lr=0.5)
    opt.step()
    held = {x: opt.state[x]["momentum_buffer"].data_ptr() for x in (p, q)}
    saved = copy.deepcopy(opt.state_dict())
    saved["state"][0]["momentum_buffer"].fill_(3.0)
    del saved["state"][1]  # a parameter that had not been stepped when the state was saved
    opt.state[q]["momentum_buffer"].fill_(2.0)
    opt.load_state_dict(saved)
    opt.step()
    assert {x: opt.state[x]["momentum_buffer"].data_ptr() for x in (p, q)} == held
    assert bool((opt.state[p]["momentum_buffer"] == 3.0).all()) and bool((opt.state[q]["momentum_buffer"] == 0.0).all())
    assert opt.state[p]["momentum_buffer"].data_ptr() != saved["state"][0]["momentum_buffer"].data_ptr()


def test_nothing_of_the_host_is_captured(launches, monkeypatch):
    """a capture would hold the address of a temporary for the rates, and would set the momentum to zero with every replay"""
    opt = optim.Muon([with_gradient(4, 6)], lr=0.5)
    capturing = [True]
    monkeypatch.setattr(optim, "_capturing", lambda device: capturing[0])
    with pytest.raises(RuntimeError, match="eager step"):
        opt.step(sync_hyperparameters=False)
    assert not launches
    capturing[0] = False
    opt.step()
    capturing[0] = True
    opt.step()  # nothing changed: nothing is copied
    opt.step(sync_hyperparameters=False)
    opt.param_groups[0]["lr"] = 0.25
    with pytest.raises(RuntimeError, match="sync_hyperparameters"):
        opt.step()
    opt.step(sync_hyperparameters=False)
    opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(3, 5))]})
    with pytest.raises(RuntimeError, match="sync_hyperparameters"):
        opt.step(sync_hyperparameters=False)  # (no row of rates for the new group)
    capturing[0] = False
    opt.sync_hyperparameters()
    capturing[0] = True
    opt.step(sync_hyperparameters=False)
    assert len(launches) == 5
