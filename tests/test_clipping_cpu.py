"""Clipping of gradients on the host: norms beyond a float's range, parameters listed twice."""
import torch

import haste_amd


def _parameters(*grads):
    parameters = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(parameters, grads):
        p.grad = g.clone()
    return parameters


def test_a_norm_beyond_a_float_clips_by_what_it_is():
    for grads in ([torch.full((2,), 3e38)], [torch.full((7,), 2e38), torch.full((5,), 3e38, dtype=torch.bfloat16)]):
        exact = sum(g.double().square().sum() for g in grads).sqrt()
        for max_norm in (1.0, 1e-3, 1e30):
            parameters = _parameters(*grads)
            assert haste_amd.clip_gradients_(parameters, max_norm).isinf()
            for p, g in zip(parameters, grads):
                want = g.double() * (max_norm / exact)
                assert ((p.grad.double() - want).abs() <= 2 * torch.finfo(g.dtype).eps * want).all()


def test_a_factor_below_a_floats_range_loses_nothing():
    g = torch.tensor([3e37, -1e37, 1e20])
    parameters = _parameters(g)
    norm = haste_amd.clip_gradients_(parameters, 1e-9)
    want = g.double() * (1e-9 / norm.double())
    assert norm.isfinite() and ((parameters[0].grad.double() - want).abs() <= 2 * torch.finfo(torch.float32).eps * want.abs()).all()


def test_infinite_gradients_are_no_numbers():
    parameters = _parameters(torch.tensor([1.0, float("inf")]))
    assert haste_amd.clip_gradients_(parameters, 1.0).isinf()
    assert parameters[0].grad[0] == 0 and parameters[0].grad[1].isnan()


def test_a_parameter_that_is_listed_twice_counts_once():
    a, b = _parameters(torch.tensor([3.0, 0.0]), torch.tensor([4.0]))
    assert haste_amd.clip_gradients_([a, b, a], 1.0) == 5
    assert (a.grad - torch.tensor([0.6, 0.0])).abs().max() <= 1e-6 and (b.grad - 0.8).abs() <= 1e-6
    shared = torch.nn.Parameter(torch.zeros(2))
    shared.grad = a.grad  # the same gradient of two parameters
    assert abs(float(haste_amd.clip_gradients_(iter([a, shared, a]), 0.3)) - 0.6) <= 1e-6
    assert abs(float(a.grad[0]) - 0.3) <= 1e-6
