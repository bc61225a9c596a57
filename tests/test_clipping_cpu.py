"""Clipping of gradients on the host: norms beyond a float's range."""
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
