"""That the bounds of state_space_bounds.py hold what float computes and fail what fewer bits compute."""
import pytest
import torch

import state_space_bounds as bounds
import state_space_formulas as formulas


def _norm_problem(D, rows):
    gen = torch.Generator().manual_seed(D)
    normal = lambda *shape: torch.randn(*shape, generator=gen).double()  # noqa: E731
    p = {k: normal(rows, 1, D) for k in ("update", "residual", "gate", "dout", "dnormed")}
    p.update({k: normal(D) for k in ("scale", "after_weight", "before_weight", "before_bias")}, centered=True, eps=1e-5)
    return p


def _float_norm(p, keep):
    """The forward pass in float32, its statistics rounded by `keep`."""
    f = {k: v.float() if torch.is_tensor(v) else v for k, v in p.items()}

    def norm(v):
        mean = keep(v.mean(-1, keepdim=True))
        inv = keep(1 / torch.sqrt((v - mean).square().mean(-1, keepdim=True) + f["eps"]))
        return (v - mean) * inv

    out = f["residual"] + norm(f["update"]) * f["after_weight"] * f["scale"] * f["gate"] * torch.sigmoid(f["gate"])
    return {"out": out, "normed": norm(out) * f["before_weight"] + f["before_bias"]}


@pytest.mark.parametrize("D", [40, 700, 8192])
def test_bounds_of_norms_tell_fewer_bits(D):
    p = _norm_problem(D, 5)
    want, magnitude = formulas.norm(p), formulas.norm(p, True)
    roundings = 8 * (bounds.ROW_SUM + 32)
    for k, v in _float_norm(p, lambda t: t).items():
        bounds.check(v, want[k], magnitude[k], roundings, k)
    for k, v in _float_norm(p, lambda t: t.bfloat16().float()).items():
        with pytest.raises(AssertionError, match="off by"):
            bounds.check(v, want[k], magnitude[k], roundings, k)


def test_bounds_below_the_normal_range():
    want = torch.tensor([3.0 * 2 ** -24, 1e-5], dtype=torch.float64)
    bounds.check(want.half(), want, want, 0, "halves")
    with pytest.raises(AssertionError, match="off by"):
        bounds.check(want.half() * 0, want, want, 0, "flushed")


def test_outputs_that_are_missing_are_seen():
    t = torch.ones(2, dtype=torch.float64)
    bounds.compare(dict(a=t.float(), b=None), dict(a=t, b=t), dict(a=t, b=t), 1, absent=("b",))
    for got in (dict(a=t.float(), b=None), dict(a=t.float())):
        with pytest.raises(AssertionError):
            bounds.compare(got, dict(a=t, b=t), dict(a=t, b=t), 1)


def test_depths_of_sums_over_partials():
    assert [bounds.parts_depth(p) for p in (1, 5, 256, 257, 1024)] == [3, 4, 66, 66 + 3, 66 + 3]
    assert bounds.parts_depth(256 * 256 + 1) == 66 + 66 + 3
