"""How far the state space operators' results may be off, by how the kernels add: like state_space_formulas.check, but a sum over a row
counts the roundings that any of its terms goes through (a few serial additions and a tree) instead of its terms, results below the
normal range are held to their own steps, and every output that is due has to be there."""
import torch

# A row of norms: 8 elements of a thread in turn, 6 additions over lanes, up to 16 wavefronts in turn.
ROW_SUM = 8 + 6 + 16


def parts_depth(parts):
    """Roundings of a sum over the partials that workgroups leave: a quarter of 256 in turn, two more for the quarters, again."""
    depth = 0
    while True:
        depth += min(-(-parts // 4), 64) + 2
        if parts <= 256:
            return depth
        parts = -(-parts // 256)


def check(got, want, magnitude, roundings, what):
    """|got - want| within half a step of got's type and `roundings` float roundings of the magnitude."""
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    info = torch.finfo(got.dtype)
    half_step = 0.0 if got.dtype == torch.float32 else info.eps / 2
    # Below the normal range a half has steps of tiny * eps; what has float's exponents may be flushed there (the exp2 and
    # reciprocal instructions do).
    least = info.tiny * info.eps if got.dtype == torch.float16 else info.tiny
    g = got.detach().cpu().double()
    assert g.isfinite().all(), what
    float_error = roundings * 2.0 ** -24 * magnitude
    bound = float_error + half_step * (want.abs() + float_error) + least
    over = (g - want).abs() - bound
    if over.numel() and over.max() > 0:
        at = over.flatten().argmax()
        raise AssertionError("%s: off by %.3e where %.3e is allowed" % (what, float((g - want).abs().flatten()[at]),
                                                                       float(bound.flatten()[at])))


def compare(got, want, magnitudes, roundings, absent=()):
    """roundings: a number, or a dict of them with one for the rest under None."""
    assert {k for k, v in got.items() if v is not None} == set(want) - set(absent)
    for k, v in got.items():
        if v is not None:
            check(v, want[k], magnitudes[k], roundings.get(k, roundings.get(None)) if isinstance(roundings, dict) else roundings, k)
