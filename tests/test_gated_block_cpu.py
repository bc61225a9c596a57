"""The operators of a gated linear recurrent block without a GPU: what they refuse, and the layers' plain forms against the formulas
and against differences."""
import ctypes

import pytest
import torch

import haste_amd
from haste_amd import layers, lib, ops

import gated_block_formulas as formulas

SUFFIXES = ("_f32", "_f16", "_bf16")
INVALID, UNSUPPORTED = 1, 2


# ---- refusals of the C entry points: nothing is read, nothing launched ----------------------
def _entry(name, *values):
    fn = lib.entry(name)
    return fn(*values, None)


def _linear(direction, sfx, R=4, C=8, D=16, x_row=8, dy_row=16, act=0, cache=None, workspace=256, bytes=1 << 30, **missing):
    a = {k: 256 for k in ("x", "kernel", "y", "dy")}
    a.update(missing)
    if direction == "forward":
        return _entry("haste_hip_linear_forward" + sfx, R, C, D, a["x"], x_row, a["kernel"], None, act, None, 0, a["y"], cache, workspace, bytes)
    return _entry("haste_hip_linear_backward" + sfx, R, C, D, a["x"], x_row, a["kernel"], act, cache, a["dy"], dy_row, 256, 256, None,
                  workspace, bytes)


def _gated(direction, sfx, T=4, N=2, D=8, admit=None, z=None, dadmit=None, dz=None, workspace=256, bytes=1 << 30, **missing):
    a = {k: 256 for k in ("x", "forget", "y", "kept", "dy", "dx", "dforget")}
    a.update(missing)
    ins = [a["x"], 16, 8, a["forget"], 16, 8, admit, 16, 8, z, 16, 8, None, None, None]
    if direction == "forward":
        return _entry("haste_hip_gated_recurrence_forward" + sfx, T, N, D, *ins, None, None, a["y"], None, None, workspace, bytes)
    return _entry("haste_hip_gated_recurrence_backward" + sfx, T, N, D, *ins, None, a["kept"], a["dy"], 16, 8, None, a["dx"], a["dforget"],
                  dadmit, dz, None, None, None, None, workspace, bytes)


@pytest.mark.parametrize("sfx", SUFFIXES)
def test_entry_points_refuse_bad_arguments(sfx):
    for direction in ("forward", "backward"):
        for bad in (dict(R=0), dict(C=0), dict(D=-1), dict(x=None), dict(kernel=None), dict(act=3), dict(act=-1), dict(x_row=7)):
            assert _linear(direction, sfx, **bad) == INVALID, (direction, bad)
        for bad in (dict(R=2 ** 30 + 1), dict(C=2 ** 20 + 1), dict(D=2 ** 20 + 1), dict(R=2 ** 30, D=2 ** 20), dict(x_row=2 ** 22 + 1)):
            assert _linear(direction, sfx, **bad) == UNSUPPORTED, (direction, bad)
        for bad in (dict(T=0), dict(N=-1), dict(D=0), dict(x=None), dict(forget=None)):
            assert _gated(direction, sfx, **bad) == INVALID, (direction, bad)
        for bad in (dict(T=2 ** 30 + 1), dict(N=2 ** 30, D=2 ** 10)):
            assert _gated(direction, sfx, **bad) == UNSUPPORTED, (direction, bad)
    assert _linear("forward", sfx, y=None) == INVALID
    for bad in (dict(dy=None), dict(act=1, cache=None), dict(dy_row=15), dict(workspace=None, D=15, dy_row=15), dict(bytes=0, D=15, dy_row=15),
                dict(workspace=257)):
        assert _linear("backward", sfx, **bad) == INVALID, bad
    assert _gated("forward", sfx, y=None) == INVALID
    assert _gated("forward", sfx, T=5000, workspace=None) == INVALID and _gated("forward", sfx, T=5000, bytes=64) == INVALID
    for bad in (dict(kept=None), dict(dy=None), dict(dx=None), dict(dforget=None), dict(admit=256), dict(z=256), dict(workspace=None), dict(bytes=8)):
        assert _gated("backward", sfx, **bad) == INVALID, bad
    step = lambda N=2, D=8, **m: _entry("haste_hip_gated_recurrence_iterate" + sfx, N, D, m.get("x", 256), 8, m.get("forget", 256), 8,  # noqa: E731
                                        None, 0, None, 0, None, None, None, m.get("h", 256), m.get("y", 256), m.get("h_out", 256))
    for bad in (dict(N=0), dict(D=0), dict(x=None), dict(forget=None), dict(h=None), dict(y=None), dict(h_out=None)):
        assert step(**bad) == INVALID, bad
    assert step(N=2 ** 30, D=2 ** 10) == UNSUPPORTED


def _clip(gradients, clipped, elements, types, max_norm=1.0, given=1, norm=64, workspace=None, bytes=0, count=None):
    n = len(gradients)
    return _entry("haste_hip_clip_gradients", n if count is None else count, (ctypes.c_void_p * n)(*gradients), (ctypes.c_void_p * n)(*clipped),
                  (ctypes.c_size_t * n)(*elements), (ctypes.c_int * n)(*types), max_norm, given, norm, 0, workspace, bytes)


def test_clipping_refuses_bad_arguments():
    far = 1 << 40
    for change in (dict(gradients=[None]), dict(clipped=[None]), dict(types=[4]), dict(types=[-1]), dict(max_norm=-1.0),
                   dict(max_norm=float("nan")), dict(norm=None), dict(given=0), dict(given=0, workspace=256, bytes=8),
                   dict(given=0, workspace=260, bytes=1 << 20), dict(count=-1)):
        call = dict(dict(gradients=[far], clipped=[far], elements=[8], types=[0]), **change)
        assert _clip(**call) == INVALID, change
    assert _clip([far], [far], [(1 << 40) + 1], [0]) == UNSUPPORTED
    # what is written and something else: twice the same, halves swapped, one byte over, an input behind another output
    for gradients, clipped, elements in (([far, far], [far, far], [8, 8]), ([far, far + 32], [far + 32, far], [8, 8]), ([far], [far + 1], [8]),
                                         ([far, far + 64], [far + 1024, far + 16], [8, 8]),
                                         ([far, far + 4096], [far + 1024, far + 1028], [8, 8])):
        assert _clip(gradients, clipped, elements, [0] * len(elements)) == INVALID, (gradients, clipped)


def test_sizes_of_workspaces():
    handle = lib.load()

    def size(name, *sizes):
        fn = handle[name]
        fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_int] * len(sizes)
        return fn(*sizes)
    linear, gated = "haste_hip_linear_workspace_bytes", "haste_hip_gated_recurrence_workspace_bytes"
    for bad in ((0, 2, 0, 8, 8, 1), (0, 3, 8, 8, 8, 1), (1, 2, 8, 2 ** 20 + 1, 8, 1), (1, 4, 2 ** 30, 8, 2 ** 20, 1)):
        assert size(linear, *bad) == 0, bad
    assert size(linear, 0, 2, 16384, 4096, 4096, 1) == 0  # nothing to copy, no pieces
    assert size(linear, 0, 2, 16384, 4095, 4096, 1) >= 16384 * 4096 * 2  # a copy of x in whole pieces
    assert size(linear, 0, 2, 16384, 4096, 4096, 0) >= (16384 + 4096) * 4096 * 2
    assert size(linear, 1, 2, 2 ** 21, 8, 2048, 1) >= 2 ** 33  # beyond 32 bits
    assert size(gated, 1, 0, 2, 8) == 0 and size(gated, 0, 2 ** 30 + 1, 2, 8) == 0 and size(gated, 1, 4, 2 ** 30, 2 ** 10) == 0
    assert size("haste_hip_gated_recurrence_kept_bytes", 4096, 4096, 4096) == 128 * 4096 * 4096 * 4  # a state for 32 steps
    assert size("haste_hip_gated_recurrence_kept_bytes", 0, 1, 1) == 0
    assert size("haste_hip_gradient_norm_workspace_bytes", -1) == 0 and size("haste_hip_gradient_norm_workspace_bytes", 1000) > 0


# ---- refusals of the ops, shapes first: they are seen without a GPU -----------------------
def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(x=_t(6)), dict(x=_t(0, 6)), dict(x=_t(2, 2, 2, 6)), dict(kernel=_t(5, 4)), dict(kernel=_t(6)), dict(kernel=_t(6, 0)),
    dict(kernel=_t(6, 4, dtype=torch.float16)), dict(bias=_t(5)), dict(bias=_t(4, dtype=torch.bfloat16)), dict(activation="relu"),
    dict(activation=None), dict(x=_t(3, 6, dtype=torch.float64), kernel=_t(6, 4, dtype=torch.float64), bias=None), {}])
def test_linear_ops_refuse(change):
    a = dict(dict(x=_t(3, 6), kernel=_t(6, 4), bias=_t(4), activation="silu"), **change)
    with pytest.raises(ValueError):
        ops.linear_forward(True, **a)
    with pytest.raises(ValueError):
        ops.linear_backward(**a, cache=_t(3, 4), dy=_t(3, 4))


@pytest.mark.parametrize("change", [
    dict(x=_t(5, 6)), dict(x=_t(5, 0, 6)), dict(x=None), dict(forget=None), dict(forget=_t(5, 2, 5)), dict(forget=_t(5, 2, 6, dtype=torch.float16)),
    dict(admit=_t(2, 5, 6)), dict(admit=None), dict(z=_t(5, 2)), dict(decay=_t(5)), dict(decay=_t(6, dtype=torch.float16)),
    dict(forget_bias=_t(1)), dict(admit_bias=_t(7)), dict(h0=_t(2, 5)), dict(h0=_t(2, 6, dtype=torch.float16)),
    dict(lengths=torch.zeros(3, dtype=torch.int64)), {}])
def test_gated_ops_refuse(change):
    a = dict(dict(x=_t(5, 2, 6), forget=_t(5, 2, 6), admit=_t(5, 2, 6), z=_t(5, 2, 6), decay=_t(6), forget_bias=_t(6), admit_bias=_t(6),
                  h0=_t(2, 6), lengths=None), **change)
    with pytest.raises(ValueError):
        ops.gated_recurrence_forward(True, **a)
    with pytest.raises(ValueError):
        ops.gated_recurrence_backward(**a, cache=_t(4), dy=_t(5, 2, 6))
    if "lengths" not in change:
        step = {k: v[0] if torch.is_tensor(v) and v.dim() == 3 else v for k, v in a.items() if k not in ("lengths", "h0")}
        with pytest.raises(ValueError):
            ops.gated_recurrence_iterate(**step, h=a["h0"])


def test_clip_ops_refuse():
    for bad in (None, [], _t(4), [_t(4)], [_t(4, dtype=torch.int32)], [None]):
        with pytest.raises(ValueError):
            ops.gradient_norm(bad)
        with pytest.raises(ValueError):
            ops.clip_gradients(bad, 1.0)


def test_layers_refuse():
    with pytest.raises(ValueError):
        layers.Linear(4, 4, activation="relu")
    x = torch.zeros(5, 2, 6)
    with pytest.raises(ValueError):
        layers.GatedRecurrence(6)(x, x)
    with pytest.raises(ValueError):
        layers.GatedRecurrence(6, admit=False)(x, x, x)
    with pytest.raises(IndexError):
        layers.GatedRecurrence(6, admit=False)(x, x, lengths=[6, 1])


# ---- the layers' plain forms ----------------------------------------------------------
def _random(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64)


def _linear_values(n, activation, residual=True):
    return dict(x=n(3, 2, 5), kernel=n(5, 4), bias=n(4), residual=n(3, 2, 4) if residual else None, dy=n(3, 2, 4), activation=activation,
                dtype=torch.float32)


def _gated_values(n, decay, admit, z, lengths, T=6):
    return dict(x=n(T, 3, 4), forget=n(T, 3, 4), admit=n(T, 3, 4) if admit else None, z=n(T, 3, 4) if z else None,
                decay=n(4).abs() + 0.1 if decay else None, forget_bias=n(4), admit_bias=n(4) if admit else None, h0=n(3, 4), dy=n(T, 3, 4),
                dh_last=n(3, 4), lengths=lengths)


@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
def test_plain_linear(activation):
    p = _linear_values(_random(1), activation)
    layer = haste_amd.Linear(5, 4, activation=activation).double()
    layer.kernel.data, layer.bias.data = p["kernel"], p["bias"]
    x, residual = p["x"].clone().requires_grad_(), p["residual"].clone().requires_grad_()
    y = layer(x, residual)
    got = dict(zip(("dx", "dkernel", "dbias", "dresidual"), torch.autograd.grad(y, [x, layer.kernel, layer.bias, residual], p["dy"])), y=y)
    want = formulas.linear(p)
    for k, (value, error) in want.items():
        assert torch.allclose(got[k].detach(), value, rtol=1e-11, atol=1e-12), k
        assert (error >= 0).all() and error.shape == value.shape
    assert torch.equal(got["dresidual"], p["dy"])


@pytest.mark.parametrize("lengths", [None, [0, 6, -3]])
@pytest.mark.parametrize("decay,admit,z", [(d, a, z) for d in (0, 1) for a in (0, 1) for z in (0, 1)])
def test_plain_gated(decay, admit, z, lengths):
    p = _gated_values(_random(2), decay, admit, z, lengths)
    layer = haste_amd.GatedRecurrence(4, bool(decay), bool(admit)).double()
    layer.forget_bias.data = p["forget_bias"]
    if decay:
        layer.log_decay.data = p["decay"].log()
    if admit:
        layer.admit_bias.data = p["admit_bias"]
    leaves = {k: p[k].clone().requires_grad_() for k in ("x", "forget", "admit", "z", "h0") if p[k] is not None}
    y, h = layer(leaves["x"], leaves["forget"], leaves.get("admit"), leaves.get("z"), leaves["h0"], lengths)
    weights = {"ddecay": layer.log_decay, "dforget_bias": layer.forget_bias, "dadmit_bias": layer.admit_bias}
    named = dict({"d" + k: v for k, v in leaves.items()}, **{k: v for k, v in weights.items() if v is not None})
    got = dict(zip(named, torch.autograd.grad([y, h], list(named.values()), [p["dy"], p["dh_last"]])), y=y, h_last=h)
    if decay:
        got["ddecay"] = got["ddecay"] / p["decay"]
    want = formulas.gated(p)
    assert set(got) == set(want)
    magnitudes = formulas.gated(p, True)
    for k in want:
        assert torch.allclose(got[k].detach(), want[k], rtol=1e-11, atol=1e-12), k
        assert (magnitudes[k] >= want[k].abs() - 1e-12).all(), k


def test_formulas_against_differences():
    """The formulas' gradients, which the kernels are held to, from differences of their values."""
    n = _random(3)
    cases = [(lambda q: {k: v for k, (v, _) in formulas.linear(q).items()}, _linear_values(n, a), dict(y="dy"), {k: "d" + k for k in ("x", "kernel", "bias")})
             for a in ("none", "gelu", "silu")]
    for decay, admit, z in ((1, 1, 1), (1, 0, 0), (0, 1, 1), (0, 0, 1)):
        p = _gated_values(n, decay, admit, z, [3, 6, 0])
        cases.append((formulas.gated, p, dict(y="dy", h_last="dh_last"), {k: "d" + k for k in (
            "x", "forget", "admit", "z", "decay", "forget_bias", "admit_bias", "h0") if p[k] is not None}))
    for function, p, ups, grads in cases:
        value = lambda q: sum((function(q)[o] * p[d]).sum() for o, d in ups.items())  # noqa: E731, B023
        gradients = function(p)
        for name, grad in grads.items():
            along = n(*p[name].shape)
            step = 1e-6
            up, down = (value(dict(p, **{name: p[name] + sign * step * along})) for sign in (1, -1))
            want = (gradients[grad] * along).sum()
            assert abs((up - down) / (2 * step) - want) <= 1e-6 * (1 + abs(want)), name


def test_the_bounds_see_a_mistake():
    """What a product that leaves out its last term, a slope of one and statistics in bfloat16 give is outside the bounds."""
    n = _random(4)
    p = dict(_linear_values(n, "gelu"), x=n(3, 2, 40).float().double(), kernel=n(40, 4).float().double() * 40 ** -0.5)
    want = formulas.linear(p)
    wrong = formulas.linear(dict(p, x=torch.cat([p["x"][..., :-1], 0 * p["x"][..., -1:]], -1)))
    for k in ("y", "dkernel"):
        with pytest.raises(AssertionError):
            formulas.check_error(wrong[k][0].float(), *want[k], k)
        formulas.check_error(want[k][0].float(), *want[k], k)
    with pytest.raises(AssertionError):
        formulas.check_error(formulas.linear(dict(p, activation="none"))["dx"][0].float(), *want["dx"], "dx")


def test_clipping_on_the_host():
    n = _random(5)
    a, b, c = (torch.nn.Parameter(n(*s).to(t)) for s, t in (((3, 4), torch.float32), ((7,), torch.float64), ((2,), torch.bfloat16)))
    unused = torch.nn.Parameter(n(2))
    for p in (a, b, c):
        p.grad = n(*p.shape).to(p.dtype)
    grads = [p.grad.double().clone() for p in (a, b, c)]
    norm = sum(g.square().sum() for g in grads).sqrt()
    got = haste_amd.clip_gradients_([a, b, c, unused], 0.5)
    assert got.dtype == torch.float64 and abs(float(got - norm)) <= 1e-12 and unused.grad is None
    for p, g in zip((a, b, c), grads):
        eps = torch.finfo(p.dtype).eps
        assert ((p.grad.double() - g * 0.5 / (norm + 1e-6)).abs() <= 2 * eps * g.abs()).all()
    before = [p.grad.clone() for p in (a, b, c)]
    haste_amd.clip_gradients_([a, b, c], 100.0)
    assert all(torch.equal(p.grad, g) for p, g in zip((a, b, c), before))
    assert float(haste_amd.clip_gradients_([unused], 1.0)) == 0
    with pytest.raises(ValueError):
        haste_amd.clip_gradients_(a, -1.0)


def test_a_block_steps_like_it_runs():
    torch.manual_seed(0)
    into, recur, back = haste_amd.Linear(6, 32, activation="silu"), haste_amd.GatedRecurrence(8), haste_amd.Linear(8, 6)
    x = torch.randn(6, 2, 6)
    y, h = recur(*into(x).chunk(4, -1))
    out, state = back(y, x), None
    for t in range(6):
        yt, state = recur.step(*into(x[t]).chunk(4, -1), state)
        assert torch.allclose(back(yt, x[t]), out[t], atol=1e-5)
    assert torch.allclose(state, h, atol=1e-5)
