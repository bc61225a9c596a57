"""The state space block's operators without a GPU: what they refuse, and the layers' plain forms against the formulas and
against differences."""
import ctypes

import pytest
import torch

import haste_amd
from haste_amd import layers, lib, ops

import state_space_formulas as formulas

SUFFIXES = ("_f32", "_f16", "_bf16")


# ---- refusals of the C entry points: nothing is read, nothing launched ----------------------
def _entry(name, *values):
    fn = lib.entry(name)
    return fn(*values, None)


def _conv_forward(sfx, T=4, N=2, D=8, W=4, x=256, kernel=256, y=256):
    return _entry("haste_hip_causal_conv_forward" + sfx, T, N, D, W, x, 16, 8, kernel, None, 1, None, None, y, None)


def _conv_backward(sfx, T=4, N=2, D=8, W=4, bytes=1 << 20, workspace=256, **missing):
    a = dict(x=256, kernel=256, dy=256, dx=256, dkernel=256)
    a.update(missing)
    return _entry("haste_hip_causal_conv_backward" + sfx, T, N, D, W, a["x"], 16, 8, a["kernel"], None, 1, None, None, a["dy"], 16, 8,
                  None, a["dx"], a["dkernel"], None, None, workspace, bytes)


def _scan(direction, sfx, T=4, N=2, D=8, S=16, G=1, workspace=256, bytes=1 << 20, z=None, dz=None, **missing):
    a = {k: 256 for k in ("x", "delta", "A", "B", "C", "y", "kept", "dy", "dx", "ddelta", "dA", "dB", "dC")}
    a.update(missing)
    ins = [a["x"], 16, 8, a["delta"], 16, 8, a["A"], a["B"], 32, 16, a["C"], 32, 16, None, z, 16, 8, None, 1]
    if direction == "forward":
        return _entry("haste_hip_selective_scan_forward" + sfx, T, N, D, S, G, *ins, None, None, a["y"], None, None, workspace, bytes)
    return _entry("haste_hip_selective_scan_backward" + sfx, T, N, D, S, G, *ins, None, a["kept"], a["dy"], 16, 8, None, a["dx"],
                  a["ddelta"], a["dA"], a["dB"], a["dC"], None, dz, None, None, workspace, bytes)


def _norm(direction, sfx, T=4, N=2, D=8, before=256, normed=256, before_bias=None, dnormed=256, workspace=256, bytes=1 << 20, **missing):
    a = {k: 256 for k in ("update", "out", "stats", "dupdate")}
    a.update(missing)
    ins = [a["update"], 16, 8, None, 0, 0, None, 0, 0, None, 256, before]
    if direction == "forward":
        return _entry("haste_hip_residual_norm_forward" + sfx, T, N, D, *ins, before_bias, 0, 1e-5, a["out"], normed, a["stats"])
    return _entry("haste_hip_residual_norm_backward" + sfx, T, N, D, *ins, 0, a["stats"], 256, 16, 8, dnormed, 16, 8, a["dupdate"],
                  None, None, None, None, None, None, workspace, bytes)


@pytest.mark.parametrize("sfx", SUFFIXES)
def test_entry_points_refuse_bad_arguments(sfx):
    INVALID, UNSUPPORTED = 1, 2
    for sizes in (dict(T=0), dict(N=0), dict(D=0), dict(W=0), dict(T=-1), dict(x=None), dict(kernel=None), dict(y=None)):
        assert _conv_forward(sfx, **sizes) == INVALID, sizes
    for sizes in (dict(W=9), dict(T=2 ** 30 + 1), dict(D=2 ** 28)):
        assert _conv_forward(sfx, **sizes) == UNSUPPORTED, sizes
    for sizes in (dict(T=0), dict(dy=None), dict(dx=None), dict(dkernel=None), dict(workspace=None)):
        assert _conv_backward(sfx, **sizes) == INVALID, sizes
    for sizes in (dict(W=9), dict(bytes=64)):
        assert _conv_backward(sfx, **sizes) == UNSUPPORTED, sizes
    for direction in ("forward", "backward"):
        for sizes in (dict(T=0), dict(N=-3), dict(S=0), dict(G=0), dict(G=3), dict(x=None), dict(delta=None), dict(A=None),
                      dict(B=None), dict(C=None)):
            assert _scan(direction, sfx, **sizes) == INVALID, (direction, sizes)
        for sizes in (dict(S=65), dict(T=2 ** 30 + 1), dict(D=2 ** 26)):
            assert _scan(direction, sfx, **sizes) == UNSUPPORTED, (direction, sizes)
        for sizes in (dict(T=0), dict(D=0), dict(update=None)):
            assert _norm(direction, sfx, **sizes) == INVALID, (direction, sizes)
        for sizes in (dict(D=8193), dict(T=2 ** 30, N=2)):
            assert _norm(direction, sfx, **sizes) == UNSUPPORTED, (direction, sizes)
    for sizes in (dict(kept=None), dict(dy=None), dict(dx=None), dict(ddelta=None), dict(dA=None), dict(dB=None), dict(dC=None),
                  dict(workspace=None), dict(z=256, dz=None), dict(z=None, dz=256)):
        assert _scan("backward", sfx, **sizes) == INVALID, sizes
    assert _scan("backward", sfx, bytes=64) == UNSUPPORTED
    assert _scan("forward", sfx, y=None) == INVALID
    for sizes in (dict(out=None), dict(normed=None), dict(before=None), dict(before=None, normed=None, before_bias=256)):
        assert _norm("forward", sfx, **sizes) == INVALID, sizes
    for sizes in (dict(stats=None), dict(dupdate=None), dict(workspace=None), dict(before=None)):
        assert _norm("backward", sfx, **sizes) == INVALID, sizes
    assert _norm("backward", sfx, bytes=64) == UNSUPPORTED
    step = lambda N=2, S=16, G=1, **m: _entry("haste_hip_selective_scan_iterate" + sfx, N, 8, S, G, m.get("x", 256), 8, 256, 8, 256, 256,  # noqa: E731
                                              16, 256, 16, None, None, 0, None, 1, m.get("h", 256), m.get("y", 256), m.get("h_out", 256))
    for sizes in (dict(N=0), dict(G=5), dict(x=None), dict(h=None), dict(y=None), dict(h_out=None)):
        assert step(**sizes) == INVALID, sizes
    assert step(S=65) == UNSUPPORTED


def test_sizes_of_workspaces():
    handle = lib.load()
    for name, count in (("haste_hip_causal_conv_workspace_bytes", 4), ("haste_hip_selective_scan_workspace_bytes", 6),
                        ("haste_hip_selective_scan_kept_bytes", 4), ("haste_hip_residual_norm_workspace_bytes", 3)):
        fn = handle[name]
        fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_int] * count
        assert fn(*[1] * count) >= 0
        assert fn(*[0] * count) == 0
        assert fn(*[1] * (count - 1), 100000 if "norm" in name else 2 ** 30) == 0
    kept = handle["haste_hip_selective_scan_kept_bytes"]
    kept.restype, kept.argtypes = ctypes.c_size_t, [ctypes.c_int] * 4
    assert kept(4096, 64, 4096, 64) == 256 * 64 * 4096 * 64 * 4  # beyond 32 bits


# ---- refusals of the ops, shapes first: they are seen without a GPU -----------------------
def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


CONV = dict(x=_t(5, 2, 6), kernel=_t(4, 6), bias=_t(6), silu=True, state=_t(3, 2, 6), lengths=None)
SCAN = dict(x=_t(5, 2, 6), delta=_t(5, 2, 6), A=_t(6, 4), B=_t(5, 2, 2, 4), C=_t(5, 2, 2, 4), D=_t(6), z=_t(5, 2, 6),
            delta_bias=_t(6), delta_softplus=True, h0=_t(2, 6, 4), lengths=None)
NORM = dict(update=_t(5, 2, 6), residual=_t(5, 2, 6), gate=_t(5, 2, 6), scale=_t(6), after_weight=_t(6), before_weight=_t(6),
            before_bias=_t(6))


@pytest.mark.parametrize("change", [
    dict(x=_t(5, 6)), dict(x=_t(0, 2, 6)), dict(x=None), dict(kernel=_t(9, 6)), dict(kernel=_t(0, 6)), dict(kernel=_t(4, 5)),
    dict(kernel=_t(4, 6, dtype=torch.float16)), dict(bias=_t(5)), dict(state=_t(4, 2, 6)), dict(state=_t(3, 2, 6, dtype=torch.float16)),
    dict(lengths=torch.zeros(3, dtype=torch.int64)), dict(lengths=torch.zeros(2, dtype=torch.int32)),
    dict(x=_t(5, 2, 6, dtype=torch.float64), state=None), {}])
def test_conv_ops_refuse(change):
    arguments = dict(CONV, **change)
    with pytest.raises(ValueError):
        ops.causal_conv_forward(**arguments)
    with pytest.raises(ValueError):
        ops.causal_conv_backward(**arguments, dy=_t(5, 2, 6))


@pytest.mark.parametrize("change", [
    dict(x=_t(5, 6)), dict(x=_t(5, 0, 6)), dict(delta=_t(5, 2, 5)), dict(delta=_t(5, 2, 6, dtype=torch.float16)), dict(A=_t(5, 4)),
    dict(A=_t(6, 65)), dict(A=_t(6, 0)), dict(A=None), dict(B=_t(5, 2, 4, 4)), dict(B=_t(5, 2, 2, 3)), dict(C=_t(5, 2, 4)), dict(B=None),
    dict(C=None), dict(D=_t(5)), dict(z=_t(2, 5, 6)), dict(delta_bias=_t(7)), dict(h0=_t(2, 6, 5)), dict(h0=_t(2, 6, 4, dtype=torch.float16)),
    dict(lengths=torch.zeros(3, dtype=torch.int64)), {}])
def test_scan_ops_refuse(change):
    arguments = dict(SCAN, **change)
    with pytest.raises(ValueError):
        ops.selective_scan_forward(True, **arguments)
    if "h0" not in change:
        with pytest.raises(ValueError):
            ops.selective_scan_backward(**arguments, cache=_t(4), dy=_t(5, 2, 6))
    step = {k: v[0] if torch.is_tensor(v) and v.dim() in (3, 4) and k != "h0" else v for k, v in arguments.items()}
    step["h"] = step.pop("h0")
    step.pop("lengths")
    if "lengths" not in change:
        with pytest.raises(ValueError):
            ops.selective_scan_iterate(**step)


@pytest.mark.parametrize("change", [
    dict(update=_t(6)), dict(update=_t(5, 0, 6)), dict(update=_t(2, 9000)), dict(residual=_t(5, 2, 5)), dict(gate=_t(2, 6)),
    dict(gate=_t(5, 2, 6, dtype=torch.float16)), dict(scale=_t(5)), dict(scale=_t(1)), dict(after_weight=_t(6, dtype=torch.float64)),
    dict(before_weight=_t(7)), dict(before_weight=None), dict(before_bias=_t(3)), {}])
def test_norm_ops_refuse(change):
    arguments = dict(NORM, **change)
    with pytest.raises(ValueError):
        ops.residual_norm_forward(**arguments)
    with pytest.raises(ValueError):
        ops.residual_norm_backward(**arguments, stats=_t(5, 2, 4), dout=_t(5, 2, 6), dnormed=None)


def test_layers_refuse():
    for bad in (lambda: layers.CausalConv(8, width=9), lambda: layers.CausalConv(8, width=0), lambda: layers.SelectiveScan(8, 65),
                lambda: layers.SelectiveScan(8, 4, groups=3)):
        with pytest.raises(ValueError):
            bad()
    conv = layers.CausalConv(6)
    with pytest.raises(IndexError):
        conv(torch.zeros(5, 2, 6), lengths=[6, 1])
    with pytest.raises(ValueError):
        conv(torch.zeros(5, 2, 6), lengths=[5, 1, 1])


# ---- the layers' plain forms ----------------------------------------------------------
def _random(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64)


def _gradients(outs, ups, leaves):
    return dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), ups)))


@pytest.mark.parametrize("lengths", [None, [0, 4, -3]])
@pytest.mark.parametrize("W,silu", [(1, True), (4, True), (3, False), (8, True)])
def test_plain_conv(W, silu, lengths):
    n = _random(W)
    p = dict(x=n(5, 3, 4), kernel=n(W, 4), bias=n(4), state=n(W - 1, 3, 4), dy=n(5, 3, 4), dstate_out=n(W - 1, 3, 4), silu=silu,
             lengths=lengths)
    layer = haste_amd.CausalConv(4, W, silu=silu).double()
    layer.kernel.data, layer.bias.data = p["kernel"], p["bias"]
    x, state = p["x"].clone().requires_grad_(), p["state"].clone().requires_grad_()
    y, last = layer(x, state, lengths)
    got = _gradients([y, last], [p["dy"], p["dstate_out"]], dict(dx=x, dstate=state, dkernel=layer.kernel, dbias=layer.bias))
    got.update(y=y, state=last)
    want = formulas.conv(p)
    assert set(got) == set(want)
    for k in want:
        assert torch.allclose(got[k].detach(), want[k], rtol=1e-12, atol=1e-12), k


@pytest.mark.parametrize("lengths", [None, [0, 6, -3]])
@pytest.mark.parametrize("G", [1, 2])
def test_plain_scan(G, lengths):
    n = _random(G)
    p = dict(x=n(6, 3, 4), delta=n(6, 3, 4), A=-n(4, 5).abs(), B=n(6, 3, G, 5), C=n(6, 3, G, 5), D=n(4), z=n(6, 3, 4),
             delta_bias=n(4), h0=n(3, 4, 5), dy=n(6, 3, 4), dh_last=n(3, 4, 5), softplus=True, lengths=lengths)
    layer = haste_amd.SelectiveScan(4, 5, G).double()
    layer.log_decay.data, layer.skip.data, layer.delta_bias.data = (-p["A"]).log(), p["D"], p["delta_bias"]
    leaves = {k: p[k].clone().requires_grad_() for k in ("x", "delta", "z", "h0")}
    leaves.update({k: p[k].flatten(2).clone().requires_grad_() for k in ("B", "C")})
    y, last = layer(leaves["x"], leaves["delta"], leaves["B"], leaves["C"], leaves["z"], leaves["h0"], lengths)
    got = _gradients([y, last], [p["dy"], p["dh_last"]],
                     dict({"d" + k: v for k, v in leaves.items()}, dA=layer.log_decay, dD=layer.skip, ddelta_bias=layer.delta_bias))
    got["dA"] = got["dA"] / p["A"]
    got.update(y=y, h_last=last)
    want = formulas.scan(p)
    assert set(got) == set(want)
    for k in want:
        assert torch.allclose(got[k].detach().view_as(want[k]), want[k], rtol=1e-11, atol=1e-12), k


@pytest.mark.parametrize("centered", [False, True])
@pytest.mark.parametrize("absent", [(), ("residual",), ("gate", "scale"), ("after",), ("before",)])
def test_plain_norm(absent, centered):
    n = _random(7)
    p = dict(update=n(3, 2, 5), residual=n(3, 2, 5), gate=n(3, 2, 5), scale=n(5), after_weight=n(5), before_weight=n(5),
             before_bias=n(5) if centered else None, dout=n(3, 2, 5), dnormed=n(3, 2, 5), centered=centered, eps=1e-5)
    layer = haste_amd.ResidualNorm(5, centered, "after" not in absent, "before" not in absent, None if "scale" in absent else 1.0).double()
    for k in ("residual", "gate"):
        if k in absent:
            p[k] = None
    for k in ("scale", "after_weight", "before_weight", "before_bias"):
        if getattr(layer, k) is None:
            p[k] = None
        else:
            getattr(layer, k).data = p[k]
    leaves = {k: p[k].clone().requires_grad_() for k in ("update", "residual", "gate") if p[k] is not None}
    out, normed = layer(leaves["update"], leaves.get("residual"), leaves.get("gate"))
    outs, ups = ([out], [p["dout"]]) if normed is None else ([out, normed], [p["dout"], p["dnormed"]])
    weights = {n_: w for n_, w in (("dscale", layer.scale), ("dafter", layer.after_weight), ("dbefore", layer.before_weight),
                                   ("dbias", layer.before_bias)) if w is not None}
    got = _gradients(outs, ups, dict({"d" + k: v for k, v in leaves.items()}, **weights))
    got["out"] = out
    if normed is not None:
        got["normed"] = normed
    want = formulas.norm(p)
    for k in got:
        assert torch.allclose(got[k].detach(), want[k], rtol=1e-10, atol=1e-11), k


def test_formulas_against_differences():
    """The formulas' gradients, which the kernels are held to, from differences of their values."""
    n = _random(3)
    scan = dict(x=n(4, 2, 4), delta=n(4, 2, 4), A=-n(4, 3).abs(), B=n(4, 2, 2, 3), C=n(4, 2, 2, 3), D=n(4), z=n(4, 2, 4), delta_bias=n(4),
                h0=n(2, 4, 3), dy=n(4, 2, 4), dh_last=n(2, 4, 3), softplus=True, lengths=[3, 4])
    conv = dict(x=n(4, 2, 3), kernel=n(3, 3), bias=n(3), state=n(2, 2, 3), dy=n(4, 2, 3), dstate_out=n(2, 2, 3), silu=True, lengths=[1, 4])
    norm = dict(update=n(3, 2, 5), residual=n(3, 2, 5), gate=n(3, 2, 5), scale=n(5), after_weight=n(5), before_weight=n(5), before_bias=n(5),
                dout=n(3, 2, 5), dnormed=n(3, 2, 5), centered=True, eps=1e-5)
    for function, p, ups, grads in (
            (formulas.scan, scan, dict(y="dy", h_last="dh_last"),
             {k: "d" + k for k in ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0")}),
            (formulas.conv, conv, dict(y="dy", state="dstate_out"), {k: "d" + k for k in ("x", "kernel", "bias", "state")}),
            (formulas.norm, norm, dict(out="dout", normed="dnormed"),
             dict(update="dupdate", residual="dresidual", gate="dgate", scale="dscale", after_weight="dafter", before_weight="dbefore",
                  before_bias="dbias"))):
        value = lambda q: sum((function(q)[o] * p[d]).sum() for o, d in ups.items())  # noqa: E731, B023
        gradients = function(p)
        for name, grad in grads.items():
            along = n(*p[name].shape)
            step = 1e-6
            up, down = (value(dict(p, **{name: p[name] + sign * step * along})) for sign in (1, -1))
            want = (gradients[grad] * along).sum()
            assert abs((up - down) / (2 * step) - want) <= 1e-6 * (1 + abs(want)), (function.__name__, name)


def test_a_block_steps_like_it_runs():
    """The layers together over a sequence, and the same one step at a time from the states they hand on."""
    torch.manual_seed(0)
    conv, scan, norm = haste_amd.CausalConv(8, 4), haste_amd.SelectiveScan(8, 4, 2), haste_amd.ResidualNorm(8)
    x, delta, B, C, z = (torch.randn(6, 2, k) for k in (8, 8, 8, 8, 8))
    u, conv_state = conv(x)
    y, h = scan(u, delta, B, C, z)
    out, normed = norm(y, x, z)
    state, hs = torch.zeros(3, 2, 8), None
    for t in range(6):
        ut, state = conv.step(x[t], state)
        yt, hs = scan.step(ut, delta[t], B[t], C[t], z[t], hs)
        ot, nt = norm(yt, x[t], z[t])
        assert torch.allclose(ot, out[t], atol=1e-5) and torch.allclose(nt, normed[t], atol=1e-5)
    assert torch.allclose(state, conv_state) and torch.allclose(hs, h, atol=1e-5)
