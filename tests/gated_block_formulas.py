"""The operators of a gated linear recurrent block and their gradients in float64, from the formulas, and how far their float
results may be off (as state_space_formulas.py has it: with magnitudes=True every factor and term is taken by its absolute value)."""
import math

import torch

from state_space_formulas import inside


def activated(kind, pre):
    """act(pre) and its slope."""
    if kind == "gelu":
        below = 0.5 * torch.special.erfc(-pre * 0.5 ** 0.5)
        return pre * below, below + pre * torch.exp(-0.5 * pre * pre) * (2 * math.pi) ** -0.5
    if kind == "silu":
        s = torch.sigmoid(pre)
        return pre * s, s * (1 + pre * (1 - s))
    return pre, torch.ones_like(pre)


def linear(p):
    """{output: (value, bound on its error before it is rounded to its type)}.

    Sums: of K terms, at most K / 16 + 16 roundings one after another (the matrix instruction adds 16 terms at a time to
    what it is given, pieces of K are added up behind) of the sum of the terms' absolute values; floats are split in three
    parts whose six products go through two such sums, and what is left out is below two more roundings.  Few tiles of floats
    go through the float instruction instead, whose four terms take at most four roundings, 32 terms at a time: within K / 32 + 32.
    act(pre): its slope is at most 1.13, and its own evaluation is off by at most 16 roundings of |pre| + |act(pre)| (exponentials of
    arguments of a few units, whose relative error is as many roundings).
    d = dy act'(pre): act'' is at most 0.8, so that it is off by 0.8 times the error of pre and 16 roundings; kept in half
    (beside bfloat16; a float otherwise) and d itself in the type of x (no half, no rounding, for float and without an activation)."""
    x, W, bias, residual, dy, kind = (p[k] for k in ("x", "kernel", "bias", "residual", "dy", "activation"))
    dtype = p["dtype"]
    x, dy, shape = x.flatten(0, -2), dy.flatten(0, -2), (*x.shape[:-1], W.shape[1])
    u = 2.0 ** -24
    (R, C), D = x.shape, W.shape[1]
    factor = 2 if dtype == torch.float32 else 1

    def depth(K):
        return (factor * (K / 16 + 16) + 4 + 32) * u

    pre = x @ W
    big = x.abs() @ W.abs()
    if bias is not None:
        pre, big = pre + bias, big + bias.abs()
    pre_error = depth(C) * big
    y, slope = activated(kind, pre)
    y_error = pre_error if kind == "none" else 1.13 * pre_error + 16 * u * (pre.abs() + y.abs())
    if residual is not None:
        r = residual.flatten(0, -2)
        y, y_error = y + r, y_error + u * (y.abs() + r.abs())
    d = dy * slope
    if kind == "none":
        d_error = torch.zeros_like(d)
    else:
        d_error = dy.abs() * (0.8 * pre_error + 16 * u)
        if dtype != torch.float32:
            d_error = d_error + d.abs() * (2.0 ** -11 + torch.finfo(dtype).eps / 2) * 1.01 + dy.abs() * 2.0 ** -24
            if dtype == torch.float16:  # below the normal range
                d_error = d_error + 2.0 ** -25
    reach = d.abs() + d_error
    out = {"y": (y, y_error), "dx": (d @ W.t(), d_error @ W.abs().t() + depth(D) * (reach @ W.abs().t())),
           "dkernel": (x.t() @ d, x.abs().t() @ d_error + depth(R) * (x.abs().t() @ reach))}
    if bias is not None:  # four rows a wavefront in turn and what workgroups leave: within R / 64 + 64
        out["dbias"] = (d.sum(0), d_error.sum(0) + (R / 64 + 64) * u * reach.sum(0))
    return {k: (v.reshape(shape if k == "y" else p["x"].shape if k == "dx" else v.shape), e.reshape(v.shape if k not in ("y", "dx") else
                shape if k == "y" else p["x"].shape)) for k, (v, e) in out.items()}


def gated(p, magnitudes=False):
    m = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    x, forget, admit, z, decay, dy = (p[k] for k in ("x", "forget", "admit", "z", "decay", "dy"))
    T, N, D = x.shape
    mask = inside(p["lengths"], T, N)[0].to(x.device)[..., None]
    zero = lambda t: torch.where(mask, t, 0.0)  # noqa: E731
    raw = zero(forget) + (0.0 if p["forget_bias"] is None else p["forget_bias"])
    r, keep = torch.sigmoid(raw), torch.sigmoid(-raw)
    if admit is not None:
        araw = zero(admit) + (0.0 if p["admit_bias"] is None else p["admit_bias"])
        i, shut = torch.sigmoid(araw), torch.sigmoid(-araw)
    else:
        i, shut = torch.ones_like(x), torch.zeros_like(x)
    x = m(zero(x))
    if decay is not None:
        a, mult = torch.exp(-decay * r), torch.sqrt(-torch.expm1(-2 * decay * r))
        scale = mult * i
    else:
        a, mult = r, torch.ones_like(r)
        scale = i if admit is not None else keep
    silu = torch.ones_like(x) if z is None else m(zero(z) * torch.sigmoid(zero(z)))
    h = x.new_zeros(N, D) if p["h0"] is None else m(p["h0"])
    hs = [h]
    for t in range(T):
        hs.append(torch.where(mask[t], a[t] * hs[-1] + scale[t] * x[t], hs[-1]))
    H = torch.stack(hs)
    out = {"y": zero(H[1:] * silu), "h_last": H[-1]}
    dy = zero(m(dy))
    c = torch.zeros_like(h) if p["dh_last"] is None else m(p["dh_last"])
    gs = [None] * T
    for t in reversed(range(T)):
        gs[t] = dy[t] * silu[t] + c
        c = torch.where(mask[t], a[t] * gs[t], c)
    g = torch.stack(gs)
    out["dh0"] = c
    out["dx"] = zero(g * scale)
    minus = (lambda p_, q: p_ + q) if magnitudes else (lambda p_, q: p_ - q)
    if decay is not None:
        dlog = g * minus(H[:-1] * a, x * i * a * a / mult)
        dforget = decay * dlog * r * keep * (1 if magnitudes else -1)
        out["ddecay"] = zero(dlog * r * (1 if magnitudes else -1)).sum((0, 1))
        dadmit = g * mult * x * i * shut
    elif admit is not None:
        dforget, dadmit = g * H[:-1] * r * keep, g * x * i * shut
    else:
        dforget, dadmit = g * minus(H[:-1], x) * r * keep, None
    out["dforget"] = zero(dforget)
    out["dforget_bias"] = out["dforget"].sum((0, 1))
    if admit is not None:
        out["dadmit"] = zero(dadmit)
        out["dadmit_bias"] = out["dadmit"].sum((0, 1))
    if z is not None:
        s = torch.sigmoid(zero(z))
        out["dz"] = zero(dy * H[1:] * (s * (1 + m(zero(z)) * (1 - s))))
    return out


def check_error(got, want, error, what):
    """|got - want| within `error` and half a step of got's type; results below the normal range to its steps there."""
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    info = torch.finfo(got.dtype)
    half_step = info.eps / 2
    least = info.tiny * info.eps if got.dtype == torch.float16 else info.tiny
    g, want, error = got.detach().double().cpu(), want.cpu(), error.cpu()
    assert g.isfinite().all(), what
    over = (g - want).abs() - (error + half_step * (want.abs() + error) + least)
    if over.numel() and over.max() > 0:
        at = over.flatten().argmax()
        raise AssertionError("%s: off by %.3e where %.3e is allowed" % (
            what, float((g - want).abs().flatten()[at]), float((g - want).abs().flatten()[at] - over.flatten()[at])))
