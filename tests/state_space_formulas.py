"""The operators of a state space block and their gradients in float64, from the formulas, and the bounds their float
results keep.

Each function takes a dict of float64 CPU tensors (absent parts None) and returns one of the outputs and gradients.  With
magnitudes=True every factor and term is taken by its absolute value: what comes out bounds every partial sum on the way to an
output, so that an output that `roundings` float operations lead to is off by at most roundings * 2^-24 of it, whatever
cancels.  A result kept in fewer bits is rounded once more, by half a step of its type at most."""
import torch


def _abs_if(magnitudes):
    return (lambda t: None if t is None else t.abs()) if magnitudes else (lambda t: t)


def inside(lengths, T, N):
    ends = torch.full((N,), T) if lengths is None else torch.as_tensor(lengths)
    ends = torch.where(ends < 0, ends + T + 1, ends)
    return torch.arange(T)[:, None] < ends, ends


def conv(p, magnitudes=False):
    m = _abs_if(magnitudes)
    x, kernel, bias, state, dy = p["x"], p["kernel"], p["bias"], p["state"], p["dy"]
    (T, N, D), W = x.shape, kernel.shape[0]
    mask, ends = inside(p["lengths"], T, N)
    state = x.new_zeros(W - 1, N, D) if state is None else state
    X = torch.cat([state, torch.where(mask[..., None], x, 0.0)])
    pre = sum(kernel[k] * X[k:k + T] for k in range(W)) + (0.0 if bias is None else bias)
    s = torch.sigmoid(pre)
    slope = s * (1 + pre * (1 - s)) if p["silu"] else torch.ones_like(pre)
    factor = s if p["silu"] else torch.ones_like(pre)
    if magnitudes:
        big = sum(m(kernel[k]) * m(X[k:k + T]) for k in range(W)) + (0.0 if bias is None else m(bias))
        # an error of pre goes into the sigmoid too, whose slope is at most 1/4
        y = big * (factor + 0.25 * big) if p["silu"] else big
        slope = s * (1 + pre.abs() * (1 - s)) + 1.1 * big if p["silu"] else slope
    else:
        y = pre * factor
    d = torch.where(mask[..., None], m(dy) * slope, 0.0)
    dX = torch.zeros_like(X)
    for k in range(W):
        dX[k:k + T] += m(kernel[k]) * d
    last = torch.stack([X[ends[n]:ends[n] + W - 1, n] for n in range(N)], 1) if W > 1 else X[:0]
    if p["dstate_out"] is not None:
        for n in range(N):
            dX[ends[n]:ends[n] + W - 1, n] += m(p["dstate_out"])[:, n]
    return {"y": torch.where(mask[..., None], y, 0.0), "state": m(last), "dx": dX[W - 1:], "dstate": dX[:W - 1],
            "dkernel": torch.stack([(d * m(X[k:k + T])).sum((0, 1)) for k in range(W)]), "dbias": d.sum((0, 1))}


def scan(p, magnitudes=False):
    m = _abs_if(magnitudes)
    x, delta, A, B, C, dy = p["x"], p["delta"], p["A"], p["B"], p["C"], p["dy"]
    T, N, D = x.shape
    S, G = A.shape[1], B.shape[2]
    mask, _ = inside(p["lengths"], T, N)
    zero = lambda t: torch.where(mask.reshape(T, N, *[1] * (t.dim() - 2)), t, 0.0)  # noqa: E731
    raw = zero(delta) + (0.0 if p["delta_bias"] is None else p["delta_bias"])
    dt = zero(torch.nn.functional.softplus(raw, threshold=80.0) if p["softplus"] else raw)
    dt_slope = torch.sigmoid(raw) if p["softplus"] else torch.ones_like(raw)
    a = torch.exp(dt[..., None] * A)
    x, B, C, dt, A = m(zero(x)), m(zero(B)), m(zero(C)), m(dt), m(A)
    B, C = B.repeat_interleave(D // G, 2), C.repeat_interleave(D // G, 2)  # [T,N,D,S]
    skip = x.new_zeros(D) if p["D"] is None else m(p["D"])
    z = None if p["z"] is None else zero(p["z"])
    if z is None:
        gate, gate_slope = torch.ones_like(x), torch.zeros_like(x)
    else:
        s = torch.sigmoid(z)
        gate, gate_slope = m(z * s), (s * (1 + m(z) * (1 - s)) if magnitudes else s * (1 + z * (1 - s)))
    h = x.new_zeros(N, D, S) if p["h0"] is None else m(p["h0"])
    hs = [h]
    for t in range(T):
        hs.append(a[t] * hs[-1] + (dt[t] * x[t])[..., None] * B[t])
    ypre = torch.stack([(C[t] * hs[t + 1]).sum(-1) for t in range(T)]) + skip * x
    q = zero(m(dy)) * gate
    G_ = torch.zeros_like(h) if p["dh_last"] is None else m(p["dh_last"])
    dx, ddelta, dA = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(A)
    dB, dC = x.new_zeros(T, N, G, S), x.new_zeros(T, N, G, S)
    groups = lambda t: t.view(N, G, D // G, S).sum(2)  # noqa: E731
    for t in reversed(range(T)):
        g = q[t][..., None] * C[t] + G_
        dC[t] = groups(q[t][..., None] * hs[t + 1])
        dB[t] = groups(g * (dt[t] * x[t])[..., None])
        du = (g * B[t]).sum(-1)
        G_ = a[t] * g
        w = G_ * hs[t]
        dx[t] = dt[t] * du + skip * q[t]
        ddelta[t] = (x[t] * du + (w * A).sum(-1)) * dt_slope[t]
        dA += (w * dt[t][..., None]).sum(0)
    dx, ddelta = zero(dx), zero(ddelta)
    return {"y": zero(ypre * gate), "h_last": hs[-1], "dx": dx, "ddelta": ddelta, "dA": dA, "dB": zero(dB), "dC": zero(dC),
            "dD": (q * x).sum((0, 1)), "dz": zero(m(dy)) * ypre * gate_slope, "ddelta_bias": ddelta.sum((0, 1)), "dh0": G_}


def norm(p, magnitudes=False):
    m = _abs_if(magnitudes)
    centered, eps = p["centered"], p["eps"]
    u, r, z, D = p["update"], p["residual"], p["gate"], p["update"].shape[-1]
    scale, after, before, bias = (p[k] for k in ("scale", "after_weight", "before_weight", "before_bias"))
    one = torch.ones(D, dtype=u.dtype)

    def unit(v, bound):
        mean = v.mean(-1, keepdim=True) if centered else torch.zeros_like(v[..., :1])
        inv = ((v - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
        return (v - mean) * inv, (bound + (bound.mean(-1, keepdim=True) if centered else 0.0)) * inv, inv

    def back(d, n, inv):
        along = (d * n).mean(-1, keepdim=True) * n
        mean = d.mean(-1, keepdim=True) if centered else 0.0
        return (d + along + mean) * inv if magnitudes else (d - along - mean) * inv

    n1, b1, inv1 = unit(u, u.abs()) if after is not None else (u, u.abs(), torch.ones_like(u[..., :1]))
    s = None if z is None else torch.sigmoid(z)
    silu = torch.ones_like(u) if z is None else z * s
    slope = torch.zeros_like(u) if z is None else s * (1 + (z.abs() if magnitudes else z) * (1 - s))
    w1 = one if after is None else after
    k = one if scale is None else scale
    out = n1 * w1 * silu * k + (0.0 if r is None else r)
    bound = (b1 * w1 * silu * k).abs() + (0.0 if r is None else r.abs())
    n2, b2, inv2 = unit(out, bound)
    if magnitudes:
        n1, n2, out, silu, w1, k = b1, b2, bound, silu.abs(), w1.abs(), k.abs()
    d = torch.zeros_like(u) if p["dout"] is None else m(p["dout"])
    result = {"out": out}
    if before is not None:
        w2 = m(before)
        result["normed"] = n2 * w2 + (0.0 if bias is None else m(bias))
        e = torch.zeros_like(u) if p["dnormed"] is None else m(p["dnormed"])
        result["dbefore"], result["dbias"] = (e * n2).flatten(0, -2).sum(0), e.flatten(0, -2).sum(0)
        d = d + back(e * w2, n2, inv2)
    result["dresidual"] = d
    result["dscale"] = (d * n1 * w1 * silu).flatten(0, -2).sum(0)
    result["dgate"] = d * k * n1 * w1 * slope
    dn = d * k * silu
    result["dafter"] = (dn * n1).flatten(0, -2).sum(0)
    result["dupdate"] = back(dn * w1, n1, inv1) if after is not None else dn * w1
    return result


def check(got, want, magnitude, roundings, what):
    """|got - want| within half a step of got's type and `roundings` float roundings of the magnitude."""
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    half_step = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny  # results below it are rounded to steps of tiny * eps
    g = got.detach().cpu().double()
    float_error = roundings * 2.0 ** -24 * magnitude
    bound = float_error + half_step * (want.abs() + float_error) + tiny
    over = (g - want).abs() - bound
    assert not g.isnan().any(), what
    assert over.max() <= 0 if over.numel() else True, "%s: off by %.3e where %.3e is allowed" % (
        what, float((g - want).abs().flatten()[over.argmax()]), float(bound.flatten()[over.argmax()]))
