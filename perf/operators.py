"""The operators of a state space block whose speed is tracked: the short causal convolution, the
selective scan, and the norms around the block with their gate and residual scale, each in training,
over prompts and for single tokens.

Sizes are those of bench.py, haste_amd/benchmark_grid.py and the tests (batch 1 .. 128, widths 300 ..
4096, 50 .. 2500 steps) and ordinary prompt lengths.  A case is a dict:

  op       "conv", "scan" or "norm"
  mode     "train": forward and backward pass; "infer": forward pass; "step": one token per row
  dtype    of the activations: float32, float16 or bfloat16 (parameters, states and statistics are
           float32)
  T, N, D  time steps, batch rows, channels
  W        conv: taps
  S, G     scan: states per channel, groups of channels that share B and C
  lengths  the batch's sequences have lengths of their own (one of them may be empty)
  state    the sequence goes on from a given state (its gradient is returned)
  batch_first   tensors are slices of projections laid out [N, T, *] instead of [T, N, *]
  centered norm: layer norm instead of root mean square norm

With `own` false run() computes the operators from elementary operations of torch, in float32, and
rounds once; with `own` true it calls haste_amd.ops.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _case(op, mode, T, N, D, dtype="bfloat16", W=0, S=0, G=0, lengths=False, state=False, batch_first=False,
          centered=False, **name):
    return dict(name, op=op, mode=mode, dtype=dtype, T=T, N=N, D=D, W=W, S=S, G=G, lengths=lengths, state=state,
                batch_first=batch_first, centered=centered)


def listed():
    return [
        # One stream's next token through the convolution and the recurrence: nothing but latency.
        _case("conv", "step", 1, 1, 1024, W=4, state=True, name="conv_step_n1"),
        _case("scan", "step", 1, 1, 1024, S=16, G=1, state=True, name="scan_step_n1"),
        # A full serving batch's next token: 32 MiB of state in, and out again.
        _case("scan", "step", 1, 128, 4096, S=16, G=1, state=True, name="scan_step_n128"),
        # One long prompt by itself: few rows, so the steps have to be shared out.
        _case("scan", "infer", 4096, 1, 2048, S=16, G=1, name="scan_prompt_n1"),
        # An ordinary training step, and a large one.
        _case("scan", "train", 1024, 8, 1024, S=16, G=1, name="scan_train"),
        _case("scan", "train", 2048, 8, 4096, S=16, G=1, name="scan_train_large"),
        # Padded sequences that go on from a state; sizes that no tile divides, channels in three groups.
        _case("scan", "train", 500, 37, 300, dtype="float32", S=11, G=3, lengths=True, state=True, name="scan_train_ragged"),
        # The convolution of the large training step, and of padded sequences stored batch first.
        _case("conv", "train", 2048, 8, 4096, W=4, name="conv_train_large"),
        _case("conv", "infer", 83, 37, 75, dtype="float16", W=3, lengths=True, state=True, batch_first=True, name="conv_infer_ragged"),
        # The norms around a block: a token, the large training step, and layer norms of an odd width in float.
        _case("norm", "step", 1, 16, 512, dtype="float16", name="norm_step"),
        _case("norm", "train", 2048, 8, 4096, name="norm_train_large"),
        _case("norm", "train", 500, 32, 1001, dtype="float32", centered=True, name="norm_train_ragged"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "conv", "norm"])
    mode = rng.choice(["train", "train", "infer", "step"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    while True:
        N, D = _spread(rng, 1, 128), _spread(rng, 64, 4096)
        T = 1 if mode == "step" else _spread(rng, 1, 4096)
        if rng.random() < 0.5:  # widths that a configuration file would have
            D = max(64, D // 64 * 64)
        S = rng.choice([16, 16, 8, 11, 32, 64]) if op == "scan" else 0
        G = rng.choice([1, 1, 2, 4]) if op == "scan" else 0
        if T * N * D * max(S, 16) > 2048 * 8 * 4096 * 16:
            continue
        if op == "scan":
            D = D // G * G
        break
    case = _case(op, mode, T, N, D, dtype=dtype, S=S, G=G)
    if op == "conv":
        case["W"] = rng.choice([4, 4, 2, 3, 5, 8])
    if op == "norm":
        case["centered"] = rng.random() < 0.5
    if mode == "step":
        case["state"] = op != "norm"
    else:
        case["batch_first"] = rng.random() < 0.25
        if op != "norm":
            case["lengths"] = rng.random() < 0.25
            case["state"] = rng.random() < 0.25
    return case


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), _DTYPES[case["dtype"]]
    T, N, D, S, G, W = (case[k] for k in ("T", "N", "D", "S", "G", "W"))
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev).to(dtype)

    def uniform(low, high, *shape):
        return low + (high - low) * torch.rand(*shape, generator=gen, device=dev)

    def projection(*widths):
        """What a projection to sum(widths) columns left: its column blocks as [T,N,width] ([N,width])."""
        if case["mode"] == "step":
            full = normal(N, sum(widths), dtype=dtype)
        elif case["batch_first"]:
            full = normal(N, T, sum(widths), dtype=dtype).transpose(0, 1)
        else:
            full = normal(T, N, sum(widths), dtype=dtype)
        return full.split(widths, dim=-1)

    s = {"case": case}
    if case["lengths"]:
        s["lengths"] = torch.randint(max(1, T // 2), T + 1, (N,), generator=gen, device=dev)
        s["lengths"][-1:] = T
        if N > 2:
            s["lengths"][1] = 0
    else:
        s["lengths"] = None
    if case["op"] == "conv":
        s["x"] = projection(D, D)[0]
        s["kernel"] = uniform(-W ** -0.5, W ** -0.5, W, D)
        s["bias"] = uniform(-W ** -0.5, W ** -0.5, D)
        s["state"] = normal(W - 1, N, D, dtype=dtype) if case["state"] else None
        if case["mode"] == "train":
            s["dy"] = normal(T, N, D, dtype=dtype)
    elif case["op"] == "scan":
        s["z"] = projection(D, D)[1]
        s["x"] = torch.nn.functional.silu(projection(D)[0].float()).to(dtype)
        s["delta"] = (0.5 * projection(D)[0].float()).to(dtype)
        _, B, C = projection(max(1, D // 16), G * S, G * S)
        s["B"], s["C"] = B.unflatten(-1, (G, S)), C.unflatten(-1, (G, S))
        # The step sizes and decays that such layers start from, and move away from.
        dt = torch.exp(uniform(math.log(1e-3), math.log(0.1), D))
        s["delta_bias"] = dt + torch.log(-torch.expm1(-dt))
        s["A"] = -torch.arange(1, S + 1, device=dev) * torch.exp(0.2 * normal(D, S))
        s["skip"] = 1 + 0.1 * normal(D)
        s["h"] = 0.3 * normal(N, D, S) if case["state"] else None
        if case["mode"] == "train":
            s["dy"] = normal(T, N, D, dtype=dtype)
            s["dh"] = normal(N, D, S) if case["state"] else None
    else:
        s["update"], s["gate"] = projection(D, D)
        s["residual"] = projection(D)[0]
        s["scale"] = uniform(0.05, 0.5, D)
        s["after_weight"], s["before_weight"] = 1 + 0.1 * normal(D), 1 + 0.1 * normal(D)
        s["before_bias"] = 0.1 * normal(D) if case["centered"] else None
        if case["mode"] == "train":
            s["dout"], s["dnormed"] = normal(T, N, D, dtype=dtype), normal(T, N, D, dtype=dtype)
    return s


def run(s):
    op, mode = s["case"]["op"], s["case"]["mode"]
    if own:
        return {"conv": _own_conv, "scan": _own_scan, "norm": _own_norm}[op](s, mode)
    return {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}[op](s, mode)


# ---- the framework's calls ----------------------------------------------------------------
def _own_conv(s, mode):
    from haste_amd import ops
    if mode == "step":
        y, state = ops.causal_conv_iterate(s["x"], s["state"], s["kernel"], s["bias"], True)
        return {"y": y, "state": state}
    y, state = ops.causal_conv_forward(s["x"], s["kernel"], s["bias"], True, s["state"], s["lengths"])
    out = {"y": y, "state": state}
    if mode == "train":
        dx, dkernel, dbias, dstate = ops.causal_conv_backward(s["x"], s["kernel"], s["bias"], True, s["state"],
                                                              s["lengths"], s["dy"])
        out.update(dx=dx, dkernel=dkernel, dbias=dbias)
        if s["state"] is not None:
            out["dstate"] = dstate
    return out


def _own_scan(s, mode):
    from haste_amd import ops
    if mode == "step":
        y, h = ops.selective_scan_iterate(s["x"], s["delta"], s["A"], s["B"], s["C"], s["h"], s["skip"], s["z"],
                                          s["delta_bias"], True)
        return {"y": y, "h": h}
    y, h, cache = ops.selective_scan_forward(mode == "train", s["x"], s["delta"], s["A"], s["B"], s["C"], s["skip"], s["z"],
                                             s["delta_bias"], True, s["h"], s["lengths"])
    out = {"y": y, "h": h}
    if mode == "train":
        dx, ddelta, dA, dB, dC, dD, dz, dbias, dh0 = ops.selective_scan_backward(
            s["x"], s["delta"], s["A"], s["B"], s["C"], s["skip"], s["z"], s["delta_bias"], True, s["h"], s["lengths"],
            cache, s["dy"], s["dh"])
        out.update(dx=dx, ddelta=ddelta, dA=dA, dB=dB, dC=dC, dskip=dD, dz=dz, dbias=dbias)
        if s["h"] is not None:
            out["dh0"] = dh0
    return out


def _own_norm(s, mode):
    from haste_amd import ops
    parts = (s["update"], s["residual"], s["gate"], s["scale"], s["after_weight"], s["before_weight"], s["before_bias"])
    out, normed, stats = ops.residual_norm_forward(*parts, centered=s["case"]["centered"])
    if mode != "train":
        return {"out": out, "normed": normed}
    names = ("dupdate", "dresidual", "dgate", "dscale", "dafter", "dbefore", "dbias")
    grads = ops.residual_norm_backward(*parts, stats, s["dout"], s["dnormed"], centered=s["case"]["centered"])
    return {"out": out, "normed": normed, **{k: g for k, g in zip(names, grads) if g is not None}}


# ---- the plain forms: elementary operations in float32, rounded once at the end -----------
def _steps(s, names):
    """The tensors as [T,N,...] in float32 (a single token as one step)."""
    found = [s[k].float() for k in names]
    return [f.unsqueeze(0) for f in found] if s["case"]["mode"] == "step" else found


def _inside(s, T, N, device):
    """[T,N]: the steps that belong to each row's sequence."""
    if s["lengths"] is None:
        return torch.ones(T, N, dtype=torch.bool, device=device)
    return torch.arange(T, device=device)[:, None] < s["lengths"]


def _plain_conv(s, mode):
    (x,) = _steps(s, ["x"])
    (T, N, D), W, dtype = x.shape, s["case"]["W"], s["x"].dtype
    kernel, inside = s["kernel"], _inside(s, T, N, x.device)[..., None]
    before = torch.zeros(W - 1, N, D, device=x.device) if s["state"] is None else s["state"].float()
    padded = torch.cat([before, torch.where(inside, x, 0.0)])
    windows = padded.unfold(0, T, 1)  # [W,N,D,T]: what each tap sees
    pre = (windows * kernel[:, None, :, None]).sum(0).permute(2, 0, 1) + s["bias"]
    sigmoid = 1 / (1 + torch.exp(-pre))
    y = torch.where(inside, pre * sigmoid, 0.0).to(dtype)
    ends = torch.full((N,), T, device=x.device) if s["lengths"] is None else s["lengths"]
    rows = ends + torch.arange(W - 1, device=x.device)[:, None]
    state = padded[rows, torch.arange(N, device=x.device)].to(dtype)
    if mode == "step":
        return {"y": y[0], "state": state}
    out = {"y": y, "state": state}
    if mode == "train":
        dpre = torch.where(inside, s["dy"].float() * sigmoid * (1 + pre * (1 - sigmoid)), 0.0)
        around = torch.nn.functional.pad(dpre, (0, 0, 0, 0, W - 1, W - 1))
        seen_by = around.unfold(0, T + W - 1, 1)  # [W,N,D,T+W-1]: the outputs that use an input, the last tap's first
        dpadded = (seen_by * kernel.flip(0)[:, None, :, None]).sum(0).permute(2, 0, 1)
        out.update(dx=dpadded[W - 1:].to(dtype), dkernel=(windows * dpre.permute(1, 2, 0)).sum((1, 3)),
                   dbias=dpre.sum((0, 1)))
        if s["state"] is not None:
            out["dstate"] = dpadded[:W - 1].to(dtype)
    return out


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t over the first axis, in place of b (a is used up): log2(T) rounds, each
    of which doubles how many steps back every step reaches."""
    k = 1
    while k < b.shape[0]:
        b[k:] += a[k:] * b[:-k]
        a[k:] = a[k:] * a[:-k]
        k *= 2
    return b


def _plain_scan(s, mode):
    x, delta, z, B, C = _steps(s, ["x", "delta", "z", "B", "C"])
    (T, N, D), G, S, dtype = x.shape, s["case"]["G"], s["case"]["S"], s["x"].dtype
    grouped = lambda t: t.unflatten(-1, (G, D // G))  # noqa: E731  [T,N,G,D/G]
    inside = _inside(s, T, N, x.device)[..., None, None]
    x, z, raw = grouped(x), grouped(z), grouped(delta + s["delta_bias"])
    A, skip = s["A"].view(G, D // G, S), s["skip"].view(G, D // G)
    dt = torch.where(inside, raw.clamp(min=0) + torch.log1p(torch.exp(-raw.abs())), 0.0)
    x = torch.where(inside, x, 0.0)
    Bs, Cs = (torch.where(inside, t, 0.0)[:, :, :, None] for t in (B, C))  # [T,N,G,1,S]
    a = torch.exp(dt[..., None] * A)
    h0 = torch.zeros(N, G, D // G, S, device=x.device) if s["h"] is None else s["h"].view(N, G, D // G, S)
    b = (dt * x)[..., None] * Bs
    b[0] += a[0] * h0
    h = _recurrence(a, b)
    sums = (h * Cs).sum(-1) + skip * x
    sigmoid = 1 / (1 + torch.exp(-z))
    y = torch.where(inside, sums * z * sigmoid, 0.0).flatten(-2).to(dtype)
    last = h[-1].reshape(N, D, S).clone()
    if mode == "step":
        return {"y": y[0], "h": last}
    out = {"y": y, "h": last}
    if mode == "train":
        dy = torch.where(inside, grouped(s["dy"].float()), 0.0)
        q = dy * z * sigmoid
        a = torch.exp(dt[..., None] * A)
        g = q[..., None] * Cs
        if s["dh"] is not None:
            g[-1] += s["dh"].view(N, G, D // G, S)
        # the same recurrence with time turned round: step t takes what step t+1 decayed
        turned = torch.ones_like(a)
        turned[1:] = a.flip(0)[:-1]
        g = _recurrence(turned, g.flip(0)).flip(0)
        del turned
        out["dC"] = (q[..., None] * h).sum(3).to(dtype)
        out["dB"] = (g * (dt * x)[..., None]).sum(3).to(dtype)
        du = (g * Bs).sum(-1)
        if s["h"] is not None:
            out["dh0"] = (g[0] * a[0]).reshape(N, D, S)
        h = torch.cat([h0[None], h[:-1]])
        decayed = g.mul_(a).mul_(h)  # the gradient of dt A
        ddt = torch.where(inside, x * du + (decayed * A).sum(-1), 0.0)
        draw_ = ddt / (1 + torch.exp(-raw))
        out.update(dx=(dt * du + skip * q).flatten(-2).to(dtype), ddelta=draw_.flatten(-2).to(dtype),
                   dA=(decayed * dt[..., None]).sum((0, 1)).view(D, S), dskip=(q * x).sum((0, 1)).view(D),
                   dz=(dy * sums * sigmoid * (1 + z * (1 - sigmoid))).flatten(-2).to(dtype),
                   dbias=draw_.sum((0, 1)).view(D))
    return out


def _plain_norm(s, mode):
    update, gate, residual = (s[k].float() for k in ("update", "gate", "residual"))
    dtype, centered = s["update"].dtype, s["case"]["centered"]
    scale, after, before = s["scale"], s["after_weight"], s["before_weight"]

    def unit(v):
        v = v - v.mean(-1, keepdim=True) if centered else v
        inv = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5)
        return v * inv, inv

    def unit_gradient(d, n, inv):
        d = d - n * (d * n).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if centered else 0.0)
        return d * inv

    u, u_inv = unit(update)
    sigmoid = 1 / (1 + torch.exp(-gate))
    silu = gate * sigmoid
    gated = u * after * silu
    out = residual + scale * gated
    n, n_inv = unit(out)
    normed = n * before + (s["before_bias"] if centered else 0.0)
    result = {"out": out.to(dtype), "normed": normed.to(dtype)}
    if mode == "train":
        dout, dnormed = s["dout"].float(), s["dnormed"].float()
        d = dout + unit_gradient(dnormed * before, n, n_inv)
        du = d * scale * silu
        result.update(dupdate=unit_gradient(du * after, u, u_inv).to(dtype), dresidual=d.to(dtype),
                      dgate=(d * scale * u * after * sigmoid * (1 + gate * (1 - sigmoid))).to(dtype),
                      dscale=(d * gated).sum((0, 1)), dafter=(du * u).sum((0, 1)), dbefore=(dnormed * n).sum((0, 1)))
        if centered:
            result["dbias"] = dnormed.sum((0, 1))
    return result


# ---- the definitions in float64: step by step, gradients by autograd ----------------------
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    train = case["mode"] == "train"
    given = {"conv": ("x", "kernel", "bias", "state"), "scan": ("x", "delta", "A", "B", "C", "skip", "z", "delta_bias", "h"),
             "norm": ("update", "residual", "gate", "scale", "after_weight", "before_weight", "before_bias")}[case["op"]]
    leaves = {k: s[k].detach().clone().requires_grad_(train) for k in given if s[k] is not None}
    with torch.set_grad_enabled(train):
        outs = {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[case["op"]](case, dict(s, **leaves))
        if train:
            upstream = {"conv": {"y": "dy"}, "scan": {"y": "dy", "h": "dh"}, "norm": {"out": "dout", "normed": "dnormed"}}
            pairs = [(outs[k], s[d]) for k, d in upstream[case["op"]].items() if s[d] is not None]
            grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [d for _, d in pairs])
            names = {"delta_bias": "dbias", "h": "dh0", "after_weight": "dafter", "before_weight": "dbefore", "before_bias": "dbias"}
            outs.update({names.get(k, "d" + k): g for k, g in zip(leaves, grads)})
    return {k: v.detach() for k, v in outs.items()}


def _exact_conv(case, s):
    x = s["x"].unsqueeze(0) if case["mode"] == "step" else s["x"]
    T, N, D = x.shape
    W, lengths = case["W"], [T] * x.shape[1] if s["lengths"] is None else s["lengths"].tolist()
    state = x.new_zeros(W - 1, N, D) if s["state"] is None else s["state"]
    ys, states = [], []
    for n, length in enumerate(lengths):
        seq = torch.cat([state[:, n], x[:length, n]])
        pre = s["bias"] + sum(s["kernel"][k] * seq[k:k + length] for k in range(W))
        ys.append(torch.cat([pre * torch.sigmoid(pre), x.new_zeros(T - length, D)]))
        states.append(seq[length:])
    y = torch.stack(ys, 1)
    return {"y": y[0] if case["mode"] == "step" else y, "state": torch.stack(states, 1)}


def _exact_scan(case, s):
    step = case["mode"] == "step"
    x, delta, z, B, C = (s[k].unsqueeze(0) if step else s[k] for k in ("x", "delta", "z", "B", "C"))
    T, N, D = x.shape
    share = D // case["G"]
    h = x.new_zeros(N, D, case["S"]) if s["h"] is None else s["h"]
    ys = []
    for t in range(T):
        dt = torch.nn.functional.softplus(delta[t] + s["delta_bias"], threshold=50.0)
        new = torch.exp(dt[..., None] * s["A"]) * h + (dt * x[t])[..., None] * B[t].repeat_interleave(share, 1)
        y = ((new * C[t].repeat_interleave(share, 1)).sum(-1) + s["skip"] * x[t]) * z[t] * torch.sigmoid(z[t])
        if s["lengths"] is not None:
            inside = (t < s["lengths"])[:, None]
            new, y = torch.where(inside[..., None], new, h), torch.where(inside, y, 0.0)
        h = new
        ys.append(y)
    return {"y": ys[0] if step else torch.stack(ys), "h": h}


def _exact_norm(case, s):
    def norm(v):
        if case["centered"]:
            return torch.nn.functional.layer_norm(v, v.shape[-1:], eps=1e-5)
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5)

    out = s["residual"] + s["scale"] * norm(s["update"]) * s["after_weight"] * torch.nn.functional.silu(s["gate"])
    normed = norm(out) * s["before_weight"]
    return {"out": out, "normed": normed + s["before_bias"] if case["centered"] else normed}


def work(case):
    T, N, D, S, G, W = (case[k] for k in ("T", "N", "D", "S", "G", "W"))
    size = 4 if case["dtype"] == "float32" else 2
    train, each = case["mode"] == "train", T * N * D
    if case["op"] == "conv":
        states = (W - 1) * N * D * (2 if case["state"] else 1)
        # x in, y out; dy in, dx out (x is at hand)
        return {"bytes": size * ((4 if train else 2) * each + states) + 4 * (W + 1) * D * (2 if train else 1),
                "flops": each * (2 * W + 5) * (3 if train else 1)}
    if case["op"] == "scan":
        states = 4 * N * D * S * (2 if case["state"] else 1)
        shared = 2 * T * N * G * S
        # x, delta, z, B, C in, y out; dy in, dx, ddelta, dz, dB, dC out
        values = 4 * each + shared + ((4 * each + shared) if train else 0)
        flops = each * (S * 7 + 12) + (each * (S * 20 + 30) if train else 0)
        return {"bytes": size * values + states * (2 if train and case["state"] else 1) + 4 * D * (S + 2) * (2 if train else 1),
                "flops": flops}
    # update, residual, gate in, out, normed out; dout, dnormed in, dupdate, dresidual, dgate out
    return {"bytes": size * (10 if train else 5) * each + 4 * 4 * D * (2 if train else 1), "flops": each * (50 if train else 18)}
