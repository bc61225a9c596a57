"""The operators of a gated linear recurrent block and of its training step whose speed is tracked: the matrix
product with bias, activation and residual (the projections around a recurrence), the gated linear recurrence,
and the global gradient norm with clipping.

Sizes are those of bench.py, haste_amd/benchmark_grid.py, perf/operators.py and the tests (batch 1 .. 128, widths
64 .. 4096, 50 .. 4096 steps).  A case is a dict:

  op       "linear", "gated" or "clip"
  mode     linear, gated: "train": forward and backward pass; "infer": forward pass; "step": one token per row
           clip: "norm": the norm alone; "clip": the norm and the scaled gradients
  dtype    of the activations, or of the gradients ("mixed": float32 vectors beside bfloat16 matrices)
  T, N     time steps, batch rows
  C, D     linear: input and output columns; gated: D channels
  activation, bias, residual   linear: what follows the product
  decay    gated: the forget gate is the exponent of a learned decay, and inputs are scaled by sqrt(1 - a^2)
  admit    gated: there is an input gate;  z: gated: the output is gated by silu(z)
  lengths  the batch's sequences have lengths of their own (one of them may be empty)
  state    the sequence goes on from a given state (its gradient is returned)
  batch_first   tensors are slices of projections laid out [N, T, *] instead of [T, N, *]
  layers, width  clip: gradients of that many layers of that width, [width, 4 width] twice and two vectors each

With `own` false run() computes the operators from elementary operations of torch, in float32, and rounds once;
with `own` true it calls haste_amd.ops.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _linear(mode, T, N, C, D, dtype="bfloat16", activation="none", bias=True, residual=False, batch_first=False, **name):
    return dict(name, op="linear", mode=mode, dtype=dtype, T=T, N=N, C=C, D=D, activation=activation, bias=bias,
                residual=residual, batch_first=batch_first)


def _gated(mode, T, N, D, dtype="bfloat16", decay=True, admit=True, z=True, lengths=False, state=False, batch_first=False, **name):
    return dict(name, op="gated", mode=mode, dtype=dtype, T=T, N=N, D=D, decay=decay, admit=admit, z=z, lengths=lengths,
                state=state, batch_first=batch_first)


def _clip(mode, layers, width, dtype="float32", **name):
    return dict(name, op="clip", mode=mode, dtype=dtype, layers=layers, width=width)


def listed():
    return [
        # One stream's next token: the projection into the block, then the recurrence.  Nothing but latency.
        _linear("step", 1, 1, 1024, 4096, activation="silu", name="linear_step_n1"),
        _gated("step", 1, 1, 1024, state=True, name="gated_step_n1"),
        # A full serving batch's next token through the projection out of the block: the weights' bytes.
        _linear("step", 1, 128, 4096, 4096, residual=True, name="linear_step_n128"),
        # An ordinary training step, and a large one.
        _linear("train", 512, 16, 1024, 2048, activation="gelu", name="linear_train"),
        _linear("train", 2048, 8, 4096, 4096, activation="silu", residual=True, name="linear_train_large"),
        # Column blocks of a projection stored batch first, in float, at sizes that no tile divides.
        _linear("train", 83, 37, 300, 1001, dtype="float32", activation="gelu", batch_first=True, name="linear_train_ragged"),
        # One long prompt by itself: few channels, so the steps have to be shared out.
        _gated("infer", 4096, 1, 2048, name="gated_prompt_n1"),
        # An ordinary training step without the learned decay, and a large one.
        _gated("train", 1024, 8, 1024, decay=False, admit=False, z=False, name="gated_train"),
        _gated("train", 2048, 8, 4096, name="gated_train_large"),
        # Padded sequences that go on from a state, at sizes that no tile divides.
        _gated("train", 500, 37, 300, dtype="float32", lengths=True, state=True, name="gated_train_ragged"),
        # The gradients of a layer of bench.py's width in float, and of a stack with float32 vectors beside bfloat16 matrices.
        _clip("clip", 1, 512, name="clip_small"),
        _clip("clip", 16, 2048, dtype="mixed", name="clip_large"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "gated", "clip"])
    if op == "clip":
        while True:
            layers, width = _spread(rng, 1, 32), _spread(rng, 32, 4096)
            dtype = rng.choice(["float32", "mixed", "bfloat16", "float16"])
            if layers * width ** 2 * (2 if dtype == "float32" else 1) <= 16 * 2048 ** 2:
                return _clip(rng.choice(["clip", "clip", "norm"]), layers, width, dtype=dtype)
    mode = rng.choice(["train", "train", "infer", "step"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    most = 2048 * 8 * 4096 // (2 if dtype == "float32" else 1)  # elements of a tensor
    while True:
        N, D = _spread(rng, 1, 128), _spread(rng, 64, 4096)
        C = _spread(rng, 64, 4096)
        T = 1 if mode == "step" else _spread(rng, 1, 4096)
        if rng.random() < 0.5:  # widths that a configuration file would have
            C, D = max(64, C // 64 * 64), max(64, D // 64 * 64)
        if T * N * (max(C, D) if op == "linear" else D) <= most:
            break
    batch_first = mode != "step" and rng.random() < 0.25
    if op == "linear":
        return _linear(mode, T, N, C, D, dtype=dtype, activation=rng.choice(["none", "gelu", "silu"]),
                       bias=rng.random() < 0.75, residual=rng.random() < 0.5, batch_first=batch_first)
    return _gated(mode, T, N, D, dtype=dtype, decay=rng.random() < 0.5, admit=rng.random() < 0.5, z=rng.random() < 0.5,
                  lengths=mode != "step" and rng.random() < 0.25, state=mode == "step" or rng.random() < 0.25,
                  batch_first=batch_first)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (scale * torch.randn(*shape, generator=gen, device=dev)).to(dtype)

    def uniform(low, high, *shape):
        return low + (high - low) * torch.rand(*shape, generator=gen, device=dev)

    s = {"case": case}
    if case["op"] == "clip":
        width = case["width"]
        matrices = torch.bfloat16 if case["dtype"] == "mixed" else _DTYPES[case["dtype"]]
        vectors = torch.float32 if case["dtype"] == "mixed" else matrices
        s["grads"] = []
        for layer in range(case["layers"]):  # gradients differ in size from layer to layer
            scale = 10.0 ** -(1 + layer % 3)
            s["grads"] += [normal(width, 4 * width, dtype=matrices, scale=scale), normal(width, 4 * width, dtype=matrices, scale=scale),
                           normal(4 * width, dtype=vectors, scale=scale), normal(4 * width, dtype=vectors, scale=scale)]
        s["max_norm"] = 1.0
        # What the optimizer reads: one buffer for each type, of which every tensor has a part.
        s["buffers"] = [torch.empty(sum(g.numel() for g in s["grads"] if g.dtype == t), dtype=t, device=dev)
                        for t in dict.fromkeys((matrices, vectors))]
        rest, s["out"] = {b.dtype: b for b in s["buffers"]}, []
        for g in s["grads"]:
            s["out"].append(rest[g.dtype][:g.numel()].view(g.shape))
            rest[g.dtype] = rest[g.dtype][g.numel():]
        return s

    dtype, T, N, D = _DTYPES[case["dtype"]], case["T"], case["N"], case["D"]

    def projection(*widths):
        """What a projection to sum(widths) columns left: its column blocks as [T,N,width] ([N,width])."""
        if case["mode"] == "step":
            full = normal(N, sum(widths), dtype=dtype)
        elif case["batch_first"]:
            full = normal(N, T, sum(widths), dtype=dtype).transpose(0, 1)
        else:
            full = normal(T, N, sum(widths), dtype=dtype)
        return full.split(widths, dim=-1)

    if case["op"] == "linear":
        C = case["C"]
        s["x"] = projection(C, C)[1] if case["batch_first"] else projection(C)[0]
        s["kernel"] = normal(C, D, dtype=dtype, scale=C ** -0.5)
        s["bias"] = normal(D, dtype=dtype, scale=0.1) if case["bias"] else None
        s["residual"] = projection(D)[0] if case["residual"] else None
        if case["mode"] == "train":
            s["dy"] = normal(T, N, D, dtype=dtype)
        return s

    if case["lengths"]:
        s["lengths"] = torch.randint(max(1, T // 2), T + 1, (N,), generator=gen, device=dev)
        s["lengths"][-1:] = T
        if N > 2:
            s["lengths"][1] = 0
    else:
        s["lengths"] = None
    s["x"], z = projection(D, D)
    s["z"] = z if case["z"] else None
    s["forget"], admit = projection(D, D)
    s["admit"] = admit if case["admit"] else None
    s["admit_bias"] = 0.1 * normal(D) if case["admit"] else None
    if case["decay"]:  # per step 0.9 .. 0.999 squared, under an open gate
        s["decay"], s["forget_bias"] = -2 * torch.log(uniform(0.9, 0.999, D)), 0.1 * normal(D)
    else:  # gates that start out remembering for a few steps up to hundreds
        s["decay"], s["forget_bias"] = None, uniform(0.5, 6.0, D)
    s["h"] = 0.3 * normal(N, D) if case["state"] else None
    if case["mode"] == "train":
        s["dy"] = normal(T, N, D, dtype=dtype)
        s["dh"] = normal(N, D) if case["state"] else None
    return s


def run(s):
    op, mode = s["case"]["op"], s["case"]["mode"]
    if own:
        return {"linear": _own_linear, "gated": _own_gated, "clip": _own_clip}[op](s, mode)
    return {"linear": _plain_linear, "gated": _plain_gated, "clip": _plain_clip}[op](s, mode)


# ---- the framework's calls ----------------------------------------------------------------
def _own_linear(s, mode):
    from haste_amd import ops
    activation = s["case"]["activation"]
    y, cache = ops.linear_forward(mode == "train", s["x"], s["kernel"], s["bias"], activation, s["residual"])
    if mode != "train":
        return {"y": y}
    dx, dkernel, dbias = ops.linear_backward(s["x"], s["kernel"], s["bias"], activation, cache, s["dy"])
    return {"y": y, "dx": dx, "dkernel": dkernel, **({} if dbias is None else {"dbias": dbias})}


def _own_gated(s, mode):
    from haste_amd import ops
    parts = s["admit"], s["z"], s["decay"], s["forget_bias"], s["admit_bias"]
    if mode == "step":
        y, h = ops.gated_recurrence_iterate(s["x"], s["forget"], s["h"], *parts)
        return {"y": y, "h": h}
    y, h, cache = ops.gated_recurrence_forward(mode == "train", s["x"], s["forget"], *parts, s["h"], s["lengths"])
    out = {"y": y, "h": h}
    if mode == "train":
        names = ("dx", "dforget", "dadmit", "dz", "ddecay", "dforget_bias", "dadmit_bias", "dh0")
        grads = ops.gated_recurrence_backward(s["x"], s["forget"], *parts, s["h"], s["lengths"], cache, s["dy"], s["dh"])
        out.update({k: g for k, g in zip(names, grads) if g is not None})
    return out


def _own_clip(s, mode):
    from haste_amd import ops
    if mode == "norm":
        return {"norm": ops.gradient_norm(s["grads"])}
    _, norm = ops.clip_gradients(s["grads"], s["max_norm"], out=s["out"])
    return {"norm": norm, "clipped": s["buffers"]}


# ---- the plain forms: elementary operations in float32, rounded once at the end -----------
def _activated(kind, pre):
    """act(pre) and its slope."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-pre))
        return pre * s, s * (1 + pre * (1 - s))
    if kind == "gelu":
        below = 0.5 * (1 + torch.erf(pre * 0.5 ** 0.5))
        return pre * below, below + pre * torch.exp(-0.5 * pre * pre) * (2 * math.pi) ** -0.5
    return pre, None


def _plain_linear(s, mode):
    dtype, shape = s["x"].dtype, s["x"].shape
    x, kernel = s["x"].float().flatten(0, -2), s["kernel"].float()
    pre = x @ kernel
    if s["bias"] is not None:
        pre = pre + s["bias"].float()
    y, slope = _activated(s["case"]["activation"], pre)
    y = y.unflatten(0, shape[:-1])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if mode == "train":
        d = s["dy"].float().flatten(0, -2)
        if slope is not None:
            d = d * slope
        out["dx"] = (d @ kernel.t()).unflatten(0, shape[:-1]).to(dtype)
        out["dkernel"] = (x.t() @ d).to(dtype)
        if s["bias"] is not None:
            out["dbias"] = d.sum(0).to(dtype)
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


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _plain_gated(s, mode):
    wide = lambda k: None if s[k] is None else s[k].float().unsqueeze(0) if mode == "step" else s[k].float()  # noqa: E731
    x, forget, admit, z = wide("x"), wide("forget"), wide("admit"), wide("z")
    (T, N, D), dtype, decay = x.shape, s["x"].dtype, s["decay"]
    inside = torch.ones(T, N, 1, dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        inside = (torch.arange(T, device=x.device)[:, None] < s["lengths"])[..., None]
    x = torch.where(inside, x, 0.0)
    raw = forget + s["forget_bias"]
    r, keep = _sigmoid(raw), _sigmoid(-raw)  # keep = 1 - r
    i = None if admit is None else _sigmoid(admit + s["admit_bias"])
    if decay is None:
        a, m = r, keep if i is None else None
    else:
        a, m = torch.exp(-decay * r), torch.sqrt(-torch.expm1(-2 * decay * r))
    scale = i if m is None else m if i is None else m * i
    u = torch.where(inside, scale * x, 0.0)
    a = torch.where(inside, a, 1.0)
    h0 = torch.zeros(N, D, device=x.device) if s["h"] is None else s["h"]
    b = u.clone()
    b[0] += a[0] * h0
    h = _recurrence(a.clone(), b)
    silu = None if z is None else z * _sigmoid(z)
    y = torch.where(inside, h if z is None else h * silu, 0.0).to(dtype)
    if mode == "step":
        return {"y": y[0], "h": h[-1].clone()}
    out = {"y": y, "h": h[-1].clone()}
    if mode == "train":
        dy = torch.where(inside, s["dy"].float(), 0.0)
        g = dy.clone() if z is None else dy * silu
        if s["dh"] is not None:
            g[-1] += s["dh"]
        # the same recurrence with time turned round: step t takes what step t+1 decayed
        turned = torch.ones_like(a)
        turned[1:] = a.flip(0)[:-1]
        g = _recurrence(turned, g.flip(0)).flip(0)
        before = torch.cat([h0[None], h[:-1]])
        out["dx"] = torch.where(inside, g * scale, 0.0).to(dtype)
        if decay is None:
            dr = g * before if i is not None else g * (before - x)
        else:
            fed = x if i is None else x * i
            dlog = g * (before * a - fed * a * a / m)  # the gradient of log a
            dr = -decay * dlog
            out["ddecay"] = torch.where(inside, -r * dlog, 0.0).sum((0, 1))
        dforget = torch.where(inside, dr * r * keep, 0.0)
        out.update(dforget=dforget.to(dtype), dforget_bias=dforget.sum((0, 1)))
        if i is not None:
            dadmit = torch.where(inside, g * (x if m is None else m * x) * i * (1 - i), 0.0)
            out.update(dadmit=dadmit.to(dtype), dadmit_bias=dadmit.sum((0, 1)))
        if z is not None:
            sigmoid = _sigmoid(z)
            out["dz"] = torch.where(inside, dy * h * sigmoid * (1 + z * (1 - sigmoid)), 0.0).to(dtype)
        if s["h"] is not None:
            out["dh0"] = a[0] * g[0]
    return out


def _plain_clip(s, mode):
    total = sum(g.float().square().sum() for g in s["grads"])
    norm = torch.sqrt(total)
    if mode == "norm":
        return {"norm": norm}
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for g, out in zip(s["grads"], s["out"]):
        out.copy_(g.float() * factor)
    return {"norm": norm, "clipped": s["buffers"]}


# ---- the definitions in float64: step by step, gradients by autograd ----------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]))
        result = {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda")}
        if case["mode"] == "clip":
            factor = min(1.0, s["max_norm"] / (norm + 1e-6))
            result["clipped"] = [torch.cat([g.double().flatten() * factor for g in s["grads"] if g.dtype == b.dtype])
                                 for b in s["buffers"]]
        return result
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    train = case["mode"] == "train"
    given = {"linear": ("x", "kernel", "bias"),
             "gated": ("x", "forget", "admit", "z", "decay", "forget_bias", "admit_bias", "h")}[case["op"]]
    leaves = {k: s[k].detach().clone().requires_grad_(train) for k in given if s[k] is not None}
    with torch.set_grad_enabled(train):
        outs = {"linear": _exact_linear, "gated": _exact_gated}[case["op"]](case, dict(s, **leaves))
        if train:
            upstream = {"linear": {"y": "dy"}, "gated": {"y": "dy", "h": "dh"}}[case["op"]]
            pairs = [(outs[k], s[d]) for k, d in upstream.items() if s[d] is not None]
            grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [d for _, d in pairs])
            outs.update({"dh0" if k == "h" else "d" + k: g for k, g in zip(leaves, grads)})
    return {k: v.detach() for k, v in outs.items()}


def _exact_linear(case, s):
    pre = torch.matmul(s["x"].flatten(0, -2), s["kernel"]).unflatten(0, s["x"].shape[:-1])
    if s["bias"] is not None:
        pre = pre + s["bias"]
    act = {"none": lambda v: v, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}
    y = act[case["activation"]](pre)
    return {"y": y if s["residual"] is None else y + s["residual"]}


def _exact_gated(case, s):
    step = case["mode"] == "step"
    x, forget, admit, z = (None if s[k] is None else s[k].unsqueeze(0) if step else s[k] for k in ("x", "forget", "admit", "z"))
    T, N, D = x.shape
    h = x.new_zeros(N, D) if s["h"] is None else s["h"]
    ys = []
    for t in range(T):
        r = torch.sigmoid(forget[t] + s["forget_bias"])
        fed = x[t] if admit is None else x[t] * torch.sigmoid(admit[t] + s["admit_bias"])
        if s["decay"] is not None:
            new = torch.exp(-s["decay"] * r) * h + torch.sqrt(-torch.expm1(-2 * s["decay"] * r)) * fed
        elif admit is not None:
            new = r * h + fed
        else:
            new = r * h + (1 - r) * fed
        y = new if z is None else new * torch.nn.functional.silu(z[t])
        if s["lengths"] is not None:
            inside = (t < s["lengths"])[:, None]
            new, y = torch.where(inside, new, h), torch.where(inside, y, 0.0)
        h = new
        ys.append(y)
    return {"y": ys[0] if step else torch.stack(ys), "h": h}


def work(case):
    if case["op"] == "clip":
        width, layers = case["width"], case["layers"]
        matrix, vector = {"float32": (4, 4), "mixed": (2, 4)}.get(case["dtype"], (2, 2))
        each = 8 * width * width * layers, 8 * width * layers
        passes = 2 if case["mode"] == "clip" else 1
        return {"bytes": passes * (each[0] * matrix + each[1] * vector), "flops": (1 + passes) * sum(each)}
    T, N, D = (case[k] for k in ("T", "N", "D"))
    size = 4 if case["dtype"] == "float32" else 2
    train, each = case["mode"] == "train", T * N * D
    if case["op"] == "linear":
        C, R = case["C"], T * N
        # x, kernel, bias, residual in, y out; dy in, dx, dkernel, dbias out
        values = R * C + C * D + D * case["bias"] + each * (2 if case["residual"] else 1)
        values += (each + R * C + C * D + D * case["bias"]) if train else 0
        return {"bytes": size * values, "flops": 2 * R * C * D * (3 if train else 1)}
    inputs = 2 + case["admit"] + case["z"]
    states = 4 * N * D * (1 + case["state"]) * (2 if train and case["state"] else 1)
    # the inputs in, y out; dy in, the inputs' gradients out
    values = inputs + 1 + ((1 + inputs) if train else 0)
    weights = 4 * D * (1 + case["decay"] + case["admit"]) * (2 if train else 1)
    return {"bytes": size * values * each + states + weights, "flops": each * (70 if train else 25)}
