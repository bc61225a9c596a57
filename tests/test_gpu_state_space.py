"""The state space block's operators on the GPU against the formulas in float64 (state_space_formulas.py, whose gradients are
checked by differences and against autograd in test_state_space_cpu.py), bounded as derived there."""
import pytest
import torch

import haste_amd
from haste_amd import ops

import state_space_formulas as formulas

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
short = lambda t: str(t).split(".")[1]  # noqa: E731


class Problem:
    """Values representable in `dtype` (activations) or float32 (the rest), as float64 on the CPU (.p) and on the GPU (.g)."""

    def __init__(self, seed, dtype):
        self.gen, self.dtype, self.p, self.g = torch.Generator().manual_seed(seed), dtype, {}, {}

    def put(self, name, value, dtype=None):
        value = value.to(dtype or self.dtype)
        self.p[name], self.g[name] = value.double(), value.cuda()

    def normal(self, name, *shape, dtype=None, scale=1.0, shift=0.0):
        self.put(name, shift + scale * torch.randn(*shape, generator=self.gen, dtype=torch.float64), dtype)

    def absent(self, *names):
        for n in names:
            self.p[n] = self.g[n] = None

    def lengths(self, lengths):
        self.p["lengths"] = lengths
        self.g["lengths"] = None if lengths is None else torch.tensor(lengths, device="cuda")

    def poison(self, *names):
        """NaN in the activations behind the rows' lengths."""
        if self.p["lengths"] is None:
            return
        T, N = self.g[names[0]].shape[:2]
        mask, _ = formulas.inside(self.p["lengths"], T, N)
        for n in names:
            if self.g[n] is not None:
                self.g[n][~mask.cuda()] = float("nan")


def compare(got, want, magnitudes, roundings):
    for k, v in got.items():
        if v is not None:
            formulas.check(v, want[k], magnitudes[k], roundings, k)


# ---- the convolution -------------------------------------------------------------------
def conv_problem(seed, dtype, T, N, D, W, bias=True, state=True, lengths=None, silu=True):
    q = Problem(seed, dtype)
    q.normal("x", T, N, D)
    q.normal("kernel", W, D, dtype=torch.float32, scale=W ** -0.5)
    q.normal("dy", T, N, D)
    q.normal("dstate_out", W - 1, N, D)
    q.normal("bias", D, dtype=torch.float32) if bias else q.absent("bias")
    q.normal("state", W - 1, N, D) if state else q.absent("state")
    q.lengths(lengths)
    q.p["silu"] = q.g["silu"] = silu
    return q


def run_conv(g):
    y, state = ops.causal_conv_forward(g["x"], g["kernel"], g["bias"], g["silu"], g["state"], g["lengths"])
    dx, dkernel, dbias, dstate = ops.causal_conv_backward(g["x"], g["kernel"], g["bias"], g["silu"], g["state"], g["lengths"],
                                                          g["dy"], g["dstate_out"])
    return dict(y=y, state=state, dx=dx, dkernel=dkernel, dbias=dbias, dstate=dstate)


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
@pytest.mark.parametrize("T,N,D,W,options", [
    (1, 1, 1, 4, {}), (1, 3, 75, 4, {}), (2, 2, 9, 8, {}), (3, 1, 64, 2, dict(silu=False)), (5, 2, 33, 1, {}),
    (7, 4, 16, 3, dict(bias=False)), (9, 3, 8, 5, dict(state=False)), (63, 2, 40, 6, {}), (64, 2, 40, 7, {}), (65, 2, 41, 8, {}),
    (130, 5, 300, 4, dict(bias=False, state=False)), (257, 3, 24, 4, {}), (20, 6, 100, 4, dict(lengths=[20, 0, 1, 2, 19, -1])),
    (70, 4, 13, 8, dict(lengths=[3, 70, 64, -2])), (6, 3, 1024, 4, dict(lengths=[0, 0, 0])), (1, 70, 2000, 4, {})])
def test_conv(T, N, D, W, options, dtype):
    print("conv", T, N, D, W, options, dtype, flush=True)
    q = conv_problem(T + D, dtype, T, N, D, W, **options)
    q.poison("x", "dy")
    compare(run_conv(q.g), formulas.conv(q.p), formulas.conv(q.p, True), 8 * W + T * N + 64)


def test_conv_gradients_may_be_left_out():
    q = conv_problem(1, torch.float32, 9, 2, 20, 4)
    q.absent("dstate_out")
    full = formulas.conv(q.p)
    dx, dkernel, dbias, dstate = ops.causal_conv_backward(q.g["x"], q.g["kernel"], q.g["bias"], True, q.g["state"], None, q.g["dy"])
    compare(dict(dx=dx, dstate=dstate), full, formulas.conv(q.p, True), 128)
    q.normal("dstate_out", 3, 2, 20)
    q.p["dy"] = q.p["dy"] * 0
    got = ops.causal_conv_backward(q.g["x"], q.g["kernel"], q.g["bias"], True, q.g["state"], None, None, q.g["dstate_out"])
    compare(dict(zip(("dx", "dkernel", "dbias", "dstate"), got)), formulas.conv(q.p), formulas.conv(q.p, True), 128)


# ---- the scan --------------------------------------------------------------------------
def scan_problem(seed, dtype, T, N, D, S, G=1, softplus=True, D_=True, z=True, bias=True, h0=True, dh=True, lengths=None):
    q = Problem(seed, dtype)
    for name in ("x", "dy"):
        q.normal(name, T, N, D)
    if softplus:
        q.normal("delta", T, N, D, scale=2.0, shift=-2.0)
    else:
        q.put("delta", 0.2 * torch.rand(T, N, D, generator=q.gen, dtype=torch.float64))
    q.put("A", -4 * torch.rand(D, S, generator=q.gen, dtype=torch.float64), torch.float32)
    for name in ("B", "C"):
        q.normal(name, T, N, G, S)
    q.normal("D", D, dtype=torch.float32) if D_ else q.absent("D")
    q.normal("z", T, N, D) if z else q.absent("z")
    q.normal("delta_bias", D, dtype=torch.float32, scale=0.5) if bias and softplus else q.absent("delta_bias")
    q.normal("h0", N, D, S, dtype=torch.float32) if h0 else q.absent("h0")
    q.normal("dh_last", N, D, S, dtype=torch.float32) if dh else q.absent("dh_last")
    q.lengths(lengths)
    q.p["softplus"] = q.g["softplus"] = softplus
    return q


NAMES = ("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dh0")


def run_scan(g):
    y, h, cache = ops.selective_scan_forward(True, g["x"], g["delta"], g["A"], g["B"], g["C"], g["D"], g["z"], g["delta_bias"],
                                             g["softplus"], g["h0"], g["lengths"])
    grads = ops.selective_scan_backward(g["x"], g["delta"], g["A"], g["B"], g["C"], g["D"], g["z"], g["delta_bias"], g["softplus"],
                                        g["h0"], g["lengths"], cache, g["dy"], g["dh_last"])
    return dict(zip(NAMES, grads), y=y, h_last=h)


SCAN_CASES = [
    (1, 1, 1, 1, {}), (1, 3, 20, 16, {}), (2, 2, 65, 4, {}), (15, 2, 64, 16, {}), (16, 2, 64, 16, {}), (17, 3, 63, 8, dict(softplus=False)),
    (33, 1, 200, 16, dict(z=False)), (40, 2, 30, 11, dict(D_=False, bias=False)), (40, 2, 48, 32, dict(h0=False)),
    (50, 2, 36, 64, dict(dh=False)), (31, 2, 40, 5, dict(G=4)), (35, 2, 390, 16, dict(G=3)), (20, 2, 70, 33, dict(G=2)),
    # long enough for the time axis to be cut
    (64, 1, 64, 16, {}), (129, 1, 64, 16, {}), (300, 2, 48, 16, dict(G=2)), (520, 1, 20, 7, {}), (400, 1, 33, 64, {}),
    (1300, 1, 9, 5, {}), (1300, 2, 20, 16, dict(lengths=[1300, 777])), (1100, 2, 8, 40, dict(lengths=[64, -1], h0=False, dh=False)),
    (20, 6, 30, 16, dict(lengths=[20, 0, 1, 16, 17, -2])), (300, 4, 40, 16, dict(lengths=[300, 0, 70, 128])),
    (200, 3, 17, 12, dict(lengths=[-1, 65, 64], h0=False)), (6, 2, 300, 16, dict(lengths=[0, 0])), (2, 90, 130, 16, {})]


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
@pytest.mark.parametrize("T,N,D,S,options", SCAN_CASES)
def test_scan(T, N, D, S, options, dtype):
    print("scan", T, N, D, S, options, dtype, flush=True)
    q = scan_problem(T + D + S, dtype, T, N, D, S, **options)
    q.poison("x", "delta", "z", "B", "C", "dy")
    # a state's step: exponent, exp2, two products, a sum, forward and backward; then the sums over states, channels, steps and rows
    compare(run_scan(q.g), formulas.scan(q.p), formulas.scan(q.p, True), 12 * T + S + D + T * N + 128)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=short)
@pytest.mark.parametrize("S", [6, 16, 24, 50])
def test_scan_of_any_number_of_channels(S, dtype):
    """Groups that end anywhere within a vector, a workgroup and the last of several workgroups; chunks of the time axis too."""
    for T in (19, 140):
        for G, share in ((3, 1), (2, 2), (2, 3), (1, 5), (2, 7), (1, 31), (2, 33), (1, 66), (1, 129), (2, 131), (1, 258)):
            print("scan channels", T, G, share, S, dtype, flush=True)
            q = scan_problem(T + share + S, dtype, T, 1, G * share, S, G)
            compare(run_scan(q.g), formulas.scan(q.p), formulas.scan(q.p, True), 12 * T + S + share + T + 128)


def test_scan_of_small_step_sizes():
    """softplus far below zero is exp, to the same relative error: y and h scale with it."""
    for shift in (-5.0, -12.0, -20.0, -60.0):
        q = scan_problem(5, torch.float32, 20, 2, 40, 16, D_=False, h0=False, dh=False, bias=False)
        q.put("delta", q.p["delta"] * 0.1 + shift)
        compare(run_scan(q.g), formulas.scan(q.p), formulas.scan(q.p, True), 12 * 20 + 16 + 40 + 40 + 128)


def test_scan_of_extreme_values():
    """Steps that forget everything, steps that change nothing, decays of zero and slow growth."""
    q = scan_problem(6, torch.float32, 150, 2, 40, 16, bias=False)
    delta = q.p["delta"].clone()
    delta[::3] = 60.0
    delta[1::5] = -200.0
    q.put("delta", delta)
    A = q.p["A"].clone()
    A[:, 0] = 0.0
    A[:, 1] = 1e-4
    A[::2] *= 100.0
    q.put("A", A, torch.float32)
    q.normal("x", 150, 2, 40, scale=0.01)
    compare(run_scan(q.g), formulas.scan(q.p), formulas.scan(q.p, True), 12 * 150 + 16 + 40 + 300 + 128)


def test_scan_without_upstream_gradients():
    q = scan_problem(8, torch.bfloat16, 100, 2, 50, 16)
    g = q.g
    _, _, cache = ops.selective_scan_forward(True, g["x"], g["delta"], g["A"], g["B"], g["C"], g["D"], g["z"], g["delta_bias"], True, g["h0"])
    got = ops.selective_scan_backward(g["x"], g["delta"], g["A"], g["B"], g["C"], g["D"], g["z"], g["delta_bias"], True, g["h0"], None,
                                      cache, None, g["dh_last"])
    q.p["dy"] = q.p["dy"] * 0
    compare(dict(zip(NAMES, got)), formulas.scan(q.p), formulas.scan(q.p, True), 2000)


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
@pytest.mark.parametrize("N,D,S,G,options", [(1, 1, 1, 1, {}), (3, 50, 16, 1, {}), (2, 64, 11, 4, dict(z=False)), (5, 30, 64, 2, dict(D_=False)),
                                             (1, 1024, 8, 1, dict(softplus=False)), (70, 90, 32, 3, dict(bias=False))])
def test_scan_step(N, D, S, G, options, dtype):
    print("scan step", N, D, S, G, options, dtype, flush=True)
    q = scan_problem(N + D + S, dtype, 1, N, D, S, G, **options)
    g = {k: v[0] if torch.is_tensor(v) and k in ("x", "delta", "B", "C", "z") else v for k, v in q.g.items()}
    y, h = ops.selective_scan_iterate(g["x"], g["delta"], g["A"], g["B"], g["C"], g["h0"], g["D"], g["z"], g["delta_bias"], g["softplus"])
    want, magnitude = formulas.scan(q.p), formulas.scan(q.p, True)
    compare(dict(y=y[None], h_last=h), want, magnitude, S + 64)
    before = g["h0"].clone()
    y2, h2 = ops.selective_scan_iterate(g["x"], g["delta"], g["A"], g["B"], g["C"], before, g["D"], g["z"], g["delta_bias"],
                                        g["softplus"], h_out=before)
    assert h2 is before and torch.equal(h2, h) and torch.equal(y2, y)


# ---- the norms ---------------------------------------------------------------------------
def norm_problem(seed, dtype, shape, centered, absent=(), shift=0.0):
    q, D = Problem(seed, dtype), shape[-1]
    for name in ("update", "residual", "gate"):
        q.absent(name) if name in absent else q.normal(name, *shape, shift=shift if name == "update" else 0.0)
    for name in ("scale", "after_weight", "before_weight", "before_bias"):
        skip = name in absent or name == "before_bias" and "before_weight" in absent
        q.absent(name) if skip else q.normal(name, D, dtype=torch.float32)
    for name in ("dout", "dnormed"):
        q.absent(name) if name in absent or name == "dnormed" and "before_weight" in absent else q.normal(name, *shape)
    q.p.update(centered=centered, eps=1e-5)
    return q


PARTS = ("update", "residual", "gate", "scale", "after_weight", "before_weight", "before_bias")


def run_norm(g, centered):
    out, normed, stats = ops.residual_norm_forward(*(g[k] for k in PARTS), centered=centered)
    grads = ops.residual_norm_backward(*(g[k] for k in PARTS), stats, g["dout"], g["dnormed"], centered=centered)
    names = ("dupdate", "dresidual", "dgate", "dscale", "dafter", "dbefore", "dbias")
    return dict(zip(names, grads), out=out, normed=normed)


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
@pytest.mark.parametrize("centered", [False, True])
@pytest.mark.parametrize("shape,options", [
    ((1, 1, 1), {}), ((1, 1, 3), {}), ((3, 5, 64), {}), ((7, 3, 511), {}), ((4, 3, 512), {}), ((4, 3, 513), {}), ((5, 2, 1001), {}),
    ((3, 2, 1030), {}), ((2, 2, 2048), {}), ((3, 1, 3000), {}), ((2, 2, 4097), {}), ((3, 1, 8192), {}), ((300, 11, 40), {}),
    ((9, 70), {}), ((6, 2, 100), dict(absent=("residual",))), ((6, 2, 100), dict(absent=("gate",))),
    ((6, 2, 100), dict(absent=("scale", "before_bias"))), ((6, 2, 100), dict(absent=("after_weight",))),
    ((6, 2, 100), dict(absent=("before_weight",))), ((6, 2, 100), dict(absent=("dout",))), ((6, 2, 100), dict(absent=("dnormed",))),
    ((6, 2, 100), dict(absent=("residual", "gate", "scale", "after_weight"))), ((6, 2, 700), dict(shift=20.0))])
def test_norm(shape, options, centered, dtype):
    print("norm", shape, options, centered, dtype, flush=True)
    q = norm_problem(shape[-1], dtype, shape, centered, **options)
    rows = q.p["update"].numel() // shape[-1]
    # every factor (two norms of D terms each, forward and backward) within D + 32 roundings, the sums over rows
    compare(run_norm(q.g, centered), formulas.norm(q.p), formulas.norm(q.p, True), 8 * (shape[-1] + 32) + rows)


# ---- any strides ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=short)
def test_rows_that_end_anywhere(dtype):
    """The last vector of a row, whole or in part; the convolution's in place too."""
    for D in list(range(1, 18)) + list(range(512, 522)):
        print("ends", D, dtype, flush=True)
        norm, conv = norm_problem(D, dtype, (3, 2, D), D % 2 == 1), conv_problem(D, dtype, 7, 2, D, 4, lengths=[7, 3])
        compare(run_norm(norm.g, D % 2 == 1), formulas.norm(norm.p), formulas.norm(norm.p, True), 8 * (D + 32) + 6)
        compare(run_conv(conv.g), formulas.conv(conv.p), formulas.conv(conv.p, True), 8 * 4 + 14 + 64)
        x, state = conv.g["x"][0], conv.g["state"].clone()
        want = ops.causal_conv_iterate(x, conv.g["state"], conv.g["kernel"], conv.g["bias"], True)
        y, _ = ops.causal_conv_iterate(x, state, conv.g["kernel"], conv.g["bias"], True, state_out=state)
        assert torch.equal(y, want[0]) and torch.equal(state, want[1])


def relaid(t, how):
    """The values of t in other memory: batch first, as a column block at an odd offset, or with channels apart."""
    if t is None or t.dim() < 3:
        return t
    if how == "batch_first":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "column_block":
        flat = t.flatten(2)
        wide = torch.full((*t.shape[:2], flat.shape[2] + 7), float("nan"), device=t.device, dtype=t.dtype)
        wide[..., 3:3 + flat.shape[2]] = flat
        return wide[..., 3:3 + flat.shape[2]].unflatten(2, t.shape[2:])
    return torch.stack([t, t], -1)[..., 0]


@pytest.mark.parametrize("how", ["batch_first", "column_block", "apart"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=short)
def test_strides(dtype, how):
    conv, scan = conv_problem(1, dtype, 21, 3, 52, 4, lengths=[21, 5, 0]), scan_problem(2, dtype, 90, 3, 52, 12, 2, lengths=[90, 5, 0])
    norm = norm_problem(3, dtype, (7, 3, 52), True)
    for run, q in ((run_conv, conv), (run_scan, scan), (lambda g: run_norm(g, True), norm)):
        want = run(q.g)
        got = run({k: relaid(v, how) if torch.is_tensor(v) and v.dtype == dtype and k not in ("h0", "dh_last") else v for k, v in q.g.items()})
        for k in want:
            assert want[k] is None or torch.equal(want[k], got[k]), (how, k)


def test_expanded_inputs():
    """One row's (or step's) values for all of them, without a copy."""
    q = scan_problem(4, torch.bfloat16, 40, 3, 30, 16)
    g = dict(q.g)
    g["z"], g["B"] = g["z"][:, :1].expand(-1, 3, -1), g["B"][:1].expand(40, -1, -1, -1)
    want = run_scan({k: v.contiguous() if torch.is_tensor(v) else v for k, v in g.items()})
    got = run_scan(g)
    assert all(torch.equal(want[k], got[k]) for k in want)


def test_strides_beyond_32_bits():
    far = torch.empty(2 ** 31 + 4096, device="cuda", dtype=torch.bfloat16)
    q = conv_problem(9, torch.bfloat16, 2, 2, 64, 4)
    x = far.as_strided((2, 2, 64), (2 ** 31 + 64, 128, 1))
    x.copy_(q.g["x"])
    want, got = run_conv(q.g), run_conv(dict(q.g, x=x))
    assert all(torch.equal(want[k], got[k]) for k in want)
    s = scan_problem(9, torch.bfloat16, 2, 2, 64, 16)
    want, got = run_scan(s.g), None
    x.copy_(s.g["x"])
    got = run_scan(dict(s.g, x=x))
    assert all(torch.equal(want[k], got[k]) for k in want)
    n = norm_problem(9, torch.bfloat16, (2, 2, 64), False)
    want = run_norm(n.g, False)
    x.copy_(n.g["update"])
    got = run_norm(dict(n.g, update=x), False)
    assert all(want[k] is None or torch.equal(want[k], got[k]) for k in want)


# ---- lengths that name no step --------------------------------------------------------------
def test_lengths_out_of_range_give_nans_for_their_rows():
    for T in (20, 200):
        c, s = conv_problem(1, torch.float32, T, 3, 24, 4, lengths=[T, T, T]), scan_problem(2, torch.float32, T, 3, 24, 16, lengths=[T, T, T])
        bad = torch.tensor([T, T + 1, -T - 2], device="cuda")
        for run, q, per_row in ((run_conv, c, {"y": 1, "state": 1, "dx": 1, "dstate": 1}),
                                (run_scan, s, {"y": 1, "h_last": 0, "dx": 1, "ddelta": 1, "dz": 1, "dB": 1, "dC": 1, "dh0": 0})):
            good, got = run(q.g), run(dict(q.g, lengths=bad))
            for k, axis in per_row.items():
                assert got[k].select(axis, 1).isnan().all() and got[k].select(axis, 2).isnan().all(), k
                assert torch.equal(got[k].select(axis, 0), good[k].select(axis, 0)), k


# ---- order, streams, graphs -------------------------------------------------------------------
def all_three(seed, dtype=torch.bfloat16):
    conv, scan = conv_problem(seed, dtype, 140, 3, 96, 4), scan_problem(seed + 1, dtype, 140, 3, 96, 16)
    norm = norm_problem(seed + 2, dtype, (140, 3, 96), False)

    def run():
        out = {"conv " + k: v for k, v in run_conv(conv.g).items()}
        out.update({"scan " + k: v for k, v in run_scan(scan.g).items()})
        out.update({"norm " + k: v for k, v in run_norm(norm.g, False).items()})
        return {k: v for k, v in out.items() if v is not None}
    return run


def same(a, b):
    return all(torch.equal(a[k], b[k]) for k in a)


def test_repeated_calls_give_the_same_bits():
    run = all_three(20)
    first = run()
    assert all(same(first, run()) for _ in range(3))


def test_two_streams_at_once():
    runs = [all_three(30), all_three(40)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [[], []]
    for _ in range(5):
        for i, (r, s) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(s):
                got[i].append(r())
    torch.cuda.synchronize()
    assert all(same(w, g) for w, gs in zip(want, got) for g in gs)


def test_graphs():
    """Two graphs of all the operators, replayed in turn with eager calls between."""
    runs = [all_three(50), all_three(60)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    captured = []
    for r in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = r()
        captured.append((graph, outs))
    for replay in range(4):
        print("replay", replay, flush=True)
        for _, outs in captured:
            for v in outs.values():
                v.zero_()
        for graph, _ in captured:
            graph.replay()
        between = runs[replay % 2]()
        torch.cuda.synchronize()
        assert all(same(w, outs) for w, (_, outs) in zip(want, captured))
        assert same(want[replay % 2], between)


# ---- in place, single steps -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=short)
@pytest.mark.parametrize("N,D,W", [(1, 1, 2), (3, 100, 4), (2, 33, 8), (4, 50, 1)])
def test_conv_steps_in_place(N, D, W, dtype):
    q = conv_problem(N + D, dtype, 11, N, D, W)
    y, last = ops.causal_conv_forward(q.g["x"], q.g["kernel"], q.g["bias"], True, q.g["state"])
    state, ys = q.g["state"].clone(), []
    for t in range(11):
        yt, out = ops.causal_conv_iterate(q.g["x"][t], state, q.g["kernel"], q.g["bias"], True, state_out=state)
        assert out is state
        ys.append(yt)
    assert torch.equal(torch.stack(ys), y) and torch.equal(state, last)


def test_outputs_that_are_given_are_checked():
    q, s = conv_problem(1, torch.float32, 1, 2, 8, 4), scan_problem(1, torch.float32, 1, 2, 8, 4)
    with pytest.raises(ValueError):
        ops.causal_conv_iterate(q.g["x"][0], q.g["state"], q.g["kernel"], state_out=torch.empty(3, 2, 9, device="cuda"))
    with pytest.raises(ValueError):
        ops.causal_conv_iterate(q.g["x"][0], None, q.g["kernel"])
    step = [s.g[k][0] if k in ("x", "delta", "B", "C") else s.g[k] for k in ("x", "delta", "A", "B", "C", "h0")]
    with pytest.raises(ValueError):
        ops.selective_scan_iterate(*step, h_out=torch.empty(2, 8, 4, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError):
        ops.selective_scan_backward(s.g["x"], s.g["delta"], s.g["A"], s.g["B"], s.g["C"], None, None, None, True, None, None, None, s.g["dy"])


# ---- the layers together -------------------------------------------------------------------------
class Block(torch.nn.Module):
    """A state space block between two norms, projections by torch."""

    def __init__(self, width, inner, states, groups):
        super().__init__()
        self.into = torch.nn.Linear(width, 2 * inner, bias=False)
        self.conv = haste_amd.CausalConv(inner, 4)
        self.select = torch.nn.Linear(inner, inner + 2 * groups * states, bias=False)
        self.scan = haste_amd.SelectiveScan(inner, states, groups)
        self.back = torch.nn.Linear(inner, width, bias=False)
        self.norm = haste_amd.ResidualNorm(width)
        self.split = [inner, groups * states, groups * states]

    def forward(self, x, residual, lengths=None):
        u, z = self.into(x).chunk(2, -1)
        u, conv_state = self.conv(u, lengths=lengths)
        delta, B, C = self.select(u).split(self.split, -1)
        y, h = self.scan(u, delta, B, C, z, lengths=lengths)
        out, normed = self.norm(self.back(y), residual)
        return out, normed, conv_state, h

    def step(self, x, residual, conv_state, h):
        u, z = self.into(x).chunk(2, -1)
        u, conv_state = self.conv.step(u, conv_state)
        delta, B, C = self.select(u).split(self.split, -1)
        y, h = self.scan.step(u, delta, B, C, z, h)
        out, normed = self.norm(self.back(y), residual)
        return out, normed, conv_state, h


@pytest.mark.parametrize("lengths", [None, [33, 0, 7]])
def test_block_trains_like_its_plain_form(lengths):
    """The fused layers against the layers' own plain form in float64 on the CPU: values and every gradient."""
    torch.manual_seed(1)
    block = Block(24, 40, 12, 2)
    plain = Block(24, 40, 12, 2).double()
    plain.load_state_dict(block.state_dict())
    block = block.cuda()
    x, r = torch.randn(33, 3, 24), torch.randn(33, 3, 24)
    results = []
    for model, to in ((block, lambda t: t.cuda()), (plain, lambda t: t.double())):
        xi, ri = to(x.clone()).requires_grad_(), to(r.clone()).requires_grad_()
        outs = model(xi, ri, lengths)
        torch.manual_seed(2)
        ups = [to(torch.randn(o.shape)) for o in outs]
        grads = torch.autograd.grad(outs, [xi, ri, *model.parameters()], ups)
        results.append([t.detach().cpu().double() for t in (*outs, *grads)])
    # float32 products of up to 99 terms on both sides of the operators; relative to the largest value
    for got, want in zip(*results):
        assert (got - want).abs().max() <= 2e-5 * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=short)
def test_block_steps_like_it_runs(dtype):
    torch.manual_seed(3)
    block = Block(24, 40, 16, 1).cuda().to(dtype)
    x, r = (torch.randn(19, 2, 24, device="cuda").to(dtype) for _ in range(2))
    with torch.no_grad():
        out, normed, conv_state, h = block(x, r)
        state, hs, outs = torch.zeros(3, 2, 40, device="cuda", dtype=dtype), None, []
        for t in range(19):
            o, n, state, hs = block.step(x[t], r[t], state, hs)
            outs.append(o)
    # the projections of torch may round a product another way for other shapes: a step of the type, and what follows from it
    tolerance = 64 * torch.finfo(dtype).eps
    assert (torch.stack(outs).float() - out.float()).abs().max() <= tolerance * out.float().abs().max()
    assert (hs - h).abs().max() <= tolerance * h.abs().max()
    assert h.dtype == torch.float32 and conv_state.dtype == dtype


def test_layers_batch_first_and_half_parameters():
    torch.manual_seed(4)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        a, b = haste_amd.SelectiveScan(20, 8).cuda().to(dtype), haste_amd.SelectiveScan(20, 8, batch_first=True).cuda().to(dtype)
        b.load_state_dict(a.state_dict())
        tensors = [torch.randn(9, 3, k, device="cuda").to(dtype).requires_grad_() for k in (20, 20, 8, 8, 20)]
        y, h = a(*tensors, lengths=[9, 4, 2])
        firsts = [t.detach().transpose(0, 1).contiguous().requires_grad_() for t in tensors]
        y2, h2 = b(*firsts, lengths=torch.tensor([9, 4, 2]))
        assert torch.equal(y2.transpose(0, 1), y) and torch.equal(h, h2)
        grads, grads2 = (torch.autograd.grad([yy, hh], [*ts, *m.parameters()], [torch.ones_like(yy), torch.ones_like(hh)])
                         for yy, hh, ts, m in ((y, h, tensors, a), (y2, h2, firsts, b)))
        for g, g2, t in zip(grads, grads2, [*tensors, *a.parameters()]):
            assert g.dtype == t.dtype
            assert torch.equal(g, g2 if g.dim() < 3 else g2.transpose(0, 1))


def test_inference_keeps_nothing_for_a_backward_pass():
    q = scan_problem(8, torch.bfloat16, 100, 2, 50, 16)
    g = q.g
    y, h, cache = ops.selective_scan_forward(False, g["x"], g["delta"], g["A"], g["B"], g["C"], g["D"], g["z"], g["delta_bias"], True, g["h0"])
    assert cache is None
    full = run_scan(g)
    assert torch.equal(y, full["y"]) and torch.equal(h, full["h_last"])


# ---- what stays apart, what may be repeated -----------------------------------------------------
def test_a_bad_value_stays_in_its_channel_and_row():
    c, s, n = conv_problem(3, torch.float32, 150, 3, 40, 4), scan_problem(3, torch.float32, 150, 3, 40, 16), norm_problem(3, torch.float32, (150, 3, 40), True)
    for run, q, name in ((run_conv, c, "x"), (run_scan, s, "x"), (lambda g: run_norm(g, True), n, "update")):
        good = run(q.g)
        for bad in (float("nan"), float("inf")):
            t = q.g[name].clone()
            t[70, 1, 5] = bad
            got = run(dict(q.g, **{name: t}))
            for k in got:
                if got[k] is None or got[k].dim() < 3 or k == "dstate" or k == "state":
                    continue
                rows = got[k] if got[k].shape[1] == 3 else got[k].transpose(0, 1)
                want = good[k] if got[k].shape[1] == 3 else good[k].transpose(0, 1)
                others = [0, 2]
                assert torch.equal(rows[:, others], want[:, others]), (k, bad)
                if name == "x" and k in ("y", "dx", "ddelta", "dz"):  # (a norm's row is one)
                    keep = [d for d in range(40) if d != 5]
                    assert torch.equal(rows[:, 1][:, keep], want[:, 1][:, keep]), (k, bad)
            if name == "x":
                assert not got["y"][70, 1, 5].isfinite() and torch.equal(got["y"][:70, 1, 5], good["y"][:70, 1, 5])


def test_backward_twice_and_refused_second_derivatives():
    torch.manual_seed(5)
    conv, scan, norm = haste_amd.CausalConv(24).cuda(), haste_amd.SelectiveScan(24, 8).cuda(), haste_amd.ResidualNorm(24).cuda()
    x, delta, B, C, z = (torch.randn(40, 2, k, device="cuda", requires_grad=True) for k in (24, 24, 8, 8, 24))
    y, _ = scan(conv(x)[0], delta, B, C, z)
    out, normed = norm(y, x, z)
    loss = (out * normed).sum()
    leaves = [x, delta, B, C, z, *conv.parameters(), *scan.parameters(), *norm.parameters()]
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    second = torch.autograd.grad(loss, leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError):
        second[0].sum().backward()


def test_steps_from_no_state():
    torch.manual_seed(6)
    conv, scan = haste_amd.CausalConv(24).cuda(), haste_amd.SelectiveScan(24, 8).cuda()
    x, delta, B, C, z = (torch.randn(1, 2, k, device="cuda") for k in (24, 24, 8, 8, 24))
    with torch.no_grad():
        y, state = conv(x)
        y1, state1 = conv.step(x[0])
        assert torch.equal(y[0], y1) and torch.equal(state, state1)
        y, h = scan(x, delta, B, C, z)
        y1, h1 = scan.step(x[0], delta[0], B[0], C[0], z[0])
        assert (y[0] - y1).abs().max() <= 1e-5 and (h - h1).abs().max() <= 1e-5


def test_outputs_that_overlap_inputs_are_refused():
    N, D, S, W = 2, 8, 4, 4
    buffer = torch.randn(W, N, D, device="cuda")
    kernel = torch.randn(W, D, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):  # the states before and after a step, a row apart
        ops.causal_conv_iterate(torch.randn(N, D, device="cuda"), buffer[:3], kernel, state_out=buffer[1:])
    with pytest.raises(ValueError, match="overlaps"):
        ops.causal_conv_iterate(buffer[3], torch.randn(3, N, D, device="cuda"), kernel, state_out=buffer[1:])
    states = torch.randn(N + 1, D, S, device="cuda")
    step = [torch.randn(N, D, device="cuda"), torch.randn(N, D, device="cuda"), -torch.rand(D, S, device="cuda"),
            torch.randn(N, S, device="cuda"), torch.randn(N, S, device="cuda")]
    with pytest.raises(ValueError, match="overlaps"):
        ops.selective_scan_iterate(*step, states[:N], h_out=states[1:])
    y, h = ops.selective_scan_iterate(*step, states[:N])
    again = states.clone()
    y2, h2 = ops.selective_scan_iterate(*step, again[:N], h_out=again[:N])
    assert torch.equal(y, y2) and torch.equal(h, again[:N]) and torch.equal(states[N], again[N])


def test_strided_states_are_copied():
    q, s = conv_problem(2, torch.float32, 1, 3, 20, 4), scan_problem(2, torch.float32, 1, 3, 20, 4)
    state = q.g["state"].transpose(0, 1).contiguous().transpose(0, 1)
    want = ops.causal_conv_iterate(q.g["x"][0], q.g["state"], q.g["kernel"], q.g["bias"], True)
    got = ops.causal_conv_iterate(q.g["x"][0], state, q.g["kernel"].t().contiguous().t(), q.g["bias"], True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = {k: v[0] if k in ("x", "delta", "B", "C", "z") else v for k, v in s.g.items()}
    h = g["h0"].transpose(1, 2).contiguous().transpose(1, 2)
    A = g["A"].t().contiguous().t()
    want = ops.selective_scan_iterate(g["x"], g["delta"], g["A"], g["B"], g["C"], g["h0"])
    got = ops.selective_scan_iterate(g["x"], g["delta"], A, g["B"], g["C"], h)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
