"""The state space block's operators at sizes beyond those of one grid, one workgroup or one turn."""
import pytest
import torch

from haste_amd import ops

import state_space_bounds as bounds
import state_space_formulas as formulas
from test_gpu_state_space import DTYPES, Problem, compare, norm_problem, run_conv, run_norm, run_scan, scan_problem

pytestmark = pytest.mark.gpu


def _scan_tensors(seed, T, N, D, S, G, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    return dict(x=normal(T, N, D), delta=normal(T, N, D), A=-torch.rand(D, S, generator=gen, device="cuda"), B=normal(T, N, G, S),
                C=normal(T, N, G, S), D=normal(D, dtype=torch.float32), z=normal(T, N, D), delta_bias=normal(D, dtype=torch.float32),
                dy=normal(T, N, D))


def _scan(g):
    ins = [g[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "delta_bias")]
    y, h, cache = ops.selective_scan_forward(True, *ins, True)
    grads = ops.selective_scan_backward(*ins, True, None, None, cache, g["dy"])
    return dict(zip(("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dh0"), grads), y=y, h_last=h)


def test_scan_with_gradients_of_B_and_C_beyond_a_grid():
    """2^30 elements of B: more than the threads that a grid has.  The groups' halves by themselves give the same bits."""
    T, N, S, G = 1024, 8, 64, 2048
    assert T * N * S * G >= 2 ** 30
    g = _scan_tensors(1, T, N, G, S, G)
    got = _scan(g)
    for half in (slice(0, G // 2), slice(G // 2, G)):
        part = {k: v[:, :, half].contiguous() if v.dim() > 2 else v[half] for k, v in g.items()}
        want = _scan(part)
        for k, v in want.items():
            mine = got[k][:, half] if k in ("h_last", "dh0") else got[k][:, :, half] if v.dim() > 2 else got[k][half]
            assert torch.equal(mine, v), k
        del part, want


def test_scan_with_more_sums_than_a_grid():
    """Gradients of parameters of more than 2^28 columns.  A channel's do not depend on the channels beside it."""
    D, S = 2 ** 22 + 2 ** 17, 64
    assert D * (S + 2) > 2 ** 28
    g = _scan_tensors(2, 1, 1, D, S, 1)
    got = _scan(g)
    for half in (slice(0, D // 2), slice(D // 2, D)):
        want = _scan({k: v if k in ("B", "C") else v[:, :, half].contiguous() if v.dim() > 2 else v[half] for k, v in g.items()})
        for k, v in want.items():
            if k in ("dB", "dC"):  # sums over the channels
                continue
            mine = got[k][:, half] if k in ("h_last", "dh0") else got[k][:, :, half] if v.dim() > 2 else got[k][half]
            assert torch.equal(mine, v), k
        del want


def test_scan_in_chunks_that_decay_and_grow_by_more_than_float_holds():
    """Over one chunk of the time axis (64 steps here) exp(A sum dt) is 2^-185 and 2^162; the states before and behind it are floats,
    and stay what they are over the other chunks (steps of 0)."""
    T, D, S = 1024, 16, 4
    q = Problem(7, torch.float32)
    delta = torch.zeros(T, 1, D, dtype=torch.float64)
    delta[320:384] = 0.25
    q.put("delta", delta)
    q.put("A", torch.tensor([-8.0, 7.0, -0.5, 0.0]).expand(D, S))
    for name in ("x", "dy"):
        q.put(name, torch.zeros(T, 1, D))
    for name in ("B", "C"):
        q.normal(name, T, 1, 1, S)
    for name in ("h0", "dh_last"):
        q.put(name, torch.tensor([1e20, 1e-30, 1.0, -3.0]).expand(1, D, S).contiguous())
    q.absent("D", "z", "delta_bias")
    q.lengths(None)
    q.p["softplus"] = q.g["softplus"] = False
    want = formulas.scan(q.p)
    assert 1e-36 < want["h_last"][..., 0].min() < 1e-35 and 1e18 < want["dh0"][..., 1].min() < 1e19
    compare(run_scan(q.g), want, formulas.scan(q.p, True), 12 * T + 512)


@pytest.mark.parametrize("T", [16, 20, 203])
def test_scan_of_states_that_forget_everything(T):
    """A of -inf: the state is the step's own input, also where the row ends within a tile (and chunks of the time axis are joined)."""
    q = scan_problem(T, torch.float32, T, 2, 24, 16, softplus=False, lengths=None)
    q.put("delta", q.p["delta"] + 0.01)
    A = q.p["A"].clone()
    A[:, ::3] = -float("inf")
    q.put("A", A)
    want, magnitude = formulas.scan(q.p), formulas.scan(q.p, True)
    got = run_scan(q.g)
    unknown = ("ddelta", "ddelta_bias")  # 0 times infinity: NaN in the formula too
    assert want["ddelta"].isnan().all() and want["dx"].isfinite().all()
    compare({k: v for k, v in got.items() if k not in unknown}, want, magnitude, 12 * T + 200)
    short = {k: v[:T - 3] if torch.is_tensor(v) and v.dim() > 2 and len(v) == T else v for k, v in q.p.items()}
    ended = run_scan(dict(q.g, lengths=torch.full((2,), T - 3, device="cuda")))
    compare({k: ended[k] for k in ("h_last", "dh0", "dA", "dD")}, formulas.scan(short), formulas.scan(short, True), 12 * T + 200)
    step = {k: v[0] if k in ("x", "delta", "B", "C", "z") else v for k, v in q.g.items()}
    _, h = ops.selective_scan_iterate(step["x"], torch.zeros_like(step["delta"]), step["A"], step["B"], step["C"], step["h0"])
    assert torch.equal(h, q.g["h0"])  # a step of 0


# ---- loops that only full grids go through: sizes from the rules by which the kernels are launched --------------
def _cus():
    return torch.cuda.get_device_properties(torch.cuda.current_device()).multi_processor_count


def _rows_for_run(T, run, vectors):
    """Batch rows with which the convolution walks runs of `run` steps: the longest that leave two wavefronts a SIMD."""
    full = _cus() * 4 * 2 * 64
    rows = -(-full // (vectors * -(-T // run)))
    assert run == 64 or rows * vectors * -(-T // (2 * run)) < full, "no number of rows takes such runs"
    return rows


def _parts(entry, sizes, columns):
    """Partials that a backward pass of these sizes leaves, from the workspace it asks for."""
    floats = ops._scratch_bytes(entry, torch.device("cuda", torch.cuda.current_device()), *sizes) // 4
    parts = floats // columns
    while True:  # what adding them takes lies behind them
        groups, scratch = -(-parts // 256), 0
        while groups > 1:
            scratch, groups = scratch + groups, -(-groups // 256)
        if (parts + scratch) * columns <= floats:
            return parts
        parts -= 1


CONV_RUNS = [(64, 63), (64, 64), (64, 65), (64, 127), (64, 128), (64, 129), (64, 200), (32, 33), (32, 64), (32, 65), (32, 96), (32, 97),
             (16, 17), (16, 32), (16, 33), (16, 49)]


@pytest.mark.parametrize("run,T", CONV_RUNS)
def test_conv_in_long_runs(run, T):
    """Runs of 16 to 64 steps, whole and in part, with states and with lengths that end anywhere; a few of the channels against the
    formulas, which know of none beside them."""
    for dtype, D, W in ((torch.bfloat16, 1021, 4), (torch.float32, 516, 8), (torch.float16, 259, 3)):
        N = _rows_for_run(T, run, -(-D // 4))
        print("conv runs", run, T, N, D, W, dtype, flush=True)
        assert _parts("haste_hip_causal_conv_workspace_bytes", (T, N, D, W), (W + 1) * D) == -(-T // run) * N
        gen = torch.Generator(device="cuda").manual_seed(T + D)
        normal = lambda *shape, to=dtype: torch.randn(*shape, generator=gen, device="cuda").to(to)  # noqa: E731, B023
        g = dict(x=normal(T, N, D), kernel=W ** -0.5 * normal(W, D, to=torch.float32), bias=normal(D, to=torch.float32),
                 state=normal(W - 1, N, D), dy=normal(T, N, D), dstate_out=normal(W - 1, N, D), silu=True)
        g["lengths"] = torch.randint(0, T + 1, (N,), generator=gen, device="cuda")
        g["lengths"][0], g["lengths"][-1] = T, -1
        behind = ~formulas.inside(g["lengths"].cpu(), T, N)[0].cuda()
        g["x"][behind] = g["dy"][behind] = float("nan")
        got = run_conv(g)
        channels = [0, 1, 5, D // 2, D - 5, D - 4, D - 2, D - 1]
        p = {k: v[..., channels].double().cpu() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in g.items()}
        p["lengths"] = g["lengths"].cpu()
        # a product, sum or slope of W taps within 8 W + 64 roundings; the parameters' sums: a run's steps in turn, then the runs
        sums = 8 * W + 64 + run + bounds.parts_depth(-(-T // run) * N)
        bounds.compare({k: v[..., channels] for k, v in got.items()}, formulas.conv(p), formulas.conv(p, True),
                       {None: 8 * W + 64, "dkernel": sums, "dbias": sums})


def _norm_rows(D, waves):
    """Rows of one turn of all workgroups."""
    threads = 64
    while threads * 8 < D:
        threads *= 2
    block = max(256, threads)
    return _cus() * 4 * waves * 64 // block * (block // threads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=lambda t: str(t).split(".")[1])
@pytest.mark.parametrize("D", [40, 513, 700, 2048, 4096, 5000, 8192])
def test_norms_of_more_rows_than_a_turn(D, dtype):
    """Three turns of the forward pass's workgroups and more of the backward pass's, the last one in part."""
    forward, backward = _norm_rows(D, 4), _norm_rows(D, 2)
    rows, centered = 2 * forward + forward // 2 + 3, (D % 1024 == 0) == (dtype == torch.float32)
    print("norm turns", D, rows, dtype, flush=True)
    assert _parts("haste_hip_residual_norm_workspace_bytes", (rows, 1, D), 4 * D) == backward
    q = norm_problem(D, dtype, (rows, 1, D), centered)
    # every factor, two norms forward and backward, within a row's sum and 32 roundings; sums over rows: turns, then workgroups
    factors = 8 * (bounds.ROW_SUM + 32)
    sums = factors + -(-rows // backward) + bounds.parts_depth(backward)
    bounds.compare(run_norm(q.g, centered), formulas.norm(q.p), formulas.norm(q.p, True),
                   {None: factors, "dscale": sums, "dafter": sums, "dbefore": sums, "dbias": sums})


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
@pytest.mark.parametrize("D,S,G", [(1024, 16, 1), (500, 64, 4), (2001, 5, 3), (1030, 30, 2)])
def test_scan_steps_of_more_rows_than_a_turn(D, S, G, dtype):
    """Workgroups go through three rows, some through two; in place too."""
    lanes = 2 if S <= 8 else 4 if S <= 16 else 8 if S <= 32 else 16
    down = _cus() * 8 // -(-D * lanes // 256)
    N = 2 * down + max(1, down // 3)
    assert down > 1
    print("scan step turns", N, D, S, dtype, flush=True)
    q = scan_problem(D + S, dtype, 1, N, D, S, G)
    g = {k: v[0] if k in ("x", "delta", "B", "C", "z") else v for k, v in q.g.items()}
    rest = [g[k] for k in ("D", "z", "delta_bias")]
    y, h = ops.selective_scan_iterate(g["x"], g["delta"], g["A"], g["B"], g["C"], g["h0"], *rest, True)
    want, magnitude = formulas.scan(q.p), formulas.scan(q.p, True)
    for k, v in dict(y=y[None], h_last=h).items():
        bounds.check(v, want[k], magnitude[k], S + 64, k)
    state = g["h0"].clone()
    y2, h2 = ops.selective_scan_iterate(g["x"], g["delta"], g["A"], g["B"], g["C"], state, *rest, True, h_out=state)
    assert h2 is state and torch.equal(state, h) and torch.equal(y2, y)


FORGET = 64  # steps after which a state is exp(-0.2 * 64) = 3e-6 of itself: what is older adds less than a rounding to an output's


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda t: str(t).split(".")[1])
@pytest.mark.parametrize("T,N,D,S,G", [(100, 520, 10, 16, 1), (60, 260, 18, 33, 1), (1300, 1, 40, 16, 2), (1300, 2, 24, 7, 1),
                                       (700, 3, 50, 30, 1), (333, 9, 131, 64, 1)])
def test_scan_within_the_roundings_of_its_memory(T, N, D, S, G, dtype):
    """Decays of exp(-0.2) and faster: errors of steps long past are forgotten with their states, so that the roundings of a result are
    those of a memory's steps however long the sequence is.  One piece of the time axis over more workgroups than CUs, and many
    chunks of it."""
    print("scan memory", T, N, D, S, G, dtype, flush=True)
    q = scan_problem(T + D, dtype, T, N, D, S, G, softplus=False)
    q.put("delta", 0.2 + 0.2 * torch.rand(T, N, D, generator=q.gen, dtype=torch.float64))
    q.put("A", -1 - 3 * torch.rand(D, S, generator=q.gen, dtype=torch.float64), torch.float32)
    if T < 1000:
        q.lengths([T, 0, T - 1] + [1 + (7 * n) % T for n in range(N - 3)])
        behind = ~formulas.inside(q.p["lengths"], T, N)[0].cuda()
        for name in ("x", "delta", "z", "B", "C", "dy"):
            q.g[name][behind] = float("nan")
    # a step of a state: exponent, exp2, two products, a sum, forward and backward.  Sums over states, over a workgroup's channels and the
    # workgroups; of parameters: steps in turn (a chunk's, or all of one piece), then chunks and rows
    each = 12 * FORGET + S + 128
    shared = each + 64 + -(-D // (16 * G))
    sums = each + T + bounds.parts_depth(T // 64 * N + N)
    bounds.compare(run_scan(q.g), formulas.scan(q.p), formulas.scan(q.p, True),
                   {None: each, "dB": shared, "dC": shared, "dA": sums, "dD": sums, "ddelta_bias": sums}, absent=("ddelta_bias",))


def test_caches_that_are_not_whole_are_refused():
    """Views of fewer bytes than they have elements, and of others than the forward pass wrote."""
    q = scan_problem(3, torch.float32, 20, 2, 24, 16)
    ins = [q.g[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "delta_bias")]
    _, _, cache = ops.selective_scan_forward(True, *ins, True, q.g["h0"])
    spread = torch.stack([cache, cache], -1)[..., 0]
    for bad in (cache[:1].expand(cache.shape), spread, cache[:-1], cache.float(), cache.cpu(), None):
        with pytest.raises(ValueError, match="cache"):
            ops.selective_scan_backward(*ins, True, q.g["h0"], None, bad, q.g["dy"])


def test_parameters_of_a_long_scan_in_one_piece():
    """dA adds up T products, here all of one sign, by tiles of 16: their sums' rounding is that of chains of 16, of T / 16 tiles and of 64
    rows, whose errors add up like steps of a random walk (sqrt(n / 3) of a step where the sum grows evenly).  A single chain of T
    would be off by sqrt(T / 3) = 52 times a rounding's 0.58 * 2^-24."""
    T, D, S, N = 8192, 16, 4, _cus() + 4
    q = Problem(11, torch.float32)
    positive = lambda *shape: 0.5 + torch.rand(*shape, generator=q.gen, dtype=torch.float64)  # noqa: E731
    for name in ("x", "dy"):
        q.put(name, positive(T, 1, D))
    q.put("delta", 0.1 * positive(T, 1, D))
    q.put("A", -positive(D, S))
    for name in ("B", "C"):
        q.put(name, positive(T, 1, 1, S))
    q.absent("D", "z", "delta_bias", "h0", "dh_last")
    q.lengths(None)
    q.p["softplus"] = q.g["softplus"] = False
    # the same row for all: enough of them that the time axis is not cut
    g = {k: v.expand(T, N, *v.shape[2:]) if torch.is_tensor(v) and v.dim() > 2 else v for k, v in q.g.items()}
    got, want = run_scan(g)["dA"].cpu().double(), N * formulas.scan(q.p)["dA"]
    assert want.min() > 0
    error = ((got - want) / want).square().mean().sqrt()
    # eight roundings for the factors of the products, whose errors have a common part
    assert error <= 2.0 ** -24 * ((16 / 3 + T / 16 / 3 + 64 / 3) ** 0.5 + 8), error
