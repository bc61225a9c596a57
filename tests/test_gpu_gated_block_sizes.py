"""Sizes, rows and values at which the operators of a gated linear recurrent block could go wrong, on the GPU against the formulas in
float64 (gated_block_formulas.py), bounded as derived there."""
import pytest
import torch

import haste_amd
from haste_amd import lib, ops

import gated_block_formulas as formulas
import state_space_bounds as bounds
from test_gpu_gated_block import PARTS, compare_linear, exact_linear, gated_problem, linear_problem, run_gated, run_linear
from test_gpu_state_space import short

pytestmark = pytest.mark.gpu


def _far(t, distance, memory):
    """The rows of t, `distance` elements apart."""
    rows = memory.as_strided(t.shape, (distance, 1))
    return rows.copy_(t)


@pytest.mark.parametrize("R,C,D", [(200, 1028, 4096), (129, 4096, 4096)])
def test_floats_of_rows_far_apart(R, C, D):
    """The last steps of long sequences, one behind the other: the products' contractions over rows are cut into short runs.  Sums of
    runs are added as pieces are, a rounding for 32 terms or more: the bound has room for one for 16 in each of two sums."""
    distance = 2 ** 22
    memory = torch.empty(R * distance, device="cuda")
    q = linear_problem(R, torch.float32, (R,), C, D, "silu")
    want = exact_linear(q)
    for name in ("x", "residual", "dy"):
        print("far", R, C, D, name, flush=True)
        compare_linear(run_linear(dict(q.g, **{name: _far(q.g[name], distance, memory)})), want)


@pytest.mark.parametrize("R,C,D", [(300, 1000, 600000), (1000, 600000, 64)])
def test_floats_of_long_rows(R, C, D):
    """More than 2^19 columns on either side of the kernel, where a contraction of the other two sizes is cut: the last columns of each."""
    print("long", R, C, D, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(D)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    g = dict(x=normal(R, C), kernel=normal(C, D) * C ** -0.5, bias=normal(D), residual=None, dy=normal(R, D), activation="none")
    got = run_linear(g)
    part = lambda **cut: {"dtype": torch.float32, "activation": "none", "residual": None,  # noqa: E731
                          **{k: g[k].double() if i is None else g[k][i].double() for k, i in cut.items()}}
    last = (slice(None), slice(-24, None))
    want = formulas.linear(part(x=None, kernel=last, bias=slice(-24, None), dy=last))  # all inputs, the last outputs
    for k, at in (("y", last), ("dkernel", last), ("dbias", slice(-24, None))):
        formulas.check_error(got[k][at], *want[k], k)
    want = formulas.linear(part(x=last, kernel=slice(-24, None), bias=None, dy=None))  # the last inputs, all outputs
    formulas.check_error(got["dx"][last], *want["dx"], "dx")
    formulas.check_error(got["dkernel"][-24:], *want["dkernel"], "dkernel")


def test_floats_cut_into_runs_of_more_pieces():
    """Runs of a contraction over rows that are cut into more pieces than the whole would be."""
    for R, C, D, distance in ((2550, 192, 2700, 237495), (16427, 128, 2112, 37069)):
        print("runs", R, C, D, distance, flush=True)
        q = linear_problem(R, torch.float32, (R,), C, D, "none")
        memory = torch.empty(R * distance, device="cuda")
        compare_linear(run_linear(dict(q.g, x=_far(q.g["x"], distance, memory))), exact_linear(q))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=short)
def test_a_single_row_in_the_scratch_memory_it_asks_for(dtype):
    """A row of a wider tensor whose rows are a multiple of 16 bytes apart, its own width is not: what lies behind the scratch memory stays."""
    element, sfx = torch.finfo(dtype).bits // 8, {torch.float32: "_f32", torch.float16: "_f16", torch.bfloat16: "_bf16"}[dtype]
    for C, D, x_row in ((77, 992, 80), (2049, 70, 2056)):
        q = linear_problem(C, dtype, (1,), C, D, "none", True, False)
        want, g = exact_linear(q), q.g
        x = torch.full((1, x_row), float("nan"), device="cuda", dtype=dtype)
        x[:, :C] = g["x"]
        got = {k: torch.full(s, 7.0, device="cuda", dtype=dtype) for k, s in (("y", (1, D)), ("dx", (1, C)), ("dkernel", (C, D)), ("dbias", (D,)))}
        for backward in (0, 1):
            print("single", C, D, backward, dtype, flush=True)
            size = ops._scratch_bytes("haste_hip_linear_workspace_bytes", x.device, backward, element, 1, C, D, 1)
            scratch = torch.full((size + 256,), 77, device="cuda", dtype=torch.uint8)
            if backward:
                lib.call("haste_hip_linear_backward" + sfx, 1, C, D, x, x_row, g["kernel"], 0, None, g["dy"], D, got["dx"], got["dkernel"],
                         got["dbias"], scratch, size)
            else:
                lib.call("haste_hip_linear_forward" + sfx, 1, C, D, x, x_row, g["kernel"], g["bias"], 0, None, 0, got["y"], None, scratch, size)
            assert (scratch[size:] == 77).all()
        compare_linear(got, want)


# ---- clipping ---------------------------------------------------------------------------
def check_scaled(got, grads, factor):
    """The factor is rounded twice and the product once, to floats or among doubles to doubles."""
    for a, g in zip(got, grads):
        want = g.double() * factor
        formulas.check_error(a, want, want.abs() * 4 * 2.0 ** (-50 if a.dtype == torch.float64 else -24), "clipped")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=short)
def test_clip_by_a_norm_beyond_a_float(dtype):
    """Finite gradients are brought to the length that is asked for, whether every workgroup adds the norm's parts up or one does."""
    for count, size in ((1, 2), (3, 8192), (130, 300001)):
        print("beyond", count, size, dtype, flush=True)
        grads = [torch.full((size,), 3e38 if i % 2 else -2.5e38, device="cuda", dtype=dtype) for i in range(count)]
        norm = float(sum(g[:1].double().square().sum() * size for g in grads).sqrt())
        assert ops.gradient_norm(grads).isinf()
        for max_norm in (1.0, 1e-6, 1e20):
            clipped, n = ops.clip_gradients(grads, max_norm)
            assert n.isinf() and n.dtype == torch.float32
            check_scaled(clipped, grads, max_norm / norm)
        same, _ = ops.clip_gradients(grads, 1.0, out=[g.clone() for g in grads])
        check_scaled(same, grads, 1.0 / norm)
        zeros, given = ops.clip_gradients(grads, 1.0, norm=n)
        assert given is n and all((z == 0).all() for z in zeros)  # an infinite norm that is given is taken for infinite


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64], ids=short)
def test_clip_by_factors_below_a_floats_range(dtype):
    few, many = torch.tensor([3e37, -1e37, 1e20, 0.0], device="cuda", dtype=dtype), torch.linspace(-2e37, 2e37, 20001, device="cuda").to(dtype)
    for grads in ([few], [few, many]):  # a norm of 3.2e37, and one of 2e37 sqrt(20001 / 3) = 1.6e39, which a float does not hold
        norm = float(sum(g.double().square().sum() for g in grads).sqrt())
        for max_norm in (1e-9, 1e-2, 0.5):
            clipped, n = ops.clip_gradients(grads, max_norm)
            assert n.isinf() if dtype != torch.float64 and norm > 3.41e38 else abs(float(n) - norm) <= norm * 2.0 ** -24
            check_scaled(clipped, grads, max_norm / norm)


def test_clip_of_doubles_in_range_and_beyond():
    for scale in (1e150, 1e-150):
        g = torch.randn(5001, device="cuda", dtype=torch.float64) * scale
        norm = float((g / scale).square().sum().sqrt()) * scale
        assert abs(float(ops.gradient_norm([g])) - norm) <= norm * 1e-14
    clipped, _ = ops.clip_gradients([torch.full((4,), 1e150, device="cuda", dtype=torch.float64)], 1.0)
    assert (clipped[0] - 0.5).abs().max() <= 1e-14
    clipped, norm = ops.clip_gradients([torch.full((4,), 1e155, device="cuda", dtype=torch.float64)], 1.0)
    assert norm.isinf() and (clipped[0] == 0).all()  # as documented: squares of doubles have a range


def test_a_parameter_that_is_listed_twice_is_clipped_once():
    """The parameters of two models that share a weight, one behind the other."""
    tied = torch.nn.Parameter(torch.zeros(100, 70, device="cuda"))
    own = [torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=t)) for n, t in ((5, torch.float32), (9001, torch.bfloat16))]
    for p in (tied, *own):
        p.grad = torch.randn(p.shape, device="cuda").to(p.dtype)
    before = [p.grad.clone() for p in (tied, *own)]
    norm = float(sum(g.double().square().sum() for g in before).sqrt())
    got = haste_amd.clip_gradients_([tied, own[0], tied, own[1]], 0.25)
    assert abs(float(got) - norm) <= norm * 2.0 ** -24
    check_scaled([p.grad for p in (tied, *own)], before, 0.25 / norm)


# ---- the recurrence --------------------------------------------------------------------
def test_every_gradient_of_extreme_gates():
    """Gates that are shut or open beyond what a float tells from 0 and 1 under decays of nothing and of everything: all gradients.  Where
    1 - a^2 is below a float's normal range it and its root's slope are 0: what enters, x sqrt(1 - a^2), is then off by 2^-63 |x| at most, and
    what reaches forget through it, |x sqrt(decay r / 2)|, by half of that."""
    T, N, D = 70, 2, 64
    q = gated_problem(17, torch.float32, T, N, D)
    forget = torch.randn(T, N, D, generator=q.gen, dtype=torch.float64)
    forget[::3], forget[1::3] = 200.0, -200.0
    q.put("forget", forget)
    q.put("admit", forget.flip(0))
    q.put("decay", torch.where(torch.arange(D) % 2 == 0, 1e-30, 1e30), torch.float32)
    p = q.p
    rate = 2 * p["decay"] * torch.sigmoid(p["forget"] + p["forget_bias"])
    cut = rate < 2.0 ** -126
    assert ((rate < 2.0 ** -140) | (rate > 2.0 ** -110)).all() and 0 < cut.sum() < cut.numel()  # none near the border
    got, want, most = run_gated(q.g), formulas.gated(p), formulas.gated(p, True)
    silu = (p["z"] * torch.sigmoid(p["z"])).abs()
    most_g = ((p["dy"].abs() * silu).sum(0) + p["dh_last"].abs()).max()  # no a is above 1
    off = cut * 2.0 ** -63 * most_g * (1 + p["x"].abs())
    entered = 2.0 ** -63 * p["x"].abs().sum(0)
    allowed = dict(dx=off, dforget=off, dadmit=off, dforget_bias=off.sum((0, 1)), dadmit_bias=off.sum((0, 1)), h_last=entered, y=entered * silu,
                   dz=entered * p["dy"].abs() * (1 + p["z"].abs()))
    roundings = 24 * T + N + 64
    assert set(got) == set(want) == {"y", "h_last", "dx", "dforget", "dadmit", "dz", "ddecay", "dforget_bias", "dadmit_bias", "dh0"}
    for k in want:
        bounds.check(got[k], want[k], most[k] + allowed.get(k, 0.0) / (roundings * 2.0 ** -24), roundings, k)
    assert (got["dforget"].cpu()[cut] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=short)
def test_steps_are_what_the_whole_is(dtype):
    for N, D, options in ((1, 1, {}), (3, 100, dict(decay=False)), (2, 33, dict(admit=False)), (4, 51, dict(decay=False, admit=False, z=False)),
                          (70, 2000, {})):
        print("steps", N, D, options, dtype, flush=True)
        q = gated_problem(N + D, dtype, 5, N, D, **options)
        full, want, most = run_gated(q.g), formulas.gated(q.p), formulas.gated(q.p, True)
        state, ys = q.g["h0"], []
        for t in range(5):
            x, forget, admit, z = (None if q.g[k] is None else q.g[k][t] for k in ("x", "forget", "admit", "z"))
            y, state = ops.gated_recurrence_iterate(x, forget, state, admit, z, *[q.g[k] for k in PARTS[2:]])
            ys.append(y)
        for k, stepped in (("y", torch.stack(ys)), ("h_last", state)):
            for value in (full[k], stepped):
                bounds.check(value, want[k], most[k], 24 * 5 + 64, k)
            # both are so far from the same value at most
            error = 2 * (24 * 5 + 64) * 2.0 ** -24 * most[k]
            half_step = 0.0 if stepped.dtype == torch.float32 else torch.finfo(dtype).eps / 2
            apart = (full[k].double() - stepped.double()).abs().cpu()
            assert (apart <= error + 2 * half_step * (want[k].abs() + error) + 2 * torch.finfo(torch.float16).tiny).all(), k
