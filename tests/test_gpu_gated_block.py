"""The operators of a gated linear recurrent block on the GPU against the formulas in float64 (gated_block_formulas.py, whose gradients
are checked by differences and against autograd in test_gated_block_cpu.py), bounded as derived there."""
import math

import pytest
import torch

import haste_amd
from haste_amd import lib, ops

import gated_block_formulas as formulas
import state_space_bounds as bounds
from test_gpu_state_space import DTYPES, Problem, relaid, short

pytestmark = pytest.mark.gpu


# ---- the projection --------------------------------------------------------------------
def linear_problem(seed, dtype, shape, C, D, activation="none", bias=True, residual=True, scale=1.0):
    q = Problem(seed, dtype)
    q.normal("x", *shape, C)
    q.normal("kernel", C, D, scale=scale * C ** -0.5)
    q.normal("bias", D) if bias else q.absent("bias")
    q.normal("residual", *shape, D) if residual else q.absent("residual")
    q.normal("dy", *shape, D)
    q.p["activation"] = q.g["activation"] = activation
    q.p["dtype"] = q.g["dtype"] = dtype
    return q


def run_linear(g):
    y, cache = ops.linear_forward(True, g["x"], g["kernel"], g["bias"], g["activation"], g["residual"])
    dx, dkernel, dbias = ops.linear_backward(g["x"], g["kernel"], g["bias"], g["activation"], cache, g["dy"])
    out = dict(y=y, dx=dx, dkernel=dkernel)
    return out if dbias is None else dict(out, dbias=dbias)


def exact_linear(q):
    """The formulas on the GPU in float64 (products of 4096 in all directions are slow on the host)."""
    return formulas.linear({k: v.cuda() if torch.is_tensor(v) else v for k, v in q.p.items()})


def compare_linear(got, want):
    assert set(got) == set(want)
    for k in want:
        formulas.check_error(got[k], *want[k], k)


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
@pytest.mark.parametrize("shape,C,D,options", [
    ((1,), 1, 1, {}), ((1,), 8, 8, dict(activation="silu")), ((1,), 75, 33, dict(activation="gelu")), ((2, 3), 7, 9, dict(bias=False)),
    ((3,), 64, 130, dict(residual=False)), ((1,), 1024, 257, {}), ((5, 3), 33, 64, dict(activation="silu", residual=False)),
    ((16,), 129, 200, {}), ((17,), 2000, 96, dict(activation="gelu")), ((33,), 96, 2001, {}), ((127,), 31, 127, {}),
    ((128,), 32, 128, dict(activation="gelu")), ((129,), 40, 129, dict(activation="silu")), ((8, 32), 64, 256, {}),
    ((257,), 300, 255, dict(activation="gelu", bias=False)), ((37, 7), 1001, 75, dict(activation="silu")), ((5, 100), 264, 520, {}),
    ((1030,), 72, 1032, dict(activation="gelu")), ((2000,), 128, 64, dict(activation="silu")), ((3, 1367), 65, 1, {})])
def test_linear(shape, C, D, options, dtype):
    print("linear", shape, C, D, options, dtype, flush=True)
    q = linear_problem(C + D, dtype, shape, C, D, **options)
    compare_linear(run_linear(q.g), exact_linear(q))


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
def test_linear_large(dtype):
    """More tiles of the largest kind than CUs, and a contraction that no stage divides."""
    for R, C, D, activation in ((4500, 1000, 4104, "silu"), (2048, 4096, 2304, "gelu")):
        print("large", R, C, D, dtype, flush=True)
        q = linear_problem(R, dtype, (R,), C, D, activation)
        compare_linear(run_linear(q.g), exact_linear(q))


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
def test_linear_ends_anywhere(dtype):
    for n in list(range(1, 18)) + [31, 32, 33, 63, 64, 65]:
        print("ends", n, dtype, flush=True)
        for R, C, D in ((n, 24, 40), (24, n, 40), (24, 40, n), (n, n, n)):
            q = linear_problem(n, dtype, (R,), C, D, "gelu")
            compare_linear(run_linear(q.g), exact_linear(q))


@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_activations_over_their_range(activation):
    """Values from -40 to 40 through a product with one: what the gate lets through of them, and its slope."""
    for dtype in DTYPES:
        v = torch.linspace(-40, 40, 4001, dtype=torch.float64).to(dtype)
        q = linear_problem(1, dtype, (4001,), 1, 1, activation, False, False)
        q.p["x"], q.g["x"] = v.double()[:, None], v.cuda()[:, None]
        q.put("kernel", torch.ones(1, 1, dtype=torch.float64))
        q.put("dy", torch.ones(4001, 1, dtype=torch.float64))
        want = exact_linear(q)
        got = run_linear(q.g)
        for k in ("y", "dx"):
            formulas.check_error(got[k], *want[k], (k, dtype))


@pytest.mark.parametrize("how", ["batch_first", "column_block", "apart"])
@pytest.mark.parametrize("dtype", DTYPES, ids=short)
def test_linear_strides(dtype, how):
    q = linear_problem(5, dtype, (21, 3), 64, 48, "silu")
    want = run_linear(q.g)
    got = run_linear({k: relaid(v, how) if torch.is_tensor(v) else v for k, v in q.g.items()})
    kernel = q.g["kernel"].t().contiguous().t()
    again = run_linear(dict(q.g, kernel=kernel))
    for k in want:
        # the float product goes by another kernel where rows do not start at 16 bytes
        assert torch.equal(want[k], again[k])
        if dtype == torch.float32 and how == "column_block":
            formulas.check_error(got[k], *exact_linear(q)[k], k)
        else:
            assert torch.equal(want[k], got[k]), (how, k)


def test_linear_from_odd_addresses():
    """Everything an element behind a 16-byte boundary."""
    q = linear_problem(6, torch.bfloat16, (40,), 64, 48, "gelu")

    def moved(t):
        flat = torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)
    want, got = run_linear(q.g), run_linear({k: moved(v) if torch.is_tensor(v) else v for k, v in q.g.items()})
    assert all(torch.equal(want[k], got[k]) for k in want)


def test_linear_expanded_inputs():
    q = linear_problem(7, torch.bfloat16, (9, 4), 32, 24, "silu")
    g = dict(q.g, x=q.g["x"][:1].expand(9, -1, -1), residual=q.g["residual"][:, :1].expand(-1, 4, -1), dy=q.g["dy"][:1, :1, :1].expand(9, 4, 24))
    want = run_linear({k: v.contiguous() if torch.is_tensor(v) else v for k, v in g.items()})
    got = run_linear(g)
    assert all(torch.equal(want[k], got[k]) for k in want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=short)
def test_linear_keeps_bad_values_to_their_rows(dtype):
    q = linear_problem(8, dtype, (300,), 72, 56, "silu")
    want, exact = run_linear(q.g), exact_linear(q)

    def unchanged(got, k, rows, columns):
        """To the bit; in float, where a tile with such values goes by another instruction than its like, within the bounds."""
        if dtype == torch.float32:
            formulas.check_error(got[k][rows][:, columns], *(t[rows][:, columns] for t in exact[k]), k)
        else:
            assert torch.equal(got[k][rows][:, columns], want[k][rows][:, columns]), k

    for bad in (float("nan"), float("inf")):
        x = q.g["x"].clone()
        x[137, 71] = bad
        got = run_linear(dict(q.g, x=x))
        others = [r for r in range(300) if r != 137]
        assert not got["y"][137].isfinite().any()
        unchanged(got, "y", others, slice(None))
        unchanged(got, "dx", others, slice(None))
        W = q.g["kernel"].clone()
        W[71, 55] = bad
        got = run_linear(dict(q.g, kernel=W))
        assert not got["y"][:, 55].isfinite().any()
        unchanged(got, "y", slice(None), slice(55))
        unchanged(got, "dkernel", slice(None), slice(55))


def test_linear_gradients_may_be_left_out():
    q = linear_problem(9, torch.bfloat16, (70,), 33, 40, "gelu")
    want = run_linear(q.g)
    g = q.g
    _, cache = ops.linear_forward(True, g["x"], g["kernel"], g["bias"], "gelu", None)
    dx, dkernel, dbias = ops.linear_backward(g["x"], g["kernel"], g["bias"], "gelu", cache, g["dy"], with_dx=False)
    assert dx is None and torch.equal(dkernel, want["dkernel"]) and torch.equal(dbias, want["dbias"])
    dx, dkernel, dbias = ops.linear_backward(g["x"], g["kernel"], None, "gelu", cache, g["dy"], with_dkernel=False)
    assert dkernel is None and dbias is None and torch.equal(dx, want["dx"])
    y, none = ops.linear_forward(False, g["x"], g["kernel"], g["bias"], "gelu", g["residual"])
    assert none is None and torch.equal(y, want["y"])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=short)
def test_linear_of_few_rows_and_more(dtype):
    """Around the numbers of rows and the lengths of the contraction at which another kernel takes over, with few and many columns."""
    for C in (2040, 2048, 2056):
        for R in (15, 16, 17, 31, 32, 33):
            print("few", R, C, dtype, flush=True)
            q = linear_problem(R + C, dtype, (R,), C, 200, "silu")
            compare_linear(run_linear(q.g), exact_linear(q))
    for R, D in ((1, 8192), (1, 8193), (16, 8200), (17, 8191), (32, 8210), (5, 20001)):
        print("wide", R, D, dtype, flush=True)
        q = linear_problem(R + D, dtype, (R,), 72, D, "gelu")
        compare_linear(run_linear(q.g), exact_linear(q))


@pytest.mark.parametrize("R,C,D", [
    (20000, 64, 72),      # small tiles, whole and in many pieces
    (300, 6000, 4200),    # dx in pieces, dkernel whole
    (9000, 520, 1030),    # odd rows, both gradients in small tiles
    (8192, 1024, 2048), (8200, 2051, 2050),  # both in large tiles in one launch
    (4096, 4096, 1024), (1100, 4104, 4104)])
def test_linear_of_every_plan(R, C, D):
    for activation in ("none", "silu"):
        print("plan", R, C, D, activation, flush=True)
        q = linear_problem(R, torch.bfloat16, (R,), C, D, activation)
        compare_linear(run_linear(q.g), exact_linear(q))


@pytest.mark.parametrize("R,C,D", [
    (3001, 300, 1001), (64, 1024, 4100), (200, 1500, 1500),  # tiles of the float instruction, in pieces and whole, of odd rows
    (70, 4096, 4096), (2048, 1030, 1024)])                  # on the other side
def test_linear_of_every_plan_of_floats(R, C, D):
    for activation in ("none", "gelu"):
        print("floats", R, C, D, activation, flush=True)
        q = linear_problem(R, torch.float32, (R,), C, D, activation)
        compare_linear(run_linear(q.g), exact_linear(q))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=short)
def test_linear_beyond_32_bits(dtype):
    """More than 2^31 outputs: the last rows and the last columns."""
    R, C, D, rows, columns = 66000, 24, 32768 + 8, 40, 16
    gen = torch.Generator(device="cuda").manual_seed(3)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
    g = dict(x=normal(R, C), kernel=normal(C, D) * C ** -0.5, bias=normal(D), residual=None, dy=normal(R, D), activation="silu")
    got = run_linear(g)
    part = lambda **cut: {"dtype": dtype, "activation": "silu", "residual": None,  # noqa: E731
                          **{k: g[k].double() if i is None else g[k][i].double() for k, i in cut.items()}}
    want = formulas.linear(part(x=slice(-rows, None), kernel=None, bias=None, dy=slice(-rows, None)))
    for k in ("y", "dx"):
        formulas.check_error(got[k][-rows:], *want[k], k)
    last = (slice(None), slice(-columns, None))
    want = formulas.linear(part(x=None, kernel=last, bias=slice(-columns, None), dy=last))
    formulas.check_error(got["y"][last], *want["y"], "y")
    formulas.check_error(got["dkernel"][last], *want["dkernel"], "dkernel")
    formulas.check_error(got["dbias"][-columns:], *want["dbias"], "dbias")


def test_linear_of_rows_far_apart():
    """The last steps of sequences that lie one behind the other, as the head of a model takes them."""
    whole = torch.empty(5, 70000, 64, device="cuda", dtype=torch.bfloat16)
    q = linear_problem(11, torch.bfloat16, (5,), 64, 64, "silu")
    want = run_linear(q.g)
    for name in ("x", "residual", "dy"):
        whole[:, -1] = q.g[name]
        got = run_linear(dict(q.g, **{name: whole[:, -1]}))
        assert all(torch.equal(want[k], got[k]) for k in want), name


def test_linear_rows_behind_the_last_are_left_alone():
    q = linear_problem(10, torch.bfloat16, (70,), 40, 33, "none", True, False)
    x, kernel, bias = q.g["x"], q.g["kernel"], q.g["bias"]
    y = torch.full((72, 33), 7.0, device="cuda", dtype=torch.bfloat16)
    size = ops._scratch_bytes("haste_hip_linear_workspace_bytes", x.device, 0, 2, 70, 40, 33, 0)
    scratch = torch.empty(size + 64, device="cuda", dtype=torch.uint8)
    scratch[size:] = 77
    lib.call("haste_hip_linear_forward_bf16", 70, 40, 33, x, 40, kernel, bias, 0, None, 0, y[1:], None, scratch, size)
    assert torch.equal(y[1:71], run_linear(q.g)["y"]) and (y[0] == 7).all() and (y[71] == 7).all()
    assert (scratch[size:] == 77).all()


# ---- the recurrence --------------------------------------------------------------------
def gated_problem(seed, dtype, T, N, D, decay=True, admit=True, z=True, biases=True, h0=True, dh=True, lengths=None):
    q = Problem(seed, dtype)
    for name in ("x", "dy"):
        q.normal(name, T, N, D)
    q.normal("forget", T, N, D, scale=2.0, shift=0.0 if decay else 1.0)
    q.normal("admit", T, N, D) if admit else q.absent("admit")
    q.normal("z", T, N, D) if z else q.absent("z")
    if decay:  # from hardly any to a factor of e^-3 a step
        q.put("decay", torch.exp(torch.empty(D, dtype=torch.float64).uniform_(-7, 1.1, generator=q.gen)), torch.float32)
    else:
        q.absent("decay")
    q.normal("forget_bias", D, dtype=torch.float32) if biases else q.absent("forget_bias")
    q.normal("admit_bias", D, dtype=torch.float32) if biases and admit else q.absent("admit_bias")
    q.normal("h0", N, D, dtype=torch.float32) if h0 else q.absent("h0")
    q.normal("dh_last", N, D, dtype=torch.float32) if dh else q.absent("dh_last")
    q.lengths(lengths)
    return q


PARTS = ("admit", "z", "decay", "forget_bias", "admit_bias")


def run_gated(g):
    parts = [g[k] for k in PARTS]
    y, h, cache = ops.gated_recurrence_forward(True, g["x"], g["forget"], *parts, g["h0"], g["lengths"])
    names = ("dx", "dforget", "dadmit", "dz", "ddecay", "dforget_bias", "dadmit_bias", "dh0")
    grads = ops.gated_recurrence_backward(g["x"], g["forget"], *parts, g["h0"], g["lengths"], cache, g["dy"], g["dh_last"])
    return dict({k: v for k, v in zip(names, grads) if v is not None}, y=y, h_last=h)


def compare_gated(got, q):
    """A step's factors are off by some 12 roundings (exponentials of arguments of a few units); T of them follow one another
    forward, as many backward; sums over steps and rows add T / 64 + 4 + 16 times in a workgroup and at most N + 64 behind it."""
    T, N, _ = q.p["x"].shape
    want = formulas.gated(q.p)
    absent = {"d" + k for k in PARTS + ("h0",) if q.p[k] is None}
    bounds.compare(got, want, formulas.gated(q.p, True), 24 * T + N + 64, absent)


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
@pytest.mark.parametrize("T,N,D,options", [
    (1, 1, 1, {}), (1, 3, 75, {}), (2, 2, 9, dict(decay=False)), (3, 1, 64, dict(admit=False)), (4, 2, 127, dict(z=False)),
    (5, 2, 128, dict(decay=False, admit=False)), (7, 2, 129, dict(biases=False)), (63, 2, 40, {}), (64, 2, 41, dict(decay=False, z=False)),
    (65, 2, 130, dict(admit=False, z=False)), (128, 1, 7, dict(h0=False, dh=False)), (130, 5, 300, {}), (257, 3, 24, dict(decay=False, admit=False)),
    (20, 6, 100, dict(lengths=[20, 0, 1, 2, 19, -1])), (200, 4, 13, dict(lengths=[3, 200, 64, -2])), (6, 3, 256, dict(lengths=[0, 0, 0])),
    (200, 5, 33, dict(lengths=[65, 127, 128, 129, 0], decay=False, admit=False, z=False))])
def test_gated(T, N, D, options, dtype):
    print("gated", T, N, D, options, dtype, flush=True)
    q = gated_problem(T + D, dtype, T, N, D, **options)
    q.poison("x", "forget", "admit", "z", "dy")
    compare_gated(run_gated(q.g), q)


@pytest.mark.parametrize("T,N,D,lengths", [(700, 1, 64, None), (1500, 2, 131, [1500, 333]), (4097, 1, 20, None), (999, 3, 5, [0, 998, 512])])
def test_gated_over_a_cut_time_axis(T, N, D, lengths):
    for options in ({}, dict(decay=False), dict(decay=False, admit=False, z=False)):
        print("cut", T, N, D, options, flush=True)
        q = gated_problem(T, torch.float32, T, N, D, lengths=lengths, **options)
        q.poison("x", "forget", "admit", "z", "dy")
        compare_gated(run_gated(q.g), q)


def test_gated_full_grid():
    """A workgroup a CU and more: the time axis in one piece."""
    q = gated_problem(2, torch.bfloat16, 70, 40, 1030)
    compare_gated(run_gated(q.g), q)


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
def test_gated_rows_that_end_anywhere(dtype):
    for D in list(range(1, 10)) + list(range(126, 132)):
        q = gated_problem(D, dtype, 9, 2, D, lengths=[9, 4])
        compare_gated(run_gated(q.g), q)


@pytest.mark.parametrize("how", ["batch_first", "column_block", "apart"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=short)
def test_gated_strides(dtype, how):
    q = gated_problem(2, dtype, 90, 3, 52, lengths=[90, 5, 0])
    want = run_gated(q.g)
    got = run_gated({k: relaid(v, how) if torch.is_tensor(v) and v.dim() == 3 else v for k, v in q.g.items()})
    assert all(torch.equal(want[k], got[k]) for k in want)


def test_gated_strides_beyond_32_bits():
    far = torch.empty(2 ** 31 + 4096, device="cuda", dtype=torch.bfloat16)
    q = gated_problem(9, torch.bfloat16, 2, 2, 64)
    x = far.as_strided((2, 2, 64), (2 ** 31 + 64, 128, 1))
    x.copy_(q.g["x"])
    want, got = run_gated(q.g), run_gated(dict(q.g, x=x))
    assert all(torch.equal(want[k], got[k]) for k in want)
    rows = far.as_strided((700, 64), (3000000, 1))
    p = linear_problem(9, torch.bfloat16, (700,), 64, 40)
    rows.copy_(p.g["x"])
    want, got = run_linear(p.g), run_linear(dict(p.g, x=rows))
    assert all(torch.equal(want[k], got[k]) for k in want)


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
def test_gated_of_one_and_two_channels_a_lane(dtype):
    """On both sides of where a lane takes two channels, and of where the time axis is cut; initial states and lengths of both."""
    for N, D in ((47, 512), (48, 512), (48, 450), (191, 65), (192, 65), (5, 2048), (40, 200), (41, 200)):
        print("lanes", N, D, dtype, flush=True)
        q = gated_problem(N, dtype, 131, N, D, lengths=[131 - 5 * n % 140 if n % 3 else 131 for n in range(N)])
        q.poison("x", "forget", "admit", "z", "dy")
        compare_gated(run_gated(q.g), q)


def test_gated_beyond_32_bits():
    """More than 2^31 elements: the last channels of the last row."""
    T, N, D, last = 264, 255, 32768, 40
    gen = torch.Generator(device="cuda").manual_seed(4)
    g = {k: torch.randn(T, N, D, generator=gen, device="cuda", dtype=torch.bfloat16) for k in ("x", "forget", "dy")}
    g.update({k: None for k in PARTS + ("h0", "dh_last", "lengths")}, decay=torch.rand(D, generator=gen, device="cuda"))
    got = run_gated(g)
    q = Problem(4, torch.bfloat16)
    q.p = {k: v if v is None else v[-last:].double().cpu() if k == "decay" else v[:, -1:, -last:].double().cpu() for k, v in g.items()}
    want, most = formulas.gated(q.p), formulas.gated(q.p, True)
    got = {k: got[k][:, -1:, -last:] if k != "h_last" else got[k][-1:, -last:] for k in ("y", "dx", "dforget", "h_last")}
    bounds.compare(got, {k: want[k] for k in got}, most, 24 * T + 64)


def test_gated_expanded_inputs():
    q = gated_problem(4, torch.bfloat16, 40, 3, 30)
    g = dict(q.g)
    g["z"], g["dy"] = g["z"][:, :1].expand(-1, 3, -1), g["dy"][:1, :1, :1].expand(40, 3, 30)
    want = run_gated({k: v.contiguous() if torch.is_tensor(v) else v for k, v in g.items()})
    got = run_gated(g)
    assert all(torch.equal(want[k], got[k]) for k in want)


def test_gated_lengths_out_of_range_give_nans_for_their_rows():
    for T in (20, 900):
        q = gated_problem(2, torch.float32, T, 3, 24, lengths=[T, T, T])
        good, got = run_gated(q.g), run_gated(dict(q.g, lengths=torch.tensor([T, T + 1, -T - 2], device="cuda")))
        for k in ("y", "dx", "dforget", "dadmit", "dz"):
            assert got[k][:, 1:].isnan().all() and torch.equal(got[k][:, 0], good[k][:, 0]), k
        for k in ("h_last", "dh0"):
            assert got[k][1:].isnan().all() and torch.equal(got[k][0], good[k][0]), k
        for k in ("ddecay", "dforget_bias", "dadmit_bias"):
            assert got[k].isnan().all(), k


def test_gated_extreme_gates():
    """Gates that are shut or open beyond what a float tells from 0 and 1, and decays of nothing and of everything."""
    T, N, D = 70, 2, 64
    for decay in (True, False):
        q = gated_problem(3, torch.float32, T, N, D, decay=decay)
        forget = torch.randn(T, N, D, generator=q.gen, dtype=torch.float64)
        forget[::3], forget[1::3] = 200.0, -200.0
        q.put("forget", forget)
        q.put("admit", forget.flip(0))
        if decay:
            q.put("decay", torch.where(torch.arange(D) % 2 == 0, 1e-30, 1e30), torch.float32)
        got = run_gated(q.g)
        if decay:  # where the decay is nothing, so is what enters, and the square root has no slope to speak of: in range, no more
            assert all(got[k].isfinite().all() for k in ("y", "h_last", "dx", "dz", "dadmit", "dh0"))
            want = formulas.gated(q.p)
            assert (got["y"].cpu() - want["y"]).abs().max() <= 1e-5 * want["y"].abs().max()
        else:
            compare_gated(got, q)
    q = gated_problem(3, torch.float32, T, N, D)
    q.g["decay"] = torch.full((D,), float("inf"), device="cuda")
    q.g["lengths"] = torch.tensor([70, 66], device="cuda")
    got = run_gated(q.g)  # nothing is remembered
    assert got["y"].isfinite().all() and got["dx"].isfinite().all() and got["h_last"].isfinite().all()


def test_gated_roundings_even_out():
    """Gates a little below 1 that multiply a state for hundreds of steps.  Each is rounded once and the product once, by a relative 2^-24 at
    most either way: a spread of sqrt(2 / 3) 2^-24 a step, of which sqrt(T) add up and sqrt(n) even out in the mean of n channels; what
    is not even-handed, two instructions' last bits, is in 1 - gate alone."""
    T, N, D = 470, 4, 1024
    q = Problem(13, torch.float32)
    q.put("forget", torch.empty(T, N, D, dtype=torch.float64).uniform_(5, 9, generator=q.gen))
    _, h, _ = ops.gated_recurrence_forward(False, torch.zeros(T, N, D, device="cuda"), q.g["forget"], h0=torch.ones(N, D, device="cuda"))
    exact = torch.sigmoid(q.p["forget"]).prod(0)
    mean = float((h.cpu().double() / exact - 1).mean())
    bound = 6 * (T * 2 / 3) ** 0.5 * 2.0 ** -24 / (N * D) ** 0.5 + T * float(torch.sigmoid(-q.p["forget"]).mean()) * 2.0 ** -22
    assert abs(mean) <= bound, (mean, bound)


def test_gated_keeps_bad_values_to_their_channels():
    for T in (150, 900):
        q = gated_problem(3, torch.float32, T, 3, 40)
        good = run_gated(q.g)
        for bad in (float("nan"), float("inf")):
            x = q.g["x"].clone()
            x[70, 1, 5] = bad
            got = run_gated(dict(q.g, x=x))
            keep = [d for d in range(40) if d != 5]
            for k in ("y", "dx", "dforget", "dadmit", "dz"):
                assert torch.equal(got[k][:, [0, 2]], good[k][:, [0, 2]]) and torch.equal(got[k][:, 1][:, keep], good[k][:, 1][:, keep]), k
            assert not got["y"][70, 1, 5].isfinite() and torch.equal(got["y"][:70, 1, 5], good["y"][:70, 1, 5])


@pytest.mark.parametrize("dtype", DTYPES, ids=short)
def test_gated_steps_in_place(dtype):
    for N, D, options in ((1, 1, {}), (3, 100, dict(decay=False)), (2, 33, dict(admit=False)), (4, 51, dict(decay=False, admit=False, z=False)),
                          (70, 2000, {})):
        q = gated_problem(N + D, dtype, 5, N, D, **options)
        full = run_gated(q.g)
        step = lambda t: [None if q.g[k] is None else q.g[k][t] for k in ("x", "forget", "admit", "z")]  # noqa: E731, B023
        state, ys = q.g["h0"].clone(), []
        for t in range(5):
            x, forget, admit, z = step(t)
            want = ops.gated_recurrence_iterate(x, forget, state.clone(), admit, z, *[q.g[k] for k in PARTS[2:]])
            y, out = ops.gated_recurrence_iterate(x, forget, state, admit, z, *[q.g[k] for k in PARTS[2:]], h_out=state)
            assert out is state and torch.equal(y, want[0]) and torch.equal(state, want[1])
            ys.append(y)
        bounds.compare(dict(y=torch.stack(ys), h_last=state), {k: formulas.gated(q.p)[k] for k in ("y", "h_last")}, formulas.gated(q.p, True), 24 * 5 + 64)
        assert full["y"].shape == (5, N, D)


def test_gated_outputs_that_are_given_are_checked():
    q = gated_problem(1, torch.float32, 1, 2, 8)
    x, forget = q.g["x"][0], q.g["forget"][0]
    states = torch.randn(3, 8, device="cuda")
    for bad in (torch.empty(2, 9, device="cuda"), torch.empty(2, 8, device="cuda", dtype=torch.float16), states[1:], x):
        with pytest.raises(ValueError):
            ops.gated_recurrence_iterate(x, forget, states[:2], h_out=bad)
    with pytest.raises(ValueError):
        ops.gated_recurrence_backward(q.g["x"], q.g["forget"], None, None, None, None, None, None, None, None, q.g["dy"])
    y, h, cache = ops.gated_recurrence_forward(True, q.g["x"], q.g["forget"])
    with pytest.raises(ValueError):  # a view of other memory
        ops.gated_recurrence_backward(q.g["x"], q.g["forget"], None, None, None, None, None, None, None, cache[:1].expand(cache.numel()), q.g["dy"])


def test_gated_gradients_may_be_left_out():
    q = gated_problem(6, torch.float32, 90, 2, 20)
    q.p["dy"] = q.p["dy"] * 0
    g = q.g
    parts = [g[k] for k in PARTS]
    y, h, cache = ops.gated_recurrence_forward(True, g["x"], g["forget"], *parts, g["h0"])
    got = ops.gated_recurrence_backward(g["x"], g["forget"], *parts, g["h0"], None, cache, None, g["dh_last"])
    names = ("dx", "dforget", "dadmit", "dz", "ddecay", "dforget_bias", "dadmit_bias", "dh0")
    bounds.compare(dict(zip(names, got)), {k: v for k, v in formulas.gated(q.p).items() if k in names}, formulas.gated(q.p, True), 24 * 90 + 66)
    y2, h2, none = ops.gated_recurrence_forward(False, g["x"], g["forget"], *parts, g["h0"])
    assert none is None and torch.equal(y, y2) and torch.equal(h, h2)


# ---- gradients, their norm and clipping ---------------------------------------------------
def exact_norm(grads):
    return math.sqrt(math.fsum(float(v) ** 2 for g in grads for v in g.detach().double().flatten().tolist())) if sum(
        g.numel() for g in grads) < 200000 else math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def check_clipped(got, grads, norm, max_norm):
    factor = min(1.0, max_norm / (norm + 1e-6))
    for a, g in zip(got, grads):
        assert a.dtype == g.dtype and a.shape == g.shape
        want = g.double() * factor
        # the factor is off by one rounding of the norm and one of its own, the product by one more: floats', or among doubles only doubles'
        formulas.check_error(a, want, want.abs() * 4 * 2.0 ** (-50 if a.dtype == torch.float64 else -24), "clipped")


SHAPES = [(1,), (7,), (0,), (512, 64), (3, 5, 7), (8192,), (16384,), (16385,), (100000,), (), (1, 1), (33, 129)]


@pytest.mark.parametrize("dtype", DTYPES + [torch.float64, None], ids=["f32", "f16", "bf16", "f64", "mixed"])
def test_clip(dtype):
    gen = torch.Generator().manual_seed(1)
    grads = [torch.randn(s, generator=gen, dtype=torch.float64).to(dtype or DTYPES[i % 3]).cuda() for i, s in enumerate(SHAPES)]
    norm = exact_norm(grads)
    wide = torch.float64 if dtype is torch.float64 else torch.float32
    got = ops.gradient_norm(grads)
    assert got.dtype == wide and got.shape == () and abs(float(got) - norm) <= norm * (1e-14 if wide is torch.float64 else 2.0 ** -24)
    for max_norm in (0.5, norm * 2, 0.0):
        clipped, n = ops.clip_gradients(grads, max_norm)
        assert torch.equal(n, got)
        check_clipped(clipped, grads, norm, max_norm)
        given, n2 = ops.clip_gradients(grads, max_norm, norm=got)
        assert n2 is got and all(torch.equal(a, b) for a, b in zip(given, clipped))
        own = [g.clone() for g in grads]
        same, _ = ops.clip_gradients(own, max_norm, out=own)
        assert same is own and all(torch.equal(a, b) for a, b in zip(own, clipped))


def test_clip_many_tensors():
    """More tensors than a launch takes, of every alignment."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    for dtype in DTYPES:
        flat = torch.randn(400000, generator=gen, device="cuda").to(dtype)
        sizes = [1 + 37 * i % 1999 for i in range(390)]
        grads = list(flat[:sum(sizes)].split(sizes))
        norm = exact_norm(grads)
        assert abs(float(ops.gradient_norm(grads)) - norm) <= norm * 2.0 ** -24
        rest = torch.full_like(flat, 3.0)
        out = list(rest[5:5 + sum(sizes)].split(sizes))
        ops.clip_gradients(grads, 1.0, out=out)
        check_clipped(out, grads, norm, 1.0)
        assert (rest[:5] == 3).all() and (rest[5 + sum(sizes):] == 3).all()


def test_clip_over_the_whole_range():
    """Gradients whose squares a float does not hold."""
    for scale in (1e25, 1e-30):
        g = torch.randn(10001, device="cuda") * scale
        norm = float(g.double().square().sum().sqrt())
        assert abs(float(ops.gradient_norm([g])) - norm) <= norm * 2.0 ** -24
    clipped, _ = ops.clip_gradients([torch.full((5,), 1e30, device="cuda")], 1.0)
    assert (clipped[0] - 5 ** -0.5).abs().max() <= 4 * 2.0 ** -24
    big = torch.full((3, 4), 300.0, device="cuda", dtype=torch.float16)
    assert abs(float(ops.gradient_norm([big])) - 300 * 12 ** 0.5) <= 300 * 12 ** 0.5 * 2.0 ** -24


def test_clip_of_no_numbers():
    a, b = torch.ones(4, device="cuda"), torch.ones(5, device="cuda", dtype=torch.bfloat16)
    a[2] = float("nan")
    clipped, norm = ops.clip_gradients([a, b], 1.0)
    assert norm.isnan() and all(c.isnan().all() for c in clipped)
    a[2] = float("inf")
    clipped, norm = ops.clip_gradients([a, b], 1.0)
    assert norm.isinf() and clipped[0][2].isnan() and (clipped[0][:2] == 0).all() and (clipped[1] == 0).all()
    empty, norm = ops.clip_gradients([torch.empty(0, device="cuda")], 1.0)
    assert norm == 0 and empty[0].numel() == 0


def test_clip_of_orders_and_overlaps():
    a = torch.randn(6, 4, 5, device="cuda")
    turned = a.permute(2, 0, 1)
    clipped, norm = ops.clip_gradients([turned], 1.0)
    assert clipped[0].stride() == turned.stride()
    check_clipped(clipped, [turned], exact_norm([turned]), 1.0)
    for bad in ([a[:, :3]], [a[:1].expand(6, 4, 5)], [a, a.cpu()]):
        with pytest.raises(ValueError):
            ops.gradient_norm(bad)
    assert abs(float(ops.gradient_norm([a, a])) - exact_norm([a]) * 2 ** 0.5) <= exact_norm([a]) * 1e-6
    flat = torch.randn(100, device="cuda")
    for grads, out in (([a, a], [a, a]), ([flat[:50], flat[50:]], [flat[50:], flat[:50]]), ([flat[:50], flat[40:90]], [flat[:50], flat[40:90]]),
                       ([flat[:50]], [flat[1:51]]), ([flat[:10], flat[20:30]], [torch.empty(10, device="cuda"), flat[5:15]])):
        before = flat.clone()
        with pytest.raises((ValueError, lib.HasteHipError)):
            ops.clip_gradients(grads, 1.0, out=out)
        assert torch.equal(before, flat)
    for out in ([torch.empty(5, device="cuda")], [torch.empty(10, device="cuda", dtype=torch.float16)], [], [torch.empty(20, device="cuda")[::2]]):
        with pytest.raises(ValueError):
            ops.clip_gradients([flat[:10]], 1.0, out=out)


def test_clip_many_large_tensors():
    """More parts of the norm than a workgroup adds up for itself, in two lists, and a tensor of more than 2^31 elements."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    for sizes in ([300001] * 130, [2 ** 31 + 16411, 77]):
        grads = [torch.randn(n, generator=gen, device="cuda", dtype=torch.bfloat16) for n in sizes]
        norm = math.sqrt(math.fsum(float(p.double().square().sum()) for g in grads for p in g.split(1 << 28)))
        got = ops.gradient_norm(grads)
        assert abs(float(got) - norm) <= norm * 2.0 ** -24
        kept = [(g[:5000].clone(), g[-5000:].clone()) for g in grads]
        same, n = ops.clip_gradients(grads, 2.0, out=grads)
        assert same is grads and torch.equal(n, got)
        for g, (head, tail) in zip(grads, kept):
            check_clipped([g[:5000], g[-5000:]], [head, tail], norm, 2.0)


# ---- order, streams, graphs, a run of all ------------------------------------------------
def all_three(seed, dtype=torch.bfloat16):
    linear, gated = linear_problem(seed, dtype, (140, 3), 72, 96, "silu"), gated_problem(seed + 1, dtype, 140, 3, 96)
    long = gated_problem(seed + 2, dtype, 900, 1, 64)
    tall = linear_problem(seed + 3, dtype, (2000,), 64, 64, "gelu")  # sums over rows in pieces

    def run():
        out = {}
        for name, values in (("linear", run_linear(linear.g)), ("gated", run_gated(gated.g)), ("long", run_gated(long.g)), ("tall", run_linear(tall.g))):
            out.update({name + " " + k: v for k, v in values.items()})
        grads = [out[k] for k in ("linear dkernel", "linear dbias", "gated ddecay", "gated dforget_bias", "tall dkernel")]
        clipped, norm = ops.clip_gradients(grads, 0.1)
        out.update({"clipped %d" % i: c for i, c in enumerate(clipped)}, norm=norm)
        return out
    return run


def same(a, b):
    return all(torch.equal(a[k], b[k]) for k in a)


def test_repeated_calls_give_the_same_bits():
    for dtype in DTYPES:
        run = all_three(20, dtype)
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=short)
def test_graphs(dtype):
    """Two graphs of all the operators, replayed in turn with eager calls between."""
    runs = [all_three(50, dtype), all_three(60, dtype)]
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


class Block(torch.nn.Module):
    """A gated linear recurrent block: projections to the gates and back, its norm and residual."""

    def __init__(self, width, inner, decay=True, batch_first=False):
        super().__init__()
        self.norm = haste_amd.ResidualNorm(width, norm_after=False, scale=None)
        self.into = haste_amd.Linear(width, 4 * inner)
        self.recur = haste_amd.GatedRecurrence(inner, decay, batch_first=batch_first)
        self.back = haste_amd.Linear(inner, width, bias=False)
        self.up, self.down = haste_amd.Linear(width, 2 * width, activation="gelu"), haste_amd.Linear(2 * width, width)

    def forward(self, x, state=None, lengths=None, step=False):
        _, normed = self.norm(x)
        u, f, a, z = self.into(normed).chunk(4, -1)
        y, state = self.recur.step(u, f, a, z, state) if step else self.recur(u, f, a, z, state, lengths)
        x = self.back(y, x)
        return self.down(self.up(x), x), state


@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("lengths", [None, [33, 0, 7]])
def test_block_trains_like_its_plain_form(lengths, decay):
    """The fused layers against the layers' own plain form in float64 on the CPU: values, every gradient, and these clipped."""
    torch.manual_seed(1)
    block, plain = Block(24, 40, decay), Block(24, 40, decay).double()
    plain.load_state_dict(block.state_dict())
    block = block.cuda()
    x = torch.randn(33, 3, 24)
    results = []
    for model, to in ((block, lambda t: t.cuda()), (plain, lambda t: t.double())):
        xi = to(x.clone()).requires_grad_()
        outs = model(xi, None, lengths)
        torch.manual_seed(2)
        torch.autograd.backward(outs, [to(torch.randn(o.shape)) for o in outs])
        grads = [p.grad.detach().clone() for p in [xi, *model.parameters()]]
        norm = haste_amd.clip_gradients_(model.parameters(), 0.5)
        results.append([t.detach().cpu().double() for t in (*outs, *grads, norm, *[p.grad for p in model.parameters()])])
    # float32 products of up to 99 terms on both sides of the operators; relative to the largest value
    for got, want in zip(*results):
        assert (got - want).abs().max() <= 2e-5 * max(1.0, float(want.abs().max()))
    assert abs(float(torch.stack([g.square().sum() for g in results[0][-len(list(plain.parameters())):]]).sum().sqrt()) - 0.5) <= 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=short)
def test_block_steps_like_it_runs(dtype):
    torch.manual_seed(3)
    block = Block(24, 40).cuda().to(dtype)
    x = torch.randn(19, 2, 24, device="cuda").to(dtype)
    with torch.no_grad():
        out, h = block(x)
        hs, outs = None, []
        for t in range(19):
            o, hs = block(x[t], hs, step=True)
            outs.append(o)
    # a projection's sums may be added in another order for other sizes: a step of the type, and what follows from it
    tolerance = 64 * torch.finfo(dtype).eps
    assert (torch.stack(outs).float() - out.float()).abs().max() <= tolerance * out.float().abs().max()
    assert (hs - h).abs().max() <= tolerance * h.abs().max()
    assert h.dtype == torch.float32 and out.dtype == dtype


def test_layers_batch_first_and_half_parameters():
    torch.manual_seed(4)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        a, b = Block(16, 24).cuda().to(dtype), Block(16, 24, batch_first=True).cuda().to(dtype)
        b.load_state_dict(a.state_dict())
        x = torch.randn(9, 3, 16, device="cuda").to(dtype).requires_grad_()
        first = x.detach().transpose(0, 1).contiguous().requires_grad_()
        results = []
        for model, given in ((a, x), (b, first)):
            y, h = model(given, None, [9, 4, 2])
            grads = torch.autograd.grad([y, h], [given, *model.parameters()], [torch.ones_like(y), torch.ones_like(h)])
            assert all(g.dtype == t.dtype for g, t in zip(grads, [given, *model.parameters()]))
            results.append((y, h, grads))
        (y, h, grads), (y2, h2, grads2) = results
        assert torch.equal(y2.transpose(0, 1), y) and torch.equal(h, h2) and torch.equal(grads2[0].transpose(0, 1), grads[0])


def test_layers_in_mixed_precision_and_frozen():
    """float parameters under bfloat16 activations, and leaves that want no gradient."""
    torch.manual_seed(5)
    block = Block(16, 24).cuda()
    x = torch.randn(9, 3, 16, device="cuda", dtype=torch.bfloat16)
    block.up.kernel.requires_grad_(False)
    y, _ = block(x)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert block.up.kernel.grad is None and block.into.kernel.grad.dtype == torch.float32
    assert all(p.grad is not None and p.grad.dtype == p.dtype for n, p in block.named_parameters() if n != "up.kernel")
    for p in block.parameters():
        p.requires_grad_(False)
    x.requires_grad_()
    block(x)[0].float().sum().backward()
    assert x.grad.dtype == torch.bfloat16 and x.grad.isfinite().all()


def test_backward_twice_and_refused_second_derivatives():
    torch.manual_seed(6)
    block = Block(16, 24).cuda()
    x = torch.randn(40, 2, 16, device="cuda", requires_grad=True)
    loss = block(x)[0].square().sum()
    leaves = [x, *block.parameters()]
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    second = torch.autograd.grad(loss, leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError):
        second[0].sum().backward()


def test_a_training_step_in_a_graph():
    """Forward pass, backward pass and clipping of a block, captured and replayed between eager steps."""
    torch.manual_seed(7)
    block = Block(16, 24).cuda()
    x = torch.randn(50, 3, 16, device="cuda")
    parameters = list(block.parameters())

    def step():
        y, _ = block(x)
        grads = torch.autograd.grad(y, parameters, torch.ones_like(y))
        return ops.clip_gradients(grads, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, norm = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        clipped, total = step()
    for replay in range(4):
        total.zero_()
        graph.replay()
        again, norm2 = step()
        torch.cuda.synchronize()
        assert torch.equal(total, norm) and torch.equal(norm2, norm)
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, clipped, again))
