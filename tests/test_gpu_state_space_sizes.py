"""The state space block's operators at sizes beyond those of one grid, one workgroup or one turn."""
import pytest
import torch

from haste_amd import ops

import state_space_formulas as formulas
from test_gpu_state_space import Problem, compare, run_scan, scan_problem

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
