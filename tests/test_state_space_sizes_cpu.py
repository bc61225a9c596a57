"""Which sizes the state space operators take, without a GPU: nothing is read, nothing launched."""
import ctypes

from haste_amd import lib

UNSUPPORTED = 2


def _refusal(name, *values):
    """The code and the reason of a call that is refused."""
    code = lib.entry(name)(*values, None)
    return code, lib.load().haste_hip_last_runtime_error().decode()


def _scan_backward(T, N, D, S, G, workspace_bytes):
    ins = [256, N * D, D, 256, N * D, D, 256, 256, N * G * S, G * S, 256, N * G * S, G * S, None, None, 0, 0, None, 1]
    return _refusal("haste_hip_selective_scan_backward_bf16", T, N, D, S, G, *ins, None, 256, 256, N * D, D, None, 256, 256, 256, 256,
                    256, None, None, None, None, 256, workspace_bytes)


def test_backward_scans_have_no_limit_of_their_own():
    """T N G S of 2^30 and more, which the forward pass takes: the small workspace is all that is wrong."""
    for sizes in ((2048, 8, 4096, 16, 4096), (1024, 8, 2048, 64, 2048), (8192, 64, 64, 64, 32)):
        assert sizes[0] * sizes[1] * sizes[3] * sizes[4] >= 2 ** 30
        code, reason = _scan_backward(*sizes, 64)
        assert code == UNSUPPORTED and "workspace is too small" in reason, (sizes, reason)


def _bytes(name, *sizes):
    fn = lib.load()[name]
    fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_int] * len(sizes)
    return fn(*sizes)


def test_workspaces_of_more_than_2_31_partials():
    """Runs of 64 steps or fewer times rows: counted in more than 32 bits."""
    T, N, D, W = 320, 2 ** 30 - 256, 1, 4
    assert _bytes("haste_hip_causal_conv_workspace_bytes", T, N, D, W) >= T // 64 * N * (W + 1) * D * 4


def test_workspaces_of_sizes_that_are_refused_are_0():
    """More workgroups than a grid has."""
    conv, scan = (64, 2 ** 22, 2 ** 12, 4), (64, 2 ** 20, 64, 16, 8)
    assert _bytes("haste_hip_causal_conv_workspace_bytes", *conv) == 0
    code, reason = _refusal("haste_hip_causal_conv_backward_f32", *conv, 256, 0, 0, 256, None, 1, None, None, 256, 0, 0, None, 256, 256,
                            None, None, 256, 2 ** 62)
    assert code == UNSUPPORTED and "too many rows" in reason
    assert _bytes("haste_hip_selective_scan_workspace_bytes", 0, *scan) == _bytes("haste_hip_selective_scan_workspace_bytes", 1, *scan) == 0
    code, reason = _scan_backward(*scan, 2 ** 62)
    assert code == UNSUPPORTED and "too many rows" in reason
    # one row less is taken
    assert _bytes("haste_hip_selective_scan_workspace_bytes", 1, 64, 2 ** 19 - 1, 64, 16, 8) > 0
    assert _bytes("haste_hip_causal_conv_workspace_bytes", 64, 2 ** 20 - 1, 2 ** 12, 4) > 0
