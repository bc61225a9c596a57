"""Which sizes and rows the operators of a gated linear recurrent block take, without a GPU: a call that is taken gets as far as its
first launch, which finds no device."""
import ctypes
import math
import random

import pytest
import torch

from haste_amd import lib, ops

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls with addresses of nothing, for machines on which nothing is launched")
INVALID, UNSUPPORTED, RUNTIME = 1, 2, 3


def _bytes(name, *sizes):
    fn = lib.load()[name]
    fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_int] * len(sizes)
    return fn(*sizes)


def _linear_bytes(backward, sfx, R, C, D, x_row):
    element = 4 if sfx == "_f32" else 2
    return _bytes("haste_hip_linear_workspace_bytes", backward, element, R, C, D, int((x_row or C) * element % 16 == 0))


def _forward(sfx, R, C, D, x_row=None, x=2 ** 12, kernel=2 ** 13, workspace=2 ** 14, size=None):
    """The code of a projection whose caller has as much scratch memory as is said to be needed (or `size` bytes)."""
    size = _linear_bytes(0, sfx, R, C, D, x_row) if size is None else size
    return lib.entry("haste_hip_linear_forward" + sfx)(R, C, D, x, x_row or C, kernel, None, 0, None, 0, 2 ** 15, None, workspace, size, None)


def _backward(sfx, R, C, D, x_row=None, dy_row=None, dx=2 ** 15, dkernel=2 ** 16, size=None):
    size = _linear_bytes(1, sfx, R, C, D, x_row) if size is None else size
    return lib.entry("haste_hip_linear_backward" + sfx)(R, C, D, 2 ** 12, x_row or C, 2 ** 13, 0, None, 2 ** 17, dy_row or D, dx, dkernel, None,
                                                        2 ** 14, size, None)


# ---- rows far apart, and long ones ----------------------------------------------------
@pytest.mark.parametrize("sfx", ["_f32", "_bf16"])
def test_long_rows_are_taken(sfx):
    """2^20 columns and rows 2^22 elements apart, whichever kernel a product goes by."""
    for sizes in (dict(R=2048, C=1024, D=600000), dict(R=2048, C=1024, D=4096, x_row=2 ** 22), dict(R=200, C=4096, D=4096, x_row=2 ** 22),
                  dict(R=2048, C=4096, D=2 ** 20), dict(R=2048, C=2 ** 20, D=1024, x_row=2 ** 22)):
        assert _forward(sfx, **sizes) == RUNTIME, sizes
    for sizes in (dict(R=2048, C=1024, D=600000), dict(R=2048, C=600000, D=1024), dict(R=2048, C=1024, D=4096, x_row=600000),
                  dict(R=4096, C=1024, D=4096, dy_row=600000), dict(R=200, C=4096, D=4096, x_row=4096000),
                  dict(R=2048, C=2 ** 20, D=1024, x_row=2 ** 22, dy_row=2 ** 22), dict(R=157, C=4096, D=4096, x_row=3000000)):
        assert _backward(sfx, **sizes, dx=None) == RUNTIME, sizes
        assert _backward(sfx, **sizes, dkernel=None) == RUNTIME, sizes


def test_products_of_long_rows_are_taken():
    """The float product by itself: short runs of a contraction, tiles whose rows are 2^22 apart."""
    product = lib.entry("haste_hip_gemm_f32")
    for trans_a, M, N, K, lda, ldb in ((0, 2048, 600000, 1024, 1024, 600000), (0, 2048, 4096, 1024, 2 ** 22, 4096), (0, 300, 2 ** 20, 4096, 4096, 2 ** 20),
                                       (0, 128, 128, 2 ** 20, 2 ** 22, 128), (1, 1024, 4096, 200, 2 ** 22, 4096),
                                       (1, 1024, 4096, 100000, 1024, 2 ** 22), (1, 600000, 64, 2048, 600000, 64)):
        assert product(trans_a, M, N, K, 2 ** 12, lda, 2 ** 13, ldb, 2 ** 15, N, 0, None) == RUNTIME, (trans_a, M, N, K, lda, ldb)
    assert product(0, 128, 128, 2 ** 20, 2 ** 12, 2 ** 22 + 2 ** 20, 2 ** 13, 128, 2 ** 15, 128, 0, None) == UNSUPPORTED


def test_scratch_memory_is_enough_for_every_run():
    """Rows so far apart that a contraction is cut: a run may want more pieces than the whole."""
    for R, C, D, x_row, dy_row in ((2550, 192, 2700, 237495, 2700), (16427, 128, 2112, 37069, 2112), (2550, 2700, 192, 2700, 237495)):
        assert _backward("_f32", R, C, D, x_row, dy_row, dx=None) == RUNTIME, (R, C, D, x_row, dy_row)
    gen = random.Random(1)
    size = lambda low, high: round(math.exp(gen.uniform(math.log(low), math.log(high))))  # noqa: E731
    for _ in range(4000):
        R, C, D = size(128, 40000), size(64, 4096), size(64, 4096)
        x_row, dy_row = size(C, 2 ** 22), size(D, 2 ** 22)
        if min(x_row, dy_row) * R < 2 ** 40:
            assert _backward("_f32", R, C, D, x_row, dy_row, dx=None) == RUNTIME, (R, C, D, x_row, dy_row)
            assert _forward("_f32", R, C, D, x_row) == RUNTIME, (R, C, D, x_row)


@pytest.mark.parametrize("sfx", ["_f32", "_f16", "_bf16"])
def test_scratch_memory_of_a_single_row(sfx):
    """x and the kernel at 16 bytes: how far the next row would be makes no difference."""
    for C, D, x_row in ((77, 992, 80), (80, 992, 80), (77, 992, 77), (77, 991, 88), (4097, 64, 4104)):
        for backward, call in ((0, _forward), (1, _backward)):
            size = _bytes("haste_hip_linear_workspace_bytes", backward, 4 if sfx == "_f32" else 2, 1, C, D, 1)
            assert call(sfx, 1, C, D, x_row, size=size) == RUNTIME, (backward, C, D, x_row)


@pytest.mark.parametrize("shape", [(2 ** 30 + 1,), (2 ** 16 + 1, 2 ** 16), (2 ** 20, 2 ** 11), (5, 2 ** 32 // 5 + 1)])
def test_more_rows_than_are_counted_are_refused(shape):
    """Steps times batch rows, each of which is in range: not to be taken for what is left of their product in 32 bits."""
    x, kernel = torch.zeros(1, 1).expand(*shape, 1), torch.zeros(1, 4)
    with pytest.raises(ValueError, match="rows"):
        ops.linear_forward(False, x, kernel)
    with pytest.raises(ValueError, match="rows"):
        ops.linear_backward(x, kernel, None, "none", None, x.expand(*shape, 4))


def test_more_gradients_than_the_norm_has_scratch_memory_for_are_refused():
    """Where the size of the scratch memory is said to be 0.  (No gradient has elements: nothing would be written if it went on.)"""
    size = lambda count: _bytes("haste_hip_gradient_norm_workspace_bytes", count)  # noqa: E731
    most = 7340032
    assert size(most) > 0 and size(most + 1) == 0
    none = (ctypes.c_void_p * (most + 1))(), (ctypes.c_size_t * (most + 1))(), (ctypes.c_int * (most + 1))()
    norm = lambda count: lib.entry("haste_hip_gradient_norm")(count, *none, 64, 0, 256, size(count), None)  # noqa: E731
    clip = lambda count, given: lib.entry("haste_hip_clip_gradients")(count, none[0], *none, 1.0, given, 64, 0, 256, size(count), None)  # noqa: E731
    assert norm(most) == RUNTIME and norm(most + 1) == UNSUPPORTED
    assert clip(most, 0) == RUNTIME and clip(most + 1, 0) == UNSUPPORTED
    assert clip(most + 1, 1) == 0  # the norm is there, and nothing to scale
