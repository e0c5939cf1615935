"""Which kernel and tiles the fused linear layer's products select, built for the CPU from the code
that the library runs: the GPU tests' sizes reach each of them, in every operand order."""
import ctypes

import pytest

import test_gpu_linear as L

KERNELS = ('FEW', 'THIN', 'TILE', 'STREAM', 'STREAM_32x256', 'STREAM_256')
FP32, FP16 = 0, 1


def _products(plan, M, K, N, dtype):
    """name -> (kernel, xi, xj, ti, tj, split) of contiguous tensors of one training step."""
    size = 4 if dtype == FP32 else 2
    got = {}
    for name, I, J, k, a, b in (('y', M, N, K, 0, 0), ('dx', M, K, N, 0, 1),
                                ('dweight', N, K, M, 1, 1)):
        direct = all(plan.emul_streamable(0, rows if layout else k, layout, rows, k, size)
                     for layout, rows in ((a, I), (b, J)))
        out = (ctypes.c_longlong * 6)()
        assert plan.emul_plan_product(I, J, k, a, b, dtype, direct, out)
        got[name] = (KERNELS[out[0]],) + tuple(out[1:])
    return got


def _sizes(test):
    """The (M, K, N) that a GPU test runs over."""
    for mark in test.pytestmark:
        if mark.name == 'parametrize' and mark.args[0] in ('shape', 'M,K,N'):
            yield from (s[:3] for s in mark.args[1])


@pytest.mark.parametrize('shape', L.WIDEST, ids=str)
def test_widest_tiles_are_selected(shape, linear_plan):
    M, K, N, name = shape
    kernel, _, _, ti, tj, split = _products(linear_plan, M, K, N, FP16)[name]
    assert (kernel, split) == ('STREAM_256', 1) and ti * tj >= 256
    assert M % 256 and N % 256 and K % 256


def test_every_kernel_is_tested(linear_plan):
    tests = [L.test_gradients, L.test_tile_shapes, L.test_many_rows_of_few_channels,
             L.test_more_rows_of_few_channels]
    seen = {FP32: set(), FP16: set()}
    for dtype, more in ((FP32, [L.test_narrow_tiles]),
                        (FP16, [L.test_widest_tiles, L.test_more_tiles_than_compute_units])):
        for test in tests + more:
            for M, K, N in _sizes(test):
                for name, p in _products(linear_plan, M, K, N, dtype).items():
                    tiles = p[1:3] if p[0] in ('TILE', 'STREAM') else ()
                    seen[dtype].add((p[0],) + tiles + (name,))
    for dtype in seen:
        want = {(k, xi, xj, name) for k in ('TILE', 'STREAM') for xi in (1, 2) for xj in (1, 2)
                for name in ('y', 'dx', 'dweight')}
        want |= {('FEW', 'y'), ('THIN', 'y'), ('THIN', 'dx'), ('STREAM_32x256', 'dweight')}
        if dtype == FP16:
            want |= {('STREAM_256', name) for name in ('y', 'dx', 'dweight')}
        assert not want - seen[dtype], want - seen[dtype]


def test_scratch_memory_covers_either_kernel(linear_plan):
    """It is planned from sizes, before the operands' alignment is known."""
    for M, K, N in list(_sizes(L.test_tile_shapes)) + list(L.SHAPES):
        for dtype in (FP32, FP16):
            for I, J, k, a, b in ((M, N, K, 0, 0), (M, K, N, 0, 1), (N, K, M, 1, 1)):
                room = linear_plan.emul_product_bytes(I, J, k, a, b, dtype)
                for direct in (0, 1):
                    out = (ctypes.c_longlong * 6)()
                    assert linear_plan.emul_plan_product(I, J, k, a, b, dtype, direct, out)
                    assert out[5] == 1 or room >= out[5] * I * J * 4
