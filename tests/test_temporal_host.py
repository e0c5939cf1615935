"""Refusals of the temporal head's C entry points and modules that need no GPU."""
import ctypes

import pytest
import torch

from tempo_amd import _lib

P = ctypes.c_void_p
ONE = P(16)  # never dereferenced: every call here must fail validation first


def test_recurrence_entry_points_reject_bad_arguments():
    lib = _lib.load()

    def forward(**kw):
        g = kw.get
        return lib.tempo_recurrence(
            g('gate', ONE), 8, 8, g('value', ONE), 8, 8, g('state', None), g('lengths', None),
            g('h', ONE), 8, 8, g('last', None), g('ckpt', None), g('B', 2), g('T', 5),
            g('D', 8), g('dtype', 0), g('ws', ONE), g('bytes', 1 << 40), None)

    def backward(**kw):
        g = kw.get
        return lib.tempo_recurrence_backward(
            g('gate', ONE), 8, 8, g('value', ONE), 8, 8, g('grad', ONE), 8, 8, None, None,
            g('ckpt', ONE), g('dgate', ONE), 8, 8, g('dvalue', ONE), 8, 8, g('dstate', None),
            g('B', 2), g('T', 5), g('D', 8), g('dtype', 0), g('ws', ONE), g('bytes', 1 << 40),
            None)

    for name in ('gate', 'value', 'h'):
        assert forward(**{name: None}) == -1
    for name in ('gate', 'value', 'grad', 'dgate', 'dvalue'):
        assert backward(**{name: None}) == -1
    assert backward(ckpt=None, T=17) == -1
    for call in (forward, backward):
        assert call(B=0) == -2 and call(T=0) == -2 and call(D=0) == -2 and call(B=-1) == -2
        assert call(dtype=3) == -5 and call(dtype=-1) == -5
        assert call(gate=P(18)) == -5 and call(value=P(17), dtype=1) == -5
        assert call(B=1 << 31, D=4) == -4 and call(B=1 << 30, D=64) == -4
        assert call(T=5000, ws=None) == -1 and call(T=5000, bytes=8) == -4
        assert call(T=5000, ws=P(18)) == -5
    assert forward(state=P(18)) == -5 and forward(last=P(18)) == -5
    assert forward(lengths=P(18)) == -5 and forward(ckpt=P(18)) == -5
    assert backward(dstate=P(18)) == -5


def test_recurrence_workspace():
    lib = _lib.load()
    ws = lib.tempo_recurrence_workspace
    assert ws(0, 5, 8, 0, 0) == -2 and ws(1, 5, 8, 9, 0) == -5
    assert ws(1, 1, 8, 0, 0) == 0 and ws(1 << 20, 40, 64, 0, 1) == 0  # time is not cut
    for backward in (0, 1):
        need = ws(1, 65536, 1024, 2, backward)
        # (A, U) in fp32 per channel and chunk, a fraction of the sequence itself
        assert 0 < need <= 65536 * 1024 * 2 // 2 and need % 8 == 0


def test_no_cpu_path():
    import tempo_amd
    x = torch.zeros(2, 3, 8)
    with pytest.raises(TypeError):
        tempo_amd.gated_recurrence(x, x)
    with pytest.raises(TypeError):
        tempo_amd.fused_linear(x, torch.zeros(4, 8))


def test_linear_entry_points_reject_bad_arguments():
    lib = _lib.load()

    def forward(**kw):
        g = kw.get
        return lib.tempo_linear(
            g('x', ONE), g('ldx', 64), g('weight', ONE), g('ldw', 64), g('bias', None),
            g('residual', None), g('ldr', 16), g('y', ONE), g('ldy', 16), g('pre', None),
            g('M', 4), g('N', 16), g('K', 64), g('dtype', 0), g('act', 0), g('ws', ONE),
            g('bytes', 1 << 40), None)

    def backward(**kw):
        g = kw.get
        return lib.tempo_linear_backward(
            g('grad', ONE), g('ldg', 16), g('pre', None), g('x', ONE), g('ldx', 64),
            g('weight', ONE), g('ldw', 64), g('dx', ONE), g('lddx', 64), g('dw', ONE),
            g('db', ONE), g('M', 4), g('N', 16), g('K', 64), g('dtype', 0), g('act', 0),
            g('ws', ONE), g('bytes', 1 << 40), None)

    for name in ('x', 'weight', 'y'):
        assert forward(**{name: None}) == -1
    for name in ('x', 'weight', 'grad', 'ws'):
        assert backward(**{name: None}) == -1
    assert backward(act=1) == -1  # its z is missing
    for call in (forward, backward):
        assert call(M=0) == -2 and call(N=0) == -2 and call(K=-1) == -2
        assert call(dtype=3) == -5 and call(act=6) == -5 and call(act=-1) == -5
        assert call(x=P(18)) == -5 and call(weight=P(17), dtype=2) == -5
        assert call(M=1 << 32) == -4 and call(N=1 << 21) == -4 and call(K=1 << 21) == -4
        assert call(ldx=-1) == -5 and call(ldw=-1) == -5
        assert call(ws=P(24), K=65536, M=100, bytes=1 << 40) == -5
        assert call(K=65536, M=100, bytes=8, lddx=65536) == -4
    assert forward(K=65536, M=100, ws=None) == -1
    assert forward(ldy=15) == -5 and backward(lddx=63) == -5 and backward(ldg=-1) == -5
    for name in ('y', 'bias', 'residual', 'pre'):
        assert forward(**{name: P(18)}) == -5
    for name in ('grad', 'dx', 'dw', 'db'):
        assert backward(**{name: P(18)}) == -5
    assert backward(pre=P(18), act=1) == -5


def test_linear_workspace():
    ws = _lib.load().tempo_linear_workspace
    assert ws(0, 1, 1, 0, 0, 0) == -2 and ws(1, 1, 1, 7, 0, 0) == -5
    assert ws(1, 1, 1, 0, 9, 0) == -5 and ws(1, 1 << 21, 1, 0, 0, 0) == -4
    assert ws(16384, 4096, 4096, 2, 0, 0) == 0  # tiles enough: the sum is not split
    assert ws(8192, 4096, 1024, 2, 3, 1) >= 8192 * 4096 * 2  # dz


def test_linear_grid_limit():
    """A product of more tiles than a launch can hold is refused by size, one below it is not."""
    workspace = _lib.load().tempo_linear_workspace
    for dtype in (0, 1, 2):
        assert workspace((1 << 31) - 1, 100, 8, dtype, 0, 0) == -4   # 2^24 tiles of 128 rows
        assert workspace((1 << 31) - 1, 100, 8, dtype, 0, 1) > 0     # 8 columns: a fixed grid
        assert workspace((1 << 31) - 1, 8, 100, dtype, 0, 0) == 0
        assert workspace((1 << 31) - 1, 8, 100, dtype, 0, 1) == -4   # dx has 100
        assert workspace(1 << 30, 100, 8, dtype, 0, 0) == 0          # 2^23


def test_results_apart_from_inputs():
    """Shared memory is told by addresses alone: exactly, against the sets of elements."""
    from tempo_amd import ops
    buf = torch.zeros(64)
    views = [torch.as_strided(buf, shape, stride, offset) for offset in (0, 1, 4, 6, 24)
             for shape, stride in (((2, 3, 4), (12, 4, 1)), ((2, 3, 2), (12, 4, 1)),
                                   ((2, 3, 2), (2, 4, 1)), ((3, 2, 2), (4, 12, 1)),
                                   ((1, 1, 8), (5, 3, 1)), ((1, 3, 1), (7, 8, 9)))]

    def elements(t):
        return set(torch.arange(64).as_strided(t.shape, t.stride(), t.storage_offset())
                   .flatten().tolist())

    told = 0
    for a in views:
        for b in views:
            shared = elements(a) & elements(b)
            try:
                ops._apart('out', a, x=b)
                assert not shared
                told += elements(b) & set(range(min(elements(a)), max(elements(a)))) != set()
            except ValueError:
                pass  # may be refused without need, too: only if their rows interleave
            if max(elements(a)) < min(elements(b)) or max(elements(b)) < min(elements(a)):
                ops._apart('out', a, x=b)
    assert told > 20  # interleaved and apart: accepted
    ops._apart('out', views[0][:0], x=views[0])
    ops._apart('out', views[0], x=views[0][:0], weight=None)


def test_rows_of_a_result_apart():
    from tempo_amd import ops
    buf = torch.zeros(400)
    for shape, stride in (((3, 5, 6), (30, 6, 1)), ((3, 5, 6), (6, 18, 1)), ((1, 5, 6), (0, 6, 1)),
                          ((3, 1, 6), (6, 0, 1)), ((0, 5, 6), (0, 6, 1)), ((4, 1), (1, 9))):
        ops._rows_apart('out', torch.as_strided(buf, shape, stride))
    for stride in ((0, 6, 1), (30, 0, 1), (29, 6, 1), (30, 5, 1), (6, 17, 1)):
        with pytest.raises(ValueError):
            ops._rows_apart('out', torch.as_strided(buf, (3, 5, 6), stride))


def test_recurrent_process_layer_refusals():
    """Before any kernel: counts that divide nothing, other ranks and channels."""
    import tempo_amd
    head = tempo_amd.RecurrentProcessLayerNHWC(8, 4)
    maps = torch.zeros(6, 8, 3, 5)
    for bad in (lambda: head(maps, 0), lambda: head(maps, 3, 0), lambda: head(maps, -3, -2),
                lambda: head(maps, -6), lambda: head(maps, 4), lambda: head(maps, 3, 4),
                lambda: head(maps[0], 1), lambda: head(maps[:, :7], 3, 2), lambda: head(None, 1)):
        with pytest.raises(ValueError):
            bad()


def test_arguments_that_are_no_tensors():
    import tempo_amd
    x = torch.zeros(2, 3, 8)
    for bad in (lambda: tempo_amd.fused_linear([1.0, 2.0], x[0]),
                lambda: tempo_amd.fused_linear(x.numpy(), x[0]),
                lambda: tempo_amd.fused_linear(None, None),
                lambda: tempo_amd.gated_recurrence([1.0, 2.0], x),
                lambda: tempo_amd.gated_recurrence(x.numpy(), x.numpy()),
                lambda: tempo_amd.gated_recurrence(None)):
        with pytest.raises(TypeError):
            bad()
