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
