"""The gated linear recurrence against its formula in 64 bits, step by step on the CPU:
types, lengths from one step to thousands, odd widths, layouts, padded batches, gradients."""
import pytest
import torch

import temporal_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# (B, T, D): one step; fewer channels than a vector; odd widths; a span and its neighbours;
# lengths at the border to cut time; many lanes with few steps; long with few lanes
SHAPES = [(1, 1, 1), (10, 1, 512), (2, 3, 7), (3, 16, 33), (2, 17, 64), (5, 4, 30),
          (1, 64, 5), (2, 65, 96), (3, 333, 77), (1, 2049, 20), (2, 1000, 256),
          (40000, 4, 16), (9000, 21, 9)]


def _inputs(B, T, D, dtype, dev, layout='plain', seed=0, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    gate = torch.randn(B, T, D, generator=gen) * spread
    value = torch.randn(B, T, D, generator=gen)
    gate, value = gate.to(dtype).to(dev), value.to(dtype).to(dev)
    if layout == 'time_major':
        gate, value = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (gate, value))
    elif layout == 'odd_rows':  # rows at odd element offsets inside larger rows
        wide = [torch.full((B, T, D + 3), float('nan'), dtype=dtype, device=dev)
                for _ in range(2)]
        for w, t in zip(wide, (gate, value)):
            w[..., 1:1 + D] = t
        gate, value = (w[..., 1:1 + D] for w in wide)
    return gate, value


def _states(B, D, dev, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(B, D, generator=gen).to(dev), torch.randn(B, D, generator=gen).to(dev))


def _lengths(B, T, dev, seed=2):
    gen = torch.Generator().manual_seed(seed)
    n = torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32)
    n[0] = T
    if B > 1:
        n[1] = 0
    if B > 2:
        n[2] = 1
    return n.to(dev)


def _train(dev, gate, value, state, lengths, grad_h, grad_last, combined=False):
    import tempo_amd
    leaves = {}
    if combined:
        leaves['gate'] = torch.cat([gate, value], dim=-1).requires_grad_(True)
        args = (leaves['gate'], None)
    else:
        leaves['gate'] = gate.detach().requires_grad_(True)
        leaves['value'] = value.detach().requires_grad_(True)
        args = (leaves['gate'], leaves['value'])
    if state is not None:
        leaves['state'] = state.detach().requires_grad_(True)
    h, last = tempo_amd.gated_recurrence(*args, state=leaves.get('state'), lengths=lengths)
    outs, seeds = [], []
    if grad_h is not None:
        outs.append(h), seeds.append(grad_h)
    if grad_last is not None:
        outs.append(last), seeds.append(grad_last)
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), seeds)))
    if combined:
        D = gate.shape[-1]
        grads['value'] = grads['gate'][..., D:]
        grads['gate'] = grads['gate'][..., :D]
    return h, last, grads


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_forward(shape, dtype, gpu_device):
    import tempo_amd
    B, T, D = shape
    gate, value = _inputs(B, T, D, dtype, gpu_device)
    state, _ = _states(B, D, gpu_device)
    ref = R.recurrence(gate, value, state)
    h, last = tempo_amd.gated_recurrence(gate, value, state=state)
    R.check(h, ref['h'], ref['h_tol'], 'h')
    R.check(last, ref['last'], ref['last_tol'], 'last')
    h2, last2 = tempo_amd.gated_recurrence(gate, value, state=state)
    assert torch.equal(h, h2) and torch.equal(last, last2)


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_gradients(shape, dtype, gpu_device):
    B, T, D = shape
    gate, value = _inputs(B, T, D, dtype, gpu_device, seed=3)
    state, grad_last = _states(B, D, gpu_device)
    grad_h = _inputs(B, T, D, dtype, gpu_device, seed=4)[1]
    ref = R.recurrence(gate, value, state, None, grad_h, grad_last)
    h, last, g = _train(gpu_device, gate, value, state, None, grad_h, grad_last)
    R.check(h, ref['h'], ref['h_tol'], 'h')
    R.check(last, ref['last'], ref['last_tol'], 'last')
    R.check(g['gate'], ref['dgate'], ref['dgate_tol'], 'dgate')
    R.check(g['value'], ref['dvalue'], ref['dvalue_tol'], 'dvalue')
    R.check(g['state'], ref['dstate'], ref['dstate_tol'], 'dstate')


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', [(4, 1, 8), (6, 4, 31), (5, 16, 24), (4, 40, 12), (7, 300, 45),
                                   (3, 1500, 8)], ids=str)
def test_padding_is_neither_read_nor_carries_gradients(shape, dtype, gpu_device):
    B, T, D = shape
    gate, value = _inputs(B, T, D, dtype, gpu_device, seed=5)
    state, grad_last = _states(B, D, gpu_device)
    lengths = _lengths(B, T, gpu_device)
    grad_h = _inputs(B, T, D, dtype, gpu_device, seed=6)[1]
    ref = R.recurrence(gate, value, state, lengths, grad_h, grad_last)
    pad = torch.arange(T, device=gpu_device)[None, :] >= lengths[:, None]
    for garbage in (float('nan'), float('inf'), torch.finfo(dtype).min):
        gg, vv, hh = (t.masked_fill(pad[..., None], garbage) for t in (gate, value, grad_h))
        h, last, g = _train(gpu_device, gg, vv, state, lengths, hh, grad_last)
        for name, got in (('h', h), ('last', last), ('dgate', g['gate']),
                          ('dvalue', g['value']), ('dstate', g['state'])):
            R.check(got, ref[name], ref[name + '_tol'], f'{name}, padding {garbage}')
        for got in (h, g['gate'], g['value']):
            assert not bool(got[pad].any())


def test_lengths_outside_the_sequence_count_as_its_ends(gpu_device):
    import tempo_amd
    gate, value = _inputs(3, 37, 12, torch.float32, gpu_device)
    odd = torch.tensor([-5, 1000, 37], dtype=torch.int32, device=gpu_device)
    even = torch.tensor([0, 37, 37], dtype=torch.int32, device=gpu_device)
    for a, b in zip(tempo_amd.gated_recurrence(gate, value, lengths=odd),
                    tempo_amd.gated_recurrence(gate, value, lengths=even)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', [(3, 5, 16), (4, 4, 13), (3, 200, 34), (6000, 4, 32)], ids=str)
@pytest.mark.parametrize('layout', ['time_major', 'odd_rows', 'combined', 'combined_time_major'])
def test_layouts_hold_the_same_values(layout, shape, dtype, gpu_device):
    B, T, D = shape
    gate, value = _inputs(B, T, D, dtype, gpu_device, seed=7)
    state, grad_last = _states(B, D, gpu_device)
    grad_h = _inputs(B, T, D, dtype, gpu_device, seed=8)[1]
    want = _train(gpu_device, gate, value, state, None, grad_h, grad_last)
    if layout.startswith('combined'):
        if layout != 'combined':
            gate, value = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (gate, value))
        got = _train(gpu_device, gate, value, state, None, grad_h, grad_last, combined=True)
    else:
        gate, value = _inputs(B, T, D, dtype, gpu_device, layout, seed=7)
        got = _train(gpu_device, gate, value, state, None, grad_h, grad_last)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    for name in want[2]:
        assert torch.equal(want[2][name], got[2][name]), name
    if layout == 'time_major':
        assert got[0].transpose(0, 1).is_contiguous()


@pytest.mark.parametrize('T', [1, 6, 50, 700])
def test_one_pass_equals_steps_with_a_carried_state(T, gpu_device):
    """Serving: T = 1 and the state updated in place, against the whole sequence."""
    import tempo_amd
    B, D = 3, 40
    gate, value = _inputs(B, T, D, torch.float32, gpu_device, seed=9)
    first, _ = _states(B, D, gpu_device)
    ref = R.recurrence(gate, value, first)
    state = first.clone()
    out = torch.empty(B, 1, D, device=gpu_device)
    for t in range(T):
        h, last = tempo_amd.gated_recurrence(gate[:, t:t + 1], value[:, t:t + 1], state=state,
                                             out=out, state_out=state)
        assert h is out and last is state
        R.check(h, ref['h'][:, t:t + 1], ref['h_tol'][:, t:t + 1], f'h at {t}')
    R.check(state, ref['last'], ref['last_tol'], 'state')
    again = first.clone()  # the whole sequence may update its state in place, too
    tempo_amd.gated_recurrence(gate, value, state=again, state_out=again)
    R.check(again, ref['last'], ref['last_tol'], 'state in place')


@pytest.mark.parametrize('T,D', [(64, 8), (5000, 4)])
def test_gates_at_their_limits(T, D, gpu_device):
    """Shut (the state stays, bit for bit), open (the value passes, bit for bit), infinite and
    the type's lowest: exactly the limits of the formula, no drift over thousands of steps."""
    import tempo_amd
    _, value = _inputs(2, T, D, torch.float32, gpu_device)
    state, _ = _states(2, D, gpu_device)
    for shut in (float('-inf'), torch.finfo(torch.float32).min, -200.0):
        h, last = tempo_amd.gated_recurrence(torch.full_like(value, shut), value, state=state)
        assert torch.equal(last, state) and torch.equal(h, state[:, None].expand_as(h))
    for wide in (float('inf'), torch.finfo(torch.float32).max, 200.0):
        h, last = tempo_amd.gated_recurrence(torch.full_like(value, wide), value, state=state)
        assert torch.equal(h, value) and torch.equal(last, value[:, -1])
    # nearly shut over the whole sequence: z = 4.5e-5 forgets next to nothing, see the bound
    gate = torch.full_like(value, -10.0)
    ref = R.recurrence(gate, value, state)
    h, last = tempo_amd.gated_recurrence(gate, value, state=state)
    R.check(h, ref['h'], ref['h_tol'], 'h')
    # a constant input is a fixed point: it stays one through any gates
    gate, _ = _inputs(2, T, D, torch.float32, gpu_device, seed=10, spread=6.0)
    h, last = tempo_amd.gated_recurrence(gate, torch.full_like(value, 0.7),
                                         state=torch.full_like(state, 0.7))
    assert float((h - 0.7).abs().max()) <= (1 + T / 32) * 2.0 ** -24


@pytest.mark.parametrize('dtype', DTYPES[1:], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('T', [3, 2000])
def test_gates_at_their_limits_in_16_bits(T, dtype, gpu_device):
    import tempo_amd
    gate, value = _inputs(2, T, 9, dtype, gpu_device, seed=21)
    state, _ = _states(2, 9, gpu_device)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    shut = torch.full_like(gate, float('-inf'))
    shut[:, 1::3] = low
    h, last = tempo_amd.gated_recurrence(shut, value, state=state)
    assert torch.equal(last, state) and torch.equal(h, state.to(dtype)[:, None].expand_as(h))
    for t, x in enumerate((float('inf'), high, float('-inf'), low, 100.0, -100.0)):
        gate[:, t::11] = x
    ref = R.recurrence(gate, value, state)
    h, last = tempo_amd.gated_recurrence(gate, value, state=state)
    R.check(h, ref['h'], ref['h_tol'], 'h')
    R.check(last, ref['last'], ref['last_tol'], 'last')


@pytest.mark.parametrize('T', [12, 300])
@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
def test_nan_stays_in_its_channel(dtype, T, gpu_device):
    import tempo_amd
    gate, value = _inputs(2, T, 12, dtype, gpu_device)
    clean, _ = tempo_amd.gated_recurrence(gate, value)
    value[1, T // 2, 3] = float('nan')
    gate[0, 7, 5] = float('nan')
    h, _ = tempo_amd.gated_recurrence(gate, value)
    bad = torch.zeros_like(h, dtype=torch.bool)
    bad[1, T // 2:, 3] = True
    bad[0, 7:, 5] = True
    assert bool(h[bad].isnan().all())
    assert torch.equal(h[~bad], clean[~bad])
    # backwards it reaches the steps in front of it, of its channel
    grad = torch.ones_like(h)
    _, _, g = _train(gpu_device, gate, value, None, None, grad, None)
    for name in g:
        other = [c for c in range(12) if c not in (3, 5)]
        assert not bool(g[name][..., other].isnan().any())


def test_gradients_are_the_differences(gpu_device):
    """Directional derivatives of the 64-bit formula against the kernel's gradients."""
    B, T, D = 3, 120, 10
    gate, value = _inputs(B, T, D, torch.float32, gpu_device, seed=11, spread=1.5)
    state, grad_last = _states(B, D, gpu_device)
    grad_h = _inputs(B, T, D, torch.float32, gpu_device, seed=12)[1]
    _, _, g = _train(gpu_device, gate, value, state, None, grad_h, grad_last)
    gen = torch.Generator().manual_seed(13)
    base = {'gate': gate, 'value': value, 'state': state}

    def loss(moved, by):
        x = {k: t.double().cpu() for k, t in base.items()}
        for k in moved:
            x[k] = x[k] + by * moved[k]
        r = R.recurrence(x['gate'], x['value'], x['state'])
        return float((r['h'] * grad_h.double().cpu()).sum() +
                     (r['last'] * grad_last.double().cpu()).sum())

    for name in base:
        d = {name: torch.randn(base[name].shape, generator=gen, dtype=torch.float64)}
        step = 1e-4
        slope = (loss(d, step) - loss(d, -step)) / (2 * step)
        mine = float((g[name].double().cpu() * d[name]).sum())
        # 64-bit differences err by step^2 = 1e-8; fp32 gradients by 1e-6 of their absolute sum
        scale = float((g[name].double().cpu() * d[name]).abs().sum())
        assert abs(slope - mine) <= 2e-6 * scale, (name, slope, mine)


@pytest.mark.parametrize('which', ['h', 'last', 'gate_only', 'expanded'])
def test_partial_gradients(which, gpu_device):
    import tempo_amd
    B, T, D = 2, 50, 18
    gate, value = _inputs(B, T, D, torch.float32, gpu_device, seed=14)
    state, grad_last = _states(B, D, gpu_device)
    grad_h = _inputs(B, T, D, torch.float32, gpu_device, seed=15)[1]
    if which in ('h', 'last'):
        gh, gl = (grad_h, None) if which == 'h' else (None, grad_last)
        ref = R.recurrence(gate, value, state, None, gh, gl)
        _, _, g = _train(gpu_device, gate, value, state, None, gh, gl)
    elif which == 'gate_only':
        ref = R.recurrence(gate, value, None, None, grad_h, None)
        leaf = gate.detach().requires_grad_(True)
        h, _ = tempo_amd.gated_recurrence(leaf, value)
        g = {'gate': torch.autograd.grad(h, leaf, grad_h)[0]}
    else:  # the gradient of a sum has no memory of its own
        ones = torch.ones(B, T, D)
        ref = R.recurrence(gate, value, None, None, ones, None)
        leaf = gate.detach().requires_grad_(True)
        h, _ = tempo_amd.gated_recurrence(leaf, value)
        h.sum().backward()
        g = {'gate': leaf.grad}
    for name in g:
        R.check(g[name], ref['d' + name], ref['d' + name + '_tol'], name)


@pytest.mark.parametrize('shape', [(0, 5, 4), (3, 0, 4)], ids=str)
def test_empty(shape, gpu_device):
    import tempo_amd
    B, T, D = shape
    gate = torch.zeros(B, T, D, device=gpu_device, requires_grad=True)
    value = torch.zeros(B, T, D, device=gpu_device)
    state = torch.randn(B, D, device=gpu_device, requires_grad=True)
    h, last = tempo_amd.gated_recurrence(gate, value, state=state)
    assert h.shape == (B, T, D) and torch.equal(last, state)
    dgate, dstate = torch.autograd.grad([h, last], [gate, state],
                                        [torch.zeros_like(h), torch.ones_like(last)])
    assert dgate.shape == gate.shape and bool((dstate == 1).all())
    h, last = tempo_amd.gated_recurrence(gate.detach(), value)
    assert not bool(last.any())


def test_refusals(gpu_device):
    import tempo_amd
    from tempo_amd import ops
    f = tempo_amd.gated_recurrence
    gate, value = _inputs(2, 5, 6, torch.float32, gpu_device)
    state = torch.zeros(2, 6, device=gpu_device)
    lengths = torch.ones(2, dtype=torch.int32, device=gpu_device)
    both, rows = torch.cat([gate, value], -1), torch.zeros(3, 6, device=gpu_device)
    for bad in (lambda: f(gate.cpu(), value), lambda: f(gate, value.half()),
                lambda: f(gate.double(), value.double()), lambda: f(gate.long(), value.long()),
                lambda: f(gate, value, state=state.half()),
                lambda: f(gate, value, lengths=lengths.long()),
                lambda: f(gate, value, out=torch.empty_like(gate, dtype=torch.float16))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: f(gate, value[:, :4]), lambda: f(gate[0], value[0]),
                lambda: f(gate[..., :5]), lambda: f(gate.transpose(1, 2), value.transpose(1, 2)),
                lambda: f(gate[..., :0], value[..., :0]),
                lambda: f(gate, value, state=state[:1]),
                lambda: f(gate, value, state=state.expand(2, 2, 6)),
                lambda: f(gate, value, state=torch.zeros(6, 2, device=gpu_device).t()),
                lambda: f(gate, value, lengths=lengths[:1]),
                lambda: f(gate, value, out=gate[:1]),
                lambda: f(gate, value, state_out=state[:1]),
                lambda: f(gate, value, out=value), lambda: f(gate, value, out=gate),
                lambda: f(both[..., :6], both[..., 6:], out=both[..., 3:9]),
                lambda: f(gate, value, state=rows[:2], state_out=rows[1:])):
        with pytest.raises(ValueError):
            bad()
    leaf = gate.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError):
        f(leaf, value, out=torch.empty_like(gate))
    with pytest.raises(NotImplementedError):
        ops.recurrence_forward(leaf, value)
    h, _ = f(leaf, value)
    (first,) = torch.autograd.grad(h.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), leaf)


def test_side_stream_and_two_calls_at_once(gpu_device):
    """Work queued on the caller's stream comes first, and calls on two streams do not share
    scratch memory."""
    import tempo_amd
    shape = (2, 4096, 64)
    ins = [_inputs(*shape, torch.float32, gpu_device, seed=20 + i) for i in range(2)]
    want = [tempo_amd.gated_recurrence(g, v) for g, v in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu_device) for _ in range(2)]
    got = []
    for rep in range(3):
        for s, (g, v) in zip(streams, ins):
            s.wait_stream(torch.cuda.current_stream(gpu_device))
            with torch.cuda.stream(s):
                x = v
                for _ in range(40):
                    x = x * 1.0
                got.append(tempo_amd.gated_recurrence(g, x))
    torch.cuda.synchronize()
    for i, (h, last) in enumerate(got):
        assert torch.equal(h, want[i % 2][0]) and torch.equal(last, want[i % 2][1])


def test_graph_replays(gpu_device):
    """A training step captured once and replayed on new inputs, with eager work between."""
    import tempo_amd
    B, T, D = 2, 2100, 48
    sets = []
    for seed in range(3):
        gate, value = _inputs(B, T, D, torch.float32, gpu_device, seed=30 + seed)
        state, grad_last = _states(B, D, gpu_device, seed=40 + seed)
        grad_h = _inputs(B, T, D, torch.float32, gpu_device, seed=50 + seed)[1]
        sets.append((gate, value, state, grad_h, grad_last))
    want = []
    for gate, value, state, grad_h, grad_last in sets:
        h, last, g = _train(gpu_device, gate, value, state, None, grad_h, grad_last)
        want.append([h.detach(), last.detach(), g['gate'], g['value'], g['state']])
        del h, last, g
    bufs = [t.clone() for t in sets[0]]
    leaves = [t.requires_grad_(True) for t in bufs[:3]]

    def one():
        h, last = tempo_amd.gated_recurrence(leaves[0], leaves[1], state=leaves[2])
        return [h.detach(), last.detach()] + list(
            torch.autograd.grad([h, last], leaves, bufs[3:]))

    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream(gpu_device).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = one()
    for rep in range(2):
        for data, ref in zip(sets, want):
            with torch.no_grad():
                for b, t in zip(bufs, data):
                    b.copy_(t)
            graph.replay()
            tempo_amd.gated_recurrence(sets[1][0], sets[1][1])  # eager work in between
            torch.cuda.synchronize()
            for a, b in zip(outs, ref):
                assert torch.equal(a, b)


def test_strides_beyond_32_bits(gpu_device):
    """Rows further apart than 2^31 elements: offsets are 64-bit."""
    import tempo_amd
    step = (1 << 31) + 64
    base = torch.empty(step + 4096, dtype=torch.float16, device=gpu_device)
    g = torch.as_strided(base, (2, 3, 32), (step, 64, 1))
    v = torch.as_strided(base, (2, 3, 32), (step, 64, 1), 32)
    gate, value = _inputs(2, 3, 32, torch.float16, gpu_device, seed=60)
    g.copy_(gate), v.copy_(value)
    want = tempo_amd.gated_recurrence(gate, value)
    got = tempo_amd.gated_recurrence(g, v)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_result_rows_overlap(gpu_device):
    """Rows of a result that coincide or run into each other are refused, as are results in the
    memory of the lengths; rows of one batch item or one step alone may have any distance."""
    import tempo_amd
    gate, value = _inputs(3, 5, 6, torch.float32, gpu_device)
    buf = torch.zeros(400, device=gpu_device)
    lengths = torch.tensor([5, 2, 0], dtype=torch.int32, device=gpu_device)
    want = tempo_amd.gated_recurrence(gate, value, lengths=lengths)

    def call(strides, at=0, shape=(3, 5, 6), **kw):
        out = torch.as_strided(buf, shape, strides, at)
        h, last = tempo_amd.gated_recurrence(gate[:shape[0], :shape[1]],
                                             value[:shape[0], :shape[1]], out=out,
                                             lengths=lengths[:shape[0]], **kw)
        assert h is out
        return h, last

    for strides in ((0, 6, 1), (30, 0, 1), (29, 6, 1), (30, 5, 1), (6, 17, 1), (0, 0, 1)):
        with pytest.raises(ValueError, match='rows overlap'):
            call(strides)
    for strides in ((30, 6, 1), (6, 18, 1), (70, 13, 1), (7, 50, 1)):
        got = call(strides)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    h, _ = call((0, 6, 1), shape=(1, 5, 6))
    assert torch.equal(h, want[0][:1])
    h, _ = call((6, 0, 1), shape=(3, 1, 6))
    assert torch.equal(h[:2], want[0][:2, :1])
    held = buf.view(torch.int32)[360:363]
    held.copy_(lengths)
    state = buf[358:376].view(3, 6)
    with pytest.raises(ValueError, match='state_out: shares memory with lengths'):
        tempo_amd.gated_recurrence(gate, value, lengths=held, state_out=state)
    with pytest.raises(ValueError, match='out: shares memory with lengths'):
        tempo_amd.gated_recurrence(gate, value, lengths=held, out=buf[300:390].view(3, 5, 6))


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('T', [1, 3, 2000])
def test_shut_gates_hide_the_largest_values(T, dtype, gpu_device):
    """Steps masked by their gate (minus infinity, the type's lowest value, -110) may hold the
    type's lowest or largest value, too: the state stays, bit for bit, and no gradient comes out
    of them."""
    gate, value = _inputs(2, T, 9, dtype, gpu_device, seed=70)
    state, grad_last = _states(2, 9, gpu_device)
    info = torch.finfo(dtype)
    for low in (float('-inf'), info.min, -110.0):
        gate.fill_(low)
        for most in (info.min, info.max):
            value.fill_(most)
            h, last, g = _train(gpu_device, gate, value, state, None, torch.zeros_like(gate),
                                grad_last)
            assert torch.equal(last, state)
            assert torch.equal(h, state.to(dtype)[:, None].expand_as(h))
            assert torch.equal(g['state'], grad_last)
            if low != -110.0:
                assert not bool(g['gate'].any()) and not bool(g['value'].any())
    # among ordinary steps
    gate, value = _inputs(2, T, 9, dtype, gpu_device, seed=71)
    masked = torch.arange(T, device=gpu_device) % 3 == 1
    gate[:, masked] = float('-inf')
    value[:, masked] = 0
    ref = R.recurrence(gate, value, state)
    value[:, masked] = info.min
    h, last, _ = _train(gpu_device, gate, value, state, None, torch.zeros_like(gate), grad_last)
    R.check(h, ref['h'], ref['h_tol'], 'h')
    R.check(last, ref['last'], ref['last_tol'], 'last')
