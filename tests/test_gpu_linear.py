"""The fused linear layer against its formula in 64 bits: types, activations, one row to many,
odd and ragged sizes, row strides, gradients."""
import pytest
import torch

import temporal_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = ['none', 'relu', 'silu', 'gelu', 'sigmoid', 'tanh']
# (M, K, N): single elements; one row; the head's widths; sizes around a tile, a step of k, a
# 16-byte chunk; long sums that are split; many rows of few channels
SHAPES = [(1, 1, 1), (1, 256, 64), (10, 256, 64), (8, 1024, 520), (2, 3, 5), (127, 63, 129),
          (128, 64, 128), (129, 65, 127), (130, 136, 260), (257, 33, 15), (300, 256, 17),
          (31, 4099, 12), (64, 2048, 64), (5000, 256, 32), (4000, 24, 40), (700, 321, 515)]


def _make(M, K, N, dtype, dev, seed=0, bias=True, residual=False, grad=False):
    gen = torch.Generator().manual_seed(seed)
    t = {'x': torch.randn(M, K, generator=gen),
         'weight': torch.randn(N, K, generator=gen) * (1.5 / K ** 0.5)}
    t['bias'] = torch.randn(N, generator=gen) * 0.5 if bias else None
    t['residual'] = torch.randn(M, N, generator=gen) if residual else None
    t['grad'] = torch.randn(M, N, generator=gen) if grad else None
    return {k: None if v is None else v.to(dtype).to(dev) for k, v in t.items()}


def _train(t, activation):
    import tempo_amd
    leaves = {k: t[k].detach().requires_grad_(True) for k in ('x', 'weight', 'bias', 'residual')
              if t[k] is not None}
    y = tempo_amd.fused_linear(leaves['x'], leaves['weight'], leaves.get('bias'),
                               leaves.get('residual'), activation)
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t['grad'])))


def _check_grads(t, activation, what=''):
    ref = R.linear(t['x'], t['weight'], t['bias'], t['residual'], activation, t['grad'])
    y, g = _train(t, activation)
    R.check(y, ref['y'], ref['y_tol'], what + 'y')
    R.check(g['x'], ref['dx'], ref['dx_tol'], what + 'dx')
    R.check(g['weight'], ref['dweight'], ref['dweight_tol'], what + 'dweight')
    if t['bias'] is not None:
        R.check(g['bias'], ref['dbias'], ref['dbias_tol'], what + 'dbias')
    if t['residual'] is not None:
        assert torch.equal(g['residual'], t['grad'])


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_forward(shape, dtype, gpu_device):
    import tempo_amd
    M, K, N = shape
    for i, act in enumerate(('none', ACTS[1 + (M + K + N) % 5])):
        t = _make(M, K, N, dtype, gpu_device, seed=i, bias=i == 1, residual=i == 1)
        ref = R.linear(t['x'], t['weight'], t['bias'], t['residual'], act)
        y = tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], t['residual'], act)
        R.check(y, ref['y'], ref['y_tol'], f'y, {act}')
        again = tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], t['residual'], act)
        assert torch.equal(y, again)


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_gradients(shape, dtype, gpu_device):
    M, K, N = shape
    for i, act in enumerate(('none', ACTS[1 + (M + K + N) % 5])):
        t = _make(M, K, N, dtype, gpu_device, seed=2 + i, bias=i == 1, residual=i == 0,
                  grad=True)
        _check_grads(t, act, f'{act} ')


@pytest.mark.parametrize('dtype', DTYPES[1:], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', [(4200, 72, 4104), (4104, 4104, 72), (72, 4104, 4104)], ids=str)
def test_more_tiles_than_compute_units(shape, dtype, gpu_device):
    """Each of the three products once large enough for the widest tiles, none of its sizes a
    multiple of them."""
    M, K, N = shape
    _check_grads(_make(M, K, N, dtype, gpu_device, seed=4, residual=True, grad=True), 'silu')


# products whose tiles are 64 or 128 rows by 64 or 128 columns, each in all three operand orders
@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', [(70, 72, 72), (67, 65, 71), (4000, 16, 520), (2000, 72, 1000),
                                   (2003, 71, 1001), (4000, 33, 1000), (4000, 520, 264),
                                   (2000, 520, 1000), (180, 520, 4000), (180, 65, 8001),
                                   (180, 130, 20000), (3999, 521, 1001), (4000, 520, 1000)],
                         ids=str)
def test_tile_shapes(shape, dtype, gpu_device):
    M, K, N = shape
    act = ACTS[(M + K + N) % 6]
    _check_grads(_make(M, K, N, dtype, gpu_device, seed=7, residual=True, grad=True), act)


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', [(16411, 256, 32), (16384, 256, 64), (16400, 321, 17),
                                   (16385, 24, 40), (20001, 64, 100), (16411, 32, 256),
                                   (16390, 520, 8), (16384, 1, 1), (16400, 130, 129),
                                   (2100, 504, 8), (2048, 248, 64), (2047, 64, 20)], ids=str)
def test_many_rows_of_few_channels(shape, dtype, gpu_device):
    M, K, N = shape
    for i, act in enumerate(('none', ACTS[1 + (M + K + N) % 5])):
        _check_grads(_make(M, K, N, dtype, gpu_device, seed=5 + i, bias=i == 0, residual=i == 1,
                           grad=True), act, f'{act} ')


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', [(65539, 256, 32), (65537, 256, 64), (66000, 221, 17),
                                   (65600, 24, 40), (65540, 32, 256), (65537, 1, 1),
                                   (65536, 64, 33), (65541, 512, 8), (65541, 513, 8),
                                   (65538, 257, 5), (32771, 63, 31), (32769, 31, 63)], ids=str)
def test_more_rows_of_few_channels(shape, dtype, gpu_device):
    M, K, N = shape
    for i, act in enumerate(('none', ACTS[1 + (M + K + N) % 5])):
        _check_grads(_make(M, K, N, dtype, gpu_device, seed=9 + i, bias=i == 0, residual=i == 1,
                           grad=True), act, f'{act} ')


# either kernel for up to 64 rows: the sums long and the columns few, the other way round, both
@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('M', [1, 8, 16, 17, 31, 33, 48, 64])
def test_few_rows_of_many_columns(M, dtype, gpu_device):
    import tempo_amd
    for K, N in ((256, 300), (1000, 1000), (1029, 999), (4096, 520), (515, 8200)):
        t = _make(M, K, N, dtype, gpu_device, seed=8, residual=True)
        ref = R.linear(t['x'], t['weight'], t['bias'], t['residual'], 'gelu')
        y = tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], t['residual'], 'gelu')
        R.check(y, ref['y'], ref['y_tol'], f'y, {K} x {N}')


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('M', [1, 15, 16, 17, 32, 33, 64, 65])
def test_few_rows(M, dtype, gpu_device):
    for K, N in ((1000, 300), (72, 33), (1029, 17), (4096, 16)):
        t = _make(M, K, N, dtype, gpu_device, seed=7, residual=True)
        import tempo_amd
        ref = R.linear(t['x'], t['weight'], t['bias'], t['residual'], 'silu')
        y = tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], t['residual'], 'silu')
        R.check(y, ref['y'], ref['y_tol'], f'y, {K} x {N}')


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('act', ACTS)
def test_activations_over_their_range(act, dtype, gpu_device):
    """K = 1 and a weight of 1: z runs over the whole range, infinities at the ends."""
    import tempo_amd
    z = torch.cat([torch.linspace(-30, 30, 4001), torch.logspace(-7, 0, 200),
                   -torch.logspace(-7, 0, 200)]).to(dtype)[:, None].to(gpu_device)
    one = torch.ones(1, 1, dtype=dtype, device=gpu_device)
    t = {'x': z, 'weight': one, 'bias': None, 'residual': None, 'grad': torch.ones_like(z)}
    _check_grads(t, act)
    ends = torch.tensor([[float('-inf')], [float('inf')], [torch.finfo(dtype).min],
                         [torch.finfo(dtype).max], [float('nan')]], dtype=dtype,
                        device=gpu_device)
    y = tempo_amd.fused_linear(ends, one, activation=act).flatten().tolist()
    low, high = {'none': (float('-inf'), float('inf')), 'relu': (0.0, float('inf')),
                 'sigmoid': (0.0, 1.0), 'tanh': (-1.0, 1.0)}.get(act, (None, float('inf')))
    assert y[1] == high and y[4] != y[4]
    if low is not None:
        assert y[0] == low
    if act in ('sigmoid', 'tanh'):
        assert y[2] == low and y[3] == high


@pytest.mark.parametrize('act', ['none', 'gelu'])
@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('K,N', [(64, 48), (33, 21)])
def test_row_strides_and_offsets(K, N, dtype, act, gpu_device):
    """Slices of larger rows at odd offsets (memory beyond them holds NaN), a transposed
    gradient, an expanded residual, more than two dimensions, a convolution's weight."""
    import tempo_amd
    M = 150
    t = _make(M, K, N, dtype, gpu_device, seed=5, residual=True, grad=True)
    want_y, want = _train(t, act)
    for offset, extra in ((1, 5), (8, 16), (0, 1)):
        s = {}
        for k in ('x', 'weight', 'residual', 'grad'):
            wide = torch.full((t[k].shape[0], t[k].shape[1] + extra + offset), float('nan'),
                              dtype=dtype, device=gpu_device)
            s[k] = wide[:, offset:offset + t[k].shape[1]]
            s[k].copy_(t[k])
        s['bias'] = torch.cat([t['bias'], t['bias']])[N:]
        y, g = _train(s, act)
        assert torch.equal(y, want_y)
        for k in want:
            assert torch.equal(g[k], want[k]), (k, offset)
        out = torch.full((M, N + extra), -7.0, dtype=dtype, device=gpu_device)
        got = tempo_amd.fused_linear(s['x'], s['weight'], s['bias'], s['residual'], act,
                                     out=out[:, :N])
        assert torch.equal(got, want_y) and bool((out[:, N:] == -7).all())
    s = dict(t, grad=t['grad'].t().contiguous().t())
    _, g = _train(s, act)
    for k in want:
        assert torch.equal(g[k], want[k]), k
    x3 = t['x'].view(3, 10, 5, K)
    y = tempo_amd.fused_linear(x3, t['weight'][:, :, None, None], t['bias'],
                               t['residual'].view(3, 10, 5, N), act)
    assert y.shape == (3, 10, 5, N) and torch.equal(y.view(M, N), want_y)
    row = t['residual'][:1].detach().requires_grad_(True)
    y = tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], row.expand(M, N), act)
    ref = R.linear(t['x'], t['weight'], t['bias'], row.expand(M, N), act)
    R.check(y, ref['y'], ref['y_tol'], 'y, shared residual')
    (d,) = torch.autograd.grad(y, row, t['grad'])
    assert torch.equal(d, t['grad'].sum(0, keepdim=True))
    one = tempo_amd.fused_linear(t['x'][3], t['weight'], t['bias'], t['residual'][3], act)
    ref1 = R.linear(t['x'][3:4], t['weight'], t['bias'], t['residual'][3:4], act)
    R.check(one[None], ref1['y'], ref1['y_tol'], 'one vector')


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('M,K,N', [(200, 72, 40), (5, 300, 33), (3000, 64, 24), (600, 33, 130)])
def test_residual_in_place(M, K, N, dtype, gpu_device):
    import tempo_amd
    t = _make(M, K, N, dtype, gpu_device, seed=8, residual=True)
    want = tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], t['residual'], 'gelu')
    stream = t['residual'].clone()
    got = tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], stream, 'gelu', out=stream)
    assert got is stream and torch.equal(got, want)


def test_channels_last_map_is_read_in_place(gpu_device):
    import tempo_amd
    m = torch.randn(2, 24, 6, 10, device=gpu_device).contiguous(memory_format=torch.channels_last)
    w = torch.randn(8, 24, 1, 1, device=gpu_device)
    y = tempo_amd.fused_linear(m.permute(0, 2, 3, 1), w)
    ref = R.linear(m.permute(0, 2, 3, 1), w.flatten(1))
    R.check(y, ref['y'], ref['y_tol'], 'y')


@pytest.mark.parametrize('want', ['x', 'weight', 'bias', 'residual'])
def test_single_gradients(want, gpu_device):
    import tempo_amd
    t = _make(200, 40, 24, torch.float32, gpu_device, seed=6, residual=True, grad=True)
    _, full = _train(t, 'silu')
    args = {k: t[k] for k in ('x', 'weight', 'bias', 'residual')}
    args[want] = t[want].detach().requires_grad_(True)
    y = tempo_amd.fused_linear(**args, activation='silu')
    (g,) = torch.autograd.grad(y, args[want], t['grad'])
    assert torch.equal(g, full[want])
    y = tempo_amd.fused_linear(**args, activation='silu')
    y.sum().backward()  # the gradient of a sum has no memory of its own
    ref = R.linear(t['x'], t['weight'], t['bias'], t['residual'], 'silu',
                   torch.ones_like(t['grad']))
    if want != 'residual':
        R.check(args[want].grad, ref['d' + want], ref['d' + want + '_tol'], want)
    else:
        assert bool((args[want].grad == 1).all())


def test_gradients_are_the_differences(gpu_device):
    t = _make(37, 29, 23, torch.float32, gpu_device, seed=7, residual=True, grad=True)
    gen = torch.Generator().manual_seed(8)
    for act in ('silu', 'gelu', 'sigmoid', 'tanh'):
        _, g = _train(t, act)
        for name in g:
            d = torch.randn(t[name].shape, generator=gen, dtype=torch.float64)

            def loss(by):
                a = {k: t[k].double().cpu() for k in ('x', 'weight', 'bias', 'residual')}
                a[name] = a[name] + by * d
                y = R.linear(a['x'], a['weight'], a['bias'], a['residual'], act)['y']
                return float((y * t['grad'].double().cpu()).sum())

            slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
            mine = float((g[name].double().cpu() * d).sum())
            scale = float((g[name].double().cpu() * d).abs().sum())
            assert abs(slope - mine) <= 2e-6 * scale, (act, name, slope, mine)


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
def test_infinity_and_nan_stay_in_their_rows(dtype, gpu_device):
    """k beyond the sum's end and rows beyond the matrix's contribute nothing, whatever lies
    there; a bad row spoils itself alone."""
    import tempo_amd
    M, K, N = 140, 37, 50
    t = _make(M, K, N, dtype, gpu_device, seed=9)
    clean = tempo_amd.fused_linear(t['x'], t['weight'], t['bias'])
    x = t['x'].clone()
    x[17, 36] = float('inf')
    x[139, 0] = float('nan')
    y = tempo_amd.fused_linear(x, t['weight'], t['bias'])
    assert not bool(torch.isfinite(y[17]).any()) and bool(y[139].isnan().all())
    keep = [i for i in range(M) if i not in (17, 139)]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
def test_relu_keeps_tiny_signs(dtype, gpu_device):
    """z that underflows in 16 bits still has relu's slope."""
    x = torch.tensor([[1e-4], [-1e-4]], device=gpu_device).to(dtype)
    w = torch.tensor([[1e-4]], device=gpu_device).to(dtype)
    t = {'x': x, 'weight': w, 'bias': None, 'residual': None, 'grad': torch.ones_like(x)}
    _, g = _train(t, 'relu')
    assert torch.equal(g['x'].flatten(), torch.stack([w[0, 0], w.new_zeros(())]))


def test_no_rows(gpu_device):
    import tempo_amd
    x = torch.zeros(0, 8, device=gpu_device, requires_grad=True)
    w = torch.ones(4, 8, device=gpu_device, requires_grad=True)
    b = torch.ones(4, device=gpu_device, requires_grad=True)
    for act in ('none', 'gelu'):
        y = tempo_amd.fused_linear(x, w, b, activation=act)
        assert y.shape == (0, 4)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 4, device=gpu_device))
        assert dx.shape == (0, 8) and not bool(dw.any()) and not bool(db.any())


def test_refusals(gpu_device):
    import tempo_amd
    from tempo_amd import ops
    f = tempo_amd.fused_linear
    t = _make(6, 8, 4, torch.float32, gpu_device, residual=True)
    x, w, b, r = t['x'], t['weight'], t['bias'], t['residual']
    for bad in (lambda: f(x.cpu(), w), lambda: f(x, w.half()), lambda: f(x, w, b.half()),
                lambda: f(x, w, b, r.half()), lambda: f(x.double(), w.double()),
                lambda: f(x.long(), w.long()), lambda: f(x, w.cpu()),
                lambda: f(x, w, out=torch.empty(6, 4, dtype=torch.half, device=gpu_device))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: f(x, w[:, :7]), lambda: f(x[0, 0], w), lambda: f(x, w[0]),
                lambda: f(x, w, b[:3]), lambda: f(x, w, b, r[:, :3]), lambda: f(x, w, b, r[:1]),
                lambda: f(x, w, activation='swish'), lambda: f(x, w.t().contiguous().t()),
                lambda: f(x.t().contiguous().t(), w), lambda: f(x, w[:0]),
                lambda: f(x[:, :0], w[:, :0]), lambda: f(x, w, out=torch.empty(4, 6)),
                lambda: f(x.view(2, 3, 8).transpose(0, 1), w),
                lambda: f(x, w, out=torch.empty(4, device=gpu_device).expand(6, 4)),
                lambda: f(x, w, out=x[:, 4:]), lambda: f(x[:4], w, out=w[:, :4]),
                lambda: f(x, torch.ones(8, 8, device=gpu_device), out=x)):
        with pytest.raises(ValueError):
            bad()
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError):
        f(leaf, w, out=torch.empty(6, 4, device=gpu_device))
    with pytest.raises(NotImplementedError):
        ops.linear_forward(leaf, w)
    (first,) = torch.autograd.grad(f(leaf, w).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), leaf)


def test_side_stream_and_two_calls_at_once(gpu_device):
    import tempo_amd
    sets = [_make(64, 4096, 64, torch.bfloat16, gpu_device, seed=10 + i) for i in range(2)]
    want = [tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], None, 'gelu') for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu_device) for _ in range(2)]
    got = []
    for rep in range(4):
        for s, t in zip(streams, sets):
            s.wait_stream(torch.cuda.current_stream(gpu_device))
            with torch.cuda.stream(s):
                x = t['x']
                for _ in range(40):
                    x = x * 1.0
                got.append(tempo_amd.fused_linear(x, t['weight'], t['bias'], None, 'gelu'))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2])


def test_graph_replays(gpu_device):
    """A training step captured once, replayed on new inputs with eager work between."""
    import tempo_amd
    sets = [_make(2000, 136, 72, torch.bfloat16, gpu_device, seed=20 + i, residual=True,
                  grad=True) for i in range(3)]
    want = []
    for t in sets:
        y, g = _train(t, 'gelu')
        want.append([y.detach()] + list(g.values()))
        del y, g
    names = ('x', 'weight', 'bias', 'residual')
    bufs = {k: sets[0][k].clone() for k in names + ('grad',)}
    leaves = [bufs[k].requires_grad_(True) for k in names]

    def one():
        y = tempo_amd.fused_linear(*leaves, activation='gelu')
        return [y.detach()] + list(torch.autograd.grad(y, leaves, bufs['grad']))

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
                for k in bufs:
                    bufs[k].copy_(data[k])
            graph.replay()
            _train(sets[1], 'gelu')  # eager work in between
            torch.cuda.synchronize()
            for a, b in zip(outs, ref):
                assert torch.equal(a, b)


@pytest.mark.parametrize('which', ['x', 'weight', 'residual', 'out', 'grad'])
def test_strides_beyond_32_bits(which, gpu_device):
    """Rows further apart than 2^31 elements: offsets are 64-bit."""
    import tempo_amd
    M = N = 3
    K = 24
    t = _make(M, K, N, torch.float16, gpu_device, seed=30, residual=True, grad=True)
    step = (1 << 30) + 1024 + 5
    far = torch.empty(2 * step + 64, dtype=torch.float16, device=gpu_device)
    want_y, want = _train(t, 'relu')
    if which == 'out':
        out = torch.as_strided(far, (M, N), (step, 1))
        tempo_amd.fused_linear(t['x'], t['weight'], t['bias'], t['residual'], 'relu', out=out)
        assert torch.equal(out, want_y)
        return
    moved = torch.as_strided(far, t[which].shape, (step, 1))
    moved.copy_(t[which])
    y, g = _train(dict(t, **{which: moved}), 'relu')
    assert torch.equal(y, want_y)
    for k in want:
        assert torch.equal(g[k], want[k]), k


@pytest.mark.parametrize('act', ACTS)
def test_gradients_where_z_leaves_the_type(act, gpu_device):
    """z beyond fp16's (bf16's) range is finite in the forward pass, and the slopes there are the
    limits: nothing but zeros and ones, in dx, dW and db."""
    import tempo_amd
    up, down = {'none': (1, 1), 'relu': (1, 0), 'silu': (1, 0), 'gelu': (1, 0)}.get(act, (0, 0))
    x = torch.tensor([[-300.0], [300.0], [0.0]], dtype=torch.float16, device=gpu_device)
    t = {'x': x, 'weight': torch.full((1, 1), 300.0, dtype=torch.float16, device=gpu_device),
         'bias': torch.zeros(1, dtype=torch.float16, device=gpu_device),
         # z = -90000 and 90000: y fits fp16 again
         'residual': x.new_tensor([[60000.0], [-60000.0], [0.0]]),
         'grad': x.new_tensor([[1.0], [1.0], [0.0]])}
    y, g = _train(t, act)
    assert bool(torch.isfinite(y).all())
    assert g['x'].flatten().tolist() == [300.0 * down, 300.0 * up, 0.0]
    assert g['weight'].item() == 300.0 * (up - down) and g['bias'].item() == up + down
    # one half step of bf16 beyond its largest value, still finite in fp32
    x = torch.tensor([[-2.0 ** 64, -2.0 ** 60], [2.0 ** 64, 2.0 ** 60]], device=gpu_device)
    w = torch.tensor([[2.0 ** 64 * (1 - 2.0 ** -8), 2.0 ** 59]], device=gpu_device)
    t = {'x': x.bfloat16(), 'weight': w.bfloat16(), 'bias': None, 'residual': None,
         'grad': x.new_ones(2, 1).bfloat16()}
    assert torch.equal(t['x'].float(), x) and torch.equal(t['weight'].float(), w)
    _, g = _train(t, act)
    assert torch.equal(g['x'].float(), torch.cat([w * down, w * up]))
    assert torch.equal(g['weight'].float(), x[:1] * down + x[1:] * up)
    # an infinity among the inputs is not hidden
    x = torch.tensor([[float('inf')], [float('nan')]], dtype=torch.float16, device=gpu_device)
    y = tempo_amd.fused_linear(x, x.new_ones(1, 1), activation=act)
    assert y[0].item() == {'sigmoid': 1.0, 'tanh': 1.0}.get(act, float('inf'))
    assert bool(y[1].isnan())


def test_out_and_residual_overlap(gpu_device):
    """A residual that is read by one workgroup after another one wrote the result over it is
    refused: shifted by a row or a channel, another distance between rows, rows that coincide.
    The same memory in the same order is not."""
    import tempo_amd
    t = _make(6, 8, 4, torch.float32, gpu_device)
    buf = torch.zeros(80, device=gpu_device)
    rows, wide = buf[:28].view(7, 4), buf[:48].view(6, 8)

    def call(residual, out, x=t['x']):
        return tempo_amd.fused_linear(x, t['weight'], t['bias'], residual, 'relu', out=out)

    for residual, out in ((rows[:6], rows[1:]), (rows[1:], rows[:6]), (rows[:6], wide[:, :4]),
                          (wide[:, :4], rows[:6]), (wide[:, :4], wide[:, 1:5]),
                          (rows[:1].expand(6, 4), rows[:6])):
        with pytest.raises(ValueError, match='shares memory with residual'):
            call(residual, out)
    bare = call(None, None)
    want = bare + 1
    wide[:, :4] = 1  # next to each other in the same rows
    call(wide[:, :4], wide[:, 4:])
    assert torch.equal(wide[:, 4:], want) and bool((wide[:, :4] == 1).all())
    for out in (rows[:6], wide[:, :4]):
        out.fill_(1)
        assert call(out.view_as(out), out) is out and torch.equal(out, want)
    out = buf[:4].view(1, 4)  # one row: its distance to the next one means nothing
    out.fill_(1)
    call(torch.as_strided(out, (1, 4), (4096, 1)), out, t['x'][:1])
    ref = R.linear(t['x'][:1], t['weight'], t['bias'], torch.ones(1, 4), 'relu')
    R.check(out, ref['y'], ref['y_tol'], 'one row')
    both = torch.zeros(6, 12, device=gpu_device)
    both[:, :8] = t['x']
    call(None, both[:, 8:], both[:, :8])
    assert torch.equal(both[:, 8:], bare) and torch.equal(both[:, :8], t['x'])
    with pytest.raises(ValueError, match='shares memory with x'):
        call(None, both[:, 7:11], both[:, :8])


# (M, K, N) with, in 16 bits, one product in 256 x 256 tiles: the forward, dx or dW, with
# remainders of rows, columns and k, sums shorter than the stages in flight, more tiles than
# compute units.  Which kernel a size selects is asserted without a GPU, in test_linear_plan.py.
WIDEST = [(4000, 520, 4008, 'y'), (4040, 1032, 4008, 'y'), (6000, 72, 4104, 'y'),
          (5000, 264, 6152, 'y'), (4040, 4008, 1032, 'dx'), (1032, 4008, 4040, 'dweight')]
# fp32 products in tiles of 64 x 128 that no size above selects
NARROW = [(9, 17209, 8), (8, 17472, 8), (13, 18688, 8), (184, 8, 8208), (47, 8, 16599)]


@pytest.mark.parametrize('dtype', DTYPES[1:], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', WIDEST, ids=str)
def test_widest_tiles(shape, dtype, gpu_device):
    M, K, N, _ = shape
    _check_grads(_make(M, K, N, dtype, gpu_device, seed=40, residual=True, grad=True), 'gelu')


@pytest.mark.parametrize('shape', NARROW, ids=str)
def test_narrow_tiles(shape, gpu_device):
    M, K, N = shape
    _check_grads(_make(M, K, N, torch.float32, gpu_device, seed=41, residual=True, grad=True),
                 'silu')


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
def test_gelu_far_down_its_tail(dtype, gpu_device):
    """K = 1 and a weight of 1, so that z is exact: gelu and its slope to one rounding and 2^-16 of
    their terms.  16 bits: 2^-18 of the approximation and 2^-24 z^2 / 2 for each rounding of the
    exponential's argument, three of them make 2^-17 at z = -9.  fp32: erfc(x) changes by
    2 x^2 + 1 = z^2 + 1 <= 82 times its argument's relative error, which is 2^-24 of the product
    and 2^-25.8 of the constant 1 / sqrt 2, 2^-17.3 in all, and the library's erfc errs itself."""
    z = torch.cat([torch.linspace(-9, 9, 3001), -torch.logspace(-4, 0.9, 500)]).to(dtype)
    z = z[:, None].to(gpu_device)
    one = torch.ones(1, 1, dtype=dtype, device=gpu_device)
    t = {'x': z, 'weight': one, 'bias': None, 'residual': None, 'grad': torch.ones_like(z)}
    y, g = _train(t, 'gelu')
    z = z.double().cpu()
    phi = torch.erfc(-z * 0.5 ** 0.5) / 2  # special.ndtr is (1 + erf) / 2: it cancels
    bell = torch.exp(-z * z / 2) * 0.3989422804014327
    own = 2.0 ** -16
    R.check(y, z * phi, R.rounding(z * phi, dtype) + own * (z * phi).abs(), 'gelu')
    R.check(g['x'], phi + z * bell, R.rounding(phi + z * bell, dtype) +
            own * (phi + z.abs() * bell), 'slope')


# long sums, in one piece and split: rows, k, columns (fp32 kernels of every kind)
EXACT = [(4, 4095, 24), (64, 4096, 512), (130, 4096, 136), (131, 4093, 77), (33000, 511, 24),
         (33000, 512, 32), (1024, 4096, 1024), (513, 1021, 515)]


@pytest.mark.parametrize('shape', EXACT, ids=str)
def test_long_fp32_sums_lose_nothing(shape, gpu_device):
    """Whole numbers whose sums stay below 2^24: every order of fp32 additions is exact, so the
    forward pass and all gradients are, to the last bit.  One factor takes 9 to 12 bits (the other
    one is -1, 0 or 1), more than bf16 or, where it is 12, fp16 operands hold: none may be
    shortened on its way, which bounds for rounded sums of this length would not show."""
    M, K, N = shape
    gen = torch.Generator().manual_seed(M)

    def wide(rows, cols, terms):  # |sum of `terms` of them| < 2^24
        most = min(4095, (2 ** 24 - 1) // terms)
        assert most > 2 ** 8
        return torch.randint(-most, most + 1, (rows, cols), generator=gen).float()

    def signs(rows, cols):
        return torch.randint(-1, 2, (rows, cols), generator=gen).float()

    for x, w, g in ((wide(M, K, max(K, M)), signs(N, K), signs(M, N)),
                    (signs(M, K), wide(N, K, max(K, N)), signs(M, N)),
                    (signs(M, K), signs(N, K), wide(M, N, max(M, N)))):
        t = {'x': x, 'weight': w, 'bias': None, 'residual': None, 'grad': g}
        t = {k: v if v is None else v.to(gpu_device) for k, v in t.items()}
        y, got = _train(t, 'none')
        x, w, g = x.double(), w.double(), g.double()
        assert torch.equal(y.double().cpu(), x @ w.t())
        assert torch.equal(got['x'].double().cpu(), g @ w)
        assert torch.equal(got['weight'].double().cpu(), g.t() @ x)


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('shape', [(153600, 256, 32), (4999, 251, 515), (5000, 256, 520),
                                   (700, 64, 40), (12, 256, 64)], ids=str)
def test_relu_of_exact_sums(shape, dtype, gpu_device):
    """relu's slope is discontinuous: where z lies within rounding of 0, two right programs may
    differ by a whole gradient.  On operands with few bits every sum is exact in any order, z's
    signs are, and the training step has to be: y, dx, dW and db are the 64-bit values, rounded
    once.  (x: multiples of 2^-6 up to 1, weight: of 2^-9 up to 55 of them, so that
    |z| 2^15 <= 64 x 55 x 256 < 2^24, and dW 2^6 <= 64 M < 2^24.)"""
    M, K, N = shape
    gen = torch.Generator().manual_seed(M)

    def lattice(most, step, *size):
        return torch.randint(-most, most + 1, size, generator=gen).float() * step

    t = {'x': lattice(64, 2.0 ** -6, M, K), 'weight': lattice(55, 2.0 ** -9, N, K),
         'bias': lattice(100, 2.0 ** -15, N), 'grad': lattice(1, 1.0, M, N)}
    x, w, b, g = (t[k].double() for k in ('x', 'weight', 'bias', 'grad'))
    z = x @ w.t() + b
    dz = g * (z > 0)
    want = {'x': dz @ w, 'weight': dz.t() @ x, 'bias': dz.sum(0)}
    t = {k: v.to(dtype).to(gpu_device) for k, v in t.items()}
    assert all(torch.equal(t[k].cpu().double(), v) for k, v in zip(t, (x, w, b, g)))
    y, got = _train(dict(t, residual=None), 'relu')
    assert torch.equal(y.cpu(), z.clamp(min=0).to(dtype))
    for k in want:
        assert torch.equal(got[k].cpu(), want[k].to(dtype)), k
