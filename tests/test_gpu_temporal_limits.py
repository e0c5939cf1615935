"""The ends of what a caller may do with the temporal head's operators: captured serving loops,
tensors of more than 2^32 elements, broadcast inputs, the smallest numbers."""
import pytest
import torch

import temporal_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _randn(dev, dtype, *shape, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).to(dev)


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
def test_captured_serving_loop(dtype, gpu_device):
    """One timestep of projection and recurrence captured with its state updated in place; replays
    carry the state on, with other lengths (0: a track without a new frame) and eager work of the
    same operators in between."""
    import tempo_amd
    B, K, D, steps = 10, 48, 24, 7
    weight, bias = _randn(gpu_device, dtype, 2 * D, K) / 4, _randn(gpu_device, dtype, 2 * D, seed=1)
    frames = _randn(gpu_device, dtype, steps, B, 1, K, seed=2)
    first = _randn(gpu_device, torch.float32, B, D, seed=3)
    lengths = torch.randint(0, 2, (steps, B), generator=torch.Generator().manual_seed(4),
                            dtype=torch.int32).to(gpu_device)
    x, n, state = frames[0].clone(), lengths[0].clone(), first.clone()
    out = torch.empty(B, 1, D, dtype=dtype, device=gpu_device)

    def one(x, n, state, out):
        both = tempo_amd.fused_linear(x, weight, bias)
        return tempo_amd.gated_recurrence(both, state=state, lengths=n, out=out, state_out=state)

    want, carried = [], first.clone()
    for t in range(steps):
        h, _ = one(frames[t], lengths[t], carried, torch.empty_like(out))
        want.append((h.clone(), carried.clone()))
    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        one(x, n, state, out)
    torch.cuda.current_stream(gpu_device).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(x, n, state, out)
    for rep in range(3):
        state.copy_(first)
        for t in range(steps):
            x.copy_(frames[t]), n.copy_(lengths[t])
            graph.replay()
            one(frames[0], lengths[0], first.clone(), torch.empty_like(out))
            torch.cuda.synchronize()
            assert torch.equal(out, want[t][0]) and torch.equal(state, want[t][1])
            skipped = lengths[t] == 0
            assert not bool(out[skipped].any())


def test_captured_recurrent_process_layer(gpu_device):
    import tempo_amd
    head = tempo_amd.RecurrentProcessLayerNHWC(24, 8).to(gpu_device)
    sets = [_randn(gpu_device, torch.float32, 12, 24, 9, 11, seed=i) for i in range(3)]
    with torch.no_grad():
        want = [head(m, 3, 2) for m in sets]
        maps, state = sets[0].clone(), torch.zeros(3 * 2 * 9 * 11, 8, device=gpu_device)
        side = torch.cuda.Stream(gpu_device)
        side.wait_stream(torch.cuda.current_stream(gpu_device))
        with torch.cuda.stream(side):
            head(maps, 3, 2, state)
        torch.cuda.current_stream(gpu_device).wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, last = head(maps, 3, 2, state)
        for rep in range(2):
            for m, (ref, ref_last) in zip(sets, want):
                maps.copy_(m)
                graph.replay()
                head(sets[1], 3, 2)
                torch.cuda.synchronize()
                for a, b in zip(out, ref):
                    assert all(torch.equal(p, q) for p, q in zip(a, b))
                assert torch.equal(last, ref_last)


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
def test_broadcast_inputs_get_summed_gradients(dtype, gpu_device):
    """One gate for all batch items, one value for all steps, one row of x for all rows, one row of
    weights for all columns: read through strides of 0."""
    import tempo_amd
    B, T, D = 3, 40, 12
    gate = _randn(gpu_device, dtype, 1, T, D).requires_grad_(True)
    value = _randn(gpu_device, dtype, B, 1, D, seed=1).requires_grad_(True)
    grad = _randn(gpu_device, dtype, B, T, D, seed=2)
    h, last = tempo_amd.gated_recurrence(gate.expand(B, T, D), value.expand(B, T, D))
    full = [t.detach().expand(B, T, D).contiguous() for t in (gate, value)]
    ref = R.recurrence(*full, None, None, grad, None)
    R.check(h, ref['h'], ref['h_tol'], 'h')
    got = torch.autograd.grad(h, (gate, value), grad)
    for g, name, dim, n in ((got[0], 'dgate', 0, B), (got[1], 'dvalue', 1, T)):
        # torch adds up n rounded terms, in fp32 at least, and rounds the sum
        want = ref[name].sum(dim, keepdim=True)
        size = (ref[name].abs() + ref[name + '_tol']).sum(dim, keepdim=True)
        R.check(g, want, ref[name + '_tol'].sum(dim, keepdim=True) + n * 2.0 ** -24 * size +
                R.rounding(size, dtype), name)

    M, K, N = 70, 24, 16
    x = _randn(gpu_device, dtype, 1, K, seed=3).requires_grad_(True)
    w = _randn(gpu_device, dtype, 1, K, seed=4).requires_grad_(True)
    grad = _randn(gpu_device, dtype, M, N, seed=5)
    y = tempo_amd.fused_linear(x.expand(M, K), w.expand(N, K), activation='tanh')
    ref = R.linear(x.detach().expand(M, K), w.detach().expand(N, K), None, None, 'tanh', grad)
    R.check(y, ref['y'], ref['y_tol'], 'y')
    got = torch.autograd.grad(y, (x, w), grad)
    for g, name, n in ((got[0], 'dx', M), (got[1], 'dweight', N)):
        want = ref[name].sum(0, keepdim=True)
        size = (ref[name].abs() + ref[name + '_tol']).sum(0, keepdim=True)
        R.check(g, want, ref[name + '_tol'].sum(0, keepdim=True) + n * 2.0 ** -24 * size +
                R.rounding(size, dtype), name)


def test_linear_of_more_than_32_bits_of_elements(gpu_device):
    """8.6 GB a tensor: 2^20 + 5 rows of 4104, forward and gradients, on operands whose sums are
    exact, against 64-bit values of rows next to every 2^32 bytes and elements."""
    import tempo_amd
    M, K, N = (1 << 20) + 5, 16, 4104
    gen = torch.Generator(device=gpu_device).manual_seed(0)

    def whole(most, *size):
        return torch.randint(-most, most + 1, size, generator=gen, device=gpu_device,
                             dtype=torch.int8).bfloat16()

    x, w = whole(3, M, K).requires_grad_(True), whole(3, N, K).requires_grad_(True)
    b = whole(2, N).requires_grad_(True)
    y = tempo_amd.fused_linear(x, w, b, activation='relu')
    grad = whole(1, M, N)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), grad)
    y, x, w, b = (t.detach() for t in (y, x, w, b))
    rows = torch.tensor([0, 1, (1 << 31) // N, (1 << 31) // N + 1, (1 << 32) // N,
                         (1 << 32) // N + 1, M - 2, M - 1] + list(range(777, M, 131101)),
                        device=gpu_device)
    z = x[rows].double() @ w.double().t().contiguous() + b.double()
    assert torch.equal(y[rows], z.clamp(min=0).bfloat16())
    dz = grad[rows].double() * (z > 0)
    assert torch.equal(dx[rows], (dz @ w.double()).bfloat16())
    # dW, db: whole numbers below 2^24, added up in fp32 here, too, a part of the rows at a time
    want_w, want_b = torch.zeros(N, K, device=gpu_device), torch.zeros(N, device=gpu_device)
    for i in range(0, M, 1 << 17):
        part = slice(i, min(i + (1 << 17), M))
        dz = grad[part] * (y[part] > 0)
        want_b += dz.sum(0, dtype=torch.float32)
        want_w += dz.float().t().contiguous() @ x[part].float()
    assert torch.equal(dw, want_w.bfloat16()) and torch.equal(db, want_b.bfloat16())


@pytest.mark.parametrize('B,T,D', [(140000, 16, 2048), (1, (1 << 22) + 37, 1032)])
def test_recurrence_of_more_than_32_bits_of_elements(B, T, D, gpu_device):
    """Batches and sequences beyond 2^32 elements, against the formula on parts of them."""
    import tempo_amd
    gen = torch.Generator(device=gpu_device).manual_seed(0)
    gate = torch.randint(-60, 61, (B, T, D), generator=gen, device=gpu_device,
                         dtype=torch.int8).half() / 16
    value = torch.randint(-64, 65, (B, T, D), generator=gen, device=gpu_device,
                          dtype=torch.int8).half() / 32
    h, last = tempo_amd.gated_recurrence(gate, value)
    if B > 1:
        for b in (0, (1 << 31) // (T * D), (1 << 32) // (T * D), B - 3):
            part = slice(b, b + 3)
            ref = R.recurrence(gate[part], value[part])
            R.check(h[part], ref['h'], ref['h_tol'], f'h of {b}')
            R.check(last[part], ref['last'], ref['last_tol'], f'last of {b}')
    else:
        for t in (0, (1 << 31) // D - 900, (1 << 32) // D - 900, T - 1800):
            # 900 steps in front forget the state, by a factor of exp(-sum z) < 2^-200
            ref = R.recurrence(gate[:, t:t + 1800], value[:, t:t + 1800])
            tail = slice(0 if t == 0 else 900, 1800)
            R.check(h[:, t:t + 1800][:, tail], ref['h'][:, tail], ref['h_tol'][:, tail],
                    f'h from {t}')
        R.check(last, ref['last'], ref['last_tol'], 'last')
    if B == 1:
        return
    del h, last
    leaf = gate.requires_grad_(True)
    h, _ = tempo_amd.gated_recurrence(leaf, value)
    (dgate,) = torch.autograd.grad(h, leaf, value)
    for b in (0, (1 << 31) // (T * D), (1 << 32) // (T * D), B - 3):
        part = slice(b, b + 3)
        ref = R.recurrence(gate.detach()[part], value[part], None, None, value[part], None)
        R.check(dgate[part], ref['dgate'], ref['dgate_tol'], f'dgate of {b}')


@pytest.mark.parametrize('dtype', DTYPES, ids=lambda d: str(d)[6:])
def test_smallest_numbers_count(dtype, gpu_device):
    """Subnormal inputs of each type are multiplied and carried as what they are."""
    import tempo_amd
    info = torch.finfo(dtype)
    tiny = torch.tensor([[1.0], [3.0], [-5.0]], dtype=torch.float64)
    tiny *= info.smallest_normal * info.eps
    x = tiny.to(dtype).to(gpu_device)
    assert torch.equal(x.double().cpu(), tiny)
    scale = 2.0 ** 10
    w = torch.full((1, 1), scale, dtype=dtype, device=gpu_device)
    assert torch.equal(tempo_amd.fused_linear(x, w).double().cpu(), tiny * scale)
    gate = torch.full((3, 1, 1), float('inf'), dtype=dtype, device=gpu_device)
    h, last = tempo_amd.gated_recurrence(gate, x[:, None])
    assert torch.equal(h, x[:, None]) and torch.equal(last.double().cpu(), tiny)


def test_arguments_that_are_no_tensors(gpu_device):
    import tempo_amd
    x, w = torch.zeros(2, 8, device=gpu_device), torch.zeros(4, 8, device=gpu_device)
    gate, state = torch.zeros(2, 3, 8, device=gpu_device), torch.zeros(2, 8, device=gpu_device)
    for bad in (lambda: tempo_amd.fused_linear(x, 3.0), lambda: tempo_amd.fused_linear(x, w, 1.0),
                lambda: tempo_amd.fused_linear(x, w, residual=1.0),
                lambda: tempo_amd.fused_linear(x, w, out=[1.0]),
                lambda: tempo_amd.fused_linear(x, w, activation=None),
                lambda: tempo_amd.gated_recurrence(gate, 1.0),
                lambda: tempo_amd.gated_recurrence(gate, gate, state=0.0),
                lambda: tempo_amd.gated_recurrence(gate, gate, state, lengths=[3, 3]),
                lambda: tempo_amd.gated_recurrence(gate, gate, state, out=[1.0]),
                lambda: tempo_amd.gated_recurrence(gate, gate, state, out=gate.clone(),
                                                   state_out=1.0)):
        with pytest.raises((TypeError, ValueError)):
            bad()
