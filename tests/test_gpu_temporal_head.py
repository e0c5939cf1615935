"""The temporal head as it is used: backbone maps through the recurrent process layer into the
unprojection, trained and streamed."""
import pytest
import torch

import cases
import temporal_ref as R

pytestmark = pytest.mark.gpu

K, C, T = 24, 15, 3


def _head(dev, dtype=torch.float32, seed=0, hw=(14, 24), V=5, B=2):
    import tempo_amd
    gen = torch.Generator().manual_seed(seed)
    head = tempo_amd.RecurrentProcessLayerNHWC(K, C)
    with torch.no_grad():
        head.weight.copy_(torch.randn(head.weight.shape, generator=gen) / K ** 0.5)
        head.bias.copy_(torch.randn(head.bias.shape, generator=gen) * 0.3)
    maps = torch.randn(T * V * B, K, *hw, generator=gen).to(dtype)
    return head.to(dev), maps.to(dev)


def _reference(head, maps, V, state=None, grads=None):
    """Both operators in 64 bits; tolerances of the run of the two: the product's error enters
    the recurrence as one of its inputs, which it scales by at most 1 (value) and by
    |v - h| / 4 (gate) at each step, over all steps that are not forgotten."""
    images, _, H, W = maps.shape
    rows = maps.permute(0, 2, 3, 1).reshape(-1, K)
    w, b = (p.detach().to(maps.dtype) for p in (head.weight.flatten(1), head.bias))
    lin = R.linear(rows, w, b)
    both = lin['y'].view(T, -1, 2 * C).transpose(0, 1)
    tol = lin['y_tol'].view(T, -1, 2 * C).transpose(0, 1)
    rec = R.recurrence(both[..., :C].to(maps.dtype), both[..., C:].to(maps.dtype), state)
    peak = both[..., C:].abs().amax(dim=1, keepdim=True)
    if state is not None:
        peak = torch.maximum(peak, state.double().cpu().abs()[:, None])
    # the reference itself rounds the product once, the kernel once: twice the tolerance
    moved = 2 * T * (tol[..., C:].amax(1, keepdim=True) +
                     tol[..., :C].amax(1, keepdim=True) * 2 * peak / 4)
    return lin, rec, both, moved


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize('memory', [torch.contiguous_format, torch.channels_last], ids=str)
def test_recurrent_process_layer_maps(memory, dtype, gpu_device):
    V, B = 5, 2
    head, maps = _head(gpu_device, dtype)
    with torch.no_grad():
        out, state = head(maps.contiguous(memory_format=memory), V, T)
    assert len(out) == T and all(len(m) == V for m in out)
    _, rec, _, moved = _reference(head, maps, V)
    H, W = maps.shape[2:]
    got = torch.stack([torch.stack(m) for m in out])  # [T,V,B,C,H,W]
    got = got.permute(1, 2, 4, 5, 0, 3).reshape(-1, T, C)
    R.check(got, rec['h'], rec['h_tol'] + moved, 'maps')
    R.check(state, rec['last'], rec['last_tol'] + moved[:, 0], 'state')
    assert out[0][0].shape == (B, C, H, W)
    assert out[0][0].is_contiguous(memory_format=torch.channels_last)


def test_one_timestep_at_a_time(gpu_device):
    V = 5
    head, maps = _head(gpu_device)
    per = maps.shape[0] // T
    with torch.no_grad():
        whole, last = head(maps, V, T)
        state = None
        for t in range(T):
            step, state = head(maps[t * per:(t + 1) * per], V, 1, state)
            _, rec, _, moved = _reference(head, maps, V)
            tol = (rec['h_tol'] + moved)[:, t]
            for v in range(V):
                a, b = step[0][v].double().cpu(), whole[t][v].double().cpu()
                lim = tol.view(V, -1, *maps.shape[2:], C)[v].permute(0, 3, 1, 2)
                assert bool(((a - b).abs() <= 2 * lim).all())
    assert state.shape == last.shape


def test_head_and_unprojection_together(gpu_device):
    """Maps go into the root volume where they lie, with the values of NCHW copies; the
    gradients of a loss on the volume reach the head's parameters and the backbone's maps."""
    import tempo_amd
    spec = dict(cfg='panoptic', B=2, cube=[12, 10, 9], hm='noise', joints=C, seed=900)
    case = cases.to_device(cases.build_root(None, full=spec), gpu_device)
    V = len(case['args'][0])
    hw = tuple(case['args'][0][0].shape[2:])
    head, maps = _head(gpu_device, hw=hw, V=V)
    layer = tempo_amd.ProjectLayer(case['image_size'], case['heatmap_size'], 'mean')
    rest = case['args'][1:]
    maps.requires_grad_(True)
    out, _ = head(maps, V, T)

    def volume(m):
        return torch.stack([layer(m[t], *rest)[0] for t in range(T)])

    with torch.no_grad():
        in_place = volume(out)
        copied = volume([[m.contiguous() for m in ms] for ms in out])
    assert torch.equal(in_place, copied)

    gen = torch.Generator(device=gpu_device).manual_seed(1)
    seed = torch.randn(in_place.shape, generator=gen, device=gpu_device)
    leaves = [[m.detach().requires_grad_(True) for m in ms] for ms in out]
    flat = [m for ms in leaves for m in ms]
    g_maps = torch.autograd.grad(volume(leaves), flat, seed)
    params = [head.weight, head.bias, maps]
    mine = torch.autograd.grad([m for ms in out for m in ms], params, g_maps, retain_graph=True)

    lin, rec, both, moved = _reference(head, maps.detach(), V)
    g = torch.stack(list(g_maps)).view(T, V, -1, C, *hw).permute(1, 2, 4, 5, 0, 3)
    g = g.reshape(-1, T, C)
    back = R.recurrence(both[..., :C].float(), both[..., C:].float(), None, None, g, None)
    d_both = torch.cat([back['dgate'], back['dvalue']], -1)
    # the kernel's gates and values are off by `moved`: sigmoid and its slope change by at most
    # a quarter of that, the states by `moved` itself
    e = torch.cat([back['dgate_tol'], back['dvalue_tol']], -1)
    peak = both.abs().amax(dim=1, keepdim=True)[..., C:]
    size = g.double().cpu().abs().flip(1).cumsum(1).flip(1)
    e = e + torch.cat([moved * size * (1 + 2 * peak), moved * size], -1) * T
    rows = maps.detach().permute(0, 2, 3, 1).reshape(-1, K)
    d_rows = d_both.transpose(0, 1).reshape(-1, 2 * C)
    e_rows = e.transpose(0, 1).reshape(-1, 2 * C)
    ref = R.linear(rows, head.weight.detach().flatten(1), head.bias.detach(), None, 'none',
                   d_rows.float())
    W64 = head.weight.detach().flatten(1).double().cpu()
    X64 = rows.double().cpu()
    R.check(mine[0].flatten(1), ref['dweight'], ref['dweight_tol'] + e_rows.t() @ X64.abs(),
            'weight')
    R.check(mine[1], ref['dbias'], ref['dbias_tol'] + e_rows.sum(0), 'bias')
    R.check(mine[2].permute(0, 2, 3, 1).reshape(-1, K), ref['dx'],
            ref['dx_tol'] + e_rows @ W64.abs(), 'backbone maps')

    # the same in one go.  The unprojection's atomics add a texel's at most 12 x 10 x 9 terms in
    # another order: each sum moves by at most 1080 x 2^-24 of its terms' magnitudes, and what
    # follows is linear in it
    whole = torch.autograd.grad(volume(out), params, seed)
    size = torch.autograd.grad(volume(leaves), flat, seed.abs())
    grown = torch.autograd.grad([m for ms in head(maps, V, T)[0] for m in ms], params,
                                [1080 * 2.0 ** -24 * m.abs() for m in size])
    for a, b, lim in zip(whole, mine, grown):
        assert float((a - b).norm()) <= 4 * float(lim.norm()) + 1e-6 * float(b.norm())


def test_parameters_and_refusals(gpu_device):
    head, maps = _head(gpu_device)
    assert sorted(head.state_dict()) == ['bias', 'weight']
    assert tuple(head.weight.shape) == (2 * C, K, 1, 1)
    with pytest.raises(ValueError):
        head(maps, 7, T)
    with pytest.raises(ValueError):
        head(maps, 5, T, state=torch.zeros(3, C, device=gpu_device))
    with pytest.raises(TypeError):
        head(maps.cpu(), 5, T)


def test_results_in_place_are_seen_by_autograd(gpu_device):
    """What was saved of a tensor, or computed from it, is out of date once it was out or
    state_out: the backward pass says so, and the project layers unproject anew."""
    import tempo_amd
    x = torch.randn(6, 8, device=gpu_device)
    w = torch.randn(8, 8, device=gpu_device)
    leaf = torch.randn(6, 8, device=gpu_device, requires_grad=True)
    gate, value = (torch.randn(3, 2, 8, device=gpu_device) for _ in range(2))

    def linear(t):
        tempo_amd.fused_linear(x, w, out=t)

    def linear_over_residual(t):
        tempo_amd.fused_linear(x, w, residual=t, out=t)

    def states(t):
        tempo_amd.gated_recurrence(gate, value, out=t.view(3, 2, 8))

    def last_state(t):
        tempo_amd.gated_recurrence(gate, value, state=t[:3], state_out=t[:3])

    for write in (linear, linear_over_residual, states, last_state):
        saved = torch.randn(6, 8, device=gpu_device)
        loss = (leaf * saved).sum()
        with torch.no_grad():
            write(saved)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            loss.backward()
        with pytest.raises(NotImplementedError):
            write(leaf)
        with torch.inference_mode():
            write(torch.zeros(6, 8, device=gpu_device))
    before = x._version, w._version, gate._version
    linear(torch.zeros(6, 8, device=gpu_device))
    states(torch.zeros(6, 8, device=gpu_device))
    assert before == (x._version, w._version, gate._version)

    spec = dict(cfg='panoptic', B=1, cube=[12, 10, 9], hm='noise', joints=C, seed=901)
    case = cases.to_device(cases.build_root(None, full=spec), gpu_device)
    layer = tempo_amd.ProjectLayer(case['image_size'], case['heatmap_size'], 'mean')
    maps = [m.contiguous(memory_format=torch.channels_last).requires_grad_(True)
            for m in case['args'][0]]
    old = layer.forward_zmax(maps, *case['args'][1:])
    rows = maps[1].detach().permute(0, 2, 3, 1)
    new = rows.clone()
    with torch.no_grad():
        tempo_amd.fused_linear(new, 2 * torch.eye(C, device=gpu_device),
                               out=maps[1].permute(0, 2, 3, 1))
    got = layer.forward_zmax(maps, *case['args'][1:])
    fresh = tempo_amd.ProjectLayer(case['image_size'], case['heatmap_size'], 'mean')
    assert torch.equal(got, fresh.forward_zmax(maps, *case['args'][1:]))
    assert not torch.equal(got, old)


@pytest.mark.parametrize('grad_mode', [True, False])
def test_forward_mode_is_refused(grad_mode, gpu_device):
    """A tangent of any tensor that the results depend on: the call raises, it returns no
    constant.  Tensors without one pass inside of a dual level."""
    import torch.autograd.forward_ad as fwd

    import tempo_amd
    from tempo_amd import ops
    gen = torch.Generator(device=gpu_device).manual_seed(0)

    def some(*shape):
        return torch.randn(*shape, generator=gen, device=gpu_device)

    def dual(t):
        return fwd.make_dual(t, torch.ones_like(t))

    linear = [some(5, 8), some(4, 8), some(4), some(5, 4)]
    rec = [some(2, 3, 8), some(2, 3, 8), some(2, 8)]
    leaf, leaf3 = linear[0].clone().requires_grad_(True), rec[0].clone().requires_grad_(True)
    y, (h, last) = tempo_amd.fused_linear(leaf, linear[1]), tempo_amd.gated_recurrence(leaf3, rec[1])
    with torch.set_grad_enabled(grad_mode), fwd.dual_level():
        for i in range(4):
            args = [dual(t) if i == j else t for j, t in enumerate(linear)]
            with pytest.raises(NotImplementedError):
                tempo_amd.fused_linear(*args, activation='gelu')
            with pytest.raises(NotImplementedError):
                tempo_amd.fused_linear(*[a if i == j else a.clone().requires_grad_(True)
                                         for j, a in enumerate(args)])
            with pytest.raises(NotImplementedError):
                ops.linear_forward(*args)
        for i in range(3):
            args = [dual(t) if i == j else t for j, t in enumerate(rec)]
            with pytest.raises(NotImplementedError):
                tempo_amd.gated_recurrence(*args)
            with pytest.raises(NotImplementedError):
                ops.recurrence_forward(*args)
        assert torch.equal(tempo_amd.fused_linear(linear[0], linear[1]), y)
        assert torch.equal(tempo_amd.gated_recurrence(*rec[:2])[1], last)
        for call in (lambda: torch.autograd.grad(y, leaf, dual(torch.ones_like(y)),
                                                 retain_graph=True),
                     lambda: torch.autograd.grad(h, leaf3, dual(torch.ones_like(h)),
                                                 retain_graph=True),
                     lambda: torch.autograd.grad(last, leaf3, dual(torch.ones_like(last)),
                                                 retain_graph=True)):
            with pytest.raises(NotImplementedError):
                call()
    with pytest.raises(RuntimeError):  # function transforms hand over tensors without memory
        torch.func.jvp(lambda x: tempo_amd.fused_linear(x, linear[1]), (linear[0],),
                       (torch.ones_like(linear[0]),))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16], ids=lambda d: str(d)[6:])
def test_half_precision_head_and_unprojection_together(dtype, gpu_device):
    """16-bit maps are widened exactly on their way into the volume: the same values as fp32
    copies of them, in any memory order, and the same gradients up to one rounding of each."""
    import tempo_amd
    spec = dict(cfg='panoptic', B=2, cube=[12, 10, 9], hm='noise', joints=C, seed=902)
    case = cases.to_device(cases.build_root(None, full=spec), gpu_device)
    V = len(case['args'][0])
    hw = tuple(case['args'][0][0].shape[2:])
    head, maps = _head(gpu_device, dtype, hw=hw, V=V)
    layer = tempo_amd.ProjectLayer(case['image_size'], case['heatmap_size'], 'mean')
    rest = case['args'][1:]
    out, _ = head(maps, V, T)
    assert all(m.dtype == dtype for ms in out for m in ms)
    with torch.no_grad():
        for ms in out:
            volume = layer(ms, *rest)[0]
            assert volume.dtype == torch.float32
            for other in ([m.contiguous() for m in ms], [m.float() for m in ms],
                          [m.float().contiguous() for m in ms]):
                assert torch.equal(layer(other, *rest)[0], volume)
    volume = layer(out[1], *rest)[0]
    seed = torch.randn(volume.shape, device=gpu_device,
                       generator=torch.Generator(device=gpu_device).manual_seed(3))
    wide = [m.detach().float().requires_grad_(True) for m in out[1]]
    want = torch.autograd.grad(layer(wide, *rest)[0], wide, seed)
    size = torch.autograd.grad(layer(wide, *rest)[0], wide, seed.abs())
    got = torch.autograd.grad(volume, out[1], seed, retain_graph=True)
    for a, b, c in zip(got, want, size):
        assert a.dtype == dtype
        # the unprojection's atomics add at most 1080 terms in another order
        lim = R.rounding(b.double(), dtype) + 1.01 * 1080 * 2.0 ** -24 * c.double().abs()
        assert bool(((a.double() - b.double()).abs() <= lim).all())
    grads = torch.autograd.grad(volume, [head.weight, head.bias], seed)
    for g, p in zip(grads, (head.weight, head.bias)):
        assert g.dtype == p.dtype and bool(torch.isfinite(g).all()) and bool(g.any())


def test_recurrent_process_layer_on_nothing_and_on_one_texel(gpu_device):
    """No images, maps without texels: empty results of the right shapes; maps of a single texel
    are channel-last in any order."""
    head, maps = _head(gpu_device)
    for images, hw, T_ in ((0, (4, 6), 2), (10, (0, 6), 2), (10, (4, 0), 1)):
        out, state = head(torch.zeros(images, K, *hw, device=gpu_device), 5, T_)
        B = images // (5 * T_)
        assert len(out) == T_ and all(m.shape == (B, C) + hw for ms in out for m in ms)
        assert state.shape == (5 * B * hw[0] * hw[1], C)
    with torch.no_grad():
        one = maps[:, :, 3:4, 7:8]
        for m in (one, one.contiguous(), one.contiguous(memory_format=torch.channels_last)):
            out, state = head(m, 5, T)
            _, rec, _, moved = _reference(head, m, 5)
            got = torch.stack([torch.stack(ms) for ms in out]).permute(1, 2, 4, 5, 0, 3)
            R.check(got.reshape(-1, T, C), rec['h'], rec['h_tol'] + moved, 'maps')
            R.check(state, rec['last'], rec['last_tol'] + moved[:, 0], 'state')
