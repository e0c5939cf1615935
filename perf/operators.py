"""Measured cases of the temporal head's operators.

Two operators stand between a 2-D backbone and the unprojection when features are carried
over time:

* ``tempo_amd.fused_linear``: the 1x1 convolution of channel-last maps, i.e. a matrix product
  with bias, activation and residual in its epilogue, and its gradients;
* ``tempo_amd.gated_recurrence``: the gated linear recurrence over timesteps,
  ``h_t = (1 - z_t) h_{t-1} + z_t v_t`` with ``z = sigmoid(gate)``, and its gradients.

``own`` chooses between the plain torch formulas below and the framework's kernels.
"""
import math

import torch

own = False

_DTYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
_ACTIVATIONS = ('none', 'relu', 'silu', 'gelu', 'sigmoid', 'tanh')


def _linear(name, M, K, N, dtype, activation='none', bias=True, residual=False, train=False):
    return {'name': name, 'op': 'linear', 'M': M, 'K': K, 'N': N, 'dtype': dtype,
            'activation': activation, 'bias': bias, 'residual': residual, 'train': train}


def _recurrence(name, B, T, D, dtype, combined=False, time_major=False, state=False,
                lengths=False, train=False):
    return {'name': name, 'op': 'recurrence', 'B': B, 'T': T, 'D': D, 'dtype': dtype,
            'combined': combined, 'time_major': time_major, 'state': state,
            'lengths': lengths, 'train': train}


def listed():
    return [
        # ten tracked people, one new frame: the projection of their embeddings
        _linear('linear_track_step', 10, 256, 64, 'bfloat16', activation='tanh'),
        # eight rows against a wide weight: bound by reading the weight
        _linear('linear_few_rows', 8, 4096, 4096, 'float16', activation='silu', residual=True),
        # four frames of the five-view 128x240 backbone maps onto gate + candidate of 32
        # channels each, half precision, channel-last
        _linear('linear_maps', 4 * 5 * 128 * 240, 256, 64, 'bfloat16'),
        # the same 2-D head's layer trained in the reference's precision, one frame
        _linear('linear_maps_train', 5 * 128 * 240, 256, 32, 'float32', activation='relu',
                train=True),
        # an ordinary training step of a wide layer
        _linear('linear_train', 8192, 1024, 4096, 'bfloat16', activation='gelu', train=True),
        # sizes that no tile divides, rows that no 16-byte load is aligned to
        _linear('linear_ragged_train', 4999, 1021, 515, 'float16', activation='silu',
                residual=True, train=True),
        # the largest product: bound by the matrix units
        _linear('linear_wide', 16384, 4096, 4096, 'bfloat16', residual=True),
        # ten tracked people, one new frame: the recurrence with its carried state
        _recurrence('recurrence_step', 10, 1, 512, 'float32', state=True),
        # four timesteps of the five-view maps, gate and candidate side by side as one
        # product leaves them, time outermost, trained in fp32
        _recurrence('recurrence_maps_train', 5 * 128 * 240, 4, 32, 'float32', combined=True,
                    time_major=True, train=True),
        # one long recording in one pass
        _recurrence('recurrence_long', 1, 65536, 1024, 'bfloat16', state=True),
        # an ordinary training step over long clips
        _recurrence('recurrence_train', 8, 2048, 1024, 'bfloat16', state=True, train=True),
        # clips of different lengths in one padded batch, odd width
        _recurrence('recurrence_ragged_train', 13, 4097, 771, 'float16', lengths=True,
                    train=True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(['float32', 'float16', 'bfloat16'])
    train = rng.random() < 0.5
    if rng.random() < 0.5:
        flops_cap = 5.4e11 if dtype != 'float32' else 1.0e11
        while True:
            M = _log_int(rng, 1, 614400)
            K = _log_int(rng, 16, 4096)
            N = _log_int(rng, 15, 4096)
            if rng.random() < 0.5:  # half of them in widths that rows stay aligned for
                K, N = -(-K // 8) * 8, -(-N // 8) * 8
            if (2.0 * M * K * N * (3 if train else 1) <= flops_cap and
                    M * (K + N) <= 1.3e8):
                break
        return {'op': 'linear', 'M': M, 'K': K, 'N': N, 'dtype': dtype,
                'activation': rng.choice(_ACTIVATIONS), 'bias': rng.random() < 0.8,
                'residual': rng.random() < 0.4, 'train': train}
    while True:
        B = _log_int(rng, 1, 153600)
        T = _log_int(rng, 1, 65536)
        D = _log_int(rng, 8, 2048)
        if rng.random() < 0.5:
            D = -(-D // 8) * 8
        if B * T * D <= 6.7e7 / (2.5 if train else 1):
            break
    return {'op': 'recurrence', 'B': B, 'T': T, 'D': D, 'dtype': dtype,
            'combined': rng.random() < 0.5, 'time_major': rng.random() < 0.5,
            'state': rng.random() < 0.5, 'lengths': rng.random() < 0.4, 'train': train}


# ------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = _DTYPES[case['dtype']]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device='cuda', dtype=torch.float32)

    state = {'case': dict(case)}
    leaves = []

    def keep(name, t):
        if t is not None and case['train']:
            t.requires_grad_(True)
            leaves.append(t)
        state[name] = t

    if case['op'] == 'linear':
        M, K, N = case['M'], case['K'], case['N']
        keep('x', normal(M, K).to(dtype))
        bound = 1.0 / math.sqrt(K)  # the initialisation of nn.Conv2d(K, N, 1)
        keep('weight', ((torch.rand(N, K, generator=gen, device='cuda') * 2 - 1) *
                        (bound * math.sqrt(3.0))).to(dtype))
        keep('bias', ((torch.rand(N, generator=gen, device='cuda') * 2 - 1) * bound).to(dtype)
             if case['bias'] else None)
        keep('residual', normal(M, N).to(dtype) if case['residual'] else None)
        state['grad'] = normal(M, N).to(dtype) if case['train'] else None
    else:
        B, T, D = case['B'], case['T'], case['D']
        # channels remember over one step to a few hundred: the gate's bias is spread
        slow = torch.linspace(-5.0, 2.0, D, device='cuda')
        shape = (T, B) if case['time_major'] else (B, T)
        if case['combined']:
            both = torch.empty(*shape, 2 * D, dtype=dtype, device='cuda')
            both[..., :D] = (normal(*shape, D) + slow).to(dtype)
            both[..., D:] = normal(*shape, D).to(dtype)
            keep('gate', both.transpose(0, 1) if case['time_major'] else both)
            state['value'] = None
        else:
            gate = (normal(*shape, D) + slow).to(dtype)
            value = normal(*shape, D).to(dtype)
            keep('gate', gate.transpose(0, 1) if case['time_major'] else gate)
            keep('value', value.transpose(0, 1) if case['time_major'] else value)
        keep('state', normal(B, D) if case['state'] else None)
        state['lengths'] = None
        if case['lengths']:
            lengths = torch.randint(0, T + 1, (B,), generator=gen, device='cuda',
                                    dtype=torch.int32)
            lengths[0] = T
            state['lengths'] = lengths
        if case['train']:
            g = normal(*shape, D).to(dtype)
            state['grad'] = g.transpose(0, 1) if case['time_major'] else g
            state['grad_last'] = normal(B, D)
    state['leaves'] = leaves
    return state


# ---------------------------------------------------------------------------- plain forms

def _activate(z, name):
    if name == 'relu':
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == 'silu':
        return z / (1 + torch.exp(-z))
    if name == 'gelu':
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == 'sigmoid':
        return 1 / (1 + torch.exp(-z))
    if name == 'tanh':
        return torch.tanh(z)
    return z


def _slope(z, name):
    if name == 'relu':
        return (z > 0).to(z.dtype)
    if name == 'silu':
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == 'gelu':
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5))) +
                z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    if name == 'sigmoid':
        s = 1 / (1 + torch.exp(-z))
        return s * (1 - s)
    if name == 'tanh':
        t = torch.tanh(z)
        return 1 - t * t
    return torch.ones_like(z)


def _plain_linear(s):
    case = s['case']
    dtype = _DTYPES[case['dtype']]
    x, w = s['x'].float(), s['weight'].float()
    z = x @ w.t()
    if s['bias'] is not None:
        z = z + s['bias'].float()
    y = _activate(z, case['activation'])
    if s['residual'] is not None:
        y = y + s['residual'].float()
    outs = [y.to(dtype)]
    if case['train']:
        dz = s['grad'].float() * _slope(z, case['activation'])
        outs += [(dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
        if s['bias'] is not None:
            outs.append(dz.sum(0).to(dtype))
        if s['residual'] is not None:
            outs.append(s['grad'])
    return outs


def _scan(a, b):
    """All states of s_t = a_t s_{t-1} + b_t (s before the first is 0), dim 1 is time, by
    doubling the span that each position has taken in."""
    step, T = 1, a.shape[1]
    a, b = a.clone(), b.clone()
    while step < T:
        b[:, step:] = b[:, step:] + a[:, step:] * b[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return b


def _plain_recurrence(s):
    case = s['case']
    dtype = _DTYPES[case['dtype']]
    B, T, D = case['B'], case['T'], case['D']
    # products of many decays: 64 bits beyond a few steps
    wide = torch.float32 if T <= 16 else torch.float64
    gate, value = s['gate'], s['value']
    if value is None:
        gate, value = gate[..., :D], gate[..., D:]
    gate, value = gate.to(wide), value.to(wide)
    z, f = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    u = z * value
    lengths = s['lengths']
    if lengths is not None:
        valid = (torch.arange(T, device=gate.device)[None, :] < lengths[:, None])[..., None]
        zero = torch.zeros((), dtype=wide, device=gate.device)
        z, f, u = (torch.where(valid, t, zero) for t in (z, f, u))
    start = s['state'].to(wide) if s['state'] is not None else gate.new_zeros(B, D)
    u[:, 0] = u[:, 0] + f[:, 0] * start
    h = _scan(f, u)
    if lengths is None:
        last = h[:, -1]
    else:
        row = (lengths.long() - 1).clamp(min=0)[:, None, None].expand(B, 1, D)
        last = torch.where((lengths > 0)[:, None], h.gather(1, row)[:, 0], start)
    outs = [h.to(dtype), last.float()]
    if case['train']:
        g, glast = s['grad'].to(wide), s['grad_last'].to(wide)
        before = torch.cat([start[:, None], h[:, :-1]], dim=1)
        if lengths is None:
            g = g.clone()
            g[:, -1] = g[:, -1] + glast
        else:
            g = torch.where(valid, g, zero)
            end = torch.arange(T, device=gate.device)[None, :] == lengths[:, None] - 1
            g = g + torch.where(end[..., None], glast[:, None], zero)
        after = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], dim=1)
        e = _scan(after.flip(1), g.flip(1)).flip(1)
        dgate = e * z * f * (value - before)
        dvalue = e * z
        if lengths is not None:
            dgate, dvalue = (torch.where(valid, t, zero) for t in (dgate, dvalue))
        if s['value'] is None:
            outs.append(torch.cat([dgate, dvalue], dim=-1).to(dtype))
        else:
            outs += [dgate.to(dtype), dvalue.to(dtype)]
        if s['state'] is not None:
            dstart = f[:, 0] * e[:, 0]
            if lengths is not None:
                dstart = torch.where((lengths > 0)[:, None], dstart, glast)
            outs.append(dstart.float())
    return outs


# ----------------------------------------------------------------------------- one pass

def run(state):
    case = state['case']
    if not own:
        with torch.no_grad():
            return _plain_linear(state) if case['op'] == 'linear' else _plain_recurrence(state)
    import tempo_amd
    with torch.set_grad_enabled(case['train']):
        if case['op'] == 'linear':
            y = tempo_amd.fused_linear(state['x'], state['weight'], state['bias'],
                                       residual=state['residual'],
                                       activation=case['activation'])
            outs, seeds = [y], [state['grad']]
        else:
            h, last = tempo_amd.gated_recurrence(state['gate'], state['value'],
                                                 state=state['state'],
                                                 lengths=state['lengths'])
            outs, seeds = [h, last], [state['grad'], state['grad_last']] if case['train'] else []
        if case['train']:
            outs = outs + list(torch.autograd.grad(outs, state['leaves'], seeds))
    return [t.detach() for t in outs]


def work(case):
    size = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'linear':
        M, K, N = case['M'], case['K'], case['N']
        rows, cols, weight = M * N, M * K, N * K
        vec = N if case['bias'] else 0
        res = rows if case['residual'] else 0
        elements = cols + weight + vec + res + rows
        flops = 2.0 * M * K * N
        if case['train']:  # the output's gradient in; those of x, weight, bias, residual out
            elements += rows + cols + weight + vec + res
            flops *= 3
        return {'bytes': float(elements * size), 'flops': flops}
    n, lanes = case['B'] * case['T'] * case['D'], case['B'] * case['D']
    elements, wide = 3 * n, lanes * (2 if case['state'] else 1)
    flops = 12.0 * n
    if case['train']:
        elements += 3 * n
        wide += lanes * (2 if case['state'] else 1)
        flops += 16.0 * n
    return {'bytes': float(elements * size + wide * 4), 'flops': flops}


# ------------------------------------------------------------------- 64-bit definitions

_EXACT = {
    'none': (lambda z: z, lambda z: torch.ones_like(z)),
    'relu': (lambda z: z.clamp(min=0), lambda z: (z > 0).double()),
    'silu': (lambda z: z * z.sigmoid(),
             lambda z: z.sigmoid() + z * z.sigmoid() * (-z).sigmoid()),
    'gelu': (lambda z: z * torch.special.ndtr(z),
             lambda z: torch.special.ndtr(z) + z * (-z * z / 2).exp() / math.sqrt(math.tau)),
    'sigmoid': (torch.sigmoid, lambda z: z.sigmoid() * (-z).sigmoid()),
    'tanh': (torch.tanh, lambda z: z.cosh().reciprocal().square()),
}


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    with torch.no_grad():
        s = prepare(dict(case, train=False), seed) if not case['train'] else prepare(case, seed)
        return _exact_linear(case, s) if case['op'] == 'linear' else _exact_recurrence(case, s)


def _exact_linear(case, s):
    act, slope = _EXACT[case['activation']]
    x, w = s['x'].double(), s['weight'].double()
    z = torch.mm(x, w.transpose(0, 1).contiguous())
    if s['bias'] is not None:
        z += s['bias'].double()
    y = act(z)
    if s['residual'] is not None:
        y = y + s['residual'].double()
    if not case['train']:
        return [y]
    dz = slope(z) * s['grad'].double()
    outs = [y, torch.mm(dz, w), torch.mm(dz.transpose(0, 1).contiguous(), x)]
    if s['bias'] is not None:
        outs.append(dz.sum(dim=0))
    if s['residual'] is not None:
        outs.append(s['grad'].double())
    return outs


def _exact_recurrence(case, s):
    """Step by step through time, forth and back."""
    B, T, D = case['B'], case['T'], case['D']
    gate, value = (s['gate'], s['value']) if s['value'] is not None else \
        s['gate'].split(D, dim=-1)
    gate = gate.transpose(0, 1).double().contiguous()  # [T,B,D]
    value = value.transpose(0, 1).double().contiguous()
    inside = None
    if s['lengths'] is not None:
        steps = torch.arange(T, device=gate.device, dtype=torch.int32)
        inside = (steps[:, None] < s['lengths'][None, :])[..., None]
    open_, shut = torch.sigmoid(gate), torch.sigmoid(-gate)
    h = torch.empty_like(gate)
    first = s['state'].double() if s['state'] is not None else gate.new_zeros(B, D)
    now = first
    for t in range(T):
        new = torch.addcmul(open_[t] * value[t], shut[t], now)
        now = new if inside is None else torch.where(inside[t], new, now)
        h[t] = now
    shown = h if inside is None else h * inside
    outs = [shown.transpose(0, 1), now]
    if not case['train']:
        return outs
    dh = s['grad'].transpose(0, 1).double().contiguous()
    dgate, dvalue = torch.empty_like(gate), torch.empty_like(gate)
    pull = s['grad_last'].double()  # gradient of the state after step t
    for t in range(T - 1, -1, -1):
        total = dh[t] + pull
        if inside is not None:
            total = torch.where(inside[t], total, torch.zeros_like(total))
        previous = h[t - 1] if t else first
        dvalue[t] = total * open_[t]
        dgate[t] = dvalue[t] * shut[t] * (value[t] - previous)
        passed = total * shut[t]
        pull = passed if inside is None else torch.where(inside[t], passed, pull)
    dgate, dvalue = dgate.transpose(0, 1), dvalue.transpose(0, 1)
    outs += [torch.cat([dgate, dvalue], dim=-1)] if s['value'] is None else [dgate, dvalue]
    if s['state'] is not None:
        outs.append(pull)
    return outs
