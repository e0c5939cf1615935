"""Plain 64-bit forms of the temporal head's operators, step by step, with the error that the
kernels' fp32 arithmetic may make at most beside each value."""
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(ref, dtype):
    """One rounding of ``ref`` to ``dtype``: half a step of the value, at least half the
    smallest subnormal."""
    info = torch.finfo(dtype)
    return ref.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def recurrence(gate, value, state=None, lengths=None, grad_h=None, grad_last=None):
    """dict of h, last and (with grad_h / grad_last) dgate, dvalue, dstate in fp64 on the CPU,
    and of their tolerances under the key + '_tol' for kernels that return ``gate.dtype``.

    Let u = 2^-24 and rho the relative error of the smaller weight w = min(z, f): the kernel's
    exponential, reciprocal and product are good to 8 u in fp32; in 16 bits the exponent's
    argument is rounded too, |g| log2(e) u ln 2 <= 32 u for |g| <= 32, in all 64 u at most.
    A step  h' = base + w (other - base)  then errs by at most  u |h'| + 2 u w D + rho w D with
    D = |v| + |h|; errors shrink by f per step, so they add up to at most n = min(T, 1/min z)
    steps' worth:  err(h) <= M (n u + 2 rho + 4 u),  M the largest |v|, |state| of the lane
    (w <= z or the error is forgotten by the factor f = w <= 1/2 at once: twice w D rho).
    Chunks add one such step per chunk.  Backwards  p' = f (dh + p)  errs relatively by at
    most 4 u + rho per step against E_t = |dh_t| + f_{t+1} E_{t+1}; weighted by the same
    products of f that make up E, n steps' worth at most n (4 u + rho) E."""
    dtype = gate.dtype
    out_dtype = dtype
    g, v = gate.double().cpu(), value.double().cpu()
    B, T, D = g.shape
    n_valid = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    inside = (torch.arange(T)[None, :] < n_valid[:, None])[..., None]
    g, v = torch.where(inside, g, torch.zeros(())), torch.where(inside, v, torch.zeros(()))
    z, f = torch.sigmoid(g), torch.sigmoid(-g)
    h = torch.zeros(B, T, D, dtype=torch.float64)
    first = state.double().cpu() if state is not None else torch.zeros(B, D, dtype=torch.float64)
    now = first
    for t in range(T):
        now = torch.where(inside[:, t], f[:, t] * now + z[:, t] * v[:, t], now)
        h[:, t] = now
    u = 2.0 ** -24
    rho = (8 if dtype == torch.float32 else 64) * u
    zmin = torch.where(inside, z, torch.ones(())).amin(dim=1) if T else torch.ones(B, D)
    n = torch.clamp(1.0 / zmin, max=float(max(T, 1)))
    # chunk boundaries: pass 2 applies one more step per chunk of at least 32 steps
    n = n * (1 + 1.0 / 16) + 2
    peak = torch.maximum(v.abs().amax(dim=1), first.abs()) if T else first.abs()
    err = peak * (n * u + 2 * rho + 4 * u)  # [B, D]
    r = {'h': h * inside, 'last': now.clone()}
    r['h_tol'] = err[:, None] * inside + rounding(r['h'], out_dtype)
    r['last_tol'] = err + rounding(r['last'], torch.float32)
    if grad_h is None and grad_last is None:
        return r
    dh = torch.zeros(B, T, D, dtype=torch.float64) if grad_h is None else grad_h.double().cpu()
    pull = torch.zeros(B, D, dtype=torch.float64) if grad_last is None else \
        grad_last.double().cpu()
    size = pull.abs()
    for name in ('dgate', 'dvalue', 'dgate_tol', 'dvalue_tol'):
        r[name] = torch.zeros(B, T, D, dtype=torch.float64)
    rel = (n + 4) * (4 * u + rho)
    zero = torch.zeros((), dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        on = inside[:, t]
        before = h[:, t - 1] if t else first
        e = torch.where(on, dh[:, t] + pull, zero)
        big = torch.where(on, dh[:, t].abs() + size, zero)
        zf = z[:, t] * f[:, t]
        r['dvalue'][:, t] = z[:, t] * e
        r['dgate'][:, t] = zf * (v[:, t] - before) * e
        r['dvalue_tol'][:, t] = z[:, t] * big * rel
        # |h| <= peak; the difference v - h errs by err + u (|v| + |h|), the factors by 2 rho
        r['dgate_tol'][:, t] = zf * big * (2 * peak * (rel + 2 * rho) + err)
        pull = torch.where(on, f[:, t] * e, pull)
        size = torch.where(on, f[:, t] * big, size)
    r['dstate'] = pull
    r['dstate_tol'] = size * rel + rounding(pull, torch.float32)
    for name in ('dgate', 'dvalue'):
        r[name + '_tol'] += rounding(r[name], out_dtype) * inside
    return r


def check(got, ref, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f'{what}: not finite'
    over = (got - ref).abs() - tol
    assert bool((over <= 0).all()), (
        f'{what}: {int((over > 0).sum())} of {over.numel()} beyond the tolerance, worst '
        f'{float((got - ref).abs().max()):.3e} at tolerance '
        f'{float(tol.flatten()[over.flatten().argmax()]):.3e}')


# ------------------------------------------------------------------------- fused linear layer

_ACT = {
    'none': (lambda z: z, lambda z: torch.ones_like(z)),
    'relu': (lambda z: z.clamp(min=0), lambda z: (z > 0).double()),
    'silu': (lambda z: z * z.sigmoid(), lambda z: z.sigmoid() * (1 + z * (-z).sigmoid())),
    'gelu': (lambda z: z * torch.special.ndtr(z),
             lambda z: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) * 0.3989422804014327),
    'sigmoid': (torch.sigmoid, lambda z: z.sigmoid() * (-z).sigmoid()),
    'tanh': (torch.tanh, lambda z: 1 - torch.tanh(z) ** 2),
}
# largest |act'|, |act''|
_STEEP = {'none': (1.0, 0.0), 'relu': (1.0, 0.0), 'silu': (1.1, 0.5), 'gelu': (1.13, 0.8),
          'sigmoid': (0.25, 0.1), 'tanh': (1.0, 0.77)}


def linear(x, weight, bias=None, residual=None, activation='none', grad=None):
    """dict of y (and dx, dweight, dbias) in fp64 on the CPU with tolerances for kernels that
    return ``x.dtype``.

    Let u = 2^-24.  A sum of n products in fp32, in any order, errs by at most
    (n + 1) u sum |a b|; the matrix units may drop what lies under the last bit of an operand's
    alignment, another n u.  z errs by dz0 = 2 (K + 2) u (|x| |W|^T + |b|), the activation by its
    steepness times that plus a few u of its own (16 bits: 2^-19 of its value, erfc's 2^-22
    absolute times |z|).  Backwards: z is kept to half a step, so act' errs by its steepness
    times (dz0 + half a step of z); dz is rounded by half a step; the products add their
    n + 1 terms' error and one rounding."""
    dtype = x.dtype
    X, W = x.double().cpu(), weight.double().cpu()
    shape = X.shape
    X = X.reshape(-1, shape[-1])
    M, K = X.shape
    N = W.shape[0]
    u = 2.0 ** -24
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    act, slope = _ACT[activation]
    steep, bend = _STEEP[activation]
    z = X @ W.t()
    z_err = X.abs() @ W.abs().t()
    if bias is not None:
        z = z + bias.double().cpu()
        z_err = z_err + bias.double().cpu().abs()
    z_err = 2 * (K + 2) * u * z_err
    own = (2.0 ** -21 if dtype == torch.float32 else 2.0 ** -19)
    a = act(z)
    y = a
    y_err = steep * z_err
    if activation != 'none' and activation != 'relu':
        y_err = y_err + own * a.abs() + 2.0 ** -22 * (z.abs() + 1)
    if residual is not None:
        res = residual.double().cpu().reshape(M, N)
        y = y + res
        y_err = y_err + 2 * u * (a.abs() + res.abs())
    r = {'y': y.reshape(shape[:-1] + (N,))}
    r['y_tol'] = (y_err + rounding(y, dtype)).reshape(r['y'].shape)
    if grad is None:
        return r
    g = grad.double().cpu().reshape(M, N)
    s = slope(z)
    dz = g * s
    s_err = bend * (z_err + half * z.abs()) + own * (1 + z.abs()) * (activation not in
                                                                     ('none', 'relu'))
    if activation == 'relu':
        # the sign of a z within its error of 0 may be either
        s_err = (z.abs() <= z_err).double()
    dz_err = g.abs() * s_err + 4 * u * dz.abs()
    dz_op = dz_err if activation == 'none' and half else \
        dz_err + (rounding(dz, dtype) if half else 0)
    if activation == 'none':
        dz_op = torch.zeros_like(dz)
    big = dz.abs() + dz_op
    r['dx'] = (dz @ W).reshape(shape)
    r['dx_tol'] = (dz_op @ W.abs() + 2 * (N + 2) * u * (big @ W.abs())).reshape(shape) + \
        rounding(r['dx'], dtype)
    r['dweight'] = dz.t() @ X
    # parts of a split sum are joined in fp32, too: twice the terms' bound covers that
    r['dweight_tol'] = dz_op.t() @ X.abs() + 2 * (M + 2) * u * (big.t() @ X.abs()) + \
        rounding(r['dweight'], dtype)
    r['dbias'] = dz.sum(0)
    r['dbias_tol'] = dz_err.sum(0) + 2 * (M + 2) * u * dz.abs().sum(0) + \
        rounding(r['dbias'], dtype)
    return r
