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
