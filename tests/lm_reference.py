"""Plain 64-bit forms of the language-model operators, with bounds on what 32-bit arithmetic may be
off: u = 2^-24 is the largest relative error of one float32 rounding, and every bound is a count of
roundings times u times the sum of the absolute values that were rounded, carried through the
formula as the values are.  A result of type t may be off by half a step, finfo(t).eps / 2, on top."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what):
    """|got - want| <= bound + half a step of got's type (and half its smallest subnormal)."""
    got64 = got.detach().double().cpu()
    want, bound = want.double().cpu(), bound.double().cpu()
    assert got64.shape == want.shape, (what, got64.shape, want.shape)
    room = bound + half_step(got.dtype) * (want.abs() + bound) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got64 - want).abs()
    bad = ~(off <= room)
    assert not bool(bad.any()), (what, int(bad.sum()), off[bad].max().item() if bad.any() else 0,
                                 bad.nonzero()[0].tolist(), got64[bad][0].item(), want[bad][0].item())


# Roundings of one step of the recurrence: the gate (expf and the reciprocal 2 ulp = 4 u each, an
# addition, a product), 1 - f times x, the product of gates and the fused multiply-add: 12.
STEP = 12 * U


def gates(gate, a, x):
    """(f, u, 1 - f)"""
    if gate == "sigmoid":
        f, rest = torch.sigmoid(a), torch.sigmoid(-a)
        return f, rest * x, rest
    return (a.exp() if gate == "log" else a), x, None


def recur(f, u, h0):
    """h_t = f_t h_{t-1} + u_t along dimension 0."""
    h, out = h0, torch.empty_like(u)
    for t in range(u.shape[0]):
        h = f[t] * h + u[t]
        out[t] = h
    return out


def linear_scan(gate, a, x, h0, dh=None, dlast=None):
    """One sequence, (tokens, dim) in float64 on the CPU: {name: (value, bound)}."""
    f, u, rest = gates(gate, a, x)
    n = x.shape[0]
    got = {}
    h = recur(f, u, h0)
    size = recur(f.abs(), u.abs(), h0.abs())          # what the absolute values add up to
    off = recur(f.abs(), STEP * size, torch.zeros_like(h0))  # each step's roundings, carried on
    got["h"] = (h, off)
    got["last"] = (h[-1], off[-1]) if n else (h0, torch.zeros_like(h0))
    if dh is None:
        return got
    # g[t]: the gradient of h_t, all of it; ahead[t]: the gate between t and t + 1
    ahead = torch.cat([f[1:], torch.ones_like(f[:1])])[:n]
    g = recur(ahead.flip(0), dh.flip(0), dlast).flip(0) if n else dh
    gsize = recur(ahead.abs().flip(0), dh.abs().flip(0), dlast.abs()).flip(0) if n else dh
    goff = recur(ahead.abs().flip(0), STEP * gsize.flip(0), torch.zeros_like(dlast)).flip(0) if n else dh
    before = torch.cat([h0[None], h[:-1]])[:n]
    bsize = torch.cat([h0.abs()[None], size[:-1]])[:n]
    boff = torch.cat([torch.zeros_like(h0)[None], off[:-1]])[:n]
    if gate == "sigmoid":
        slope = f * rest
        got["da"] = (g * (before - x) * slope,
                     ((goff + STEP * g.abs()) * (before - x).abs() + g.abs() * (boff + STEP * (bsize + x.abs()))) * slope)
        got["dx"] = (g * rest, (goff + STEP * g.abs()) * rest)
    else:
        slope = f if gate == "log" else torch.ones_like(f)
        got["da"] = (g * before * slope, ((goff + STEP * g.abs()) * before.abs() + g.abs() * (boff + STEP * bsize)) * slope.abs())
        got["dx"] = (g, goff)
    got["dh0"] = (f[0] * g[0], (f[0] * goff[0]).abs() + STEP * gsize[0] * f[0].abs()) if n else (dlast, torch.zeros_like(dlast))
    return got
