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
# An exponential below float32's smallest normal number, 2^-126, counts as 0: a gate is off by less than that, and
# what it multiplies by less than that times its size.
FLUSH = 2.0 ** -126


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
    flush = FLUSH * torch.cat([h0.abs()[None], size[:-1]])[:n]
    off = recur(f.abs(), STEP * size + flush, torch.zeros_like(h0))  # each step's roundings, carried on
    got["h"] = (h, off)
    got["last"] = (h[-1], off[-1]) if n else (h0, torch.zeros_like(h0))
    if dh is None:
        return got
    # g[t]: the gradient of h_t, all of it; ahead[t]: the gate between t and t + 1
    ahead = torch.cat([f[1:], torch.ones_like(f[:1])])[:n]
    g = recur(ahead.flip(0), dh.flip(0), dlast).flip(0) if n else dh
    gsize = recur(ahead.abs().flip(0), dh.abs().flip(0), dlast.abs()).flip(0) if n else dh
    gflush = FLUSH * torch.cat([gsize[1:], dlast.abs()[None]])[:n]
    goff = recur(ahead.abs().flip(0), (STEP * gsize + gflush).flip(0), torch.zeros_like(dlast)).flip(0) if n else dh
    before = torch.cat([h0[None], h[:-1]])[:n]
    bsize = torch.cat([h0.abs()[None], size[:-1]])[:n]
    boff = torch.cat([torch.zeros_like(h0)[None], off[:-1]])[:n]
    if gate == "sigmoid":
        slope = f * rest
        got["da"] = (g * (before - x) * slope,
                     ((goff + STEP * g.abs()) * (before - x).abs() + g.abs() * (boff + STEP * (bsize + x.abs()))) * slope + FLUSH * gsize * (bsize + x.abs()))
        got["dx"] = (g * rest, (goff + STEP * g.abs()) * rest + FLUSH * gsize)
    else:
        slope = f if gate == "log" else torch.ones_like(f)
        got["da"] = (g * before * slope, ((goff + STEP * g.abs()) * before.abs() + g.abs() * (boff + STEP * bsize)) * slope.abs() + FLUSH * gsize * bsize)
        got["dx"] = (g, goff)
    got["dh0"] = (f[0] * g[0], (f[0] * goff[0]).abs() + STEP * gsize[0] * f[0].abs() + FLUSH * gsize[0]) if n else (dlast, torch.zeros_like(dlast))
    return got


class Run:
    """A value with a bound on what 32-bit arithmetic may be off: running error analysis.  Every
    operation carries the bounds of its operands on and adds its own roundings, as many units u of the
    result's size as are given (1 for a rounded operation, 4 for a function within 2 ulp)."""

    def __init__(self, value, bound=None):
        self.v = value
        self.e = torch.zeros_like(value) if bound is None else bound

    def _new(self, value, bound, roundings):
        return Run(value, bound + roundings * U * (value.abs() + bound))

    def __add__(self, o):
        return self._new(self.v + o.v, self.e + o.e, 1)

    def __sub__(self, o):
        return self._new(self.v - o.v, self.e + o.e, 1)

    def __mul__(self, o):
        if not isinstance(o, Run):
            o = Run(torch.as_tensor(float(o), dtype=torch.float64).to(self.v.device))
        return self._new(self.v * o.v, self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e, 1)

    def call(self, f, slope, roundings=4):
        """f of the value; slope: a bound on |f'| around it."""
        return self._new(f(self.v), slope * self.e, roundings)

    def sum(self, dim, keepdim=False, chain=None):
        """A sum in which every term passes through at most `chain` additions."""
        n = self.v.shape[dim] if chain is None else chain
        size = (self.v.abs() + self.e).sum(dim, keepdim=keepdim)
        return Run(self.v.sum(dim, keepdim=keepdim), self.e.sum(dim, keepdim=keepdim) + n * U * size)

    def index(self, f):
        return Run(f(self.v), f(self.e))


def norm_residual(z, residual, post, gate, act, scale, pre, eps, dout=None, dnormed=None):
    """Rows of float64 on the CPU, gate expanded to rows or None: {name: Run}; the gradients of post,
    pre and gate before they are summed over rows are post_rows, pre_rows and gate_rows."""
    dim = z.shape[1]
    chain = 16 + 5 + 6  # a thread's elements, its warp, the block's warps
    # The sums that come behind the first norm may be put together from sums of products of the inputs and of
    # 1 / rms(z), 2^n of it: the roundings of each part, and the 25 u of 1 / rms(z), count by the size of the parts.
    # (Unless they cancel to less than a quarter, when they are summed directly.)
    parts = (chain + 25 + 8) * U

    def scaled(y, size=None):  # y / rms(y) and 1 / rms(y)
        mean = (y * y).sum(1, True, chain) * (1.0 / dim)
        if size is not None:
            mean.e = mean.e + parts * torch.minimum(size.sum(1, keepdim=True), 8 * (y.v * y.v).sum(1, keepdim=True)) / dim
        ms = Run(mean.v + eps, mean.e + U * (mean.v + eps))
        r = ms.call(lambda m: m.rsqrt(), 0.51 * (ms.v - ms.e).clamp(min=1e-300) ** -1.5)
        return y * r, r

    got = {}
    z_ = Run(z)
    zn, rz = scaled(z_) if post is not None else (z_, None)
    n = zn * Run(post) if post is not None else zn
    if gate is not None:
        sig = torch.sigmoid(gate)
        value = {"none": gate, "sigmoid": sig, "silu": gate * sig}[act]
        g = Run(value, 0 * value if act == "none" else 12 * U * value.abs())
        t = 1 - sig if act != "none" else None
        slope = {"none": lambda: Run(torch.ones_like(gate)), "sigmoid": lambda: Run(sig * t, 26 * U * sig * t),
                 "silu": lambda: Run(sig * (1 + gate * t), 30 * U * sig * (1 + (gate * t).abs()))}[act]()
    else:
        g = Run(torch.ones_like(z))
    o = n * g * scale
    branch = o.v.abs()
    rest = residual.abs() if residual is not None else torch.zeros_like(z)
    if residual is not None:
        o = o + Run(residual)
    got["out"] = o
    if pre is not None:
        on, ro = scaled(o, (branch + rest) ** 2)
        got["normed"] = on * Run(pre)
    if dout is None:
        return got
    d = Run(dout)
    if pre is not None:
        v = Run(dnormed) * Run(pre)
        mean = (v * on).sum(1, True, chain + 2) * (1.0 / dim)
        mean.e = mean.e + parts * (v.v.abs() * (branch + rest)).sum(1, keepdim=True) * ro.v / dim
        k = (ro.v * mean.v).abs()
        got["pre_rows"] = Run(dnormed) * on
        d = d + ro * (v - on * mean)
    got["dresidual"] = d
    ds = d * scale
    if gate is not None:
        got["gate_rows"] = ds * n * slope
    dn = ds * g
    if post is not None:
        got["post_rows"] = dn * zn
        w = dn * Run(post)
        mean = (w * zn).sum(1, True, chain + 2) * (1.0 / dim)
        size = dout.abs()
        if pre is not None:
            size = size + ro.v * v.v.abs() + k * ro.v * (branch + rest)
        mean.e = mean.e + parts * ((g.v * post * scale).abs() * zn.v.abs() * size).sum(1, keepdim=True) / dim
        got["dz"] = rz * (w - zn * mean)
    else:
        got["dz"] = dn
    return got


def token_logprobs(x, targets, top, dlp=None, dent=None):
    """Rows of float64 on the CPU: {name: (value, bound)}, top_index without a bound.  The bounds count the
    roundings of x - r (u |x - r|), its product (u) and 2^d (4 u) into each exponential, the chain of additions,
    and the logarithm's 2 ulp."""
    rows, vocab = x.shape
    most = x.max(1, keepdim=True).values
    dead = torch.isinf(most)                      # nothing but -inf
    far = torch.where(dead | torch.isinf(x), torch.zeros_like(x), x - torch.where(dead, 0.0, most))
    p = torch.where(dead, torch.zeros_like(x), torch.softmax(torch.where(dead, 0.0, x), 1))
    logp = torch.where(dead | torch.isinf(x), torch.zeros_like(x), torch.log_softmax(torch.where(dead, 0.0, x), 1))
    chain = vocab / 128 + 60                      # additions and rebasings a term passes through
    # what d = (x - r) log2(e) is off, in natural units, weighted: the relative error of s
    rel = (p * (6 * far.abs() + 8) * U).sum(1) + chain * U
    log_s = torch.where(dead[:, 0], 0.0, (torch.logsumexp(torch.where(dead, 0.0, x), 1) - torch.where(dead[:, 0], 0.0, most[:, 0])))
    lse = torch.where(dead[:, 0], most[:, 0], torch.logsumexp(torch.where(dead, 0.0, x), 1))
    off = rel + 8 * U * (log_s + 1)               # of log s
    got = {"lse": (lse, off + U * torch.where(dead[:, 0], 0.0, lse.abs())),
           "entropy": (-(p * logp).sum(1), off + (p * far.abs() * (6 * far.abs() + chain + 12) * U).sum(1) + 4 * U * (log_s + 1) + (p * far.abs()).sum(1) * rel)}
    row = torch.arange(rows)
    if targets is not None:
        t = targets.clamp(0, vocab - 1)
        got["logprob"] = (torch.where(torch.isinf(x[row, t]), -torch.inf, logp[row, t]), off + 4 * U * (far[row, t].abs() + log_s))
    if top:
        order = torch.where(torch.isnan(x), torch.inf, x).sort(dim=1, descending=True, stable=True).indices[:, :top]
        got["top_index"] = order
        got["top_logprob"] = (torch.where(torch.isinf(x.gather(1, order)), -torch.inf, logp.gather(1, order)),
                              off[:, None] + 4 * U * (far.gather(1, order).abs() + log_s[:, None]))
    if dlp is not None:
        hit = torch.zeros_like(x)
        hit[row, targets] = 1
        hit[dead[:, 0]] = 0
        ent = got["entropy"][0]
        g = dlp[:, None] * (hit - p) - dent[:, None] * p * (logp + ent[:, None])
        # log p from lse: its rounding (or 2^-16 at most), x - lse, the product, and the exponential
        lost = off + torch.where(dead[:, 0], 0.0, torch.minimum(lse.abs(), torch.full_like(lse, 256.0))) * U
        rel_p = lost[:, None] + (4 * logp.abs() + 8) * U
        size = dlp.abs()[:, None] + dent.abs()[:, None] * (logp.abs() + ent[:, None])
        got["dlogits"] = (g, p * (size * (rel_p + 6 * U) + dent.abs()[:, None] * (lost[:, None] + got["entropy"][1][:, None] + 4 * U * logp.abs()))
                          + 2 * U * (hit * dlp[:, None].abs())
                          # a probability below float32's smallest normal number, 2^-126, counts as 0, so p is off by
                          # less than that, and p (dlp + dH (log p + H)) by less than that times the bracket
                          + 2.0 ** -126 * size)
    return got
