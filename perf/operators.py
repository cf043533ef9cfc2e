"""The cases on which the language-model operators are measured: the gated linear recurrence
(`linear_scan` and its gradient, `linear_scan_step`), the norms around a block fused with its gate and
residual (`norm_residual` and its gradient) and the log probabilities of given tokens
(`token_logprobs` and its gradient).

`own` false: the operators' plain forms, elementary torch operations in float32.
`own` true: the calls a user makes of tcu_scope_b200.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # One new token for each of 64 sequences of a recurrent layer; states live in a pool of slots.
        {"name": "step 64 x 2048", "op": "step", "batch": 64, "dim": 2048, "pool": 96, "gate": "log",
         "a_type": "bf16", "type": "bf16"},
        # A training step of one recurrent layer: forward, then the gradients.
        {"name": "scan train 8 x 2048 x 2560", "op": "scan", "batch": 8, "tokens": 2048, "dim": 2560,
         "gate": "log", "a_type": "bf16", "type": "bf16", "packed": False, "train": True},
        # One long document read in before generation, continued from an earlier state, decays in 32 bits.
        {"name": "scan 1 x 65537 x 1024", "op": "scan", "batch": 1, "tokens": 65537, "dim": 1024,
         "gate": "decay", "a_type": "f32", "type": "bf16", "packed": False, "train": False},
        # Sequences of many lengths packed one behind the other, as a fine-tuning batch is; gates from logits.
        {"name": "scan train packed 37 sequences", "op": "scan", "batch": 37, "tokens": 20011, "dim": 1000,
         "gate": "sigmoid", "a_type": "f16", "type": "f16", "packed": True, "train": True},
        # One new token for each of 16 sequences: both norms around a block, its learned gate, the residual.
        {"name": "norm 16 x 4096", "op": "norm", "rows": 16, "dim": 4096, "type": "bf16", "w_type": "bf16",
         "groups": 1, "act": "none", "pre": True, "residual": True, "train": False},
        # A training step through the same, 16384 tokens.
        {"name": "norm train 16384 x 4096", "op": "norm", "rows": 16384, "dim": 4096, "type": "bf16",
         "w_type": "f32", "groups": 1, "act": "none", "pre": True, "residual": True, "train": True},
        # The gated norm behind a recurrence, a gate for every element, an odd width in 32 bits.
        {"name": "norm train 1777 x 1111 f32", "op": "norm", "rows": 1777, "dim": 1111, "type": "f32",
         "w_type": "f32", "groups": 1777, "act": "silu", "pre": False, "residual": False, "train": True},
        # Eight long prompts, a gate row for each of them.
        {"name": "norm 32768 x 5120", "op": "norm", "rows": 32768, "dim": 5120, "type": "f16", "w_type": "f16",
         "groups": 8, "act": "sigmoid", "pre": True, "residual": True, "train": False},
        # What a server answers with each sampled token: its log probability and the 20 best alternatives.
        {"name": "logprobs 16 x 128000 top 20", "op": "logprobs", "rows": 16, "vocab": 128000, "type": "bf16",
         "top": 20, "masked": 0.3, "train": False},
        # Scoring of given texts.
        {"name": "logprobs 4096 x 128000 top 8", "op": "logprobs", "rows": 4096, "vocab": 128000,
         "type": "bf16", "top": 8, "masked": 0.0, "train": False},
        # A policy update: log probabilities and entropies, then the gradient of the logits; rows of odd length.
        {"name": "logprobs train 2048 x 100003", "op": "logprobs", "rows": 2048, "vocab": 100003,
         "type": "bf16", "top": 0, "masked": 0.0, "train": True},
        # A small batch with logits in 32 bits.
        {"name": "logprobs train 300 x 32000 f32", "op": "logprobs", "rows": 300, "vocab": 32000, "type": "f32",
         "top": 5, "masked": 0.1, "train": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan", "norm", "norm", "norm", "logprobs", "logprobs", "logprobs"])
    kind = rng.choice(["f16", "bf16", "bf16", "f32"])
    if op == "step":
        batch = _spread(rng, 1, 512)
        return {"op": op, "batch": batch, "dim": _spread(rng, 64, 8192), "pool": batch + rng.randint(0, 64),
                "gate": rng.choice(["decay", "log", "sigmoid"]), "a_type": rng.choice([kind, "f32"]), "type": kind}
    if op == "scan":
        dim = rng.choice([_spread(rng, 64, 4096), 64 * rng.randint(1, 64)])
        packed = rng.random() < 0.4
        elements = _spread(rng, 1 << 16, 1 << 25)
        batch = _spread(rng, 1, 64)
        tokens = max(1, min(elements // dim // (1 if packed else batch), 65537))
        return {"op": op, "batch": batch, "tokens": max(tokens, batch) if packed else tokens, "dim": dim,
                "gate": rng.choice(["decay", "log", "sigmoid"]), "a_type": rng.choice([kind, "f32"]), "type": kind,
                "packed": packed, "train": rng.random() < 0.6}
    if op == "norm":
        dim = rng.choice([_spread(rng, 64, 8192), 64 * rng.randint(1, 128)])
        groups = rng.choice([1, 1, rng.randint(2, 16), 0])
        pre, train = rng.random() < 0.6, rng.random() < 0.5
        most = (1 << 27) // BYTES[kind] // (2 if train else 1) // dim
        rows = _spread(rng, 1, min(32768, most))
        rows = -(-rows // max(groups, 1)) * max(groups, 1)
        return {"op": op, "rows": rows, "dim": dim, "type": kind, "w_type": rng.choice([kind, "f32"]),
                "groups": groups or rows, "act": rng.choice(["none", "sigmoid", "silu"]), "pre": pre,
                "residual": pre or rng.random() < 0.5, "train": train}
    vocab = _spread(rng, 1000, 160000)
    train = rng.random() < 0.4
    return {"op": op, "rows": _spread(rng, 1, min(4096, (1 << 27) // vocab)), "vocab": vocab, "type": kind,
            "top": rng.choice([0, 1, rng.randint(2, 32)]), "masked": rng.choice([0.0, 0.0, 0.5]), "train": train}


# ---------------------------------------------------------------------------------------- inputs


def _gates(case, shape, normal):
    """Gates of layers that remember between a few and about a thousand tokens."""
    if case["gate"] == "sigmoid":
        g = 3 + 2 * normal(*shape)
    else:
        g = -torch.exp(-4 + 1.5 * normal(*shape)).clamp_(max=8.0)
        if case["gate"] == "decay":
            g = torch.exp(g)
    return g.to(TYPES[case["a_type"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    s = dict(case)
    kind = TYPES[case["type"]]
    if case["op"] == "step":
        b, d = case["batch"], case["dim"]
        s["a"], s["x"] = _gates(case, (b, d), normal), normal(b, d).to(kind)
        s["state"] = normal(case["pool"], d)
        s["slots"] = torch.randperm(case["pool"], generator=gen, device="cuda")[:b].to(torch.int32)
    elif case["op"] == "scan":
        b, t, d = case["batch"], case["tokens"], case["dim"]
        shape = (t, d) if case["packed"] else (b, t, d)
        s["a"], s["x"] = _gates(case, shape, normal), normal(*shape).to(kind)
        s["h0"] = normal(b, d)
        s["offsets"] = None
        if case["packed"]:
            cuts = torch.randint(0, t + 1, (b - 1,), generator=gen, device="cuda").sort().values
            ends = torch.tensor([0, t], device="cuda")
            s["offsets"] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
        if case["train"]:
            s["dh"], s["dlast"] = normal(*shape).to(kind), normal(b, d)
    elif case["op"] == "norm":
        r, d = case["rows"], case["dim"]
        w_kind = TYPES[case["w_type"]]
        s["z"] = (normal(r, d) * (0.5 + normal(r, 1).abs())).to(kind)
        s["res"] = (3 * normal(r, d)).to(kind) if case["residual"] else None
        s["post"] = (1 + 0.2 * normal(d)).to(w_kind)
        s["gate_rows"] = (0.5 + 0.5 * normal(case["groups"], d)).to(kind)
        s["pre_w"] = (1 + 0.2 * normal(d)).to(w_kind) if case["pre"] else None
        s["scale"] = 0.75
        if case["train"]:
            s["dout"] = normal(r, d).to(kind)
            s["dnormed"] = normal(r, d).to(kind) if case["pre"] else None
    else:
        r, v = case["rows"], case["vocab"]
        logits = 2.5 * normal(r, v)
        target = torch.randint(0, v, (r,), generator=gen, device="cuda")
        row = torch.arange(r, device="cuda")
        logits[row, target] += 12 * torch.rand(r, generator=gen, device="cuda")  # some rows sure, some not
        if case["masked"]:  # tokens that the grammar of the answer forbids
            out = torch.rand(v, generator=gen, device="cuda") < case["masked"]
            keep = logits[row, target].clone()
            logits[:, out] = -math.inf
            logits[row, target] = keep
        s["logits"], s["target"] = logits.to(kind), target
        if case["train"]:
            s["dlp"], s["dent"] = normal(r), 0.1 * normal(r)
    return s


# ------------------------------------------------------------------------------------ plain forms


def _gated(gate, a, x):
    """(f, u, 1 - f) of h_t = f h_{t-1} + u."""
    if gate == "sigmoid":
        keep, take = 1 / (1 + torch.exp(-a)), 1 / (1 + torch.exp(a))
        return keep, take * x, take
    return (torch.exp(a) if gate == "log" else a), x, None


def _recur(f, u):
    """h_t = f_t h_{t-1} + u_t along dimension 1, by pairs: neighbours are joined, the half as long
    recurrence is solved, and its answers are spread back."""
    n = f.shape[1]
    if n == 1:
        return u
    m = n // 2
    f0, f1, u0, u1 = f[:, 0:2 * m:2], f[:, 1::2], u[:, 0:2 * m:2], u[:, 1::2]
    odd = _recur(f1 * f0, f1 * u0 + u1)
    h = torch.empty_like(u)
    h[:, 1::2] = odd
    h[:, 0] = u[:, 0]
    k = n - n // 2 - 1  # even places behind the first
    h[:, 2::2] = f[:, 2::2] * odd[:, :k] + u[:, 2::2]
    return h


def _plain_scan(s):
    a, x, h0 = s["a"].float(), s["x"].float(), s["h0"]
    f, u, take = _gated(s["gate"], a, x)
    shape = x.shape
    if s["packed"]:
        f, u = f[None], u[None]
        off = s["offsets"].long()
        full = off[1:] > off[:-1]
        first, end = off[:-1][full], off[1:][full] - 1
        lane = torch.zeros_like(first)
        of_seq = full.nonzero()[:, 0]
    else:
        lane = torch.arange(shape[0], device=x.device)
        first, end, of_seq = torch.zeros_like(lane), torch.full_like(lane, shape[1] - 1), lane
    start_f = f[lane, first]
    cut, u = f.clone(), u.clone()
    cut[lane, first] = 0
    u[lane, first] += start_f * h0[of_seq]
    h = _recur(cut, u)
    last = h0.clone()
    last[of_seq] = h[lane, end]
    kind = s["x"].dtype
    y = h.reshape(shape).to(kind)
    if not s["train"]:
        return {"h": y, "last": last}
    dh = s["dh"].float().reshape(u.shape).clone()
    dh[lane, end] += s["dlast"][of_seq]
    ahead = torch.cat([cut[:, 1:], torch.zeros_like(cut[:, :1])], 1)
    g = _recur(ahead.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    before[lane, first] = h0[of_seq]
    dh0 = s["dlast"].clone()
    dh0[of_seq] = start_f * g[lane, first]
    g, before, f = g.reshape(shape), before.reshape(shape), f.reshape(shape)
    if s["gate"] == "sigmoid":
        da, dx = g * (before - x) * f * take, g * take
    else:
        da, dx = (g * before * f if s["gate"] == "log" else g * before), g
    return {"h": y, "last": last, "da": da.to(s["a"].dtype), "dx": dx.to(kind), "dh0": dh0}


def _plain_step(s):
    f, u, _ = _gated(s["gate"], s["a"].float(), s["x"].float())
    at = s["slots"].long()
    h = f * s["state"][at] + u
    s["state"][at] = h
    return {"h": h.to(s["x"].dtype), "state": s["state"]}


def _act(kind, g):
    """The gate and its derivative."""
    if kind == "none":
        return g, torch.ones_like(g)
    sig = 1 / (1 + torch.exp(-g))
    if kind == "sigmoid":
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


def _plain_norm(s):
    z, rows, dim, groups = s["z"].float(), s["rows"], s["dim"], s["groups"]
    kind = s["z"].dtype
    post = s["post"].float()
    gate, slope = _act(s["act"], s["gate_rows"].float())
    gate, slope = gate[:, None], slope[:, None]  # groups, 1, dim
    each = (groups, rows // groups, dim)
    rz = torch.rsqrt((z * z).mean(1, keepdim=True) + EPS)
    zn = z * rz
    n = zn * post
    out = (s["scale"] * gate * n.reshape(each)).reshape(rows, dim)
    if s["residual"]:
        out = out + s["res"].float()
    got = {"out": out.to(kind)}
    if s["pre"]:
        pre = s["pre_w"].float()
        ro = torch.rsqrt((out * out).mean(1, keepdim=True) + EPS)
        on = out * ro
        got["normed"] = (on * pre).to(kind)
    if not s["train"]:
        return got
    do = s["dout"].float()
    if s["pre"]:
        du = s["dnormed"].float()
        v = du * pre
        got["dpre"] = (du * on).sum(0).to(s["pre_w"].dtype)
        do = do + ro * (v - on * (v * on).mean(1, keepdim=True))
    if s["residual"]:
        got["dres"] = do.to(kind)
    d3 = do.reshape(each) * s["scale"]
    got["dgate"] = ((d3 * n.reshape(each)).sum(1) * slope[:, 0]).to(kind)
    dn = (d3 * gate).reshape(rows, dim)
    got["dpost"] = (dn * zn).sum(0).to(s["post"].dtype)
    v = dn * post
    got["dz"] = (rz * (v - zn * (v * zn).mean(1, keepdim=True))).to(kind)
    return got


def _plain_logprobs(s):
    x, target, k = s["logits"].float(), s["target"], s["top"]
    rows = torch.arange(x.shape[0], device=x.device)
    most = x.max(1, keepdim=True).values
    e = torch.exp(x - most)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    p = e / total
    entropy = log_total - torch.where(p > 0, p * (x - most), 0.0).sum(1, keepdim=True)
    lse = most + log_total
    got = {"logprob": x[rows, target] - lse[:, 0], "entropy": entropy[:, 0], "lse": lse[:, 0]}
    if k:
        # a whole number for each logit that orders as (value, lower index first), so that none are equal
        bits = (x + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, -(1 << 31) - bits, bits)
        key = bits * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=x.device))
        got["top_index"] = key.topk(k, 1).indices
        got["top_logprob"] = x.gather(1, got["top_index"]) - lse
    if s["train"]:
        logp = x - lse
        d = -p * s["dlp"][:, None] - s["dent"][:, None] * torch.where(p > 0, p * (logp + entropy), 0.0)
        d[rows, target] += s["dlp"]
        got["dlogits"] = d.to(s["logits"].dtype)
    return got


# ------------------------------------------------------------------------------- one pass of a case


def run(s):
    if own:
        return _own(s)
    return {"step": _plain_step, "scan": _plain_scan, "norm": _plain_norm, "logprobs": _plain_logprobs}[s["op"]](s)


def _own(s):
    import tcu_scope_b200 as tcu

    if s["op"] == "step":
        return {"h": tcu.linear_scan_step(s["a"], s["x"], s["state"], gate=s["gate"], slots=s["slots"]),
                "state": s["state"]}
    if s["op"] == "scan":
        if not s["train"]:
            h, last = tcu.linear_scan(s["a"], s["x"], gate=s["gate"], h0=s["h0"], offsets=s["offsets"])
            return {"h": h, "last": last}
        states = tcu.linear_scan_states(s["x"], offsets=s["offsets"])
        h, last = tcu.linear_scan(s["a"], s["x"], gate=s["gate"], h0=s["h0"], offsets=s["offsets"], states=states)
        da, dx, dh0 = tcu.linear_scan_backward(s["dh"], s["a"], s["x"], states, gate=s["gate"], dlast=s["dlast"],
                                               offsets=s["offsets"])
        return {"h": h, "last": last, "da": da, "dx": dx, "dh0": dh0}
    if s["op"] == "norm":
        args = dict(post_weight=s["post"], gate=s["gate_rows"], gate_act=s["act"], scale=s["scale"],
                    pre_weight=s["pre_w"], eps=EPS)
        out, normed = tcu.norm_residual(s["z"], s["res"], **args)
        got = {"out": out}
        if s["pre"]:
            got["normed"] = normed
        if s["train"]:
            d = tcu.norm_residual_backward(s["dout"], s["dnormed"], s["z"], s["res"], **args)
            got.update(dz=d.dz, dgate=d.dgate, dpost=d.dpost_weight)
            if s["residual"]:
                got["dres"] = d.dresidual
            if s["pre"]:
                got["dpre"] = d.dpre_weight
        return got
    lp = tcu.token_logprobs(s["logits"], s["target"], top=s["top"])
    got = {"logprob": lp.logprob, "entropy": lp.entropy, "lse": lp.lse}
    if s["top"]:
        got.update(top_index=lp.top_index, top_logprob=lp.top_logprob)
    if s["train"]:
        got["dlogits"] = tcu.token_logprobs_backward(s["logits"], s["target"], lp.lse, lp.entropy,
                                                     dlogprob=s["dlp"], dentropy=s["dent"])
    return got


# ------------------------------------------------------------------------------------------ work


def work(case):
    n, e = 1, BYTES[case["type"]]
    if case["op"] == "step":
        n = case["batch"] * case["dim"]
        return {"bytes": n * (BYTES[case["a_type"]] + 2 * e + 8) + 4 * case["batch"], "flops": 4 * n}
    if case["op"] == "scan":
        ends = 4 * case["batch"] * case["dim"]
        n = case["tokens"] * case["dim"] * (1 if case["packed"] else case["batch"])
        if case["train"]:  # a, x, dh in; h, da, dx out
            return {"bytes": n * (2 * BYTES[case["a_type"]] + 4 * e) + 4 * ends, "flops": 10 * n}
        return {"bytes": n * (BYTES[case["a_type"]] + 2 * e) + 2 * ends, "flops": 3 * n}
    if case["op"] == "norm":
        n, w = case["rows"] * case["dim"], BYTES[case["w_type"]] * case["dim"]
        arrays = 2 + case["residual"] + case["pre"]  # z, out
        ends = (1 + case["pre"]) * w + case["groups"] * case["dim"] * e
        if case["train"]:  # and dout, dz
            return {"bytes": n * e * (arrays + 2 + case["residual"] + case["pre"]) + 2 * ends, "flops": 30 * n}
        return {"bytes": n * e * arrays + ends, "flops": 10 * n}
    n = case["rows"] * case["vocab"]
    small = case["rows"] * (8 + 12 + 12 * case["top"])
    return {"bytes": n * e * (2 if case["train"] else 1) + small, "flops": n * (10 if case["train"] else 5)}


# ------------------------------------------------------------- from the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"step": _exact_step, "scan": _exact_scan, "norm": _exact_norm, "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_gate(s):
    a, x = s["a"].double(), s["x"].double()
    if s["gate"] == "sigmoid":
        return torch.sigmoid(a), x * torch.sigmoid(-a)
    return (a.exp() if s["gate"] == "log" else a), x


def _exact_step(s):
    f, u = _exact_gate(s)
    state = s["state"].double()
    slots = s["slots"].tolist()
    h = torch.stack([f[i] * state[j] + u[i] for i, j in enumerate(slots)])
    for i, j in enumerate(slots):
        state[j] = h[i]
    return {"h": h, "state": state}


def _exact_scan(s):
    """Token by token, forwards and back, one sequence at a time where they are packed."""
    if s["packed"]:
        cuts = s["offsets"].tolist()
        parts = [slice(i, j) for i, j in zip(cuts, cuts[1:])]
        if s["tokens"] > 30000:
            return None
    f, u = _exact_gate(s)
    names = ["h", "da", "dx"] if s["train"] else ["h"]
    got = {n: torch.empty_like(f) for n in names}
    last = s["h0"].double()
    dh0 = s["dlast"].double() if s["train"] else None
    if s["packed"]:
        for i, part in enumerate(parts):
            _one_exact(s, f, u, got, part, last[i], dh0[i] if s["train"] else None)
    else:
        # the sequences side by side: time first
        s = dict(s, **{n: s[n].transpose(0, 1) for n in ("a", "x", "dh") if n in s})
        got = {n: v.transpose(0, 1) for n, v in got.items()}
        _one_exact(s, f.transpose(0, 1), u.transpose(0, 1), got, slice(0, s["tokens"]), last, dh0)
        got = {n: v.transpose(0, 1) for n, v in got.items()}
    got["last"] = last
    if s["train"]:
        got["dh0"] = dh0
    return got


def _one_exact(s, f, u, got, part, h, g):
    """The sequence whose time steps are `part`, from the state h, which becomes the last one, and with
    the last state's gradient g, which becomes the first one's."""
    for t in range(part.start, part.stop):
        h.mul_(f[t]).add_(u[t])
        got["h"][t] = h
    if g is None:
        return
    h0 = s["h0"].double()
    if s["packed"]:
        h0 = h0[_sequence_of(s, part)]
    for t in range(part.stop - 1, part.start - 1, -1):
        before = got["h"][t - 1] if t > part.start else h0
        d = s["dh"][t].double() + g
        if s["gate"] == "sigmoid":
            got["da"][t] = d * (before - s["x"][t].double()) * f[t] * torch.sigmoid(-s["a"][t].double())
            got["dx"][t] = d * torch.sigmoid(-s["a"][t].double())
        else:
            got["da"][t] = d * before * (f[t] if s["gate"] == "log" else 1.0)
            got["dx"][t] = d
        torch.mul(d, f[t], out=g)


def _sequence_of(s, part):
    """The last sequence that begins at part.start: those before it there are empty."""
    return max(i for i, v in enumerate(s["offsets"].tolist()[:-1]) if v == part.start)


def _exact_norm(s):
    """The gradients by autograd, not from written-out formulas."""
    names = ["z", "post", "gate_rows"] + (["res"] if s["residual"] else []) + (["pre_w"] if s["pre"] else [])
    v = {n: s[n].double().requires_grad_(s["train"]) for n in names}
    per = s["rows"] // s["groups"]
    gate = {"none": lambda g: g, "sigmoid": torch.sigmoid, "silu": lambda g: g * torch.sigmoid(g)}[s["act"]](v["gate_rows"])
    n = v["z"] / (v["z"].pow(2).mean(1, keepdim=True) + EPS).sqrt() * v["post"]
    out = s["scale"] * gate.repeat_interleave(per, 0) * n
    if s["residual"]:
        out = out + v["res"]
    got, ends, grads = {"out": out}, [out], [s["dout"].double()] if s["train"] else []
    if s["pre"]:
        got["normed"] = out / (out.pow(2).mean(1, keepdim=True) + EPS).sqrt() * v["pre_w"]
        ends.append(got["normed"])
        if s["train"]:
            grads.append(s["dnormed"].double())
    if s["train"]:
        d = dict(zip(names, torch.autograd.grad(ends, [v[n] for n in names], grads)))
        to = {"z": "dz", "post": "dpost", "gate_rows": "dgate", "res": "dres", "pre_w": "dpre"}
        got.update({to[n]: t for n, t in d.items()})
    return {n: t.detach() for n, t in got.items()}


def _exact_logprobs(s):
    k, parts = s["top"], []
    for i in range(0, s["rows"], 256):
        x = s["logits"][i:i + 256].double()
        target = s["target"][i:i + 256, None]
        logp = torch.log_softmax(x, 1)
        p = logp.exp()
        entropy = -(p * logp.masked_fill(p == 0, 0.0)).sum(1)
        part = {"logprob": logp.gather(1, target)[:, 0], "entropy": entropy, "lse": torch.logsumexp(x, 1)}
        if k:
            order = x.sort(dim=1, descending=True, stable=True).indices[:, :k]
            part.update(top_index=order, top_logprob=logp.gather(1, order))
        if s["train"]:
            dlp, dent = (s[n][i:i + 256, None].double() for n in ("dlp", "dent"))
            hit = torch.zeros_like(p).scatter_(1, target, 1.0)
            part["dlogits"] = dlp * (hit - p) - dent * p * (logp.masked_fill(p == 0, 0.0) + entropy[:, None])
        parts.append(part)
    return {n: torch.cat([q[n] for q in parts]) for n in parts[0]}
