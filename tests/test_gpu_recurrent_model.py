"""The language-model operators one after the other, as a small model with recurrent layers uses them: embeddings,
layers of a norm, projections, the gated recurrence and the gated norm with its residual, logits, log
probabilities and entropies; a training step with every gradient, and generation token by token, against
the same model in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
DIM, INNER, VOCAB, LAYERS, EPS = 48, 64, 101, 2, 1e-6


def parameters(seed):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    p = {"embed": n(VOCAB, DIM), "norm0": 1 + 0.1 * n(DIM), "head": n(DIM, VOCAB) / DIM ** 0.5}
    for i in range(LAYERS):
        p[f"in{i}"] = n(DIM, 3 * INNER) / DIM ** 0.5   # gate logits, inputs and output gates of the recurrence
        p[f"out{i}"] = n(INNER, DIM) / INNER ** 0.5
        p[f"post{i}"] = 1 + 0.1 * n(INNER)
        p[f"norm{i + 1}"] = 1 + 0.1 * n(DIM)
        p[f"scale{i}"] = 0.5 + 0.1 * n(DIM)
    return p


def plain(p, tokens, targets, lengths):
    """Mean log probability of the targets plus a little entropy, by autograd in 64 bits; logits too."""
    x = p["embed"][tokens]
    u = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * p["norm0"]
    for i in range(LAYERS):
        a, v, o = (u @ p[f"in{i}"]).split(INNER, -1)
        f = torch.sigmoid(a + 2)
        rows, at = [], 0
        for n in lengths:
            h = torch.zeros(INNER, dtype=x.dtype)
            for t in range(at, at + n):
                h = f[t] * h + (1 - f[t]) * v[t]
                rows.append(h)
            at += n
        h = torch.stack(rows)
        y = h / (h.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * p[f"post{i}"] * (o * torch.sigmoid(o))
        x = x + 0.7 * p[f"scale{i}"] * (y @ p[f"out{i}"])
        u = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * p[f"norm{i + 1}"]
    logits = u @ p["head"]
    logp = torch.log_softmax(logits, -1)
    entropy = -(logp.exp() * logp).sum(-1)
    return logp.gather(-1, targets[:, None])[:, 0], entropy, logits


def forward(tcu, p, tokens, offsets, targets):
    """The model on the operators; everything that the backward pass wants, too."""
    keep = {}
    x = p["embed"][tokens]
    # the first norm alone: no block before it
    keep["x0"] = x
    _, u = tcu.norm_residual(x, pre_weight=p["norm0"], eps=EPS)
    for i in range(LAYERS):
        proj = u @ p[f"in{i}"]
        proj[:, :INNER] += 2
        a, v, o = proj[:, :INNER], proj[:, INNER:2 * INNER], proj[:, 2 * INNER:]  # views: rows 3 * INNER apart
        states = tcu.linear_scan_states(v, offsets)
        h, _ = tcu.linear_scan(a, v, gate="sigmoid", offsets=offsets, states=states)
        y, _ = tcu.norm_residual(h, post_weight=p[f"post{i}"], gate=o, gate_act="silu", eps=EPS)
        z = y @ p[f"out{i}"]
        keep[i] = (u, a, v, o, states, h, y, z, x)
        x, u = tcu.norm_residual(z, x, gate=p[f"scale{i}"], scale=0.7, pre_weight=p[f"norm{i + 1}"], eps=EPS)
    keep["u"] = u
    keep["logits"] = u @ p["head"]
    return keep, tcu.token_logprobs(keep["logits"], targets)


def backward(tcu, p, tokens, offsets, targets, keep, lp, dlp, dent):
    g = {}
    dlogits = tcu.token_logprobs_backward(keep["logits"], targets, lp.lse, lp.entropy, dlogprob=dlp, dentropy=dent)
    g["head"] = keep["u"].t() @ dlogits
    du, dx = dlogits @ p["head"].t(), None
    for i in reversed(range(LAYERS)):
        u, a, v, o, states, h, y, z, x = keep[i]
        d = tcu.norm_residual_backward(dx, du, z, x, gate=p[f"scale{i}"], scale=0.7, pre_weight=p[f"norm{i + 1}"], eps=EPS)
        g[f"scale{i}"], g[f"norm{i + 1}"], dx = d.dgate, d.dpre_weight, d.dresidual
        g[f"out{i}"] = y.t() @ d.dz
        dy = d.dz @ p[f"out{i}"].t()
        d = tcu.norm_residual_backward(dy, None, h, post_weight=p[f"post{i}"], gate=o, gate_act="silu", eps=EPS)
        g[f"post{i}"] = d.dpost_weight
        da, dv, _ = tcu.linear_scan_backward(d.dz, a, v, states, gate="sigmoid", offsets=offsets)
        dproj = torch.cat([da, dv, d.dgate], 1)
        g[f"in{i}"] = u.t() @ dproj
        du = dproj @ p[f"in{i}"].t()
    d = tcu.norm_residual_backward(dx, du, keep["x0"], pre_weight=p["norm0"], eps=EPS)
    g["norm0"] = d.dpre_weight
    g["embed"] = torch.zeros_like(p["embed"]).index_add_(0, tokens, d.dz)
    return g


def batch(seed, lengths):
    g = torch.Generator().manual_seed(seed)
    n = sum(lengths)
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return (torch.randint(0, VOCAB, (n,), generator=g), torch.randint(0, VOCAB, (n,), generator=g), offsets)


@pytest.fixture(autouse=True)
def full_precision_products():
    """The products between the operators are torch's: in 32 bits, not TF32."""
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = old


def test_training_step_matches_the_model_in_64_bits():
    """The roundings of a chain of about a thousand operations on values of size 1 to 10, none of them amplified by
    more than the model's slopes (below 100): 1e3 * 2^-24 * 100 would be 6e-3 at the worst, all of one sign; as they
    fall on both sides a hundredth of that, relative to the size of each result, is held."""
    import tcu_scope_b200 as tcu
    lengths = [7, 0, 1, 40, 16]
    tokens, targets, offsets = batch(3, lengths)
    p64 = {k: v.requires_grad_() for k, v in parameters(5).items()}
    dlp = torch.full((sum(lengths),), -1.0 / sum(lengths), dtype=torch.float64)
    logp, entropy, _ = plain(p64, tokens, targets, lengths)
    want = torch.autograd.grad((logp * dlp).sum() + (entropy * 0.01 * dlp).sum(), list(p64.values()))
    p = {k: v.detach().float().cuda() for k, v in p64.items()}
    dev = [t.cuda() for t in (tokens, offsets, targets)]
    keep, lp = forward(tcu, p, *dev)
    g = backward(tcu, p, *dev, keep, lp, dlp.float().cuda(), (0.01 * dlp).float().cuda())
    for got, ref in ((lp.logprob, logp.detach()), (lp.entropy, entropy.detach())):
        assert float((got.double().cpu() - ref).norm() / ref.norm()) < 6e-5
    for (name, _), ref in zip(p64.items(), want):
        off = float((g[name].double().cpu() - ref).norm() / ref.norm())
        assert off < 6e-5, (name, off)
    assert tcu.device_error() == 0


def test_captured_training_step_follows_new_data():
    import tcu_scope_b200 as tcu
    lengths = [30, 20, 14]
    tokens, targets, offsets = (t.cuda() for t in batch(4, lengths))
    p = {k: v.float().cuda() for k, v in parameters(6).items()}
    dlp = torch.full((64,), 0.1, device="cuda")

    def step():
        keep, lp = forward(tcu, p, tokens, offsets, targets)
        return backward(tcu, p, tokens, offsets, targets, keep, lp, dlp, dlp)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    tokens.copy_(tokens.flip(0))
    for t in p.values():
        t.mul_(1.01)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    for name in want:
        if name == "embed":  # torch adds rows of the same token up in any order
            assert torch.allclose(captured[name], want[name], rtol=1e-4, atol=1e-6)
        else:
            assert torch.equal(captured[name], want[name]), name


def test_tokens_one_by_one_are_the_sequence_at_once():
    """Generation from slots of a pool, in the model's order, gives the logits of the whole sequence (to the roundings of
    either, see above)."""
    import tcu_scope_b200 as tcu
    lengths = [25, 25, 25]
    tokens, targets, offsets = batch(8, lengths)
    p = {k: v.float().cuda() for k, v in parameters(7).items()}
    keep, _ = forward(tcu, p, tokens.cuda(), offsets.cuda(), targets.cuda())
    whole = keep["logits"].view(3, 25, VOCAB)
    pools = [torch.zeros(5, INNER, device="cuda") for _ in range(LAYERS)]
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    for t in range(25):
        x = p["embed"][tokens.view(3, 25)[:, t].cuda()]
        _, u = tcu.norm_residual(x, pre_weight=p["norm0"], eps=EPS)
        for i in range(LAYERS):
            proj = u @ p[f"in{i}"]
            proj[:, :INNER] += 2
            h = tcu.linear_scan_step(proj[:, :INNER], proj[:, INNER:2 * INNER], pools[i], gate="sigmoid", slots=slots)
            y, _ = tcu.norm_residual(h, post_weight=p[f"post{i}"], gate=proj[:, 2 * INNER:], gate_act="silu", eps=EPS)
            x, u = tcu.norm_residual(y @ p[f"out{i}"], x, gate=p[f"scale{i}"], scale=0.7, pre_weight=p[f"norm{i + 1}"], eps=EPS)
        logits = u @ p["head"]
        assert float((logits - whole[:, t]).norm() / whole[:, t].norm()) < 6e-5
    best = tcu.token_logprobs(logits, top=3)
    assert best.logprob is None and torch.equal(best.top_index[:, 0], logits.argmax(1))
    assert all(bool((pool[[1, 3]] == 0).all()) for pool in pools)
