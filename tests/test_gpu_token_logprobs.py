"""Log probabilities of given tokens with entropy and alternatives, and the gradient of the logits, against the
plain 64-bit formulas, at the vocabularies, masks, ties and layouts where they can go wrong."""
import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def check(tcu, logits, targets, top, seed=0, names=("logprob", "entropy", "lse")):
    g = torch.Generator().manual_seed(seed)
    rows = logits.shape[0]
    dlp, dent = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    got = tcu.token_logprobs(logits, targets, top=top)
    d = tcu.token_logprobs_backward(logits, targets, got.lse, got.entropy, dlogprob=dlp, dentropy=dent)
    want = ref.token_logprobs(logits.double().cpu(), targets.cpu().long(), top, dlp.double().cpu(), dent.double().cpu())
    for name in names:
        finite = torch.isfinite(want[name][0])
        mine = getattr(got, name).cpu()
        assert torch.equal(mine[~finite].double(), want[name][0][~finite]), name
        ref.assert_within(mine[finite], want[name][0][finite], want[name][1][finite], name)
    if top:
        assert torch.equal(got.top_index.cpu(), want["top_index"])
        finite = torch.isfinite(want["top_logprob"][0])
        mine = got.top_logprob.cpu()
        assert torch.equal(mine[~finite].double(), want["top_logprob"][0][~finite])
        ref.assert_within(mine[finite], want["top_logprob"][0][finite], want["top_logprob"][1][finite], "top")
    else:
        assert got.top_logprob is None and got.top_index is None
    ref.assert_within(d, *want["dlogits"], "dlogits")
    again = tcu.token_logprobs(logits, targets, top=top)
    assert all(p is None or torch.equal(p, q) for p, q in zip(got, again))
    return got, d


def make(rows, vocab, kind, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(rows, vocab, generator=g)).to(kind)
    return x.cuda(), torch.randint(0, vocab, (rows,), generator=g).cuda()


@pytest.mark.parametrize("kind", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (4, 33), (7, 129), (200, 300), (9, 1000), (3, 2048),
                                        (2, 4097), (400, 5003), (1, 32000), (6, 50001), (2, 131072), (1, 300007)])
def test_vocabularies_match_reference(kind, rows, vocab):
    import tcu_scope_b200 as tcu
    x, t = make(rows, vocab, kind, rows + vocab)
    for top in sorted({0, 1, min(5, vocab), min(32, vocab)}):
        check(tcu, x, t, top)


@pytest.mark.parametrize("kind", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [40, 1000, 20011])
def test_masked_tokens(kind, vocab):
    """-inf and the type's lowest value in masked places; rows in which a mask leaves one token, or none."""
    import tcu_scope_b200 as tcu
    for low in (float("-inf"), torch.finfo(kind).min):
        x, t = make(6, vocab, kind, vocab)
        keep = torch.rand(6, vocab, generator=torch.Generator().manual_seed(1)).cuda() < 0.02
        keep[0] = False                       # nothing is left
        keep[1] = False
        keep[1, vocab // 2] = True            # one token is left
        keep[2:, t[2]] = True
        keep[3] = True
        x = x.masked_fill(~keep, low)
        t[1] = vocab // 2
        t[4] = int((~keep[4]).nonzero()[0, 0])  # a target that the mask forbids
        got, d = check(tcu, x, t, 8)
        if low == float("-inf"):
            assert got.lse[0] == low and got.logprob[0] == low and got.entropy[0] == 0 and bool((d[0] == 0).all())
            assert got.top_index[0].tolist() == list(range(8))
            assert got.logprob[1] == 0 and got.entropy[1] == 0


@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_ties_go_to_the_lowest_index(vocab):
    import tcu_scope_b200 as tcu
    g = torch.Generator().manual_seed(vocab)
    for levels in (1, 2, 5, 40):
        x = torch.randint(0, levels, (3, vocab), generator=g).to(BF16).cuda() - 1
        x[x == 0] = torch.where(torch.rand(int((x == 0).sum()), generator=g).cuda() < 0.5, 0.0, -0.0).to(BF16)  # -0 is 0
        t = torch.randint(0, vocab, (3,), generator=g).cuda()
        for top in (1, 7, 32):
            check(tcu, x, t, top)


@pytest.mark.parametrize("order", ["rising", "falling", "organ"])
def test_sorted_rows(order):
    """Every element is better than all before it, or none is."""
    import tcu_scope_b200 as tcu
    x = torch.arange(9001.0).cuda() / 100 - 45
    x = {"rising": x, "falling": x.flip(0), "organ": -x.abs()}[order][None]
    check(tcu, x.contiguous(), torch.tensor([5]).cuda(), 32)


def test_large_logits_and_sure_rows():
    """Rows far from 0, where lse itself loses digits, and rows with one near certain token."""
    import tcu_scope_b200 as tcu
    x, t = make(8, 3001, F32, 3)
    x[0] += 200
    x[1] -= 250
    x[2] += 3000
    x[3] -= 1e6
    x[4, t[4]] += 40
    x[5, t[5]] += 100
    x[6] *= 1e30
    check(tcu, x, t, 4)
    got = tcu.token_logprobs(x, t)
    assert float(got.logprob[4]) <= 0 and float(got.entropy[5]) >= 0


def test_nan_and_infinity_stay_in_their_rows():
    import tcu_scope_b200 as tcu
    x, t = make(4, 700, F32, 3)
    x[1, 40] = float("nan")
    x[1, 600] = -float("nan")
    x[2, 50] = float("inf")
    got = tcu.token_logprobs(x, t, top=3)
    for v in (got.lse, got.logprob, got.entropy):
        assert v.isnan().tolist() == [False, True, True, False]
    assert got.top_index[1, :2].tolist() == [40, 600] and got.top_index[2, 0] == 50
    d = tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=torch.ones(4).cuda())
    assert d.isnan().any(1).tolist() == [False, True, True, False]


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_ignored_and_wrong_targets(kind):
    import tcu_scope_b200 as tcu
    x, t = make(6, 500, BF16, 5)
    want, d_want = check(tcu, x, t, 2)
    t2 = t.to(kind).clone()  # (a tensor of its own where kind is t's type already)
    t2[1] = -100
    one = torch.ones(6).cuda()
    got = tcu.token_logprobs(x, t2)
    assert tcu.device_error() == 0
    t2[2], t2[3] = 500, -1
    got = tcu.token_logprobs(x, t2)
    assert tcu.device_error() == 8
    out = [1, 2, 3]
    assert bool((got.logprob[out] == 0).all()) and torch.equal(got.entropy, want.entropy)
    assert torch.equal(got.logprob[[0, 4, 5]], want.logprob[[0, 4, 5]])
    d = tcu.token_logprobs_backward(x, t2, got.lse, got.entropy, dlogprob=one, dentropy=one)
    assert tcu.device_error() == 8
    none = tcu.token_logprobs_backward(x, None, got.lse, got.entropy, dentropy=one)
    full = tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=one, dentropy=one)
    assert torch.equal(d[out], none[out]) and torch.equal(d[[0, 4, 5]], full[[0, 4, 5]])
    got = tcu.token_logprobs(x, t.to(kind).masked_fill(t == t[0], 3), ignore_index=3)
    assert float(got.logprob[0]) == 0 and tcu.device_error() == 0


def test_strided_unaligned_and_shaped_logits():
    import tcu_scope_b200 as tcu
    wide = (2 * torch.randn(12, 3333, generator=torch.Generator().manual_seed(2))).to(BF16).cuda()
    t = torch.arange(12).cuda() * 200
    for i, j in ((0, 3328), (1, 3001), (5, 2900), (8, 3333)):
        check(tcu, wide[:, i:j], t, 6)
    check(tcu, wide[::3, 7:], t[:4], 6)
    check(tcu, wide[:1].expand(12, 3333), t, 6)
    flat, _ = check(tcu, wide, t, 6)
    shaped = tcu.token_logprobs(wide.view(3, 4, 3333), t.view(3, 4), top=6)
    assert shaped.logprob.shape == (3, 4) and shaped.top_index.shape == (3, 4, 6)
    assert all(torch.equal(p.flatten(), q.flatten()) for p, q in zip(flat, shaped))
    one = tcu.token_logprobs(wide[0], t[0], top=6)
    assert one.lse.shape == () and torch.equal(one.top_index, flat.top_index[0])
    empty = tcu.token_logprobs(wide[:0], t[:0], top=2)
    assert empty.lse.shape == (0,) and empty.top_index.shape == (0, 2)
    assert tcu.token_logprobs_backward(wide[:0], t[:0], empty.lse, empty.entropy, dlogprob=empty.lse).shape == (0, 3333)


@pytest.mark.parametrize("vocab", [512, 3331])
def test_gradient_over_the_logits(vocab):
    import tcu_scope_b200 as tcu
    x, t = make(9, vocab, BF16, 7)
    got = tcu.token_logprobs(x, t)
    one = torch.ones(9).cuda()
    want = tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=one, dentropy=one)
    copy = x.clone()
    assert tcu.token_logprobs_backward(copy, t, got.lse, got.entropy, dlogprob=one, dentropy=one, out=copy) is copy
    assert torch.equal(copy, want)
    zero = tcu.token_logprobs_backward(x, None, got.lse)
    assert bool((zero == 0).all())
    # an output that begins at another place of its 16 bytes than the logits do
    room = torch.empty(9 * vocab + 1, dtype=BF16, device="cuda")
    out = room[1:].view(9, vocab)
    assert torch.equal(tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=one, dentropy=one, out=out), want)


@pytest.mark.parametrize("kind", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(3, 20011), (64, 20016), (5, 100003), (150, 100000)])
def test_gradient_over_the_logits_of_rows_far_from_zero(kind, rows, vocab):
    """Rows whose lse has lost digits are summed once more for the gradient: all of a row is read before any
    of it is overwritten, however many blocks a row of ordinary size has."""
    import tcu_scope_b200 as tcu
    x, t = make(rows, vocab, kind, rows + vocab)
    x[0] += 3000
    x[2:-1] -= 20000 if kind == F16 else 1e6  # the last row and row 1 stay as they are
    x[2::3] += 19000 if kind == F16 else 1e6 - 1000
    got = tcu.token_logprobs(x, t)
    assert int((got.lse.abs() > 256).sum()) >= rows - 2
    g = torch.Generator().manual_seed(3)
    dlp, dent = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    want = tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=dlp, dentropy=dent)
    few = slice(0, 4)
    bound = ref.token_logprobs(x[few].double().cpu(), t[few].cpu(), 0, dlp[few].double().cpu(), dent[few].double().cpu())
    ref.assert_within(want[few], *bound["dlogits"], "dlogits")
    for _ in range(3):
        over = x.clone()
        tcu.token_logprobs_backward(over, t, got.lse, got.entropy, dlogprob=dlp, dentropy=dent, out=over)
        assert torch.equal(over, want)


@pytest.mark.parametrize("vocab", [2, 5, 64, 5000, 40000])
def test_gradient_of_equal_logits_far_from_zero(vocab):
    """All p are 1 / vocab, whatever the logits are.  Up to |lse| of 32 lse is off by half its step (2^-20) and its own
    error, above it log2 s by 2 ulp (4 u log2 vocab) and the exponential by 4 u; one product and, at the target, a sum."""
    import math

    import tcu_scope_b200 as tcu
    values = [0.0, 3.7, 20.3, 31.9, 33.3, 40.1, 77.7, 100.3, 150.9, 200.1, 255.4, 900.7, -21.2, -90.7, -200.3, -255.9]
    x = torch.tensor(values).cuda()[:, None].expand(len(values), vocab).contiguous()
    t = torch.full((len(values),), vocab - 1).cuda()
    got = tcu.token_logprobs(x, t)
    d = tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=torch.ones(len(values)).cuda()).double().cpu()
    u, p = 2.0 ** -24, 1.0 / vocab
    far = [v for v, lse in enumerate(got.lse.tolist()) if abs(lse) > 32]
    near = [v for v in range(len(values)) if v not in far]
    assert len(far) >= 8 and len(near) >= 4
    rel = (4 * math.log2(vocab) + 4 + 2) * u
    for rows, off in ((far, rel), (near, rel + 2.0 ** -20)):
        assert float((d[rows, :-1] + p).abs().max()) <= off * p
        assert float((d[rows, -1] - (1 - p)).abs().max()) <= off * p + 2 * u


def test_gradient_against_differences():
    import tcu_scope_b200 as tcu
    x, t = make(3, 11, F32, 8, spread=1.0)
    g = torch.Generator().manual_seed(1)
    dlp, dent = torch.randn(3, generator=g).cuda(), torch.randn(3, generator=g).cuda()
    got = tcu.token_logprobs(x, t)
    d = tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=dlp, dentropy=dent).cpu()

    def loss(x):
        w = ref.token_logprobs(x, t.cpu(), 0)
        return float((w["logprob"][0] * dlp.double().cpu()).sum() + (w["entropy"][0] * dent.double().cpu()).sum())

    for i in range(33):
        up, down = x.double().cpu(), x.double().cpu()
        up.view(-1)[i] += 1e-5
        down.view(-1)[i] -= 1e-5
        # third derivatives below 100: the quotient is within 1e-8
        assert abs((loss(up) - loss(down)) / 2e-5 - float(d.view(-1)[i])) < 1e-6


def test_other_stream_and_captured_graph():
    import tcu_scope_b200 as tcu
    x, t = make(20, 20000, BF16, 2)
    one = torch.ones(20).cuda()

    def run():
        got = tcu.token_logprobs(x, t, top=4)
        return [*got, tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=one, dentropy=one)]

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    x.copy_(x.flip(0))
    want = run()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_far_rows():
    """More than 2^31 logits in one call: the last rows are what they are alone."""
    import tcu_scope_b200 as tcu
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GiB of free device memory")
    rows, vocab = 17000, 128001
    x = torch.empty(rows, vocab, dtype=BF16, device="cuda").normal_()
    t = torch.randint(0, vocab, (rows,), device="cuda")
    one = torch.ones(rows, device="cuda")
    got = tcu.token_logprobs(x, t, top=3)
    tail = slice(rows - 40, rows)
    want = tcu.token_logprobs(x[tail], t[tail], top=3)
    # 40 rows are read by more blocks each than 17000, so sums are joined in another order
    assert torch.equal(got.top_index[tail], want.top_index)
    assert torch.allclose(got.lse[tail], want.lse, rtol=3e-7, atol=0)
    d = tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=one, dentropy=one)
    w = tcu.token_logprobs_backward(x[tail], t[tail], got.lse[tail], got.entropy[tail], dlogprob=one[tail], dentropy=one[tail])
    assert torch.equal(d[tail], w)
