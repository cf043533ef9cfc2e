"""The gated linear recurrence, its gradient and its form for single tokens, against the plain 64-bit
recurrence, at the lengths, widths, layouts and offsets where it can go wrong."""
import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
GATES = ["decay", "log", "sigmoid"]


def inputs(gate, shape, a_type, x_type, seed):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if gate == "sigmoid":
        a = 3 + 2 * n(*shape)
    else:
        a = -torch.exp(-3 + 1.5 * n(*shape))
        a = a.exp() * torch.sign(n(*shape) + 1.5) if gate == "decay" else a
    return a.to(a_type).cuda(), n(*shape).to(x_type).cuda(), n


def check(got, want, what):
    for name, t in got.items():
        value, bound = want[name]
        ref.assert_within(t, value, bound, (what, name))


def run_batch(tcu, gate, a, x, h0, dh, dlast):
    states = tcu.linear_scan_states(x)
    h, last = tcu.linear_scan(a, x, gate=gate, h0=h0, states=states)
    da, dx, dh0 = tcu.linear_scan_backward(dh, a, x, states, gate=gate, dlast=dlast)
    return dict(h=h, last=last, da=da, dx=dx, dh0=dh0)


def check_batch(gate, a, x, h0, dh, dlast, got, what):
    cpu = lambda t: t.double().cpu()  # noqa: E731
    for b in range(x.shape[0]):
        want = ref.linear_scan(gate, cpu(a[b]), cpu(x[b]), cpu(h0[b]), cpu(dh[b]), cpu(dlast[b]))
        check({k: v[b] for k, v in got.items()}, want, (what, b))


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("a_type,x_type", [(F32, F32), (BF16, BF16), (F32, BF16), (F16, F16), (F32, F16)])
@pytest.mark.parametrize("batch,tokens,dim", [(2, 1, 128), (1, 63, 4), (2, 64, 130), (1, 65, 129), (3, 200, 33),
                                              (1, 1100, 256), (2, 513, 1)])
def test_batch_matches_reference(gate, a_type, x_type, batch, tokens, dim):
    import tcu_scope_b200 as tcu
    a, x, n = inputs(gate, (batch, tokens, dim), a_type, x_type, 7 * tokens + dim)
    h0, dlast, dh = n(batch, dim).cuda(), n(batch, dim).cuda(), n(batch, tokens, dim).to(x_type).cuda()
    got = run_batch(tcu, gate, a, x, h0, dh, dlast)
    check_batch(gate, a, x, h0, dh, dlast, got, (gate, batch, tokens, dim))
    again = run_batch(tcu, gate, a, x, h0, dh, dlast)
    assert all(torch.equal(got[k], again[k]) for k in got)  # the same bits every time


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("dim", [64, 96, 131])
def test_packed_sequences_match_reference(gate, wide, dim):
    """Empty sequences, single tokens, chunk borders; rows outside all sequences."""
    import tcu_scope_b200 as tcu
    lengths = [0, 1, 64, 0, 63, 65, 2, 300, 0]
    first, rest = 5, 70
    ends = torch.tensor([first] + lengths).cumsum(0)
    tokens, batch = int(ends[-1]) + rest, len(lengths)
    a, x, n = inputs(gate, (tokens, dim), BF16, BF16, dim)
    h0, dlast, dh = n(batch, dim).cuda(), n(batch, dim).cuda(), n(tokens, dim).to(BF16).cuda()
    # what lies outside the sequences must not matter
    for t in (a, x, dh):
        t[:first] = float("nan")
        t[tokens - rest:] = float("nan")
    offsets = ends.to(wide).cuda()
    states = tcu.linear_scan_states(x, offsets)
    mine = torch.full_like(x, 7.0)
    h, last = tcu.linear_scan(a, x, gate=gate, h0=h0, offsets=offsets, states=states)
    h2, _ = tcu.linear_scan(a, x, gate=gate, h0=h0, offsets=offsets, out=mine)
    da, dx, dh0 = tcu.linear_scan_backward(dh, a, x, states, gate=gate, dlast=dlast, offsets=offsets)
    da2, dx2, _ = tcu.linear_scan_backward(dh, a, x, states, gate=gate, dlast=dlast, offsets=offsets,
                                           da=torch.full_like(a, 7.0), dx=torch.full_like(x, 7.0))
    outside = torch.ones(tokens, dtype=torch.bool)
    cpu = lambda t: t.double().cpu()  # noqa: E731
    for b, (i, j) in enumerate(zip(ends[:-1].tolist(), ends[1:].tolist())):
        outside[i:j] = False
        want = ref.linear_scan(gate, cpu(a[i:j]), cpu(x[i:j]), cpu(h0[b]), cpu(dh[i:j]), cpu(dlast[b]))
        check(dict(h=h[i:j], da=da[i:j], dx=dx[i:j], last=last[b], dh0=dh0[b]), want, (gate, b))
    for new, old in ((h, h2), (da, da2), (dx, dx2)):
        assert bool((new[outside.cuda()] == 0).all()) and bool((old[outside.cuda()] == 7).all())
        assert torch.equal(new[~outside.cuda()], old[~outside.cuda()])
    assert tcu.device_error() == 0


TYPES = [(F32, F32), (BF16, BF16), (F32, BF16), (F16, F16), (F32, F16)]


def device_inputs(gate, shape, a_type, x_type, seed):
    """As inputs(), made on the GPU: many columns."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if gate == "sigmoid":
        a = 3 + 2 * n(*shape)
    else:
        a = -torch.exp(-3 + 1.5 * n(*shape))
        a = a.exp() * torch.sign(n(*shape) + 1.5) if gate == "decay" else a
    return a.to(a_type), n(*shape).to(x_type), n


def some_channels(dim):
    """The ends of the columns of 64, and others."""
    return sorted({c for c in (0, 1, 63, 64, 127, dim // 2, dim // 3, dim - 65, dim - 2, dim - 1) if 0 <= c < dim})


def check_channels(gate, a, x, h0, dh, dlast, got, what):
    """check_batch() at some channels, those of all sequences side by side."""
    batch, tokens, dim = x.shape
    ch = some_channels(dim)
    pick = lambda t: t[..., ch].double().cpu()  # noqa: E731
    rows = lambda t: pick(t).transpose(0, 1).reshape(tokens, -1)  # noqa: E731
    flat = lambda t: pick(t).reshape(-1)  # noqa: E731
    want = ref.linear_scan(gate, rows(a), rows(x), flat(h0), rows(dh), flat(dlast))
    for name, t in got.items():
        t = t[..., ch].reshape(-1) if name in ("last", "dh0") else t[..., ch].transpose(0, 1).reshape(tokens, -1)
        ref.assert_within(t, *want[name], (what, name))


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("a_type,x_type", TYPES)
@pytest.mark.parametrize("batch,dim", [(37, 2048), (36, 2057)])
def test_a_warp_for_each_of_many_columns(gate, a_type, x_type, batch, dim):
    """Where there are eight columns for every SM the gradient goes through a sequence with one warp: windows of 32
    rows with two states each, a ring that wraps, lengths around the borders of both."""
    import tcu_scope_b200 as tcu
    for tokens in (33, 47, 64, 65, 289) if a_type == x_type else (31, 177):
        a, x, n = device_inputs(gate, (batch, tokens, dim), a_type, x_type, tokens)
        h0, dlast, dh = n(batch, dim), n(batch, dim), n(batch, tokens, dim).to(x_type)
        got = run_batch(tcu, gate, a, x, h0, dh, dlast)
        check_channels(gate, a, x, h0, dh, dlast, got, (gate, tokens))
        again = run_batch(tcu, gate, a, x, h0, dh, dlast)
        assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("a_type,x_type", TYPES)
@pytest.mark.parametrize("batch,tokens,dim", [(8, 300, 1280), (8, 1111, 1210), (3, 2050, 3200)])
def test_a_block_for_each_column(gate, a_type, x_type, batch, tokens, dim):
    """As many columns as SMs and more: the warps of one block share a sequence, with several windows each."""
    import tcu_scope_b200 as tcu
    a, x, n = device_inputs(gate, (batch, tokens, dim), a_type, x_type, tokens)
    h0, dlast, dh = n(batch, dim), n(batch, dim), n(batch, tokens, dim).to(x_type)
    got = run_batch(tcu, gate, a, x, h0, dh, dlast)
    check_channels(gate, a, x, h0, dh, dlast, got, (gate, tokens))


def lengths_of(kind):
    """Lengths of packed sequences: at and above the number that is ranked, and batches whose mean says little."""
    g = torch.Generator().manual_seed(len(kind))
    if kind in ("96", "97", "300"):
        n = int(kind)
        lengths = torch.randint(0, 60, (n,), generator=g)
        lengths[torch.rand(n, generator=g) < 0.1] = 0
        lengths[n // 3], lengths[n - 1], lengths[5] = 700, 150, 0
        return lengths.tolist()
    if kind == "1100":
        return torch.randint(0, 5, (1100,), generator=g).tolist()
    return [5] * 20 + [0, 350, 1] + [3] * 27 if kind == "one long" else [2000] + [32] * 30


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("a_type,x_type", [(BF16, BF16), (F32, F16), (F32, F32)])
@pytest.mark.parametrize("kind", ["96", "97", "300", "1100", "one long", "long first"])
@pytest.mark.parametrize("dim", [72, 1033, 2048])
def test_packed_batches_match_reference(gate, a_type, x_type, kind, dim):
    import tcu_scope_b200 as tcu
    lengths = lengths_of(kind)
    first, rest = 3, 9
    ends = torch.tensor([first] + lengths).cumsum(0)
    tokens, batch = int(ends[-1]) + rest, len(lengths)
    a, x, n = device_inputs(gate, (tokens, dim), a_type, x_type, dim)
    h0, dlast, dh = n(batch, dim), n(batch, dim), n(tokens, dim).to(x_type)
    offsets = ends.to(torch.int32).cuda()

    def run():
        states = tcu.linear_scan_states(x, offsets)
        h, last = tcu.linear_scan(a, x, gate=gate, h0=h0, offsets=offsets, states=states)
        da, dx, dh0 = tcu.linear_scan_backward(dh, a, x, states, gate=gate, dlast=dlast, offsets=offsets)
        return dict(h=h, last=last, da=da, dx=dx, dh0=dh0)

    got = run()
    ch = some_channels(dim)
    cpu = {k: t[..., ch].double().cpu() for k, t in dict(a=a, x=x, h0=h0, dh=dh, dlast=dlast).items()}
    few = {k: t[..., ch] for k, t in got.items()}
    for k in ("h", "da", "dx"):
        assert bool((got[k][:first] == 0).all()) and bool((got[k][tokens - rest:] == 0).all())
    long = [b for b in range(batch) if lengths[b] > 100]
    for b in sorted({*long, *range(0, batch, 1 + batch // 40), 5, batch - 1}):
        i, j = int(ends[b]), int(ends[b + 1])
        want = ref.linear_scan(gate, cpu["a"][i:j], cpu["x"][i:j], cpu["h0"][b], cpu["dh"][i:j], cpu["dlast"][b])
        check(dict(h=few["h"][i:j], da=few["da"][i:j], dx=few["dx"][i:j], last=few["last"][b], dh0=few["dh0"][b]), want, (gate, b))
    again = run()
    assert all(torch.equal(got[k], again[k]) for k in got)
    assert tcu.device_error() == 0


def test_strided_and_unaligned_inputs():
    """a and x as column blocks of one projection, a shifted view, a gate broadcast over the batch."""
    import tcu_scope_b200 as tcu
    batch, tokens, dim = 2, 130, 96
    _, _, n = inputs("log", (1, 1, 1), F32, F32, 3)
    proj = (-n(batch, tokens, 2 * dim + 8).abs()).to(BF16).cuda()
    h0, dlast, dh = n(batch, dim).cuda(), n(batch, dim).cuda(), n(batch, tokens, dim).to(BF16).cuda()
    for a, x in [(proj[..., :dim], proj[..., dim:2 * dim]), (proj[..., 1:dim + 1], proj[..., dim + 3:2 * dim + 3]),
                 (proj[:1, :, :dim].expand(batch, tokens, dim), proj[..., 2:dim + 2]),
                 (proj[:, :1, 4:dim + 4].expand(batch, tokens, dim), proj.flip(1)[..., 4:dim + 4])]:
        for d in (dh, dh.transpose(0, 1).contiguous().transpose(0, 1)):
            got = run_batch(tcu, "log", a, x, h0, d, dlast)
            check_batch("log", a, x, h0, d, dlast, got, "strided")


def test_defaults_and_in_place_state():
    """No h0, no dlast, no dh; last written over h0; an empty time axis."""
    import tcu_scope_b200 as tcu
    a, x, n = inputs("decay", (2, 150, 40), F32, F32, 1)
    zero, h0 = torch.zeros(2, 40).cuda(), n(2, 40).cuda()
    states = tcu.linear_scan_states(x)
    h, last = tcu.linear_scan(a, x, states=states)
    want, _ = tcu.linear_scan(a, x, h0=zero)
    assert torch.equal(h, want)
    da, dx, dh0 = tcu.linear_scan_backward(None, a, x, states, dlast=h0)
    full = tcu.linear_scan_backward(torch.zeros_like(x), a, x, states, dlast=h0)
    assert all(torch.equal(p, q) for p, q in zip((da, dx, dh0), full))
    none = tcu.linear_scan_backward(None, a, x, states)
    assert all(bool((t == 0).all()) for t in none)
    state = h0.clone()
    want, wlast = tcu.linear_scan(a, x, h0=h0)
    h, last = tcu.linear_scan(a, x, h0=state, last=state)
    assert last is state and torch.equal(state, wlast) and torch.equal(h, want)
    empty = x[:, :0]
    h, last = tcu.linear_scan(a[:, :0], empty, h0=h0)
    assert h.shape == (2, 0, 40) and torch.equal(last, h0)
    assert torch.equal(tcu.linear_scan(a[:, :0], empty)[1], zero)
    dh0 = tcu.linear_scan_backward(empty, a[:, :0], empty, tcu.linear_scan_states(empty), dlast=h0)[2]
    assert torch.equal(dh0, h0)


def test_pieces_of_a_sequence_join():
    """A sequence read in pieces, the state handed on, is the sequence read at once."""
    import tcu_scope_b200 as tcu
    a, x, n = inputs("sigmoid", (1, 700, 72), F32, F32, 9)
    cpu = lambda t: t.double().cpu()  # noqa: E731
    want = ref.linear_scan("sigmoid", cpu(a[0]), cpu(x[0]), torch.zeros(72, dtype=torch.float64))
    state = torch.zeros(1, 72).cuda()
    parts = [tcu.linear_scan(a[:, i:j], x[:, i:j], gate="sigmoid", h0=state, last=state)[0]
             for i, j in ((0, 1), (1, 65), (65, 66), (66, 500), (500, 700))]
    check(dict(h=torch.cat(parts, 1)[0], last=state[0]), want, "pieces")


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("a_type,x_type", [(F32, F32), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("dim", [1, 128, 130, 2053])
def test_step_matches_reference(gate, a_type, x_type, dim):
    import tcu_scope_b200 as tcu
    batch, pool = 9, 12
    a, x, n = inputs(gate, (batch, dim), a_type, x_type, dim)
    state = n(pool, dim).cuda()
    slots = torch.tensor([3, 11, -1, 0, 7, 5, -5, 2, 1])
    for kind in (torch.int32, torch.int64, None):
        pool_state, out = state.clone(), torch.full((batch, dim), 5.0, dtype=x_type).cuda()
        at = torch.arange(batch) if kind is None else slots
        given = None if kind is None else slots.to(kind).cuda()
        h = tcu.linear_scan_step(a, x, pool_state, gate=gate, slots=given, out=out)
        fresh = tcu.linear_scan_step(a, x, state.clone(), gate=gate, slots=given)
        want = state.double().cpu()
        for b, s in enumerate(at.tolist()):
            if s < 0:
                assert bool((h[b] == 5).all()) and bool((fresh[b] == 0).all())
                continue
            one = ref.linear_scan(gate, a[b:b + 1].double().cpu(), x[b:b + 1].double().cpu(), want[s])
            ref.assert_within(h[b], one["last"][0], one["last"][1], ("step", b))
            assert torch.equal(fresh[b], h[b])
            ref.assert_within(pool_state[s], one["last"][0], one["last"][1], ("state", b))
        for s in range(pool):
            if s not in at.tolist():
                assert torch.equal(pool_state[s], state[s])
    assert tcu.device_error() == 0


def test_wrong_indices_are_left_out_and_reported():
    """Checked in the kernel before anything is addressed with them."""
    import tcu_scope_b200 as tcu
    a, x, n = inputs("decay", (6, 64), F32, F32, 2)
    state = n(4, 64).cuda()
    before = state.clone()
    slots = torch.tensor([2, 4, 1 << 30, 2, -1, 0], dtype=torch.int32).cuda()  # past the pool, and 2 twice
    h = tcu.linear_scan_step(a, x, state, slots=slots)
    assert tcu.device_error() == 8 and tcu.device_error() == 0
    assert bool((h[[1, 2, 3, 4]] == 0).all()) and torch.equal(state[[1, 3]], before[[1, 3]])
    assert torch.equal(h[0], state[2]) and torch.equal(h[5], state[0])
    offsets = torch.tensor([0, 4, 2, 6, 9], dtype=torch.int32).cuda()  # sequence 1 decreases, sequence 3 passes the end
    h0 = n(4, 64).cuda()
    out = torch.full((6, 64), 3.0).cuda()
    h, last = tcu.linear_scan(a, x, h0=h0, offsets=offsets, out=out)
    assert tcu.device_error() == 8
    assert torch.equal(last[1], h0[1]) and torch.equal(last[3], h0[3])
    # `last` is joined from maps of several rows, h row by row: each is within its bound of the 64-bit
    # value, and they need not have the same bits
    want = ref.linear_scan("decay", a[2:6].double().cpu(), x[2:6].double().cpu(), h0[2].double().cpu())
    ref.assert_within(last[2], *want["last"], "last")
    ref.assert_within(h[5], *want["last"], "h")


def offsets_that_decrease():
    """(tokens, offsets) with sequences that share rows, or (the last) states."""
    even = list(range(0, 1207, 6))  # 201 sequences of 6 rows
    def changed(**at):
        return [at.get(f"o{i}", v) for i, v in enumerate(even)]
    return [(600, [0, 300, 100, 600]), (600, [0, 50, 120, 60, 400, 600]), (600, [200, 600, 0, 400, 300, 500]),
            (1206, changed(o57=5000)), (1206, changed(o57=-9, o126=1300)), (1206, changed(o60=0)),
            (1206, changed(o133=700, o140=650)), (1206, changed(o3=1000, o150=30)), (1206, even[::-1]),
            (688, [672, 688] + list(range(0, 641, 16)))]


@pytest.mark.parametrize("case", range(10))
@pytest.mark.parametrize("dim", [64, 136])
def test_sequences_that_share_rows(case, dim):
    """A sequence that is in order with all others runs; of those that share rows or are out of order at most one
    does, the same one every time, forward and backward; the rest count as empty."""
    import tcu_scope_b200 as tcu
    tokens, offsets = offsets_that_decrease()[case]
    batch = len(offsets) - 1
    a, x, n = inputs("decay", (tokens, dim), F32, BF16, case)
    h0, dlast, dh = n(batch, dim).cuda(), n(batch, dim).cuda(), n(tokens, dim).to(BF16).cuda()
    at = torch.tensor(offsets, dtype=torch.int64).cuda()

    def run():
        states = tcu.linear_scan_states(x, at)
        h, last = tcu.linear_scan(a, x, h0=h0, offsets=at, states=states, out=torch.full_like(x, 7.0))
        da, dx, dh0 = tcu.linear_scan_backward(dh, a, x, states, dlast=dlast, offsets=at, da=torch.full_like(a, 7.0),
                                               dx=torch.full_like(x, 7.0))
        return dict(h=h, da=da, dx=dx, last=last, dh0=dh0)

    got = run()
    assert tcu.device_error() == 8
    for _ in range(3):
        again = run()
        assert all(torch.equal(got[k], again[k]) for k in got)
    tcu.device_error()
    well = [b for b in range(batch) if 0 <= offsets[b] < offsets[b + 1] <= tokens]
    owner = [None] * tokens
    cpu = lambda t: t.double().cpu()  # noqa: E731
    for b in range(batch):
        i, j = offsets[b], offsets[b + 1]
        if torch.equal(got["last"][b], h0[b]):
            assert torch.equal(got["dh0"][b], dlast[b])
            assert b not in well or any(offsets[k + 1] > i if k < b else offsets[k] < j for k in well if k != b), b
            continue
        assert b in well and owner[i:j] == [None] * (j - i), b
        owner[i:j] = [b] * (j - i)
        want = ref.linear_scan("decay", cpu(a[i:j]), cpu(x[i:j]), cpu(h0[b]), cpu(dh[i:j]), cpu(dlast[b]))
        check({k: v[b] if k in ("last", "dh0") else v[i:j] for k, v in got.items()}, want, b)
    free = torch.tensor([o is None for o in owner]).cuda()
    for k in ("h", "da", "dx"):
        assert bool((got[k][free] == 7).all())
    assert bool(free.all()) == (case == 8)  # something runs, unless nothing can


@pytest.mark.parametrize("tokens,offsets", [
    (6, [0, 6, 2]), (6, [5, 0, 6]), (500, [0, 400, 100]), (500, [450, 20, 480]), (500, [300, 320, 100, 130, 420, 60]),
    (500, [-4, 30, 90]), (500, [10, 30, 600]), (500, [700, 800]), (500, [480, 490, -3]),
    (700, [690] + [7 * i for i in range(1, 99)] + [3]), (700, [695, 699] + [7 * i for i in range(1, 99)] + [3])])
@pytest.mark.parametrize("dim", [64, 200])
def test_cleared_rows_are_no_sequences(tokens, offsets, dim):
    """New outputs have zeros before the first and behind the last sequence; where offsets decrease, rows of a
    sequence that lies there all the same are not among them."""
    import tcu_scope_b200 as tcu
    batch = len(offsets) - 1
    a, x, n = inputs("decay", (tokens, dim), F32, BF16, tokens)
    h0, dlast, dh = n(batch, dim).cuda(), n(batch, dim).cuda(), n(tokens, dim).to(BF16).cuda()
    at = torch.tensor(offsets, dtype=torch.int32).cuda()
    states = tcu.linear_scan_states(x, at)
    h2, last2 = tcu.linear_scan(a, x, h0=h0, offsets=at, out=torch.full_like(x, 7.0), states=states)
    da2, dx2, dh02 = tcu.linear_scan_backward(dh, a, x, states, dlast=dlast, offsets=at, da=torch.full_like(a, 7.0),
                                              dx=torch.full_like(x, 7.0))
    well = [(i, j) for i, j in zip(offsets, offsets[1:]) if 0 <= i < j <= tokens]
    for _ in range(5):
        h, last = tcu.linear_scan(a, x, h0=h0, offsets=at)
        da, dx, dh0 = tcu.linear_scan_backward(dh, a, x, states, dlast=dlast, offsets=at)
        assert torch.equal(last, last2) and torch.equal(dh0, dh02)
        for new, old in ((h, h2), (da, da2), (dx, dx2)):
            for i, j in well:
                if not bool((old[i:j] == 7).all()):  # it ran
                    assert torch.equal(new[i:j], old[i:j])
            before = max(0, min([offsets[0], tokens] + [i for i, _ in well]))
            behind = max([offsets[-1], 0] + [j for _, j in well])
            assert bool((new[:before] == 0).all()) and bool((new[behind:] == 0).all())
    assert tcu.device_error() in ((0, 8) if tokens == 700 else (8,))


def test_overflowing_products_do_not_spoil_a_zero_state():
    """Gates above 1 whose product leaves float32 while the state is 0, and gates of 0."""
    import tcu_scope_b200 as tcu
    x = torch.zeros(1, 256, 32).cuda()
    x[:, 200] = 1
    a = torch.full_like(x, 1e6)
    a[:, 201:] = 0.5
    h, _ = tcu.linear_scan(a, x)
    want = torch.zeros(256)
    want[200:] = 0.5 ** torch.arange(56.0)
    assert torch.equal(h[0].cpu(), want[:, None].expand(256, 32))
    a[:, 210] = 0
    assert bool((tcu.linear_scan(a, x)[0][:, 210:] == 0).all())
    a[:, 220] = float("nan")
    h = tcu.linear_scan(a, x)[0]
    assert bool(h[:, 220:].isnan().all()) and not bool(h[:, :220].isnan().any())


def test_gradient_against_differences():
    import tcu_scope_b200 as tcu
    for gate in GATES:
        a, x, n = inputs(gate, (1, 70, 3), F32, F32, 4)
        h0, dh, dlast = n(1, 3).cuda(), n(1, 70, 3).cuda(), n(1, 3).cuda()
        got = run_batch(tcu, gate, a, x, h0, dh, dlast)
        loss = lambda a, x, h0: sum((p.double().cpu() * q.double().cpu()).sum() for p, q in  # noqa: E731
                                    zip((lambda w: (w["h"][0], w["last"][0]))(
                                        ref.linear_scan(gate, a.double().cpu()[0], x.double().cpu()[0], h0.double().cpu()[0])),
                                        (dh[0], dlast[0])))
        for name, t in (("da", a), ("dx", x), ("dh0", h0)):
            for i in range(0, t.numel(), max(1, t.numel() // 7)):
                args = {"a": a.double().cpu(), "x": x.double().cpu(), "h0": h0.double().cpu()}
                up, down = ({k: v.clone() for k, v in args.items()} for _ in range(2))
                up[name[1:]].view(-1)[i] += 1e-5
                down[name[1:]].view(-1)[i] -= 1e-5
                slope = float(loss(**up) - loss(**down)) / 2e-5
                # second differences of the loss are below 1e3 here, so the quotient is within 1e-7
                assert abs(slope - float(got[name].view(-1)[i])) < 1e-4 * max(1.0, abs(slope)), (gate, name, i)


def test_other_stream_and_captured_graph():
    import tcu_scope_b200 as tcu
    a, x, n = inputs("log", (2, 300, 256), BF16, BF16, 6)
    h0, dlast, dh = n(2, 256).cuda(), n(2, 256).cuda(), n(2, 300, 256).to(BF16).cuda()
    want = run_batch(tcu, "log", a, x, h0, dh, dlast)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_batch(tcu, "log", a, x, h0, dh, dlast)
    side.synchronize()
    assert all(torch.equal(want[k], got[k]) for k in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run_batch(tcu, "log", a, x, h0, dh, dlast)
    for t in (a, x, h0, dh, dlast):
        t.copy_(t.flip(0))
    want = run_batch(tcu, "log", a, x, h0, dh, dlast)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(want[k], got[k]) for k in want)


def test_long_axis_and_far_elements():
    """More than 2^31 elements in one call: a gate of 0 every 64 tokens makes every 64th state known."""
    import tcu_scope_b200 as tcu
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of free device memory")
    tokens, dim = (1 << 20) + 77, 2056
    x = torch.ones(1, tokens, dim, dtype=BF16, device="cuda")
    a = torch.ones(1, tokens, 1, dtype=BF16, device="cuda")
    a[:, ::64] = 0
    a = a.expand(1, tokens, dim).contiguous()
    h, last = tcu.linear_scan(a, x)
    ramp = (torch.arange(tokens, device="cuda") % 64 + 1).to(BF16)
    assert bool((h[0, :, ::257] == ramp[:, None]).all())
    assert bool((h[0, -200:] == ramp[-200:, None]).all()) and bool((last == float(ramp[-1])).all())
