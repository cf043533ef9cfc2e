"""The norms around a block with its gate and residual, and their gradient, against the plain 64-bit
formulas, at the widths, row counts, gates and layouts where they can go wrong."""
import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def make(rows, dim, kind, w_kind, groups, seed, residual=True, post=True, pre=True):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(z=(2 * n(rows, dim)).to(kind).cuda(), residual=(3 * n(rows, dim)).to(kind).cuda() if residual else None,
                post=(1 + 0.3 * n(dim)).to(w_kind).cuda() if post else None,
                gate=n(groups, dim).to(kind).cuda() if groups else None,
                pre=(1 + 0.3 * n(dim)).to(w_kind).cuda() if pre else None,
                dout=n(rows, dim).to(kind).cuda(), dnormed=n(rows, dim).to(kind).cuda() if pre else None)


def run(tcu, s, act, scale=0.75, eps=1e-6, **more):
    args = dict(post_weight=s["post"], gate=s["gate"], gate_act=act, scale=scale, pre_weight=s["pre"], eps=eps)
    out, normed = tcu.norm_residual(s["z"], s["residual"], **args)
    d = tcu.norm_residual_backward(s["dout"], s["dnormed"], s["z"], s["residual"], **args, **more)
    return out, normed, d


def check(s, act, out, normed, d, scale=0.75, eps=1e-6):
    cpu = {k: None if t is None else t.double().cpu() for k, t in s.items()}
    rows = cpu["z"].shape[0]
    gate = cpu["gate"]
    groups = None if gate is None else gate.shape[0]
    if gate is not None:
        gate = gate.repeat_interleave(rows // groups, 0)
    want = ref.norm_residual(cpu["z"], cpu["residual"], cpu["post"], gate, act, scale, cpu["pre"], eps, cpu["dout"],
                             cpu["dnormed"] if cpu["dnormed"] is not None else None)
    ref.assert_within(out, want["out"].v, want["out"].e, "out")
    if normed is not None:
        ref.assert_within(normed, want["normed"].v, want["normed"].e, "normed")
    ref.assert_within(d.dz, want["dz"].v, want["dz"].e, "dz")
    if s["residual"] is not None:
        ref.assert_within(d.dresidual, want["dresidual"].v, want["dresidual"].e, "dresidual")
    else:
        assert d.dresidual is None
    for name, t, rows_of in (("post", d.dpost_weight, "post_rows"), ("pre", d.dpre_weight, "pre_rows")):
        if s[name] is None:
            assert t is None
        else:
            w = want[rows_of].sum(0)
            ref.assert_within(t, w.v, w.e, name)
    if gate is not None:
        w = want["gate_rows"].index(lambda t: t.reshape(groups, rows // groups, -1)).sum(1)
        ref.assert_within(d.dgate, w.v, w.e, "dgate")
    else:
        assert d.dgate is None


@pytest.mark.parametrize("kind,w_kind", [(F32, F32), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (40, 64), (9, 100), (701, 256), (5, 257), (33, 512), (17, 520),
                                      (12, 1111), (700, 96), (6, 4096), (3, 5000), (2, 8200), (2, 16384), (2, 16383)])
def test_widths_match_reference(kind, w_kind, rows, dim):
    import tcu_scope_b200 as tcu
    for act, groups in (("none", 1), ("silu", rows)):
        s = make(rows, dim, kind, w_kind, groups, rows + dim)
        check(s, act, *run(tcu, s, act))


@pytest.mark.parametrize("rows,groups", [(1, 1), (64, 1), (64, 4), (700, 350), (3000, 3000), (2368, 8), (999, 333), (999, 3)])
@pytest.mark.parametrize("dim", [72, 600])
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
def test_shared_gates_match_reference(rows, groups, dim, act):
    import tcu_scope_b200 as tcu
    s = make(rows, dim, BF16, F32, groups, rows + groups)
    got = run(tcu, s, act)
    check(s, act, *got)
    again = run(tcu, s, act)
    assert all(torch.equal(p, q) for p, q in zip([*got[:2], *got[2]], [*again[:2], *again[2]]))


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("groups", [0, 2])
@pytest.mark.parametrize("dim", [40, 1000])
def test_every_part_can_be_left_out(residual, post, pre, groups, dim):
    import tcu_scope_b200 as tcu
    s = make(26, dim, F32, F32, groups, 5, residual, post, pre)
    check(s, "sigmoid", *run(tcu, s, "sigmoid"))


def test_missing_gradients_are_zero():
    import tcu_scope_b200 as tcu
    s = make(10, 300, F32, F32, 1, 8)
    for gone in ("dout", "dnormed"):
        zero = torch.zeros_like(s["dout"])
        d = run(tcu, {**s, gone: None}, "none")[2]
        want = run(tcu, {**s, gone: zero}, "none")[2]
        assert all(torch.equal(p, q) for p, q in zip(d, want))


def test_zero_rows_and_large_values():
    import tcu_scope_b200 as tcu
    s = make(6, 200, F32, F32, 1, 8)
    s["z"][2] = 0
    s["residual"][2] = 0
    s["z"][3] *= 1e15
    s["residual"][3] *= 1e-15
    s["z"][4] *= 1e-18
    out, normed, d = run(tcu, s, "none")
    check(s, "none", out, normed, d)
    assert bool((out[2] == 0).all()) and bool((normed[2] == 0).all())
    s["z"][1, 7] = float("nan")
    out, normed, d = run(tcu, s, "none")
    assert bool(out[1].isnan().all()) and not bool(out[[0, 2, 3, 4, 5]].isnan().any())


@pytest.mark.parametrize("dim", [100, 512, 1111, 4096])
def test_branch_that_cancels_the_residual(dim):
    """The second norm's sum must not be put together from parts that cancel."""
    import tcu_scope_b200 as tcu
    s = make(9, dim, F32, F32, 1, 8)
    z = s["z"].double()
    n = z / (z.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * s["post"].double() * s["gate"].double() * 0.75
    for row, left in enumerate((0.0, 1e-6, 1e-4, 1e-2, 0.1, 0.4, 0.6, 1.0, 2.0)):
        s["residual"][row] = (-n[row] + left * s["residual"][row].double()).float()
    check(s, "none", *run(tcu, s, "none"))


@pytest.mark.parametrize("dim", [200, 1000])
def test_parts_beyond_float32(dim):
    """Products of large rows and weights leave float32 although the row's sum of squares and all results do not."""
    import tcu_scope_b200 as tcu
    s = make(5, dim, F32, F32, 1, 8)
    s["z"][1] *= 1e17
    s["z"][3] *= 1e17
    s["residual"][3] = 0
    s["post"] *= 1000
    check(s, "none", *run(tcu, s, "none"))


@pytest.mark.parametrize("kind", [BF16, F32])
@pytest.mark.parametrize("dim", [200, 1000, 4096])
@pytest.mark.parametrize("post", [False, True])
def test_gradient_of_rows_of_any_size(kind, dim, post):
    """Rows whose 1 / rms has a square or a cube beyond float32, while the sum of squares is not."""
    import tcu_scope_b200 as tcu
    for size, eps in ((1e13, 1e-6), (1e15, 1e-6), (1e17, 1e-6), (1e-14, 0.0), (1e-17, 0.0)):
        for plain in (True, False):  # without a residual, and with one that sets the size of `out` where z is normed
            s = make(4, dim, kind, F32, 0 if plain else 1, 8, residual=not plain, post=post)
            s["z"] *= size / 3
            if not plain:
                s["residual"] *= size / 3
            zero = {**s, "dout": torch.zeros_like(s["z"])}
            none = run(tcu, {**s, "dout": None}, "none", eps=eps)
            check(zero, "none", *none, eps=eps)
            s["dout"] *= 1 / size  # as large as what comes through the norm
            check(s, "none", *run(tcu, s, "none", eps=eps), eps=eps)


def test_no_rows():
    import tcu_scope_b200 as tcu
    s = make(1, 48, BF16, F32, 1, 8)
    s = {k: v if k in ("post", "pre", "gate") else v[:0] for k, v in s.items()}
    out, normed, d = run(tcu, s, "none")
    assert out.shape == (0, 48) and d.dz.shape == (0, 48)
    assert all(bool((t == 0).all()) for t in (d.dpost_weight, d.dgate, d.dpre_weight))


@pytest.mark.parametrize("kind", [BF16, F32])
def test_strided_and_unaligned_rows(kind):
    import tcu_scope_b200 as tcu
    s = make(24, 136, kind, kind, 24, 2)
    wide = torch.randn(24, 5 * 136 + 24, generator=torch.Generator().manual_seed(1)).to(kind).cuda()
    for shift in (0, 1, 8):
        names = ["z", "residual", "gate", "dout", "dnormed"]
        for i, name in enumerate(names):
            s[name] = wide[:, i * 136 + shift:(i + 1) * 136 + shift]
        check(s, "silu", *run(tcu, s, "silu"))
    # the residual and the gradient broadcast from one row
    s["residual"], s["dout"] = wide[:1, :136].expand(24, 136), wide[:1, 136:272].expand(24, 136)
    check(s, "silu", *run(tcu, s, "silu"))


def test_three_dimensions_and_gates_of_sequences():
    import tcu_scope_b200 as tcu
    s = make(2 * 9, 80, F32, F32, 2, 4)
    flat = run(tcu, s, "silu")
    three = {k: v.view(2, 9, 80) if k in ("z", "residual", "dout", "dnormed") else v for k, v in s.items()}
    three["gate"] = s["gate"].view(2, 1, 80)
    got = run(tcu, three, "silu")
    assert got[0].shape == (2, 9, 80) and got[2].dgate.shape == (2, 1, 80)
    assert all(torch.equal(p.flatten(), q.flatten()) for p, q in zip([*flat[:2], *flat[2]], [*got[:2], *got[2]]))
    s1 = {**s, "gate": s["gate"][:1]}
    vec = {**s, "gate": s["gate"][0]}
    assert all(torch.equal(p.flatten(), q.flatten()) for p, q in zip(run(tcu, s1, "none")[2], run(tcu, vec, "none")[2]))


@pytest.mark.parametrize("dim", [64, 1000])
def test_results_over_inputs(dim):
    """The buffers that the documentation allows to be shared."""
    import tcu_scope_b200 as tcu
    s = make(30, dim, BF16, BF16, 1, 6)
    out, normed, d = run(tcu, s, "none")
    args = dict(post_weight=s["post"], gate=s["gate"], scale=0.75, pre_weight=s["pre"])
    z, r = s["z"].clone(), s["residual"].clone()
    o, u = tcu.norm_residual(z, r, **args, out=r, normed=z)
    assert o is r and u is z and torch.equal(o, out) and torch.equal(u, normed)
    z = s["z"].clone()
    assert torch.equal(tcu.norm_residual(z, s["residual"], **args, out=z)[0], out)
    for over in ("dout", "dnormed", "z"):
        t = {k: None if v is None else v.clone() for k, v in s.items()}
        more = dict(dz=t[over])
        if over != "dout":
            more["dresidual"] = t["dout"]
        got = run(tcu, t, "none", **more)[2]
        assert all(torch.equal(p, q) for p, q in zip(got, d)), over


def test_gradient_against_differences():
    import tcu_scope_b200 as tcu
    s = make(4, 6, F32, F32, 2, 9)
    d = run(tcu, s, "silu")[2]
    cpu = {k: t.double().cpu() for k, t in s.items()}

    def loss(c):
        w = ref.norm_residual(c["z"], c["residual"], c["post"], c["gate"].repeat_interleave(2, 0), "silu", 0.75, c["pre"], 1e-6)
        return float((w["out"].v * cpu["dout"]).sum() + (w["normed"].v * cpu["dnormed"]).sum())

    for name, got in (("z", d.dz), ("residual", d.dresidual), ("post", d.dpost_weight), ("gate", d.dgate), ("pre", d.dpre_weight)):
        for i in range(cpu[name].numel()):
            up, down = ({k: v.clone() for k, v in cpu.items()} for _ in range(2))
            up[name].view(-1)[i] += 1e-5
            down[name].view(-1)[i] -= 1e-5
            slope = (loss(up) - loss(down)) / 2e-5
            # the third derivatives are below 1e3, so the quotient is within 1e-7 of the slope
            assert abs(slope - float(got.view(-1)[i])) < 2e-5 * max(1.0, abs(slope)), (name, i)


def test_other_stream_captured_graph_and_own_workspace():
    import tcu_scope_b200 as tcu
    s = make(300, 1024, BF16, F32, 1, 3)
    want = run(tcu, s, "none")
    need = tcu._lib.load().tcu_norm_residual_workspace_bytes(300, 1024, 1)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # NaN where it is read before it is written
    flat = lambda g: [*g[:2], *g[2]]  # noqa: E731
    assert all(torch.equal(p, q) for p, q in zip(flat(want), flat(run(tcu, s, "none", workspace=ws))))
    with pytest.raises(tcu.TcuError, match="workspace"):
        run(tcu, s, "none", workspace=ws[:-64])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(tcu, s, "none")
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(flat(want), flat(got)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(tcu, s, "none")
    for t in (s["z"], s["dout"]):
        t.copy_(t.flip(0))
    want = run(tcu, s, "none")
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(flat(want), flat(got)))
