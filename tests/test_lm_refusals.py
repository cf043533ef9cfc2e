"""Calls that the language-model operators refuse: nothing here reaches a GPU."""
import struct

import pytest
import torch

INVALID, UNSUPPORTED = 1, 2


@pytest.fixture()
def lib(built_library):
    import tcu_scope_b200 as tcu
    return tcu._lib.load()


def pack(layout, **fields):
    """The bytes of an argument struct from its fields' names; what is not named is 0."""
    return struct.pack(f"={len(layout)}q", *[fields.pop(f, 0) for f in layout]), assert_empty(fields)


def assert_empty(fields):
    assert not fields, fields


def fields_of(name):
    """The fields of a struct of the header, in order."""
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "tcu_scope.h")).read(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", text).group(1)
    out = []
    for line in body.split(";"):
        words = re.sub(r"\b(const|void|float|double|int64_t)\b|\*", " ", line).replace(",", " ").split()
        out += words
    return out


SCAN = dict(a=0x1000, x=0x2000, h=0x3000, batch=2, tokens=8, dim=16, type=2, a_type=2)


@pytest.mark.parametrize("change,status", [
    (dict(type=9), UNSUPPORTED), (dict(a_type=0), UNSUPPORTED), (dict(gate=3), UNSUPPORTED),
    (dict(a=0), INVALID), (dict(x=0), INVALID), (dict(h=0), INVALID), (dict(x=0x2001), INVALID),
    (dict(a=0x1002, a_type=1), INVALID), (dict(h0=0x5002), INVALID), (dict(batch=-1), INVALID),
    (dict(tokens=1 << 41), INVALID), (dict(batch=1 << 30, tokens=1 << 30), INVALID),
    (dict(offsets=0x7004, offsets_are_64bit=1), INVALID),
    (dict(batch=0), 0), (dict(dim=0, a=0), 0),
])
def test_linear_scan_c_refusals(lib, change, status):
    args, _ = pack(fields_of("tcu_linear_scan_args"), **{**SCAN, **change})
    assert lib.tcu_linear_scan(args, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(states=0), INVALID), (dict(da=0), INVALID), (dict(dx=0x6001), INVALID), (dict(dlast=2), INVALID),
    (dict(type=7), UNSUPPORTED), (dict(batch=0), 0),
])
def test_linear_scan_backward_c_refusals(lib, change, status):
    base = dict(a=0x1000, x=0x2000, dh=0x3000, states=0x4000, da=0x5000, dx=0x6000, batch=2, tokens=8, dim=16,
                type=0, a_type=1)
    args, _ = pack(fields_of("tcu_linear_scan_backward_args"), **{**base, **change})
    assert lib.tcu_linear_scan_backward(args, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(pool=1), INVALID), (dict(state=0), INVALID), (dict(state=0x4002), INVALID), (dict(gate=-1), UNSUPPORTED),
    (dict(batch=0), 0),
])
def test_linear_scan_step_c_refusals(lib, change, status):
    base = dict(a=0x1000, x=0x2000, h=0x3000, state=0x4000, batch=2, pool=2, dim=16, type=1, a_type=1)
    args, _ = pack(fields_of("tcu_linear_scan_step_args"), **{**base, **change})
    assert lib.tcu_linear_scan_step(args, None) == status


def test_null_arguments(lib):
    for name in ("tcu_linear_scan", "tcu_linear_scan_backward", "tcu_linear_scan_step"):
        assert getattr(lib, name)(None, None) == INVALID


def test_states_rows(lib):
    assert lib.tcu_linear_scan_states_rows(3, 16, 0) == 3 and lib.tcu_linear_scan_states_rows(3, 17, 0) == 6
    assert lib.tcu_linear_scan_states_rows(3, 17, 1) == 4 and lib.tcu_linear_scan_states_rows(3, 0, 0) == 0


def test_python_structs_match_the_header(built_library):
    import tcu_scope_b200.lm as lm
    for layout, name in ((lm._SCAN, "tcu_linear_scan_args"), (lm._SCAN_BACKWARD, "tcu_linear_scan_backward_args"),
                         (lm._STEP, "tcu_linear_scan_step_args")):
        assert layout.size == 8 * len(fields_of(name)), name


def test_cpu_tensors_are_refused(built_library):
    import tcu_scope_b200 as tcu
    x = torch.zeros(1, 4, 8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        tcu.linear_scan(x, x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        tcu.linear_scan_backward(x, x, x, x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        tcu.linear_scan_step(x[0], x[0], x[0])


def test_tangents_are_refused(built_library):
    """Forward-mode autograd would lose them; inside a Function with a jvp of its own they are not there."""
    import torch.autograd.forward_ad as fw
    import tcu_scope_b200.lm as lm
    x, i, cuda = torch.ones(3), torch.zeros(3, dtype=torch.int32), torch.device("cuda", 0)

    class Here:  # the CPU under the name of a GPU
        type = "cuda"

        def __ne__(self, other):
            return other != torch.device("cpu")

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(x):
            lm._inputs(Here(), ("x",), (x,))
            return 2 * x

        @staticmethod
        def setup_context(ctx, inputs, output):
            pass

        @staticmethod
        def jvp(ctx, t):
            return 2 * t

    with fw.dual_level():
        dual = fw.make_dual(x, x)
        for t in (dual, dual[1:]):
            for names, tensors in ((("x",), (t,)), (("x", "a"), (t, None))):
                with pytest.raises(RuntimeError, match="tangent"):
                    lm._inputs(cuda, names, tensors)
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                lm._inputs(cuda, ("x",), (t,))
        for t in (x, i, fw.unpack_dual(dual).primal):
            with pytest.raises(RuntimeError, match="cpu"):
                lm._inputs(cuda, ("x",), (t,))
        assert torch.equal(fw.unpack_dual(Twice.apply(dual)).tangent, 2 * x)


@pytest.mark.gpu
def test_every_operator_refuses_tangents():
    import torch.autograd.forward_ad as fw
    import tcu_scope_b200 as tcu
    x, w, s = torch.ones(2, 4, 8, device="cuda"), torch.ones(8, device="cuda"), torch.ones(4, 8, device="cuda")
    states, at, t = tcu.linear_scan_states(x), torch.tensor([0, 4], device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    one = torch.ones(4, device="cuda")
    with fw.dual_level():
        dual = lambda v: fw.make_dual(v, torch.ones_like(v))  # noqa: E731
        for call in (lambda: tcu.linear_scan(x, dual(x)), lambda: tcu.linear_scan(dual(x), x),
                     lambda: tcu.linear_scan(s, s, h0=dual(w[None]), offsets=at),
                     lambda: tcu.linear_scan_backward(dual(x), x, x, states), lambda: tcu.linear_scan_step(s, dual(s), s.clone()),
                     lambda: tcu.linear_scan_step(s, s, dual(s.clone())), lambda: tcu.norm_residual(dual(x), pre_weight=w),
                     lambda: tcu.norm_residual(x, pre_weight=dual(w)), lambda: tcu.norm_residual(x, dual(x)),
                     lambda: tcu.norm_residual_backward(dual(x), None, x), lambda: tcu.token_logprobs(dual(s), t),
                     lambda: tcu.token_logprobs_backward(s, t, one, dlogprob=dual(one))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        h, last = tcu.linear_scan(s, s, h0=w[None], offsets=at)  # tensors without one are taken
        assert float(last[0, 0]) == 5


@pytest.mark.gpu
def test_linear_scan_python_refusals():
    import tcu_scope_b200 as tcu
    x = torch.zeros(2, 4, 8, device="cuda")
    s = tcu.linear_scan_states(x)
    with pytest.raises(TypeError):
        tcu.linear_scan(x.half(), x)
    with pytest.raises(TypeError):
        tcu.linear_scan(x.double(), x.double())
    with pytest.raises(ValueError):
        tcu.linear_scan(x, x, gate="tanh")
    with pytest.raises(ValueError):
        tcu.linear_scan(x[:1], x)
    with pytest.raises(ValueError):
        tcu.linear_scan(x[0], x[0])
    with pytest.raises(ValueError):
        tcu.linear_scan(x.transpose(1, 2), x.transpose(1, 2))
    with pytest.raises(ValueError):
        tcu.linear_scan(x, x, h0=torch.zeros(2, 7, device="cuda"))
    with pytest.raises(ValueError):
        tcu.linear_scan(x, x, h0=torch.zeros(2, 8, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError):
        tcu.linear_scan(x, x, states=s[:1])
    with pytest.raises(ValueError):
        tcu.linear_scan(x, x, out=torch.zeros(2, 8, 4, device="cuda").transpose(1, 2))
    with pytest.raises(ValueError):
        tcu.linear_scan(x, x, offsets=torch.zeros(3, device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError):
        tcu.linear_scan(x[0], x[0], offsets=torch.zeros(3, device="cuda"))
    with pytest.raises(RuntimeError):
        tcu.linear_scan(x[0], x[0], offsets=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="gradient"):
        tcu.linear_scan(x, x.clone().requires_grad_())
    with torch.no_grad():
        tcu.linear_scan(x, x.clone().requires_grad_())
    with pytest.raises(ValueError):
        tcu.linear_scan_backward(x[:, :3], x, x, s)
    with pytest.raises(ValueError):
        tcu.linear_scan_backward(x, x, x, s[:1])
    with pytest.raises(ValueError):
        tcu.linear_scan_step(x[0], x[0], torch.zeros(3, 8, device="cuda"))
    with pytest.raises(ValueError):
        tcu.linear_scan_step(x[0], x[0], torch.zeros(4, 8, device="cuda"), slots=torch.zeros(3, device="cuda", dtype=torch.int32))


NORM = dict(z=0x1000, post_weight=0x2000, out=0x3000, rows=4, dim=64, type=0, weight_type=1)


@pytest.mark.parametrize("change,status", [
    (dict(type=3), UNSUPPORTED), (dict(weight_type=2), UNSUPPORTED), (dict(act=3), UNSUPPORTED),
    (dict(dim=16385), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(gate=0x4000, gate_rows=3), INVALID),
    (dict(gate=0x4000, gate_rows=0), INVALID), (dict(z=0), INVALID), (dict(out=0), INVALID), (dict(z=0x1001), INVALID),
    (dict(post_weight=0x2002), INVALID), (dict(pre_weight=0x5000), INVALID), (dict(rows=0), 0),
])
def test_norm_residual_c_refusals(lib, change, status):
    args, _ = pack(fields_of("tcu_norm_residual_args"), **{**NORM, **change})
    assert lib.tcu_norm_residual(args, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(dz=0), INVALID), (dict(dgate=0x6000), INVALID), (dict(dpre_weight=0x6000), INVALID), (dict(workspace=0), 5),
    (dict(workspace=0x7008), 5), (dict(workspace_bytes=16), 5), (dict(dresidual=0x8001), INVALID),
    (dict(rows=0, dpost_weight=0), 0),
])
def test_norm_residual_backward_c_refusals(lib, change, status):
    base = dict(z=0x1000, dout=0x1100, post_weight=0x2000, dz=0x3000, dpost_weight=0x5000, workspace=0x7000,
                workspace_bytes=1 << 30, rows=4, dim=64, type=0, weight_type=1)
    args, _ = pack(fields_of("tcu_norm_residual_backward_args"), **{**base, **change})
    assert lib.tcu_norm_residual_backward(args, None) == status


def test_norm_structs_and_workspace(lib):
    import tcu_scope_b200.lm as lm
    for layout, name in ((lm._NORM, "tcu_norm_residual_args"), (lm._NORM_BACKWARD, "tcu_norm_residual_backward_args")):
        assert layout.size == 8 * len(fields_of(name)), name
    ws = lib.tcu_norm_residual_workspace_bytes
    assert ws(0, 64, 1) == 0 and ws(10, 0, 1) == 0
    assert ws(1 << 20, 4096, 1) >= ws(100, 4096, 1) > 0
    for name in ("tcu_norm_residual", "tcu_norm_residual_backward"):
        assert getattr(lib, name)(None, None) == INVALID


@pytest.mark.gpu
def test_norm_residual_python_refusals():
    import tcu_scope_b200 as tcu
    z = torch.zeros(2, 4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for bad in (dict(z=z.double(), post_weight=w), dict(z=z, post_weight=w.half()), dict(z=z, post_weight=w[:7])):
        with pytest.raises((TypeError, ValueError)):
            tcu.norm_residual(bad.pop("z"), **bad)
    with pytest.raises(ValueError):
        tcu.norm_residual(z, z[:1], post_weight=w)
    with pytest.raises(ValueError):
        tcu.norm_residual(z, post_weight=w, gate_act="tanh")
    for shape in ((1, 4, 8), (4, 8), (3, 8), (2, 4, 1)):  # a gate for each token, broadcast over the batch, is not one of consecutive rows
        with pytest.raises(ValueError):
            tcu.norm_residual(z, post_weight=w, gate=torch.zeros(shape, device="cuda"))
    for shape in ((8,), (1, 1, 8), (2, 1, 8), (2, 4, 8)):
        tcu.norm_residual(z, post_weight=w, gate=torch.zeros(shape, device="cuda"))
    with pytest.raises(ValueError):
        tcu.norm_residual(z, post_weight=w, normed=z)
    with pytest.raises(ValueError):
        tcu.norm_residual(z.transpose(1, 2), post_weight=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="stride"):
        tcu.norm_residual(torch.zeros(4, 2, 8, device="cuda").transpose(0, 1)[:, :3], post_weight=w)
    with pytest.raises(tcu.TcuError):
        tcu.norm_residual(torch.zeros(2, 16385, device="cuda"), post_weight=torch.ones(16385, device="cuda"))
    with pytest.raises(RuntimeError, match="gradient"):
        tcu.norm_residual(z, post_weight=w.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        tcu.norm_residual(z, post_weight=w.cpu())
    with pytest.raises(ValueError):
        tcu.norm_residual_backward(z, z, z, post_weight=w)
    with pytest.raises(ValueError):
        tcu.norm_residual_backward(z, None, z, post_weight=w, dresidual=z)
    with pytest.raises(ValueError):
        tcu.norm_residual_backward(z[:1], None, z, post_weight=w)


LOGPROBS = dict(logits=0x1000, targets=0x2000, logprob=0x3000, entropy=0x4000, lse=0x5000, rows=3, vocab=100,
                row_stride=100, type=2, targets_are_64bit=1)


@pytest.mark.parametrize("change,status", [
    (dict(type=5), UNSUPPORTED), (dict(top=33, vocab=200), UNSUPPORTED), (dict(top=-1), UNSUPPORTED),
    (dict(top=4), INVALID), (dict(top=4, vocab=3, top_logprob=0x6000, top_index=0x7000), INVALID),
    (dict(top=4, top_logprob=0x6000, top_index=0x7004), INVALID), (dict(targets=0), INVALID), (dict(targets=0x2004), INVALID),
    (dict(logits=0), INVALID), (dict(logits=0x1001), INVALID), (dict(vocab=0), INVALID), (dict(rows=-1), INVALID),
    (dict(vocab=1 << 31), INVALID), (dict(rows=1 << 31), INVALID), (dict(lse=0x5002), INVALID), (dict(rows=0), 0),
])
def test_token_logprobs_c_refusals(lib, change, status):
    args, _ = pack(fields_of("tcu_token_logprobs_args"), **{**LOGPROBS, **change})
    assert lib.tcu_token_logprobs(args, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(lse=0), INVALID), (dict(dlogits=0), INVALID), (dict(dlogits=0x6001), INVALID), (dict(targets=0), INVALID),
    (dict(dentropy=0x8000, entropy=0), INVALID), (dict(type=-1), UNSUPPORTED), (dict(rows=0), 0),
])
def test_token_logprobs_backward_c_refusals(lib, change, status):
    base = dict(logits=0x1000, targets=0x2000, lse=0x3000, entropy=0x4000, dlogprob=0x5000, dlogits=0x6000, rows=3,
                vocab=100, row_stride=100, type=0)
    args, _ = pack(fields_of("tcu_token_logprobs_backward_args"), **{**base, **change})
    assert lib.tcu_token_logprobs_backward(args, None) == status


def test_logprob_structs(lib):
    import tcu_scope_b200.lm as lm
    for layout, name in ((lm._LOGPROBS, "tcu_token_logprobs_args"), (lm._LOGPROBS_BACKWARD, "tcu_token_logprobs_backward_args")):
        assert layout.size == 8 * len(fields_of(name)), name
    for name in ("tcu_token_logprobs", "tcu_token_logprobs_backward"):
        assert getattr(lib, name)(None, None) == INVALID


@pytest.mark.gpu
def test_token_logprobs_python_refusals():
    import tcu_scope_b200 as tcu
    x, t = torch.zeros(3, 50, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        tcu.token_logprobs(x.double(), t)
    for bad in (t[:2], t.float(), t[:, None]):
        with pytest.raises(ValueError):
            tcu.token_logprobs(x, bad)
    with pytest.raises(RuntimeError):
        tcu.token_logprobs(x, t.cpu())
    with pytest.raises(ValueError):
        tcu.token_logprobs(x, t, top=51)
    with pytest.raises(tcu.TcuError):
        tcu.token_logprobs(x, t, top=33)
    with pytest.raises(ValueError):
        tcu.token_logprobs(x.t(), torch.zeros(50, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="gradient"):
        tcu.token_logprobs(x.clone().requires_grad_(), t)
    got = tcu.token_logprobs(x, t)
    with pytest.raises(ValueError):
        tcu.token_logprobs_backward(x, None, got.lse, got.entropy, dlogprob=got.lse)
    with pytest.raises(ValueError):
        tcu.token_logprobs_backward(x, t, got.lse, dentropy=got.lse)
    with pytest.raises(ValueError):
        tcu.token_logprobs_backward(x, t, got.lse[:2], got.entropy, dlogprob=got.lse)
    with pytest.raises(ValueError):
        tcu.token_logprobs_backward(x, t, got.lse, got.entropy, dlogprob=got.lse, out=x.half())
