"""CPU: what token embedding, cross attention and distillation refuse, through the C ABI and through the host side, without a GPU call."""
import ctypes as C

import pytest
import torch

import dualvgr_videoqa_amd as dv
from dualvgr_videoqa_amd import _lib as L
from dualvgr_videoqa_amd import head as HD
from dualvgr_videoqa_amd import inputs as IN

E_DIMS, E_NULL, E_WORKSPACE, E_ALIGN, E_KIND = -1, -2, -3, -4, -5
_buf = (C.c_char * 8192)()
A = (C.addressof(_buf) + 255) // 256 * 256          # an address that is only ever looked at


def test_embedding_refusals():
    f, b, ws = IN.load().dvgr_embed_forward, IN.load().dvgr_embed_backward, IN.load().dvgr_embed_workspace_bytes
    assert f(A, 10, 8, 3, A, 4, 1.0, A, None, None) == E_KIND
    assert f(A, 0, 8, 0, A, 4, 1.0, A, None, None) == E_DIMS
    assert f(A, 10, 0, 0, A, 4, 1.0, A, None, None) == E_DIMS
    assert f(A, 10, 8, 0, A, -1, 1.0, A, None, None) == E_DIMS
    assert f(A, 10, 8, 0, A, 1 << 26, 1.0, A, None, None) == E_DIMS
    assert f(A, (1 << 31) - 1, 8, 0, A, 4, 1.0, A, None, None) == E_DIMS
    assert f(None, 10, 8, 0, A, 4, 1.0, A, None, None) == E_NULL
    assert f(A, 10, 8, 0, None, 4, 1.0, A, None, None) == E_NULL
    assert f(A, 10, 8, 0, A, 4, 1.0, None, None, None) == E_NULL
    assert f(None, 10, 8, 0, None, 0, 1.0, None, None, None) == 0                     # nothing to do
    need = ws(9000, 10, 8, 0)
    assert need > 0 and ws(100, 10, 8, 0) == 0 and ws(0, 10, 8, 0) == 0 and ws(-1, 10, 8, 0) == 0 and ws(100, 10, 8, 9) == 0
    assert b(A, A, 9000, 10, 8, 0, 1.0, -1, None, A, need, None) == E_NULL
    assert b(None, A, 9000, 10, 8, 0, 1.0, -1, A, A, need, None) == E_NULL
    assert b(A, A, 9000, 10, 8, 0, 1.0, -1, A, None, need, None) == E_NULL
    assert b(A, A, 9000, 10, 8, 0, 1.0, -1, A, A, need - 1, None) == E_WORKSPACE
    assert b(A, A, 9000, 10, 8, 0, 1.0, -1, A, A + 8, need, None) == E_ALIGN
    assert b(A, A, 9000, 10, 8, 7, 1.0, -1, A, A, need, None) == E_KIND


def test_distillation_refusals():
    lib = HD.load()
    f, b, ws = lib.dvgr_distill_forward, lib.dvgr_distill_backward, lib.dvgr_distill_workspace_bytes
    ok = dict(z=A, ld=100, e=0, R=4, C=100, v=A, ev=0, i=A, K=5, T=1.0, red=2, rows=A, total=A, stats=A, ws=None, wb=0)

    def fwd(**kw):
        d = {**ok, **kw}
        return f(d["z"], d["ld"], d["e"], d["R"], d["C"], d["v"], d["ev"], d["i"], d["K"], d["T"], d["red"], d["rows"], d["total"], d["stats"],
                 d["ws"], d["wb"], None)

    for kw in (dict(e=3), dict(ev=-1), dict(red=3), dict(red=-1)):
        assert fwd(**kw) == E_KIND, kw
    for kw in (dict(ld=99), dict(C=0), dict(K=0), dict(K=1025), dict(T=0.0), dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")), dict(R=-1),
               dict(R=1 << 22)):
        assert fwd(**kw) == E_DIMS, kw
    for kw in (dict(z=None), dict(v=None), dict(i=None), dict(rows=None), dict(total=None), dict(stats=None)):
        assert fwd(**kw) == E_NULL, kw
    for kw in (dict(stats=A + 4), dict(z=A + 2), dict(v=A + 1, ev=1)):
        assert fwd(**kw) == E_ALIGN, kw
    big = dict(R=1, C=100000, ld=100000)
    need = ws(1, 100000)
    assert need > 0 and ws(1 << 20, 100000) == 0 and ws(0, 5) == 0
    assert fwd(**big) == E_NULL and fwd(**big, ws=A, wb=need - 1) == E_WORKSPACE and fwd(**big, ws=A + 8, wb=need) == E_ALIGN
    assert b(A, 100, 0, 4, 100, A, 0, A, 5, 1.0, A, A, 2, A, 100, None) == E_DIMS          # stride of the upstream gradient: 0 or 1
    assert b(A, 100, 0, 4, 100, A, 0, A, 5, 1.0, A, A, 0, A, 99, None) == E_DIMS
    assert b(A, 100, 0, 4, 100, A, 0, A, 5, 1.0, A, None, 0, A, 100, None) == E_NULL
    assert b(A, 100, 0, 4, 100, A, 0, A, 5, 1.0, A, A, 0, None, 100, None) == E_NULL
    assert b(A, 100, 0, 4, 100, A, 0, A, 5, 1.0, A, A, 0, A + 2, 100, None) == E_ALIGN
    assert b(None, 100, 0, 0, 100, None, 0, None, 5, 1.0, None, None, 0, None, 100, None) == 0


def problem(**kw):
    p = L.AttnProblem(B=2, Lq=3, Lk=5, H=4, Hk=2, Dh=16, elem=0, scale=0.25)
    for n in "qkvo":
        setattr(p, n, L.AttnView(A, 1024, 64, 16))
    p.lse = A
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_attention_refusals():
    lib = L.load()
    assert C.sizeof(L.AttnView) == 32 and C.sizeof(L.AttnProblem) == 32 + 4 * 32 + 5 * 8 and C.sizeof(L.AttnGrads) == 4 * 32
    assert lib.dvgr_attn_check(C.byref(problem())) == 0 and lib.dvgr_attn_check(None) == E_NULL
    for kw in (dict(B=-1), dict(Lq=-1), dict(Lk=-1), dict(H=0), dict(Hk=0), dict(H=5), dict(Dh=0), dict(Dh=12), dict(Dh=136), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(Lk=1 << 30), dict(Lq=1 << 29), dict(B=1 << 24)):
        assert lib.dvgr_attn_check(C.byref(problem(**kw))) == E_DIMS, kw
        assert lib.dvgr_attn_forward(C.byref(problem(**kw)), None, 0, None) == E_DIMS, kw
    assert lib.dvgr_attn_check(C.byref(problem(elem=5))) == E_KIND
    none, off, odd = L.AttnView(None, 1024, 64, 16), L.AttnView(A + 8, 1024, 64, 16), L.AttnView(A, 1024, 65, 16)
    for n in "qkvo":
        assert lib.dvgr_attn_forward(C.byref(problem(**{n: none})), None, 0, None) == E_NULL
        assert lib.dvgr_attn_forward(C.byref(problem(**{n: off})), None, 0, None) == E_ALIGN
        assert lib.dvgr_attn_forward(C.byref(problem(**{n: odd})), None, 0, None) == E_ALIGN
    assert lib.dvgr_attn_forward(C.byref(problem(B=0)), None, 0, None) == 0 and lib.dvgr_attn_forward(C.byref(problem(Lq=0)), None, 0, None) == 0
    long = problem(Lk=100000, Lq=1)
    need = lib.dvgr_attn_forward_workspace_bytes(C.byref(long))
    assert need > 0 and lib.dvgr_attn_forward(C.byref(long), None, 0, None) == E_NULL
    assert lib.dvgr_attn_forward(C.byref(long), A, need - 1, None) == E_WORKSPACE and lib.dvgr_attn_forward(C.byref(long), A + 4, need, None) == E_ALIGN
    g = lambda **kw: L.AttnGrads(**{n: kw.get(n, L.AttnView(A, 1024, 64, 16)) for n in ("g_o", "g_q", "g_k", "g_v")})  # noqa: E731
    p = problem(Lq=40)
    need = lib.dvgr_attn_backward_workspace_bytes(C.byref(p))
    back = lambda q, gr, ws=A, n=need: lib.dvgr_attn_backward(C.byref(q), C.byref(gr) if gr else None, ws, n, None)  # noqa: E731
    assert need > 0 and back(p, None) == E_NULL and back(p, g(g_o=none)) == E_NULL and back(p, g(g_k=none)) == E_NULL
    assert back(problem(Lq=40, lse=None), g()) == E_NULL and back(p, g(), None) == E_NULL
    assert back(p, g(), A, need - 1) == E_WORKSPACE and back(p, g(), A + 8) == E_ALIGN
    for n in ("g_o", "g_q", "g_k", "g_v"):
        assert back(p, g(**{n: odd})) == E_ALIGN
    assert back(problem(B=0), g()) == 0


def test_host_side_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dv.embed_tokens(torch.zeros(4, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dv.TokenEmbedding(4, 8)(torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dv.distillation_loss(torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dv.cross_attention(torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1, 8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dv.CrossAttention(64, 2)(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64))


def test_constructors_refuse():
    for kw in (dict(module_dim=100, num_heads=8), dict(module_dim=768, num_heads=4), dict(module_dim=768, num_heads=8, key_heads=3),
               dict(module_dim=24, num_heads=2)):
        with pytest.raises(ValueError):
            dv.CrossAttention(**kw)
    assert set(dv.TokenEmbedding(4, 8, padding_idx=1).state_dict()) == {"weight"}
    assert {k.split(".")[0] for k in dv.CrossAttention(64, 2).state_dict()} == {"query", "key_value", "out"}


def test_projections_refuse_what_their_kernels_cannot_read():
    lin = dv.HipLinear(64, 32)
    for t in (torch.bfloat16, torch.float16, torch.float64):
        with pytest.raises(RuntimeError, match="fp32 on one device; the input"):
            lin(torch.zeros(3, 64, dtype=t))
    for shape in ((3, 60), (3, 68), (64, 3), ()):
        with pytest.raises(RuntimeError, match="64 input features"):
            lin(torch.zeros(shape))
    with pytest.raises(RuntimeError, match="fp32 on one device; the weight"):
        dv.HipLinear(64, 32).to(torch.bfloat16)(torch.zeros(3, 64))
    cast = dv.HipLinear(64, 32)
    cast.bias = torch.nn.Parameter(cast.bias.detach().half())
    with pytest.raises(RuntimeError, match="fp32 on one device; the bias"):
        cast(torch.zeros(3, 64))

    attend = dv.CrossAttention(64, 2, state_dim=48, dtype="bf16")
    x, s = torch.zeros(1, 2, 64), torch.zeros(1, 5, 48)
    for t in (torch.float64, torch.int64):
        with pytest.raises(RuntimeError, match="in fp32, bf16 or fp16"):
            attend(x.to(t), s)
        with pytest.raises(RuntimeError, match="in fp32, bf16 or fp16"):
            attend(x, s.to(t))
    with pytest.raises(RuntimeError, match="batch, length, features"):
        attend.states(s[0])
    with pytest.raises(RuntimeError, match="48 input features"):
        attend.states(x)
    assert attend.half() is attend                                  # nn.Module's own cast, then refused by name
    with pytest.raises(RuntimeError, match="fp32 on one device; the weight"):
        attend(x, s)


def test_the_look_at_a_captured_backward_finds_leaves_behind_views_and_copies():
    ops = L.torch_ops()
    x, w = torch.randn(3, 4, 10, requires_grad=True), torch.randn(10, 8, requires_grad=True)
    found = lambda t: {id(u) for u in ops.dbg_leaves(t)}  # noqa: E731
    assert found(x.reshape(-1, 10)) == {id(x)} == found(x.transpose(0, 2).contiguous()) == found(x[:, :, :5])
    y = x.view(12, 10) @ w
    assert found(y) == {id(x), id(w)} == found(torch.cat([y[:, :4].float(), y[:, 4:]]).exp())
    assert found(y.detach()) == set() and found(x) == set()
    assert not ops.dbg_refuses_capture(y)                           # nothing of a device


def _calls():
    ids = torch.zeros(2, 3, dtype=torch.int64)
    x = torch.randn(1, 4, 2, 8)
    return [(lambda t: dv.embed_tokens(t, ids[0]), torch.randn(5, 8)), (lambda z: dv.distillation_loss(z, torch.zeros(2, 3), ids), torch.randn(2, 9)),
            (lambda q: dv.cross_attention(q, x, x), x), (lambda k: dv.cross_attention(x, k, x), x), (lambda v: dv.cross_attention(x, x, v), x)]


def test_inputs_with_a_tangent_and_traces_are_refused():
    import torch.autograd.forward_ad as fwd
    for call, t in _calls():
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(fwd.make_dual(t, torch.ones_like(t)))
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, t, check_trace=False)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call(t)


def test_attention_stays_under_a_launch_of_2_32_threads():
    # dK and dV: 512 threads for 128 keys, workgroups rounded up to a multiple of 8; D: 256 threads for 64 rows
    check = lambda **kw: L.load().dvgr_attn_check(C.byref(problem(B=1, H=1, Hk=1, **kw)))  # noqa: E731
    for tiles in range((1 << 23) - 16, 1 << 23):
        grid = (tiles + 7) // 8 * 8
        assert (check(Lk=128 * tiles - 1) == 0) == (grid * 512 < 1 << 32), tiles
    assert check(Lq=(1 << 30) - 1) == E_DIMS and check(Lq=(1 << 30) - 128) == 0
