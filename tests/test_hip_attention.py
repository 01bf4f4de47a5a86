"""GPU: attention to an encoder's states (include/dvgr_attn.h, attention.cross_attention) against 64 bits.

Tolerances, element by element, from the arithmetic.  A score is an fp32 dot product of Dh terms: off by (Dh + 4) 2^-24 of the sum
of its terms' sizes; a probability by E = that error + 2^-20 (its exponential and its row's sum), relative, and by half a step of
the type where the matrix unit takes it (h = finfo.eps / 2 for bf16 / fp16, 0 for fp32; fp16 also 2^-25, half its smallest number).
So o is off by (2 E + h + Lk 2^-24) sum p|v|, then half a step of its type; dS = p (dP - D) by 2 E of its size, by p times the
errors of dP (Dh 2^-24 sum |do||v|) and of D (sum |do| times o's error), and by half a step; the sums over keys and rows pass that on.
fp16 score gradients are scaled, so their smallest number is 2^-24 of the largest |do| of the tensor."""
import pytest
import torch

import dualvgr_videoqa_amd as dv
from dualvgr_videoqa_amd.attention import cross_attention

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def half(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def mm(a, b):
    return torch.matmul(a.contiguous(), b.contiguous())


def reference(q, k, v, lens, mask, scale, up):
    """(value, tolerance) of o, dq, dk, dv, per head group in (B, Hk, G * Lq, Dh) / (B, Hk, Lk, Dh) order, 64 bits."""
    t = q.dtype
    B, Lq, H, Dh = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G, h = H // Hk, half(t)
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    rows = lambda x: x.double().view(B, Lq, Hk, G, Dh).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, Dh)  # noqa: E731
    back = lambda x: x.view(B, Hk, G, Lq, Dh).permute(0, 3, 1, 2, 4).reshape(B, Lq, H, Dh)  # noqa: E731
    live = torch.ones(B, 1, 1, Lk, dtype=torch.bool, device=q.device)
    if lens is not None:
        live = live & (torch.arange(Lk, device=q.device) < lens.view(B, 1, 1, 1))
    if mask is not None:
        live = live & mask.view(B, 1, 1, Lk)
    clean = lambda x: torch.where(live.view(B, Lk, 1, 1), x.double(), 0.0).transpose(1, 2).contiguous()  # noqa: E731
    Q, K, V, D = rows(q), clean(k), clean(v), rows(up)
    S = mm(Q, K.transpose(2, 3)) * scale
    some = live.any(3, keepdim=True)
    P = torch.where(live & some, torch.softmax(torch.where(live, S, -torch.inf).masked_fill(~some, 0.0), 3), 0.0)
    E = (Dh + 4) * U * scale * mm(Q.abs(), K.abs().transpose(2, 3))
    E = torch.where(live, E, 0.0).amax(3, keepdim=True) * 2 + 2.0 ** -20 if Lk else torch.zeros_like(S[..., :1])
    step = lambda x: x.abs() * (torch.finfo(t).eps / 2) + torch.finfo(t).smallest_normal * torch.finfo(t).eps  # noqa: E731
    o, A = mm(P, V), mm(P, V.abs())
    o_tol = (2 * E + h + Lk * U) * A + tiny * V.abs().sum(2, keepdim=True)
    o_all = o_tol + step(o)
    rt = G * Lq
    dV = mm(P.transpose(2, 3), D)
    dV_tol = mm((P * (E + h) + tiny).transpose(2, 3), D.abs()) + rt * U * mm(P.transpose(2, 3), D.abs()) + step(dV)
    dP = mm(D, V.transpose(2, 3))
    delta = (D * o).sum(3, keepdim=True)
    dS = P * (dP - delta)
    dP_err = (Dh + 2) * U * mm(D.abs(), V.abs().transpose(2, 3))
    delta_err = (D.abs() * (o_all + Dh * U * o.abs())).sum(3, keepdim=True)
    tiny_s = 2.0 ** -24 * float(D.abs().max()) if t == torch.float16 else 0.0
    dS_err = dS.abs() * (2 * E + h + 4 * U) + P * (1 + E) * (dP_err + delta_err) + torch.where(live, tiny_s, 0.0)
    dQ, dK = mm(dS, K) * scale, mm(dS.transpose(2, 3), Q) * scale
    dQ_tol = scale * mm(dS_err + Lk * U * dS.abs(), K.abs()) + step(dQ)
    dK_tol = scale * mm((dS_err + rt * U * dS.abs()).transpose(2, 3), Q.abs()) + step(dK)
    out = lambda x: x.transpose(1, 2)  # noqa: E731
    return [(back(o), back(o_all)), (back(dQ), back(dQ_tol)), (out(dK), out(dK_tol)), (out(dV), out(dV_tol))]


def check(q, k, v, lens=None, mask=None, scale=None, up=None):
    up = torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(99), device="cuda").to(q.dtype) if up is None else up
    o = cross_attention(q, k, v, lens, mask, scale)
    grads = torch.autograd.grad(o, [q, k, v], up)
    with torch.no_grad():
        want = reference(q, k, v, lens, mask, scale or q.shape[3] ** -0.5, up)
        assert torch.equal(cross_attention(q, k, v, lens, mask, scale), o)
    for name, got, (w, tol) in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), want):
        assert got.dtype == q.dtype and got.shape == w.shape
        off = ((got.double() - w).abs() - tol)
        assert not torch.isnan(got).any(), name
        assert float(off.max() if off.numel() else 0.0) <= 0, (name, float(off.max()), float((got.double() - w).norm() / w.norm()))
    return o.detach(), grads


def tensors(B, Lq, Lk, H, Hk, Dh, t, seed=0, sharp=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + Lq * 7 + Lk)
    q = (torch.randn(B, Lq, H, Dh, generator=gen, device="cuda") * sharp).to(t)
    kv = torch.randn(B, Lk, 2, Hk, Dh, generator=gen, device="cuda").to(t)
    return q.requires_grad_(True), kv[:, :, 0].detach().requires_grad_(True), kv[:, :, 1].detach().requires_grad_(True), gen


SHAPES = [  # B, Lq, Lk, H, Hk, Dh
    (1, 1, 1, 1, 1, 8), (2, 3, 5, 2, 1, 32), (3, 20, 15, 8, 8, 96), (2, 33, 31, 4, 2, 40), (2, 32, 32, 1, 1, 64), (1, 129, 33, 2, 2, 128),
    (2, 15, 200, 4, 4, 96), (1, 1, 129, 8, 2, 64), (2, 7, 128, 8, 1, 72), (1, 64, 65, 3, 3, 16), (1, 200, 321, 4, 2, 120), (2, 257, 64, 2, 1, 104),
    (1, 130, 513, 1, 1, 128)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(t, shape):
    q, k, v, gen = tensors(*shape, t)
    a = check(q, k, v)
    b = check(q, k, v)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))      # the same inputs, the same bits


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(5, 20, 50, 4, 2, 96), (5, 3, 300, 8, 2, 64), (5, 150, 140, 2, 2, 32), (5, 40, 30, 2, 1, 128)])
def test_lengths_and_masks_that_leave_rows_empty(t, shape):
    B, Lq, Lk, H, Hk, Dh = shape
    q, k, v, gen = tensors(*shape, t)
    lens = torch.tensor([0, 1, Lk, Lk + 9, -4], device="cuda")
    mask = torch.rand(B, Lk, generator=gen, device="cuda") < 0.5
    mask[2] = False
    mask[3, :Lk - 2] = False
    mask[3, Lk - 2:] = True
    for ln, mk in ((lens, None), (None, mask), (lens, mask), (lens.int(), mask)):
        o, (dq, dk, dvv) = check(q, k, v, ln, mk)
        for b in range(B):
            n = Lk if ln is None else max(0, min(Lk, int(ln[b])))
            there = torch.arange(Lk, device="cuda") < n
            if mk is not None:
                there &= mk[b]
            if not bool(there.any()):
                assert (o[b] == 0).all() and (dq[b] == 0).all()
            assert (dk[b][~there] == 0).all() and (dvv[b][~there] == 0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,Lk", [(5, 150), (140, 150), (140, 20)])
def test_what_lies_in_keys_that_are_not_there_is_never_used(t, Lq, Lk):
    q, k, v, gen = tensors(3, Lq, Lk, 4, 2, 64, t)
    lens = torch.tensor([Lk - 7, Lk // 2, 0], device="cuda")
    mask = torch.rand(3, Lk, generator=gen, device="cuda") < 0.7
    want = check(q, k, v, lens, mask)
    gone = ~(mask & (torch.arange(Lk, device="cuda") < lens[:, None]))
    for bad in (float("nan"), float("inf"), -torch.finfo(t).max):
        k2, v2 = k.detach().clone(), v.detach().clone()
        k2[gone], v2[gone] = bad, bad
        o = cross_attention(q, k2.requires_grad_(True), v2.requires_grad_(True), lens, mask)
        got = torch.autograd.grad(o, [q, k2, v2], torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(99), device="cuda").to(t))
        assert torch.equal(o, want[0]) and all(torch.equal(x, y) for x, y in zip(got, want[1]))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,H,Hk,Lk,Dh", [(1, 8, 2, 5000, 128), (2, 4, 4, 2049, 64), (1, 32, 1, 1025, 96), (3, 1, 1, 640, 32)])
def test_one_word_over_a_long_video_splits_the_keys(t, B, H, Hk, Lk, Dh):
    q, k, v, gen = tensors(B, 1, Lk, H, Hk, Dh, t)
    lens = torch.randint(1, Lk + 1, (B,), generator=gen, device="cuda")
    mask = torch.rand(B, Lk, generator=gen, device="cuda") < 0.9
    check(q, k, v)
    check(q, k, v, lens, mask)
    check(q, k, v, torch.zeros_like(lens))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,Dh", [(1, 50, 2100, 2, 1, 64), (1, 3000, 20, 2, 1, 96), (2, 700, 300, 3, 1, 128), (1, 33, 1300, 1, 1, 40),
                                             (3, 1025, 65, 2, 2, 32)])
def test_small_batches_are_split_over_keys_and_rows(t, B, Lq, Lk, H, Hk, Dh):
    q, k, v, gen = tensors(B, Lq, Lk, H, Hk, Dh, t)
    a, b = check(q, k, v), check(q, k, v)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))
    check(q, k, v, torch.randint(0, Lk + 1, (B,), generator=gen, device="cuda"), torch.rand(B, Lk, generator=gen, device="cuda") < 0.8)


@pytest.mark.parametrize("t", TYPES)
def test_strides_and_alignment(t):
    q, k, v, gen = tensors(2, 20, 70, 4, 2, 64, t)
    want = check(q, k, v)
    packed = lambda x: x.detach().permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3).requires_grad_(True)  # heads first  # noqa: E731

    def shifted(x):                                                 # heads that no 16-byte load fits: copied
        flat = torch.zeros(x.numel() + 1, device="cuda", dtype=t)[1:].view(x.shape)
        flat.copy_(x.detach())
        return flat.requires_grad_(True)

    for f in (packed, shifted, lambda x: x.detach().transpose(2, 3).contiguous().transpose(2, 3).requires_grad_(True)):
        got = check(f(q), f(k), f(v))
        assert torch.equal(got[0], want[0]) and all(torch.equal(x, y) for x, y in zip(got[1], want[1]))
    one = k.detach()[:1].expand(2, -1, -1, -1).requires_grad_(True)  # one video for two questions
    check(q, one, one.detach().clone().requires_grad_(True))
    up = torch.randn(2, 4, 20, 64, generator=gen, device="cuda").to(t).transpose(1, 2)
    check(q, k, v, up=up)
    check(q, k, v, up=torch.ones(1, device="cuda", dtype=t).expand(q.shape))
    check(q, k, v, mask=(torch.rand(70, 2, generator=gen, device="cuda") < 0.5).t())


@pytest.mark.parametrize("t", TYPES)
def test_scores_of_any_size(t):
    q, k, v, _ = tensors(2, 40, 90, 2, 2, 64, t, sharp=30.0)        # one key takes nearly all
    check(q, k, v)
    check(q, k, v, scale=1e-3)
    q2, k2, v2, _ = tensors(2, 5, 300, 2, 2, 64, t, sharp=0.0)      # all equal
    check(q2, k2, v2)


def test_small_upstream_gradients_of_half_precision_do_not_vanish():
    q, k, v, gen = tensors(2, 40, 500, 4, 4, 64, torch.float16)
    up = (torch.randn(q.shape, generator=gen, device="cuda") * 2.0 ** -9).half()
    o = cross_attention(q, k, v)
    small = torch.autograd.grad(o, [q, k, v], up)
    o = cross_attention(q, k, v)
    large = torch.autograd.grad(o, [q, k, v], up * 2.0 ** 9)        # the same, 2^9 larger: the scale takes powers of two out
    for a, b in zip(small, large):
        assert float((a.double() * 2.0 ** 9 - b.double()).abs().max()) <= float(b.double().abs().max()) * 2.0 ** -10 + 2.0 ** -25 * 2 ** 9


@pytest.mark.parametrize("shape", [(32, 33, 70, 8, 8, 40), (16, 257, 33, 16, 8, 96), (64, 100, 130, 4, 4, 128), (32, 1030, 64, 1, 1, 32), (64, 2100, 40, 1, 1, 64)])
@pytest.mark.parametrize("t", TYPES)
def test_many_rows_of_many_heads(t, shape):
    q, k, v, gen = tensors(*shape, t)
    B, _, Lk = shape[:3]
    check(q, k, v, torch.randint(0, Lk + 1, (B,), generator=gen, device="cuda"), torch.rand(B, Lk, generator=gen, device="cuda") < 0.9)
    check(q, k, v)


@pytest.mark.parametrize("t", TYPES)
def test_scores_that_grow_and_fall_from_key_to_key(t):
    # the running maximum moves by less and by more than 2^8 between tiles, up and down, in some rows only
    B, Lq, Lk, H, Dh = 16, 130, 400, 16, 32
    q, k, v, gen = tensors(B, Lq, Lk, H, H, Dh, t)
    with torch.no_grad():
        slope = torch.linspace(-3.0, 3.0, Lk, device="cuda")[None, :, None, None]
        k.copy_((k.float() * slope.abs() + 0.4 * slope).to(t))
    check(q, k, v)
    check(q[:2].detach().requires_grad_(True), k[:2].detach().requires_grad_(True), v[:2].detach().requires_grad_(True))


@pytest.mark.parametrize("shape,lens", [((3, 700, 700, 4, 2, 64), [0, 1, 700]), ((2, 1100, 20, 2, 1, 96), [20, 3]), ((5, 600, 300, 3, 3, 128), [300, 129, 128, 127, 5]),
                                        ((4, 1000, 513, 2, 2, 32), [0, 0, 0, 0]), ((4, 1000, 513, 2, 2, 40), [0, 0, 0, 1]), ((2, 1500, 32, 1, 1, 128), [0, 32]),
                                        ((1, 3001, 400, 1, 1, 128), None), ((2, 1024, 30, 3, 1, 16), None)])
@pytest.mark.parametrize("t", TYPES)
def test_gradients_of_keys_shared_by_workgroups(t, shape, lens):
    q, k, v, gen = tensors(*shape, t)
    n = None if lens is None else torch.tensor(lens, device="cuda")
    check(q, k, v, n)
    check(q, k, v, n, torch.rand(shape[0], shape[2], generator=gen, device="cuda") < 0.8)


@pytest.mark.parametrize("worst", [float("nan"), float("inf")])
@pytest.mark.parametrize("Lq,Lk", [(5, 40), (5, 100), (40, 20), (40, 100)])
@pytest.mark.parametrize("t", TYPES)
def test_an_upstream_gradient_that_is_not_finite_reaches_what_it_touches(t, Lq, Lk, worst):
    q, k, v, _ = tensors(2, Lq, Lk, 2, 1, 32, t)
    mask = torch.ones(2, Lk, dtype=torch.bool, device="cuda")
    mask[:, 3] = False
    lens = torch.tensor([Lk - 2, Lk], device="cuda")
    up = torch.ones_like(q)
    up[0, 2, 1] = worst                                             # one query of one head of sample 0
    gq, gk, gv = torch.autograd.grad(cross_attention(q, k, v, lens, mask), [q, k, v], up)
    assert not torch.isfinite(gq[0, 2, 1]).any()
    assert torch.isfinite(gq[0, 2, 0]).all() and torch.isfinite(gq[0, :2]).all() and torch.isfinite(gq[0, 3:]).all()
    there = mask[0] & (torch.arange(Lk, device="cuda") < Lk - 2)
    assert not torch.isfinite(gk[0][there]).any() and not torch.isfinite(gv[0][there]).any()
    assert not gk[0][~there].any() and not gv[0][~there].any()
    assert all(torch.isfinite(x[1]).all() for x in (gq, gk, gv))


def test_gradients_against_differences():
    q, k, v, gen = tensors(2, 9, 40, 4, 2, 24, torch.float32, sharp=1.0)
    lens = torch.tensor([40, 23], device="cuda")
    w = torch.randn(q.shape, generator=gen, device="cuda")
    o = cross_attention(q, k, v, lens)
    size = float((o.detach().double() * w).abs().sum())
    grads = torch.autograd.grad(o, [q, k, v], w)
    for i, g in enumerate(grads):
        d = torch.randn(g.shape, generator=gen, device="cuda")

        def diff(h):
            out = []
            with torch.no_grad():
                for s in (1, -1):
                    x = [q, k, v]
                    x[i] = x[i] + s * h * d
                    out.append((cross_attention(*x, lens).double() * w).sum())
            return float(out[0] - out[1]) / (2 * h)

        wide, near, along = diff(2.0 ** -5), diff(2.0 ** -6), float((g.double() * d).sum())
        # a central difference's error falls fourfold with half the step; an output is off by less than 2^-18 of its size
        assert abs((4 * near - wide) / 3 - along) <= abs(wide - near) + size * 2.0 ** -18 * 2 ** 6


def test_only_the_wanted_gradients():
    q, k, v, _ = tensors(2, 9, 40, 4, 2, 32, torch.float32)
    up = torch.ones_like(q)
    all3 = torch.autograd.grad(cross_attention(q, k, v), [q, k, v], up)
    assert torch.equal(torch.autograd.grad(cross_attention(q, k.detach(), v.detach()), q, up)[0], all3[0])
    assert torch.equal(torch.autograd.grad(cross_attention(q.detach(), k, v.detach()), k, up)[0], all3[1])
    assert torch.equal(torch.autograd.grad(cross_attention(q.detach(), k.detach(), v), v, up)[0], all3[2])


def test_nothing_to_attend_to_and_nobody_to_attend():
    for B, Lq, Lk in ((2, 5, 0), (0, 5, 7), (2, 0, 7)):
        q, k, v, _ = tensors(B, Lq, Lk, 4, 2, 32, torch.bfloat16)
        o = cross_attention(q, k, v)
        assert o.shape == q.shape and (o == 0).all()
        for g, x in zip(torch.autograd.grad(o.sum(), [q, k, v]), (q, k, v)):
            assert g.shape == x.shape and (g == 0).all()


def test_offsets_beyond_32_bits():
    Lk = 70000                                                      # keys 65536 elements apart: the last lies 9 GB behind the first
    big = torch.zeros(Lk * 65536, device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = big.view(1, Lk, 1, 65536)
    k0, v0 = (torch.randn(1, Lk, 1, 64, generator=gen, device="cuda").bfloat16() for _ in range(2))
    wide[..., :64], wide[..., 64:128] = k0, v0
    q = torch.randn(1, 2, 1, 64, generator=gen, device="cuda").bfloat16()
    with torch.no_grad():
        assert torch.equal(cross_attention(q, wide[..., :64], wide[..., 64:128]), cross_attention(q, k0, v0))


def test_another_stream_and_a_captured_graph():
    q, k, v, gen = tensors(2, 12, 700, 4, 2, 64, torch.float16)
    lens = torch.tensor([700, 300], device="cuda")
    up = torch.randn(q.shape, generator=gen, device="cuda").half()

    def step():
        o = cross_attention(q, k, v, lens)
        return (o.detach(), *torch.autograd.grad(o, [q, k, v], up))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:                                                # two graphs in flight: each has workspaces of its own
        with torch.cuda.graph(g):
            held.append(step())
    for i in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=gen, device="cuda"))
        lens.copy_(torch.randint(0, 701, (2,), generator=gen, device="cuda"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for h in held:
            assert all(torch.equal(a, b) for a, b in zip(h, want))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_module_against_its_formula_and_word_by_word(dtype):
    torch.manual_seed(0)
    m = dv.CrossAttention(128, 4, state_dim=96, key_heads=2, dtype=dtype).cuda()
    x, s = torch.randn(3, 6, 128, device="cuda"), torch.randn(3, 50, 96, device="cuda")
    lens = torch.tensor([50, 20, 1], device="cuda")
    y = m(x, s, lens)
    y.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for n, p in m.named_parameters() if n != "key_value.bias")
    with torch.no_grad():
        kv = m.states(s)
        for l in range(6):                                          # an answer written word by word over keys made once
            one = m(x[:, l:l + 1], kv=kv, lens=lens)
            assert float((one - y[:, l:l + 1]).abs().max()) <= (1e-5 if dtype == "fp32" else 4e-2)
        W = lambda lin, z: z.double() @ lin.weight.double().t() + lin.bias.double()  # noqa: E731
        q, kvd = W(m.query, x).view(3, 6, 4, 32), W(m.key_value, s).view(3, 50, 2, 2, 32)
        k, v = kvd[:, :, 0].repeat_interleave(2, 2), kvd[:, :, 1].repeat_interleave(2, 2)
        sc = torch.einsum("blhd,bjhd->bhlj", q.cpu(), k.cpu()) / 32 ** 0.5
        sc = sc.masked_fill(torch.arange(50) >= lens.cpu().view(3, 1, 1, 1), -torch.inf)
        o = torch.einsum("bhlj,bjhd->blhd", sc.softmax(3), v.cpu()).reshape(3, 6, 128)
        want = o @ m.out.weight.double().cpu().t() + m.out.bias.double().cpu()
        assert float((y.cpu() - want).abs().max()) <= (1e-5 if dtype == "fp32" else 4e-2)


@pytest.mark.parametrize("B,Lq,Lk,H", [(2, 3, 40, 2), (2, 3, 500, 2), (1, 1, 5000, 2), (2, 200, 300, 2), (64, 300, 70, 4), (16, 40, 33, 16), (1, 3000, 20, 2)])
@pytest.mark.parametrize("t,size,scale", [(torch.float32, 1e5, 1.0), (torch.float32, 1e18, 1.0), (torch.float32, 2.0, 1e30), (torch.bfloat16, 1e6, 1.0),
                                          (torch.bfloat16, 3.0, 1e28), (torch.float16, 60000.0, 1.0), (torch.float16, 0.5, 1e20)])
def test_finite_scores_of_any_size(t, size, scale, B, Lq, Lk, H):
    # one number of each head carries the score: size^2 scale = 4e9 to 1e36 for the best key, at most 7/8 of it for the others
    Dh, gen = 32, torch.Generator(device="cuda").manual_seed(Lk)
    q, k = torch.zeros(B, Lq, H, Dh, device="cuda", dtype=t), torch.zeros(B, Lk, H, Dh, device="cuda", dtype=t)
    v = torch.randn(B, Lk, H, Dh, generator=gen, device="cuda").to(t)
    up = (torch.randn(B, Lq, H, Dh, generator=gen, device="cuda") * 2.0 ** -6).to(t)
    q[..., 3] = size
    k[..., 3] = (torch.linspace(-0.875, 0.875, Lk, device="cuda") * size).to(t)[None, :, None]
    best, twin = Lk // 3, Lk - 2
    k[:, best, :, 3] = size
    q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True)
    o = cross_attention(q, k, v, scale=scale)
    assert torch.equal(o, v[:, best:best + 1].expand(B, Lq, H, Dh))                      # all of the best key, to the bit
    gq, gk, gv = torch.autograd.grad(o, [q, k, v], up)
    want = up.double().sum(1)
    step = torch.finfo(t).eps / 2
    assert ((gv[:, best].double() - want).abs() <= want.abs() * step + Lq * 2.0 ** -24 * up.double().abs().sum(1)).all()
    gv[:, best] = 0
    assert (gv == 0).all()
    # p (dP - D) = 0 for the best key up to the rounding of two sums of Dh products, for every row of it; and 0 for the others
    err = (2 * Dh * 2.0 ** -24) * (up.double().abs() * v[:, best:best + 1].double().abs()).sum(3, keepdim=True)
    # (a bound beyond the type's largest number allows what such a number rounds to, an infinity: fp16 at scale 1e20, where the bound is
    # 1e20 x 0.5 x 2^-18 x sum |up v|, at least 1e10 while the sum is over 2^-14, and the largest number 65504)
    for got, bound in ((gq, scale * size * err * 1.01), (gk[:, best], scale * size * 1.01 * err.sum(1))):
        assert (got.double().abs() <= torch.where(bound > torch.finfo(t).max, torch.inf, bound)).all()
    gk[:, best] = 0
    assert (gk == 0).all()
    with torch.no_grad():                                           # two keys share the maximum
        k[:, twin, :, 3] = size
        o = cross_attention(q, k, v, scale=scale).double()
        want = (v[:, best:best + 1].double() + v[:, twin:twin + 1].double()) / 2
        assert ((o - want).abs() <= want.abs() * step + 2.0 ** -22).all()


@pytest.mark.parametrize("B,Lq,Lk,H,Hk", [(2, 6, 40, 2, 2), (2, 5, 300, 4, 2), (2, 70, 20, 2, 1), (2, 70, 300, 2, 2), (64, 300, 70, 4, 4)])
def test_large_values_of_half_precision_do_not_hold_the_gradient_back(B, Lq, Lk, H, Hk):
    # values near the type's largest, flat upstream gradients: differences of dO V^T of 2^19 largest |dO|, where a scaled score gradient of p = 1/2
    # is beyond the type; the queries are small, so that the gradients themselves are not
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = (torch.randn(B, Lq, H, 128, generator=gen, device="cuda") * 2.0 ** -4).half()
    k = (torch.randn(B, Lk, Hk, 128, generator=gen, device="cuda") * 2.0 ** -4).half()
    sign = torch.where(torch.rand(128, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    v = torch.randn(B, Lk, Hk, 128, generator=gen, device="cuda")
    q[..., 0], k[..., 0] = 16.0, 0.0
    for j in (1, Lk - 2):                                           # two keys share each row, with opposite values
        k[:, j, :, 0] = 16.0
        v[:, j] = 60000.0 * sign * (1 if j == 1 else -1)
    up = (torch.ones(B, Lq, H, 128, device="cuda") * sign * 2.0 ** -12).half()
    up[:, ::2] = -up[:, ::2]
    check(q.requires_grad_(True), k.requires_grad_(True), v.half().requires_grad_(True), up=up)


@pytest.mark.parametrize("shape", [(2, 20, 60, 4, 2, 64), (2, 15, 500, 4, 4, 96), (1, 1, 3000, 8, 2, 64), (2, 200, 330, 2, 1, 128), (64, 140, 70, 4, 4, 32), (1, 1500, 30, 1, 1, 64)])
@pytest.mark.parametrize("t", TYPES)
def test_rows_with_scores_of_very_different_size_side_by_side(t, shape):
    # some rows of a tile are beyond what is taken off with the scaling, some are not, and keys grow so that a row passes from one to the other
    q, k, v, gen = tensors(*shape, t, sharp=1.0)
    size = torch.tensor([1.0, 40.0, 1.0, 3000.0, 200.0], device="cuda")
    with torch.no_grad():
        q.mul_(size[torch.arange(shape[1], device="cuda") % 5].to(t)[None, :, None, None])
        k.mul_(torch.linspace(0.01, 8.0, shape[2], device="cuda").to(t)[None, :, None, None])
    check(q, k, v)
    lens = torch.randint(1, shape[2] + 1, (shape[0],), generator=gen, device="cuda")
    check(q, k, v, lens, torch.rand(shape[0], shape[2], generator=gen, device="cuda") < 0.8)
