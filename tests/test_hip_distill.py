"""GPU: distillation from a teacher's top logits (include/dvgr_head.h, losses.distillation_loss) against 64 bits.

Tolerances, from fp32 arithmetic (u = 2^-24): a logit's distance from its row's maximum, in powers of two, is off by at most
(2 L + 8) u with L the largest distance; the sum over the classes by (C / 256 + 16) u relative.  p and q are off by both, relative; the
loss by T^2 times the errors of its two logarithms and of p; the gradient by its parts' errors, then half a step of its type."""
import pytest
import torch

import dualvgr_videoqa_amd as dv

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def reference(z, v, idx, T):
    z, v, C = z.double() / T, v.double() / T, z.shape[1]
    there = (idx >= 0) & (idx < C)
    v = torch.where(there, v, -torch.inf)
    some = (v > -torch.inf).any(1, keepdim=True)
    logp = torch.where(some, torch.log_softmax(torch.where(some, v, 0.0), 1), -torch.inf)
    p = torch.where(there & some, logp.exp(), 0.0)
    logq = torch.log_softmax(z, 1)
    at = idx.clamp(0, C - 1)
    lq = logq.gather(1, at)
    rows = torch.where(p > 0, p * (logp - lq), 0.0).sum(1) * T * T
    spread = torch.where(p > 0, p * ((logp - lq).abs() + 1), 0.0).sum(1)
    q = torch.where(some, logq.exp(), 0.0)
    full = torch.zeros_like(q).scatter_add_(1, at, p)
    L = float((z.max(1, keepdim=True).values - z)[torch.isfinite(z)].max()) + float((v.max() - v[torch.isfinite(v)].min()) if bool(some.any()) else 0)
    e = ((2 * L * 1.4427 + 8) * 2 + C / 256 + 16) * U
    return rows, T * T * spread * 2 * e, T * (q - full), T * (q + full) * 2 * e, some.squeeze(1)


def check(z, v, idx, T, reduction="mean", up=None):
    rows, rows_tol, grad, grad_tol, some = reference(z.detach(), v, idx, T)
    n = max(1, int(some.sum()))
    loss = dv.distillation_loss(z, v, idx, T, reduction)
    up = torch.ones((), device="cuda") if up is None else up
    if reduction == "none":
        up = up.expand(rows.shape) if up.dim() == 0 else up
        want, tol, w = rows, rows_tol, up.double()[:, None]
    else:
        w = up.double() / (n if reduction == "mean" else 1)
        f = 1 / n if reduction == "mean" else 1.0
        want, tol = rows.sum() * f, rows_tol.sum() * f + rows.abs().sum() * f * 4 * U
    assert loss.dtype == torch.float32
    assert ((loss.double() - want).abs() <= tol + want.abs() * 2 * U).all(), (loss, want, tol)
    g, = torch.autograd.grad(loss, z, up.float())
    assert g.dtype == z.dtype and g.shape == z.shape
    want = grad * w
    tol = grad_tol * w.abs() + want.abs() * (torch.finfo(z.dtype).eps / 2 + 4 * U) + torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps / 2
    worst = ((g.double() - want).abs() - tol).max()
    assert float(worst) <= 0, float(worst)
    with torch.no_grad():
        assert torch.equal(dv.distillation_loss(z, v, idx, T, reduction), loss)
    return loss, g


def case(R, C, K, t, seed, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(R, C, generator=gen, device="cuda") * spread
    v, idx = (z + torch.randn(R, C, generator=gen, device="cuda")).topk(K, 1)
    return z.to(t).requires_grad_(True), v, idx


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("R,C,K,T", [(1, 1, 1, 1.0), (3, 2, 2, 4.0), (64, 1000, 10, 2.0), (5, 1023, 1000, 1.0), (7, 4099, 129, 0.5),
                                     (2, 70001, 50, 2.0), (1, 131072, 1024, 3.0), (1500, 33, 5, 1.0), (130, 8193, 1, 2.0)])
def test_loss_and_gradient(t, R, C, K, T):
    z, v, idx = case(R, C, K, t, R + C)
    scale = torch.tensor(1024.0 if t == torch.float16 else 1.0, device="cuda")
    for reduction in ("mean", "sum", "none"):
        a = check(z, v.to(t), idx, T, reduction, scale)
    b = check(z, v.to(t), idx, T, "none", scale)
    assert all(torch.equal(x, y) for x, y in zip(a, b))             # the same inputs, the same bits


def test_rows_of_the_teacher_in_another_type_and_upstream_by_row():
    z, v, idx = case(33, 500, 20, torch.bfloat16, 3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    check(z, v, idx.int().long(), 2.0, "none", torch.randn(33, generator=gen, device="cuda"))
    assert torch.equal(dv.distillation_loss(z, v, idx.int(), 2.0), dv.distillation_loss(z, v, idx, 2.0))


@pytest.mark.parametrize("R,C", [(9, 300), (3, 40000)])
def test_ragged_lists_repeated_classes_and_rows_without_entries(R, C):
    z, v, idx = case(R, C, 12, torch.float32, 5)
    idx[0, 3:] = -1                                                 # a short list
    idx[1, :] = -1                                                  # none
    idx[2, 4:8] = idx[2, 4]                                         # the same class four times
    v[2, 9] = -torch.inf                                            # listed with probability 0
    idx[2, 10], v[2, 10] = C, torch.nan                             # outside the classes: never looked at
    v[0, 5] = torch.nan
    for reduction in ("mean", "sum", "none"):
        loss, g = check(z, v, idx, 2.0, reduction)
        assert (g[1] == 0).all()
    rows = dv.distillation_loss(z, v, idx, 2.0, "none")
    assert float(rows[1].detach()) == 0.0
    idx.fill_(-1)
    for reduction in ("mean", "sum"):
        loss = dv.distillation_loss(z, v, idx, 2.0, reduction)
        assert float(loss.detach()) == 0.0 and (torch.autograd.grad(loss, z)[0] == 0).all()


def test_classes_the_student_excludes():
    z, v, idx = case(4, 900, 8, torch.float32, 6)
    with torch.no_grad():
        z[:, 100:200] = -torch.inf                                  # q = 0 there
    idx[:, 0], v[:, 0] = 150, -torch.inf                            # listed, but with p = 0: adds nothing
    keep = (idx < 100) | (idx >= 200)
    idx[:, 1:] = torch.where(keep[:, 1:], idx[:, 1:], -1)
    _, g = check(z, v, idx, 1.0)
    assert (g[:, 100:200] == 0).all()
    idx[0, 1], v[0, 1] = 150, 5.0
    rows = dv.distillation_loss(z, v, idx, 1.0, "none").detach()
    assert float(rows[0]) == float("inf") and torch.isfinite(rows[1:]).all()


def test_not_a_number_is_passed_on():
    z, v, idx = case(3, 50, 1, torch.float32, 7)
    v[1, 0] = torch.nan
    rows = dv.distillation_loss(z, v, idx, 1.0, "none").detach()
    assert torch.isnan(rows[1]) and torch.isfinite(rows[0]) and torch.isfinite(rows[2])


def test_strided_logits_and_leading_dimensions():
    z, v, idx = case(12, 1000, 6, torch.bfloat16, 8)
    want, gw = check(z, v, idx, 2.0)
    # rows at another alignment give their elements to other threads, so sums run in another order: held to the bounds, not to the bits
    wide = torch.zeros(12, 1004, device="cuda", dtype=torch.bfloat16)
    wide[:, :1000] = z.detach()
    check(wide[:, :1000].requires_grad_(True), v, idx, 2.0)
    wide.requires_grad_(True)
    g, = torch.autograd.grad(dv.distillation_loss(wide[:, :1000], v, idx, 2.0), wide)
    assert (g[:, 1000:] == 0).all() and (g[:, :1000] != 0).any()
    odd = torch.zeros(12 * 1001 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(12, 1001)[:, :1000]
    odd.copy_(z.detach())
    check(odd.requires_grad_(True), v, idx, 2.0)
    three = z.detach().view(3, 4, 1000).requires_grad_(True)
    rows = dv.distillation_loss(three, v.view(3, 4, 6), idx.view(3, 4, 6), 2.0, "none")
    assert rows.shape == (3, 4) and torch.equal(rows.view(-1), dv.distillation_loss(z, v, idx, 2.0, "none"))
    last = z.detach().t().contiguous().t().requires_grad_(True)     # classes not along the last stride
    assert torch.equal(dv.distillation_loss(last, v, idx, 2.0), want)


def test_a_single_row_that_is_a_column_of_another_tensor():
    x = torch.randn(37, 1, generator=torch.Generator().manual_seed(8)).cuda().requires_grad_(True)
    z = x.t()                                                       # (1, 37), its one row's stride is 1
    assert z.stride() == (1, 1)
    v, idx = torch.randn(1, 3, generator=torch.Generator().manual_seed(9)).cuda(), torch.tensor([[4, 0, 36]], device="cuda")
    dv.distillation_loss(z, v, idx, 1.5).backward()
    y = x.detach().t().clone().requires_grad_(True)
    dv.distillation_loss(y, v, idx, 1.5).backward()
    assert torch.equal(x.grad.t(), y.grad)


def test_gradient_against_differences():
    z, v, idx = case(6, 77, 9, torch.float32, 9)
    gen = torch.Generator(device="cuda").manual_seed(10)
    d = torch.randn(6, 77, generator=gen, device="cuda")
    loss = dv.distillation_loss(z, v, idx, 1.5, "sum")
    g, = torch.autograd.grad(loss, z)
    along = float((g.double() * d).sum())

    def diff(h):
        with torch.no_grad():
            a, b = (dv.distillation_loss(z + s * h * d, v, idx, 1.5, "none").double().sum() for s in (1, -1))
        return float(a - b) / (2 * h)

    wide, near = diff(2.0 ** -4), diff(2.0 ** -5)
    # the error of a central difference falls fourfold with half the step; the rows are off by a few 2^-22 of their size each
    assert abs((4 * near - wide) / 3 - along) <= abs(wide - near) + 2.0 ** -22 * 16 * 6 * float(loss.detach()) * 2 ** 5


def test_empty_batch():
    z = torch.empty(0, 10, device="cuda", requires_grad=True)
    v, idx = torch.empty(0, 3, device="cuda"), torch.empty(0, 3, device="cuda", dtype=torch.int64)
    loss = dv.distillation_loss(z, v, idx)
    assert float(loss.detach()) == 0.0 and torch.autograd.grad(loss, z)[0].shape == (0, 10)
    assert dv.distillation_loss(z, v, idx, reduction="none").shape == (0,)


def test_another_stream_and_a_captured_graph():
    z, v, idx = case(40, 9000, 30, torch.bfloat16, 11)

    def step():
        loss = dv.distillation_loss(z, v, idx, 2.0)
        return loss.detach(), torch.autograd.grad(loss, z)[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    gen = torch.Generator(device="cuda").manual_seed(12)
    for k in range(3):
        with torch.no_grad():
            z.copy_(torch.randn(40, 9000, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


@pytest.mark.parametrize("C", [700, 40000])                         # a row in one workgroup, in shares
@pytest.mark.parametrize("t,base,T", [(torch.float32, 3e9, 1.0), (torch.float32, 1e10, 1.0), (torch.float32, -1e10, 1.0), (torch.float32, 3e38, 2.0),
                                      (torch.float32, -3e38, 1.0), (torch.float32, 5000.0, 1e-6), (torch.bfloat16, 1e12, 1.0), (torch.bfloat16, 30000.0, 1e-6),
                                      (torch.float16, 60000.0, 1e-6), (torch.float16, -4000.0, 1e-6)])
def test_finite_logits_of_any_size(t, base, T, C):
    # two classes share the maximum, everything else is thousands of exponents below it: q = 1/2, 1/2, 0, .. to the last bit
    z = torch.full((3, C), base, device="cuda", dtype=t)
    step = 2.0 ** -3 * abs(base)
    z -= torch.linspace(0.5, 1.0, C, device="cuda").to(t) * torch.tensor(step, device="cuda").to(t)
    assert torch.isfinite(z).all()
    z[:, 5], z[:, C - 7] = base, base
    z.requires_grad_(True)
    idx = torch.tensor([[5, 9], [C - 7, 5], [5, -1]], device="cuda")
    v = torch.full((3, 2), base, device="cuda", dtype=t)
    v[0, 1] = torch.tensor(base - step, device="cuda").to(t)        # p = (1, 0); (1/2, 1/2); (1)
    rows = dv.distillation_loss(z, v, idx, T, "none")
    ln2 = 0.6931471805599453
    want = torch.tensor([ln2, 0.0, ln2], device="cuda", dtype=torch.float64) * T * T
    assert ((rows.double() - want).abs() <= 2.0 ** -20 * T * T).all(), rows
    up = 1.0 / T                                                    # (the gradient's factor is T: fp16 would lose 1e-6)
    g, = torch.autograd.grad(rows, z, torch.full_like(rows, up))
    want = torch.zeros(3, C, device="cuda", dtype=torch.float64)
    want[0, 5], want[0, C - 7], want[2, 5], want[2, C - 7] = -0.5, 0.5, -0.5, 0.5
    assert ((g.double() - want).abs() <= 2.0 ** -10).all()
