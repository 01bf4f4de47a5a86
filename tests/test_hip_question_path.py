"""GPU: the question-side operators as a program uses them -- together, in the training step, and where they refuse."""
import pytest
import torch
import torch.nn as nn

import dualvgr_videoqa_amd as dv
from dualvgr_videoqa_amd import synth
from test_hip_model import model_inputs

pytestmark = pytest.mark.gpu


class Reader(nn.Module):
    """words -> embedding -> attention to the video's frames -> answers"""

    def __init__(self, words, answers, dim, frames_dim):
        super().__init__()
        self.embed = dv.TokenEmbedding(words, dim, padding_idx=0, scale=dim ** 0.5)
        self.attend = dv.CrossAttention(dim, 4, state_dim=frames_dim, key_heads=2)
        self.answer = dv.HipLinear(dim, answers)

    def forward(self, tokens, frames, lens):
        x = self.embed(tokens)
        return self.answer((x + self.attend(x, frames, lens)).mean(1))


def plain(sd, tokens, frames, lens, values, indices, T, dim):
    """the same program in 64 bits on the CPU: (loss, gradients)"""
    p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in sd.items()}
    x = p["embed.weight"][tokens] * dim ** 0.5
    lin = lambda n, z: z @ p[n + ".weight"].t() + p[n + ".bias"]  # noqa: E731
    B, L, _ = x.shape
    q = lin("attend.query", x).view(B, L, 4, dim // 4)
    kv = lin("attend.key_value", frames.double()).view(B, -1, 2, 2, dim // 4)
    k, v = kv[:, :, 0].repeat_interleave(2, 2), kv[:, :, 1].repeat_interleave(2, 2)
    s = torch.einsum("blhd,bjhd->bhlj", q, k) * (dim // 4) ** -0.5
    s = s.masked_fill(torch.arange(k.shape[1]) >= lens.view(-1, 1, 1, 1), -torch.inf)
    o = torch.einsum("bhlj,bjhd->blhd", s.softmax(3), v).reshape(B, L, dim)
    z = lin("answer", (x + lin("attend.out", o)).mean(1))
    logp, logq = torch.log_softmax(values.double() / T, 1), torch.log_softmax(z / T, 1).gather(1, indices)
    loss = (logp.exp() * (logp - logq)).sum(1).mean() * T * T
    loss.backward()
    grads = {k: t.grad for k, t in p.items()}
    grads["embed.weight"][0] = 0
    return float(loss.detach()), grads


def test_embedding_attention_and_distillation_together():
    torch.manual_seed(3)
    dim, B, L, F = 64, 6, 7, 90
    m = Reader(50, 40, dim, 48).cuda()
    g = torch.Generator().manual_seed(4)
    tokens, frames = torch.randint(0, 50, (B, L), generator=g), torch.randn(B, F, 48, generator=g)
    lens = torch.tensor([90, 1, 33, 64, 65, 17])
    values, indices = torch.randn(B, 40, generator=g).topk(5, 1)
    args = tokens.cuda(), frames.cuda(), lens.cuda()
    loss = dv.distillation_loss(m(*args), values.cuda(), indices.cuda(), 2.0)
    loss.backward()
    want, grads = plain(m.state_dict(), tokens, frames, lens, values, indices, 2.0, dim)
    # fp32 throughout: chains of dot products of up to 128 terms, a few 2^-24 of their size each
    assert abs(float(loss.detach()) - want) <= 2e-5 * abs(want)
    for n, p in m.named_parameters():
        off = (p.grad.cpu().double() - grads[n]).abs().max()
        assert float(off) <= 5e-5 * float(grads[n].abs().max()) + (1e-7 if n == "attend.key_value.bias" else 0), (n, float(off))
    again = {n: p.grad.clone() for n, p in m.named_parameters()}
    m.zero_grad()
    dv.distillation_loss(m(*args), values.cuda(), indices.cuda(), 2.0).backward()
    assert torch.equal(m.embed.weight.grad, again["embed.weight"])
    m.embed.check_tokens()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())


def test_one_pass_of_gradient_steps_runs():
    torch.manual_seed(5)
    m = Reader(30, 20, 64, 48).cuda()
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    values, indices = torch.randn(8, 20, device="cuda").topk(4, 1)
    for i in range(3):
        opt.zero_grad()
        z = m(torch.randint(0, 30, (8, 5), device="cuda"), torch.randn(8, 40, 48, device="cuda"), torch.randint(1, 41, (8,), device="cuda"))
        dv.distillation_loss(z, values, indices).backward()
        opt.step()
    assert all(torch.isfinite(p).all() for p in m.parameters())


def small_step(weight, teacher_on, lr=0.0, keep=False):
    V, D, Wd, N, Fr, Lr, B, T, vq, va = 64, 64, 32, 5, 3, 2, 8, 6, 40, 10
    vocab = {"question_token_to_idx": {str(i): i for i in range(vq)}, "answer_token_to_idx": {str(i): i for i in range(va)}}
    torch.manual_seed(11)
    m = dv.DualVGR(vision_dim=V, module_dim=D, word_dim=Wd, vocab=vocab, num_of_nodes=N, graph_module="GAT", graph_layers=1, unit_layers=Lr, dtype="fp32")
    m = m.cuda().train().set_dropout_enabled(False)
    app, mot, q, qlen = [torch.from_numpy(x).cuda() for x in model_inputs(B, N, Fr, V, T, vq, 5)]
    answers = torch.arange(B).cuda() % va
    g = torch.Generator().manual_seed(6)
    values, indices = torch.randn(B, va, generator=g).topk(4, 1)
    indices[2] = -1                                                 # a pair the teacher says nothing about
    teacher = (values.cuda(), indices.cuda())
    step = dv.TrainStep(m, lr=lr, max_norm=1e9, distill_weight=weight, distill_temperature=2.0)
    out = step(app, mot, q, qlen, answers, teacher=teacher if teacher_on else None)
    grads = {n: p.grad.clone() for n, p in step.other}
    first = out, grads, step.unit.last_flat_grad.clone(), teacher
    return first + (step, (app, mot, q, qlen, answers)) if keep else first


def test_a_teacher_in_the_training_step():
    base, g0, u0, _ = small_step(0.0, False)
    assert "distill" not in base
    one, g1, u1, teacher = small_step(0.5, True)
    two, g2, u2, _ = small_step(1.0, True)
    z = one["logits"].detach().requires_grad_(True)
    kd = dv.distillation_loss(z, *teacher, 2.0)
    gz, = torch.autograd.grad(kd, z)
    assert torch.equal(one["distill"], kd.detach())
    # the cross entropy adds its 8 terms atomically: each of 8 roundings is half a step of at most the sum, in either run
    assert abs(float(one["ce"] - base["ce"])) <= 2 * 8 * 2.0 ** -24 * float(base["ce"])
    assert abs(float(one["loss"] - base["loss"]) - 0.5 * float(kd.detach())) <= 1e-6 * float(one["loss"])
    # the last bias sees the logits' gradient alone: the sum over the 8 pairs of (q - p) / 8, whose q moves by no more than the logits do
    # from run to run (the step adds atomically; the forward's own gate is 1e-4 of their size)
    bias = [n for n in g0 if n.endswith("classifier.5.bias")][0]
    noise = 1e-4 * float(z.detach().abs().max())
    for w, g in ((0.5, g1), (1.0, g2)):
        assert float(((g[bias] - g0[bias]) - w * gz.sum(0)).abs().max()) <= noise
    assert float(gz.sum(0).abs().max()) > 20 * noise
    assert float((u2 - u0).abs().max()) > 0
    with pytest.raises(ValueError):
        small_step(0.0, True)
    with pytest.raises(ValueError):
        small_step(0.5, False)


def test_the_weight_of_the_teacher_may_move_between_steps():
    _, _, _, teacher, step, batch = small_step(0.5, True, keep=True)
    bias = [n for n, _ in step.other if n.endswith("classifier.5.bias")][0]
    seen = {}
    for w in (0.5, 4.0):
        step.distill_weight = w
        out = step(*batch, teacher=teacher)
        seen[w] = dict(step.other)[bias].grad.clone()
    z = out["logits"].detach().requires_grad_(True)
    gz, = torch.autograd.grad(dv.distillation_loss(z, *teacher, 2.0), z)
    # (lr = 0: the logits are those of the first step up to its atomics, 1e-4 of their size as above)
    assert float((seen[4.0] - seen[0.5] - 3.5 * gz.sum(0)).abs().max()) <= 1e-4 * float(z.detach().abs().max())


def test_refusals_on_the_device():
    t = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    ids = t(3, dtype=torch.int64)
    for bad, args in (("takes fp32", (t(4, 8, dtype=torch.float64), ids)), ("integers", (t(4, 8), t(3))), ("integers", (t(4, 8), t(3, dtype=torch.bool))),
                      ("vocab, wd", (t(4), ids)), ("vocab, wd", (t(0, 8), ids)), ("tokens are on", (t(4, 8), ids.cpu()))):
        with pytest.raises(RuntimeError, match=bad):
            dv.embed_tokens(*args)
    for p in (4, -5):
        with pytest.raises(RuntimeError, match="padding_idx"):
            dv.embed_tokens(t(4, 8), ids, padding_idx=p)
    with pytest.raises(RuntimeError, match="one int32"):
        dv.embed_tokens(t(4, 8), ids, bad=t(1))

    z, v, i = t(2, 9), t(2, 3), t(2, 3, dtype=torch.int64)
    for bad, args in (("takes fp32", (z.double(), v, i)), ("logits \\(", (z, v, i[:1])), ("logits \\(", (z, v[:1], i[:1])), ("int64 or int32", (z, v, v)),
                      ("one device", (z, v, i.cpu())), ("entries a row", (z, t(2, 0), t(2, 0, dtype=torch.int64))),
                      ("entries a row", (t(2, 2000), t(2, 1025), t(2, 1025, dtype=torch.int64))), ("temperature", (z, v, i, 0.0)),
                      ("temperature", (z, v, i, float("nan"))), ("reduction", (z, v, i, 1.0, "batchmean"))):
        with pytest.raises(RuntimeError, match=bad):
            dv.distillation_loss(*args)

    q, k = t(2, 3, 4, 16), t(2, 5, 2, 16)
    for bad, args in (("takes fp32", (q.double(), k.double(), k.double())), ("one type", (q, k.half(), k.half())), ("one device", (q, k.cpu(), k)),
                      ("q \\(B", (q[0], k, k)), ("q \\(B", (q, k, k[:, :4])), ("q \\(B", (q[:1], k, k)), ("multiple of the key heads", (q[:, :, :3], k, k)),
                      ("head size", (t(2, 3, 4, 12), t(2, 5, 2, 12), t(2, 5, 2, 12))), ("head size", (t(2, 3, 4, 136), t(2, 5, 2, 136), t(2, 5, 2, 136))),
                      ("lens", (q, k, k, t(3, dtype=torch.int64))), ("lens", (q, k, k, t(2))), ("lens", (q, k, k, torch.zeros(2, dtype=torch.int64))),
                      ("mask", (q, k, k, None, t(2, 5))), ("mask", (q, k, k, None, t(2, 4, dtype=torch.bool))), ("scale", (q, k, k, None, None, 0.0)),
                      ("scale", (q, k, k, None, None, -1.0)), ("scale", (q, k, k, None, None, float("inf")))):
        with pytest.raises(RuntimeError, match=bad):
            dv.cross_attention(*args)
    with pytest.raises(RuntimeError, match="states or the keys"):
        dv.CrossAttention(64, 2).cuda()(t(1, 4, 64))


def test_a_gradient_says_when_it_is_differentiated_again():
    table = torch.randn(5, 8, device="cuda", requires_grad=True)
    up = torch.randn(3, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(dv.embed_tokens(table, torch.arange(3, device="cuda")), table, up, create_graph=True)
    assert torch.equal(g.detach()[:3], up.detach())
    with pytest.raises(RuntimeError, match="differentiated again"):
        g.sum().backward()
    z = torch.randn(2, 9, device="cuda", requires_grad=True)
    loss = dv.distillation_loss(z, torch.randn(2, 3, device="cuda"), torch.zeros(2, 3, device="cuda", dtype=torch.int64))
    loss.backward(retain_graph=True)
    first = z.grad.clone()
    loss.backward()                                                 # twice over one graph: the gradients add up
    assert torch.equal(z.grad, 2 * first)
    with pytest.raises(RuntimeError):
        loss.backward()                                             # its tensors are gone
    q = torch.randn(1, 2, 1, 8, device="cuda", requires_grad=True)
    o = dv.cross_attention(q, q.detach(), q.detach())
    with torch.no_grad():
        q.add_(1.0)                                                 # what the backward needs is not what it was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


@pytest.mark.parametrize("which", ["distil", "attend"])
def test_captured_backwards_refuse_while_an_eager_graph_of_a_leaf_lives(which):
    x = torch.randn(2, 6, 1, 16, device="cuda", requires_grad=True)
    v, i = torch.randn(2, 3, device="cuda"), torch.zeros(2, 3, device="cuda", dtype=torch.int64)
    z = torch.randn(2, 16, device="cuda", requires_grad=True)
    call = (lambda: dv.distillation_loss(z, v, i)) if which == "distil" else (lambda: dv.cross_attention(x, x, x).sum())
    leaf = z if which == "distil" else x
    alive = dv.distillation_loss(z, v, i) if which == "distil" else dv.cross_attention(x, x, x)
    up = torch.ones((), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
        with pytest.raises(RuntimeError, match="captured while"):
            torch.autograd.grad(out, leaf, up)
        del out
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g, = torch.autograd.grad(call(), leaf, up)
    want, = torch.autograd.grad(call(), leaf, up)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(g, want)


def test_two_streams_at_once():
    gen = torch.Generator(device="cuda").manual_seed(8)
    q = torch.randn(4, 40, 4, 64, generator=gen, device="cuda").bfloat16().requires_grad_(True)
    kv = torch.randn(4, 900, 4, 64, generator=gen, device="cuda").bfloat16()
    table = torch.randn(9000, 64, generator=gen, device="cuda", requires_grad=True)
    tokens = torch.randint(0, 9000, (9000,), generator=gen, device="cuda")
    up = torch.randn(9000, 64, generator=gen, device="cuda")

    def work():
        o = dv.cross_attention(q, kv, kv)
        return [o.detach(), *torch.autograd.grad(o, q, torch.ones_like(o)), *torch.autograd.grad(dv.embed_tokens(table, tokens), table, up)]

    want = work()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_two_byte_embeddings_feed_the_attention_module(t, dtype):
    torch.manual_seed(9)
    embed, attend = dv.TokenEmbedding(40, 64, scale=8.0).cuda().to(t), dv.CrossAttention(64, 2, state_dim=48, dtype=dtype).cuda()
    tokens = torch.randint(0, 40, (3, 5), device="cuda")
    frames = torch.randn(3, 20, 48, device="cuda").to(t).requires_grad_(True)
    words = embed(tokens)
    words.retain_grad()
    y = attend(words, frames)
    assert words.dtype == t and y.dtype == torch.float32
    y.square().sum().backward()
    wide, states = words.detach().float().requires_grad_(True), frames.detach().float().requires_grad_(True)
    z = attend(wide, states)                                        # the same numbers in fp32
    assert torch.equal(y, z)
    z.square().sum().backward()
    # nothing differs but the one rounding to the input's type (half a step, and half the smallest number)
    for got, want in ((words.grad, wide.grad), (frames.grad, states.grad)):
        assert got.dtype == t
        assert ((got.double() - want.double()).abs() <= want.double().abs() * torch.finfo(t).eps / 2 + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2).all()
    assert embed.weight.grad.dtype == t and torch.isfinite(embed.weight.grad).all()


@pytest.mark.parametrize("dtype,tol", [("fp32", 2e-6), ("bf16x3", 2e-5)])
@pytest.mark.parametrize("rows", [1, 2, 3, 4])
def test_projections_of_a_few_words_have_gradients(dtype, tol, rows):
    # (the bounds of the same products at other sizes: fp32 sums of up to 64 terms, operands split into two bf16 halves)
    torch.manual_seed(10)
    lin = dv.HipLinear(64, 24, dtype=dtype).cuda()
    x, up = torch.randn(rows, 64, device="cuda", requires_grad=True), torch.randn(rows, 24, device="cuda")
    grads = torch.autograd.grad(lin(x), [x, lin.weight, lin.bias], up)
    u, w, z = up.double(), lin.weight.detach().double(), x.detach().double()
    for got, want in zip(grads, (u @ w, u.t() @ z, u.sum(0))):
        assert got.shape == want.shape and float((got - want).abs().max()) <= tol * float(want.abs().max())


def test_an_answer_of_one_word_is_trained():
    torch.manual_seed(11)
    attend = dv.CrossAttention(64, 2, key_heads=1, state_dim=48).cuda()
    x, s = torch.randn(1, 1, 64, device="cuda", requires_grad=True), torch.randn(1, 2, 48, device="cuda", requires_grad=True)
    up = torch.randn(1, 1, 64, device="cuda")
    grads = torch.autograd.grad(attend(x, s), [x, s, *attend.parameters()], up)
    p = {n: t.detach().cpu().double().requires_grad_(True) for n, t in attend.named_parameters()}
    y, z = x.detach().cpu().double().requires_grad_(True), s.detach().cpu().double().requires_grad_(True)
    lin = lambda n, t: t @ p[n + ".weight"].t() + p[n + ".bias"]  # noqa: E731
    q, kv = lin("query", y).view(2, 32), lin("key_value", z).view(2, 2, 32)
    o = torch.softmax(q @ kv[:, 0].t() * 32 ** -0.5, 1) @ kv[:, 1]
    want = torch.autograd.grad(lin("out", o.reshape(1, 1, 64)), [y, z, *p.values()], up.cpu().double())
    # fp32 throughout: chains of dot products of up to 64 terms, a few 2^-24 of their size each (the keys' bias has no gradient: a sum that cancels)
    for got, w in zip(grads, want):
        assert float((got.cpu().double() - w).abs().max()) <= 5e-5 * float(w.abs().max()) + 1e-7


def test_the_whole_path_captured_and_replayed_between_eager_work():
    torch.manual_seed(12)
    m = Reader(50, 40, 64, 48).cuda()
    gen = torch.Generator(device="cuda").manual_seed(13)
    B, L, F = 16, 9, 70
    tokens, frames = torch.randint(0, 50, (B, L), generator=gen, device="cuda"), torch.randn(B, F, 48, generator=gen, device="cuda")
    lens = torch.randint(1, F + 1, (B,), generator=gen, device="cuda")
    values, indices = torch.randn(B, 40, generator=gen, device="cuda").topk(5, 1)
    names = [n for n, _ in m.named_parameters()]

    def step():
        loss = dv.distillation_loss(m(tokens, frames, lens), values, indices, 2.0)
        return [loss.detach(), *torch.autograd.grad(loss, list(m.parameters()))]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(5):
        tokens.copy_(torch.randint(0, 50, (B, L), generator=gen, device="cuda"))
        frames.copy_(torch.randn(B, F, 48, generator=gen, device="cuda"))
        lens.copy_(torch.randint(1, F + 1, (B,), generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        # what the projections add atomically (their biases' sums over 16 shares of up to B F rows) may differ in its last bits
        for n, a, b in zip(["loss", *names], held, want):
            assert float((a - b).abs().max()) <= 2e-5 * float(b.abs().max()) + 1e-7, (i, n)


def test_which_graphs_a_captured_backward_may_not_run_into():
    # nothing is run backward here: the look at the nodes alone, from eager code and from inside a capture
    refuses = dv._lib.torch_ops().dbg_refuses_capture
    x, z = torch.randn(2, 6, 1, 16, device="cuda", requires_grad=True), torch.randn(2, 3, 16, device="cuda", requires_grad=True)
    assert refuses(x.view(2, 96)) and refuses(z.transpose(1, 2).contiguous())              # eager, on the null stream
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        w = torch.randn(3, device="cuda", requires_grad=True)
        assert not refuses(w.exp())                                 # eager, on another stream: it joins the capture and leaves it again
    graph = torch.cuda.CUDAGraph()
    alive = x.view(2, 96)
    with torch.cuda.graph(graph):
        y, u = x.reshape(-1, 16).float() * 2, z.view(6, 16) * 2
        seen = refuses(y), refuses(u)
    assert seen == (True, False)                                    # x has a graph outside, z has none
    del alive, y, u
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x.reshape(-1, 16).float() * 2
        seen = refuses(y)
    assert not seen


@pytest.mark.parametrize("which", ["logits of three dimensions", "logits along the other stride", "keys and values of one tensor", "projections"])
def test_captured_backwards_refuse_a_leaf_behind_views_and_copies(which):
    v, i = torch.randn(2, 3, 3, device="cuda"), torch.zeros(2, 3, 3, device="cuda", dtype=torch.int64)
    if which == "projections":
        m = dv.CrossAttention(32, 2, state_dim=16).cuda()
        x, s = torch.randn(2, 4, 32, device="cuda"), torch.randn(2, 5, 16, device="cuda")
        leaf, call = m.query.weight, lambda: m(x, s).sum()
        alive = m.query(x)
    elif which == "keys and values of one tensor":
        leaf = torch.randn(2, 6, 2, 1, 16, device="cuda", requires_grad=True)
        q, call = torch.randn(2, 3, 1, 16, device="cuda"), lambda: dv.cross_attention(q, leaf[:, :, 0], leaf[:, :, 1]).sum()
        alive = dv.cross_attention(q, leaf[:, :, 1], leaf[:, :, 0])
    elif which == "logits of three dimensions":
        leaf = torch.randn(2, 3, 16, device="cuda", requires_grad=True)
        call = lambda: dv.distillation_loss(leaf, v, i)  # noqa: E731
        alive = call()
    else:
        leaf = torch.randn(16, 6, device="cuda", requires_grad=True)
        call = lambda: dv.distillation_loss(leaf.t(), v.view(6, 3), i.view(6, 3))  # noqa: E731
        alive = call()
    call().backward()                                               # eager ones run
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
        with pytest.raises(RuntimeError, match="captured while"):
            torch.autograd.grad(out, leaf)
        del out
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g, = torch.autograd.grad(call(), leaf)
    want, = torch.autograd.grad(call(), leaf)
    graph.replay()
    torch.cuda.synchronize()
    assert float((g - want).abs().max()) <= 1e-5 * float(want.abs().max())      # (a projection's weight gradient may add atomically)


def test_a_captured_projection_refuses_while_an_eager_graph_of_its_weight_lives():
    lin, x = dv.HipLinear(32, 16).cuda(), torch.randn(5, 32, device="cuda")
    alive = lin(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lin(x)
        with pytest.raises(RuntimeError, match="HipLinear: this backward is being captured while"):
            torch.autograd.grad(out, lin.weight, torch.ones_like(out))
        del out
    assert alive.shape == (5, 16)


def test_a_gradient_of_a_constant_upstream_says_when_it_is_differentiated_again():
    # a gradient penalty: the first gradient depends on the inputs, whatever comes from above
    z, x = torch.randn(2, 9, device="cuda", requires_grad=True), torch.randn(1, 3, 2, 8, device="cuda", requires_grad=True)
    v, i = torch.randn(2, 3, device="cuda"), torch.zeros(2, 3, device="cuda", dtype=torch.int64)
    for call, leaf in ((lambda: dv.distillation_loss(z, v, i), z), (lambda: dv.distillation_loss(z.view(2, 1, 9), v[:, None], i[:, None], reduction="sum"), z),
                       (lambda: dv.cross_attention(x, x.detach(), x.detach()).sum(), x), (lambda: dv.cross_attention(x.detach(), x, x.detach()).sum(), x),
                       (lambda: dv.cross_attention(x.detach(), x.detach(), x).sum(), x)):
        g, = torch.autograd.grad(call(), leaf, create_graph=True)
        assert torch.equal(g.detach(), torch.autograd.grad(call(), leaf)[0])
        with pytest.raises(RuntimeError, match="differentiated again"):
            g.square().sum().backward()
    table = torch.randn(5, 8, device="cuda", requires_grad=True)    # linear: a constant upstream gives a constant gradient
    g, = torch.autograd.grad(dv.embed_tokens(table, torch.arange(3, device="cuda")).sum(), table, create_graph=True)
    assert not g.requires_grad


def test_a_gradient_through_projections_says_when_it_is_differentiated_again():
    torch.manual_seed(14)
    m, lin = dv.CrossAttention(32, 2, state_dim=16).cuda(), dv.HipLinear(16, 8).cuda()
    x, s, y = torch.randn(2, 4, 32, device="cuda", requires_grad=True), torch.randn(2, 5, 16, device="cuda"), torch.randn(3, 16, device="cuda", requires_grad=True)
    for call, leaf in ((lambda: m(x, s).sum(), x), (lambda: lin(y).sum(), y), (lambda: lin(y.detach()).square().sum(), lin.weight)):
        g, = torch.autograd.grad(call(), leaf, create_graph=True)
        want, = torch.autograd.grad(call(), leaf)
        assert float((g.detach() - want).abs().max()) <= 1e-5 * float(want.abs().max())
        with pytest.raises(RuntimeError, match="differentiated again"):
            (call() + g.square().sum()).backward()                  # a penalty beside a loss


def test_transforms_and_traces_are_refused_on_the_device():
    import torch.autograd.forward_ad as fwd
    ids, x = torch.zeros(2, 3, device="cuda", dtype=torch.int64), torch.randn(1, 4, 2, 8, device="cuda")
    for call, t in ((lambda t: dv.embed_tokens(t, ids[0]), torch.randn(5, 8, device="cuda")),
                    (lambda z: dv.distillation_loss(z, torch.zeros(2, 3, device="cuda"), ids), torch.randn(2, 9, device="cuda")),
                    (lambda k: dv.cross_attention(x, k, x), x)):
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(fwd.make_dual(t, torch.ones_like(t)))
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, t, check_trace=False)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(torch.stack([t, t]))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda y: call(y).sum())(t)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (t,), (t,))
        assert torch.isfinite(call(t)).all()


def test_a_schedule_of_the_teachers_weight_passes_through_zero():
    _, _, _, teacher, step, batch = small_step(0.5, True, keep=True)
    bias = [n for n, _ in step.other if n.endswith("classifier.5.bias")][0]
    none, g0, _, _ = small_step(0.0, False)
    for w in (0.25, 0.0, 0.25):
        step.distill_weight = w
        out = step(*batch, teacher=teacher)
        grad = dict(step.other)[bias].grad.clone()
        z = out["logits"].detach().requires_grad_(True)
        kd = dv.distillation_loss(z, *teacher, 2.0)
        gz, = torch.autograd.grad(kd, z)
        assert torch.equal(out["distill"], kd.detach())
        assert abs(float(out["loss"] - none["loss"]) - w * float(kd.detach())) <= 1e-6 * float(none["loss"])
        # (lr = 0: the logits are those of the first step up to its atomics, 1e-4 of their size)
        assert float((grad - g0[bias] - w * gz.sum(0)).abs().max()) <= 1e-4 * float(z.detach().abs().max())
    step.distill_weight = 0.0
    step(*batch)                                                    # no teacher and no weight
    step.distill_weight = 0.5
    with pytest.raises(ValueError):
        step(*batch)


def _teacher_rank(rank, world, rendezvous, q):
    """A rank of TrainStep on GPU 0, gradients averaged over gloo through host memory; its teacher lists other numbers of pairs."""
    import torch.distributed as dist
    torch.cuda.set_device(0)
    dist.init_process_group("gloo", init_method=rendezvous, rank=rank, world_size=world)
    try:
        seen = {}
        for w in (0.5, 0.0):
            _, _, _, (values, indices), step, batch = small_step(0.5, True, keep=True)
            indices[rank + 1:] = -1                                 # rank + 1 pairs; 2 of the batch's are never listed
            step.world, step.distill_weight = world, w
            real = step.opt.step

            def averaged(segs):
                for seg in segs:
                    h = seg[2].cpu()
                    dist.all_reduce(h)
                    seg[2].copy_(h / world)
                return real(segs)

            step.opt.step = averaged
            out = step(*batch, teacher=(values, indices))
            bias = [n for n, _ in step.other if n.endswith("classifier.5.bias")][0]
            seen[w] = (dict(step.other)[bias].grad.cpu(), float(out["distill"]), out["logits"].detach().cpu(), values.cpu(), indices.cpu(),
                       float(out["loss"] - out["ce"]))
        q.put((rank, {w: tuple(x.numpy() if torch.is_tensor(x) else x for x in t) for w, t in seen.items()}))
    finally:
        dist.destroy_process_group()


@pytest.mark.timeout(300)
def test_a_teacher_that_lists_other_numbers_of_pairs_on_the_ranks():
    import torch.multiprocessing as mp
    from test_hip_parallel import _rendezvous
    world = 2
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    rendezvous = _rendezvous()
    procs = [ctx.Process(target=_teacher_rank, args=(r, world, rendezvous, q)) for r in range(world)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=240) for _ in range(world))
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    _, d, z, v, i, _ = zip(*(got[r][0.5] for r in range(world)))
    z = torch.cat([torch.from_numpy(x) for x in z]).double().requires_grad_(True)
    v, i = (torch.cat([torch.from_numpy(x) for x in t]) for t in (v, i))
    listed = (i >= 0).any(1)
    assert int(listed.sum()) == 3                                   # 1 of rank 0, 2 of rank 1
    logp, logq = torch.log_softmax(v.double()[listed] / 2, 1), torch.log_softmax(z[listed] / 2, 1).gather(1, i[listed])
    want = (logp.exp() * (logp - logq)).sum(1).mean() * 4           # the concatenated batch's mean
    gz, = torch.autograd.grad(want, z)
    assert abs(sum(d) / world - float(want)) <= 1e-5 * float(want)
    assert abs((got[0][0.0][1] + got[1][0.0][1]) / world - float(want)) <= 1e-4 * float(want)      # (reported at weight 0 as well)
    # the last bias's averaged gradient: with and without the term (lr does not matter: first steps of equal models, atomics 1e-4 of the logits)
    for r in range(world):
        moved = torch.from_numpy(got[r][0.5][0] - got[r][0.0][0]).double()
        assert float((moved - 0.5 * gz.sum(0)).abs().max()) <= 1e-4 * float(z.detach().abs().max())
    assert float(gz.sum(0).abs().max()) > 1e-3 * float(z.detach().abs().max())      # a mean over shards would be off by more than the bound


def test_a_teacher_without_ranks_to_ask_is_refused():
    _, _, _, teacher, step, batch = small_step(0.5, True, keep=True)
    step.world = 2
    with pytest.raises(RuntimeError, match="needs torch.distributed"):
        step(*batch, teacher=teacher)


def test_a_captured_backward_runs_beside_an_eager_graph_of_another_stream():
    # a wrapper that keeps accumulation nodes makes them on a side stream, and captures on yet another one
    gen = torch.Generator(device="cuda").manual_seed(15)
    x, z = torch.randn(2, 6, 2, 16, generator=gen, device="cuda", requires_grad=True), torch.randn(3, 20, generator=gen, device="cuda", requires_grad=True)
    table, ids = torch.randn(30, 8, generator=gen, device="cuda", requires_grad=True), torch.randint(0, 30, (3, 4), generator=gen, device="cuda")
    lin = dv.HipLinear(16, 8).cuda()
    leaves = [x, z, table, lin.weight]

    def step():
        loss = dv.cross_attention(x, x, x).square().sum() + dv.distillation_loss(z, table[:3, :4].detach(), ids, 2.0)
        loss = loss + dv.embed_tokens(table, ids).square().sum() + lin(x.view(24, 16)).square().sum()
        return torch.autograd.grad(loss, leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = [t.view_as(t) for t in leaves]
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
    assert len(alive) == 4
