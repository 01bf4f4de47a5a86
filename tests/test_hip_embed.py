"""GPU: token embedding with scaling and its gradient by sorted tokens (include/dvgr_inputs.h, inputs.embed_tokens) against 64 bits.

Tolerances: a result is rounded to its type once (half a step, finfo.eps / 2 relative, half the smallest subnormal below that);
in front of it stands one fp32 product, or an fp32 sum of m terms (m 2^-24 of the sum of their magnitudes)."""
import pytest
import torch

import dualvgr_videoqa_amd as dv

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(want, t):
    return want.abs() * (torch.finfo(t).eps / 2) + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def check_embed(table, tokens, scale, padding, up, y, g):
    t, vocab = table.dtype, table.shape[0]
    E, flat = table.double(), tokens.reshape(-1)
    ok = (flat >= 0) & (flat < vocab)
    want = torch.where(ok[:, None], scale * E[flat.clamp(0, vocab - 1)], 0.0).view(*tokens.shape, -1)
    assert ((y.double() - want).abs() <= half_step(want, t) + want.abs() * 2.0 ** -23).all()
    if g is None:
        return
    keep = ok if padding is None else ok & (flat != padding % vocab)
    u = up.reshape(flat.numel(), -1).double()
    want, size = torch.zeros_like(E), torch.zeros_like(E)
    want.index_add_(0, flat[keep], scale * u[keep])
    size.index_add_(0, flat[keep], abs(scale) * u[keep].abs())
    most = int(torch.bincount(flat[keep], minlength=1).max()) if int(keep.sum()) else 0
    assert ((g.double() - want).abs() <= half_step(want, t) + size * (most + 2) * 2.0 ** -24).all()


def tokens_of(kind, n, vocab, gen):
    if kind == "zipf":
        return ((float(vocab) ** torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)).long() - 1).clamp_(0, vocab - 1)
    if kind == "one":
        return torch.full((n,), vocab // 2, device="cuda")
    if kind == "last":
        return torch.full((n,), vocab - 1, device="cuda")
    return torch.randint(0, vocab, (n,), generator=gen, device="cuda")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind,n,vocab,wd,padding", [
    ("uniform", 1, 1, 1, None), ("uniform", 31, 7, 8, 0), ("uniform", 32, 255, 300, None), ("uniform", 33, 256, 64, None),
    ("one", 64, 3, 40, None), ("one", 5000, 1000, 96, None), ("one", 100, 9, 17, 4), ("last", 257, 65536, 24, None),
    ("zipf", 960, 4000, 300, 0), ("zipf", 3001, 10007, 301, None), ("zipf", 20000, 70000, 136, -1), ("uniform", 4097, 300, 1025, None),
    ("zipf", 40000, 500, 520, 3)])
def test_values_and_gradient(t, kind, n, vocab, wd, padding):
    gen = torch.Generator(device="cuda").manual_seed(n + wd)
    table = torch.randn(vocab, wd, generator=gen, device="cuda").to(t).requires_grad_(True)
    tokens = tokens_of(kind, n, vocab, gen)
    up = torch.randn(n, wd, generator=gen, device="cuda").to(t)
    y = dv.embed_tokens(table, tokens, scale=3.7, padding_idx=padding)
    g, = torch.autograd.grad(y, table, up)
    check_embed(table.detach(), tokens, 3.7, padding, up, y.detach(), g)
    y2 = dv.embed_tokens(table, tokens, scale=3.7, padding_idx=padding)
    g2, = torch.autograd.grad(y2, table, up)
    assert torch.equal(g, g2) and torch.equal(y, y2)                # the same inputs, the same bits
    with torch.no_grad():
        assert torch.equal(dv.embed_tokens(table, tokens, scale=3.7), y)


def test_a_long_batch_of_few_tokens_takes_the_larger_sort_tiles():
    gen = torch.Generator(device="cuda").manual_seed(1)
    n, vocab, wd = (1 << 18) + 77, 50, 16
    table = torch.randn(vocab, wd, generator=gen, device="cuda").requires_grad_(True)
    tokens = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
    up = torch.randn(n, wd, generator=gen, device="cuda")
    y = dv.embed_tokens(table, tokens)
    g, = torch.autograd.grad(y, table, up)
    check_embed(table.detach(), tokens, 1.0, None, up, y.detach(), g)


@pytest.mark.parametrize("t", TYPES)
def test_tokens_outside_the_table(t):
    emb = dv.TokenEmbedding(10, 24, padding_idx=2, scale=2.0).to("cuda", t)
    tokens = torch.tensor([[1, 2, 10], [-1, 9, 1 << 40]]).cuda()
    y = emb(tokens)
    assert (y[0, 2] == 0).all() and (y[1, 0] == 0).all() and (y[1, 2] == 0).all()
    up = torch.randn_like(y)
    y.backward(up)
    check_embed(emb.weight.detach(), tokens, 2.0, 2, up, y.detach(), emb.weight.grad)
    with pytest.raises(IndexError):
        emb.check_tokens()
    emb(tokens[:, 1:2])
    emb.check_tokens()


def test_module_matches_torch_on_strided_inputs():
    gen = torch.Generator(device="cuda").manual_seed(5)
    emb = dv.TokenEmbedding(50, 20, padding_idx=-3).cuda()
    ref = torch.nn.Embedding(50, 20, padding_idx=-3).cuda()
    ref.load_state_dict(emb.state_dict())
    tokens = torch.randint(0, 50, (9, 14), generator=gen, device="cuda", dtype=torch.int32)[:, ::2]
    up = torch.randn(20, 9, 7, generator=gen, device="cuda").permute(1, 2, 0)
    y, yr = emb(tokens), ref(tokens.long())
    y.backward(up)
    yr.backward(up)
    assert torch.equal(y, yr) and float((emb.weight.grad - ref.weight.grad).abs().max()) < 1e-5
    one = emb(tokens[:1, :1])                                       # an upstream gradient that is one value broadcast
    one.sum().backward()
    assert dv.embed_tokens(emb.weight, tokens[:0]).shape == (0, 7, 20)


def test_rows_at_any_alignment():
    gen = torch.Generator(device="cuda").manual_seed(6)
    flat = torch.randn(1 + 40 * 16, generator=gen, device="cuda").half()
    table = flat[1:].view(40, 16).requires_grad_(True)              # two bytes past a 16-byte boundary
    tokens = torch.randint(0, 40, (100,), generator=gen, device="cuda")
    up = torch.randn(1 + 1600, generator=gen, device="cuda").half()[1:].view(100, 16)
    y = dv.embed_tokens(table, tokens, 0.5)
    g, = torch.autograd.grad(y, table, up)
    check_embed(table.detach(), tokens, 0.5, None, up, y.detach(), g)


def test_empty_batch_gives_a_zero_gradient():
    table = torch.randn(7, 5, device="cuda", requires_grad=True)
    y = dv.embed_tokens(table, torch.empty(0, dtype=torch.int64, device="cuda"))
    g, = torch.autograd.grad(y.sum(), table)
    assert y.shape == (0, 5) and (g == 0).all()


def test_another_stream_and_a_captured_graph():
    gen = torch.Generator(device="cuda").manual_seed(7)
    table = torch.randn(300, 64, generator=gen, device="cuda").requires_grad_(True)
    tokens = torch.randint(0, 300, (500,), generator=gen, device="cuda")
    up = torch.randn(500, 64, generator=gen, device="cuda")

    def step():
        y = dv.embed_tokens(table, tokens, 2.0, padding_idx=1)
        return y.detach(), torch.autograd.grad(y, table, up)[0]

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
    for k in range(3):
        tokens.copy_(torch.randint(0, 300, (500,), generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_a_captured_backward_refuses_while_an_eager_graph_of_the_same_leaf_lives():
    table = torch.randn(30, 16, device="cuda", requires_grad=True)
    tokens = torch.arange(20, device="cuda")
    alive = dv.embed_tokens(table, tokens)
    up = torch.ones(20, 16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dv.embed_tokens(table, tokens)
        with pytest.raises(RuntimeError, match="captured while"):
            torch.autograd.grad(y, table, up)
        del y
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g, = torch.autograd.grad(dv.embed_tokens(table, tokens), table, up)
    graph.replay()
    torch.cuda.synchronize()
    assert (g[:20] == 1).all() and (g[20:] == 0).all()
