"""The workloads of the question-side operators: token embedding, cross attention to a video's states, distillation of answers.

`listed()` and `draw()` give the cases, `prepare()` what a program has in hand, `run()` one pass: in plain torch operations, or
(`own`) as a user of the framework calls it; `exact()` the definition in 64 bits."""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # a batch of questions (64 pairs x 15 words, 4000 words of 300 features) in a training step of the shipped configuration
        {"name": "embed questions train fp32", "op": "embed", "type": "fp32", "n": 960, "vocab": 4000, "wd": 300, "pad": True, "train": True},
        # the next word of 64 answers being written: one token each, latency alone
        {"name": "embed one word serve bf16", "op": "embed", "type": "bf16", "n": 64, "vocab": 32000, "wd": 768, "pad": False, "train": False},
        # a corpus batch of captions with its padding, Zipf-like words
        {"name": "embed corpus train bf16", "op": "embed", "type": "bf16", "n": 65536, "vocab": 50000, "wd": 1024, "pad": True, "train": True},
        # rows that no vector load fits, no padding word
        {"name": "embed odd rows train fp16", "op": "embed", "type": "fp16", "n": 3001, "vocab": 10007, "wd": 301, "pad": False, "train": True},
        # 20 clips of every video look at the words of its question (the reasoning unit's sizes, 8 heads of 96)
        {"name": "attend clips-words train fp32", "op": "attend", "type": "fp32", "B": 64, "Lq": 20, "Lk": 15, "H": 8, "Hk": 8, "Dh": 96, "mask": False, "train": True},
        # the words of a question look at every frame of its video (64 clips x 16 frames), some frames dropped by a mask
        {"name": "attend words-frames train bf16", "op": "attend", "type": "bf16", "B": 64, "Lq": 15, "Lk": 1024, "H": 8, "Hk": 8, "Dh": 96, "mask": True, "train": True},
        # long captions over long videos, shared key heads: the matrix units' case
        {"name": "attend long train bf16", "op": "attend", "type": "bf16", "B": 2, "Lq": 4096, "Lk": 4096, "H": 16, "Hk": 4, "Dh": 128, "mask": False, "train": True},
        # one word of 64 answers over the states of their videos
        {"name": "attend one word serve fp16", "op": "attend", "type": "fp16", "B": 64, "Lq": 1, "Lk": 2048, "H": 16, "Hk": 4, "Dh": 64, "mask": False, "train": False},
        # one word of one answer over hours of frames: the work has to be split over the states
        {"name": "attend one word long serve bf16", "op": "attend", "type": "bf16", "B": 1, "Lq": 1, "Lk": 65536, "H": 32, "Hk": 8, "Dh": 128, "mask": False, "train": False},
        # the answer head's batch: 1000 answers, the teacher's first 10
        {"name": "distil answers train fp32", "op": "distil", "type": "fp32", "R": 64, "C": 1000, "K": 10, "train": True},
        # a batch of words over a vocabulary
        {"name": "distil words train bf16", "op": "distil", "type": "bf16", "R": 4096, "C": 32000, "K": 64, "train": True},
        # a large vocabulary of odd size: rows that start at every alignment
        {"name": "distil odd vocabulary train fp16", "op": "distil", "type": "fp16", "R": 1023, "C": 100003, "K": 50, "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "attend", "distil"])
    kind = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.75
    if op == "embed":
        wd = _log(rng, 64, 1024)
        if rng.random() < 0.7:
            wd = max(8, wd // 8 * 8)
        n = _log(rng, 64, 65536)
        return {"op": op, "type": kind, "n": n, "vocab": _log(rng, 1000, 50000), "wd": wd, "pad": rng.random() < 0.5, "train": train}
    if op == "attend":
        Hk = rng.choice([1, 2, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 4])
        Dh = rng.choice([32, 40, 64, 80, 96, 128])
        if not train:
            B, Lq = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 16])
            Lk = _log(rng, 256, 65536)
        else:
            B, Lq, Lk = _log(rng, 1, 64), _log(rng, 4, 4096), _log(rng, 4, 4096)
        most = 2.0 ** 28 if kind == "fp32" else 2.0 ** 30
        while 1.0 * B * H * Lq * Lk > most / 4 or 1.0 * B * Hk * Lk * Dh > 2.0 ** 27:
            B, Lk = max(1, B // 2), max(4, (Lk * 3) // 4)
        return {"op": op, "type": kind, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hk": Hk, "Dh": Dh, "mask": rng.random() < 0.4, "train": train}
    C, K = _log(rng, 100, 131072), _log(rng, 1, 128)
    R = max(1, min(_log(rng, 16, 8192), 2 ** 27 // C))
    return {"op": op, "type": kind, "R": R, "C": C, "K": min(K, C), "train": train}


def _mean_len(case):
    return 0.75 * case["Lk"] if case["B"] > 1 else 1.0 * case["Lk"]


def work(case):
    es = SIZES[case["type"]]
    if case["op"] == "embed":
        n, V, wd = case["n"], case["vocab"], case["wd"]
        b = 8 * n + es * wd * (min(n, V) + n)
        if case["train"]:
            b += es * wd * (n + V)
        return {"bytes": b, "flops": (2 if case["train"] else 1) * n * wd}
    if case["op"] == "attend":
        B, Lq, Lk, H, Hk, Dh = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "Dh"))
        L = _mean_len(case)
        b = es * B * Dh * (2 * Lq * H + 2 * L * Hk)
        f = 4.0 * B * H * Lq * L * Dh
        if case["train"]:
            b += es * B * Dh * (2 * Lq * H + 2 * Lk * Hk)
            f += 10.0 * B * H * Lq * L * Dh
        return {"bytes": b, "flops": f}
    R, C, K = case["R"], case["C"], case["K"]
    b = R * C * es + R * K * (es + 8)
    if case["train"]:
        b += R * C * es
    return {"bytes": b, "flops": (6 if case["train"] else 4) * R * C}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(t)

    s = {"op": case["op"], "train": case["train"]}
    if case["op"] == "embed":
        n, V, wd = case["n"], case["vocab"], case["wd"]
        tokens = (float(V) ** torch.rand(n, generator=g, device="cuda", dtype=torch.float64)).long() - 1      # few words are most of a text
        tokens = tokens.clamp_(0, V - 1)
        if case["pad"]:
            tokens[torch.rand(n, generator=g, device="cuda") < 0.25] = 0
        s.update(table=normal(V, wd).requires_grad_(case["train"]), tokens=tokens, scale=math.sqrt(wd), padding_idx=0 if case["pad"] else None)
        if case["train"]:
            s["up"] = normal(n, wd)
        return s
    if case["op"] == "attend":
        B, Lq, Lk, H, Hk, Dh = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "Dh"))
        q = (2.0 * normal(B, Lq, H, Dh)).to(t)
        kv = normal(B, Lk, 2, Hk, Dh)                      # one projection gives keys and values side by side
        s.update(q=q.requires_grad_(case["train"]), k=kv[:, :, 0].detach().requires_grad_(case["train"]),
                 v=kv[:, :, 1].detach().requires_grad_(case["train"]), lens=None, mask=None)
        if B > 1:
            s["lens"] = torch.randint(Lk - Lk // 2, Lk + 1, (B,), generator=g, device="cuda")
        if case["mask"]:
            s["mask"] = torch.rand(B, Lk, generator=g, device="cuda") < 0.9
        if case["train"]:
            s["up"] = normal(B, Lq, H, Dh)
        return s
    R, C, K = case["R"], case["C"], case["K"]
    z = torch.randn(R, C, generator=g, device="cuda").mul_(2.0)
    teacher = z + torch.randn(R, C, generator=g, device="cuda")
    values, indices = teacher.topk(K, dim=1)
    # a training loop in half precision scales its loss: the gradient of a mean over many rows would otherwise leave the type's range
    s.update(logits=z.to(t).requires_grad_(case["train"]), values=values.to(t), indices=indices, temperature=2.0,
             up=torch.tensor(65536.0 if t == torch.float16 else 1.0, device="cuda"))
    return s


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"embed": _plain_embed, "attend": _plain_attend, "distil": _plain_distil}[s["op"]](s)


def _own(s):
    import dualvgr_videoqa_amd as dv
    if s["op"] == "embed":
        if not s["train"]:
            with torch.no_grad():
                return dv.embed_tokens(s["table"], s["tokens"], scale=s["scale"], padding_idx=s["padding_idx"])
        y = dv.embed_tokens(s["table"], s["tokens"], scale=s["scale"], padding_idx=s["padding_idx"])
        return [y, *torch.autograd.grad(y, [s["table"]], s["up"])]
    if s["op"] == "attend":
        if not s["train"]:
            with torch.no_grad():
                return dv.cross_attention(s["q"], s["k"], s["v"], lens=s["lens"], mask=s["mask"])
        o = dv.cross_attention(s["q"], s["k"], s["v"], lens=s["lens"], mask=s["mask"])
        return [o, *torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["up"])]
    if not s["train"]:
        with torch.no_grad():
            return dv.distillation_loss(s["logits"], s["values"], s["indices"], temperature=s["temperature"])
    loss = dv.distillation_loss(s["logits"], s["values"], s["indices"], temperature=s["temperature"])
    return [loss, *torch.autograd.grad(loss, [s["logits"]], s["up"])]


def _plain_embed(s):
    table, tokens, t = s["table"], s["tokens"], s["table"].dtype
    y = (table[tokens].float() * s["scale"]).to(t)
    if not s["train"]:
        return y
    up = s["up"].float() * s["scale"]
    if s["padding_idx"] is not None:
        up = up * (tokens != s["padding_idx"]).unsqueeze(1)
    g = torch.zeros(table.shape, device=table.device, dtype=torch.float32)
    return [y, g.index_add_(0, tokens, up).to(t)]


def _plain_attend(s):
    q, k, v, t = s["q"], s["k"], s["v"], s["q"].dtype
    B, Lq, H, Dh = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = 1.0 / math.sqrt(Dh)
    rows = lambda x: x.float().view(B, Lq, Hk, G, Dh).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, Dh)  # noqa: E731
    back = lambda x: x.view(B, Hk, G, Lq, Dh).permute(0, 3, 1, 2, 4).reshape(B, Lq, H, Dh).to(t)  # noqa: E731
    qf, kf, vf = rows(q), k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous()
    live = torch.ones(B, 1, 1, Lk, dtype=torch.bool, device=q.device)
    if s["lens"] is not None:
        live = live & (torch.arange(Lk, device=q.device) < s["lens"].view(B, 1, 1, 1))
    if s["mask"] is not None:
        live = live & s["mask"].view(B, 1, 1, Lk)
    x = (qf @ kf.transpose(2, 3).contiguous()).mul_(scale).masked_fill_(~live, -math.inf)
    top = x.amax(3, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(3, keepdim=True).clamp_min(1e-37)
    o = p @ vf
    if not s["train"]:
        return back(o)
    up = rows(s["up"])
    dv = p.transpose(2, 3).contiguous() @ up
    dp = up @ vf.transpose(2, 3).contiguous()
    ds = p * (dp - (up * o).sum(3, keepdim=True)) * scale
    dq = ds @ kf
    dk = ds.transpose(2, 3).contiguous() @ qf
    return [back(o), back(dq), dk.transpose(1, 2).to(t).contiguous(), dv.transpose(1, 2).to(t).contiguous()]


def _plain_distil(s):
    z, T, t = s["logits"].float() / s["temperature"], s["temperature"], s["logits"].dtype
    a = s["values"].float() / T
    a = a - a.amax(1, keepdim=True)
    logp = a - torch.exp(a).sum(1, keepdim=True).log()
    p = torch.exp(logp)
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    logq = z.gather(1, s["indices"]) - total.log()
    loss = (p * (logp - logq)).sum(1).mean() * (T * T)
    if not s["train"]:
        return loss
    g = (e / total).scatter_add_(1, s["indices"], -p) * (T / z.shape[0] * s["up"])
    return [loss, g.to(t)]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if s["op"] == "embed":
            E, up = s["table"].double(), s["up"].double() if s["train"] else None
            y = s["scale"] * torch.index_select(E, 0, s["tokens"])
            if not s["train"]:
                return y
            grad = torch.zeros_like(E)
            keep = torch.ones_like(s["tokens"], dtype=torch.bool) if s["padding_idx"] is None else s["tokens"] != s["padding_idx"]
            grad.index_put_((s["tokens"][keep],), up[keep], accumulate=True)
            return [y, s["scale"] * grad]
        if s["op"] == "attend":
            return _exact_attend(s)
        z = s["logits"].double() / s["temperature"]
        T2 = s["temperature"] ** 2
        logp = torch.log_softmax(s["values"].double() / s["temperature"], 1)
        logq = torch.log_softmax(z, 1)
        R = z.shape[0]
        loss = T2 / R * sum((logp[r].exp() * (logp[r] - logq[r, s["indices"][r]])).sum() for r in range(R))
        if not s["train"]:
            return loss
        d = logq.exp()
        d.scatter_add_(1, s["indices"], -logp.exp())
        return [loss, d * (s["up"].double() * T2 / s["temperature"] / R)]


def _exact_attend(s):
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    B, Lq, H, Dh = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G, c = H // Hk, Dh ** -0.5
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        n = Lk if s["lens"] is None else int(s["lens"][b])
        at = torch.arange(n, device=q.device)
        if s["mask"] is not None:
            at = at[s["mask"][b, :n]]
        if not len(at):
            continue
        kb, vb = k[b, at].repeat_interleave(G, 1).permute(1, 2, 0).contiguous(), v[b, at].repeat_interleave(G, 1).permute(1, 0, 2).contiguous()
        qb = q[b].permute(1, 0, 2).contiguous()
        w = torch.softmax(c * torch.bmm(qb, kb), 2)
        ob = torch.bmm(w, vb)
        o[b] = ob.permute(1, 0, 2)
        if not s["train"]:
            continue
        ub = s["up"][b].double().permute(1, 0, 2).contiguous()
        dw = torch.bmm(ub, vb.permute(0, 2, 1).contiguous())
        dx = c * w * (dw - (dw * w).sum(2, keepdim=True))
        dq[b] = torch.bmm(dx, kb.permute(0, 2, 1).contiguous()).permute(1, 0, 2)
        dk[b, at] = torch.bmm(dx.permute(0, 2, 1).contiguous(), qb).view(Hk, G, len(at), Dh).sum(1).permute(1, 0, 2)
        dv[b, at] = torch.bmm(w.permute(0, 2, 1).contiguous(), ub).view(Hk, G, len(at), Dh).sum(1).permute(1, 0, 2)
    return [o, dq, dk, dv] if s["train"] else o
