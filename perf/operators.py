"""The training pass of the video block's attention as measurable cases: attention that keeps its softmax statistics,
attention's gradients, and the Q/K RMSNorm + rotation with its gradients.

With ``own`` false, ``run`` computes an operator from elementary torch operations in 32 bits; with ``own`` true it
calls ``opengenie_b200.ltx_ops``.  Sizes: 2304 and 9216 tokens are the 576p windows of the benchmark (4 and 16 latent
frames of 18 x 32 = 576 tokens), 28800 the 720p-class window (16 frames of 45 x 40 = 1800) with the 4 heads that one of
8 GPUs holds, 1024 the prompt context, 32 heads of 128 the block's width.
"""

import math

import torch

own = False

HEAD = 128
EPS = 1e-6


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the shortest window a test drives through the block: latency of one forward call
        _attn("fwd", "forward, 64 tokens", 1, 64, 64, 32, 32),
        # queries of two short clips over two prompts of unequal length, padded to the longer one
        _attn("fwd", "forward, padded prompts", 2, 2304, 1024, 32, 32, kv_lengths="1024,333"),
        # the 720p-class window, frame by frame: a token sees its own and all earlier latent frames
        _attn("fwd", "forward, 16 frames of 1800", 1, 28800, 28800, 4, 4, causal_block=1800),
        # a small token-causal sequence with shared key/value heads and an odd length
        _attn("bwd", "backward, 129 tokens", 2, 129, 129, 8, 2, causal_block=1),
        # the benchmark's self-attention, dense
        _attn("bwd", "backward, 9216 tokens", 1, 9216, 9216, 32, 32),
        # video queries over one padded prompt: many queries, few keys
        _attn("bwd", "backward, prompt of 1000", 1, 9216, 1024, 32, 32, kv_lengths="1000"),
        # two clips of unequal length, frame-causal, four query heads to a key head
        _attn("bwd", "backward, two clips", 2, 2305, 2305, 32, 8, causal_block=576, q_lengths="2305,1729",
              kv_lengths="2305,1729"),
        # one new token for each of four sequences
        _norm("nfwd", "norm + rotation, 4 tokens", 4, 1, 32, 8, "head", 128, False, False, "bf16"),
        # a norm for each head, half of the head rotated in neighbouring pairs
        _norm("nfwd", "norm + rotation, 9216 tokens", 1, 9216, 32, 32, "head", 64, True, False, "fp32"),
        # gradients for a short odd sequence
        _norm("nbwd", "norm gradient, 77 tokens", 1, 77, 32, 8, "head", 128, False, False, "fp32"),
        # gradients with shared key heads, two clips
        _norm("nbwd", "norm gradient, two clips", 2, 4099, 32, 8, "head", 128, True, False, "bf16"),
        # gradients of the video block's own norm: over all heads at once, a rotation table for each head
        _norm("nbwd", "norm gradient, whole rows", 1, 9216, 32, 32, "row", 128, False, True, "bf16"),
    ]


def _attn(op, name, batch, q_tokens, kv_tokens, heads, kv_heads, causal_block=0, q_lengths="", kv_lengths=""):
    return {"name": name, "op": op, "batch": batch, "q_tokens": q_tokens, "kv_tokens": kv_tokens, "heads": heads,
            "kv_heads": kv_heads, "causal_block": causal_block, "q_lengths": q_lengths, "kv_lengths": kv_lengths}


def _norm(op, name, batch, tokens, heads, kv_heads, norm, rotary, interleaved, per_head, weights):
    return {"name": name, "op": op, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "norm": norm, "rotary": rotary, "interleaved": interleaved, "per_head": per_head, "weights": weights}


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["fwd", "bwd", "nfwd", "nbwd"])
    heads = rng.choice([1, 2, 4, 8, 16, 32])
    kv_heads = heads // rng.choice([d for d in (1, 1, 2, 4, 8) if d <= heads])
    if op in ("nfwd", "nbwd"):
        norm = rng.choice(["head", "head", "row", "none"])
        per_head = kv_heads == heads and rng.random() < 0.3
        batch = rng.randint(1, 4)
        tokens = _log_int(rng, 1, 9216 * 32 // (heads * batch) if heads >= 4 else 20000)
        case = _norm(op, "", batch, min(tokens, 20000), heads, kv_heads, norm, rng.choice([32, 64, 96, 128]),
                     rng.random() < 0.5, per_head, rng.choice(["bf16", "fp32"]))
    else:
        batch = rng.randint(1, 4)
        most = (28800 ** 2 * 4 if op == "fwd" else 9216 ** 2 * 32) // (heads * batch)
        # A softmax over a single key is constant: its dq and dk are zero but for rounding and say nothing, so the
        # gradients' sequences and lengths start at 16 (or are empty, all but the batch's first).
        least = 16 if op == "bwd" else 1
        q_tokens = _log_int(rng, least, min(28800, math.isqrt(most)))
        kv_tokens = q_tokens if rng.random() < 0.6 else _log_int(rng, least, min(28800, most // q_tokens))
        causal_block = rng.choice([0, 0, 1, _log_int(rng, 2, 1800)])
        lengths = lambda n: ",".join(str(rng.randint(least, n) if i == 0 or rng.random() < 0.9 else 0)  # noqa: E731
                                     for i in range(batch))
        padded = rng.random() if kv_tokens == q_tokens or not causal_block else 1.0
        case = _attn(op, "", batch, q_tokens, kv_tokens, heads, kv_heads, causal_block,
                     lengths(q_tokens) if padded < 0.2 else "", lengths(kv_tokens) if padded < 0.4 else "")
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _lengths(text, batch, full):
    return [int(n) for n in text.split(",")] if text else [full] * batch


def _visible(case):
    """(query, key) pairs that the masks leave, for one head."""
    pairs = 0
    n, m, block = case["q_tokens"], case["kv_tokens"], case["causal_block"]
    for ql, kl in zip(_lengths(case["q_lengths"], case["batch"], n), _lengths(case["kv_lengths"], case["batch"], m)):
        if not block:
            pairs += ql * kl
            continue
        for i in range(ql):
            at = i + m - n
            pairs += min(kl, (at // block + 1) * block) if at >= 0 else 0
    return pairs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    s = dict(case)
    b, h, kh = case["batch"], case["heads"], case["kv_heads"]
    if case["op"] in ("nfwd", "nbwd"):
        n = case["tokens"]
        # rows of one packed projection, as the block's Q/K/V GEMM writes them
        rows = (randn(b, n, (h + 2 * kh) * HEAD) * 1.7).to(torch.bfloat16)
        s["q"], s["k"] = rows[..., :h * HEAD], rows[..., h * HEAD:(h + kh) * HEAD]
        kind = torch.bfloat16 if case["weights"] == "bf16" else torch.float32
        wide = {"head": (HEAD, HEAD), "row": (h * HEAD, kh * HEAD), "none": (0, 0)}[case["norm"]]
        s["qw"], s["kw"] = ((1 + 0.1 * randn(w)).to(kind) if w else None for w in wide)
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * freq + 6.0 * torch.rand(
            (h if case["per_head"] else 1, 1, 1), device="cuda", generator=gen)
        tables = angle.cos()[None], angle.sin()[None]
        s["cos"], s["sin"] = (t.to(torch.bfloat16) if case["per_head"] else t[:, 0].float() for t in tables)
        if case["op"] == "nbwd":
            s["dq"], s["dk"] = randn(b, n, h * HEAD).to(torch.bfloat16), randn(b, n, kh * HEAD).to(torch.bfloat16)
        return s
    n, m = case["q_tokens"], case["kv_tokens"]
    if n == m:  # self-attention: views of one packed projection
        rows = randn(b, n, (h + 2 * kh) * HEAD).to(torch.bfloat16)
        s["q"], s["k"], s["v"] = rows.split([h * HEAD, kh * HEAD, kh * HEAD], dim=-1)
    else:
        rows = randn(b, m, 2 * kh * HEAD).to(torch.bfloat16)
        s["q"] = randn(b, n, h * HEAD).to(torch.bfloat16)
        s["k"], s["v"] = rows.split([kh * HEAD, kh * HEAD], dim=-1)
    for name, full in (("q_lengths", n), ("kv_lengths", m)):
        s[name] = torch.tensor(_lengths(case[name], b, full), device="cuda", dtype=torch.int32) if case[name] else None
    if case["op"] == "bwd":
        s["out"], s["lse"] = _attention(s)  # what the forward pass left for the backward pass
        s["dout"] = randn(b, n, h * HEAD).to(torch.bfloat16)
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["op"] == "fwd":
        if own:
            from opengenie_b200 import ltx_ops

            return ltx_ops.attention_with_lse(s["q"], s["k"], s["v"], s["heads"], kv_heads=s["kv_heads"],
                                              causal_block=s["causal_block"], q_lengths=s["q_lengths"],
                                              kv_lengths=s["kv_lengths"])
        return _attention(s)
    if s["op"] == "bwd":
        if own:
            from opengenie_b200 import ltx_ops

            return ltx_ops.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["heads"],
                                              kv_heads=s["kv_heads"], causal_block=s["causal_block"],
                                              q_lengths=s["q_lengths"], kv_lengths=s["kv_lengths"])
        return _attention_gradients(s)
    if s["op"] == "nfwd":
        if own:
            from opengenie_b200 import ltx_ops

            return ltx_ops.fused_qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], EPS, s["cos"], s["sin"], s["heads"],
                                              kv_heads=s["kv_heads"], norm=s["norm"], interleaved=s["interleaved"])
        return tuple(_norm_rotate(s[x], s[x + "w"], s) for x in "qk")
    if own:
        from opengenie_b200 import ltx_ops

        grads = ltx_ops.fused_qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], EPS, s["cos"],
                                                    s["sin"], s["heads"], kv_heads=s["kv_heads"], norm=s["norm"],
                                                    interleaved=s["interleaved"])
        return [g for g in grads if g is not None]
    (dq, dqw), (dk, dkw) = (_norm_rotate_gradients(s["d" + x], s[x], s[x + "w"], s) for x in "qk")
    return [g for g in (dq, dk, dqw, dkw) if g is not None]


# ---------------------------------------------------------------------------------------------- plain forms
def _heads_first(x, heads):
    """[B, L, H*128] -> 32-bit [B, H, L, 128]."""
    return x.float().unflatten(-1, (heads, HEAD)).transpose(1, 2)


def _mask(s):
    """Pairs that a query may not see, [B, 1, L, L_kv]."""
    n, m, b = s["q_tokens"], s["kv_tokens"], s["batch"]
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")[None, :]
    hidden = torch.zeros((b, 1, n, m), device="cuda", dtype=torch.bool)
    if s["causal_block"]:
        hidden |= j // s["causal_block"] > torch.div(i + m - n, s["causal_block"], rounding_mode="floor")
    if s["q_lengths"] is not None:
        hidden |= i >= s["q_lengths"].view(b, 1, 1, 1)
    if s["kv_lengths"] is not None:
        hidden |= j >= s["kv_lengths"].view(b, 1, 1, 1)
    return hidden


def _scores(s):
    group = s["heads"] // s["kv_heads"]
    q = _heads_first(s["q"], s["heads"]) * HEAD ** -0.5
    k = _heads_first(s["k"], s["kv_heads"]).repeat_interleave(group, dim=1)
    scores = q @ k.transpose(-1, -2)
    if s["causal_block"] or s["q_lengths"] is not None or s["kv_lengths"] is not None:
        scores.masked_fill_(_mask(s), -math.inf)
    return scores


def _attention(s):
    v = _heads_first(s["v"], s["kv_heads"]).repeat_interleave(s["heads"] // s["kv_heads"], dim=1)
    p = _scores(s)
    top = p.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)  # a row that sees no key
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / total.clamp_min(1e-30)
    return out.transpose(1, 2).flatten(2).to(torch.bfloat16), (top + total.log()).squeeze(-1)


def _attention_gradients(s):
    group = s["heads"] // s["kv_heads"]
    q, dout, out = (_heads_first(s[x], s["heads"]) for x in ("q", "dout", "out"))
    k, v = (_heads_first(s[x], s["kv_heads"]).repeat_interleave(group, dim=1) for x in ("k", "v"))
    lse = s["lse"].unsqueeze(-1)
    p = _scores(s).sub_(torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)).exp_()
    dv = p.transpose(-1, -2) @ dout
    ds = (dout @ v.transpose(-1, -2)).sub_((dout * out).sum(-1, keepdim=True)).mul_(p).mul_(HEAD ** -0.5)
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    dk, dv = (g.unflatten(1, (s["kv_heads"], group)).sum(2) for g in (dk, dv))
    return tuple(g.transpose(1, 2).flatten(2).to(torch.bfloat16) for g in (dq, dk, dv))


def _tables(x, s):
    """cos and sin for x [B, L, H, 128], in 32 bits."""
    c, d = s["cos"].float(), s["sin"].float()
    return (c.transpose(1, 2), d.transpose(1, 2)) if s["per_head"] else (c.unsqueeze(2), d.unsqueeze(2))


def _turn(x, cos, sin, s):
    """Rotates the first `rotary` columns of each head."""
    r = s["rotary"]
    turned, rest = x[..., :r], x[..., r:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if s["interleaved"] else turned.chunk(2, dim=-1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if s["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, rest), -1)


def _inverse_rms(x, s):
    squares = x.square().mean(-1, keepdim=True)
    if s["norm"] == "row":
        squares = squares.mean(-2, keepdim=True)
    return torch.rsqrt(squares + EPS)


def _norm_rotate(x, weight, s):
    y = x.float().unflatten(-1, (-1, HEAD))
    if s["norm"] != "none":
        y = y * _inverse_rms(y, s) * weight.float().view(-1, HEAD)
    return _turn(y, *_tables(y, s), s).flatten(2).to(torch.bfloat16)


def _norm_rotate_gradients(dy, x, weight, s):
    x, g = x.float().unflatten(-1, (-1, HEAD)), dy.float().unflatten(-1, (-1, HEAD))
    cos, sin = _tables(x, s)
    g = _turn(g, cos, -sin, s)
    if s["norm"] == "none":
        return g.flatten(2).to(torch.bfloat16), None
    r = _inverse_rms(x, s)
    unit = x * r
    dw = (g * unit).double().sum((0, 1, 2) if s["norm"] == "head" else (0, 1)).flatten().float()
    g = g * weight.float().view(-1, HEAD)
    along = (g * unit).mean(-1, keepdim=True)
    if s["norm"] == "row":
        along = along.mean(-2, keepdim=True)
    return (r * (g - unit * along)).flatten(2).to(torch.bfloat16), dw


# ---------------------------------------------------------------------------------------------- work
def work(case):
    b, h, kh = case["batch"], case["heads"], case["kv_heads"]
    if case["op"] in ("nfwd", "nbwd"):
        elements = b * case["tokens"] * (h + kh) * HEAD
        tables = case["tokens"] * case["rotary"] * (2 * h if case["per_head"] else 4)
        wide = {"head": 2 * HEAD, "row": (h + kh) * HEAD, "none": 0}[case["norm"]]
        size = 2 if case["weights"] == "bf16" else 4
        if case["op"] == "nfwd":
            return {"bytes": 4 * elements + tables + wide * size, "flops": 9 * elements}
        return {"bytes": 6 * elements + tables + wide * (size + 4), "flops": 16 * elements}
    q, kv = b * case["q_tokens"] * h * HEAD, b * case["kv_tokens"] * kh * HEAD
    lse = 4 * b * case["q_tokens"] * h
    pairs = _visible(case) * h * HEAD
    if case["op"] == "fwd":  # reads q, k, v; writes out and the statistics; two products
        return {"bytes": 2 * (2 * q + 2 * kv) + lse, "flops": 4 * pairs}
    # reads q, k, v, out, dout and the statistics; writes three gradients; five products
    return {"bytes": 2 * (4 * q + 4 * kv) + lse, "flops": 10 * pairs}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("nfwd", "nbwd"):
        return _exact_norm(s)
    b, n, m, h, kh = (case[x] for x in ("batch", "q_tokens", "kv_tokens", "heads", "kv_heads"))
    scale, block = 1 / math.sqrt(HEAD), case["causal_block"]
    seen_q = _lengths(case["q_lengths"], b, n)
    seen_k = _lengths(case["kv_lengths"], b, m)
    at = torch.arange(n, device="cuda") + (m - n)
    last = (torch.div(at, block, rounding_mode="floor") + 1) * block if block else torch.full_like(at, m)
    wide = lambda x, i, head: s[x][i, :, head * HEAD:(head + 1) * HEAD].double()  # noqa: E731
    if case["op"] == "fwd":
        out = torch.zeros((b, n, h * HEAD), device="cuda", dtype=torch.float64)
        lse = torch.full((b, h, n), -math.inf, device="cuda", dtype=torch.float64)
    else:
        dq = torch.zeros((b, n, h * HEAD), device="cuda", dtype=torch.float64)
        dk, dv = (torch.zeros((b, m, kh * HEAD), device="cuda", dtype=torch.float64) for _ in range(2))
    for i in range(b):
        limit = last.clamp(0, seen_k[i])
        limit[seen_q[i]:] = 0
        rows = torch.nonzero(limit > 0).flatten()
        if not rows.numel():
            continue
        see = torch.arange(m, device="cuda") < limit[rows, None]
        for head in range(h):
            low, high = head * HEAD, (head + 1) * HEAD
            g = head * kh // h
            k, v, q = wide("k", i, g), wide("v", i, g), wide("q", i, head)[rows]
            z = torch.einsum("id,jd->ij", q, k).mul_(scale).masked_fill_(~see, -math.inf)
            if case["op"] == "fwd":
                lse[i, head, rows] = torch.logsumexp(z, -1)
                out[i, rows, low:high] = torch.softmax(z, -1) @ v
                continue
            p = torch.exp(z - s["lse"][i, head, rows, None].double())
            do, o = wide("dout", i, head)[rows], wide("out", i, head)[rows]
            dv[i, :, g * HEAD:(g + 1) * HEAD] += torch.einsum("ij,id->jd", p, do)
            p *= torch.einsum("id,jd->ij", do, v) - torch.einsum("id,id->i", do, o)[:, None]
            dq[i, rows, low:high] = torch.einsum("ij,jd->id", p, k) * scale
            dk[i, :, g * HEAD:(g + 1) * HEAD] += torch.einsum("ij,id->jd", p, q) * scale
    return (out, lse) if case["op"] == "fwd" else (dq, dk, dv)


def _exact_norm(s):
    """The rotation as a product of complex numbers; gradients by differentiating the forward form."""
    def forward(x, w):
        x = x.unflatten(-1, (x.shape[-1] // HEAD, HEAD))
        if s["norm"] != "none":
            squares = (x * x).flatten(2).mean(-1)[..., None, None] if s["norm"] == "row" else (x * x).mean(-1)[..., None]
            x = x / (squares + EPS).sqrt() * w.view(-1, HEAD)
        angle = torch.complex(s["cos"].double(), s["sin"].double())
        angle = angle.transpose(1, 2) if s["per_head"] else angle[:, :, None]
        r = s["rotary"]
        pairs = x[..., :r].unflatten(-1, (r // 2, 2)) if s["interleaved"] else x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * angle)
        z = z.flatten(-2) if s["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat((z, x[..., r:]), -1).flatten(2)

    given = {x: s[x].double().requires_grad_() for x in ("q", "k", "qw", "kw") if s[x] is not None}
    q, k = forward(given["q"], given.get("qw")), forward(given["k"], given.get("kw"))
    if s["op"] == "nfwd":
        return q.detach(), k.detach()
    return list(torch.autograd.grad((q, k), list(given.values()), (s["dq"].double(), s["dk"].double())))
