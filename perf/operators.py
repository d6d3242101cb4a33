"""Performance cases of the operators that answer many questions about one prompt: attention over a prompt that the whole
batch shares (``prefix_attention``), the mixture-of-experts block for the few tokens of a decode step (``moe_block``), and the
scores of given tokens (``token_logprobs``), each with its plain form in elementary torch operations and an exact form in 64
bits. ``own`` selects which of the first two ``run`` computes.

Shapes are the model variants' (heads, widths, expert counts, vocabulary 201088 stored in rows of 204800)."""

from __future__ import annotations

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
VOCAB, PADDED_VOCAB = 201088, 204800
# (query heads, kv heads, head dim) of the model variants
HEADS = {"lyra-tiny": (4, 2, 64), "lyra-small": (16, 4, 128), "lyra-medium": (32, 8, 128), "gpt-oss": (64, 8, 64)}


def listed() -> list[dict]:
    """Cases: the smallest calls of each operator (latency), ordinary ones and the largest."""

    def prefix(name, heads, B, T, P, S, window=0, kind="bf16"):
        Nq, Nkv, D = HEADS[heads]
        return dict(name=name, op="prefix_attention", Nq=Nq, Nkv=Nkv, D=D, B=B, T=T, P=P, S=S, window=window, kind=kind, sinks=True)

    return [
        # four answers to one short prompt, one new token each: latency counts
        prefix("prefix-decode-few", "lyra-small", 4, 1, 777, 64),
        # a serving batch behind one system prompt, one new token each
        prefix("prefix-decode-batch", "gpt-oss", 64, 1, 8192, 512),
        # the same with quantised caches (serving with --fp8)
        prefix("prefix-decode-e4m3", "lyra-medium", 32, 1, 4096, 256, kind="e4m3"),
        # multiple-choice scoring: the continuations of eight questions behind the same in-context examples
        prefix("prefix-choices", "gpt-oss", 32, 24, 1333, 24),
        # many samples of one long document
        prefix("prefix-decode-long", "gpt-oss", 256, 1, 32768, 1024),
        # one token of one sequence, small model: launch latency
        dict(name="moe-one-token-tiny", op="moe_block", C=256, H=512, E=4, k=2, shared=1, F=1, bias=False, kind="bf16"),
        # one chat, one token
        dict(name="moe-one-token", op="moe_block", C=2880, H=2880, E=32, k=4, shared=0, F=1, bias=True, kind="bf16"),
        # a few samples, routed and shared experts
        dict(name="moe-eight-tokens", op="moe_block", C=2048, H=2048, E=15, k=3, shared=1, F=8, bias=False, kind="bf16"),
        # a serving batch that touches most of 128 quantised experts
        dict(name="moe-batch-e4m3", op="moe_block", C=2880, H=2880, E=128, k=4, shared=0, F=64, bias=True, kind="e4m3"),
        # the next-token distribution of one sequence, with twenty alternatives
        dict(name="logprobs-one-row", op="token_logprobs", N=1, V=VOCAB, stride=PADDED_VOCAB, top_k=20, kind="fp32", grad=False),
        # one block of rows of the evaluation harness
        dict(name="logprobs-scoring", op="token_logprobs", N=2048, V=VOCAB, stride=PADDED_VOCAB, top_k=4, kind="bf16", grad=False),
        # a training objective on the log probability and the entropy of sampled tokens
        dict(name="logprobs-gradient", op="token_logprobs", N=1024, V=VOCAB, stride=VOCAB, top_k=0, kind="bf16", grad=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_any(rng) -> dict:
    op = rng.choice(["prefix_attention", "moe_block", "token_logprobs"])
    if op == "prefix_attention":
        Nq, Nkv, D = rng.choice([*HEADS.values(), (12, 4, 64), (10, 2, 128)])       # groups of 3 and 5 heads too
        T = 1 if rng.random() < 0.6 else rng.randint(2, 40)
        S = T + _log_int(rng, 1, 1500) - (1 if rng.random() < 0.3 else 0)
        return dict(op=op, Nq=Nq, Nkv=Nkv, D=D, B=_log_int(rng, 1, 256), T=T, P=_log_int(rng, 1, 32768), S=S,
                    window=rng.choice([0, 0, 128]), kind=rng.choice(["bf16", "e4m3"]), sinks=rng.random() < 0.8)
    if op == "moe_block":
        kind = rng.choice(["bf16", "e4m3"])
        unit = 8 if kind == "bf16" else 16
        E = rng.choice([4, 7, 15, 31, 32, 63, 128])
        return dict(op=op, C=unit * _log_int(rng, 128 // unit, 4096 // unit), H=unit * _log_int(rng, 128 // unit, 4096 // unit), E=E,
                    k=rng.randint(1, 4), shared=rng.choice([0, 1]), F=_log_int(rng, 1, 64), bias=rng.random() < 0.5, kind=kind)
    V = rng.choice([VOCAB, _log_int(rng, 1000, VOCAB)])
    grad = rng.random() < 0.4
    return dict(op=op, N=_log_int(rng, 1, 2048), V=V, stride=V + (rng.choice([0, 1, 64, 515]) if not grad else 0),
                top_k=0 if grad else rng.choice([0, 1, 5, 20, 32]), kind=rng.choice(["bf16", "fp32"]), grad=grad)


def draw(rng) -> dict:
    """One more case of the ranges above that is no larger than the largest listed case of its operator."""
    most: dict[str, list[float]] = {}
    for c in listed():
        w = work(c)
        top = most.setdefault(c["op"], [0.0, 0.0])
        top[0], top[1] = max(top[0], w["bytes"]), max(top[1], w["flops"])
    while True:
        c = _draw_any(rng)
        w = work(c)
        if w["bytes"] <= most[c["op"]][0] and w["flops"] <= most[c["op"]][1]:
            return c


def work(case: dict) -> dict:
    """Bytes and operations of one pass: every input once, every output once."""
    c = case
    if c["op"] == "prefix_attention":
        row = 2 * c["D"] if c["kind"] == "bf16" else c["D"] + 4
        own_keys = (c["S"] + c["T"]) / 2                       # positions are uniform over what the cache can hold
        window = c["window"]
        if window:                                             # a sliding layer sees the last `window` positions only
            own_seen = min(own_keys, window)
            prefix_seen = min(c["P"], max(window - own_keys, 0))
        else:
            own_seen, prefix_seen = own_keys, c["P"]
        caches = 2 * c["Nkv"] * row * (prefix_seen + c["B"] * own_seen)
        qo = 2 * 2 * c["B"] * c["Nq"] * c["T"] * c["D"]
        return {"bytes": caches + qo, "flops": 4.0 * c["B"] * c["Nq"] * c["T"] * c["D"] * (prefix_seen + own_seen)}
    if c["op"] == "moe_block":
        touched = c["E"] * (1 - (1 - c["k"] / c["E"]) ** c["F"]) + c["shared"]      # expected number of distinct experts
        size = 2 if c["kind"] == "bf16" else 1
        per_expert = 3 * c["C"] * c["H"]
        rows = c["F"] * (c["k"] + c["shared"])
        return {"bytes": touched * per_expert * size + 4 * c["C"] * c["E"] + 4 * c["F"] * c["C"], "flops": 2.0 * rows * per_expert}
    size = 2 if c["kind"] == "bf16" else 4
    cells = c["N"] * c["V"]
    return {"bytes": cells * size * (3 if c["grad"] else 1) + c["N"] * (16 + 12 * c["top_k"]), "flops": cells * (12.0 if c["grad"] else 6.0)}


# --------------------------------------------------------------------------- inputs
def _quantise(x: torch.Tensor, block: tuple[int, int]):
    """e4m3 values and fp32 block scales (block maximum / largest e4m3 number) over the last two axes."""
    r, n = block
    t = x.float().reshape(*x.shape[:-2], x.shape[-2] // r, r, x.shape[-1] // n, n)
    amax = t.abs().amax(dim=(-3, -1))
    scale = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    q = (t / scale[..., :, None, :, None]).clamp(-448.0, 448.0).to(E4M3).reshape(x.shape)
    return q, scale


def prepare(case: dict, seed: int):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)
    if c["op"] == "prefix_attention":
        B, T, P, S, Nq, Nkv, D = (c[n] for n in ("B", "T", "P", "S", "Nq", "Nkv", "D"))
        st = {"case": c, "q": randn(B, Nq, T, D).bfloat16(), "sinks": randn(Nq) if c["sinks"] else None}
        st["pos"] = torch.randint(0, S - T + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        for name, shape in (("pk", (Nkv, P, D)), ("pv", (Nkv, P, D)), ("k", (B, Nkv, S, D)), ("v", (B, Nkv, S, D))):
            x = randn(*shape)
            st[name] = _quantise(x, (1, D)) if c["kind"] == "e4m3" else x.bfloat16()
        return st
    if c["op"] == "moe_block":
        C, H, E, F = c["C"], c["H"], c["E"], c["F"]
        n = E + c["shared"]
        st = {"case": c, "x": randn(F, C).bfloat16(), "norm": 1 + 0.1 * randn(C), "router": randn(C, E) * (0.5 / math.sqrt(C)), "router_bias": 0.1 * randn(E)}
        up, down = [], []
        for _ in range(n):
            u, d = randn(C, 2 * H) / math.sqrt(C), randn(H, C) / math.sqrt(H)
            if c["kind"] == "e4m3":
                up.append(_quantise(u, (math.gcd(C, 256), math.gcd(2 * H, 256))))
                down.append(_quantise(d, (math.gcd(H, 256), math.gcd(C, 256))))
            else:
                up.append(u.bfloat16())
                down.append(d.bfloat16())
        if c["kind"] == "e4m3":
            st["up"] = tuple(torch.stack([t[i].view(torch.uint8) if i == 0 else t[i] for t in up]) for i in (0, 1))
            st["down"] = tuple(torch.stack([t[i].view(torch.uint8) if i == 0 else t[i] for t in down]) for i in (0, 1))
            st["up"], st["down"] = (st["up"][0].view(E4M3), st["up"][1]), (st["down"][0].view(E4M3), st["down"][1])
        else:
            st["up"], st["down"] = torch.stack(up).view(n, C, 2, H), torch.stack(down)
        st["up_bias"] = 0.1 * randn(n, 2, H) if c["bias"] else None
        st["down_bias"] = 0.1 * randn(n, C) if c["bias"] else None
        return st
    N, V = c["N"], c["V"]
    logits = torch.full((N, c["stride"]), float("-inf"), device=dev)
    logits[:, :V] = 2.5 * randn(N, V)
    logits = logits if c["kind"] == "fp32" else logits.bfloat16()
    st = {"case": c, "logits": logits, "targets": torch.randint(0, V, (N,), generator=g, device=dev)}
    if c["grad"]:
        st["g_logprob"], st["g_entropy"] = randn(N), 0.1 * randn(N)
    return st


# --------------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


def _wide(x, dtype):
    """A cache as numbers of ``dtype``: bf16 values, or e4m3 values times the scale of their row."""
    if isinstance(x, tuple):
        return x[0].to(dtype) * x[1].to(dtype)
    return x.to(dtype)


def _plain_prefix(st):
    c = st["case"]
    B, T, P, S, Nq, Nkv, D, window = (c[n] for n in ("B", "T", "P", "S", "Nq", "Nkv", "D", "window"))
    rep = Nq // Nkv
    q = st["q"].float().view(B, Nkv, rep, T, D) * D ** -0.5
    own_at = st["pos"].long()[:, None] + torch.arange(T, device=q.device)           # index of the query among the row's own positions
    i, j = torch.arange(S, device=q.device), torch.arange(P, device=q.device)
    see_own = i <= own_at[..., None]                                                  # [B, T, S]
    see_prefix = j <= (P + own_at)[..., None]                                         # [B, T, P]
    if window:
        see_own = see_own & (i > own_at[..., None] - window)
        see_prefix = see_prefix & (j > (P + own_at)[..., None] - window)
    out = torch.empty(B, Nkv, rep, T, D, device=q.device)
    for h in range(Nkv):                                                              # one kv head at a time bounds the scores' memory
        qh = q[:, h]
        s_p = (qh.reshape(-1, D) @ _wide(_index(st["pk"], h), torch.float32).t()).view(B, rep, T, P)
        s_o = qh.reshape(B, rep * T, D).bmm(_wide(_index(st["k"], (slice(None), h)), torch.float32).transpose(1, 2)).view(B, rep, T, S)
        s_p = s_p.masked_fill(~see_prefix[:, None], float("-inf"))
        s_o = s_o.masked_fill(~see_own[:, None], float("-inf"))
        m = torch.maximum(s_p.amax(-1, keepdim=True), s_o.amax(-1, keepdim=True))
        if st["sinks"] is not None:
            sink = st["sinks"].view(Nkv, 1, rep, 1, 1)[h]
            m = torch.maximum(m, sink)
        e_p, e_o = torch.exp(s_p - m), torch.exp(s_o - m)
        total = e_p.sum(-1, keepdim=True) + e_o.sum(-1, keepdim=True)
        if st["sinks"] is not None:
            total = total + torch.exp(sink - m)
        o = (e_p.view(-1, P) @ _wide(_index(st["pv"], h), torch.float32)).view(B, rep * T, D)
        o = o + e_o.view(B, rep * T, S).bmm(_wide(_index(st["v"], (slice(None), h)), torch.float32))
        out[:, h] = o.view(B, rep, T, D) / total
    return out.view(B, Nq, T, D).to(torch.bfloat16)


def _index(x, at):
    return tuple(t[at] for t in x) if isinstance(x, tuple) else x[at]


def _expert(w, e, dtype):
    """Weights of one expert as ``[K, N]`` of ``dtype`` (e4m3: value times the scale of its block)."""
    if not isinstance(w, tuple):
        t = w[e].to(dtype)
        return t.reshape(t.shape[0], -1)
    q, s = w[0][e].to(dtype), w[1][e].to(dtype)
    r, n = q.shape[0] // s.shape[0], q.shape[1] // s.shape[1]
    return (q.view(s.shape[0], r, s.shape[1], n) * s[:, None, :, None]).view(q.shape)


BETA, LIMIT, EPS, RESIDUAL = 1.702, 7.0, 1e-5, 0.25


def _moe(st, dtype):
    c = st["case"]
    F, k, shared, E = c["F"], c["k"], c["shared"], c["E"]
    x64 = st["x"].double()
    xn64 = x64 * torch.rsqrt((x64 * x64).mean(-1, keepdim=True) + EPS) * st["norm"].double()
    logits = xn64 @ st["router"].double() + st["router_bias"].double()               # 64 bits: near-equal experts must not change places
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    vals, idx = order.values[:, :k], order.indices[:, :k]
    ex = torch.exp(vals - vals[:, :1])
    scores = ex / ex.sum(-1, keepdim=True)
    xn = xn64.to(dtype)
    mixed = torch.zeros(F, c["C"], dtype=dtype, device=xn.device)
    chosen = torch.unique(idx).tolist() + list(range(E, E + shared))
    for e in chosen:
        if e < E:
            hit = idx == e
            weight = (scores * hit).sum(-1).to(dtype)
            rows = hit.any(-1).nonzero()[:, 0]
        else:
            weight = torch.ones(F, dtype=dtype, device=xn.device)
            rows = torch.arange(F, device=xn.device)
        t = xn[rows] @ _expert(st["up"], e, dtype)
        if st["up_bias"] is not None:
            t = t + st["up_bias"][e].reshape(-1).to(dtype)
        gate, lin = t[:, : c["H"]].clamp(max=LIMIT), t[:, c["H"]:].clamp(-LIMIT, LIMIT)
        a = (lin + 1) * gate / (1 + torch.exp(-BETA * gate))
        y = a @ _expert(st["down"], e, dtype)
        if st["down_bias"] is not None:
            y = y + st["down_bias"][e].to(dtype)
        mixed[rows] += weight[rows, None] * y
    return st["x"].to(dtype) + RESIDUAL * mixed, scores, idx


def _plain_moe(st):
    out, scores, idx = _moe(st, torch.float32)
    return out.to(torch.bfloat16), scores.float(), idx


def _logprobs(st, dtype):
    c = st["case"]
    x = st["logits"][:, : c["V"]].to(dtype)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    logprob = (x.gather(1, st["targets"][:, None]) - lse)[:, 0]
    entropy = (torch.log(total) - (e * (x - m)).sum(-1, keepdim=True) / total)[:, 0]
    return x, e / total, lse, logprob, entropy


def _logprob_gradient(st, dtype):
    x, p, lse, logprob, entropy = _logprobs(st, dtype)
    g_l, g_h = st["g_logprob"].to(dtype)[:, None], st["g_entropy"].to(dtype)[:, None]
    grad = -p * (g_l + g_h * (x - lse + entropy[:, None]))
    grad.scatter_add_(1, st["targets"][:, None], g_l)
    return logprob, entropy, grad


def _plain_logprobs(st):
    c = st["case"]
    if c["grad"]:
        logprob, entropy, grad = _logprob_gradient(st, torch.float32)
        return logprob, entropy, grad.to(st["logits"].dtype)
    x, _, lse, logprob, entropy = _logprobs(st, torch.float32)
    order = torch.sort(x, dim=-1, descending=True, stable=True)                       # equal logits: the lower token first
    k = c["top_k"]
    return logprob, entropy, order.values[:, :k] - lse, order.indices[:, :k]


def _own_prefix(st):
    from lyra_b200.nn.quant import QArray
    from lyra_b200.ops import api as ops

    D = st["case"]["D"]
    cache = lambda x: QArray(x[0], x[1], (1, D)) if isinstance(x, tuple) else x
    return ops.prefix_attention(st["q"], cache(st["pk"]), cache(st["pv"]), cache(st["k"]), cache(st["v"]), st["sinks"], D ** -0.5,
                                st["case"]["window"], st["pos"])


def _own_moe(st):
    from lyra_b200.nn.quant import QArray
    from lyra_b200.ops import api as ops

    c = st["case"]
    weight = lambda w: QArray(w[0], w[1], (w[0].shape[1] // w[1].shape[1], w[0].shape[2] // w[1].shape[2])) if isinstance(w, tuple) else w
    return ops.moe_block(st["x"], st["norm"], EPS, st["router"], st["router_bias"], weight(st["up"]), st["up_bias"], weight(st["down"]),
                         st["down_bias"], c["k"], c["shared"], BETA, LIMIT, RESIDUAL)


def _own_logprobs(st):
    from lyra_b200.ops import api as ops

    c = st["case"]
    if c["grad"]:
        logits = st["logits"].detach().requires_grad_()
        r = ops.token_logprobs(logits, st["targets"], vocab_size=c["V"])
        (grad,) = torch.autograd.grad((r.logprob, r.entropy), logits, (st["g_logprob"], st["g_entropy"]))
        return r.logprob.detach(), r.entropy.detach(), grad
    r = ops.token_logprobs(st["logits"], st["targets"], c["top_k"], vocab_size=c["V"])
    return r.logprob, r.entropy, r.top_logprobs, r.top_ids


_run_plain = {"prefix_attention": _plain_prefix, "moe_block": _plain_moe, "token_logprobs": _plain_logprobs}
_run_own = {"prefix_attention": _own_prefix, "moe_block": _own_moe, "token_logprobs": _own_logprobs}


# --------------------------------------------------------------------------- exact values
def exact(case: dict, seed: int):
    """The outputs of ``run`` from the operators' definitions in 64 bits, written apart from the plain forms: attention as one
    softmax over the concatenated keys of each row, the experts by token, the scores by ``log p`` itself."""
    st = prepare(case, seed)
    c = case
    f64 = torch.float64
    if c["op"] == "prefix_attention":
        B, T, P, S, Nq, Nkv, D, window = (c[n] for n in ("B", "T", "P", "S", "Nq", "Nkv", "D", "window"))
        rep = Nq // Nkv
        out = torch.zeros(B, Nq, T, D, dtype=f64, device="cuda")
        pk, pv = _wide(st["pk"], f64), _wide(st["pv"], f64)
        where = torch.cat([torch.arange(P, device="cuda"), P + torch.arange(S, device="cuda")])      # absolute position of every key
        sinks = st["sinks"].double() if st["sinks"] is not None else None
        for b in range(B):
            kb = torch.cat([pk, _wide(_index(st["k"], b), f64)], dim=1)                               # [Nkv, P + S, D]
            vb = torch.cat([pv, _wide(_index(st["v"], b), f64)], dim=1)
            at = P + int(st["pos"][b]) + torch.arange(T, device="cuda")[:, None]
            hidden = where > at
            if window:
                hidden |= where <= at - window
            s = torch.einsum("nrtd,nsd->nrts", st["q"][b].double().view(Nkv, rep, T, D), kb) / math.sqrt(D)
            s.masked_fill_(hidden, float("-inf"))
            if sinks is not None:
                s = torch.cat([s, sinks.view(Nkv, rep, 1, 1).expand(Nkv, rep, T, 1)], dim=-1)
            p = torch.softmax(s, dim=-1)[..., : P + S]
            out[b] = torch.einsum("nrts,nsd->nrtd", p, vb).reshape(Nq, T, D)
        return out
    if c["op"] == "moe_block":
        x = st["x"].double()
        xn = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * st["norm"].double()
        logits = xn @ st["router"].double() + st["router_bias"].double()
        ids = torch.argsort(-logits, dim=-1, stable=True)[:, : c["k"]]
        scores = torch.softmax(logits.gather(1, ids), dim=-1)
        by_expert: dict[int, list] = {}
        for f, row in enumerate(ids.tolist()):
            for slot, e in enumerate(row):
                by_expert.setdefault(e, []).append((f, scores[f, slot]))
        for e in range(c["E"], c["E"] + c["shared"]):
            by_expert[e] = [(f, torch.ones((), dtype=f64, device="cuda")) for f in range(c["F"])]
        total = torch.zeros_like(x)
        for e, uses in by_expert.items():
            w_up, w_down = _expert(st["up"], e, f64), _expert(st["down"], e, f64)
            f = torch.tensor([u[0] for u in uses], device="cuda")
            h = xn[f] @ w_up
            h = h if st["up_bias"] is None else h + st["up_bias"][e].double().flatten()
            g, l = h.chunk(2, dim=-1)
            g, l = torch.clamp(g, max=LIMIT), torch.clamp(l, -LIMIT, LIMIT)
            y = (g * torch.sigmoid(BETA * g) * (l + 1)) @ w_down
            y = y if st["down_bias"] is None else y + st["down_bias"][e].double()
            total.index_add_(0, f, torch.stack([u[1] for u in uses])[:, None] * y)
        return x + RESIDUAL * total, scores, ids
    V, k = c["V"], c["top_k"]
    rows: list[list] = [[], [], [], []]
    for n in range(0, c["N"], 128):                                                   # blocks of rows bound the memory
        x = st["logits"][n:n + 128, :V].double()
        t = st["targets"][n:n + 128]
        lp = torch.log_softmax(x, dim=-1)
        p = lp.exp()
        h = -(p * lp).sum(-1)
        rows[0].append(lp[torch.arange(x.shape[0], device="cuda"), t])
        rows[1].append(h)
        if c["grad"]:
            hot = torch.zeros_like(p)
            hot[torch.arange(x.shape[0], device="cuda"), t] = 1
            gl, gh = st["g_logprob"][n:n + 128].double()[:, None], st["g_entropy"][n:n + 128].double()[:, None]
            rows[2].append((gl * (hot - p) - gh * p * (lp + h[:, None])).float())       # 32 bits here: 64 would need twice the memory
        elif k:
            ids = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :k]
            rows[2].append(lp.gather(1, ids))
            rows[3].append(ids)
    if c["grad"]:
        return torch.cat(rows[0]), torch.cat(rows[1]), torch.cat(rows[2])
    empty = torch.zeros(c["N"], 0, device="cuda")
    return (torch.cat(rows[0]), torch.cat(rows[1]), torch.cat(rows[2]) if k else empty.double(), torch.cat(rows[3]) if k else empty.long())
