"""Attention over a shared prefix and own caches: the CPU path against one softmax over the concatenated keys in 64 bits, refusals; the
kernels against the same over heads, lengths, windows, cache types, strides and odd rows.

Tolerance of the kernels. The inputs are taken as they are (bf16, or e4m3 times its scale, which the kernels keep exact). A probability
is rounded to bf16 before the product with V: at most 2^-8 of it, so sum p |v| / L times 2^-8 in the output. Scores are fp32 sums of D
products, off by at most D * 2^-24 of sum |q k| * scale, and exp2 turns an error of a score into the same relative error of p, in the
numerator and in the denominator: twice ``score_error``; 2^-16 of sum p |v| / L covers the fp32 sums. The output is rounded once: 2^-8 of it."""

import pytest
import torch

from lyra_b200.nn.quant import QArray, dequantize, quantize
from lyra_b200.ops import api as ops

E4M3 = torch.float8_e4m3fn


def make(B, Nq, Nkv, T, P, S, D, prefix_quant=False, own_quant=False, sinks=True, device="cpu", seed=0, dtype=torch.bfloat16, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    cache = lambda q, *s: quantize(r(*s) * 2, E4M3, (1, D)) if q else r(*s).to(dtype)
    a = dict(q=(gain * r(B, Nq, T, D)).to(dtype), pk=cache(prefix_quant, Nkv, P, D), pv=cache(prefix_quant, Nkv, P, D), k=cache(own_quant, B, Nkv, S, D),
             v=cache(own_quant, B, Nkv, S, D), sinks=r(Nq) if sinks else None)
    return {key: (t.to(device) if t is not None else None) for key, t in a.items()}


def call(a, pos, window=0, scale=None, **kw):
    with torch.no_grad():
        return ops.prefix_attention(a["q"], a["pk"], a["pv"], a["k"], a["v"], a["sinks"], scale or a["q"].shape[-1] ** -0.5, window, pos, **kw)


def wide(t):
    return (t.qval.double() * t.scale.double()) if isinstance(t, QArray) else t.double()


def definition(a, pos, window=0, scale=None):
    """``(out, bound)`` sequence by sequence, over the visible keys alone."""
    q = a["q"].double()
    B, Nq, T, D = q.shape
    pk, pv, k, v = (wide(a[n]) for n in ("pk", "pv", "k", "v"))
    P, S, Nkv = pk.shape[1], k.shape[2], pk.shape[0]
    scale = scale or D ** -0.5
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        p0 = int(pos[b]) if isinstance(pos, torch.Tensor) and pos.numel() > 1 else int(pos)
        if p0 < 0:
            continue
        for t in range(T):
            at = P + p0 + t
            lo = max(0, at - window + 1) if window else 0
            end = min(p0 + t + 1, S)
            keys = torch.cat([pk[:, min(lo, P):], k[b][:, max(lo - P, 0):end]], dim=1).repeat_interleave(Nq // Nkv, 0)
            vals = torch.cat([pv[:, min(lo, P):], v[b][:, max(lo - P, 0):end]], dim=1).repeat_interleave(Nq // Nkv, 0)
            s = torch.einsum("nd,nsd->ns", q[b, :, t], keys) * scale
            mag = torch.einsum("nd,nsd->ns", q[b, :, t].abs(), keys.abs()) * scale
            full = torch.cat([s, a["sinks"].double()[:, None]], 1) if a["sinks"] is not None else s
            if full.shape[1] == 0:
                continue
            p = torch.softmax(full, dim=1)[:, : s.shape[1]]
            out[b, :, t] = torch.einsum("ns,nsd->nd", p, vals)
            weight = torch.einsum("ns,nsd->nd", p, vals.abs())
            score_error = (D * 2.0**-24 * mag.amax(1, keepdim=True) + 2.0**-20) if s.shape[1] else torch.zeros(Nq, 1, dtype=q.dtype, device=q.device)
            bound[b, :, t] = (2.0**-8 + 2 * score_error + 2.0**-16) * weight
    return out, bound + 2.0**-8 * (out.abs() + bound) + 1e-30


def rows(B, S, T, seed, device, idle=False):
    g = torch.Generator().manual_seed(seed)
    pos = torch.randint(0, S - T + 1, (B,), generator=g, dtype=torch.int32)
    pos[0] = S - T
    if B > 1:
        pos[1] = 0
    if idle and B > 2:
        pos[2] = -1
    return pos.to(device)


@pytest.mark.parametrize("window", [0, 5, 40])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("quant", [False, True])
def test_cpu_path_follows_the_definition(window, sinks, quant):
    a = make(4, 6, 2, 3, 21, 12, 8, prefix_quant=quant, sinks=sinks)
    pos = rows(4, 12, 3, 1, "cpu", idle=True)
    out = call({**a, "q": a["q"].double()}, pos, window)
    want, _ = definition(a, pos, window)
    # dequantize forms value * scale in fp32: 2^-24 of each key and value; scores (8 products below 10) shift by less than 1e-5
    assert (out - want).abs().max() < (1e-4 if quant else 1e-12)
    assert out[2].abs().max() == 0


def test_cpu_path_equals_attention_over_the_joined_cache():
    """The same keys as one prefix + own cache and as one long cache (decode attention): equal results."""
    a = make(2, 4, 2, 1, 9, 6, 8)
    joined = {n: torch.cat([a[p][None].expand(2, -1, -1, -1), a[n]], dim=2) for n, p in (("k", "pk"), ("v", "pv"))}
    got = call(a, 3)
    want = ops.decode_attention(a["q"], joined["k"], joined["v"], a["sinks"], 8 ** -0.5, 0, 9 + 3)
    assert (got.float() - want.float()).abs().max() <= 2 ** -8 * want.float().abs().max()


def test_cpu_empty_rows_and_masked_nan():
    a = make(2, 2, 1, 1, 0, 5, 8, sinks=False)
    a["k"][:, :, 3:] = float("nan")
    a["v"][:, :, 3:] = float("nan")
    assert torch.isfinite(call(a, 2)).all()
    none = make(2, 2, 1, 1, 0, 0, 8, sinks=False)
    assert call(none, torch.zeros(1, dtype=torch.int32)).abs().max() == 0


def test_refusals():
    a = make(2, 4, 2, 1, 6, 5, 8)

    def bad(pos=0, window=0, scale=None, **change):
        with pytest.raises(ValueError):
            call({**a, **change}, pos, window, scale)

    bad(q=a["q"][0])
    bad(pk=a["pk"][None])
    bad(pk=a["pk"][:, :5])
    bad(pk=a["pk"][:1], pv=a["pv"][:1])
    bad(k=a["k"][:1], v=a["v"][:1])
    bad(pk=quantize(a["pk"].float(), E4M3, (1, 8)))
    bad(pk=quantize(a["pk"].float(), E4M3, (2, 8)), pv=quantize(a["pv"].float(), E4M3, (2, 8)))
    bad(sinks=a["sinks"][:3])
    bad(pos=5)
    bad(window=-1)
    bad(scale=-1.0)
    bad(pos=torch.zeros(3, dtype=torch.int32))
    bad(pos=torch.zeros(2))
    with pytest.raises(ValueError):
        ops.prefix_attention(a["q"].float().requires_grad_(), a["pk"], a["pv"], a["k"], a["v"], a["sinks"], 1.0, 0, 0)
    with pytest.raises(ValueError):
        call(a, 0, implementation="b200")


def check_numbers_of_other_types(device):
    """A window beyond any 32-bit number or written as a float, a position far below zero; a position that is no integer is refused."""
    a = make(2, 2, 1, 1, 40, 30, 64, device=device)
    everything = call(a, 3, 0)
    assert torch.equal(call(a, 3, 2**32 + 5), everything) and torch.equal(call(a, 3, 70.0), everything)
    assert torch.equal(call(a, 3, 9.0), call(a, 3, 9)) and not torch.equal(call(a, 3, 9), everything)
    assert call(a, -2**32, 0).abs().max() == 0
    for pos in (1.0, 2.5, None):
        with pytest.raises(ValueError):
            call(a, pos)


def test_numbers_of_other_types_cpu():
    check_numbers_of_other_types("cpu")


# --------------------------------------------------------------------------- GPU
@pytest.mark.gpu
def test_numbers_of_other_types_gpu():
    check_numbers_of_other_types("cuda")


def check(a, pos, window=0, scale=None):
    from lyra_b200.ops import native

    out = call(a, pos, window, scale)
    native.check_status()
    want, bound = definition(a, pos, window, scale)
    assert out.shape == want.shape and out.dtype == torch.bfloat16
    err = (out.double() - want).abs()
    assert (err <= bound).all(), (float((err / bound).max()), int((err > bound).sum()))
    assert torch.equal(call(a, pos, window, scale), out)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("B,Nq,Nkv,D,T,P,S", [
    (1, 4, 2, 64, 1, 1, 1), (3, 16, 4, 128, 1, 127, 40), (2, 64, 8, 64, 1, 128, 300), (5, 12, 4, 64, 1, 129, 33), (4, 10, 2, 128, 1, 1000, 17), (40, 32, 8, 128, 1, 700, 70),
    (17, 64, 8, 64, 1, 2500, 600), (2, 16, 16, 64, 1, 300, 9), (2, 40, 2, 64, 1, 260, 50), (3, 16, 4, 128, 2, 400, 30), (2, 64, 8, 64, 24, 333, 24),
    (3, 32, 8, 128, 7, 140, 500), (2, 12, 4, 64, 40, 64, 90), (1, 8, 8, 64, 100, 129, 260)])
def test_shapes_gpu(B, Nq, Nkv, D, T, P, S, quant):
    a = make(B, Nq, Nkv, T, P, S, D, quant, quant, device="cuda", seed=P + S)
    check(a, rows(B, S, T, P, "cuda", idle=True))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 16, 128, 1000])
@pytest.mark.parametrize("T", [1, 9])
def test_windows_gpu(window, T):
    """Windows inside the own cache, across the border into the prefix, and wider than both; each sequence has its own border."""
    a = make(6, 16, 4, T, 391, 150, 64, device="cuda", seed=window)
    check(a, rows(6, 150, T, window, "cuda"), window)
    check(make(3, 16, 4, T, 391, 150, 128, True, False, sinks=False, device="cuda"), rows(3, 150, T, 2, "cuda"), window)


@pytest.mark.gpu
@pytest.mark.parametrize("kinds", [(False, True), (True, False)])
def test_prefix_and_own_cache_of_different_types_gpu(kinds):
    check(make(3, 16, 4, 1, 300, 77, 128, *kinds, device="cuda"), rows(3, 77, 1, 5, "cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("P,S", [(0, 64), (200, 0), (0, 0)])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("T", [1, 20])
def test_empty_sides_gpu(P, S, sinks, T):
    a = make(3, 8, 2, T, P, S, 64, sinks=sinks, device="cuda")
    pos = torch.tensor([0, max(S - T, 0), -1], dtype=torch.int32, device="cuda")
    out = check(a, pos)
    assert out[2].abs().max() == 0
    if P == S == 0:
        assert out.abs().max() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("gain", [0.0, 30.0])
def test_flat_and_sharp_scores_gpu(quant, gain):
    check(make(3, 16, 4, 1, 1500, 60, 64, quant, quant, device="cuda", gain=gain), rows(3, 60, 1, 7, "cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
def test_scores_far_from_zero_and_rising_gpu(quant):
    """All scores around -400 (a reference of zero would lose every probability), and scores that rise by hundreds along the prefix (the
    running maximum moves in every tile)."""
    B, Nq, Nkv, P, S, D = 2, 8, 2, 900, 40, 64
    a = make(B, Nq, Nkv, 1, P, S, D, sinks=False, device="cuda")
    a["q"][..., 0] = 40.0
    for n, sign in (("pk", -1.0), ("k", -1.0)):
        a[n][..., 0] = sign * 80.0
    pos = rows(B, S, 1, 1, "cuda")
    pack = lambda t: quantize(t.float(), E4M3, (1, D)) if quant else t
    b = {n: (pack(t) if n in ("pk", "pv", "k", "v") else t) for n, t in a.items()}
    check(b, pos)
    a["pk"][..., 0] = torch.linspace(-80, 80, P, device="cuda")
    b = {n: (pack(t) if n in ("pk", "pv", "k", "v") else t) for n, t in a.items()}
    check(b, pos)


@pytest.mark.gpu
def test_places_that_are_not_visible_are_not_read_gpu():
    """NaN behind each sequence's last position, behind the prefix in its buffer, and before a window that no sequence reaches."""
    B, Nq, Nkv, P, S, D = 4, 16, 4, 500, 96, 64
    a = make(B, Nq, Nkv, 1, P, S, D, device="cuda")
    pos = rows(B, S, 1, 3, "cuda")
    for b in range(B):
        a["k"][b, :, int(pos[b]) + 1:] = float("nan")
        a["v"][b, :, int(pos[b]) + 1:] = float("nan")
    buffers = {}
    for n in ("pk", "pv"):
        buf = torch.full((1, Nkv, P + 100, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        buf[0, :, :P] = a[n]
        buffers[n] = buf
    clean = {**a, "k": a["k"].nan_to_num(0.0), "v": a["v"].nan_to_num(0.0)}
    views = {**a, **{n: buffers[n][0, :, :P] for n in buffers}}
    assert torch.equal(call(views, pos), call(clean, pos))
    window = 100
    for n in buffers:
        buffers[n][0, :, : P - window + 1] = float("inf")
    assert torch.equal(call(views, pos, window), call(clean, pos, window))
    assert torch.isfinite(call(views, pos, window)).all()


@pytest.mark.gpu
def test_layouts_and_positions_gpu():
    """Strided queries and prefixes, bases off the 16-byte boundary, an int position, one device value, int64 positions."""
    B, Nq, Nkv, T, P, S, D = 3, 16, 4, 2, 300, 50, 64
    a = make(B, Nq, Nkv, T, P, S, D, device="cuda")
    pos = rows(B, S, T, 4, "cuda")
    want = call(a, pos)
    q = a["q"].transpose(1, 2).contiguous().transpose(1, 2)
    wide_q = torch.zeros(B, T, 3 * Nq * D, dtype=torch.bfloat16, device="cuda")
    wide_q[:, :, Nq * D:2 * Nq * D] = q.transpose(1, 2).reshape(B, T, -1)
    fused = wide_q[:, :, Nq * D:2 * Nq * D].view(B, T, Nq, D).transpose(1, 2)
    odd = torch.zeros(a["pk"].numel() + 3, dtype=torch.bfloat16, device="cuda")[3:].view_as(a["pk"]).copy_(a["pk"])
    token_major = a["pk"].transpose(0, 1).contiguous().transpose(0, 1)
    for change in ({"q": q}, {"q": fused}, {"pk": odd}, {"pk": token_major}, {"k": a["k"].transpose(1, 2).contiguous().transpose(1, 2)}):
        assert torch.equal(call({**a, **change}, pos), want)
    assert torch.equal(call(a, pos.long()), want)
    one = call(a, torch.full((B,), 7, dtype=torch.int32, device="cuda"))
    assert torch.equal(call(a, 7), one) and torch.equal(call(a, torch.tensor(7, dtype=torch.int32, device="cuda")), one)
    e8 = make(B, Nq, Nkv, T, P + 20, S, D, True, True, device="cuda")
    cut = {n: QArray(e8[n].qval[:, :P], e8[n].scale[:, :P], (1, D)) for n in ("pk", "pv")}
    packed = {n: QArray(t.qval.contiguous(), t.scale.contiguous(), t.block) for n, t in cut.items()}
    assert torch.equal(call({**e8, **cut}, pos), call({**e8, **packed}, pos))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(a, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)


@pytest.mark.gpu
def test_refusals_gpu():
    a = make(2, 4, 2, 1, 6, 5, 32, device="cuda")
    with pytest.raises(ValueError):
        call(a, 0)                                             # head dim
    a = make(2, 4, 2, 1, 6, 5, 64, device="cuda")
    for change in ({"pk": a["pk"].float(), "pv": a["pv"].float()}, {"k": a["k"].half(), "v": a["v"].half()}, {"sinks": a["sinks"].cpu()}):
        with pytest.raises(ValueError):
            call({**a, **change}, 0)


@pytest.mark.gpu
def test_replay_with_other_positions_gpu():
    a = make(3, 16, 4, 1, 300, 64, 128, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    want = []
    for step in (0, 5, 63):
        pos.fill_(step)
        want.append(call(a, pos).clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(a, pos)
    for step, w in zip((0, 5, 63), want):
        pos.fill_(step)
        graph.replay()
        assert torch.equal(out, w)
