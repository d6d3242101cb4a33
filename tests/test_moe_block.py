"""The one-kernel mixture-of-experts block: the CPU path against the definition in 64 bits, refusals, the arithmetic of the
kernel's unit runs; the kernel against the definition over token counts, widths, expert counts, weight types and odd routings.

Tolerances of the kernel. Three roundings to bf16, each at most 2^-8 relative (half a step): of x * norm, of the SwiGLU result, of
the output. ``bound`` carries them through the block as intervals (every term off in the worst direction) and adds 2^-16 of the sums'
magnitudes for fp32 accumulation (up to 2^8 terms in a row per accumulator). As errors of one sign are not what happens, the
relative root mean square error is held to 3 * 2^-8 as well: one 2^-8 for each rounding, whose error in a sum of independent terms
has at most the relative size in the mean square that it has in each term. Router logits see no rounding: scores to 2^-18."""

import math

import pytest
import torch

from lyra_b200.nn.quant import QArray, dequantize, quantize
from lyra_b200.ops import api as ops

E4M3 = torch.float8_e4m3fn
BETA, LIMIT, EPS = 1.702, 7.0, 1e-5


def make(F, C, H, E, k, shared, bias=True, quant=False, device="cpu", seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    n = E + shared
    a = dict(x=r(F, C).to(dtype), norm=1 + 0.1 * r(C), router=r(C, E) / math.sqrt(C), router_bias=0.1 * r(E) if bias else None,
             up=r(n, C, 2, H) / math.sqrt(C), up_bias=0.1 * r(n, 2, H) if bias else None, down=r(n, H, C) / math.sqrt(H),
             down_bias=0.1 * r(n, C) if bias else None)
    if quant:
        a["up"] = quantize(a["up"].reshape(n, C, 2 * H), E4M3, (math.gcd(C, 256), math.gcd(2 * H, 256)))
        a["down"] = quantize(a["down"], E4M3, (math.gcd(H, 256), math.gcd(C, 256)))
    else:
        a["up"], a["down"] = a["up"].to(dtype), a["down"].to(dtype)
    return {key: (v.to(device) if v is not None else None) for key, v in a.items()}


def call(a, k, shared, rs=4.0, **kw):
    return ops.moe_block(a["x"], a["norm"], EPS, a["router"], a["router_bias"], a["up"], a["up_bias"], a["down"], a["down_bias"], k, shared, BETA, LIMIT, rs, **kw)


def wide(w, n, C, H):
    up = dequantize(w, torch.float32) if isinstance(w, QArray) else w
    return up.double()


def definition(a, k, shared, rs=4.0):
    """``(out, scores, idx, bound)`` in 64 bits by token and expert; ``bound`` is the interval of the kernel's roundings."""
    x = a["x"].double()
    F, C = x.shape
    up, down = wide(a["up"], 0, 0, 0), wide(a["down"], 0, 0, 0)
    n, H = down.shape[0], down.shape[1]
    up = up.reshape(n, C, 2 * H)
    E = n - shared
    xn = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * a["norm"].double()
    logits = xn @ a["router"].double() + (a["router_bias"].double() if a["router_bias"] is not None else 0)
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    idx, scores = order.indices[:, :k], torch.softmax(order.values[:, :k], dim=-1)
    half, acc = 2.0**-8, 2.0**-16
    out, bound = x.clone(), torch.zeros_like(x)
    for f in range(F):
        for e, s in [*zip(idx[f].tolist(), scores[f].tolist()), *((E + i, 1.0) for i in range(shared))]:
            t = xn[f] @ up[e]
            err_t = (half + acc) * (xn[f].abs() @ up[e].abs())
            if a["up_bias"] is not None:
                t = t + a["up_bias"][e].reshape(-1).double()
            g, l = t[:H].clamp(max=LIMIT), t[H:].clamp(-LIMIT, LIMIT)
            act = (l + 1) * g * torch.sigmoid(BETA * g)
            # |d(g sigmoid(b g))/dg| <= 1.1 everywhere; the product of both errors is second order and kept
            err = err_t[H:] * (g * torch.sigmoid(BETA * g)).abs() + 1.1 * err_t[:H] * ((l + 1).abs() + err_t[H:])
            err = err + half * (act.abs() + err)
            y = act @ down[e]
            err_y = err @ down[e].abs() + acc * (act.abs() @ down[e].abs())
            if a["down_bias"] is not None:
                y = y + a["down_bias"][e].double()
            out[f] += rs * s * y
            bound[f] += abs(rs) * s * err_y + 2.0**-18 * (rs * s * y).abs()
    bound = bound + half * (out.abs() + bound)
    return out, scores, idx, bound


def test_cpu_path_follows_the_definition():
    for quant in (False, True):
        a = make(5, 48, 32, 6, 3, 1, quant=quant)
        out, scores, idx = call(a, 3, 1)
        want, s, i, _ = definition(a, 3, 1)
        assert out.dtype == torch.bfloat16 and torch.equal(idx, i)
        assert (scores - s).abs().max() < 1e-6
        assert ((out.double() - want).abs() <= 2**-8 * want.abs() + 1e-4).all()      # one rounding at the end, the rest in fp32


def test_cpu_path_ties_take_the_lower_expert():
    a = make(3, 16, 16, 5, 2, 0)
    a["router"].zero_()
    a["router_bias"].zero_()
    _, scores, idx = call(a, 2, 0)
    assert idx.tolist() == [[0, 1]] * 3 and torch.equal(scores, torch.full((3, 2), 0.5))


def test_refusals():
    a = make(2, 16, 16, 4, 2, 1)

    def bad(k=2, shared=1, **change):
        with pytest.raises(ValueError):
            call({**a, **change}, k, shared)

    bad(k=0)
    bad(k=5)
    bad(shared=5)
    bad(x=a["x"][0])
    bad(norm=a["norm"][:8])
    bad(router=a["router"][:, :3])
    bad(router_bias=a["router_bias"][:3])
    bad(up=a["up"].reshape(5, 16, 32))
    bad(up_bias=a["up_bias"][:, :1])
    bad(down=a["down"][:4])
    bad(down_bias=a["down_bias"].reshape(16, 5))
    bad(up=QArray(a["up"].reshape(5, 16, 32).to(E4M3), torch.ones(5, 1, 1), (16, 16)))
    bad(x=a["x"].float().requires_grad_())
    with pytest.raises(ValueError):
        call(a, 2, 1, implementation="b200")


@pytest.mark.parametrize("U", [1, 2, 7, 63, 147, 148, 149, 1000, 8100, 123457])
@pytest.mark.parametrize("G", [1, 2, 5, 64, 148])
@pytest.mark.parametrize("per", [1, 3, 45])
def test_unit_runs(U, G, per):
    """The kernel's bookkeeping restated: contiguous runs cover every unit once, ``owner`` finds them, the CTAs ``first .. last`` that the
    last arriver of a panel waits for all have a part of it, and no CTA needs a third slot for a cut panel."""
    U = U * per
    size, rem = U // G, U % G
    begin = [c * size + min(c, rem) for c in range(G + 1)]
    wide = rem * (size + 1)
    owner = lambda u: u // (size + 1) if u < wide else rem + (u - wide) // size
    assert begin[0] == 0 and begin[G] == U
    for u in range(0, U, max(1, U // 997)):
        c = owner(u)
        assert begin[c] <= u < begin[c + 1]
    cut = {c: [] for c in range(G)}
    for q in range(0, U // per, max(1, U // per // 499)):
        for c in range(owner(q * per), owner(q * per + per - 1) + 1):
            assert begin[c] < (q + 1) * per and q * per < begin[c + 1] and begin[c] != begin[c + 1]
            if not (begin[c] <= q * per and (q + 1) * per <= begin[c + 1]):
                cut[c].append(0 if begin[c] >= q * per else 1)
                assert (begin[c] // per == q) == (cut[c][-1] == 0)
    assert all(len(slots) == len(set(slots)) <= 2 for slots in cut.values())


# --------------------------------------------------------------------------- GPU
def check(a, k, shared, rs=4.0):
    from lyra_b200.ops import native

    with torch.no_grad():
        out, scores, idx = call(a, k, shared, rs)
        native.check_status()
    want, s, i, bound = definition(a, k, shared, rs)
    assert torch.equal(idx, i)
    assert (scores - s).abs().max() < 2**-18
    err = (out.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    assert err.norm() <= 3 * 2**-8 * want.norm(), float(err.norm() / want.norm())
    with torch.no_grad():
        again = call(a, k, shared, rs)
    assert torch.equal(again[0], out) and torch.equal(again[1], scores)       # the result does not depend on which CTA came last
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("F,C,H,E,k,shared,bias", [
    (1, 16, 16, 4, 1, 0, True), (1, 256, 512, 4, 2, 1, False), (2, 80, 48, 7, 2, 1, True), (8, 512, 208, 15, 3, 1, False), (9, 272, 400, 5, 2, 0, True),
    (17, 128, 64, 3, 1, 2, True), (33, 144, 1008, 9, 4, 4, False), (64, 1040, 80, 4, 4, 0, True), (64, 512, 512, 256, 8, 0, True), (5, 2880, 320, 32, 4, 0, True)])
def test_shapes_gpu(F, C, H, E, k, shared, bias, quant):
    if E + shared > 256:
        pytest.skip("too many experts")
    check(make(F, C, H, E, k, shared, bias, quant, "cuda", seed=F + C), k, shared)


@pytest.mark.gpu
@pytest.mark.parametrize("C,H", [(8, 8), (24, 40), (264, 72), (1000, 712)])
def test_widths_off_the_tile_gpu(C, H):
    check(make(6, C, H, 5, 2, 1, True, False, "cuda", seed=C), 2, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("F", [1, 7, 8, 16, 24, 32, 40, 63, 64])
@pytest.mark.parametrize("quant", [False, True])
def test_all_tokens_on_one_expert_gpu(F, quant):
    a = make(F, 160, 96, 6, 1, 0, True, quant, "cuda", seed=F)
    a["router_bias"][4] = 50.0
    check(a, 1, 0)


@pytest.mark.gpu
def test_odd_routings_gpu():
    """Equal logits, masked experts, tokens of zeros; a token of NaN spoils its own row only."""
    a = make(6, 64, 64, 5, 2, 0, True, False, "cuda")
    a["router"].zero_()
    a["router_bias"].zero_()
    check(a, 2, 0)
    a["router_bias"][0] = float("-inf")
    a["router_bias"][3] = torch.finfo(torch.float32).min
    check(a, 2, 0)
    a = make(6, 64, 64, 5, 2, 1, True, False, "cuda")
    a["x"][3].zero_()
    check(a, 2, 1)
    with torch.no_grad():
        clean, _, _ = call(a, 2, 1)
        a["x"][2, 5] = float("nan")
        spoilt, scores, idx = call(a, 2, 1)
    others = [0, 1, 3, 4, 5]
    assert torch.isnan(spoilt[2]).all() and torch.isnan(scores[2]).all() and idx[2].tolist() == [0, 1]
    assert torch.equal(spoilt[others], clean[others])


@pytest.mark.gpu
def test_weights_of_experts_nobody_chose_are_not_looked_at_gpu():
    a = make(4, 64, 48, 6, 1, 0, True, False, "cuda")
    a["router_bias"][2] = 40.0
    for e in (0, 1, 3, 4, 5):
        a["up"][e] = float("nan")
        a["down"][e] = float("inf")
    with torch.no_grad():
        out, _, idx = call(a, 1, 0)
    assert (idx == 2).all() and torch.isfinite(out).all()


@pytest.mark.gpu
def test_every_e4m3_code_gpu():
    """All 254 numbers of the format as weights of the up-projection (one column each) against their values. The NaN code is kept: it
    makes its hidden unit NaN, and that every output (the down-projection is dense, 0 * NaN = NaN)."""
    C, H = 16, 256
    a = make(1, C, H, 1, 1, 0, False, False, "cuda")
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes[codes % 128 == 127] = 0
    up = torch.zeros(1, C, 2 * H, dtype=torch.uint8, device="cuda")
    up[0, 3, H:] = codes                                                   # linear half: one non-zero input row
    up[0, :, :H] = torch.full((), 0.5, device="cuda").to(E4M3).view(torch.uint8)
    down = torch.zeros(1, H, C, device="cuda")

    def run():
        b = {**a, "up": QArray(up.view(E4M3), torch.ones(1, 1, 1, device="cuda"), (C, 2 * H)), "down": quantize(down, E4M3, (16, 16))}
        with torch.no_grad():
            return ops.moe_block(b["x"], b["norm"], EPS, b["router"], None, b["up"], None, b["down"], None, 1, 0, BETA, 1e4, 1.0)[0]

    x = a["x"].double()
    xn = x / torch.sqrt((x * x).mean() + EPS) * a["norm"].double()
    w = up.view(E4M3).double()[0]
    t, size = (xn @ w)[0], (xn.abs() @ w.abs())[0]
    act = (t[H:] + 1) * t[:H] * torch.sigmoid(BETA * t[:H])
    for start in range(0, H, C):
        down.zero_()
        for c in range(C):
            down[0, start + c, c] = 1.0
        magnitude = x[0].abs() + (size[H:] + 1)[start:start + C] * size[0] * 1.1
        assert ((run()[0].double() - (x[0] + act[start:start + C])).abs() <= 4 * 2**-8 * magnitude).all()
    for code in (127, 255):
        up[0, 5, H + 17] = code
        assert torch.isnan(run()).all()
        up[0, 5, H + 17] = 0
    assert torch.isfinite(run()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("beta,limit", [(1e-4, 1000.0), (2.8e-5, 7.0), (1.702, 0.0)])
def test_hidden_units_of_any_size_with_e4m3_weights_gpu(beta, limit):
    """Gates far below zero under a small beta make hidden units of up to 0.2785 (limit + 1) / beta, beyond fp16 unless they are scaled.
    The weights copy hidden units to the output one by one. Tolerance: the gate and the linear half carry the rounding of x * norm to fp16
    (2^-11, as do both products with their sums of one term) and the hidden unit, fp16 after a power of two, 2^-11 of itself or half a step
    of the smallest size, 2^-25 times that power (bound / 60000, rounded up); the output 2^-8 of itself. |d(g sigmoid(b g)) / dg| <= 1.1."""
    C, H = 16, 16
    a = make(1, C, H, 1, 1, 0, False, False, "cuda")
    x = torch.linspace(-2.0, 2.0, C, device="cuda").to(torch.bfloat16)[None]
    eye = torch.eye(C, device="cuda")
    up = torch.cat([eye, eye], 1)[None].to(E4M3)
    for gate_scale in (1.0, 1 / beta):
        for linear_scale in (1.0, max(limit, 1.0)):
            scale = torch.tensor([[[gate_scale, linear_scale]]], device="cuda")
            w_up = QArray(up, scale, (16, 16))
            w_down = QArray(eye[None].to(E4M3), torch.ones(1, 1, 1, device="cuda"), (16, 16))
            with torch.no_grad():
                out = ops.moe_block(x, a["norm"], EPS, a["router"], None, w_up, None, w_down, None, 1, 0, beta, limit, 1.0)[0]
            xd = x.double()
            xn = xd / torch.sqrt((xd * xd).mean() + EPS) * a["norm"].double()
            g, l = (xn * gate_scale).clamp(max=limit), (xn * linear_scale).clamp(-limit, limit)
            s = g * torch.sigmoid(beta * g)
            act = (l + 1) * s
            step = 2.0**-11 * 1.05
            err = (step * (xn * linear_scale).abs()) * s.abs() + 1.1 * step * (xn * gate_scale).abs() * ((l + 1).abs() * 1.001 + 1e-3)
            top = (limit + 1) * max(limit, 0.279 / beta)
            err = err + step * act.abs() + 2.0**-25 * max(1.0, 2 * top / 60000)
            err = err + 2.0**-8 * ((xd + act).abs() + err)
            assert ((out.double() - (xd + act)).abs() <= err).all(), ((out.double() - (xd + act)).abs() / err).max()


@pytest.mark.gpu
def test_sizes_of_hidden_units_that_are_refused_gpu():
    from lyra_b200.ops import decode

    a = make(2, 64, 48, 6, 2, 1, True, True, "cuda")
    for beta, limit in ((0.0, 7.0), (-1.0, 7.0), (1e-6, 7.0), (1.702, 2e4), (1.702, -1.0), (float("nan"), 7.0)):
        with pytest.raises(ValueError), torch.no_grad():
            ops.moe_block(a["x"], a["norm"], EPS, a["router"], a["router_bias"], a["up"], a["up_bias"], a["down"], a["down_bias"], 2, 1, beta, limit, 1.0)
        assert not decode.moe_block_supported(2, 64, 48, 6, 1, 2, a["up"], a["down"], beta, limit)


@pytest.mark.gpu
def test_refusals_and_layouts_gpu():
    from lyra_b200.ops import decode

    a = make(4, 64, 48, 6, 2, 1, True, False, "cuda")
    with torch.no_grad():
        want = call(a, 2, 1)[0]
        big = torch.zeros(4, 130, dtype=torch.bfloat16, device="cuda")
        big[:, 3:67] = a["x"]
        assert torch.equal(call({**a, "x": big[:, 3:67]}, 2, 1)[0], want)                     # strided, off the 16-byte boundary
        masters = {**a, "up": a["up"].float(), "down": a["down"].float()}
        assert torch.equal(call(masters, 2, 1)[0], want)                                       # fp32 masters through their bf16 copies
        out, scores, idx = call({**a, "x": a["x"][:0]}, 2, 1)
        assert out.shape == (0, 64) and idx.shape == (0, 2)
        for change in ({"x": a["x"].float()}, {"x": a["x"].repeat(17, 1)}, {"down": quantize(a["down"], E4M3, (16, 16))}):
            with pytest.raises(ValueError):
                call({**a, **change}, 2, 1)
    narrow = make(2, 20, 16, 4, 1, 0, device="cuda")
    with pytest.raises(ValueError), torch.no_grad():
        call(narrow, 1, 0)
    assert not decode.moe_block_supported(65, 64, 64, 4, 0, 1, a["up"], a["down"])
    assert not decode.moe_block_supported(1, 64, 64, 16, 0, 9, a["up"], a["down"])


@pytest.mark.gpu
def test_two_streams_and_graphs_gpu():
    """Workspaces are a call's own: two captured graphs replayed at the same time on two streams give what eager calls give."""
    inputs = [make(3, 256, 128, 8, 2, 1, True, False, "cuda", seed=s) for s in (1, 2)]
    graphs, outs = [], []
    with torch.no_grad():
        want = [call(a, 2, 1)[0].clone() for a in inputs]
        torch.cuda.synchronize()
        for a in inputs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(call(a, 2, 1)[0])
            graphs.append(g)
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(20):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
