"""Scores of given tokens: the CPU path against the definition in 64 bits and against differences, refusals; the kernel against
the definition in 64 bits over types, alignments, row counts (one to several CTAs per row) and rows where it can go wrong.

Tolerances. Forward: every term of s = sum e^{x-m} carries the error of the subtraction and of exp2 (2 ulp) plus the summation
(a thread adds fewer than 4096 terms, the tree 20 more levels): relative 4096 * 2^-24 / 2 worst case, about 1.3e-4 if all errors
had one sign; they do not, and the tests use shapes with at most 512 terms per thread: 512 * 2^-24 = 3.1e-5 for log s, and the
same times the largest |x - m| that still has weight (below 20) for the entropy: 6.1e-4; plus half an ulp of the result.
Gradient: see the test."""

import math

import pytest
import torch

from lyra_b200.ops import api as ops

NAN = float("nan")
INF = float("inf")


def exact(logits, targets, k, vocab):
    x = logits[..., :vocab].double()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    p = e / e.sum(-1, keepdim=True)
    logp = (x - m) - torch.log(e.sum(-1, keepdim=True))
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    picked = logp.gather(-1, targets.long().clamp(0, vocab - 1)[..., None])[..., 0]
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :k]
    return picked, entropy, logp.gather(-1, order), order, p, logp


def exact_gradient(logits, targets, vocab, gl, gh):
    _, entropy, _, _, p, logp = exact(logits, targets, 0, vocab)
    gl = torch.where(targets < 0, torch.zeros_like(gl), gl).double()[..., None]
    gh = gh.double()[..., None]
    hot = torch.zeros_like(p).scatter_(-1, targets.long().clamp(0, vocab - 1)[..., None], 1.0)
    g = gl * (hot - p) - gh * p * (torch.where(p > 0, logp, torch.zeros_like(logp)) + entropy[..., None])
    return torch.cat([g, g.new_zeros(*g.shape[:-1], logits.shape[-1] - vocab)], dim=-1)


def test_cpu_path_follows_the_definition():
    torch.manual_seed(0)
    logits = torch.randn(3, 5, 70, dtype=torch.float64) * 3
    logits[0, 0, 7] = -INF
    targets = torch.randint(0, 64, (3, 5))
    r = ops.token_logprobs(logits, targets, 6, vocab_size=64)
    lp, h, top, ids, _, _ = exact(logits, targets, 6, 64)
    assert torch.equal(r.top_ids, ids)
    for got, want in ((r.logprob, lp), (r.entropy, h), (r.top_logprobs, top)):
        assert (got - want).abs().max() < 1e-12


def test_cpu_gradient_against_formula_and_differences():
    torch.manual_seed(1)
    logits = (torch.randn(4, 19, dtype=torch.float64) * 2).requires_grad_()
    targets = torch.tensor([3, 0, -1, 11])
    gl, gh = torch.randn(4, dtype=torch.float64), torch.randn(4, dtype=torch.float64)

    def objective(x):
        r = ops.token_logprobs(x, targets, 0, vocab_size=17)
        return (r.logprob * gl + r.entropy * gh).sum()

    (g,) = torch.autograd.grad(objective(logits), logits)
    assert (g - exact_gradient(logits.detach(), targets, 17, gl, gh)).abs().max() < 1e-12
    step = 1e-6
    for i in range(4):
        for v in (0, 3, 11, 16, 18):
            d = torch.zeros_like(logits)
            d[i, v] = step
            slope = (objective(logits.detach() + d) - objective(logits.detach() - d)) / (2 * step)
            assert abs(float(slope - g[i, v])) < 1e-7
    assert g[2].abs().max() > 0 and g[:, 17:].abs().max() == 0


def edge_rows():
    """Rows where a softmax goes wrong, their targets, and what logprob and entropy have to be (None: the definition)."""
    V = 40
    base = torch.linspace(-3, 3, V)
    low = torch.finfo(torch.float32).min
    rows = [base, torch.full((V,), low), torch.full((V,), -INF), base.clone(), base.clone(), base.clone(), base.clone(), torch.full((V,), -INF), base.clone(),
            base.clone(), torch.full((V,), 7.25)]
    rows[3][5] = NAN
    rows[4][5] = INF
    rows[5][:30] = -INF
    rows[6][:30] = low
    rows[7][9] = 1.5
    targets = torch.tensor([2, 3, 4, 5, 6, 2, 35, 9, -100, V, 39])
    return torch.stack(rows), targets


def check_edges(device):
    logits, targets = edge_rows()
    V = logits.shape[1]
    x = logits.to(device).requires_grad_()
    r = ops.token_logprobs(x, targets.to(device), 3)
    lp, h = r.logprob.detach().cpu().double(), r.entropy.detach().cpu().double()
    want, want_h, top, ids, _, _ = exact(logits, targets, 3, V)
    for i in (0, 1, 5, 6, 7, 8, 9, 10):                       # rows with a distribution
        assert abs(float(h[i] - want_h[i])) < 1e-5, i
        assert torch.equal(r.top_ids[i].cpu(), ids[i]), i
        a, b = r.top_logprobs[i].cpu().double(), top[i]
        assert torch.equal(torch.isinf(a), torch.isinf(b)) and (torch.isinf(a) | ((a - b).abs() < 1e-5)).all(), i
    for i in (0, 1, 6, 7, 10):
        assert abs(float(lp[i] - want[i])) < 1e-5, i
    assert lp[5] == -INF and lp[8] == 0 and torch.isnan(lp[9])
    for i in (2, 3, 4):
        assert torch.isnan(lp[i]) and torch.isnan(h[i]) and torch.isnan(r.top_logprobs[i]).all()
    assert r.top_ids[3].tolist()[:2] == [5, 39] and r.top_ids[4].tolist()[:2] == [5, 39] and r.top_ids[2].tolist() == [0, 1, 2]
    good = torch.tensor([0, 1, 6, 7, 8, 10])
    (g,) = torch.autograd.grad((r.logprob + r.entropy)[good.to(device)].sum(), x)
    ones = torch.ones(len(good))
    want_g = exact_gradient(logits[good], targets[good], V, ones, ones)
    assert (g[good.to(device)].cpu().double() - want_g).abs().max() < 1e-5


def test_edges_on_the_cpu():
    check_edges("cpu")


def test_refusals():
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.long)
    for bad in (lambda: ops.token_logprobs(x, t[:1]), lambda: ops.token_logprobs(x, t.float()), lambda: ops.token_logprobs(x, t, 9),
                lambda: ops.token_logprobs(x, t, -1), lambda: ops.token_logprobs(x, t, vocab_size=9), lambda: ops.token_logprobs(x, t, vocab_size=0),
                lambda: ops.token_logprobs(torch.zeros(2, 64), t, 33), lambda: ops.token_logprobs(x, t, implementation="b200")):
        with pytest.raises(ValueError):
            bad()


def test_no_rows():
    r = ops.token_logprobs(torch.zeros(0, 8), torch.zeros(0, dtype=torch.long), 2)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 2)


# --------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,pad,k", [(1, 1, 0, 1), (3, 2, 5, 2), (1, 201088, 0, 20), (5, 65537, 0, 32), (1, 100003, 1, 5), (2, 131, 3, 32), (160, 20011, 0, 4),
                                       (40, 33001, 7, 1), (80, 40000, 0, 7), (400, 1000, 24, 3)])
def test_forward_gpu(dtype, N, V, pad, k):
    torch.manual_seed(V + N)
    buf = (torch.randn(N, V + pad, device="cuda") * 3).to(dtype)
    buf[:, V:] = NAN                                           # padding columns must not be looked at
    targets = torch.randint(0, V, (N,), device="cuda")
    r = ops.token_logprobs(buf, targets, k, vocab_size=V)
    lp, h, top, ids, _, _ = exact(buf, targets, k, V)
    assert torch.equal(r.top_ids, ids)
    assert (r.logprob - lp).abs().max() < 3.1e-5 + 2**-24 * 40
    assert (r.top_logprobs - top).abs().max() < 3.1e-5 + 2**-24 * 40
    assert (r.entropy - h).abs().max() < 6.1e-4
    again = ops.token_logprobs(buf, targets, k, vocab_size=V)
    assert all(torch.equal(a, b) for a, b in zip(r, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 30, 200])
@pytest.mark.parametrize("kind", ["constant", "few values", "ascending", "descending"])
def test_alternatives_of_tied_and_sorted_rows_gpu(dtype, N, kind):
    """Many equal logits overflow the candidate buffer (the slow selection), sorted rows are the worst case of a running list."""
    torch.manual_seed(3)
    V, k = 50021, 11
    x = {"constant": torch.zeros(N, V), "few values": torch.randint(0, 3, (N, V)).float(), "ascending": torch.linspace(-9, 9, V).expand(N, V),
         "descending": torch.linspace(9, -9, V).expand(N, V)}[kind].to(dtype).contiguous().cuda()
    targets = torch.arange(N, device="cuda")
    r = ops.token_logprobs(x, targets, k)
    lp, h, top, ids, _, _ = exact(x, targets, k, V)
    assert torch.equal(r.top_ids, ids)
    assert (r.top_logprobs - top).abs().max() < 3.2e-5 and (r.logprob - lp).abs().max() < 3.2e-5 and (r.entropy - h).abs().max() < 6.1e-4


@pytest.mark.gpu
def test_edges_gpu():
    check_edges("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,W", [(1, 1, 1), (3, 17, 17), (2, 201088, 201088), (5, 10001, 10007), (64, 4096, 4100), (7, 999, 999)])
def test_gradient_gpu(dtype, N, V, W):
    torch.manual_seed(N)
    buf = (torch.randn(N, W, device="cuda") * 3).to(dtype)
    x = buf.requires_grad_()
    targets = torch.randint(0, V, (N,), device="cuda")
    targets[N // 2] = -1
    gl, gh = torch.randn(N, device="cuda"), torch.randn(N, device="cuda")
    r = ops.token_logprobs(x, targets, 0, vocab_size=V)
    peak = torch.softmax(buf.detach()[:, :V].double(), -1).amax(-1, keepdim=True)

    def check(got, gl_, gh_):
        # The result's own rounding is at most half a step of the value compared (2^-8 of it in bf16, 2^-24 in fp32). p carries the
        # 3.2e-5 of log s relative to itself and enters times |g_l|, and times |g_H| (|log p| + H) with the entropy's 6.1e-4.
        want = exact_gradient(buf.detach(), targets, V, gl_, gh_)
        rounding = (2**-8 if dtype == torch.bfloat16 else 2**-24) * want.abs()
        bound = rounding + 3.3e-5 * want.abs() + (6.1e-4 * gh_.abs() + 3.3e-5 * gl_.abs())[:, None] * peak + 1e-12
        assert ((got.double() - want).abs() <= bound).all()
        assert got[:, V:].abs().sum() == 0

    check(torch.autograd.grad((r.logprob, r.entropy), x, (gl, gh), retain_graph=True)[0], gl, gh)
    check(torch.autograd.grad(r.logprob, x, gl, retain_graph=True)[0], gl, gh * 0)
    check(torch.autograd.grad(r.entropy, x, gh)[0], gl * 0, gh)


@pytest.mark.gpu
def test_layouts_gpu():
    """Leading dimensions, a padded row stride that leaves rows off the 16-byte boundary, transposed and expanded logits, int32
    targets, another stream."""
    torch.manual_seed(5)
    big = torch.randn(6, 5, 1203, device="cuda").bfloat16()
    x = big[:, 1:4, 3:1200]
    targets = torch.randint(0, x.shape[-1], x.shape[:-1], device="cuda", dtype=torch.int32)
    want = exact(x, targets, 4, x.shape[-1])
    for y in (x, big.transpose(0, 1).contiguous().transpose(0, 1)[:, 1:4, 3:1200], x.transpose(0, 2).contiguous().transpose(0, 2)):
        r = ops.token_logprobs(y, targets, 4)
        assert r.logprob.shape == (6, 3) and r.top_ids.shape == (6, 3, 4) and torch.equal(r.top_ids, want[3])
        assert (r.logprob - want[0]).abs().max() < 3.2e-5
    one = x[:1, :1].expand(6, 3, -1)
    assert torch.equal(ops.token_logprobs(one, targets[:1, :1].expand(6, 3), 4).top_ids, want[3][:1, :1].expand(6, 3, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = ops.token_logprobs(x, targets, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(r.top_ids, want[3])
    with pytest.raises(ValueError):
        ops.token_logprobs(x.half(), targets)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, targets.cpu())


def check_one_row_without_leading_dimensions(device):
    torch.manual_seed(8)
    logits, target = torch.randn(301, device=device, requires_grad=True), torch.tensor(17, device=device)
    r = ops.token_logprobs(logits, target, 3)
    want = exact(logits.detach()[None], target[None], 3, 301)
    assert r.logprob.shape == () and r.entropy.shape == () and r.top_logprobs.shape == (3,) and torch.equal(r.top_ids, want[3][0])
    assert abs(float(r.logprob.detach()) - float(want[0])) < 3.2e-5 and abs(float(r.entropy.detach()) - float(want[1])) < 6.1e-4
    (g,) = torch.autograd.grad(r.logprob, logits)
    one = torch.ones(1, device=device)
    assert g.shape == logits.shape and (g - exact_gradient(logits.detach()[None], target[None], 301, one, 0 * one)[0]).abs().max() < 1e-5


def test_one_row_without_leading_dimensions_cpu():
    check_one_row_without_leading_dimensions("cpu")


@pytest.mark.gpu
def test_one_row_without_leading_dimensions_gpu():
    check_one_row_without_leading_dimensions("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N", [(torch.float32, 2), (torch.bfloat16, 200)])
def test_widest_rows_gpu(dtype, N):
    """2^22 columns of which one 16-byte vector in 64 holds ties above all else: the slowest selection. One column more is refused.

    Tolerance: a thread adds up 16384 terms of at most 1: 16384 * 2^-24 / 2 = 4.9e-4 relative, once in log s and once in u / s."""
    from lyra_b200.ops import native

    V, per = 1 << 22, 16 // torch.empty(0, dtype=dtype).element_size()
    x = torch.zeros(N, V + 1, dtype=dtype, device="cuda")
    x[:, :V].view(N, -1, 64, per)[:, :, 0] = 1.0
    t = torch.zeros(N, dtype=torch.long, device="cuda")
    r = ops.token_logprobs(x, t, 32, vocab_size=V)
    native.check_status()
    i = torch.arange(32, device="cuda")
    assert (r.top_ids == i // per * 64 * per + i % per).all()
    ones, zeros = V / 64 * math.e, V * 63 / 64
    lse = math.log(ones + zeros)
    assert (r.logprob - (1 - lse)).abs().max() < 1e-3 and (r.entropy - (lse - ones / (ones + zeros))).abs().max() < 1e-3
    with pytest.raises(ValueError):
        ops.token_logprobs(x, t)


@pytest.mark.gpu
def test_replay_in_a_graph_gpu():
    x = torch.randn(9, 5000, device="cuda").requires_grad_()
    targets = torch.randint(0, 5000, (9,), device="cuda")

    def step():
        r = ops.token_logprobs(x, targets, 3)
        (g,) = torch.autograd.grad((r.logprob.sum(), r.entropy.sum()), x)
        return (*(t.detach() for t in r), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))
