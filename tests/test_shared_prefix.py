"""Generation and evaluation behind a shared prefix: the same tokens and scores as running every sequence from its first token, and the
whole decode path with all its operators together (prefix attention, one-kernel MoE block, token scores), eager and replayed."""

from dataclasses import replace

import pytest
import torch

from lyra_b200.config import Mode
from lyra_b200.evals.common import Doc, Scorer, continuation_scores, prefix_cache, shared_beginning, token_scores
from lyra_b200.generate import BatchedGenerator, InferenceConfig, apply_inference_overrides, init_cache
from lyra_b200.model import ModelCache, ModelWeights, model_apply
from tests.helpers import small_config


def hidden_of(c, w, tokens, device="cpu"):
    cache = init_cache(c, tokens.shape[1], device, tokens.shape[0])
    with torch.no_grad():
        return model_apply(tokens, w, cache, replace(c, mode=Mode.PREFILL), return_hidden_states=True)[0]


@pytest.mark.parametrize("fp8", [False, True])
def test_model_behind_a_prefix_equals_the_joined_sequence(fp8):
    c = small_config(compute_dtype=torch.float32, seq_len=64)
    if fp8:
        c = replace(c, quantize_cache=True)
    w = ModelWeights.init(0, c)
    g = torch.Generator().manual_seed(0)
    prefix, own = torch.randint(0, 500, (21,), generator=g), torch.randint(0, 500, (3, 6), generator=g)
    cfg = replace(c, mode=Mode.PREFILL)
    shared = prefix_cache(w, c, prefix)
    cache = ModelCache.share(shared, cfg, 3, 8, "cpu")
    with torch.no_grad():
        first, _, cache = model_apply(own[:, :4], w, cache, cfg, return_hidden_states=True)
        assert cache.pos == 4 and cache.prefix_len == 21
        rest, _, cache = model_apply(own[:, 4:5], w, cache, replace(c, mode=Mode.DECODE), return_hidden_states=True)
        last, _, cache = model_apply(own[:, 5:], w, cache, replace(c, mode=Mode.DECODE), return_hidden_states=True)
    got = torch.cat([first, rest, last], dim=1)
    joined = torch.cat([prefix[None].expand(3, -1), own], dim=1)
    if fp8:      # token by token, so that every position reads the quantised cache as it does behind the prefix
        whole = init_cache(c, 27, "cpu", 3)
        with torch.no_grad():
            _, _, whole = model_apply(joined[:, :21], w, whole, cfg, return_hidden_states=True)
            steps = []
            for t in range(21, 27):
                h, _, whole = model_apply(joined[:, t:t + 1], w, whole, replace(c, mode=Mode.DECODE), return_hidden_states=True)
                steps.append(h)
        want = torch.cat(steps, 1)
    else:
        want = hidden_of(c, w, joined)[:, 21:]
    # the same fp32 terms in another order; a near-equal choice of experts would differ by far more
    assert (got - want).abs().max() < 1e-4 * want.abs().max()
    with pytest.raises(ValueError):
        ModelCache.share(cache, cfg, 2, 4, "cpu")


def test_a_batch_is_no_shared_prefix():
    c = small_config()
    with pytest.raises(ValueError):
        ModelCache.share(init_cache(c, 8, "cpu", 2), c, 3, 4, "cpu")


def test_batched_generation_behind_a_prefix():
    c = small_config(compute_dtype=torch.float32, sample_temperature=0.0, seq_len=64)
    w = ModelWeights.init(0, c)
    g = torch.Generator().manual_seed(1)
    prefix, prompts = torch.randint(0, 500, (15,), generator=g), torch.randint(0, 500, (3, 5), generator=g)
    gen = BatchedGenerator(w, c, batch=3, capacity=16, device="cpu")
    with_prefix = gen.decode(gen.prefill(prompts, prefix), 6)
    plain = BatchedGenerator(w, c, batch=3, capacity=40, device="cpu")
    joined = torch.cat([prefix[None].expand(3, -1), prompts], dim=1)
    assert torch.equal(with_prefix, plain.decode(plain.prefill(joined), 6))
    alone = BatchedGenerator(w, c, batch=3, capacity=16, device="cpu")
    assert torch.equal(gen.decode(gen.prefill(prompts), 6), alone.decode(alone.prefill(prompts), 6))     # and without one again
    for bad in (prefix[None], prefix[:0], torch.zeros(62, dtype=torch.long)):
        with pytest.raises(ValueError):
            gen.prefill(prompts, bad)


def test_generation_behind_a_prefix_ends_with_the_model_s_positions():
    """A cache may be larger than what the model's positions leave behind the prefix: the last token that fits is generated, one more is
    refused, in steps and (before anything runs) in a recorded sequence of steps."""
    c = small_config(compute_dtype=torch.float32, sample_temperature=0.0, seq_len=32, rope_scale=1.0)
    w = ModelWeights.init(0, c)
    gen = BatchedGenerator(w, c, batch=2, capacity=30, device="cpu")
    prefix, prompts = torch.arange(20), torch.arange(10).view(2, 5)
    first = gen.prefill(prompts, prefix)
    assert gen.decode(first, 8).shape == (2, 8)                # 20 + 5 + 7 positions
    for run in (gen.decode, gen._decode_graph):
        first = gen.prefill(prompts, prefix)
        with pytest.raises(ValueError, match="32"):
            run(first, 9)


def test_fused_moe_decode_is_opt_in_and_follows_the_step_by_step_path():
    c = small_config(compute_dtype=torch.float32, sample_temperature=0.0)
    assert not c.fused_moe_decode
    fused = apply_inference_overrides(c, InferenceConfig(weights="x", fused_moe=True))
    assert fused.fused_moe_decode
    w = ModelWeights.init(0, c)
    prompts = torch.randint(0, 500, (2, 7), generator=torch.Generator().manual_seed(2))
    outs = []
    for cfg in (c, fused):
        gen = BatchedGenerator(w, cfg, batch=2, capacity=16, device="cpu")
        outs.append(gen.decode(gen.prefill(prompts), 5))
    assert torch.equal(*outs)


def test_resume_ignores_the_decode_option():
    from lyra_b200.training.train import MODEL_FIELDS_IGNORED_ON_RESUME

    assert "fused_moe_decode" in MODEL_FIELDS_IGNORED_ON_RESUME


def test_scorer_with_a_shared_prefix_gives_the_same_scores():
    c = small_config(vocab_size=201088, padded_vocab_size=204800, n_layers=2, mlp_map=("dense", "moe"), seq_len=400, compute_dtype=torch.float32)
    w = ModelWeights.init(0, c)
    shots = "Question: sky?\nAnswer: blue\n\nQuestion: grass?\nAnswer: green\n\n"
    docs = [Doc(shots + "Question: snow?\nAnswer:", ("white", "black as night", "red"), 0, True), Doc(shots + "Question: coal?\nAnswer:", ("black", "white"), 0, True),
            Doc("Unlike the others:", ("x", "yes"), 1, True), Doc("word " * 100, ("cut from the left",), 0)]
    apart = Scorer(w, c, batch_size=3).score(docs)
    together = Scorer(w, c, batch_size=3, share_prefix=True).score(docs)
    assert all(abs(a - b) < 1e-3 * max(1.0, abs(a)) for x, y in zip(apart, together) for a, b in zip(x, y))
    reqs = sorted(Scorer(w, c).requests(docs), key=lambda r: r.ids)
    group = [r for r in reqs if r.doc < 2]
    common = shared_beginning(group)
    assert 32 <= common < min(r.scored_from for r in group) and len({tuple(r.ids[:common]) for r in group}) == 1
    one = [r for r in reqs if r.doc == 0]
    assert shared_beginning(one) == one[0].scored_from - 1          # the choices of one question share all of it but its last token


def test_token_scores_against_the_logits():
    c = small_config(compute_dtype=torch.float32)
    w = ModelWeights.init(0, c)
    tokens = torch.randint(0, 500, (2, 9), generator=torch.Generator().manual_seed(3))
    hidden = hidden_of(c, w, tokens)
    targets = torch.cat([tokens[:, 1:], torch.full((2, 1), -1)], dim=1)
    got = token_scores(hidden, targets, w, c, top_k=3, row_block=4)
    logp = torch.log_softmax((hidden @ w.tok.emb[:500].to(hidden.dtype).t()).double(), -1)
    want = logp[:, :-1].gather(-1, targets[:, :-1, None])[..., 0]
    assert (got.logprob[:, :-1] - want).abs().max() < 1e-4 and got.logprob[:, -1].abs().max() == 0
    assert (got.entropy + (logp.exp() * logp).sum(-1)).abs().max() < 1e-4
    assert got.top_ids.shape == (2, 9, 3) and torch.equal(got.top_ids[..., 0], logp.argmax(-1))


# --------------------------------------------------------------------------- GPU
def gpu_model(fp8: bool):
    from lyra_b200.variants import model_variant

    c = replace(model_variant("tiny"), sample_temperature=0.0, seq_len=1024)
    if fp8:
        c = replace(apply_inference_overrides(c, InferenceConfig(weights="x", fp8=True)), sample_temperature=0.0, quant_block=(64, 64))
    w = ModelWeights.init(0, c, device="cuda:0")
    return c, (ModelWeights.quantize(w, c) if fp8 else w)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("fused", [False, True])
def test_decode_behind_a_prefix_gpu(fp8, fused):
    """Prefix attention, the MoE block and the cache append together: eager steps and a replayed graph give the same tokens, and hidden
    states close to those of the joined sequence."""
    from lyra_b200.ops import native

    c, w = gpu_model(fp8)
    c = replace(c, fused_moe_decode=fused)
    g = torch.Generator(device="cuda").manual_seed(4)
    prefix, prompts = (torch.randint(0, c.vocab_size, s, generator=g, device="cuda") for s in ((300,), (6, 9)))
    eager = BatchedGenerator(w, c, batch=6, capacity=40, device="cuda:0")
    first = eager.prefill(prompts, prefix)
    a = eager.decode(first, 12)
    replayed = BatchedGenerator(w, c, batch=6, capacity=40, device="cuda:0", use_cuda_graph=True)
    for _ in range(2):                                          # the second prefill brings a new cache and a new recording
        b = replayed.decode(replayed.prefill(prompts, prefix), 12)
        assert torch.equal(a, b)
    # teacher-forced hidden states, behind the prefix and as one sequence
    joined = torch.cat([prefix[None].expand(6, -1), prompts], dim=1)
    cfg = replace(c, mode=Mode.PREFILL)
    with torch.no_grad():
        cache = ModelCache.share(prefix_cache(w, c, prefix), cfg, 6, 16, "cuda:0")
        h, _, _ = model_apply(prompts, w, cache, cfg, return_hidden_states=True)
        whole = init_cache(c, 320, "cuda:0", 6)
        hw, _, _ = model_apply(joined, w, whole, cfg, return_hidden_states=True)
    native.check_status()
    # two paths of the same bf16 model (with --fp8 one of them reads the prompt's own keys unquantised): a few roundings per layer
    err = (h.float() - hw[:, 300:].float()).norm() / hw[:, 300:].float().norm()
    assert err < (0.1 if fp8 else 0.03), float(err)


@pytest.mark.gpu
def test_fused_moe_steps_follow_the_step_by_step_path_gpu():
    c, w = gpu_model(False)
    tokens = torch.randint(0, c.vocab_size, (4, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    hidden = []
    with torch.no_grad():
        for fused in (False, True):
            cfg = replace(c, mode=Mode.DECODE, fused_moe_decode=fused)
            cache = init_cache(cfg, 8, "cuda:0", 4)
            hidden.append(model_apply(tokens, w, cache, cfg, return_hidden_states=True)[0].float())
    # both round the normalised input, the hidden units and each layer's output to bf16 (2^-8 each) at other places
    assert (hidden[0] - hidden[1]).norm() < 6 * 2**-8 * hidden[0].norm()


@pytest.mark.gpu
def test_scores_behind_a_prefix_gpu():
    """A scoring pass: prefix attention over several own tokens, logits, token scores with alternatives."""
    c, w = gpu_model(False)
    g = torch.Generator(device="cuda").manual_seed(6)
    prefix, own = (torch.randint(0, c.vocab_size, s, generator=g, device="cuda") for s in ((200,), (5, 11)))
    targets = torch.cat([own[:, 1:], torch.full((5, 1), -1, device="cuda")], dim=1)
    got = continuation_scores(w, c, prefix_cache(w, c, prefix), own, targets, top_k=4)
    joined = torch.cat([prefix[None].expand(5, -1), own], dim=1)
    want = token_scores(hidden_of(c, w, joined, "cuda:0")[:, 200:], targets, w, c, top_k=4)
    assert got.logprob[:, -1].abs().max() == 0 and got.top_ids.shape == (5, 11, 4)
    # hidden states differ by a few bf16 roundings; a random model's logits have a spread of about 1
    assert (got.logprob - want.logprob).abs().max() < 0.1 and (got.entropy - want.entropy).abs().max() < 0.05
    docs = [Doc("The sky above the port was the color of " * 6, ("television", "tuned to a dead channel"), 0, True)]
    a, b = (Scorer(w, c, batch_size=2, device="cuda:0", share_prefix=s).score(docs) for s in (False, True))
    assert all(abs(x - y) < 0.02 * abs(x) for p, q in zip(a, b) for x, y in zip(p, q))
