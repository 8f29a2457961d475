"""Incremental generation against recomputing the whole sequence for every step."""
import math

import pytest
import torch

import exploration_b200 as eb


def small_model(seed=0, vocab=19, dim=32, heads=4, layers=2):
    torch.manual_seed(seed)
    model = eb.BaselineModel(vocab, dim=dim, heads=heads, layers=layers).eval()
    with torch.no_grad():
        model.embedding.weight.mul_(20)      # logits of a spread that makes ties and near ties unlikely
    return model


def full_logp(model, tokens):
    with torch.no_grad():
        return torch.log_softmax(model(torch.tensor([tokens], device=model.embedding.weight.device))[0, -1].double(), -1)


def search_by_recomputation(model, prompt, steps, beams, eos):
    """Beam search that runs the whole sequence through the model for every candidate."""
    live = [(0.0, list(prompt), False)]
    for _ in range(steps):
        pool = []
        for w, (score, tokens, ended) in enumerate(live):
            if ended:
                pool.append((-score, w, tokens + [eos], True))
                continue
            logp = full_logp(model, tokens)
            for t in range(len(logp)):
                pool.append((-(score + float(logp[t])), w, tokens + [t], t == eos))
        pool.sort(key=lambda c: c[:2])
        live = [(-c[0], c[2], c[3]) for c in pool[:beams]]
    return live


PROMPTS = [[3, 1, 4, 1, 5], [9], list(range(18)), [2] * 33]


@pytest.mark.parametrize("chunk", [4096, 7])
@pytest.mark.parametrize("beams,eos", [(1, None), (3, None), (4, 5)])
def test_generate_equals_recomputation(beams, eos, chunk):
    model = small_model()
    tokens, scores = eb.generate(model, PROMPTS, 6, beams=beams, eos=eos, page=16, prefill_chunk=chunk)
    for g, prompt in enumerate(PROMPTS):
        for b, (score, want, _) in enumerate(search_by_recomputation(model, prompt, 6, beams, eos)):
            assert tokens[g, b].tolist() == want[len(prompt):]
            assert abs(float(scores[g, b]) - score) < 1e-4


def test_generate_stops_when_every_beam_has_ended():
    model = small_model()
    with torch.no_grad():
        # The next token after anything is 7.
        model.final_norm.weight.zero_()
        model.final_norm.bias.copy_(100 * model.embedding.weight[7])
    tokens, scores = eb.generate(model, [[1, 2], [3]], 40, beams=1, eos=7)
    assert tokens.shape == (2, 1, 16) and bool((tokens == 7).all())
    assert bool(torch.isfinite(scores).all())


def test_generate_refusals():
    model = small_model()
    for call, message in [
            (lambda: eb.generate(model, [], 3), "prompts"), (lambda: eb.generate(model, [[1]], 0), "new tokens"),
            (lambda: eb.generate(model, [[]], 3), "at least one token"),
            (lambda: eb.generate(model, [[1]], 3, beams=33), "beams"),
            (lambda: eb.generate(model, [[1]], 3, eos=19), "eos"),
            (lambda: eb.generate(model, [[1]], 3, page=24), "power of two"),
            (lambda: eb.generate(eb.StackModel(19, dim=32, heads=4), [[1]], 3), "incremental")]:
        with pytest.raises(ValueError, match=message):
            call()


def test_cache_shares_prompt_pages():
    cache = eb.PagedCache(2, 1, 8, [40, 5], 20, beams=3, page=16)
    assert cache.tables.shape == (2, 3, 4)
    assert bool((cache.tables[0, :, :2] == cache.tables[0, :1, :2]).all())
    own = torch.cat((cache.tables[0, :, 2:].flatten(), cache.tables[1, :, :2].flatten(), cache.spare.flatten(),
                     cache.tables[0, 0, :2]))
    assert own.unique().numel() == own.numel() == cache.k.shape[1]


@pytest.mark.gpu
@pytest.mark.parametrize("beams,eos", [(1, None), (4, 5)])
def test_generate_on_the_gpu(native, beams, eos):
    """fp32: the same hypotheses as on the CPU; head dim 8 runs the CUDA-core attention."""
    model = small_model()
    want, want_scores = eb.generate(model, PROMPTS, 8, beams=beams, eos=eos, page=16)
    got, scores = eb.generate(model.cuda(), PROMPTS, 8, beams=beams, eos=eos, page=16, prefill_chunk=11)
    assert torch.equal(got.cpu(), want)
    torch.testing.assert_close(scores.cpu(), want_scores, atol=1e-3, rtol=0)
    assert native.device_errors(torch.cuda.current_device()) == (0, 0)


@pytest.mark.gpu
def test_generate_bf16_scores_are_the_models(native):
    """bf16 autocast, tensor-core attention (prompts as chunks, then few rows): scores match a full pass."""
    torch.manual_seed(1)
    model = eb.BaselineModel(64, dim=256, heads=4, layers=3).cuda().eval()
    with torch.no_grad():
        model.embedding.weight.mul_(20)
    prompts = [torch.randint(0, 64, (n,)).tolist() for n in (300, 45, 1)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        tokens, scores = eb.generate(model, prompts, 20, beams=3)
        for g, prompt in enumerate(prompts):
            for b in range(3):
                ids = torch.tensor([prompt + tokens[g, b].tolist()], device="cuda")
                with torch.no_grad():
                    logp = torch.log_softmax(model(ids)[0].float(), -1)
                at = torch.arange(len(prompt) - 1, len(prompt) + 19, device="cuda")
                total = logp[at, tokens[g, b]].sum()
                # Twenty steps, each a difference of logits of size about 10 known to bf16's 2^-8.
                assert abs(float(total - scores[g, b])) < 20 * 2 * 10 * 2.0 ** -8
    assert native.device_errors(torch.cuda.current_device()) == (0, 0)
