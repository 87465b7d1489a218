"""The example's generation by drafted tokens: it runs, and its tokens are the model's own choice."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location(
        "paged_generation", os.path.join(ROOT, "examples", "paged_generation.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("steps", [0, 60])
def test_drafted_tokens_are_the_models(dev, steps):
    ex = _example()
    torch.manual_seed(0)
    model = ex.Model().to(dev)
    ex.train(model, dev, steps) if steps else None
    gen = torch.Generator().manual_seed(7)
    patterns = [torch.randperm(ex.VOCAB, generator=gen)[:n] for n in (3, 5, 8)]
    prompts = [p.repeat(4)[:len(p) * 2 + i] for i, p in enumerate(patterns)]
    count = 30
    tokens, taken = ex.generate_drafted(model, dev, prompts, count)
    assert tokens.shape == (3, count) and 1 <= taken <= count
    cos, sin = ex.tables(dev)
    for prompt, row in zip(prompts, tokens):
        whole = torch.cat([prompt, row[:-1]]).to(dev)
        before = torch.cat([whole[:1], whole[:-1]])
        at = torch.arange(len(whole), device=dev)
        with torch.no_grad():
            x, fused = model.fused(whole, before)
            q, k, v = ex.parts(fused)
            attended = ex.fs.flagsparse_attention_packed(
                ex.rotated(q, cos[at], sin[at]), ex.rotated(k, cos[at], sin[at]), v,
                torch.tensor([0, len(whole)], device=dev))
            logits = model.logits(x, attended)[len(prompt) - 1:]
        # each attention output is off by at most 2 roundings of its largest value in each of two
        # ways, and the last layers pass it on by the sums of their weights' magnitudes
        gain = float((model.read.weight.abs() @ model.join.weight.abs()).sum(1).max().detach())
        bound = 4 * 2.0**-8 * float(v.abs().max()) * gain
        chosen = logits.gather(1, row.to(dev)[:, None])[:, 0]
        assert float((logits.amax(1) - chosen).max()) <= 2 * bound


def test_trees_of_what_followed_before():
    ex = _example()
    assert ex.draft([5], 3, 4) == ([5], [-1])
    assert ex.draft([1, 2, 3, 1, 2, 4, 1], 2, 2) == ([1, 2, 3, 4], [-1, 0, 1, 1])
    assert ex.draft([7, 8, 7], 1, 5) == ([7, 8, 7], [-1, 0, 1])
