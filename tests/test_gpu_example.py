"""The example of a small model, trained on packed sequences and generating through a paged cache."""

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


def test_it_learns_and_generates(dev):
    ex = _example()
    torch.manual_seed(0)
    model = ex.Model().to(dev)
    losses = ex.train(model, dev, 150)
    # a uniform guess over the vocabulary starts it; what follows is settled by the pattern
    assert losses[0] > 3.0 and losses[-1] < 1.0
    gen = torch.Generator().manual_seed(7)
    patterns = [torch.randperm(ex.VOCAB, generator=gen)[:n] for n in (3, 5, 8)]
    prompts = [p.repeat(4)[:len(p) * 2 + i] for i, p in enumerate(patterns)]
    tokens, logits = ex.generate(model, dev, prompts, 20)

    # the cache's way and the whole sequence at once give the same logits, to 16-bit attention
    cos, sin = ex.tables(dev)
    for b, prompt in enumerate(prompts):
        whole = torch.cat([prompt.to(dev), tokens[b, :-1]])
        before = torch.cat([whole[:1], whole[:-1]])
        at = torch.arange(len(whole), device=dev)
        with torch.no_grad():
            x, fused = model.fused(whole, before)
            q, k, v = ex.parts(fused)
            attended = ex.fs.flagsparse_attention_packed(
                ex.rotated(q, cos[at], sin[at]), ex.rotated(k, cos[at], sin[at]), v,
                torch.tensor([0, len(whole)], device=dev))
            want = model.logits(x, attended)[len(prompt) - 1:]
        # each attention output is off by at most 2 roundings of its largest value in each of two
        # ways, and the last layers pass it on by the sums of their weights' magnitudes
        gain = float((model.read.weight.abs() @ model.join.weight.abs()).sum(1).max().detach())
        bound = 4 * 2.0**-8 * float(v.abs().max()) * gain
        assert float((logits[b] - want).abs().max()) <= bound


def test_gradients_reach_every_parameter(dev):
    ex = _example()
    torch.manual_seed(1)
    model = ex.Model().to(dev)
    ex.train(model, dev, 1)
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
