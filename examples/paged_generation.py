"""A one-layer language model that is trained on packed sequences and generates through a paged cache.

    python examples/paged_generation.py

Training runs ``flagsparse_attention_packed`` and its gradient over sequences of different lengths,
packed one after the other.  Generation runs the prompts through the same call while
``flagsparse_paged_append`` stores their keys and values, then goes on token by token with
``flagsparse_paged_append`` and ``flagsparse_attention_paged``.  The task: a sequence repeats a short
pattern, so that the model has to attend to where it saw the last token before.
"""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import flagsparse_amd as fs  # noqa: E402

VOCAB, WIDTH, HEADS, KV_HEADS, DIM, PAGE, LONGEST = 32, 128, 4, 2, 64, 16, 256


def tables(device):
    """cos and sin of the rotation by position."""
    half = DIM // 2
    turn = torch.arange(LONGEST, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(half, device=device, dtype=torch.float64) / half)
    return turn.cos().float(), turn.sin().float()


def rotated(x, cos, sin):
    """The rotation of paged_append, for training: elements half a head apart."""
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos[:, None] - b * sin[:, None], a * sin[:, None] + b * cos[:, None]],
                     -1).to(x.dtype)


class Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.embed = torch.nn.Embedding(VOCAB, WIDTH)
        self.previous = torch.nn.Embedding(VOCAB, WIDTH)
        self.project = torch.nn.Linear(WIDTH, (HEADS + 2 * KV_HEADS) * DIM, bias=False)
        self.join = torch.nn.Linear(HEADS * DIM, WIDTH, bias=False)
        self.read = torch.nn.Linear(WIDTH, VOCAB)

    def fused(self, tokens, before):
        """Hidden states, and queries, keys and values side by side as [tokens, heads, dim]."""
        x = self.embed(tokens) + self.previous(before)
        return x, self.project(x).view(len(tokens), HEADS + 2 * KV_HEADS, DIM).to(torch.bfloat16)

    def logits(self, x, attended):
        return self.read(x + self.join(attended.flatten(1).to(x.dtype)))


def parts(fused):
    return fused[:, :HEADS], fused[:, HEADS:HEADS + KV_HEADS], fused[:, HEADS + KV_HEADS:]


def batch(generator, device, lengths):
    """Packed tokens, the token before each, the next of each, positions and offsets."""
    rows = []
    for n in lengths:
        period = int(torch.randint(3, 9, (1,), generator=generator))
        pattern = torch.randperm(VOCAB, generator=generator)[:period]
        rows.append(pattern.repeat(n // period + 2)[:n + 1])
    tokens = torch.cat([r[:-1] for r in rows]).to(device)
    before = torch.cat([torch.cat([r[:1], r[:-2]]) for r in rows]).to(device)
    following = torch.cat([r[1:] for r in rows]).to(device)
    positions = torch.cat([torch.arange(n) for n in lengths]).to(device)
    indptr = torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).to(device)
    return tokens, before, following, positions, indptr


def train(model, device, steps, seed=1):
    """Losses of the steps; every step has sequences of its own lengths."""
    gen = torch.Generator().manual_seed(seed)
    cos, sin = tables(device)
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        lengths = torch.randint(20, 120, (24,), generator=gen).tolist()
        tokens, before, following, positions, indptr = batch(gen, device, lengths)
        pattern = fs.prepare_attention_packed(indptr)  # for every layer's forward and backward
        x, fused = model.fused(tokens, before)
        q, k, v = parts(fused)
        attended = fs.flagsparse_attention_packed(rotated(q, cos[positions], sin[positions]),
                                                  rotated(k, cos[positions], sin[positions]), v,
                                                  prepared=pattern)
        loss = torch.nn.functional.cross_entropy(model.logits(x, attended), following)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def generate(model, device, prompts, count):
    """[prompt, count] new tokens and their logits [prompt, count, vocabulary]."""
    cos, sin = tables(device)
    batch_size = len(prompts)
    # every sequence gets the pages that it will need; in what order they lie does not matter
    held = torch.tensor([-(-(len(p) + count) // PAGE) for p in prompts])
    indptr = torch.cat([torch.zeros(1, dtype=torch.int64), held.cumsum(0)]).to(device)
    pages = int(held.sum())
    cache = torch.zeros(2, pages, PAGE, KV_HEADS, DIM, dtype=torch.bfloat16, device=device)
    kv = fs.prepare_paged_kv(cache[0], cache[1], indptr, torch.randperm(pages, device=device))
    lengths = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=device)

    # the prompts: stored, and attended to where they are
    tokens = torch.cat(prompts).to(device)
    before = torch.cat([torch.cat([p[:1], p[:-1]]) for p in prompts]).to(device)
    offsets = torch.cat([lengths.new_zeros(1), lengths.cumsum(0, dtype=torch.int32)])
    x, fused = model.fused(tokens, before)
    q, k, v = parts(fused)
    # queries and keys lie side by side, so both come back rotated
    turned = fs.flagsparse_paged_append(k, v, lengths, offsets, prepared=kv,
                                        q=fused[:, :HEADS + KV_HEADS], cos=cos, sin=sin)
    attended = fs.flagsparse_attention_packed(turned[:, :HEADS], turned[:, HEADS:], v, offsets)
    last = offsets[1:].long() - 1
    logits = model.logits(x[last], attended[last])

    all_tokens, all_logits, current = [], [], tokens[last]
    for step in range(count):
        chosen = logits.argmax(-1)
        all_tokens.append(chosen)
        all_logits.append(logits)
        if step + 1 == count:
            break
        lengths += 1
        x, fused = model.fused(chosen, current)
        q, k, v = parts(fused)
        turned = fs.flagsparse_paged_append(k, v, lengths, prepared=kv, q=q, cos=cos, sin=sin)
        attended = fs.flagsparse_attention_paged(turned, lengths, prepared=kv)
        logits = model.logits(x, attended)
        current = chosen
    assert all_tokens[0].shape == (batch_size,)
    return torch.stack(all_tokens, 1), torch.stack(all_logits, 1)


def main():
    device = torch.device("cuda:0")
    torch.manual_seed(0)
    model = Model().to(device)
    losses = train(model, device, 150)
    print(f"loss: first {losses[0]:.3f}, last {losses[-1]:.3f}")
    gen = torch.Generator().manual_seed(7)
    patterns = [torch.randperm(VOCAB, generator=gen)[:n] for n in (3, 5, 8)]
    prompts = [p.repeat(4)[:len(p) * 2 + i] for i, p in enumerate(patterns)]
    tokens, _ = generate(model, device, prompts, 12)
    for p, prompt, row in zip(patterns, prompts, tokens.tolist()):
        print("pattern", p.tolist(), "after", prompt.tolist(), "->", row)


if __name__ == "__main__":
    main()
