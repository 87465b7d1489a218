"""A one-layer language model that is trained on packed sequences and generates through a paged cache.

    python examples/paged_generation.py

Training runs ``flagsparse_attention_packed`` and its gradient over sequences of different lengths,
packed one after the other.  Generation runs the prompts through the same call while
``flagsparse_paged_append`` stores their keys and values, then goes on token by token with
``flagsparse_paged_append`` and ``flagsparse_attention_paged``; or several tokens at a step, by trees of
drafted tokens (``flagsparse_attention_paged_tree``), of which those that the model agrees with stay
(``flagsparse_paged_keep``).  The task: a sequence repeats a short pattern, so that the model has to attend to where
it saw the last token before.
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


def read_prompts(model, device, prompts, room):
    """(the cache with ``room`` places behind each prompt, lengths, last tokens, logits after them)."""
    cos, sin = tables(device)
    # every sequence gets the pages that it will need; in what order they lie does not matter
    held = torch.tensor([-(-(len(p) + room) // PAGE) for p in prompts])
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
    return kv, lengths, tokens[last], model.logits(x[last], attended[last])


@torch.no_grad()
def generate(model, device, prompts, count):
    """[prompt, count] new tokens and their logits [prompt, count, vocabulary]."""
    cos, sin = tables(device)
    kv, lengths, current, logits = read_prompts(model, device, prompts, count)
    all_tokens, all_logits = [], []
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
    return torch.stack(all_tokens, 1), torch.stack(all_logits, 1)


def draft(text, breadth, depth):
    """(tokens, parents) of a tree that starts at the last token of a text: what followed the token's last
    ``breadth`` places before, ``depth`` tokens each."""
    tokens, parents = [text[-1]], [-1]
    places = [i for i, token in enumerate(text[:-1]) if token == text[-1]]
    for place in places[-breadth:]:
        at = 0
        for token in text[place + 1:place + 1 + depth]:
            same = [i for i, p in enumerate(parents) if p == at and tokens[i] == token]
            if not same:
                tokens.append(token)
                parents.append(at)
            at = same[0] if same else len(tokens) - 1
    return tokens, parents


@torch.no_grad()
def generate_drafted(model, device, prompts, count, breadth=3, depth=5):
    """([prompt, count] new tokens, the steps that they took): each step reads a tree of drafted tokens for each
    sequence, and goes on from the last one of those that the model would have chosen."""
    cos, sin = tables(device)
    most = 1 + breadth * depth
    kv, lengths, _, logits = read_prompts(model, device, prompts, count + 2 * most)
    texts = [p.tolist() + [int(t)] for p, t in zip(prompts, logits.argmax(-1))]
    steps = 0
    while min(len(text) - len(p) for text, p in zip(texts, prompts)) < count:
        trees = [draft(text, breadth, depth) if len(text) - len(p) < count else ([], [])
                 for text, p in zip(texts, prompts)]
        tokens = torch.tensor([t for tree in trees for t in tree[0]], device=device)
        before = torch.tensor([tree[0][p] if p >= 0 else text[-2] for tree, text in zip(trees, texts)
                               for p in tree[1]], device=device)
        parents = torch.tensor([p for tree in trees for p in tree[1]], dtype=torch.int32, device=device)
        new = torch.tensor([len(tree[0]) for tree in trees], dtype=torch.int32)
        offsets = torch.cat([new.new_zeros(1), new.cumsum(0, dtype=torch.int32)]).to(device)
        lengths = lengths + new.to(device)
        x, fused = model.fused(tokens, before)
        q, k, v = parts(fused)
        turned = fs.flagsparse_paged_append(k, v, lengths, offsets, prepared=kv, q=q, cos=cos, sin=sin,
                                            parents=parents)
        attended = fs.flagsparse_attention_paged_tree(turned, lengths, offsets, parents=parents,
                                                      longest=most, prepared=kv)
        chosen = model.logits(x, attended).argmax(-1).tolist()
        keep, at = torch.zeros(len(tokens), dtype=torch.bool), 0
        for text, (drafted, ups) in zip(texts, trees):
            here = 0 if drafted else None
            while here is not None:  # down the tree as long as a child is what the model chooses
                keep[at + here] = True
                text.append(chosen[at + here])
                here = next((i for i, p in enumerate(ups) if p == here and drafted[i] == text[-1]), None)
            at += len(drafted)
        lengths = fs.flagsparse_paged_keep(keep.to(device), lengths, offsets, prepared=kv)
        steps += 1
    return torch.tensor([text[len(p):len(p) + count] for text, p in zip(texts, prompts)]), steps


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
    tokens, steps = generate_drafted(model, device, prompts, 40)
    print(f"40 tokens each by drafts in {steps} steps: {tokens.tolist()}")


if __name__ == "__main__":
    main()
