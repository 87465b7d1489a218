"""Attention over packed sequences and over a paged cache, as data: the calls whose speed matters.

Three operators that a language model's program makes of sequences of different lengths, which are
rows of a CSR pattern (``indptr`` over tokens, or over the pages of a cache):

* ``append``: new keys and values, rotated by their positions, written into a paged cache;
* ``decode``: one new query per sequence over all that the cache holds of it;
* ``packed`` (forward) and ``train`` (forward and gradients): whole prompts, one after the other in
  one array.

A case is a dict of plain values; ``longest`` and ``ragged`` give the sequences' lengths, which are
the same for every seed, and everything else is made on the GPU from the seed.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_EMPTY = float("-inf")


def listed():
    return [
        # one decoding step of a small batch: latency and launches are all of it
        {"name": "append_step", "op": "append", "batch": 16, "past": 500, "new": 1,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "page": 16,
         "interleaved": False, "dtype": "bf16"},
        # a batch of prompts enters the cache: a copy with a rotation, half of each head turned
        {"name": "append_prompts", "op": "append", "batch": 24, "past": 40, "new": 2000,
         "ragged": True, "heads": 16, "kv_heads": 16, "dim": 64, "rot": 32, "page": 32,
         "interleaved": True, "dtype": "f16"},
        # one user of a small model, a short conversation
        {"name": "decode_one", "op": "decode", "batch": 1, "longest": 1000, "ragged": False,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "window": 0, "lse": False,
         "dtype": "f16"},
        # a serving batch in mid-flight: slots at all stages, some empty
        {"name": "decode_batch", "op": "decode", "batch": 96, "longest": 4096, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "lse": False,
         "dtype": "bf16"},
        # a few very long documents: the cache's bytes are all of it, split over its length
        {"name": "decode_long", "op": "decode", "batch": 6, "longest": 131072, "ragged": False,
         "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "lse": True,
         "dtype": "bf16"},
        # one shared head under an odd number of queries, odd pages, a sliding window
        {"name": "decode_window", "op": "decode", "batch": 33, "longest": 20011, "ragged": True,
         "heads": 23, "kv_heads": 1, "dim": 80, "page": 24, "window": 8191, "lse": False,
         "dtype": "f16"},
        # a few short prompts: latency
        {"name": "packed_short", "op": "packed", "batch": 3, "longest": 130, "ragged": True,
         "heads": 8, "kv_heads": 8, "dim": 64, "causal": True, "window": 0, "more": 0,
         "dtype": "f16"},
        # prompts of a serving batch, packed, odd lengths
        {"name": "packed_prompts", "op": "packed", "batch": 16, "longest": 2047, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "window": 0, "more": 0,
         "dtype": "bf16"},
        # one long document
        {"name": "packed_long", "op": "packed", "batch": 1, "longest": 16384, "ragged": False,
         "heads": 16, "kv_heads": 2, "dim": 128, "causal": True, "window": 0, "more": 0,
         "dtype": "bf16"},
        # a reader that looks both ways at other sequences than its own
        {"name": "train_cross", "op": "train", "batch": 7, "longest": 300, "ragged": True,
         "heads": 12, "kv_heads": 12, "dim": 96, "causal": False, "window": 0, "more": 213,
         "dtype": "f16"},
        # a training batch of packed texts, a sliding window over the longer ones
        {"name": "train_packed", "op": "train", "batch": 12, "longest": 2500, "ragged": True,
         "heads": 16, "kv_heads": 4, "dim": 64, "causal": True, "window": 1024, "more": 0,
         "dtype": "bf16"},
        # a training batch of full rows
        {"name": "train_rows", "op": "train", "batch": 2, "longest": 4096, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "window": 0, "more": 0,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(["append", "decode", "decode", "packed", "train"])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    while kv * group > 64:
        group = rng.choice([1, 2, 3, 4])
    c = {"op": op, "heads": kv * group, "kv_heads": kv, "ragged": rng.random() < 0.7,
         "dim": rng.choice([40, 64, 72, 80, 96, 112, 128, 128]), "dtype": rng.choice(["bf16", "f16"])}
    if op == "append":
        c |= {"batch": _log_int(rng, 1, 128), "past": _log_int(rng, 1, 600),
              "page": rng.choice([8, 16, 32, 48, 64, 128]), "interleaved": rng.random() < 0.5}
        c["new"] = 1 if rng.random() < 0.5 else _log_int(rng, 2, 30000 // c["batch"] + 2)
        c["rot"] = c["dim"] // rng.choice([1, 2]) // 2 * 2
    elif op == "decode":
        c["batch"] = _log_int(rng, 1, 128)
        c["longest"] = min(_log_int(rng, 1, 131072),
                           6 * 131072 * 8 * 128 // (c["batch"] * kv * c["dim"]))
        c |= {"page": rng.choice([8, 16, 24, 32, 64, 100, 256]), "lse": rng.random() < 0.5,
              "window": _log_int(rng, 16, 8192) if rng.random() < 0.25 else 0}
    else:
        c["longest"] = _log_int(rng, 2, 6000)
        # the scores of a padded batch stay under those of the largest case
        room = (1 << 30) // max(1, (c["longest"] * c["longest"] * c["heads"]))
        c["batch"] = max(1, min(room, _log_int(rng, 1, 32)))
        c["causal"] = rng.random() < 0.75
        c["window"] = _log_int(rng, 16, 4096) if c["causal"] and rng.random() < 0.3 else 0
        c["more"] = _log_int(rng, 1, 500) if rng.random() < 0.3 else 0
    return c


def _lengths(case, longest, least):
    """A length for each sequence: all of the longest, or spread over the logarithm with the longest
    first; they follow from the case alone."""
    if not case["ragged"]:
        return [longest] * case["batch"]
    r = random.Random("%d/%d" % (case["batch"], longest))
    more = [int(math.exp(r.uniform(0, math.log(longest + 1)))) for _ in range(case["batch"] - 1)]
    if len(more) > 6:
        more[5] = 0  # a slot of the batch that holds no sequence
    return [max(least, n) for n in [longest] + more]


def _sizes(case):
    """(queries, keys) of each sequence."""
    if case["op"] == "append":
        new = _lengths(case, case["new"], 0 if case["new"] > 1 else 1)
        past = _lengths(case, case["past"], 0)
        return new, [p + n for p, n in zip(reversed(past), new)]
    keys = _lengths(case, case["longest"], 0)
    if case["op"] == "decode":
        return [1] * case["batch"], keys
    return keys, [n + case["more"] if n else 0 for n in keys]


def _pairs(case):
    """Pairs of a query and a key that it sees, over all sequences."""
    total = 0
    for nq, nk in zip(*_sizes(case)):
        if case["op"] == "decode":
            total += min(nk, case["window"] or nk)
        elif not case["causal"]:
            total += nq * nk
        else:
            w = case["window"] or nk
            seen = torch.arange(nk - nq + 1, nk + 1)
            total += int(seen.clamp(0, w).sum())
    return total


def work(case):
    nq, nk = _sizes(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        # q, k and v read and written once, the rows of the table that the tokens turn by
        return {"bytes": sum(nq) * (4 * d * (h + 2 * g) + 4 * case["rot"]),
                "flops": 3 * sum(nq) * case["rot"] * (h + g)}
    flops = 4 * _pairs(case) * h * d
    if case["op"] == "decode":
        seen = sum(min(n, case["window"] or n) for n in nk)
        return {"bytes": 2 * d * (2 * seen * g + 2 * case["batch"] * h), "flops": flops}
    data = 2 * d * (2 * sum(nq) * h + 2 * sum(nk) * g) + 4 * sum(nq) * h
    if case["op"] == "packed":
        return {"bytes": data, "flops": flops}
    # backward: q, k, v, out and its gradient read, three gradients written; scores once more and
    # four products for the three gradients
    return {"bytes": 2 * data + 2 * d * (2 * sum(nq) * h + 2 * sum(nk) * g), "flops": 3.5 * flops}


def _indptr(lengths):
    p = [0]
    for n in lengths:
        p.append(p[-1] + n)
    return torch.tensor(p, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    nq, nk = _sizes(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, gain=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * gain).to(dt)

    s = {"case": case, "q": normal(sum(nq), h, d, gain=1.5)}
    if case["op"] in ("append", "decode"):
        page = case["page"]
        held = [-(-n // page) for n in nk]
        n_pages = sum(held) + 3  # some pages belong to nobody
        s |= {"k_pages": normal(n_pages, page, g, d), "v_pages": normal(n_pages, page, g, d),
              "indptr": _indptr(held), "longest": max(nk),
              "indices": torch.randperm(n_pages, generator=gen, device="cuda")[:sum(held)].to(torch.int32),
              "lengths": torch.tensor(nk, dtype=torch.int32, device="cuda")}
        if own:
            import flagsparse_amd as fs

            s["kv"] = fs.prepare_paged_kv(s["k_pages"], s["v_pages"], s["indptr"], s["indices"])
    if case["op"] == "append":
        half = case["rot"] // 2
        turn = torch.arange(max(nk), device="cuda", dtype=torch.float64)[:, None] * torch.exp(
            torch.arange(half, device="cuda", dtype=torch.float64) * (-math.log(10000.0) / half))
        s |= {"k": normal(sum(nq), g, d), "v": normal(sum(nq), g, d), "tokens": _indptr(nq),
              "cos": turn.cos().float(), "sin": turn.sin().float()}
    elif case["op"] != "decode":
        s |= {"k": normal(sum(nk), g, d), "v": normal(sum(nk), g, d), "indptr": _indptr(nq),
              "k_indptr": _indptr(nk), "longest_q": max(nq), "longest_k": max(nk)}
        if case["op"] == "train":
            s["grad"] = normal(sum(nq), h, d)
        if own:
            import flagsparse_amd as fs

            s["pattern"] = fs.prepare_attention_packed(s["indptr"], s["k_indptr"])
    return s


def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


# ---- the framework's calls ----


def _own_append(s):
    import flagsparse_amd as fs

    q = fs.flagsparse_paged_append(s["k"], s["v"], s["lengths"], s["tokens"], prepared=s["kv"],
                                   q=s["q"], cos=s["cos"], sin=s["sin"],
                                   interleaved=s["case"]["interleaved"])
    return q, s["k_pages"], s["v_pages"]


def _own_decode(s):
    import flagsparse_amd as fs

    c = s["case"]
    return fs.flagsparse_attention_paged(s["q"], s["lengths"], prepared=s["kv"],
                                         window=c["window"] or None, return_lse=c["lse"])


def _own_packed(s):
    import flagsparse_amd as fs

    c = s["case"]
    return fs.flagsparse_attention_packed(s["q"], s["k"], s["v"], prepared=s["pattern"],
                                          causal=c["causal"], window=c["window"] or None,
                                          return_lse=True)


def _own_train(s):
    import flagsparse_amd as fs

    c = s["case"]
    out, lse = _own_packed(s)
    grads = fs.flagsparse_attention_packed_backward(
        s["grad"], s["q"], s["k"], s["v"], out, lse, prepared=s["pattern"], causal=c["causal"],
        window=c["window"] or None)
    return out, lse, *grads


_own = {"append": _own_append, "decode": _own_decode, "packed": _own_packed, "train": _own_train}


# ---- the plain form: elementary operations in 32 bits, rounded once ----


def _turn(x, cos, sin, interleaved):
    """x [tokens, heads, dim] in 32 bits with its first 2 * cos.shape[1] elements rotated by pairs:
    neighbours (interleaved), or the element half the rotated part further on."""
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    x = x.float()
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2] = a * cos - b * sin
        y[..., 1:2 * half:2] = a * sin + b * cos
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half] = a * cos - b * sin
        y[..., half:2 * half] = a * sin + b * cos
    return y


def _plain_append(s):
    c = s["case"]
    tokens = s["tokens"].long()
    at = torch.arange(s["k"].shape[0], device="cuda")
    row = torch.searchsorted(tokens, at, right=True) - 1
    pos = s["lengths"].long()[row] - tokens[row + 1] + at
    page = s["indices"].long()[s["indptr"].long()[row] + pos // c["page"]]
    cos, sin = s["cos"][pos], s["sin"][pos]
    dt = s["k"].dtype
    s["k_pages"][page, pos % c["page"]] = _turn(s["k"], cos, sin, c["interleaved"]).to(dt)
    s["v_pages"][page, pos % c["page"]] = s["v"]
    return _turn(s["q"], cos, sin, c["interleaved"]).to(dt), s["k_pages"], s["v_pages"]


def _softmax(scores, seen):
    """(weights, log of the sums of exponentials) over the last axis; a row that sees nothing has no
    weights and a logarithm of minus infinity."""
    scores = scores.masked_fill(~seen, _EMPTY)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == _EMPTY, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / total.masked_fill(total == 0, 1.0), (total.log() + top).squeeze(-1)


def _plain_decode(s):
    c = s["case"]
    b, h, g, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    pos = torch.arange(s["longest"], device="cuda")
    at = s["indptr"].long()[:-1, None] + pos // c["page"]
    page = s["indices"].long()[at.clamp(max=s["indices"].numel() - 1)]
    k = s["k_pages"][page, pos % c["page"]].float().permute(0, 2, 3, 1).contiguous()
    v = s["v_pages"][page, pos % c["page"]].float().permute(0, 2, 1, 3).contiguous()
    n = s["lengths"].long()[:, None]
    seen = (pos < n) & (pos >= n - (c["window"] or s["longest"]))
    q = s["q"].float().view(b, g, h // g, d)
    p, lse = _softmax(torch.matmul(q, k) * d ** -0.5, seen[:, None, None])
    out = torch.matmul(p, v).reshape(b, h, d).to(s["q"].dtype)
    return (out, lse.reshape(b, h)) if c["lse"] else out


def _pad(x, indptr, longest):
    """Packed [tokens, heads, dim] as 32-bit [sequences, heads, longest, dim], and each token's place."""
    at = torch.arange(x.shape[0], device="cuda")
    row = torch.searchsorted(indptr, at, right=True) - 1
    pos = at - indptr[row]
    y = torch.zeros(indptr.numel() - 1, longest, x.shape[1], x.shape[2], device="cuda")
    y[row, pos] = x.float()
    return y.transpose(1, 2).contiguous(), row, pos


def _plain_scores(s):
    c = s["case"]
    g = c["kv_heads"]
    iq, ik = s["indptr"].long(), s["k_indptr"].long()
    q, row, pos = _pad(s["q"], iq, s["longest_q"])
    k, krow, kpos = _pad(s["k"], ik, s["longest_k"])
    v = _pad(s["v"], ik, s["longest_k"])[0]
    q = q.reshape(q.shape[0], g, -1, q.shape[3])  # the queries of a group's heads, one after the other
    nq, nk = (iq[1:] - iq[:-1])[:, None, None], (ik[1:] - ik[:-1])[:, None, None]
    i = torch.arange(s["longest_q"], device="cuda")[:, None]
    j = torch.arange(s["longest_k"], device="cuda")
    seen = (i < nq) & (j < nk)
    if c["causal"]:
        seen = seen & (j <= i + nk - nq)
    if c["window"]:
        seen = seen & (j > i + nk - nq - c["window"])
    scale = c["dim"] ** -0.5
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    seen = seen.repeat(1, c["heads"] // g, 1)[:, None]
    p, lse = _softmax(scores, seen)
    del scores
    return q, k, v, p, lse, scale, (row, pos), (krow, kpos)


def _packed_again(x, heads, row, pos, dt):
    x = x.reshape(x.shape[0], heads, -1, x.shape[3])
    return x[row, :, pos].to(dt)


def _plain_packed(s):
    q, k, v, p, lse, scale, at, kat = _plain_scores(s)
    h = s["case"]["heads"]
    out = _packed_again(torch.matmul(p, v), h, *at, s["q"].dtype)
    return out, _packed_again(lse[..., None], h, *at, torch.float32).squeeze(-1)


def _plain_train(s):
    q, k, v, p, lse, scale, at, kat = _plain_scores(s)
    h, g, dt = s["case"]["heads"], s["case"]["kv_heads"], s["q"].dtype
    go = _pad(s["grad"], s["indptr"].long(), s["longest_q"])[0].reshape(q.shape)
    out = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), go)
    ds = torch.matmul(go, v.transpose(2, 3).contiguous())
    ds = p * (ds - (go * out).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    return (_packed_again(out, h, *at, dt),
            _packed_again(lse[..., None], h, *at, torch.float32).squeeze(-1),
            _packed_again(dq, h, *at, dt), _packed_again(dk, g, *kat, dt),
            _packed_again(dv, g, *kat, dt))


_plain = {"append": _plain_append, "decode": _plain_decode, "packed": _plain_packed,
          "train": _plain_train}


# ---- the definition in 64 bits, one sequence and head at a time ----


def _exact_rows(q, k, v, first, case):
    """(out, lse) of one head's queries [n, dim], the first of which is at position ``first``."""
    i = torch.arange(q.shape[0], device="cuda")[:, None] + first
    j = torch.arange(k.shape[0], device="cuda")
    hidden = torch.zeros(q.shape[0], k.shape[0], dtype=torch.bool, device="cuda")
    if case.get("causal", True):
        hidden |= j > i
    if case["window"]:
        hidden |= j <= i - case["window"]
    x = (q @ k.T) / math.sqrt(case["dim"])
    x = torch.where(hidden, torch.full_like(x, _EMPTY), x)
    lse = torch.logsumexp(x, 1)
    w = torch.where(hidden, torch.zeros_like(x), torch.exp(x - lse.detach()[:, None]))
    if q.requires_grad:  # the weights' own sum carries the gradient of the logarithm
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    return w @ v, lse


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    nq, nk = _sizes(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        return _exact_append(case, s, nq, nk)
    q = s["q"].double()
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], _EMPTY, dtype=torch.float64, device="cuda")
    train = case["op"] == "train"
    dq, tq, tk = torch.zeros_like(q), 0, 0
    if case["op"] != "decode":
        k, v = s["k"].double(), s["v"].double()
        dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for b in range(case["batch"]):
        if case["op"] == "decode":
            at = s["indptr"][b:b + 2].tolist()
            pages = s["indices"][at[0]:at[1]].long()
            kb = s["k_pages"][pages].flatten(0, 1)[:nk[b]].double()
            vb = s["v_pages"][pages].flatten(0, 1)[:nk[b]].double()
        else:
            kb, vb = k[tk:tk + nk[b]], v[tk:tk + nk[b]]
        rows = slice(tq, tq + nq[b])
        for a in range(h if nq[b] and nk[b] else 0):
            one = a // (h // g)
            x, y, z = q[rows, a], kb[:, one], vb[:, one]
            if train:
                x, y, z = (t.clone().requires_grad_() for t in (x, y, z))
            o, e = _exact_rows(x, y, z, nk[b] - nq[b], case)
            out[rows, a], lse[rows, a] = o.detach(), e.detach()
            if train:
                gx, gy, gz = torch.autograd.grad(o, (x, y, z), s["grad"][rows, a].double())
                dq[rows, a] = gx
                dk[tk:tk + nk[b], one] += gy
                dv[tk:tk + nk[b], one] += gz
        tq, tk = tq + nq[b], tk + nk[b]
    if case["op"] == "decode":
        return (out, lse) if case["lse"] else out
    return (out, lse, dq, dk, dv) if train else (out, lse)


def _exact_append(case, s, nq, nk):
    """Each pair as a complex number times the table's."""
    half = case["rot"] // 2
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    q, table = s["q"].double(), torch.complex(s["cos"].double(), s["sin"].double())

    def turned(x, turn):
        two = x[..., :2 * half].reshape(*x.shape[:-1], *((half, 2) if case["interleaved"] else (2, half)))
        if not case["interleaved"]:
            two = two.transpose(-1, -2)
        two = torch.view_as_real(torch.view_as_complex(two.contiguous()) * turn[:, None])
        if not case["interleaved"]:
            two = two.transpose(-1, -2)
        return torch.cat([two.flatten(-2), x[..., 2 * half:]], -1)

    t, at = 0, s["indptr"].tolist()
    for b in range(case["batch"]):
        if not nq[b]:
            continue
        new = slice(t, t + nq[b])
        pos = torch.arange(nk[b] - nq[b], nk[b], device="cuda")
        page = s["indices"][at[b]:at[b + 1]].long()[pos // case["page"]]
        q[new] = turned(q[new], table[pos])
        k_pages[page, pos % case["page"]] = turned(s["k"][new].double(), table[pos])
        v_pages[page, pos % case["page"]] = s["v"][new].double()
        t += nq[b]
    return q, k_pages, v_pages
