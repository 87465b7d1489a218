"""What a program that drafts, branches and forgets makes of packed sequences and a paged cache, as data.

* ``decode``, ``packed``, ``train``: attention under a sliding window with a few first tokens that stay
  visible (sinks), of one new token over a cache, of whole prompts, and forward with gradients;
* ``tree``: attention of a tree of drafted tokens over a cache that holds them at its end;
* ``accept``: drafted tokens enter the cache, turned by their depth in the tree, and those that were
  accepted close up behind the cached text;
* ``evict``: tokens of long sequences are given up, the others go to pages of their own;
* ``copy``: pages are copied, as forks of sequences need it.

A case is a dict of plain values; the sequences' lengths follow from it alone, everything else is made on
the GPU from the seed.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_EMPTY = float("-inf")
_DRAFTS = 256  # drafted tokens of one sequence, at most


def listed():
    return [
        # one decoding step of a few chats that outgrew their window: latency
        {"name": "sinks_step", "op": "decode", "batch": 4, "longest": 2000, "ragged": False,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "window": 512, "sinks": 4, "lse": False,
         "dtype": "f16"},
        # a serving batch of streams of all ages under a long window
        {"name": "sinks_streams", "op": "decode", "batch": 64, "longest": 60000, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 4096, "sinks": 64, "lse": True,
         "dtype": "bf16"},
        # long prompts of a layer with a window
        {"name": "sinks_prompt", "op": "packed", "batch": 2, "longest": 8192, "ragged": False,
         "heads": 16, "kv_heads": 4, "dim": 128, "window": 1024, "sinks": 4, "more": 0,
         "dtype": "bf16"},
        # training on texts of odd lengths, more first tokens than a block of keys
        {"name": "sinks_train_odd", "op": "train", "batch": 6, "longest": 1501, "ragged": True,
         "heads": 12, "kv_heads": 4, "dim": 96, "window": 200, "sinks": 70, "more": 0,
         "dtype": "f16"},
        # a training batch of full rows: every first key takes gradients from all later queries
        {"name": "sinks_train_rows", "op": "train", "batch": 4, "longest": 4096, "ragged": False,
         "heads": 16, "kv_heads": 4, "dim": 64, "window": 512, "sinks": 16, "more": 0,
         "dtype": "bf16"},
        # one user of a small model, a few drafted tokens: latency
        {"name": "tree_one", "op": "tree", "batch": 1, "longest": 1200, "ragged": False, "drafts": 8,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "window": 0, "sinks": 0, "lse": False,
         "chain": False, "dtype": "f16"},
        # drafts of different sizes in a batch, one key head, odd pages, a window and sinks
        {"name": "tree_window", "op": "tree", "batch": 33, "longest": 20011, "ragged": True,
         "drafts": 26, "heads": 23, "kv_heads": 1, "dim": 80, "page": 24, "window": 2047, "sinks": 5,
         "lse": True, "chain": False, "dtype": "f16"},
        # wide trees over long texts: as much work for the matrix units as for memory
        {"name": "tree_wide", "op": "tree", "batch": 8, "longest": 30000, "ragged": False,
         "drafts": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "sinks": 0,
         "lse": False, "chain": False, "dtype": "bf16"},
        # the cache's part of a step with drafts: latency
        {"name": "accept_step", "op": "accept", "batch": 16, "longest": 900, "ragged": True,
         "drafts": 26, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"},
        # half the tokens of long sequences are given up: a gather at memory's rate
        {"name": "evict_half", "op": "evict", "batch": 16, "longest": 8192, "ragged": False,
         "kv_heads": 8, "dim": 128, "page": 64, "share": 0.5, "dtype": "bf16"},
        # a few samples branch off a prompt: latency
        {"name": "copy_forks", "op": "copy", "pages": 7, "spare": 50, "page": 16, "kv_heads": 8,
         "dim": 128, "dtype": "f16"},
        # a cache makes room: thousands of pages move
        {"name": "copy_many", "op": "copy", "pages": 4001, "spare": 5000, "page": 16, "kv_heads": 8,
         "dim": 128, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(["decode", "packed", "train", "train", "tree", "tree", "tree", "accept", "evict",
                     "copy"])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    while kv * group > 64:
        group = rng.choice([1, 2, 3, 4])
    dim = rng.choice([40, 64, 72, 80, 96, 112, 128, 128])
    c = {"op": op, "kv_heads": kv, "dim": dim, "dtype": rng.choice(["bf16", "f16"])}
    if op in ("decode", "packed", "train", "tree", "accept"):
        c |= {"heads": kv * group, "ragged": rng.random() < 0.7}
    if op not in ("packed", "train"):
        c["page"] = rng.choice([8, 16, 24, 32, 64, 100, 256])
    if op in ("packed", "train", "decode"):
        c |= {"window": _log_int(rng, 16, 4096), "sinks": _log_int(rng, 1, 128)}
    if op == "decode":
        c |= {"batch": _log_int(rng, 1, 128), "lse": rng.random() < 0.5}
        c["longest"] = min(_log_int(rng, 1, 100000), (1 << 28) // (c["batch"] * kv))
        c["window"] = min(c["window"], (1 << 28) // (c["batch"] * kv * dim))
    elif op in ("packed", "train"):
        c["longest"] = _log_int(rng, 2, 6000)
        # the scores of a padded batch stay under those of the largest case
        room = (1 << 30) // max(1, c["longest"] * c["longest"] * c["heads"])
        c["batch"] = max(1, min(room, _log_int(rng, 1, 32)))
        c["more"] = _log_int(rng, 1, 500) if rng.random() < 0.3 else 0
    elif op == "tree":
        c |= {"batch": _log_int(rng, 1, 64), "drafts": _log_int(rng, 1, 160),
              "lse": rng.random() < 0.5, "chain": rng.random() < 0.25, "window": 0, "sinks": 0}
        # keys and scores of a padded batch stay under those of the largest case
        room = min((1 << 27) // (c["batch"] * kv * dim),
                   (1 << 28) // (c["batch"] * c["heads"] * c["drafts"]))
        c["longest"] = max(c["drafts"], min(_log_int(rng, 1, 30000), room))
        if rng.random() < 0.4:
            c |= {"window": _log_int(rng, 4, 4096), "sinks": _log_int(rng, 1, 100)}
    elif op == "accept":
        c |= {"batch": _log_int(rng, 1, 128), "longest": _log_int(rng, 1, 2000)}
        c["drafts"] = _log_int(rng, 1, min(160, 8000 // c["batch"]))
    elif op == "evict":
        c |= {"batch": _log_int(rng, 1, 64), "ragged": rng.random() < 0.5,
              "share": rng.choice([0.1, 0.5, 0.9])}
        c["longest"] = min(_log_int(rng, 16, 30000), (1 << 27) // (c["batch"] * kv * dim))
    else:
        most = 4001 * 16 * 8 * 128 // (c["page"] * kv * dim)
        c |= {"pages": _log_int(rng, 1, max(1, most)), "spare": _log_int(rng, 1, 5000)}
        c["spare"] = min(c["spare"], 2 * most + 1)
    return c


def _lengths(case, longest, least, salt=0):
    """A length for each sequence: all of the longest, or spread over the logarithm with the longest
    first; they follow from the case alone."""
    if not case["ragged"]:
        return [longest] * case["batch"]
    r = random.Random("%d/%d/%d" % (case["batch"], longest, salt))
    more = [int(math.exp(r.uniform(0, math.log(longest + 1)))) for _ in range(case["batch"] - 1)]
    if len(more) > 6:
        more[5] = 0  # a slot of the batch that holds no sequence
    return [max(least, n) for n in [longest] + more]


def _sizes(case):
    """(queries, keys) of each sequence."""
    keys = _lengths(case, case["longest"], 0)
    if case["op"] in ("decode", "evict"):
        return [1] * case["batch"], keys
    if case["op"] in ("tree", "accept"):
        new = _lengths(case, case["drafts"], 0, 1)
        return new, [n + m for n, m in zip(new, reversed(keys))]
    return keys, [n + case["more"] if n else 0 for n in keys]


def _kept(case):
    return [int(n * case["share"]) for n in _sizes(case)[1]]


def _pairs(case):
    """(pairs of a query and a key that it sees, keys that any query sees), over all sequences; of a
    tree's drafted keys a query's own alone is sure."""
    pairs = keys = 0
    w, s = case["window"], case["sinks"]
    for nq, nk in zip(*_sizes(case)):
        if not nq:
            continue
        if case["op"] == "tree":
            past = nk - nq
            seen = past if not w else min(past, w - 1 + min(s, max(0, past + 1 - w)))
            pairs, keys = pairs + nq * (max(0, seen) + 1), keys + max(0, seen) + nq
            continue
        p = torch.arange(nk - nq, nk, dtype=torch.int64)  # the queries' positions
        first = (p + 1 - w).clamp(min=0)
        pairs += int((p + 1 - first + first.clamp(max=s)).sum())
        at = int(first[0]) if nq else nk
        keys += nk - at + min(s, at)
    return pairs, keys


def work(case):
    g, d = case["kv_heads"], case["dim"]
    if case["op"] == "copy":
        return {"bytes": 8 * case["pages"] * case["page"] * g * d, "flops": 0}
    nq, nk = _sizes(case)
    if case["op"] == "evict":
        # marks, and both rows of each token that stays, read and written
        return {"bytes": sum(nk) + 8 * sum(_kept(case)) * g * d, "flops": 0}
    h = case["heads"]
    if case["op"] == "accept":
        # q, k and v read and written once, the table's rows; what moves goes by the tree
        return {"bytes": sum(nq) * (4 * d * (h + 2 * g) + 4 * d), "flops": 3 * sum(nq) * d * (h + g)}
    pairs, keys = _pairs(case)
    if case["op"] in ("decode", "tree"):
        return {"bytes": 2 * d * (2 * keys * g + 2 * sum(nq) * h), "flops": 4 * pairs * h * d}
    data = 2 * d * (2 * sum(nq) * h + 2 * keys * g) + 4 * sum(nq) * h
    if case["op"] == "packed":
        return {"bytes": data, "flops": 4 * pairs * h * d}
    # backward: q, k, v, out and its gradient read, three gradients written; scores once more and
    # four products for the three gradients
    return {"bytes": 2 * data + 2 * d * (2 * sum(nq) * h + 2 * sum(nk) * g),
            "flops": 14 * pairs * h * d}


def _indptr(lengths):
    p = [0]
    for n in lengths:
        p.append(p[-1] + n)
    return torch.tensor(p, dtype=torch.int32, device="cuda")


def _trees(sizes, chain, gen):
    """Parents of each sequence's drafted tokens, by place: near ones, now and then the text itself."""
    if chain:
        parents = [torch.arange(-1, n - 1) for n in sizes]
        return torch.cat(parents).to(torch.int32).to("cuda")
    at = torch.cat([torch.arange(n) for n in sizes]).to("cuda")
    r = torch.rand(2, at.numel(), generator=gen, device="cuda")
    back = 1 + (r[0] * torch.clamp(at, max=9)).long()
    return torch.where(r[1] < 0.05, -1, at - torch.clamp(back, max=at + 1)).clamp(min=-1).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    g, d, op = case["kv_heads"], case["dim"], case["op"]

    def normal(*shape, gain=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * gain).to(dt)

    def some(n, of):
        return torch.randperm(of, generator=gen, device="cuda")[:n].to(torch.int32)

    s = {"case": case}
    if op == "copy":
        n, page = 2 * case["pages"] + case["spare"], case["page"]
        both = some(2 * case["pages"], n)
        s |= {"k_pages": normal(n, page, g, d), "v_pages": normal(n, page, g, d),
              "sources": both[::2].contiguous(), "targets": both[1::2].contiguous()}
        if own:
            import flagsparse_amd as fs

            s["kv"] = fs.prepare_paged_kv(s["k_pages"], s["v_pages"], _indptr([case["pages"]]),
                                          s["sources"])
        return s
    nq, nk = _sizes(case)
    if op in ("packed", "train"):
        h = case["heads"]
        s |= {"q": normal(sum(nq), h, d, gain=1.5), "k": normal(sum(nk), g, d),
              "v": normal(sum(nk), g, d), "indptr": _indptr(nq), "k_indptr": _indptr(nk),
              "longest_q": max(nq), "longest_k": max(nk)}
        if op == "train":
            s["grad"] = normal(sum(nq), h, d)
        if own:
            import flagsparse_amd as fs

            s["pattern"] = fs.prepare_attention_packed(s["indptr"], s["k_indptr"])
        return s
    page = case["page"]
    held = [-(-n // page) for n in nk]
    kept = [-(-n // page) for n in _kept(case)] if op == "evict" else []
    n_pages = sum(held) + sum(kept) + 3  # some pages belong to nobody
    table = some(sum(held) + sum(kept), n_pages)
    s |= {"k_pages": normal(n_pages, page, g, d), "v_pages": normal(n_pages, page, g, d),
          "indptr": _indptr(held), "indices": table[:sum(held)].contiguous(), "longest": max(nk),
          "lengths": torch.tensor(nk, dtype=torch.int32, device="cuda")}
    if op != "evict":
        s["q"] = normal(sum(nq), case["heads"], d, gain=1.5)
    if op in ("tree", "accept"):
        s |= {"tokens": _indptr(nq), "drafts": max(nq),
              "parents": _trees(nq, case.get("chain", False), gen)}
    if op == "accept":
        half = d // 2
        turn = torch.arange(max(nk), device="cuda", dtype=torch.float64)[:, None] * torch.exp(
            torch.arange(half, device="cuda", dtype=torch.float64) * (-math.log(10000.0) / half))
        s |= {"k": normal(sum(nq), g, d), "v": normal(sum(nq), g, d), "cos": turn.cos().float(),
              "sin": turn.sin().float()}
        # accepted: a random drafted token of each sequence with all before it
        row, pos = _rows(s["tokens"], sum(nq))
        size = (s["tokens"][1:] - s["tokens"][:-1]).long()
        leaf = (torch.rand(case["batch"], generator=gen, device="cuda") * size).long()
        s["keep"] = _ancestors(s)[0][row, leaf[row], pos]
    if op == "evict":
        s |= {"kept_indptr": _indptr(kept), "kept_indices": table[sum(held):].contiguous()}
        keep = torch.zeros(sum(nk), dtype=torch.bool, device="cuda")
        at = 0
        for n, m in zip(nk, _kept(case)):
            keep[at + some(m, n).long()] = True
            at += n
        s |= {"keep": keep, "tokens": _indptr(nk)}
    if own:
        import flagsparse_amd as fs

        s["kv"] = fs.prepare_paged_kv(s["k_pages"], s["v_pages"], s["indptr"], s["indices"])
        if op == "evict":
            s["into"] = fs.prepare_paged_kv(s["k_pages"], s["v_pages"], s["kept_indptr"],
                                            s["kept_indices"])
    return s


def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


# ---- the framework's calls ----


def _own_decode(s):
    import flagsparse_amd as fs

    c = s["case"]
    return fs.flagsparse_attention_paged(s["q"], s["lengths"], prepared=s["kv"], window=c["window"],
                                         sinks=c["sinks"], return_lse=c["lse"])


def _own_packed(s):
    import flagsparse_amd as fs

    c = s["case"]
    return fs.flagsparse_attention_packed(s["q"], s["k"], s["v"], prepared=s["pattern"],
                                          window=c["window"], sinks=c["sinks"], return_lse=True)


def _own_train(s):
    import flagsparse_amd as fs

    c = s["case"]
    out, lse = _own_packed(s)
    grads = fs.flagsparse_attention_packed_backward(
        s["grad"], s["q"], s["k"], s["v"], out, lse, prepared=s["pattern"], window=c["window"],
        sinks=c["sinks"])
    return out, lse, *grads


def _own_tree(s):
    import flagsparse_amd as fs

    c = s["case"]
    return fs.flagsparse_attention_paged_tree(
        s["q"], s["lengths"], s["tokens"], parents=None if c["chain"] else s["parents"],
        longest=s["drafts"], prepared=s["kv"], window=c["window"] or None, sinks=c["sinks"],
        return_lse=c["lse"])


def _own_accept(s):
    import flagsparse_amd as fs

    q = fs.flagsparse_paged_append(s["k"], s["v"], s["lengths"], s["tokens"], parents=s["parents"],
                                   prepared=s["kv"], q=s["q"], cos=s["cos"], sin=s["sin"])
    n = fs.flagsparse_paged_keep(s["keep"], s["lengths"], s["tokens"], prepared=s["kv"])
    return q, s["k_pages"], s["v_pages"], n


def _own_evict(s):
    import flagsparse_amd as fs

    n = fs.flagsparse_paged_keep(s["keep"], s["lengths"], s["tokens"], prepared=s["kv"],
                                 into=s["into"])
    return s["k_pages"], s["v_pages"], n


def _own_copy(s):
    import flagsparse_amd as fs

    fs.flagsparse_paged_copy(s["sources"], s["targets"], prepared=s["kv"])
    return s["k_pages"], s["v_pages"]


_own = {"decode": _own_decode, "packed": _own_packed, "train": _own_train, "tree": _own_tree,
        "accept": _own_accept, "evict": _own_evict, "copy": _own_copy}


# ---- the plain form: elementary operations in 32 bits, rounded once ----


def _rows(indptr, n):
    """(sequence, place in it) of each of n packed tokens."""
    at = torch.arange(n, device="cuda")
    row = torch.searchsorted(indptr.long(), at, right=True) - 1
    return row, at - indptr.long()[row]


def _softmax(scores, seen):
    """(weights, log of the sums of exponentials) over the last axis; a row that sees nothing has no
    weights and a logarithm of minus infinity."""
    scores = scores.masked_fill(~seen, _EMPTY)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == _EMPTY, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / total.masked_fill(total == 0, 1.0), (total.log() + top).squeeze(-1)


def _places(s, first, n_max):
    """(positions [batch, n], which of them hold a token): the sinks before ``first`` and what follows
    from ``first`` on, n_max at most."""
    sinks = s["case"]["sinks"]
    e = torch.arange(min(s["longest"], n_max) + sinks, device="cuda")
    first, n = first[:, None], s["lengths"].long()[:, None]
    pos = torch.where(e < sinks, e, first + e - sinks)
    return pos, torch.where(e < sinks, pos < first, pos < n)


def _held(s, pos):
    """Keys [batch, heads, dim, n] and values [batch, heads, n, dim] at the positions, in 32 bits."""
    page = s["case"]["page"]
    at = s["indptr"].long()[:-1, None] + pos // page
    at = s["indices"].long()[at.clamp(max=s["indices"].numel() - 1)]
    k = s["k_pages"][at, pos % page].float().permute(0, 2, 3, 1).contiguous()
    return k, s["v_pages"][at, pos % page].float().permute(0, 2, 1, 3).contiguous()


def _plain_decode(s):
    c = s["case"]
    b, h, g, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    first = (s["lengths"].long() - c["window"]).clamp(min=0)
    pos, seen = _places(s, first, c["window"])
    k, v = _held(s, pos)
    p, lse = _softmax(torch.matmul(s["q"].float().view(b, g, h // g, d), k) * d ** -0.5,
                      seen[:, None, None])
    out = torch.matmul(p, v).reshape(b, h, d).to(s["q"].dtype)
    return (out, lse.reshape(b, h)) if c["lse"] else out


def _ancestors(s):
    """(which drafted tokens lie on the way of each, itself among them [batch, T, T], depths [batch, T])."""
    t = s["drafts"]
    row, pos = _rows(s["tokens"], s["parents"].numel())
    way = torch.eye(t, device="cuda").repeat(s["case"]["batch"], 1, 1)
    up = s["parents"].long()
    on = up >= 0
    way[row[on], pos[on], up[on]] = 1.0
    for _ in range(max(1, t - 1).bit_length()):
        way = (torch.matmul(way, way.clone()) > 0).float()
    return way > 0, way.sum(-1).long() - 1


def _plain_tree(s):
    c = s["case"]
    b, h, g, d, t = c["batch"], c["heads"], c["kv_heads"], c["dim"], s["drafts"]
    w, dt = c["window"], s["q"].dtype
    row, at = _rows(s["tokens"], s["q"].shape[0])
    size = s["tokens"].long()[1:] - s["tokens"].long()[:-1]
    past = s["lengths"].long() - size
    first = (past + 1 - w).clamp(min=0) if w else torch.zeros_like(past)
    pos, there = _places(s, first, w + t if w else s["longest"])
    k, v = _held(s, pos)
    way, depth = _ancestors(s)
    drafted = (pos - past[:, None]).clamp(min=0, max=t - 1)
    cached = pos < past[:, None]
    seen = cached[:, None] | torch.gather(way, 2, drafted[:, None].expand(b, t, pos.shape[1]))
    if w:
        p_key = torch.where(cached, pos, past[:, None] + torch.gather(depth, 1, drafted))[:, None]
        seen &= (p_key > (past[:, None] + depth - w)[:, :, None]) | (p_key < c["sinks"])
    seen &= there[:, None]
    q = torch.zeros(b, t, h, d, device="cuda")
    q[row, at] = s["q"].float()
    q = q.view(b, t, g, h // g, d).permute(0, 2, 1, 3, 4).reshape(b, g, t * (h // g), d)
    seen = seen.repeat_interleave(h // g, 1)[:, None]
    p, lse = _softmax(torch.matmul(q, k) * d ** -0.5, seen)

    def packed(x):
        x = x.reshape(b, g, t, h // g, -1).permute(0, 2, 1, 3, 4).reshape(b, t, h, -1)
        return x[row, at]

    out = packed(torch.matmul(p, v)).to(dt)
    return (out, packed(lse[..., None]).squeeze(-1)) if c["lse"] else out


def _pad(x, indptr, longest):
    """Packed [tokens, heads, dim] as 32-bit [sequences, heads, longest, dim], and each token's place."""
    row, pos = _rows(indptr, x.shape[0])
    y = torch.zeros(indptr.numel() - 1, longest, x.shape[1], x.shape[2], device="cuda")
    y[row, pos] = x.float()
    return y.transpose(1, 2).contiguous(), row, pos


def _plain_scores(s):
    c = s["case"]
    g = c["kv_heads"]
    q, row, pos = _pad(s["q"], s["indptr"], s["longest_q"])
    k, krow, kpos = _pad(s["k"], s["k_indptr"], s["longest_k"])
    v = _pad(s["v"], s["k_indptr"], s["longest_k"])[0]
    q = q.reshape(q.shape[0], g, -1, q.shape[3])  # the queries of a group's heads, one after the other
    iq, ik = s["indptr"].long(), s["k_indptr"].long()
    nq, nk = (iq[1:] - iq[:-1])[:, None, None], (ik[1:] - ik[:-1])[:, None, None]
    i = torch.arange(s["longest_q"], device="cuda")[:, None]
    j = torch.arange(s["longest_k"], device="cuda")
    at = i + nk - nq
    seen = (i < nq) & (j < nk) & (j <= at) & ((j > at - c["window"]) | (j < c["sinks"]))
    scale = c["dim"] ** -0.5
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    p, lse = _softmax(scores, seen.repeat(1, c["heads"] // g, 1)[:, None])
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
    go = _pad(s["grad"], s["indptr"], s["longest_q"])[0].reshape(q.shape)
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


def _turn(x, cos, sin):
    """x [tokens, heads, dim] in 32 bits, its halves rotated as pairs."""
    x, cos, sin = x.float(), cos[:, None], sin[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _slot(s, indptr, indices, row, pos):
    page = s["case"]["page"]
    return indices.long()[indptr.long()[row] + pos // page], pos % page


def _plain_accept(s):
    dt = s["k"].dtype
    tokens, lengths = s["tokens"].long(), s["lengths"].long()
    row, at = _rows(tokens, s["k"].shape[0])
    past = lengths - (tokens[1:] - tokens[:-1])
    turned = past[row] + _ancestors(s)[1][row, at]
    cos, sin = s["cos"][turned], s["sin"][turned]
    q = _turn(s["q"], cos, sin).to(dt)
    here = _slot(s, s["indptr"], s["indices"], row, past[row] + at)
    s["k_pages"][here], s["v_pages"][here] = _turn(s["k"], cos, sin).to(dt), s["v"]
    keep = s["keep"]
    count = torch.cat([keep.new_zeros(1, dtype=torch.long), keep.long().cumsum(0)])
    row, at = row[keep], at[keep]
    to = past[row] + (count[:-1] - count[tokens[:-1]][_rows(tokens, keep.numel())[0]])[keep]
    here = _slot(s, s["indptr"], s["indices"], row, past[row] + at)
    there = _slot(s, s["indptr"], s["indices"], row, to)
    s["k_pages"][there], s["v_pages"][there] = s["k_pages"][here], s["v_pages"][here]
    return q, s["k_pages"], s["v_pages"], (past + count[tokens[1:]] - count[tokens[:-1]]).to(torch.int32)


def _plain_evict(s):
    tokens, keep = s["tokens"].long(), s["keep"]
    row, pos = _rows(tokens, keep.numel())
    count = torch.cat([keep.new_zeros(1, dtype=torch.long), keep.long().cumsum(0)])
    to = (count[:-1] - count[tokens[:-1]][row])[keep]
    here = _slot(s, s["indptr"], s["indices"], row[keep], pos[keep])
    there = _slot(s, s["kept_indptr"], s["kept_indices"], row[keep], to)
    s["k_pages"][there], s["v_pages"][there] = s["k_pages"][here], s["v_pages"][here]
    return s["k_pages"], s["v_pages"], (count[tokens[1:]] - count[tokens[:-1]]).to(torch.int32)


def _plain_copy(s):
    a, b = s["sources"].long(), s["targets"].long()
    s["k_pages"][b], s["v_pages"][b] = s["k_pages"][a], s["v_pages"][a]
    return s["k_pages"], s["v_pages"]


_plain = {"decode": _plain_decode, "packed": _plain_packed, "train": _plain_train, "tree": _plain_tree,
          "accept": _plain_accept, "evict": _plain_evict, "copy": _plain_copy}


# ---- the definition in 64 bits, one sequence and head at a time ----


def _exact_rows(q, k, v, hidden):
    """(out, lse) of one head's queries [n, dim]."""
    x = (q @ k.T) / math.sqrt(q.shape[1])
    x = torch.where(hidden, torch.full_like(x, _EMPTY), x)
    lse = torch.logsumexp(x, 1)
    w = torch.where(hidden, torch.zeros_like(x), torch.exp(x - lse.detach()[:, None]))
    if q.requires_grad:  # the weights' own sum carries the gradient of the logarithm
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    return w @ v, lse


def _exact_paths(parents):
    """For each drafted token the places on its way, from itself up."""
    paths = []
    for i, p in enumerate(parents):
        paths.append([i] + (paths[p] if p >= 0 else []))
    return paths


def _exact_hidden(case, nq, nk, parents):
    """[nq, nk]: what the queries, the last tokens of nk, do not see."""
    j = torch.arange(nk, device="cuda")
    if case["op"] != "tree":
        i = torch.arange(nk - nq, nk, device="cuda")[:, None]
        return (j > i) | ((j <= i - case["window"]) & (j >= case["sinks"]))
    past, paths = nk - nq, _exact_paths(parents)
    hidden = torch.ones(nq, nk, dtype=torch.bool)
    for i, path in enumerate(paths):
        hidden[i, :past] = False
        p = past + len(path) - 1
        if case["window"]:
            hidden[i, min(past, case["sinks"]):min(past, max(0, p - case["window"] + 1))] = True
            hidden[i, :min(past, case["sinks"])] = False
        for up, a in enumerate(path):
            if not case["window"] or up < case["window"] or p - up < case["sinks"]:
                hidden[i, past + a] = False
    return hidden.cuda()


def exact(case, seed):
    global own
    if case["op"] in ("copy", "evict"):
        return None  # nothing is computed
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    nq, nk = _sizes(case)
    if case["op"] == "accept":
        return _exact_accept(case, s, nq, nk)
    h, g = case["heads"], case["kv_heads"]
    q = s["q"].double()
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], _EMPTY, dtype=torch.float64, device="cuda")
    train, paged = case["op"] == "train", case["op"] in ("decode", "tree")
    dq, tq, tk = torch.zeros_like(q), 0, 0
    if not paged:
        k, v = s["k"].double(), s["v"].double()
        dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    else:
        table = s["indptr"].tolist()
    for b in range(case["batch"]):
        if paged:
            pages = s["indices"][table[b]:table[b + 1]].long()
            kb = s["k_pages"][pages].flatten(0, 1)[:nk[b]].double()
            vb = s["v_pages"][pages].flatten(0, 1)[:nk[b]].double()
        else:
            kb, vb = k[tk:tk + nk[b]], v[tk:tk + nk[b]]
        rows = slice(tq, tq + nq[b])
        if nq[b] and nk[b]:
            parents = s["parents"][rows].tolist() if case["op"] == "tree" else None
            hidden = _exact_hidden(case, nq[b], nk[b], parents)
        for a in range(h if nq[b] and nk[b] else 0):
            one = a // (h // g)
            x, y, z = q[rows, a], kb[:, one], vb[:, one]
            if train:
                x, y, z = (t.clone().requires_grad_() for t in (x, y, z))
            o, e = _exact_rows(x, y, z, hidden)
            out[rows, a], lse[rows, a] = o.detach(), e.detach()
            if train:
                gx, gy, gz = torch.autograd.grad(o, (x, y, z), s["grad"][rows, a].double())
                dq[rows, a] = gx
                dk[tk:tk + nk[b], one] += gy
                dv[tk:tk + nk[b], one] += gz
        tq, tk = tq + nq[b], tk + nk[b]
    if paged:
        return (out, lse) if case["lse"] else out
    return (out, lse, dq, dk, dv) if train else (out, lse)


def _exact_accept(case, s, nq, nk):
    """Each pair as a complex number times the table's; then the accepted tokens one after the other."""
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    q, table = s["q"].double(), torch.complex(s["cos"].double(), s["sin"].double())

    def turned(x, turn):
        two = x.reshape(*x.shape[:-1], 2, -1).transpose(-1, -2).contiguous()
        two = torch.view_as_real(torch.view_as_complex(two) * turn[:, None])
        return two.transpose(-1, -2).flatten(-2)

    t, at, lengths = 0, s["indptr"].tolist(), []
    for b in range(case["batch"]):
        new, past = slice(t, t + nq[b]), nk[b] - nq[b]
        if not nq[b]:
            lengths.append(past)
            continue
        depth = torch.tensor([len(p) - 1 for p in _exact_paths(s["parents"][new].tolist())],
                             device="cuda")
        q[new] = turned(q[new], table[past + depth])
        pages = s["indices"][at[b]:at[b + 1]].long()
        pos = torch.arange(past, nk[b], device="cuda")
        here = pages[pos // case["page"]], pos % case["page"]
        k_pages[here] = turned(s["k"][new].double(), table[past + depth])
        v_pages[here] = s["v"][new].double()
        to = past
        for i, stays in enumerate(s["keep"][new].tolist()):
            if stays:
                one, two = divmod(past + i, case["page"]), divmod(to, case["page"])
                for x in (k_pages, v_pages):
                    x[pages[two[0]], two[1]] = x[pages[one[0]], one[1]]
                to += 1
        lengths.append(to)
        t += nq[b]
    return q, k_pages, v_pages, torch.tensor(lengths, dtype=torch.int32, device="cuda")
