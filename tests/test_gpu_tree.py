"""Attention of trees of drafted tokens over a paged cache, against the formulas in 64 bits."""

import copy
import math
import random

import pytest
import torch

import flagsparse_amd as fs
from oracle import attention as ref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _indptr(lengths, dev):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).to(dev)


def _normal(seed, *shape, dtype, gain=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * gain).to(dtype)


def _tree(n, seed, roots=0.1, back=9):
    r = random.Random(seed)
    return [-1 if i == 0 or r.random() < roots else max(0, i - r.randint(1, back)) for i in range(n)]


def _ways(parents):
    ways = []
    for i, p in enumerate(parents):
        ways.append(([] if p < 0 else ways[p]) + [i])
    return ways


def _masks(past, trees, window=None, sinks=0):
    """What each drafted token sees, [drafted, past + drafted] for each sequence, by positions."""
    masks = []
    for n, parents in zip(past, trees):
        m = torch.zeros(len(parents), n + len(parents), dtype=torch.bool)
        for i, way in enumerate(_ways(parents)):
            own = n + len(way) - 1
            seen = [(p, p) for p in range(n)] + [(n + a, n + d) for d, a in enumerate(way)]
            for place, pos in seen:
                m[i, place] = not window or pos > own - window or pos < sinks
        masks.append(m)
    return masks


def _cache(dev, lengths, page, heads, dim, dtype, seed=1, order="tokens", room=0):
    """(prepared cache, keys, values): pages in a random order, NaN where no token lies."""
    held = [-(-n // page) + room for n in lengths]
    gen = torch.Generator().manual_seed(seed)
    indices = torch.randperm(sum(held) + 2, generator=gen)[:sum(held)]
    both, kept = [], []
    for which in (0, 1):
        x = torch.full((sum(held) + 2, page, heads, dim), float("nan"), dtype=dtype)
        rows = [_normal(seed + 10 * b + which + 2, n, heads, dim, dtype=dtype)
                for b, n in enumerate(lengths)]
        at = 0
        for r, m in zip(rows, held):
            full = torch.full((m * page, heads, dim), float("nan"), dtype=dtype)
            full[:len(r)] = r
            x[indices[at:at + m]] = full.view(m, page, heads, dim)
            at += m
        x = x.to(dev)
        both.append(x if order == "tokens" else x.transpose(1, 2).contiguous().transpose(1, 2))
        kept.append(rows)
    return fs.prepare_paged_kv(*both, _indptr(held, dev), indices.to(torch.int32).to(dev)), *kept


def _check(dev, past, trees, page, heads, kv_heads, dim, dtype, window=None, sinks=0, scale=None,
           longest=None, chain=False, order="tokens", room=0):
    new = [len(t) for t in trees]
    print(f"tree {past} + {new} page={page} heads={heads}/{kv_heads} dim={dim} {dtype} "
          f"window={window} sinks={sinks} longest={longest}", flush=True)
    lengths = [a + b for a, b in zip(past, new)]
    kv, k, v = _cache(dev, lengths, page, kv_heads, dim, dtype, order=order, room=room)
    q = _normal(99, sum(new), heads, dim, dtype=dtype, gain=1.5).to(dev)
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = fs.flagsparse_attention_paged_tree(
        q, n, _indptr(new, dev), parents=None if chain else parents, longest=longest, prepared=kv,
        window=window, sinks=sinks, scale=scale, return_lse=True)
    torch.cuda.synchronize()
    want = ref.packed(q, torch.cat(k), torch.cat(v), new, lengths, True, None,
                      dim**-0.5 if scale is None else scale, masks=_masks(past, trees, window, sinks))
    ref.check("out", out, want["out"])
    ref.check("lse", lse, want["lse"])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("past", [[0], [1], [15, 16, 17], [0, 31, 0, 33, 1], [63, 64, 65, 127],
                                  [128, 255, 256, 257], [1000], [2500, 3, 700], [245, 1270]])
def test_lengths(dev, past, dtype):
    _check(dev, past, [_tree(11, s) for s in range(len(past))], 16, 4, 2, 128, dtype)


@pytest.mark.parametrize("new", [[1], [2], [0, 3, 0], [31, 32, 33], [64, 1, 63], [256], [200, 0, 17, 256]])
def test_drafted_tokens(dev, new):
    past = [(37 * i + 5) % 90 for i in range(len(new))]
    trees = [_tree(n, s) for s, n in enumerate(new)]
    _check(dev, past, trees, 16, 4, 2, 64, BF)
    _check(dev, past, trees, 16, 3, 3, 64, HF, longest=max(new))


def test_shapes_of_trees(dev):
    star, deep = [-1] + [0] * 20, [-1] + list(range(40))
    roots = [-1] * 33
    pairs = [-1] + [i // 2 for i in range(62)]
    _check(dev, [70, 3, 0, 300], [star, deep, roots, pairs], 16, 4, 1, 64, BF)
    _check(dev, [70, 3, 0, 300], [star, deep, roots, pairs], 16, 4, 1, 64, BF, window=6, sinks=2)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 48, 64, 72, 80, 96, 112, 120, 128])
def test_dims(dev, dim):
    trees = [_tree(9, 1), _tree(14, 2)]
    _check(dev, [100, 37], trees, 16, 3, 1, dim, HF)
    _check(dev, [100, 37], trees, 16, 4, 4, dim, BF)


@pytest.mark.parametrize("page", [1, 2, 3, 5, 8, 24, 33, 64, 100, 256, 1024])
def test_pages_that_end_anywhere(dev, page):
    trees = [_tree(9, 1), _tree(14, 2), _tree(3, 3)]
    _check(dev, [150, 1, 333], trees, page, 4, 2, 64, BF)
    _check(dev, [150, 1, 333], trees, page, 4, 2, 64, BF, order="heads", room=2)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (8, 1), (15, 1), (16, 1), (17, 1),
                                            (33, 1), (64, 2), (24, 8), (23, 1)])
def test_heads(dev, heads, kv_heads):
    _check(dev, [200, 45], [_tree(5, 1), _tree(8, 2)], 16, heads, kv_heads, 64, BF)
    _check(dev, [200, 45], [_tree(1, 1), _tree(2, 2)], 16, heads, kv_heads, 128, HF)


@pytest.mark.parametrize("sinks", [0, 1, 4, 33, 300, 5000])
@pytest.mark.parametrize("window", [1, 2, 7, 31, 100, 256, 300, 10000])
def test_windows(dev, window, sinks):
    _check(dev, [0, 3, 64, 300, 700], [_tree(20, s, back=3) for s in range(5)], 16, 4, 2, 64, HF,
           window=window, sinks=sinks)


def test_windows_smaller_than_a_tree_is_deep(dev):
    deep = [-1] + list(range(99))
    for window, sinks in ((1, 0), (3, 0), (10, 12), (40, 1), (99, 0), (100, 0)):
        _check(dev, [0, 8, 50], [deep, _tree(100, 1, back=2), deep], 16, 2, 1, 64, BF, window=window,
               sinks=sinks)


def test_chains(dev):
    chains = [[-1] + list(range(n - 1)) for n in (5, 1, 70)]
    _check(dev, [90, 0, 400], chains, 16, 4, 2, 64, BF, chain=True)
    _check(dev, [90, 0, 400], chains, 16, 4, 2, 128, HF, chain=True, window=20, sinks=3)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.25])
def test_scale(dev, scale):
    _check(dev, [90, 200], [_tree(6, 1), _tree(7, 2)], 16, 2, 1, 64, HF, scale=scale)


def test_long_sequences(dev):
    _check(dev, [30011], [_tree(21, 1)], 64, 8, 1, 128, BF)
    _check(dev, [20000, 5, 9000], [_tree(64, 1), _tree(3, 2), _tree(40, 3)], 32, 2, 2, 64, HF)
    _check(dev, [30000, 20000], [_tree(33, 1), _tree(12, 2)], 64, 8, 2, 128, BF, window=4096, sinks=64)


def test_many_sequences(dev):
    past = [(7 * i) % 40 for i in range(300)]
    _check(dev, past, [_tree(i % 5, i) for i in range(300)], 8, 2, 1, 64, BF)


def test_one_token_is_the_paged_call(dev):
    lengths = [300, 50, 1, 0]
    kv, k, v = _cache(dev, lengths, 16, 2, 64, BF)
    q, n = _normal(9, 4, 8, 64, dtype=BF).to(dev), torch.tensor([300, 50, 1, 17], device=dev)
    got = fs.flagsparse_attention_paged_tree(q, n, prepared=kv)
    want = ref.packed(q[:3], torch.cat(k), torch.cat(v), [1] * 3, lengths[:3], True, None, 0.125)
    ref.check("out", got[:3], want["out"])
    assert torch.isnan(got[3]).all()  # its pages hold nothing


@pytest.mark.parametrize("heads", [2, 24, 40])
def test_one_token_under_a_window_that_starts_anywhere(dev, heads):
    # a piece that ends where all see its keys, in a step that is not whole; LDS holds what others left
    x = _normal(5, 4096, 8, 128, dtype=BF).to(dev)
    fs.flagsparse_attention_packed(x, x, x, torch.tensor([0, 4096], device=dev))
    past = list(range(230, 790))
    _check(dev, past, [[-1]] * len(past), 16, heads, 1, 64, BF, window=100)


def test_lists_stay_for_the_graphs_that_read_them(dev):
    kv, _, _ = _cache(dev, [300], 16, 1, 64, BF)
    n = torch.tensor([300], dtype=torch.int32, device=dev)
    q = _normal(3, 4, 2, 64, dtype=BF).to(dev)
    fs.flagsparse_attention_paged_tree(q, n, prepared=kv, window=9)
    (first,) = kv._lists.values()
    for window in range(10, 140):
        fs.flagsparse_attention_paged_tree(q, n, prepared=kv, window=window)
    assert any(kept is first for kept in kv._lists.values())


def test_as_many_tokens_as_a_table_may_hold(dev):
    # one page for all places: the softmax is that of one page, the sum of the weights is that of them all
    page, times = 1 << 20, 2047
    k = _normal(1, 1, page, 1, 8, dtype=BF).to(dev)
    v = _normal(2, 1, page, 1, 8, dtype=BF).to(dev)
    kv = fs.prepare_paged_kv(k, v, torch.tensor([0, times], device=dev), torch.zeros(times, dtype=torch.int32,
                                                                                    device=dev))
    q = _normal(3, 1, 2, 8, dtype=BF).to(dev)
    n = torch.tensor([page * times], dtype=torch.int32, device=dev)
    out, lse = fs.flagsparse_attention_paged_tree(q, n, prepared=kv, return_lse=True)
    s = (k[0, :, 0].double() @ q[0].double().T) * 8**-0.5  # [page, heads]
    want = torch.softmax(s, 0).T @ v[0, :, 0].double()
    # a weight and the result are rounded to 8 bits, half a step each; sums in 32 bits are small beside it
    bound = 2 * 2.0**-8 * (torch.softmax(s, 0).T @ v[0, :, 0].double().abs())
    assert bool(((out[0].double() - want).abs() <= bound).all())
    # sums in 32 bits, of all 2^18 pieces of 8192 keys one after the other, and a factor for each 8 of them: at most
    # (2^18 + 2^15) 2^-24 of the sum; in a piece 2^9 a lane, 2^-15; weights and scores some 2^-20 more
    assert float((lse[0].double() - (torch.logsumexp(s, 0) + math.log(times))).abs().max()) <= 2.0**-5


def test_what_is_not_as_it_should_be_is_nan(dev):
    past, new = [90, 40, 7], [9, 12, 5]
    trees = [_tree(n, s) for s, n in enumerate(new)]
    kv, k, v = _cache(dev, [a + b for a, b in zip(past, new)], 16, 2, 64, BF)
    q = _normal(9, 30, 4, 64, dtype=BF).to(dev)
    tokens = torch.tensor([1, 10, 22, 27], device=dev)  # a row before the first, three after the last
    n = torch.tensor([99, 52, 12], device=dev)
    flat = [0] + [p for t in trees for p in t] + [0, 0, 0]
    parents = torch.tensor(flat, device=dev)

    def call(**kw):
        out, lse = fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, prepared=kv,
                                                      return_lse=True, **kw)
        bad = torch.isnan(out.float()).all(-1)
        assert torch.equal(bad, torch.isnan(out.float()).any(-1)) and torch.equal(bad, torch.isnan(lse))
        assert torch.equal(bad.any(1), bad.all(1))
        return bad.all(1).cpu().nonzero().flatten().tolist()

    outside = [0, 27, 28, 29]
    assert call() == outside and call(longest=12) == outside
    assert call(longest=9) == [0, *range(10, 22), 27, 28, 29]
    for bad in (8, -1, 113, 2**40):  # less than the drafted tokens, or more than the pages hold
        n[0] = bad
        assert call() == [*range(10), 27, 28, 29]
    n[0] = 99
    # a parent that does not come earlier takes its token and those after it on their ways
    for bad in (4, 5, 100, -2, -2**40, 2**40):
        parents[1 + 4] = bad
        fallen = [1 + i for i, way in enumerate(_ways(trees[0])) if 4 in way]
        assert call() == sorted(outside + fallen)
        assert call(window=3) == sorted(outside + fallen)
    parents[5] = flat[5]
    # tokens that lead nowhere
    for bad in ([0, -5, 22, 27], [0, 50, 22, 27], [-3, 10, 22, 27], [2**33, 10, 22, 2**33]):
        tokens.copy_(torch.tensor(bad))
        call()
    torch.cuda.synchronize()


def test_hidden_keys_may_be_anything(dev):
    # keys of other branches, and those behind the sinks and before the window
    past, trees = [500], [[-1, 0, 0, 1, 2, 3, 4]]
    kv, k, v = _cache(dev, [507], 16, 2, 64, HF)
    q, n = _normal(5, 7, 4, 64, dtype=HF).to(dev), torch.tensor([507], device=dev)
    parents = torch.tensor(trees[0], device=dev)

    def call(**kw):
        return fs.flagsparse_attention_paged_tree(q, n, parents=parents, prepared=kv, **kw)

    clean, near = call(), call(window=100, sinks=5)
    at = 500 + 2
    kv.k_pages[kv.indices[at // 16].long(), at % 16] = float("nan")
    dirty = call()
    for row, way in enumerate(_ways(trees[0])):
        assert torch.isnan(dirty[row]).all() if 2 in way else torch.equal(dirty[row], clean[row])
    kv.k_pages[kv.indices[at // 16].long(), at % 16] = k[0][at].to(dev)
    hidden = torch.arange(5, 401, device=dev)
    kv.k_pages[kv.indices.long()[hidden // 16], hidden % 16] = float("inf")
    kv.v_pages[kv.indices.long()[hidden // 16], hidden % 16] = float("nan")
    assert torch.equal(call(window=100, sinks=5), near)


def test_strides_outputs_and_index_types(dev):
    past, new = [64, 20], [3, 4]
    trees = [_tree(n, s) for s, n in enumerate(new)]
    kv, k, v = _cache(dev, [67, 24], 16, 2, 64, HF)
    fused = _normal(5, 7, 8, 64, dtype=HF).to(dev)
    q = fused[:, 2:6]
    n, tokens = torch.tensor([67, 24], device=dev), torch.tensor([0, 3, 7], device=dev)
    parents = torch.tensor([p for t in trees for p in t], device=dev)
    out = torch.zeros(4, 7, 64, dtype=HF, device=dev).transpose(0, 1)
    assert fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, prepared=kv, out=out) is out
    want = ref.packed(q, torch.cat(k), torch.cat(v), new, [67, 24], True, None, 0.125,
                      masks=_masks(past, trees))
    ref.check("out", out, want["out"])
    odd = torch.zeros(7, 4, 65, dtype=HF, device=dev)[:, :, 1:]
    fs.flagsparse_attention_paged_tree(q, n.int(), tokens.int(), parents=parents.int(), prepared=kv, out=odd)
    assert torch.equal(odd, out)
    same = q.clone()
    fs.flagsparse_attention_paged_tree(same, n, tokens, parents=parents, prepared=kv, out=same)
    assert torch.equal(same, out)
    direct = fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, k_pages=kv.k_pages,
                                                v_pages=kv.v_pages, indptr=kv.indptr, indices=kv.indices)
    assert torch.equal(direct, out)


def test_graphs_streams_and_equal_bits(dev):
    past, new = [900, 3, 2000, 77], [20, 64, 0, 9]
    trees = [_tree(n, s) for s, n in enumerate(new)]
    kv, _, _ = _cache(dev, [a + b for a, b in zip(past, new)], 16, 2, 128, BF)
    n = torch.tensor([a + b for a, b in zip(past, new)], dtype=torch.int32, device=dev)
    q, tokens = _normal(2, 93, 16, 128, dtype=BF).to(dev), _indptr(new, dev)
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)

    def step(kv=kv):
        return fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, longest=64, prepared=kv,
                                                  return_lse=True)

    graph = torch.cuda.CUDAGraph()
    want = step()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    with torch.cuda.graph(graph):
        got = step()
    for lengths in ([920, 67, 2000, 86], [500, 66, 1000, 80], [920, 67, 2000, 86]):
        n.copy_(torch.tensor(lengths))
        eager = step()
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, got))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    again = copy.deepcopy(kv)
    for _, pieces, _, _, _ in kv._lists.values():
        pieces.zero_()  # the copy works on its own arrays
    assert all(torch.equal(a, b) for a, b in zip(want, step(again)))


def test_a_capture_needs_a_call_before(dev):
    kv, _, _ = _cache(dev, [40], 16, 1, 64, BF)
    q, n = _normal(1, 4, 2, 64, dtype=BF).to(dev), torch.tensor([40], dtype=torch.int32, device=dev)
    kv._on()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(graph):
            fs.flagsparse_attention_paged_tree(q, n, prepared=kv)


def test_offsets_past_32_bits(dev):
    pages, page, g, d = 17000, 64, 16, 128
    kp = torch.empty(pages, page, g, d, dtype=BF, device=dev)
    vp = torch.empty(pages, page, g, d, dtype=BF, device=dev)
    assert kp.numel() > 2**31
    ix = torch.tensor([pages - 1, 3, pages - 2], dtype=torch.int32, device=dev)
    n = torch.tensor([150], dtype=torch.int32, device=dev)
    kv = fs.prepare_paged_kv(kp, vp, torch.tensor([0, 3], device=dev), ix)
    k, v = (_normal(s, 150, g, d, dtype=BF) for s in (1, 2))
    fs.flagsparse_paged_append(k.to(dev), v.to(dev), n, torch.tensor([0, 150], device=dev), prepared=kv)
    tree = _tree(10, 1)
    q = _normal(3, 10, g, d, dtype=BF).to(dev)
    got = fs.flagsparse_attention_paged_tree(q, n, parents=torch.tensor(tree, device=dev), prepared=kv)
    ref.check("out", got, ref.packed(q, k, v, [10], [150], True, None, d**-0.5,
                                     masks=_masks([140], [tree]))["out"])


def test_refusals(dev):
    kv, _, _ = _cache(dev, [40, 30], 16, 2, 64, BF)
    q = _normal(1, 6, 4, 64, dtype=BF).to(dev)
    n, tokens = torch.tensor([40, 30], device=dev), torch.tensor([0, 2, 6], device=dev)
    call = fs.flagsparse_attention_paged_tree
    for bad in ({"longest": -1}, {"longest": 257}, {"sinks": 3}, {"window": 0}, {"scale": float("nan")},
                {"parents": torch.zeros(5, dtype=torch.int32, device=dev)},
                {"parents": torch.zeros(6, dtype=torch.int32)}):
        with pytest.raises(ValueError):
            call(q, n, tokens, prepared=kv, **bad)
    with pytest.raises(TypeError):
        call(q, n, tokens, prepared=kv, parents=torch.zeros(6, device=dev))
    for bad in ((q[:5], n, None), (q, n[:1], tokens), (q, n, tokens[:2]), (q[:, :3], n, tokens),
                (q, n.cpu(), tokens), (q[:, :, :56], n, tokens)):
        with pytest.raises(ValueError):
            call(*bad, prepared=kv)
    with pytest.raises(ValueError):
        call(q, n, prepared=kv, longest=2)
    # without a prepared cache the indices are checked too
    cache = {"k_pages": kv.k_pages, "v_pages": kv.v_pages, "indptr": kv.indptr, "indices": kv.indices}
    for kw in ({"parents": torch.tensor([-1, 1, -1, 0, 0, 0], device=dev)},
               {"parents": torch.tensor([-1, 0, -1, 0, -2, 0], device=dev)}, {"longest": 3}):
        with pytest.raises(ValueError):
            call(q, n, tokens, **kw, **cache)
    for bad in ([0, 3, 5], [1, 2, 6], [0, 7, 6]):
        with pytest.raises(ValueError):
            call(q, n, torch.tensor(bad, device=dev), **cache)
    with pytest.raises(ValueError):
        call(q, torch.tensor([40, 3], device=dev), tokens, **cache)


def test_no_tokens(dev):
    kv, _, _ = _cache(dev, [40, 30], 16, 2, 64, BF)
    q = torch.empty(0, 4, 64, dtype=BF, device=dev)
    n, tokens = torch.tensor([40, 30], device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    for t in (None, tokens):
        out, lse = fs.flagsparse_attention_paged_tree(q, n, t, prepared=kv, return_lse=True)
        assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    empty = fs.prepare_paged_kv(kv.k_pages, kv.v_pages, torch.tensor([0], device=dev),
                                torch.zeros(0, dtype=torch.int32, device=dev))
    q = torch.zeros(3, 4, 64, dtype=BF, device=dev)
    out = fs.flagsparse_attention_paged_tree(q, n[:0], torch.zeros(1, dtype=torch.int32, device=dev),
                                             prepared=empty)
    assert torch.isnan(out).all()


def _long_cache(dev, batch, pages, heads, dim, dtype):
    """A cache of ``batch`` sequences with room for pages * 64 tokens each, all in the same pages."""
    k, v = (_normal(s, pages, 64, heads, dim, dtype=dtype).to(dev) for s in (1, 2))
    table = torch.arange(pages, dtype=torch.int32, device=dev).repeat(batch)
    return fs.prepare_paged_kv(k, v, torch.arange(0, batch * pages + 1, pages, device=dev), table)


def test_memory_goes_by_the_drafted_tokens(dev):
    # no bound of the drafted tokens, room for long texts: what a call takes goes by the tokens that there are
    batch, heads, dim, each = 64, 16, 64, 6
    kv = _long_cache(dev, batch, 512, 4, dim, BF)
    n = torch.full((batch,), 900, dtype=torch.int32, device=dev)
    q, tokens = _normal(3, batch * each, heads, dim, dtype=BF).to(dev), _indptr([each] * batch, dev)
    parents = torch.full((batch * each,), -1, dtype=torch.int32, device=dev)
    want = fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, longest=each, prepared=kv)
    assert fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, prepared=kv).shape == q.shape
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(dev)
    before = torch.cuda.memory_allocated(dev)
    out = fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, prepared=kv)
    torch.cuda.synchronize()
    taken = torch.cuda.max_memory_allocated(dev) - before
    # pieces of 256 tokens at least, the output beside them; the allocator gives a block whole where less than 1 MiB
    # of it would be left
    assert taken <= 512 * 64 // 256 * batch * each * heads * (dim + 2) * 4 + 2 * q.numel() + (2 << 20), taken
    # two orders of the same sums, weights rounded to 8 bits by other maxima in each
    s = float(kv.v_pages.float().abs().max())
    assert float((out.float() - want.float()).abs().max()) <= 4 * 2.0**-8 * s


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (23, 1, 80)])
def test_partial_sums_of_ragged_trees(dev, heads, kv_heads, dim):
    # many pieces, drafts of very different sizes, with a bound of them and without: sums by pieces and by tokens
    past, new = [9000, 30, 4000, 0, 700], [3, 90, 0, 5, 1]
    trees = [_tree(n, s) for s, n in enumerate(new)]
    _check(dev, past, trees, 64, heads, kv_heads, dim, BF)
    _check(dev, past, trees, 64, heads, kv_heads, dim, HF, longest=90, window=3000, sinks=7)
    past, new = [6000, 5000, 300], [4, 4, 4]
    trees = [_tree(n, s) for s, n in enumerate(new)]
    _check(dev, past, trees, 64, heads, kv_heads, dim, BF, longest=4)
    _check(dev, past, trees, 64, heads, kv_heads, dim, HF, room=60)


@pytest.mark.parametrize("heads,window,sinks", [(4, None, 0), (12, 700, 5)])
def test_other_numbers_of_drafts_use_the_same_lists(dev, heads, window, sinks):
    # after the first call of a program others build nothing: they can be captured whatever they draft
    kv = _long_cache(dev, 4, 100, 2, 64, BF)
    n = torch.full((4,), 6000, dtype=torch.int32, device=dev)

    def call(new, longest=None):
        q = _normal(sum(new), sum(new), heads, 64, dtype=BF).to(dev)
        tokens, parents = _indptr(new, dev), torch.full((sum(new),), -1, dtype=torch.int32, device=dev)

        def run():
            return fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, longest=longest, prepared=kv,
                                                      window=window, sinks=sinks)
        return run

    call([1, 0, 2, 1])()
    lists, streams = list(kv._lists), torch.cuda.Stream(dev)
    for new, longest in (([3, 3, 3, 3], 3), ([20, 1, 0, 7], None), ([256, 256, 256, 256], None), ([40, 1, 2, 3], 64)):
        run, graph = call(new, longest), torch.cuda.CUDAGraph()
        streams.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.graph(graph, stream=streams):
            got = run()
        for _ in range(2):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, run())
    assert list(kv._lists) == lists


def test_what_is_not_finite_between_the_windows_of_rows(dev):
    # text that the windows of less deep rows hold and those of deeper rows do not
    past, trees, window = [500, 40], [[-1, 0, 1, 2, 3, 4, 5], [-1, -1]], 100
    kv, k, v = _cache(dev, [507, 42], 16, 2, 64, HF)
    q, n = _normal(5, 9, 4, 64, dtype=HF).to(dev), torch.tensor([507, 42], device=dev)
    parents, tokens = torch.tensor(sum(trees, []), device=dev), _indptr([7, 2], dev)

    def call(**kw):
        return fs.flagsparse_attention_paged_tree(q, n, tokens, parents=parents, prepared=kv, window=window, **kw)

    def at(place):
        return kv.indices[place // 16].long(), place % 16

    clean = call()
    for place, sees in ((400, 0), (401, 1), (403, 3), (407, 7)):  # position 500 + depth sees what is past 400 + depth
        kv.k_pages[at(place)] = float("nan")
        dirty = call()
        assert torch.isnan(dirty[:sees]).all() and torch.equal(dirty[sees:], clean[sees:])
        kv.k_pages[at(place)] = k[0][place].to(dev)
        for bad in (float("nan"), float("inf")):
            kv.v_pages[at(place)] = bad
            dirty = call()
            assert not torch.isfinite(dirty[:sees]).any() and torch.equal(dirty[7:], clean[7:])
            if sees == 0:  # before all windows: not read
                assert torch.equal(dirty, clean)
        kv.v_pages[at(place)] = v[0][place].to(dev)
    assert torch.equal(call(), clean)


def test_the_ends_of_as_many_tokens_as_a_table_may_hold_count_once(dev):
    # keys of score 0 in one page for all places but the first, one in the middle and the last, each of whose pages has
    # one key that weighs as much as all others or more, at its first, an inner and its last place
    page, times = 1 << 20, 2047
    k, v = (torch.zeros(4, page, 1, 8, dtype=BF, device=dev) for _ in range(2))
    v[0] = 1
    table = torch.zeros(times, dtype=torch.int32, device=dev)
    heavy = ((0, 1, 0, 8.0), (1000, 2, 777777, -8.0), (times - 1, 3, page - 1, 8.0))
    for entry, which, slot, value in heavy:
        table[entry] = which
        v[which] = 1
        k[which, slot], v[which, slot] = 2, value
    kv = fs.prepare_paged_kv(k, v, torch.tensor([0, times], device=dev), table)
    q = torch.full((1, 2, 8), 4.0, dtype=BF, device=dev)
    q[0, 1] = 3.875
    n = torch.tensor([page * times], dtype=torch.int32, device=dev)
    out, lse = fs.flagsparse_attention_paged_tree(q, n, prepared=kv, return_lse=True)
    others = page * times - 3
    for head, x in enumerate((4.0, 3.875)):
        w = math.exp(8 * 2 * x * 8**-0.5)
        total = others + 3 * w
        want = (others + w * sum(value for _, _, _, value in heavy)) / total
        # sums in 32 bits of 2^18 pieces in turn, (2^18 + 2^15) 2^-24 and 2^-15 in a piece, less than 2^-5 of the sum,
        # above and below; weights and the result are rounded to 8 bits.  A heavy key twice or
        # not at all is off by twice as much
        bound = (2 * 2.0**-5 + 2 * 2.0**-8) * (others + 24 * w) / total
        assert float((out[0, head].double() - want).abs().max()) <= bound, (head, out[0, head], want, bound)
        assert abs(float(lse[0, head]) - math.log(total)) <= 2.0**-5
