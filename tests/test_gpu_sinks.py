"""Windows with first tokens that stay visible: packed attention, its gradient, and one new token over a
paged cache, against the formulas in 64 bits."""

import copy

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


def _inputs(dev, q_len, k_len, heads, kv_heads, dim, dtype, seed=1):
    return (_normal(seed, sum(q_len), heads, dim, dtype=dtype, gain=1.5).to(dev),
            _normal(seed + 1, sum(k_len), kv_heads, dim, dtype=dtype).to(dev),
            _normal(seed + 2, sum(k_len), kv_heads, dim, dtype=dtype).to(dev),
            _normal(seed + 3, sum(q_len), heads, dim, dtype=dtype).to(dev))


def _both(dev, q_len, k_len, heads, kv_heads, dim, dtype, window, sinks, scale=None, seed=1):
    print(f"attention {q_len} {k_len} heads={heads}/{kv_heads} dim={dim} {dtype} window={window} "
          f"sinks={sinks}", flush=True)
    q, k, v, g = _inputs(dev, q_len, k_len, heads, kv_heads, dim, dtype, seed)
    kw = {"window": window, "sinks": sinks, "scale": scale}
    ip, kp = _indptr(q_len, dev), _indptr(k_len, dev)
    out, lse = fs.flagsparse_attention_packed(q, k, v, ip, kp, return_lse=True, **kw)
    grads = fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, ip, kp, **kw)
    torch.cuda.synchronize()
    want = ref.packed(q, k, v, q_len, k_len, True, window, dim**-0.5 if scale is None else scale, g,
                      sinks=sinks)
    for name, got in zip(("out", "lse", "q", "k", "v"), (out, lse, *grads)):
        ref.check(name, got, want[name])


@pytest.mark.parametrize("sinks", [1, 4, 31, 32, 33, 63, 64, 65, 130, 1000])
@pytest.mark.parametrize("window", [1, 2, 64, 65, 200])
def test_window_and_sinks(dev, window, sinks):
    _both(dev, [300, 40, 129], [300, 40, 129], 4, 2, 64, BF, window, sinks)
    _both(dev, [100, 200], [333, 150], 2, 1, 128, HF, window, sinks)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lengths", [[1], [2, 1], [31, 33], [64, 0, 63], [65], [127, 128, 129],
                                     [255, 1, 257], [700]])
def test_lengths(dev, lengths, dtype):
    _both(dev, lengths, lengths, 4, 2, 64, dtype, 17, 3)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [8, 24, 40, 64, 72, 96, 104, 120, 128])
def test_dims(dev, dim, dtype):
    _both(dev, [150, 70], [150, 70], 3, 1, dim, dtype, 20, 5)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (7, 1), (16, 2), (24, 8), (9, 3), (60, 4)])
def test_heads(dev, heads, kv_heads):
    _both(dev, [90, 300], [90, 300], heads, kv_heads, 128, BF, 70, 4)


@pytest.mark.parametrize("q_len,k_len", [([5, 200], [300, 1]), ([200], [40]), ([130, 64], [0, 64]),
                                         ([0, 70], [70, 0]), ([1, 1, 1], [500, 65, 2]),
                                         ([300], [129]), ([0, 0, 3], [9, 0, 900])])
def test_other_keys(dev, q_len, k_len):
    # more queries than keys: the first ones see nothing; and keys that no query sees
    _both(dev, q_len, k_len, 4, 2, 64, BF, 30, 7)
    _both(dev, q_len, k_len, 2, 2, 128, HF, 5, 80)


def test_no_queries(dev):
    _both(dev, [0, 0], [9, 700], 2, 2, 64, BF, 30, 7)
    _both(dev, [0], [100], 4, 1, 96, HF, 30, 70)


def test_many_first_keys(dev):
    # jobs hold as many queries as there are first keys
    _both(dev, [1900, 100], [1900, 100], 2, 1, 64, BF, 50, 700)
    _both(dev, [1300], [1500], 4, 2, 128, HF, 3, 1200)


def test_jobs_of_queries(dev):
    # first keys under more queries than one job of 512 or of the window has, in ragged batches
    _both(dev, [1700], [1700], 2, 1, 64, BF, 100, 4)
    _both(dev, [511, 512, 513, 0, 1030, 3], [511, 512, 513, 0, 1030, 3], 4, 2, 64, HF, 20, 70)
    _both(dev, [1500, 30], [1600, 700], 2, 2, 128, BF, 600, 33)
    _both(dev, [1] * 70 + [600] + [2] * 70, [1] * 70 + [600] + [2] * 70, 2, 1, 64, BF, 8, 2)


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("lengths,heads", [([64], 4), ([65] * 3, 60), ([600], 40), ([520, 3], 54),
                                           ([2100], 16)])
def test_shares_of_a_tile(dev, lengths, heads, dim):
    # few and many workgroups, shares of a group's heads
    _both(dev, lengths, lengths, heads, 2, dim, BF, 530, 6)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_scale(dev, scale):
    _both(dev, [100, 20], [100, 20], 2, 1, 32, HF, 11, 2, scale=scale)


def test_no_window_to_leave_is_the_causal_call(dev):
    # a window that holds everything, and first keys that reach into it, hide nothing
    lengths = [300, 20]
    q, k, v, g = _inputs(dev, lengths, lengths, 4, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev))
    want = ref.packed(q, k, v, lengths, lengths, True, None, 0.125, g)
    for window, sinks in ((300, 5), (2**31 - 1, 2**31 - 1), (10, 300), (2**40, 2**40), (1, 299)):
        kw = {"prepared": p, "window": window, "sinks": sinks}
        out, lse = fs.flagsparse_attention_packed(q, k, v, return_lse=True, **kw)
        grads = fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, **kw)
        for name, got in zip(("out", "lse", "q", "k", "v"), (out, lse, *grads)):
            ref.check(name, got, want[name])


def test_no_sinks_is_the_call_without(dev):
    lengths = [200, 20]
    q, k, v, g = _inputs(dev, lengths, lengths, 4, 2, 64, HF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev))
    for sinks in (0, None):
        out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, window=30, sinks=sinks,
                                                  return_lse=True)
        want, _ = fs.flagsparse_attention_packed(q, k, v, prepared=p, window=30, return_lse=True)
        assert torch.equal(out, want)


def test_autograd_is_the_backward_call(dev):
    lengths = [100, 31]
    q, k, v, g = _inputs(dev, lengths, lengths, 4, 2, 64, HF)
    kw = {"prepared": fs.prepare_attention_packed(_indptr(lengths, dev)), "window": 40, "sinks": 3}
    out, lse = fs.flagsparse_attention_packed(q, k, v, return_lse=True, **kw)
    want = fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, **kw)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    res = fs.flagsparse_attention_packed(*leaves, **kw)
    res.backward(g)
    assert torch.equal(res, out)
    for t, w in zip(leaves, want):
        assert torch.equal(t.grad, w)


def test_gradient_against_differences(dev):
    # the slope of f(t) = sum(grad * out(x + t d)) in 64 bits by central differences, against the
    # kernels' gradient along d
    lengths, h, g, d, t, window, sinks = [40, 23], 2, 1, 64, 1e-5, 9, 3
    q, k, v, grad = _inputs(dev, lengths, lengths, h, g, d, HF)
    ip = _indptr(lengths, dev)
    kw = {"window": window, "sinks": sinks}
    out, lse = fs.flagsparse_attention_packed(q, k, v, ip, return_lse=True, **kw)
    grads = fs.flagsparse_attention_packed_backward(grad, q, k, v, out, lse, ip, **kw)
    want = ref.packed(q, k, v, lengths, lengths, True, window, d**-0.5, grad, sinks=sinks)
    xs = [x.cpu().double() for x in (q, k, v)]

    def f(*a):
        total, at = 0.0, 0
        for n in lengths:
            m = ref.seen(n, n, True, window, sinks)
            for head in range(h):
                r = ref.one(a[0][at:at + n, head], a[1][at:at + n, head // (h // g)],
                            a[2][at:at + n, head // (h // g)], m, d**-0.5)
                total += float((r["out"] * grad[at:at + n, head].cpu().double()).sum())
            at += n
        return total

    for which, name in enumerate("qkv"):
        gen = torch.Generator().manual_seed(which)
        way = torch.randn(xs[which].shape, generator=gen, dtype=torch.float64)
        up, down = list(xs), list(xs)
        up[which], down[which] = xs[which] + t * way, xs[which] - t * way
        slope = (f(*up) - f(*down)) / (2 * t)
        got = float((grads[which].cpu().double() * way).sum())
        bound = float((ref.SLACK * want[name][1] * way.abs()).sum())
        # differences: t^2 of third derivatives, and 2^-52 |f| / t of rounding
        assert abs(got - slope) <= bound + 1e-6 * (1 + abs(slope)), (name, got, slope, bound)


def test_equal_bits_graphs_and_streams(dev):
    lengths = [900, 1, 633]
    q, k, v, g = _inputs(dev, lengths, lengths, 8, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev))
    kw = {"prepared": p, "window": 100, "sinks": 5}

    def both():
        out, lse = fs.flagsparse_attention_packed(q, k, v, return_lse=True, **kw)
        return (out, lse, *fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, **kw))

    first = both()
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        eager = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, got, eager))
    again = copy.deepcopy(p)
    p._sequences.zero_()  # the copy works on its own arrays
    for t in p._tiles.values():
        t.zero_()
    kw["prepared"] = again
    assert all(torch.equal(a, b) for a, b in zip(first, both()))


def test_sequences_do_not_touch_each_other(dev):
    lengths = [77, 50, 530, 9]
    q, k, v, g = _inputs(dev, lengths, lengths, 4, 2, 64, BF)
    kw = {"prepared": fs.prepare_attention_packed(_indptr(lengths, dev)), "window": 20, "sinks": 6}

    def both():
        out, lse = fs.flagsparse_attention_packed(q, k, v, return_lse=True, **kw)
        return (out, lse, *fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, **kw))

    clean = both()
    bad = slice(77, 127)
    for t in (q, k, v, g):
        t[bad] = float("nan")
    dirty = both()
    keep = torch.ones(sum(lengths), dtype=torch.bool, device=dev)
    keep[bad] = False
    for a, b in zip(clean, dirty):
        assert torch.equal(a[keep], b[keep])


def test_keys_out_of_sight_may_be_anything(dev):
    # keys behind the first ones and before the window, chosen away whatever they are
    n, window, sinks = 400, 50, 4
    q, k, v, _ = _inputs(dev, [n], [n], 2, 2, 64, BF)
    ip = _indptr([n], dev)
    clean = fs.flagsparse_attention_packed(q, k, v, ip, window=window, sinks=sinks)
    k[sinks:100] = float("nan")
    out = fs.flagsparse_attention_packed(q, k, v, ip, window=window, sinks=sinks)
    last = 100 + window - 1  # the first query that has left them all
    assert torch.equal(out[:sinks], clean[:sinks]) and torch.equal(out[last:], clean[last:])
    assert torch.isnan(out[sinks:last]).all()


def test_refusals(dev):
    q = _normal(1, 8, 2, 64, dtype=BF).to(dev)
    ip = _indptr([8], dev)
    for kw in ({"sinks": 4}, {"sinks": -1, "window": 3}, {"sinks": 2, "causal": False},
               {"sinks": 2, "window": 3, "causal": False}):
        with pytest.raises(ValueError):
            fs.flagsparse_attention_packed(q, q, q, ip, **kw)
        lse = torch.zeros(8, 2, device=dev)
        with pytest.raises(ValueError):
            fs.flagsparse_attention_packed_backward(q, q, q, q, q, lse, ip, **kw)
    pages = q.view(1, 8, 2, 64)
    kv = fs.prepare_paged_kv(pages, pages, torch.tensor([0, 1], device=dev),
                             torch.tensor([0], device=dev))
    n = torch.tensor([8], device=dev)
    for kw in ({"sinks": 4}, {"sinks": -1, "window": 3}):
        with pytest.raises(ValueError):
            fs.flagsparse_attention_paged(q[:1], n, prepared=kv, **kw)


# ---- one new token over a cache ----


def _cache(dev, lengths, page, heads, dim, dtype, seed=1):
    """(prepared cache, keys, values): pages in a random order, NaN where no token lies."""
    held = [-(-n // page) for n in lengths]
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
        both.append(x.to(dev))
        kept.append(rows)
    return fs.prepare_paged_kv(*both, _indptr(held, dev), indices.to(torch.int32).to(dev)), *kept


def _decode(dev, lengths, page, heads, kv_heads, dim, dtype, window, sinks, scale=None):
    print(f"paged attention {lengths} page={page} heads={heads}/{kv_heads} dim={dim} {dtype} "
          f"window={window} sinks={sinks}", flush=True)
    kv, k, v = _cache(dev, lengths, page, kv_heads, dim, dtype)
    q = _normal(99, len(lengths), heads, dim, dtype=dtype, gain=1.5).to(dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = fs.flagsparse_attention_paged(q, n, prepared=kv, window=window, sinks=sinks,
                                             scale=scale, return_lse=True)
    again = fs.flagsparse_attention_paged(q, n, prepared=kv, window=window, sinks=sinks, scale=scale)
    assert torch.equal(out, again)
    # a hidden key would be an infinity or NaN if it were read: left out
    want = ref.packed(q, torch.cat(k), torch.cat(v), [1] * len(lengths), lengths, True, window,
                      dim**-0.5 if scale is None else scale, sinks=sinks)
    ref.check("out", out, want["out"])
    ref.check("lse", lse, want["lse"])


@pytest.mark.parametrize("sinks", [1, 4, 33, 64, 200, 256, 300, 5000])
@pytest.mark.parametrize("window", [1, 31, 100, 255, 256, 300])
def test_decode(dev, window, sinks):
    _decode(dev, [0, 1, 64, 300, 700, 1111], 16, 4, 2, 64, HF, window, sinks)


@pytest.mark.parametrize("page", [1, 3, 16, 100, 1024])
def test_decode_pages(dev, page):
    _decode(dev, [150, 1, 999], page, 4, 2, 128, BF, 77, 9)


@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 8), (17, 1, 80), (64, 2, 40), (24, 8, 128)])
def test_decode_heads(dev, heads, kv_heads, dim):
    _decode(dev, [200, 45, 3000], 24, heads, kv_heads, dim, BF, 60, 5)


def test_decode_long(dev):
    _decode(dev, [30011, 20000], 64, 8, 1, 128, BF, 4096, 64)
    _decode(dev, [20000, 5, 9000], 32, 2, 2, 64, HF, 700, 1300)
    _decode(dev, [(37 * i) % 900 for i in range(300)], 8, 2, 1, 64, BF, 100, 4)


def test_decode_numbers_past_32_bits(dev):
    _decode(dev, [300, 20], 16, 4, 2, 64, BF, 2**40, 2**40)
    _decode(dev, [300, 20], 16, 4, 2, 64, BF, 100, 2**31 - 1)


def test_decode_hidden_keys_are_not_read(dev):
    lengths = [700]
    kv, k, v = _cache(dev, lengths, 16, 2, 64, HF)
    q, n = _normal(5, 1, 4, 64, dtype=HF).to(dev), torch.tensor(lengths, device=dev)
    clean = fs.flagsparse_attention_paged(q, n, prepared=kv, window=100, sinks=5)
    hidden = kv.indices.long()[torch.arange(5, 600, device=dev) // 16]
    kv.k_pages[hidden, torch.arange(5, 600, device=dev) % 16] = float("nan")
    kv.v_pages[hidden, torch.arange(5, 600, device=dev) % 16] = float("inf")
    assert torch.equal(fs.flagsparse_attention_paged(q, n, prepared=kv, window=100, sinks=5), clean)
    for bad in (701 + 100, -1, 2**40):
        n.fill_(bad)
        assert torch.isnan(fs.flagsparse_attention_paged(q, n, prepared=kv, window=100, sinks=5)).all()


def test_tokens_through_a_cache_are_the_packed_rows(dev):
    # token by token through the cache gives what packed attention gives of the whole
    n, g, h, d, page = 60, 2, 4, 64, 16
    kp = torch.full((8, page, g, d), float("nan"), dtype=BF, device=dev)
    vp = torch.full((8, page, g, d), float("nan"), dtype=BF, device=dev)
    kv = fs.prepare_paged_kv(kp, vp, torch.tensor([0, 4, 8], device=dev),
                             torch.tensor([4, 0, 7, 5, 1, 3, 6, 2], device=dev))
    q, k, v = (_normal(s, 2, n, m, d, dtype=BF).to(dev) for s, m in ((1, h), (2, g), (3, g)))
    length = torch.zeros(2, dtype=torch.int32, device=dev)
    outs = []
    for t in range(n):
        length += 1
        fs.flagsparse_paged_append(k[:, t], v[:, t], length, prepared=kv)
        outs.append(fs.flagsparse_attention_paged(q[:, t], length, prepared=kv, window=11, sinks=3))
    want = ref.packed(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), [n, n], [n, n], True, 11,
                      d**-0.5, sinks=3)
    ref.check("out", torch.stack(outs, 1).flatten(0, 1), want["out"])


def test_memory_of_short_sequences(dev):
    # gradients of many short sequences take what the call without first tokens does, and of those with jobs
    # room by their queries
    def taken(lengths, sinks):
        q, k, v, g = _inputs(dev, lengths, lengths, 4, 2, 64, BF)
        kw = {"prepared": fs.prepare_attention_packed(_indptr(lengths, dev)), "window": 20, "sinks": sinks}
        out, lse = fs.flagsparse_attention_packed(q, k, v, return_lse=True, **kw)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats(dev)
        before = torch.cuda.memory_allocated(dev)
        fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, **kw)
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated(dev) - before

    # the allocator gives a block whole where less than 1 MiB of it would be left: three gradients and a workspace
    more = 4 << 20
    short, slot = [30] * 3000, 2 * 64 * 64 * 4 * 2  # 64 keys, keys and values, of 64 numbers, two key heads
    assert taken(short, 4) <= taken(short, 0) + more
    mixed = short + [900]
    assert taken(mixed, 4) <= taken(mixed, 0) + 2 * (sum(mixed) // 512 + 1) * slot + more


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (12, 2)])
def test_short_sequences_beside_those_with_jobs(dev, heads, kv_heads):
    # those with as many queries as one job take their first keys' gradients in the tiles themselves, shares and all
    for lengths in ([3] * 90 + [700, 0, 512, 513] + [40] * 30 + [1100], [512, 300], [0, 5, 0, 513, 0]):
        _both(dev, lengths, lengths, heads, kv_heads, 64, BF, 30, 6)
    _both(dev, [40, 600, 0, 90], [300, 650, 70, 9], heads, kv_heads, 96, HF, 25, 100)
    _both(dev, [300] * 9, [300] * 9, heads, kv_heads, 128, HF, 200, 130)


def test_first_keys_that_reach_the_window_are_the_causal_call(dev):
    # to the bit, without lists of their own: also as a graph's first call
    lengths = [300, 20, 0, 513]
    q, k, v, g = _inputs(dev, lengths, [n + 30 for n in lengths], 6, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev), _indptr([n + 30 for n in lengths], dev))

    def both(**kw):
        out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, return_lse=True, **kw)
        return (out, lse, *fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, prepared=p, **kw))

    want, side = both(), torch.cuda.Stream(dev)
    for window, sinks in ((500, 43), (1, 542), (542, 1), (2**40, 7)):
        graph = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.graph(graph, stream=side):
            got = both(window=window, sinks=sinks)
        for _ in range(2):
            for t in got:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, got))
    hidden = both(window=500, sinks=42)  # one key of one query
    assert not torch.equal(hidden[0][832], want[0][832])


@pytest.mark.parametrize("batch", [70, 5000])
def test_jobs_among_very_many_sequences(dev, batch):
    # their sequences are searched for, 64 at a look, and again where there are more
    lengths = [1 + i % 3 for i in range(batch)]
    for at, n in ((0, 700), (batch // 2, 1100), (batch - 1, 513)):
        lengths[at] = n
    _both(dev, lengths, lengths, 2, 1, 64, BF, 2, 1)
    lengths = [0] * (batch // 2) + [900] + [0] * batch + [2, 600, 0]
    _both(dev, lengths, lengths, 2, 1, 64, HF, 30, 40)
