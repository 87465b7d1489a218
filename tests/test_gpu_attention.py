"""Attention over packed sequences, forward and backward, against the formulas in 64 bits."""

import copy

import pytest
import torch

import flagsparse_amd as fs
from oracle import attention as ref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _indptr(lengths, dev, dtype=torch.int32):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(dtype).to(dev)


def _normal(seed, *shape, dtype, dev, gain=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * gain).to(dtype).to(dev)


def _inputs(dev, q_len, k_len, heads, kv_heads, dim, dtype, seed=1):
    return (_normal(seed, sum(q_len), heads, dim, dtype=dtype, dev=dev, gain=1.5),
            _normal(seed + 1, sum(k_len), kv_heads, dim, dtype=dtype, dev=dev),
            _normal(seed + 2, sum(k_len), kv_heads, dim, dtype=dtype, dev=dev),
            _normal(seed + 3, sum(q_len), heads, dim, dtype=dtype, dev=dev))


def _both(dev, q_len, k_len, heads, kv_heads, dim, dtype, causal, window, scale=None, seed=1):
    print(f"attention {q_len} {k_len} heads={heads}/{kv_heads} dim={dim} {dtype} causal={causal} "
          f"window={window}", flush=True)
    q, k, v, g = _inputs(dev, q_len, k_len, heads, kv_heads, dim, dtype, seed)
    kw = {"causal": causal, "window": window, "scale": scale}
    ip, kp = _indptr(q_len, dev), _indptr(k_len, dev)
    out, lse = fs.flagsparse_attention_packed(q, k, v, ip, kp, return_lse=True, **kw)
    grads = fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, ip, kp, **kw)
    torch.cuda.synchronize()
    want = ref.packed(q, k, v, q_len, k_len, causal, window,
                      dim**-0.5 if scale is None else scale, g)
    for name, got in zip(("out", "lse", "q", "k", "v"), (out, lse, *grads)):
        ref.check(name, got, want[name])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", [[1], [2, 1], [31, 33], [64, 0, 63], [65], [127, 128, 129],
                                     [255, 1, 257], [700]])
def test_lengths(dev, lengths, causal, dtype):
    _both(dev, lengths, lengths, 4, 2, 64, dtype, causal, None)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 56, 64, 72, 80, 96, 104, 112, 120, 128])
def test_dims(dev, dim, dtype):
    _both(dev, [150, 70], [150, 70], 3, 1, dim, dtype, True, None)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (7, 1), (16, 2), (24, 8), (9, 3)])
def test_heads(dev, heads, kv_heads):
    _both(dev, [90, 300], [90, 300], heads, kv_heads, 128, BF, True, None)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_len,k_len", [([5, 200], [300, 1]), ([200], [40]), ([130, 64], [0, 64]),
                                         ([0, 70], [70, 0]), ([1, 1, 1], [500, 65, 2]),
                                         ([300], [129])])
def test_other_keys(dev, q_len, k_len, causal):
    # more queries than keys: the first ones see nothing under the causal mask
    _both(dev, q_len, k_len, 4, 2, 64, BF, causal, None)
    _both(dev, q_len, k_len, 2, 2, 128, HF, causal, None)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 128, 200, 5000])
def test_window(dev, window):
    _both(dev, [300, 40, 129], [300, 40, 129], 4, 2, 64, BF, True, window)
    _both(dev, [100, 200], [333, 150], 2, 1, 128, HF, True, window)


def test_many_sharing_few(dev):
    # few key tiles under many heads: shares of a group's heads are summed by another launch
    _both(dev, [130], [130], 16, 1, 64, BF, True, None)
    _both(dev, [70, 3], [200, 64], 24, 2, 128, HF, True, 50)
    _both(dev, [90], [0], 8, 1, 64, BF, False, None)
    _both(dev, [33, 0], [40, 10], 60, 4, 40, BF, True, None)


def test_long_chains_with_many_heads(dev):
    # more workgroups than the chip takes at once, and chains that are shared by more waves
    _both(dev, [1300], [1300], 4, 2, 128, BF, True, None)
    _both(dev, [1, 1500], [1100, 1200], 2, 1, 64, HF, True, 1050)
    _both(dev, [40] * 70, [40] * 70, 16, 8, 96, HF, True, None)


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("lengths,heads", [([64], 4), ([65], 4), ([64] * 5, 60), ([65] * 3, 60),
                                           ([600], 40), ([520, 3], 54), ([300, 65], 8)])
def test_shares_of_a_tile(dev, lengths, heads, dim):
    # few and many workgroups, chains of one step of keys and of several
    _both(dev, lengths, lengths, heads, 2, dim, BF, True, None)
    _both(dev, lengths, lengths, heads, 2, dim, HF, False, None)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_scale(dev, scale):
    _both(dev, [100, 20], [100, 20], 2, 1, 32, HF, True, None, scale=scale)


def test_long_rows(dev):
    _both(dev, [3000], [3000], 2, 1, 128, BF, True, None)
    _both(dev, [40], [9000], 2, 1, 64, HF, True, None)
    _both(dev, [2500], [30], 2, 1, 64, BF, False, None)


@pytest.mark.parametrize("gain", [40.0, 1e-3])
def test_peaked_and_flat_scores(dev, gain):
    q, k, v, g = _inputs(dev, [200], [200], 2, 2, 64, HF)
    q = (q * gain).to(HF)
    out, lse = fs.flagsparse_attention_packed(q, k, v, _indptr([200], dev), return_lse=True)
    want = ref.packed(q, k, v, [200], [200], True, None, 0.125)
    ref.check("out", out, want["out"])
    ref.check("lse", lse, want["lse"])


def test_slices_of_one_projection(dev):
    lengths, h, g, d = [70, 133], 4, 2, 64
    fused = _normal(3, sum(lengths), h + 2 * g, d, dtype=BF, dev=dev)
    q, k, v = fused[:, :h], fused[:, h:h + g], fused[:, h + g:]
    grad = _normal(4, h, sum(lengths), d, dtype=BF, dev=dev).transpose(0, 1)  # heads first in memory
    ip = _indptr(lengths, dev, torch.int64)
    p = fs.prepare_attention_packed(ip)
    out = torch.full((h, sum(lengths), d), 7.0, dtype=BF, device=dev).transpose(0, 1)
    got, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, out=out, return_lse=True)
    assert got is out
    grads = fs.flagsparse_attention_packed_backward(grad, q, k, v, out, lse, prepared=p)
    want = ref.packed(q, k, v, lengths, lengths, True, None, d**-0.5, grad)
    for name, x in zip(("out", "lse", "q", "k", "v"), (out, lse, *grads)):
        ref.check(name, x, want[name])


def test_unaligned_inputs_and_outputs_are_copied(dev):
    lengths, h, g, d = [50, 7], 2, 1, 40
    wide = [_normal(i, sum(lengths), n, d + 3, dtype=HF, dev=dev) for i, n in ((1, h), (2, g), (3, g))]
    q, k, v = (t[:, :, 1:d + 1] for t in wide)
    room = torch.zeros(sum(lengths), h, d + 3, dtype=HF, device=dev)
    out = room[:, :, 2:d + 2]
    fs.flagsparse_attention_packed(q, k, v, _indptr(lengths, dev), out=out)
    want = ref.packed(q, k, v, lengths, lengths, True, None, d**-0.5)
    ref.check("out", out, want["out"])
    assert not room[:, :, :2].any() and not room[:, :, d + 2:].any()


def test_broadcast_inputs_and_their_gradients(dev):
    # one token's values for every key, through an expanded view: autograd sums over the copies
    lengths, h, d = [60, 80], 2, 64
    q, k, _, g = _inputs(dev, lengths, lengths, h, h, d, BF)
    row = _normal(9, 1, h, d, dtype=BF, dev=dev).requires_grad_()
    q.requires_grad_()
    v = row.expand(sum(lengths), h, d)
    out = fs.flagsparse_attention_packed(q, k, v, _indptr(lengths, dev))
    dq, drow = torch.autograd.grad(out, (q, row), g)
    want = ref.packed(q, k, v, lengths, lengths, True, None, d**-0.5, g)
    ref.check("out", out, want["out"])
    ref.check("q", dq, want["q"])
    total, bound = want["v"]
    # the sum over the copies is torch's, in its own order, rounded to the type
    ref.check("v", drow, (total.sum(0, keepdim=True), bound.sum(0, keepdim=True) +
                          ref.U[BF] * total.abs().sum(0, keepdim=True)))


def test_autograd_is_the_backward_call(dev):
    lengths = [100, 31]
    q, k, v, g = _inputs(dev, lengths, lengths, 4, 2, 64, HF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev))
    out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, window=40, return_lse=True)
    want = fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, prepared=p, window=40)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    res = fs.flagsparse_attention_packed(*leaves, prepared=p, window=40)
    res.backward(g)
    assert torch.equal(res, out)
    for t, w in zip(leaves, want):
        assert torch.equal(t.grad, w)
    with pytest.raises(RuntimeError):
        fs.flagsparse_attention_packed(*leaves, prepared=p, out=torch.empty_like(out))


@pytest.mark.parametrize("causal", [True, False])
def test_gradient_against_differences(dev, causal):
    # the slope of f(t) = sum(grad * out(x + t d)) in 64 bits by central differences, against the
    # kernels' gradient along d
    lengths, h, g, d, t = [40, 23], 2, 1, 64, 1e-5
    q, k, v, grad = _inputs(dev, lengths, lengths, h, g, d, HF)
    ip = _indptr(lengths, dev)
    out, lse = fs.flagsparse_attention_packed(q, k, v, ip, causal=causal, return_lse=True)
    grads = fs.flagsparse_attention_packed_backward(grad, q, k, v, out, lse, ip, causal=causal)
    want = ref.packed(q, k, v, lengths, lengths, causal, None, d**-0.5, grad)
    xs = [x.cpu().double() for x in (q, k, v)]

    def f(*a):
        total, at = 0.0, 0
        for n in lengths:
            m = ref.seen(n, n, causal, None)
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


def test_sequences_do_not_touch_each_other(dev):
    lengths = [77, 50, 130, 9]
    q, k, v, g = _inputs(dev, lengths, lengths, 4, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev))

    def both():
        out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, return_lse=True)
        return (out, lse, *fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, prepared=p))

    clean = both()
    bad = slice(77, 127)
    for t in (q, k, v, g):
        t[bad] = float("nan")
    v[bad] = float("inf")
    dirty = both()
    keep = torch.ones(sum(lengths), dtype=torch.bool, device=dev)
    keep[bad] = False
    for a, b in zip(clean, dirty):
        assert torch.equal(a[keep], b[keep])


def test_keys_that_are_not_finite_reach_the_rows_that_see_them(dev):
    # a masked score is chosen away, whatever it is
    n, h = 150, 2
    q, k, v, _ = _inputs(dev, [n], [n], h, h, 64, BF)
    ip = _indptr([n], dev)
    clean = fs.flagsparse_attention_packed(q, k, v, ip)
    k[100, 0, 3] = float("nan")
    k[120, 1] = float("inf")
    out = fs.flagsparse_attention_packed(q, k, v, ip)
    assert torch.equal(out[:100, 0], clean[:100, 0]) and torch.equal(out[:120, 1], clean[:120, 1])
    assert torch.isnan(out[100:, 0]).all() and torch.isnan(out[120:, 1]).all()


def test_equal_calls_give_equal_bits(dev):
    lengths = [400, 1, 233]
    q, k, v, g = _inputs(dev, lengths, lengths, 8, 2, 128, BF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev))

    def both():
        out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, return_lse=True)
        return (out, lse, *fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, prepared=p))

    first = both()
    for _ in range(3):
        for a, b in zip(first, both()):
            assert torch.equal(a, b)
    again = copy.deepcopy(p)
    for t in p._tiles.values():
        t.zero_()  # the copy works on its own arrays
    p = again
    for a, b in zip(first, both()):
        assert torch.equal(a, b)


def test_offsets_past_32_bits(dev):
    # rows so far apart that the last ones lie past 2^31 elements
    n, h, d, step = 33, 1, 64, 1 << 26
    room = torch.empty(n * step, dtype=BF, device=dev)
    assert room.numel() > 2**31
    q, k, v, g = _inputs(dev, [n], [n], h, h, d, BF)
    views = [room[64 * i:].as_strided((n, h, d), (step, d, 1)) for i in range(5)]
    for t, x in zip(views, (q, k, v, g)):
        t.copy_(x)
    ip = _indptr([n], dev)
    out, lse = fs.flagsparse_attention_packed(*views[:3], ip, out=views[4], return_lse=True)
    grads = fs.flagsparse_attention_packed_backward(views[3], *views[:3], out, lse, ip)
    want = ref.packed(q, k, v, [n], [n], True, None, d**-0.5, g)
    for name, x in zip(("out", "lse", "q", "k", "v"), (out, lse, *grads)):
        ref.check(name, x, want[name])


@pytest.mark.parametrize("d", [64, 128])
def test_the_longest_steps_between_tokens(dev, d):
    # the longest that the kernels take as they are: a tile's rows span almost 2^31 bytes
    n, step = 300, 1 << 23
    room = torch.empty(n * step, dtype=BF, device=dev)
    q, k, v, g = _inputs(dev, [n], [n], 1, 1, d, BF)
    views = [room[d * i:].as_strided((n, 1, d), (step, d, 1)) for i in range(5)]
    for t, x in zip(views, (q, k, v, g)):
        t.copy_(x)
    ip = _indptr([n], dev)
    out, lse = fs.flagsparse_attention_packed(*views[:3], ip, out=views[4], return_lse=True)
    grads = fs.flagsparse_attention_packed_backward(views[3], *views[:3], out, lse, ip)
    want = ref.packed(q, k, v, [n], [n], True, None, d**-0.5, g)
    for name, x in zip(("out", "lse", "q", "k", "v"), (out, lse, *grads)):
        ref.check(name, x, want[name])


def test_nothing_to_do(dev):
    for q_len, k_len in (([], []), ([0, 0], [0, 0]), ([0], [5]), ([5], [0])):
        q, k, v, g = _inputs(dev, q_len, k_len, 2, 1, 64, HF)
        ip, kp = _indptr(q_len, dev), _indptr(k_len, dev)
        out, lse = fs.flagsparse_attention_packed(q, k, v, ip, kp, return_lse=True)
        grads = fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, ip, kp)
        assert not out.any() and (lse == float("-inf")).all()
        for x, t in zip(grads, (q, k, v)):
            assert x.shape == t.shape and not x.any()


def test_other_streams_and_graphs(dev):
    lengths = [200, 77]
    q, k, v, g = _inputs(dev, lengths, lengths, 4, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev))

    def both():
        out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, return_lse=True)
        return (out, lse, *fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, prepared=p))

    want = both()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream(dev).wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in (5, 6, 7):
        for t in (q, k, v, g):
            t.copy_(_normal(seed, *t.shape, dtype=BF, dev=dev))
            seed += 10
        want = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_index_arrays_are_not_checked_in_a_capture(dev, monkeypatch):
    q, k, v, _ = _inputs(dev, [10], [10], 2, 2, 64, BF)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError):
        fs.flagsparse_attention_packed(q, k, v, _indptr([10], dev))


def test_refusals(dev):
    q, k, v, g = _inputs(dev, [10], [10], 4, 2, 64, BF)
    ip = _indptr([10], dev)
    call = fs.flagsparse_attention_packed
    out, lse = call(q, k, v, ip, return_lse=True)
    p = fs.prepare_attention_packed(ip)
    bad = [
        (TypeError, lambda: call(q.float(), k, v, ip)),
        (TypeError, lambda: call(q, k.half(), v, ip)),
        (TypeError, lambda: call(None, k, v, ip)),
        (ValueError, lambda: call(q[0], k, v, ip)),
        (ValueError, lambda: call(q.cpu(), k, v, ip)),
        (ValueError, lambda: call(q, k.cpu(), v, ip)),
        (ValueError, lambda: call(q[:, :3], k, v, ip)),
        (ValueError, lambda: call(q, k, v[:, :1], ip)),
        (ValueError, lambda: call(q, k[:, :, :32], v, ip)),
        (ValueError, lambda: call(q[:9], k, v, ip)),
        (ValueError, lambda: call(q, k[:9], v[:9], ip)),
        (ValueError, lambda: call(q, k, v)),
        (ValueError, lambda: call(q, k, v, ip.cpu())),
        (ValueError, lambda: call(q, k, v, ip.flip(0))),
        (ValueError, lambda: call(q, k, v, ip + 1)),
        (ValueError, lambda: call(q, k, v, ip, _indptr([4, 6], dev))),
        (TypeError, lambda: call(q, k, v, ip.float())),
        (TypeError, lambda: call(q, k, v, prepared=ip)),
        (ValueError, lambda: call(q, k, v, ip, window=0)),
        (ValueError, lambda: call(q, k, v, ip, window=3, causal=False)),
        (ValueError, lambda: call(q, k, v, ip, out=out[:9])),
        (TypeError, lambda: call(q, k, v, ip, out=out.half())),
        (NotImplementedError, lambda: call(q[:, :, :4], k[:, :, :4], v[:, :, :4], ip)),
        (NotImplementedError, lambda: call(*(torch.zeros(10, 1, 136, dtype=BF, device=dev),) * 3, ip)),
        (ValueError, lambda: fs.flagsparse_attention_packed_backward(g[:9], q, k, v, out, lse,
                                                                     prepared=p)),
        (TypeError, lambda: fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse.double(),
                                                                    prepared=p)),
        (TypeError, lambda: fs.flagsparse_attention_packed_backward(g, q, k, v, out.half(), lse,
                                                                    prepared=p)),
    ]
    for n, (kind, f) in enumerate(bad):
        with pytest.raises(kind):
            f()
            pytest.fail(f"refusal {n} did not come")


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (1, 1), (4, 2)])
@pytest.mark.parametrize("q_len,k_len", [([0], [5]), ([0, 0], [70, 3])])
def test_gradients_of_a_batch_without_queries(dev, q_len, k_len, heads, kv_heads):
    # where the heads of a group are not shared out the workspace has no bytes
    q, k, v, g = _inputs(dev, q_len, k_len, heads, kv_heads, 64, BF)
    p = fs.prepare_attention_packed(_indptr(q_len, dev), _indptr(k_len, dev))
    for _ in range(2):
        out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, return_lse=True)
        grads = fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, prepared=p)
        for x, t in zip(grads, (q, k, v)):
            assert x.shape == t.shape and not x.any()
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    fs.flagsparse_attention_packed(*leaves, prepared=p).backward(g)
    for t in leaves:
        assert t.grad.shape == t.shape and not t.grad.any()


def test_outputs_over_inputs(dev):
    # written after everything is read: over the queries, the keys, the values, or slices of each
    lengths, h, d = [300, 65, 1], 4, 64
    n = sum(lengths)
    ip = _indptr(lengths, dev)
    first = _normal(1, n + 1, 3 * h, d, dtype=BF, dev=dev)

    def parts():
        fused = first.clone()
        return fused, fused[:n, :h], fused[:n, h:2 * h], fused[:n, 2 * h:]

    _, q, k, v = parts()
    want = fs.flagsparse_attention_packed(q, k, v, ip)
    for place in (lambda f: f[:n, :h], lambda f: f[:n, h:2 * h], lambda f: f[:n, 2 * h:],
                  lambda f: f[1:, :h], lambda f: f[1:, 2:h + 2], lambda f: f[:n, 2 * h - 1:3 * h - 1]):
        fused, q, k, v = parts()
        out = place(fused)
        assert fs.flagsparse_attention_packed(q, k, v, ip, out=out) is out
        assert torch.equal(out, want)


def test_batches_that_are_too_long(dev):
    for n in (2**31 - 1023, 2**31 - 1, 2**33):
        with pytest.raises(ValueError):
            fs.prepare_attention_packed(torch.tensor([0, n], device=dev))
        with pytest.raises(ValueError):
            fs.prepare_attention_packed(torch.tensor([0, 1], device=dev), torch.tensor([0, n], device=dev))


def test_one_token_of_a_wider_array(dev):
    # the step of an axis of one element is no multiple of anything, and contiguous() keeps it
    h, g, d = 4, 2, 64
    wide = _normal(1, 3, (h + 2 * g) * d + 3, dtype=BF, dev=dev)[:, :-3].unflatten(1, (-1, d))[:1]
    assert wide.stride(0) % 8 and wide.is_contiguous()
    q, k, v = wide[:, :h], wide[:, h:h + g], wide[:, h + g:]
    grad = _normal(4, 2, h * d + 5, dtype=BF, dev=dev)[:, :h * d].unflatten(1, (h, d))[:1]
    ip = _indptr([1], dev)
    out, lse = fs.flagsparse_attention_packed(q, k, v, ip, return_lse=True)
    grads = fs.flagsparse_attention_packed_backward(grad, q, k, v, out, lse, ip)
    want = ref.packed(q, k, v, [1], [1], True, None, d**-0.5, grad)
    for name, x in zip(("out", "lse", "q", "k", "v"), (out, lse, *grads)):
        ref.check(name, x, want[name])


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_scales_that_are_not_finite(dev, scale):
    q, k, v, g = _inputs(dev, [10], [10], 2, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr([10], dev))
    out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, return_lse=True)
    for _ in range(2):
        with pytest.raises(ValueError):
            fs.flagsparse_attention_packed(q, k, v, prepared=p, scale=scale)
        with pytest.raises(ValueError):
            fs.flagsparse_attention_packed_backward(g, q, k, v, out, lse, prepared=p, scale=scale)


def test_tangents_are_refused(dev):
    # forward-mode derivatives have no kernel: an error, never an output without its tangent
    q, k, v, _ = _inputs(dev, [10], [10], 2, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr([10], dev))
    for _ in range(2):
        want = fs.flagsparse_attention_packed(q, k, v, prepared=p)
    with torch.autograd.forward_ad.dual_level():
        for which in range(3):
            args = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if i == which else t
                    for i, t in enumerate((q, k, v))]
            with pytest.raises(NotImplementedError):
                fs.flagsparse_attention_packed(*args, prepared=p)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                fs.flagsparse_attention_packed(*args, prepared=p)
        assert torch.equal(fs.flagsparse_attention_packed(q, k, v, prepared=p), want)


def test_tangents_of_the_gradient_are_refused(dev):
    q, k, v, g = _inputs(dev, [10], [10], 2, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr([10], dev))
    out, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, return_lse=True)
    args = [g, q, k, v, out, lse]
    for _ in range(2):
        fs.flagsparse_attention_packed_backward(*args, prepared=p)
    leaf = q.clone().requires_grad_()
    res = fs.flagsparse_attention_packed(leaf, k, v, prepared=p)
    with torch.autograd.forward_ad.dual_level():
        for i, t in enumerate(args):
            dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(NotImplementedError):
                fs.flagsparse_attention_packed_backward(*args[:i], dual, *args[i + 1:], prepared=p)
        dual = torch.autograd.forward_ad.make_dual(g, torch.ones_like(g))
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(res, leaf, dual)


@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([2048], 2, 1, 64), ([700] * 4, 16, 8, 128),
                                                        ([300, 65], 4, 2, 40)])
@pytest.mark.parametrize("gain,v_gain", [(2.0**-13, 1.0), (2.0**-10, 1.0), (1000.0, 30.0)])
def test_small_and_large_gradients_in_float16(dev, gain, v_gain, lengths, heads, kv_heads, dim):
    # dS lies far from 1: below float16's normal numbers, or past its largest, while the gradient
    # that is looked at lies among them, by a large q beside a small k or the other way round.
    # Scores do not change with it, nor does dS
    print(f"gradients times {gain} {v_gain} {lengths} {heads} {kv_heads} {dim}", flush=True)
    q, k, v, g = _inputs(dev, lengths, lengths, heads, kv_heads, dim, HF)
    v, g = (v * v_gain).to(HF), (g.float() * gain).to(HF)
    p = fs.prepare_attention_packed(_indptr(lengths, dev))
    for up, names in ((64.0, "k" if gain < 1 else "q"), (1 / 64.0, "q" if gain < 1 else "k")):
        a, b = (q.float() * up).to(HF), (k.float() / up).to(HF)
        out, lse = fs.flagsparse_attention_packed(a, b, v, prepared=p, return_lse=True)
        grads = dict(zip("qkv", fs.flagsparse_attention_packed_backward(g, a, b, v, out, lse,
                                                                        prepared=p)))
        want = ref.packed(a, b, v, lengths, lengths, True, None, dim**-0.5, g, small=0.0)
        for name in names + "v":
            ref.check(name, grads[name], want[name])


def test_one_key_above_all_others_in_float16(dev):
    # a key that outweighs the others by 16 e-folds and has a value of zero: the output is what the
    # others' small weights leave of it.  Weights are rounded as 2^11 times themselves
    n, h, d = 4096, 2, 64
    q = torch.zeros(3, h, d, dtype=HF)
    q[..., 0] = 16.0
    k = torch.zeros(n, h, d, dtype=HF)
    k[..., 0] = -8.0
    v = _normal(1, n, h, d, dtype=HF, dev="cpu").abs()
    k[77], v[77] = 0.0, 0.0
    q, k, v = (t.to(dev) for t in (q, k, v))
    out = fs.flagsparse_attention_packed(q, k, v, _indptr([3], dev), _indptr([n], dev), causal=False)
    ref.check("out", out, ref.packed(q, k, v, [3], [n], False, None, d**-0.5, small=2.0**-11)["out"])


def test_flags_of_the_library_are_not_cut_to_32_bits(dev):
    from flagsparse_amd import _abi, attention

    q, k, v, _ = _inputs(dev, [100], [100], 2, 2, 64, BF)
    p = fs.prepare_attention_packed(_indptr([100], dev))
    want, lse = fs.flagsparse_attention_packed(q, k, v, prepared=p, return_lse=True)
    out = torch.empty_like(q)
    head = list(attention._PACKED.unpack(attention._pack(p, q, k, v, True, 0, 0.125, out)))
    assert head[8] == 1
    head[8] = 1 << 32
    args = attention._PACKED.pack(*head) + attention._PACKED_AT.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, 0)
    _abi.check(_abi.lib().fsp_attention_packed(args, p._on()), "fsp_attention_packed")
    assert torch.equal(out, want)


@pytest.mark.parametrize("which", ["q", "k", "v", "qk", "qv", "kv"])
def test_gradients_of_some_inputs(dev, which):
    lengths = [100, 31]
    arrays = dict(zip("qkvg", _inputs(dev, lengths, lengths, 4, 2, 64, BF)))
    g = arrays.pop("g")
    p = fs.prepare_attention_packed(_indptr(lengths, dev))
    out, lse = fs.flagsparse_attention_packed(*arrays.values(), prepared=p, return_lse=True)
    want = fs.flagsparse_attention_packed_backward(g, *arrays.values(), out, lse, prepared=p)
    leaves = {n: t.clone().requires_grad_(n in which) for n, t in arrays.items()}
    res, stat = fs.flagsparse_attention_packed(*leaves.values(), prepared=p, return_lse=True)
    assert torch.equal(res, out) and torch.equal(stat, lse) and not stat.requires_grad
    res.backward(g)
    for (n, t), w in zip(leaves.items(), want):
        assert torch.equal(t.grad, w) if n in which else t.grad is None
