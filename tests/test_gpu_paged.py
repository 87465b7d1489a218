"""A paged cache: appending with the rotation of positions, and attention of one new token, against the
formulas in 64 bits."""

import copy

import pytest
import torch

import flagsparse_amd as fs
from oracle import attention as ref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _normal(seed, *shape, dtype, gain=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * gain).to(dtype)


def _cache(dev, lengths, page, heads, dim, dtype, spare=2, room=0, order="tokens", seed=1,
           stale=float("nan")):
    """(k_pages, v_pages, indptr, indices, k, v): a cache on the GPU whose pages hold k and v, lists
    of [length, heads, dim] on the CPU, in a random order, ``room`` pages more than a sequence
    needs; every other place holds ``stale``."""
    held = [-(-n // page) + room for n in lengths]
    total = sum(held) + spare
    gen = torch.Generator().manual_seed(seed)
    indices = torch.randperm(total, generator=gen)[:sum(held)].to(torch.int32)
    indptr = torch.tensor([0] + held).cumsum(0).to(torch.int32)
    shape = (total, page, heads, dim) if order == "tokens" else (total, heads, page, dim)
    both, kept = [], []
    for which in (0, 1):
        x = torch.full(shape, stale, dtype=dtype)
        view = x if order == "tokens" else x.transpose(1, 2)
        kept.append([])
        for b, n in enumerate(lengths):
            rows = _normal(seed + 10 * b + which + 2, n, heads, dim, dtype=dtype)
            kept[-1].append(rows)
            for j in range(n):
                view[int(indices[int(indptr[b]) + j // page]), j % page] = rows[j]
        x = x.to(dev)
        both.append(x if order == "tokens" else x.transpose(1, 2))
    return both[0], both[1], indptr.to(dev), indices.to(dev), kept[0], kept[1]


def _want(q, k, v, lengths, window, scale):
    """ref.packed of one query per sequence, with the tokens a window hides left out."""
    if window:
        k = [t[max(0, n - window):] for t, n in zip(k, lengths)]
        v = [t[max(0, n - window):] for t, n in zip(v, lengths)]
        lengths = [min(n, window) for n in lengths]
    return ref.packed(q, torch.cat(k), torch.cat(v), [1] * len(lengths), lengths, True, None, scale)


def _decode(dev, lengths, page, heads, kv_heads, dim, dtype, window=None, scale=None, order="tokens",
            room=0):
    print(f"paged attention {lengths} page={page} heads={heads}/{kv_heads} dim={dim} {dtype} "
          f"window={window} {order}", flush=True)
    kp, vp, ip, ix, k, v = _cache(dev, lengths, page, kv_heads, dim, dtype, order=order, room=room)
    q = _normal(99, len(lengths), heads, dim, dtype=dtype, gain=1.5).to(dev)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = fs.flagsparse_attention_paged(q, n, prepared=kv, window=window, scale=scale,
                                             return_lse=True)
    torch.cuda.synchronize()
    want = _want(q, k, v, lengths, window, dim**-0.5 if scale is None else scale)
    ref.check("out", out, want["out"])
    ref.check("lse", lse, want["lse"])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lengths", [[1], [0], [15, 16, 17], [0, 31, 0, 33, 1], [63, 64, 65, 127],
                                     [128, 129, 255, 256, 257], [1000], [2500, 3, 700]])
def test_lengths(dev, lengths, dtype):
    _decode(dev, lengths, 16, 4, 2, 128, dtype)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 48, 64, 72, 80, 96, 112, 120, 128])
def test_dims(dev, dim):
    _decode(dev, [100, 37], 16, 3, 1, dim, HF)
    _decode(dev, [100, 37], 16, 4, 4, dim, BF)


@pytest.mark.parametrize("page", [1, 2, 3, 5, 8, 24, 33, 64, 100, 256, 1024])
def test_pages_that_end_anywhere(dev, page):
    _decode(dev, [150, 1, 333], page, 4, 2, 64, BF)
    _decode(dev, [150, 1, 333], page, 4, 2, 64, BF, order="heads", room=2)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (8, 1), (15, 1), (16, 1), (17, 1),
                                            (33, 1), (64, 2), (24, 8), (23, 1)])
def test_heads(dev, heads, kv_heads):
    _decode(dev, [200, 45], 16, heads, kv_heads, 64, BF)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 300, 10000])
def test_window(dev, window):
    _decode(dev, [0, 1, 64, 300, 700], 16, 4, 2, 64, HF, window=window)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.25])
def test_scale(dev, scale):
    _decode(dev, [90, 200], 16, 2, 1, 64, HF, scale=scale)


def test_long_sequences(dev):
    _decode(dev, [30011], 64, 8, 1, 128, BF)
    _decode(dev, [20000, 5, 9000], 32, 2, 2, 64, HF)


def test_many_sequences(dev):
    _decode(dev, [(7 * i) % 40 for i in range(700)], 8, 2, 1, 64, BF)


@pytest.mark.parametrize("heads,batch", [(16, 60), (10, 220)])
def test_pieces_over_rounds_of_workgroups(dev, heads, batch):
    # two pieces each, more than the chip takes at once: joined by the last to arrive, or another launch
    g, d, page, each = heads // 2, 64, 64, 24
    kp, vp = (_normal(s, batch * each, page, g, d, dtype=BF) for s in (1, 2))
    lengths = [page * each - 13 * i % 700 for i in range(batch)]
    k, v = ([x[each * b:each * (b + 1)].flatten(0, 1)[:n] for b, n in enumerate(lengths)]
            for x in (kp, vp))
    kv = fs.prepare_paged_kv(kp.to(dev), vp.to(dev), torch.arange(batch + 1, device=dev) * each,
                             torch.arange(batch * each, device=dev))
    q, n = _normal(3, batch, heads, d, dtype=BF).to(dev), torch.tensor(lengths, device=dev)
    out, lse = fs.flagsparse_attention_paged(q, n, prepared=kv, return_lse=True)
    for _ in range(20):
        again, _ = fs.flagsparse_attention_paged(q, n, prepared=kv, return_lse=True)
        assert torch.equal(out, again)
    want = _want(q, k, v, lengths, None, d**-0.5)
    ref.check("out", out, want["out"])
    ref.check("lse", lse, want["lse"])


def test_caches_past_the_last_level(dev):
    # a table of more than 256 MB is read by other loads
    pages, page, g, d, n = 16 * 1024, 64, 2, 128, 3000
    kp = torch.empty(pages, page, g, d, dtype=HF, device=dev)
    vp = torch.empty(pages, page, g, d, dtype=HF, device=dev)
    k, v = (_normal(s, n, g, d, dtype=HF) for s in (1, 2))
    kv = fs.prepare_paged_kv(kp, vp, torch.tensor([0, 50, pages], device=dev),
                             torch.arange(pages, device=dev).flip(0))
    lengths = torch.tensor([n, 1], device=dev)
    fs.flagsparse_paged_append(torch.cat([k, k[:1]]).to(dev), torch.cat([v, v[:1]]).to(dev), lengths,
                               torch.tensor([0, n, n + 1], device=dev), prepared=kv)
    q = _normal(3, 2, 6, d, dtype=HF).to(dev)
    out, lse = fs.flagsparse_attention_paged(q, lengths, prepared=kv, return_lse=True)
    want = _want(q, [k, k[:1]], [v, v[:1]], [n, 1], None, d**-0.5)
    ref.check("out", out, want["out"])
    ref.check("lse", lse, want["lse"])


def test_lengths_change_and_tables_are_copies(dev):
    lengths = [300, 50]
    kp, vp, ip, ix, k, v = _cache(dev, lengths, 16, 2, 64, BF)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    other = copy.deepcopy(kv)
    q = _normal(99, 2, 4, 64, dtype=BF).to(dev)
    ix.zero_()  # the prepared object keeps what it checked
    ip.zero_()
    n = torch.tensor(lengths, dtype=torch.int64, device=dev)
    for now in ([300, 50], [1, 0], [299, 49], [17, 33]):
        n.copy_(torch.tensor(now))
        want = _want(q, [t[:m] for t, m in zip(k, now)], [t[:m] for t, m in zip(v, now)], now, None,
                     0.125)
        got = fs.flagsparse_attention_paged(q, n, prepared=kv)
        ref.check("out", got, want["out"])
        assert torch.equal(got, fs.flagsparse_attention_paged(q, n, prepared=other))
    # what the pages cannot hold is NaN, and nothing outside them is read
    n.copy_(torch.tensor([305, -1]))
    assert torch.isnan(fs.flagsparse_attention_paged(q, n, prepared=kv)).all()
    n.copy_(torch.tensor([2**40, 50]))
    got, lse = fs.flagsparse_attention_paged(q, n, prepared=kv, return_lse=True)
    assert torch.isnan(got[0]).all() and torch.isnan(lse[0]).all()
    assert not torch.isnan(got[1]).any() and not torch.isnan(lse[1]).any()


def test_shared_pages_and_strided_queries(dev):
    # two sequences read the same first pages; q is a slice of a fused projection
    kp, vp, ip, ix, k, v = _cache(dev, [64], 16, 2, 64, HF)
    kv = fs.prepare_paged_kv(kp, vp, torch.tensor([0, 4, 6], device=dev), torch.cat([ix, ix[:2]]))
    fused = _normal(5, 2, 8, 64, dtype=HF).to(dev)
    q = fused[:, 2:6]
    n = torch.tensor([64, 20], device=dev)
    out = torch.zeros(4, 2, 64, dtype=HF, device=dev).transpose(0, 1)
    assert fs.flagsparse_attention_paged(q, n, prepared=kv, out=out) is out
    want = _want(q, [k[0], k[0][:20]], [v[0], v[0][:20]], [64, 20], None, 0.125)
    ref.check("out", out, want["out"])
    odd = torch.zeros(2, 4, 65, dtype=HF, device=dev)[:, :, 1:]
    fs.flagsparse_attention_paged(q, n, prepared=kv, out=odd)
    assert torch.equal(odd, out)


def test_offsets_past_32_bits(dev):
    pages, page, g, d = 17000, 64, 16, 128
    kp = torch.empty(pages, page, g, d, dtype=BF, device=dev)
    vp = torch.empty(pages, page, g, d, dtype=BF, device=dev)
    assert kp.numel() > 2**31
    ix = torch.tensor([pages - 1, 3, pages - 2], dtype=torch.int32, device=dev)
    ip = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    n = torch.tensor([150], dtype=torch.int32, device=dev)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    k, v = (_normal(s, 150, g, d, dtype=BF) for s in (1, 2))
    fs.flagsparse_paged_append(k.to(dev), v.to(dev), n, torch.tensor([0, 150], device=dev),
                               prepared=kv)
    assert torch.equal(kp[ix[2].long(), 21, 15].cpu(), k[149, 15])
    q = _normal(3, 1, g, d, dtype=BF).to(dev)
    got = fs.flagsparse_attention_paged(q, n, prepared=kv)
    ref.check("out", got, _want(q, [k], [v], [150], None, d**-0.5)["out"])


# ---- appending ----


def _table(rows, half):
    t = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(half, dtype=torch.float64) / half)
    return t.cos().float(), t.sin().float()


def _turned(x, pos, cos, sin, interleaved):
    """(rotated, bound) of x [tokens, heads, dim]: two products and a sum in 32 bits, one rounding."""
    u, x = ref.U[x.dtype], x.double()
    half = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    y, e = x.clone(), torch.zeros_like(x)
    lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else \
        (slice(0, half), slice(half, 2 * half))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    e[..., lo] = e[..., hi] = 2.0**-22 * (a.abs() + b.abs())
    return y, e + u * y.abs() * (e > 0) + 1e-7 * (e > 0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half", [(64, 32), (128, 64), (128, 32), (80, 20), (72, 17), (40, 1),
                                      (8, 4), (64, 0), (120, 60)])
def test_append(dev, dim, half, interleaved, dtype):
    past, new, page, g, h = [0, 17, 40, 5, 0], [1, 3, 0, 30, 16], 12, 2, 6
    print(f"append dim={dim} half={half} interleaved={interleaved} {dtype}", flush=True)
    total = [a + b for a, b in zip(past, new)]
    kp, vp, ip, ix, k, v = _cache(dev, total, page, g, dim, dtype, room=1, stale=3.0)
    pos = torch.cat([torch.arange(a, a + b) for a, b in zip(past, new)])
    tokens = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev)
    kn, vn, q = (_normal(s, sum(new), n, dim, dtype=dtype) for s, n in ((7, g), (8, g), (9, h)))
    cos, sin = _table(60, half)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    before = kp.clone(), vp.clone()
    got = fs.flagsparse_paged_append(
        kn.to(dev), vn.to(dev), torch.tensor(total, device=dev), tokens, prepared=kv, q=q.to(dev),
        cos=cos.to(dev) if half else None, sin=sin.to(dev) if half else None,
        interleaved=interleaved)
    ref.check("q", got, _turned(q, pos, cos, sin, interleaved))
    seq = torch.repeat_interleave(torch.arange(5), torch.tensor(new))
    page_of = ix.cpu().long()[ip.cpu().long()[seq] + pos // page]
    ref.check("k", kp.cpu()[page_of, pos % page], _turned(kn, pos, cos, sin, interleaved))
    assert torch.equal(vp.cpu()[page_of, pos % page], vn)
    for now, then in ((kp, before[0]), (vp, before[1])):  # nothing else changes
        now, then = now.cpu(), then.cpu()
        now[page_of, pos % page] = 0
        then[page_of, pos % page] = 0
        assert torch.equal(now, then)


def test_append_steps_then_attention(dev):
    # token by token through the cache gives what packed attention gives of the whole
    n, g, h, d, page = 40, 2, 4, 64, 16
    kp = torch.full((8, g, page, d), float("nan"), dtype=BF, device=dev).transpose(1, 2)
    vp = torch.full((8, g, page, d), float("nan"), dtype=BF, device=dev).transpose(1, 2)
    kv = fs.prepare_paged_kv(kp, vp, torch.tensor([0, 3, 6], device=dev),
                             torch.tensor([4, 0, 7, 1, 3, 6], device=dev))
    q, k, v = (_normal(s, 2, n, m, d, dtype=BF).to(dev) for s, m in ((1, h), (2, g), (3, g)))
    length = torch.zeros(2, dtype=torch.int32, device=dev)
    cos, sin = (t.to(dev) for t in _table(48, 32))
    outs, turned = [], []
    for t in range(n):
        length += 1
        turned.append(fs.flagsparse_paged_append(k[:, t], v[:, t], length, prepared=kv, q=q[:, t],
                                                 cos=cos, sin=sin))
        outs.append(fs.flagsparse_attention_paged(turned[-1], length, prepared=kv))
    keys = torch.stack([kp[[4, 0, 7]].flatten(0, 1)[:n], kp[[1, 3, 6]].flatten(0, 1)[:n]])
    want = ref.packed(torch.stack(turned, 1).flatten(0, 1), keys.flatten(0, 1), v.flatten(0, 1),
                      [n, n], [n, n], True, None, d**-0.5)
    ref.check("out", torch.stack(outs, 1).flatten(0, 1), want["out"])


def test_tokens_without_a_place(dev):
    kp, vp, ip, ix, _, _ = _cache(dev, [20, 10], 16, 1, 64, HF, stale=2.0)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    before = kp.clone()
    k = _normal(1, 2, 1, 64, dtype=HF).to(dev)
    q = _normal(2, 2, 3, 64, dtype=HF).to(dev)
    cos, sin = (t.to(dev) for t in _table(16, 32))
    for lengths in ([33, 17], [0, -5], [2**35, -2**35]):
        n = torch.tensor(lengths, device=dev)
        got = fs.flagsparse_paged_append(k, k, n, prepared=kv, q=q)
        assert torch.isnan(got).all() and torch.equal(kp, before)
    # past the table of the rotation, in the pages
    got = fs.flagsparse_paged_append(k, k, torch.tensor([17, 16], device=dev), prepared=kv, q=q,
                                     cos=cos, sin=sin)
    assert torch.isnan(got[0]).all() and not torch.isnan(got[1]).any()
    page = ix[2].long()
    assert not torch.equal(kp[page, 15], before[page, 15])
    kp[page, 15] = before[page, 15]
    assert torch.equal(kp, before)
    # tokens of no sequence: the offsets end before the tokens do
    got = fs.flagsparse_paged_append(k, k, torch.tensor([5, 5], device=dev),
                                     torch.tensor([0, 1, 1], device=dev), prepared=kv, q=q)
    assert not torch.isnan(got[0]).any() and torch.isnan(got[1]).all()


def test_streams_graphs_and_equal_bits(dev):
    lengths = [900, 3, 2000, 77]
    kp, vp, ip, ix, _, _ = _cache(dev, lengths, 16, 2, 128, BF)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    cos, sin = (t.to(dev) for t in _table(3000, 64))
    k, q = _normal(1, 4, 2, 128, dtype=BF).to(dev), _normal(2, 4, 16, 128, dtype=BF).to(dev)

    def step():
        r = fs.flagsparse_paged_append(k, k, n, prepared=kv, q=q, cos=cos, sin=sin)
        return fs.flagsparse_attention_paged(r, n, prepared=kv, return_lse=True)

    want = step()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (3, 4, 5):
        q.copy_(_normal(seed, 4, 16, 128, dtype=BF))
        n.copy_(torch.tensor([900 - seed, 1, 2000 - 100 * seed, 0]))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b, ) or torch.equal(torch.isnan(a), torch.isnan(b)) and \
                torch.equal(a.nan_to_num(), b.nan_to_num())


def test_without_a_prepared_object(dev):
    lengths = [40, 0, 7]
    kp, vp, ip, ix, k, v = _cache(dev, lengths, 16, 2, 64, HF)
    q = _normal(3, 3, 4, 64, dtype=HF).to(dev)
    n = torch.tensor(lengths, device=dev)
    parts = {"k_pages": kp, "v_pages": vp, "indptr": ip, "indices": ix}
    out = fs.flagsparse_attention_paged(q, n, **parts)
    ref.check("out", out, _want(q, k, v, lengths, None, 0.125)["out"])
    new = _normal(4, 3, 2, 64, dtype=HF).to(dev)
    with pytest.raises(ValueError):  # sequence 1 has no pages
        fs.flagsparse_paged_append(new, new, n + 1, **parts)
    with pytest.raises(ValueError):
        fs.flagsparse_attention_paged(q, n - 1, **parts)
    with pytest.raises(ValueError):
        fs.flagsparse_attention_paged(q, n, k_pages=kp, v_pages=vp, indptr=ip)


def test_empty_batch(dev):
    kp = torch.zeros(1, 16, 1, 64, dtype=BF, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    kv = fs.prepare_paged_kv(kp, kp.clone(), torch.zeros(1, dtype=torch.int32, device=dev), none)
    q = torch.zeros(0, 2, 64, dtype=BF, device=dev)
    out, lse = fs.flagsparse_attention_paged(q, none, prepared=kv, return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    assert fs.flagsparse_paged_append(q[:, :1], q[:, :1], none, prepared=kv) is None


def test_refusals(dev):
    kp, vp, ip, ix, _, _ = _cache(dev, [20, 10], 16, 2, 64, BF)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    n = torch.tensor([20, 10], device=dev)
    q = torch.zeros(2, 4, 64, dtype=BF, device=dev)
    k = torch.zeros(2, 2, 64, dtype=BF, device=dev)
    cos, sin = (t.to(dev) for t in _table(32, 32))
    prep, paged, add = (fs.prepare_paged_kv, fs.flagsparse_attention_paged,
                        fs.flagsparse_paged_append)
    bad = [
        (TypeError, lambda: prep(kp.float(), vp.float(), ip, ix)),
        (TypeError, lambda: prep(kp, vp.half(), ip, ix)),
        (ValueError, lambda: prep(kp[0], vp[0], ip, ix)),
        (ValueError, lambda: prep(kp, vp[1:], ip, ix)),
        (ValueError, lambda: prep(kp.cpu(), vp.cpu(), ip, ix)),
        (ValueError, lambda: prep(kp.transpose(2, 3), vp.transpose(2, 3), ip, ix)),
        (NotImplementedError, lambda: prep(kp[..., :4], vp[..., :4], ip, ix)),
        (IndexError, lambda: prep(kp, vp, ip, ix + 100)),
        (IndexError, lambda: prep(kp, vp, ip, ix - 100)),
        (ValueError, lambda: prep(kp, vp, ip + 1, ix)),
        (ValueError, lambda: prep(kp, vp, ip, ix[:-1])),
        (ValueError, lambda: prep(kp, vp, ip[[0, 2, 1, 2]], ix)),
        (ValueError, lambda: prep(kp, vp, ip.cpu(), ix)),
        (TypeError, lambda: prep(kp, vp, ip, ix.float())),
        (TypeError, lambda: paged(q.half(), n, prepared=kv)),
        (TypeError, lambda: paged(q, n, prepared=ip)),
        (TypeError, lambda: paged(q, n.float(), prepared=kv)),
        (ValueError, lambda: paged(q, n[:1], prepared=kv)),
        (ValueError, lambda: paged(q, n.cpu(), prepared=kv)),
        (ValueError, lambda: paged(q[:1], n, prepared=kv)),
        (ValueError, lambda: paged(q[:, :3], n, prepared=kv)),
        (ValueError, lambda: paged(q[:, :, :32], n, prepared=kv)),
        (ValueError, lambda: paged(q, n, prepared=kv, window=0)),
        (ValueError, lambda: paged(q, n, prepared=kv, out=q[:1])),
        (ValueError, lambda: add(k[:, :1], k, n, prepared=kv)),
        (ValueError, lambda: add(k[:1], k, n, prepared=kv)),
        (ValueError, lambda: add(k[:1], k[:1], n, prepared=kv)),
        (ValueError, lambda: add(k, k, n, n, prepared=kv)),
        (ValueError, lambda: add(k, k, n, prepared=kv, cos=cos)),
        (ValueError, lambda: add(k, k, n, prepared=kv, cos=cos, sin=sin[:1])),
        (TypeError, lambda: add(k, k, n, prepared=kv, cos=cos.half(), sin=sin)),
        (ValueError, lambda: add(k, k, n, prepared=kv, cos=torch.cat([cos, cos], 1),
                                 sin=torch.cat([sin, sin], 1))),
        (ValueError, lambda: add(k, k, n, prepared=kv, q=q[:1])),
        (ValueError, lambda: add(k, k, n, prepared=kv, out=q)),
    ]
    for i, (kind, f) in enumerate(bad):
        with pytest.raises(kind):
            f()
            pytest.fail(f"refusal {i} did not come")


def test_tokens_of_no_sequence_at_all(dev):
    # an empty batch whose offsets leave every token out
    kp = torch.zeros(1, 16, 1, 64, dtype=BF, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    kv = fs.prepare_paged_kv(kp, kp.clone(), torch.zeros(1, dtype=torch.int32, device=dev), none)
    q = _normal(1, 5, 3, 64, dtype=BF).to(dev)
    for _ in range(2):
        room = [torch.zeros(5, 3, 64, dtype=BF, device=dev) for _ in range(4)]
        del room  # what a fresh array is likely to hold
        got = fs.flagsparse_paged_append(q[:, :1], q[:, :1], none, torch.zeros(1, device=dev,
                                         dtype=torch.int32), prepared=kv, q=q)
        assert torch.isnan(got).all()
    out = torch.zeros(5, 3, 65, dtype=BF, device=dev)[:, :, 1:]
    assert fs.flagsparse_paged_append(q[:, :1], q[:, :1], none, torch.zeros(1, device=dev,
                                      dtype=torch.int32), prepared=kv, q=q, out=out) is out
    assert torch.isnan(out).all() and not kp.any()


@pytest.mark.parametrize("tokens", [3, 700])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half", [(40, 20), (64, 32), (72, 17), (80, 40), (96, 48), (112, 56), (128, 64)])
def test_append_over_its_queries(dev, dim, half, interleaved, tokens):
    # out on q, on a slice that is partly q's, on k and on v: what the call gives elsewhere
    g, h, page = 2, 32, 16
    pages = -(-tokens // page)
    cos, sin = (t.to(dev) for t in _table(tokens, half))
    first = _normal(1, tokens + 1, h + 2 * g, dim, dtype=HF).to(dev)
    n, at = torch.tensor([tokens], device=dev), torch.tensor([0, tokens], device=dev)

    def call(place):
        kp, vp = torch.zeros(2, pages, page, g, dim, dtype=HF, device=dev)
        kv = fs.prepare_paged_kv(kp, vp, torch.tensor([0, pages], device=dev),
                                 torch.arange(pages, device=dev))
        fused = first.clone()
        q, k, v = fused[:tokens, :h], fused[:tokens, h:h + g], fused[:tokens, h + g:]
        out = None if place is None else place(fused)
        got = fs.flagsparse_paged_append(k, v, n, at, prepared=kv, q=q, cos=cos, sin=sin,
                                         interleaved=interleaved, out=out)
        assert out is None or got is out
        return got.clone(), kp, vp

    want = call(None)
    for place in (lambda f: f[:tokens, :h], lambda f: f[1:, :h], lambda f: f[:tokens, 2 * g:],
                  lambda f: f[:tokens, 1:h + 1]):
        for a, b in zip(call(place), want):
            assert torch.equal(a, b)


def test_paged_attention_over_its_queries(dev):
    lengths = [900, 3, 0, 77]
    kp, vp, ip, ix, _, _ = _cache(dev, lengths, 16, 2, 64, BF)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    first = _normal(1, 5, 8, 64, dtype=BF).to(dev)
    want = fs.flagsparse_attention_paged(first[:4], n, prepared=kv)
    for place in (lambda f: f[:4], lambda f: f[1:]):
        room = first.clone()
        out = place(room)
        assert fs.flagsparse_attention_paged(room[:4], n, prepared=kv, out=out) is out
        assert torch.equal(out, want)


def test_graphs_of_a_warm_stream_beside_its_calls(dev):
    # two graphs captured on a stream that has run the call, replayed on others beside it
    lengths = [900, 3, 2000, 77]
    kp, vp, ip, ix, _, _ = _cache(dev, lengths, 16, 2, 64, BF)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    q = _normal(2, 4, 40, 64, dtype=BF).to(dev)
    streams = [torch.cuda.Stream(dev) for _ in range(3)]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        want = fs.flagsparse_attention_paged(q, n, prepared=kv)
        assert kv._counts  # the pieces are joined in the kernel
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[0]):
                held = fs.flagsparse_attention_paged(q, n, prepared=kv)
            graphs.append((g, held))
    torch.cuda.synchronize()
    for _ in range(30):
        got = []
        for (g, _), s in zip(graphs, streams[1:]):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[0]):
            got = [fs.flagsparse_attention_paged(q, n, prepared=kv) for _ in range(3)]
        torch.cuda.synchronize()
        for x in (*got, *(held for _, held in graphs)):
            assert torch.equal(x, want)
    for counts in kv._counts.values():
        assert not counts.any()


def test_the_longest_sequence(dev):
    # one page, named over and over: the last token that a table can hold, and what it sees
    page, g, h, d, n = 1024, 1, 2, 8, 2**31 - 1024
    kp, vp = torch.zeros(2, 1, page, g, d, dtype=BF, device=dev)
    k, v = (_normal(s, page, g, d, dtype=BF) for s in (1, 2))
    kp.copy_(k[None]), vp.copy_(v[None])
    with pytest.raises(ValueError):
        fs.prepare_paged_kv(kp[:, :512], vp[:, :512], torch.tensor([0, 2**22 - 1], device=dev),
                            torch.zeros(2**22 - 1, dtype=torch.int32, device=dev))
    kv = fs.prepare_paged_kv(kp, vp, torch.tensor([0, n // page], device=dev),
                             torch.zeros(n // page, dtype=torch.int32, device=dev))
    assert kv.room == n
    q = _normal(3, 1, h, d, dtype=BF).to(dev)
    length = torch.tensor([n], dtype=torch.int32, device=dev)
    k[-1], v[-1] = 2.0, 3.0
    fs.flagsparse_paged_append(k[-1:].to(dev), v[-1:].to(dev), length, prepared=kv)
    assert torch.equal(kp[0].cpu(), k) and torch.equal(vp[0].cpu(), v)
    for window in (1, 700, 5000):
        out, lse = fs.flagsparse_attention_paged(q, length, prepared=kv, window=window, return_lse=True)
        at = torch.arange(n - window, n) % page
        want = ref.packed(q, k[at], v[at], [1], [window], True, None, d**-0.5)
        ref.check("out", out, want["out"])
        ref.check("lse", lse, want["lse"])
    length += 1
    assert torch.isnan(fs.flagsparse_attention_paged(q, length, prepared=kv, window=700)).all()


def test_one_token_and_one_head_of_wider_arrays(dev):
    # the step of an axis of one element is no multiple of anything
    g, h, d, n = 1, 3, 64, 40
    kp, vp, ip, ix, k, v = _cache(dev, [n], 16, g, d, BF)
    kp, vp = (t.as_strided(t.shape, (*t.stride()[:2], 5, 1)) for t in (kp, vp))
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    fused = _normal(5, 2, (h + 2 * g) * d + 3, dtype=BF).to(dev)[:, :-3].unflatten(1, (-1, d))[:1]
    assert fused.stride(0) % 8 and fused.is_contiguous()
    length = torch.tensor([n], device=dev)
    got = fs.flagsparse_paged_append(fused[:, h:h + g], fused[:, h + g:], length, prepared=kv,
                                     q=fused[:, :h])
    assert torch.equal(got, fused[:, :h])
    out = fs.flagsparse_attention_paged(fused[:, :h], length, prepared=kv)
    k, v = k[0].clone(), v[0].clone()
    k[-1], v[-1] = fused[0, h:h + g].cpu(), fused[0, h + g:].cpu()
    ref.check("out", out, _want(fused[:, :h], [k], [v], [n], None, d**-0.5)["out"])


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 1e39])
def test_scales_that_are_not_finite(dev, scale):
    kp, vp, ip, ix, _, _ = _cache(dev, [20], 16, 2, 64, BF)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    q = torch.zeros(1, 4, 64, dtype=BF, device=dev)
    with pytest.raises(ValueError):
        fs.flagsparse_attention_paged(q, torch.tensor([20], device=dev), prepared=kv, scale=scale)


def test_pages_whose_storage_moves(dev):
    # the tensors are the caller's: what they hold at the time of a call is what is read and written
    lengths = [300, 50]
    kp, vp, ip, ix, k, v = _cache(dev, lengths, 16, 2, 64, BF)
    kv = fs.prepare_paged_kv(kp, vp, ip, ix)
    n = torch.tensor(lengths, device=dev)
    q = _normal(99, 2, 4, 64, dtype=BF).to(dev)
    new = _normal(98, 2, 2, 64, dtype=BF).to(dev)
    for _ in range(2):
        fs.flagsparse_paged_append(new, new, n, prepared=kv)
        fs.flagsparse_attention_paged(q, n, prepared=kv)
    old = kp.detach(), vp.detach()  # keeps the old storage
    kp.data, vp.data = kp * 2, vp * 0.5
    before = [t.clone() for t in old]
    k, v = [t * 2 for t in k], [t * 0.5 for t in v]
    for b in range(2):
        k[b][-1] = v[b][-1] = new[b].cpu() * 4
    for _ in range(2):
        fs.flagsparse_paged_append(new * 4, new * 4, n, prepared=kv)
        out = fs.flagsparse_attention_paged(q, n, prepared=kv)
        ref.check("out", out, _want(q, k, v, lengths, None, 0.125)["out"])
    for a, b in zip(old, before):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    kp.data = kp[:-1]
    with pytest.raises(ValueError):
        fs.flagsparse_attention_paged(q, n, prepared=kv, scale=0.5)


def test_one_key_above_all_others_in_float16(dev):
    # as with packed sequences: weights are rounded as 2^11 times themselves
    n, g, h, d, page = 250, 1, 2, 64, 16
    q = torch.zeros(1, h, d, dtype=HF)
    q[..., 0] = 16.0
    k = torch.zeros(n, g, d, dtype=HF)
    k[..., 0] = -8.0
    v = _normal(1, n, g, d, dtype=HF).abs()
    k[77], v[77] = 0.0, 0.0
    kp, vp = (torch.zeros(16, page, g, d, dtype=HF) for _ in range(2))
    kp.view(-1, g, d)[:n], vp.view(-1, g, d)[:n] = k, v
    out = fs.flagsparse_attention_paged(
        q.to(dev), torch.tensor([n], device=dev), k_pages=kp.to(dev), v_pages=vp.to(dev),
        indptr=torch.tensor([0, 16], device=dev), indices=torch.arange(16, device=dev))
    ref.check("out", out, ref.packed(q, k, v, [1], [n], True, None, d**-0.5, small=2.0**-11)["out"])


@pytest.mark.parametrize("lengths", [[900, 3, 2000, 77], [7000, 1, 520]])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(33, 1, 72, HF), (40, 2, 40, BF), (23, 1, 80, HF),
                                                      (6, 2, 120, BF), (64, 2, 128, HF), (4, 4, 8, BF)])
def test_pieces_of_odd_heads_and_dims(dev, heads, kv_heads, dim, dtype, lengths):
    # several pieces a sequence, joined by the last of them to arrive or by another launch, with head
    # tiles that are not full, several to a key head, and dims that fill no tile
    _decode(dev, lengths, 16, heads, kv_heads, dim, dtype)
    _decode(dev, lengths, 16, heads, kv_heads, dim, dtype, window=600, room=3)
