"""Drafted tokens into a paged cache, the accepted ones kept, pages copied: moves are exact, what is rotated is
within one rounding of 64 bits; and a generation with drafts is the generation without."""

import copy

import pytest
import torch

import flagsparse_amd as fs
from oracle import attention as ref
from tests.test_gpu_tree import _cache, _indptr, _masks, _normal, _tree, _ways

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _table(rows, half):
    t = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(half, dtype=torch.float64) / max(half, 1))
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


def _bits(t):
    return t.contiguous().view(torch.int16)


def _slots(kv, b, places):
    """(pages, slots) of a sequence's places."""
    first = int(kv.indptr[b])
    places = torch.as_tensor(places, dtype=torch.long, device=kv.device)
    return kv.indices.long()[first + places // kv.page_size], places % kv.page_size


# ---- appending drafts ----


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half", [(64, 32), (128, 64), (80, 20), (72, 17), (64, 0)])
def test_append_drafts(dev, dim, half, interleaved, dtype):
    past, new, g, h = [0, 17, 40, 5, 300], [1, 30, 0, 256, 70], 2, 6
    trees = [_tree(n, s) for s, n in enumerate(new)]
    total = [a + b for a, b in zip(past, new)]
    kv, _, _ = _cache(dev, total, 12, g, dim, dtype, room=1)
    ways = [_ways(t) for t in trees]
    turn = torch.tensor([p + len(w) - 1 for p, ws in zip(past, ways) for w in ws])
    kn, vn, q = (_normal(s, sum(new), n, dim, dtype=dtype) for s, n in ((7, g), (8, g), (9, h)))
    cos, sin = _table(600, half)
    kw = {"cos": cos.to(dev), "sin": sin.to(dev), "interleaved": interleaved} if half else {}
    got = fs.flagsparse_paged_append(
        kn.to(dev), vn.to(dev), torch.tensor(total, device=dev), _indptr(new, dev), prepared=kv,
        q=q.to(dev), parents=torch.tensor([p for t in trees for p in t], device=dev), **kw)
    ref.check("q", got, _turned(q, turn, cos, sin, interleaved))
    want = _turned(kn, turn, cos, sin, interleaved)
    at = 0
    for b, n in enumerate(new):
        here = _slots(kv, b, range(past[b], total[b]))
        ref.check("k", kv.k_pages[here], tuple(t[at:at + n] for t in want))
        assert torch.equal(kv.v_pages[here].cpu(), vn[at:at + n])
        at += n


def test_append_drafts_one_each_and_a_chain(dev):
    # a chain is rotated as the tokens of a text are; one token each is at its place
    kv, _, _ = _cache(dev, [40, 20], 16, 2, 64, BF)
    cos, sin = (t.to(dev) for t in _table(64, 32))
    n, tokens = torch.tensor([40, 20], device=dev), torch.tensor([0, 9, 12], device=dev)
    k, q = (_normal(s, 12, m, 64, dtype=BF).to(dev) for s, m in ((1, 2), (2, 4)))
    plain = fs.flagsparse_paged_append(k, k, n, tokens, prepared=kv, q=q, cos=cos, sin=sin)
    before = _bits(kv.k_pages).clone()
    chain = torch.tensor([*range(-1, 8), *range(-1, 2)], device=dev)
    got = fs.flagsparse_paged_append(k, k, n, tokens, prepared=kv, q=q, cos=cos, sin=sin, parents=chain)
    assert torch.equal(got, plain) and torch.equal(_bits(kv.k_pages), before)
    none = torch.full((2,), -1, device=dev)
    one = fs.flagsparse_paged_append(k[:2], k[:2], n, prepared=kv, q=q[:2], cos=cos, sin=sin, parents=none)
    assert torch.equal(one, fs.flagsparse_paged_append(k[:2], k[:2], n, prepared=kv, q=q[:2], cos=cos, sin=sin))
    none[1] = 0
    one = fs.flagsparse_paged_append(k[:2], k[:2], n, prepared=kv, q=q[:2], cos=cos, sin=sin, parents=none)
    assert not torch.isnan(one[0]).any() and torch.isnan(one[1]).all()


def test_append_drafts_without_a_way(dev):
    past, new = [90, 40], [9, 12]
    trees = [_tree(n, s) for s, n in enumerate(new)]
    kv, _, _ = _cache(dev, [a + b for a, b in zip(past, new)], 16, 2, 64, BF)
    k, q = (_normal(s, 21, m, 64, dtype=BF).to(dev) for s, m in ((1, 2), (2, 4)))
    n, tokens = torch.tensor([99, 52], device=dev), _indptr(new, dev)
    flat = [p for t in trees for p in t]
    for bad in (4, 7, 100, -2, -2**40, 2**40):
        before = kv.k_pages.clone()
        parents = torch.tensor(flat, device=dev)
        parents[4] = bad
        got = fs.flagsparse_paged_append(k, k, n, tokens, prepared=kv, q=q, parents=parents)
        fallen = [i for i, way in enumerate(_ways(trees[0])) if 4 in way]
        assert torch.isnan(got.float()).all(-1).all(-1).cpu().nonzero().flatten().tolist() == fallen
        here = _slots(kv, 0, [90 + i for i in fallen])
        assert torch.equal(_bits(kv.k_pages[here]), _bits(before[here]))
    # tokens that lead nowhere: no parent outside the array is looked at
    for bad in ([-3, 9, 21], [0, 9, 2**31 - 1], [0, 2**40, 21], [-2**40, 5, 2**40], [30, 9, 21]):
        parents = torch.tensor(flat, device=dev)
        got = fs.flagsparse_paged_append(k, k, n, torch.tensor(bad, device=dev), prepared=kv, q=q,
                                         parents=parents)
        if bad[0] < 0:
            assert torch.isnan(got[:5].float()).all()
        if bad[2] > 21:
            assert torch.isnan(got[9:].float()).all()
    # more than 256 of a sequence
    kv, _, _ = _cache(dev, [300], 16, 2, 64, BF)
    k = _normal(1, 257, 2, 64, dtype=BF).to(dev)
    got = fs.flagsparse_paged_append(k, k, torch.tensor([300], device=dev), torch.tensor([0, 257], device=dev),
                                     prepared=kv, q=k, parents=torch.zeros(257, device=dev).long() - 1)
    assert torch.isnan(got).all()
    # past the table of the rotation by depth, not by place
    cos, sin = (t.to(dev) for t in _table(45, 32))
    star = torch.tensor([-1] + [0] * 19, device=dev)
    got = fs.flagsparse_paged_append(k[:20], k[:20], torch.tensor([63], device=dev),
                                     torch.tensor([0, 20], device=dev), prepared=kv, q=k[:20], cos=cos,
                                     sin=sin, parents=star)
    assert not torch.isnan(got).any()
    got = fs.flagsparse_paged_append(k[:20], k[:20], torch.tensor([64], device=dev),
                                     torch.tensor([0, 20], device=dev), prepared=kv, q=k[:20], cos=cos,
                                     sin=sin, parents=star)
    assert not torch.isnan(got[0]).any() and torch.isnan(got[1:]).all()


# ---- keeping tokens ----


def _marks(counts, share, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.rand(n, generator=gen) < share for n in counts]


def _kept_rows(rows, count, marks):
    """The rows of one sequence that stay."""
    past = len(rows) - count
    return torch.cat([rows[:past], rows[past:][marks]])


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (HF, 128), (BF, 8), (HF, 72), (BF, 120)])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.9, 1.0])
def test_keep_in_place(dev, share, dim, dtype):
    lengths, new = [0, 1, 40, 300, 700, 33, 3000], [0, 1, 13, 64, 700, 0, 2500]
    kv, k, v = _cache(dev, lengths, 16, 2, dim, dtype, room=1)
    before = kv.k_pages.clone(), kv.v_pages.clone()
    marks = _marks(new, share, 1)
    n = torch.tensor(lengths, device=dev)
    got = fs.flagsparse_paged_keep(torch.cat(marks).to(dev), n, _indptr(new, dev), prepared=kv)
    assert got.dtype == torch.int32
    assert got.tolist() == [a - b + int(m.sum()) for a, b, m in zip(lengths, new, marks)]
    changed = torch.zeros(kv.n_pages, 16, dtype=torch.bool, device=dev)
    for b in range(len(lengths)):
        here = _slots(kv, b, range(int(got[b])))
        for pages, rows in ((kv.k_pages, k[b]), (kv.v_pages, v[b])):
            assert torch.equal(pages[here].cpu(), _kept_rows(rows, new[b], marks[b]))
        changed[_slots(kv, b, range(lengths[b] - new[b], lengths[b]))] = True
    for now, then in zip((kv.k_pages, kv.v_pages), before):  # nothing else changes
        assert torch.equal(_bits(now[~changed]), _bits(then[~changed]))


@pytest.mark.parametrize("page,to_page,order", [(16, 16, "tokens"), (1, 5, "tokens"), (100, 24, "heads"),
                                                (64, 256, "tokens"), (33, 8, "heads")])
@pytest.mark.parametrize("share", [0.0, 0.5, 1.0])
def test_keep_into_other_pages(dev, share, page, to_page, order):
    lengths, new = [0, 1, 40, 300, 700, 33, 3000, 1500], [0, 1, 13, 300, 64, 0, 2500, 3]
    kv, k, v = _cache(dev, lengths, page, 3, 64, BF, room=1)
    to, _, _ = _cache(dev, lengths, to_page, 3, 64, BF, seed=5, order=order, room=1)
    before = _bits(kv.k_pages).clone(), to.k_pages.clone(), to.v_pages.clone()
    marks = _marks(new, share, 2)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    for _ in range(2):
        got = fs.flagsparse_paged_keep(torch.cat(marks).to(dev), n, _indptr(new, dev), prepared=kv, into=to)
    assert got.tolist() == [a - b + int(m.sum()) for a, b, m in zip(lengths, new, marks)]
    assert torch.equal(_bits(kv.k_pages), before[0])
    changed = torch.zeros(to.n_pages, to_page, dtype=torch.bool, device=dev)
    for b in range(len(lengths)):
        here = _slots(to, b, range(int(got[b])))
        for pages, rows in ((to.k_pages, k[b]), (to.v_pages, v[b])):
            assert torch.equal(pages[here].cpu(), _kept_rows(rows, new[b], marks[b]))
        changed[here] = True
    for now, then in zip((to.k_pages, to.v_pages), before[1:]):
        assert torch.equal(_bits(now[~changed]), _bits(then[~changed]))


def test_marks_at_any_address(dev):
    lengths = [2000, 900]
    kv, k, _ = _cache(dev, lengths, 16, 1, 64, HF)
    to, _, _ = _cache(dev, lengths, 16, 1, 64, HF, seed=5)
    n = torch.tensor(lengths, device=dev)
    for skip in range(5):
        for new in ([1997, 3], [5, 900], [64, 61]):
            marks = _marks(new, 0.5, skip)
            keep = torch.cat([torch.ones(skip, dtype=torch.bool), *marks,
                              torch.ones(7, dtype=torch.bool)]).to(dev)[skip:skip + sum(new)]
            got = fs.flagsparse_paged_keep(keep, n, _indptr(new, dev), prepared=kv, into=to)
            for b in range(2):
                want = _kept_rows(k[b], new[b], marks[b])
                assert int(got[b]) == len(want)
                assert torch.equal(to.k_pages[_slots(to, b, range(len(want)))].cpu(), want)


def test_keep_as_many_for_each_and_strided_marks(dev):
    kv, k, _ = _cache(dev, [40, 30], 16, 2, 64, BF)
    n = torch.tensor([40, 30], device=dev)
    marks = _marks([8, 8], 0.5, 3)
    wide = torch.zeros(16, 2, dtype=torch.bool)
    wide[:, 1] = torch.cat(marks)
    got = fs.flagsparse_paged_keep(wide.to(dev)[:, 1], n, prepared=kv)
    for b in range(2):
        want = _kept_rows(k[b], 8, marks[b])
        assert int(got[b]) == len(want)
        assert torch.equal(kv.k_pages[_slots(kv, b, range(len(want)))].cpu(), want)


def test_keep_where_nothing_can_move(dev):
    kv, _, _ = _cache(dev, [40, 30, 9], 16, 2, 64, BF)
    to, _, _ = _cache(dev, [48, 16, 16], 16, 2, 64, BF, seed=5)
    keep, tokens = torch.zeros(20, dtype=torch.bool, device=dev), torch.tensor([0, 10, 18, 20], device=dev)
    keep[9] = keep[17] = True
    n = torch.tensor([40, 30, 9], device=dev)
    before = _bits(kv.k_pages).clone(), _bits(to.k_pages).clone()
    for bad in ([9, -1, 1], [49, 2**40, 17], [-2**40, 7, 33]):
        n.copy_(torch.tensor(bad))
        for kw in ({}, {"into": to}):
            assert fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, **kw).tolist() == [-1, -1, -1]
    n.copy_(torch.tensor([40, 30, 9]))
    for bad in ([0, -5, 18, 20], [0, 30, 18, 20], [2**33, 10, 2**33, 20]):
        # what belongs to no tokens is not moved; what does may be
        for kw in ({}, {"into": to}):
            fs.flagsparse_paged_keep(keep, n, torch.tensor(bad, device=dev), prepared=kv, **kw)
    torch.cuda.synchronize()
    kv.k_pages.view(torch.int16).copy_(before[0])
    to.k_pages.view(torch.int16).copy_(before[1])
    # 23 of the second sequence stay, and its other pages hold 16
    got = fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, into=to)
    assert got.tolist() == [31, -1, 7]
    assert torch.equal(_bits(to.k_pages[to.indices[3].long()]), before[1][to.indices[3].long()])


def test_keep_in_graphs_and_on_streams(dev):
    lengths, new = [700, 90], [20, 7]
    kv, k, _ = _cache(dev, lengths, 16, 2, 64, BF)
    to, _, _ = _cache(dev, lengths, 16, 2, 64, BF, seed=5)
    keep, tokens = torch.cat(_marks(new, 0.5, 1)).to(dev), _indptr(new, dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    start = kv.k_pages.clone(), kv.v_pages.clone()

    def both():
        return (fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, into=to),
                fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv))

    want = both()
    after = _bits(kv.k_pages).clone(), _bits(to.k_pages).clone()
    assert torch.equal(want[0], want[1])
    graph = torch.cuda.CUDAGraph()
    kv.k_pages.copy_(start[0])
    kv.v_pages.copy_(start[1])
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(3):
        kv.k_pages.copy_(start[0])
        kv.v_pages.copy_(start[1])
        to.k_pages.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert torch.equal(_bits(kv.k_pages), after[0])
        for b in range(2):
            here = _slots(to, b, range(int(got[0][b])))
            assert torch.equal(_bits(to.k_pages[here]), after[1][here])
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        again = fs.flagsparse_paged_keep(keep, n, tokens, prepared=copy.deepcopy(kv), into=copy.deepcopy(to))
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(again, want[0])


def test_another_table_of_the_same_pages(dev):
    # what a call moves goes by the arguments it is given, not by those of an earlier call
    kv, k, _ = _cache(dev, [40], 16, 2, 64, BF)
    keep, n = torch.ones(40, dtype=torch.bool, device=dev), torch.tensor([40], dtype=torch.int32, device=dev)
    room = torch.zeros(2, 9, 16, 2, 64, dtype=BF, device=dev)
    for pages in ([0, 1, 2], [5, 3, 8], [7, 6, 4]):
        to = fs.prepare_paged_kv(room[0], room[1], torch.tensor([0, 3], device=dev),
                                 torch.tensor(pages, device=dev))
        room.zero_()
        fs.flagsparse_paged_keep(keep, n, prepared=kv, into=to)
        assert torch.equal(room[0][pages].flatten(0, 1)[:40].cpu(), k[0])
        del to


# ---- copying pages ----


@pytest.mark.parametrize("order", ["tokens", "heads", "apart"])
@pytest.mark.parametrize("page,heads,dim,dtype", [(16, 2, 64, BF), (1, 1, 8, HF), (33, 3, 72, BF),
                                                  (256, 8, 128, HF)])
def test_copy(dev, page, heads, dim, dtype, order):
    n = 40
    if order == "apart":
        room = _normal(1, n, page, 3, heads, dim, dtype=dtype).to(dev)
        kp, vp = room[:, :, 0], room[:, :, 2]
    else:
        kp, vp = (_normal(s, n, page, heads, dim, dtype=dtype).to(dev) for s in (1, 2))
        if order == "heads":
            kp, vp = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kp, vp))
    pages = torch.randperm(n, generator=torch.Generator().manual_seed(3))
    sources, targets = pages[:13].to(dev), pages[13:26].to(torch.int32).to(dev)
    sources[3] = sources[4]  # one page to two others
    targets[5] = sources[5]  # and one to itself
    want = kp.clone(), vp.clone()
    for x in want:
        x[targets.long()] = x[sources]
    fs.flagsparse_paged_copy(sources, targets, k_pages=kp, v_pages=vp)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    kv = fs.prepare_paged_kv(kp, vp, torch.tensor([0], device=dev), targets[:0])
    fs.flagsparse_paged_copy(targets[:1], sources[:1], prepared=kv)
    assert torch.equal(kp, want[0])


def test_copy_of_numbers_outside_the_cache(dev):
    kv, _, _ = _cache(dev, [40], 16, 2, 64, BF)
    before = _bits(kv.k_pages).clone()
    bad = torch.tensor([-1, 5, 100, -2**40, 2**40, 0, 1, 2], device=dev)
    fs.flagsparse_paged_copy(bad, torch.tensor([0, 5, 0, 1, 1, -1, 5, 2**33], device=dev), prepared=kv)
    assert torch.equal(_bits(kv.k_pages), before)
    none = bad[:0]
    fs.flagsparse_paged_copy(none, none, prepared=kv)


def test_many_pages_and_offsets_past_32_bits(dev):
    pages, page, g, d = 17000, 64, 16, 128
    kp = torch.zeros(pages, page, g, d, dtype=BF, device=dev)
    vp = torch.zeros(pages, page, g, d, dtype=BF, device=dev)
    assert kp.numel() > 2**31
    rows = _normal(1, 5, page, g, d, dtype=BF).to(dev)
    kp[100:105], vp[100:105] = rows, rows.flip(0)
    targets = torch.tensor([pages - 1, 3, 16999 - 5, 16400, 8], device=dev)
    fs.flagsparse_paged_copy(torch.arange(100, 105, device=dev), targets, k_pages=kp, v_pages=vp)
    assert torch.equal(kp[targets], rows) and torch.equal(vp[targets], rows.flip(0))
    small = torch.arange(6000, dtype=torch.float32, device=dev).to(HF)[:, None, None, None].expand(
        6000, 16, 1, 8).contiguous()
    other = small.clone()
    fs.flagsparse_paged_copy(torch.arange(0, 3000, device=dev), torch.arange(3000, 6000, device=dev),
                             k_pages=small, v_pages=other)
    assert torch.equal(small[3000:], small[:3000]) and torch.equal(other, small)


def test_refusals(dev):
    kv, _, _ = _cache(dev, [40, 30], 16, 2, 64, BF)
    other, _, _ = _cache(dev, [40], 16, 2, 64, BF)
    half, _, _ = _cache(dev, [40, 30], 16, 2, 64, HF)
    heads, _, _ = _cache(dev, [40, 30], 16, 4, 64, BF)
    n, tokens = torch.tensor([40, 30], device=dev), torch.tensor([0, 2, 6], device=dev)
    keep = torch.ones(6, dtype=torch.bool, device=dev)
    cache = {"k_pages": kv.k_pages, "v_pages": kv.v_pages, "indptr": kv.indptr, "indices": kv.indices}
    for bad in ((keep[:5], n, None), (keep[None], n, tokens), (keep.cpu(), n, tokens), (keep, n[:1], tokens),
                (keep, n, tokens[:2])):
        with pytest.raises(ValueError):
            fs.flagsparse_paged_keep(*bad, prepared=kv)
    with pytest.raises(TypeError):
        fs.flagsparse_paged_keep(keep.int(), n, tokens, prepared=kv)
    with pytest.raises(TypeError):
        fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, into=kv.k_pages)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, into=kv)
    for _ in range(2):  # a call that was made before, or not
        for into in (other, half, heads):
            with pytest.raises(ValueError):
                fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, into=into)
        fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv)
    for bad in ([0, 2, 5], [1, 2, 6], [0, 7, 6], [0, 0, 40]):
        with pytest.raises(ValueError):
            fs.flagsparse_paged_keep(keep, n, torch.tensor(bad, device=dev), **cache)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_keep(keep, torch.tensor([1, 30], device=dev), tokens, **cache)
    k = torch.zeros(6, 2, 64, dtype=BF, device=dev)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_append(k, k, n, tokens, parents=torch.zeros(5, device=dev).int(), prepared=kv)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_append(k, k, n, tokens, parents=torch.zeros(6, device=dev).int(), **cache)
    pages = {"k_pages": kv.k_pages, "v_pages": kv.v_pages}
    a, b = torch.tensor([0, 1], device=dev), torch.tensor([2, 3], device=dev)
    for s, t in ((a, b[:1]), (a[None], b), (a.cpu(), b), (a, torch.tensor([2, 2], device=dev)),
                 (a, torch.tensor([1, 2], device=dev))):
        with pytest.raises(ValueError):
            fs.flagsparse_paged_copy(s, t, **pages)
    for s, t in ((a - 1, b), (a, b + 100)):
        with pytest.raises(IndexError):
            fs.flagsparse_paged_copy(s, t, **pages)
    with pytest.raises(TypeError):
        fs.flagsparse_paged_copy(a.float(), b, **pages)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_copy(a, b)


# ---- together ----


@pytest.mark.parametrize("window,sinks", [(None, 0), (24, 5)])
def test_drafting_is_the_text_read_at_once(dev, window, sinks):
    """Steps of drafts over a cache, some accepted, the sequences branched by copied pages: the queries of the
    tokens that stay see what packed attention shows them of the text they ended up in."""
    g, h, d, page, steps, room = 2, 8, 64, 8, 6, 12
    gen = torch.Generator().manual_seed(7)
    pages = torch.full((2, 60, page, g, d), float("nan"), dtype=BF, device=dev)
    table = torch.randperm(60, generator=gen)[:3 * room].view(3, room)
    cos, sin = (t.to(dev) for t in _table(room * page, d // 2))

    def cache(rows):
        return fs.prepare_paged_kv(pages[0], pages[1], torch.arange(len(rows) + 1, device=dev) * room,
                                   table[rows].flatten().to(dev))

    # two sequences go on from prompts; later the first one's text is shared by the third
    kv, lengths = cache([0, 1]), torch.tensor([13, 21], dtype=torch.int32, device=dev)
    texts = [_normal(11, 13, h + 2 * g, d, dtype=BF), _normal(12, 21, h + 2 * g, d, dtype=BF)]
    fused = torch.cat(texts).to(dev)
    fs.flagsparse_paged_append(fused[:, h:h + g], fused[:, h + g:], lengths, torch.tensor([0, 13, 34], device=dev),
                               prepared=kv, q=fused[:, :h], cos=cos, sin=sin)
    seen = [[], []]  # (place in the text, rotated query, output) of the accepted tokens
    for step in range(steps):
        if step == 3:
            # pages that are full are shared by the table, the one being filled is copied
            full = int(lengths[0]) // page
            table[2, :full] = table[0, :full]
            fs.flagsparse_paged_copy(table[0, full:full + 1].to(dev), table[2, full:full + 1].to(dev), prepared=kv)
            kv, lengths = cache([0, 1, 2]), torch.cat([lengths, lengths[:1]])
            texts.append(texts[0].clone())
            seen.append([])
        new = [int(torch.randint(1, 9, (1,), generator=gen)) for _ in texts]
        trees = [_tree(n, 10 * step + b, roots=0.2, back=3) for b, n in enumerate(new)]
        drafts = [_normal(100 * step + b, n, h + 2 * g, d, dtype=BF) for b, n in enumerate(new)]
        fused, tokens = torch.cat(drafts).to(dev), _indptr(new, dev)
        parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
        lengths = lengths + torch.tensor(new, dtype=torch.int32, device=dev)
        q = fs.flagsparse_paged_append(fused[:, h:h + g], fused[:, h + g:], lengths, tokens, prepared=kv,
                                       q=fused[:, :h], cos=cos, sin=sin, parents=parents)
        out = fs.flagsparse_attention_paged_tree(q, lengths, tokens, parents=parents, longest=8, prepared=kv,
                                                 window=window, sinks=sinks)
        keep = []
        for b, (n, tree) in enumerate(zip(new, trees)):
            way = _ways(tree)[int(torch.randint(0, n, (1,), generator=gen))]
            keep.append(torch.zeros(n, dtype=torch.bool))
            keep[-1][way] = True
            at = len(texts[b])
            first = sum(new[:b])
            seen[b] += [(at + i, q[first + a], out[first + a]) for i, a in enumerate(way)]
            texts[b] = torch.cat([texts[b], drafts[b][way]])
        lengths = fs.flagsparse_paged_keep(torch.cat(keep).to(dev), lengths, tokens, prepared=kv)
        assert lengths.tolist() == [len(t) for t in texts]
    for b, text in enumerate(texts):
        n = len(text)
        pos = torch.arange(n)
        here = _slots(kv, b, range(n))
        k, v = kv.k_pages[here], kv.v_pages[here]
        ref.check("k", k, _turned(text[:, h:h + g], pos, cos.cpu(), sin.cpu(), False))
        assert torch.equal(v.cpu(), text[:, h + g:])
        at = torch.tensor([i for i, _, _ in seen[b]])
        q = torch.zeros(n, h, d, dtype=BF)
        q[at] = torch.stack([x for _, x, _ in seen[b]]).cpu()
        turned = _turned(text[:, :h], pos, cos.cpu(), sin.cpu(), False)
        ref.check("q", q[at], tuple(x[at] for x in turned))
        want = ref.packed(q, k, v, [n], [n], True, window, d**-0.5, sinks=sinks)["out"]
        ref.check("out", torch.stack([x for _, _, x in seen[b]]), tuple(x[at] for x in want))


@pytest.mark.parametrize("share", [0.0, 0.5, 1.0])
def test_keep_into_other_pages_of_long_texts(dev, share):
    # so many marks that they are counted by pieces first: ragged texts, marks of all and of some of a text
    lengths, new = [40000, 0, 17, 20000, 3001, 33000], [39000, 0, 17, 20000, 1, 5]
    kv, k, v = _cache(dev, lengths, 16, 1, 8, BF, room=1)
    to, _, _ = _cache(dev, [40000, 0, 17, 15000, 3001, 33000], 24, 1, 8, BF, seed=5, room=1)
    before = to.k_pages.clone(), to.v_pages.clone()
    marks = _marks(new, share, 2)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    keep = torch.cat([torch.ones(3, dtype=torch.bool), *marks]).to(dev)[3:]
    want = [a - b + int(m.sum()) for a, b, m in zip(lengths, new, marks)]
    for _ in range(2):
        got = fs.flagsparse_paged_keep(keep, n, _indptr(new, dev), prepared=kv, into=to)
        assert got.tolist() == [-1 if b == 3 and share == 1.0 else m for b, m in enumerate(want)]  # no room for all
    changed = torch.zeros(to.n_pages, 24, dtype=torch.bool, device=dev)
    for b in range(len(lengths)):
        here = _slots(to, b, range(max(0, int(got[b]))))
        if int(got[b]) >= 0:
            for pages, rows in ((to.k_pages, k[b]), (to.v_pages, v[b])):
                assert torch.equal(pages[here].cpu(), _kept_rows(rows, new[b], marks[b]))
        changed[here] = True
    for now, then in zip((to.k_pages, to.v_pages), before):
        assert torch.equal(_bits(now[~changed]), _bits(then[~changed]))
    for bad in ([-1, 1, 16, 40000, 0, 4], [2**40, 17, 4000, 19999, -2**40, 2**31 - 1]):
        got = fs.flagsparse_paged_keep(keep, torch.tensor(bad, device=dev), _indptr(new, dev), prepared=kv, into=to)
        assert got[0] == got[2] == got[4] == got[5] == -1 and got[3] == -1
    for bad in ([0, 2**30, 17, 20000, 59018, 59023], [-5, 39000, 0, 39017, 0, 59018, 2**31 - 1]):
        fs.flagsparse_paged_keep(keep, n, torch.tensor((bad + [59023])[:7], device=dev), prepared=kv, into=to)
    torch.cuda.synchronize()


def test_keep_of_long_texts_in_a_graph(dev):
    lengths = [30000, 900]
    kv, k, _ = _cache(dev, lengths, 16, 2, 64, BF)
    to, _, _ = _cache(dev, lengths, 16, 2, 64, BF, seed=5)
    keep, tokens = torch.cat(_marks(lengths, 0.5, 1)).to(dev), _indptr(lengths, dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, into=to)
    with torch.cuda.graph(graph):
        got = fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, into=to)
    for seed in range(3):
        marks = _marks(lengths, 0.1 + 0.4 * seed, seed)
        keep.copy_(torch.cat(marks))
        eager = fs.flagsparse_paged_keep(keep, n, tokens, prepared=kv, into=to)
        to.k_pages.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, got)
        for b in range(2):
            here = _slots(to, b, range(int(got[b])))
            assert torch.equal(to.k_pages[here].cpu(), _kept_rows(k[b], lengths[b], marks[b]))


def test_keep_into_other_pages_takes_time_by_the_tokens(dev):
    # eight times the tokens of a text: eight times the time and not its square, 64 times
    def time_of(tokens):
        k, v, k2, v2 = (torch.zeros(tokens // 64, 64, 1, 8, dtype=BF, device=dev) for _ in range(4))
        table = torch.arange(tokens // 64, dtype=torch.int32, device=dev)
        ends = torch.tensor([0, tokens // 64], device=dev)
        kv, to = fs.prepare_paged_kv(k, v, ends, table), fs.prepare_paged_kv(k2, v2, ends, table)
        keep = torch.arange(tokens, device=dev) % 2 == 0
        n = torch.tensor([tokens], dtype=torch.int32, device=dev)
        best = float("inf")
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                got = fs.flagsparse_paged_keep(keep, n, prepared=kv, into=to)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        assert got.tolist() == [tokens // 2]
        return best

    assert time_of(1 << 21) <= 24 * time_of(1 << 18)


@pytest.mark.parametrize("dtype,half,interleaved", [(BF, 32, False), (HF, 32, True), (HF, 20, False), (BF, 17, True)])
def test_a_text_goes_on_after_tokens_were_given_up(dev, dtype, half, interleaved):
    # its kept keys stay where they stood in the text, and so do those that come after them
    dim, g, h, text, new = 64, 2, 4, [300, 41, 128], [3, 1, 5]
    cos, sin = _table(400, half)
    kw = {"cos": cos.to(dev), "sin": sin.to(dev), "interleaved": interleaved}
    kv, _, _ = _cache(dev, text, 16, g, dim, dtype, room=1)
    to, _, _ = _cache(dev, text, 16, g, dim, dtype, seed=5, room=1)
    k, v = (_normal(s, sum(text), g, dim, dtype=dtype) for s in (1, 2))
    n = torch.tensor(text, dtype=torch.int32, device=dev)
    fs.flagsparse_paged_append(k.to(dev), v.to(dev), n, _indptr(text, dev), prepared=kv, **kw)
    marks = _marks(text, 0.4, 3)
    left = fs.flagsparse_paged_keep(torch.cat(marks).to(dev), n, _indptr(text, dev), prepared=kv, into=to)
    pos = [m.nonzero().flatten() for m in marks]

    def check(cache, lengths, turns, key, value):
        at = 0
        for b, turn in enumerate(turns):
            here = _slots(cache, b, range(int(lengths[b]) - len(turn), int(lengths[b])))
            ref.check("k", cache.k_pages[here],
                      tuple(t for t in _turned(key[at:at + len(turn)], turn, cos, sin, interleaved)))
            assert torch.equal(cache.v_pages[here].cpu(), value[at:at + len(turn)])
            at += len(turn)

    check(to, left, pos, torch.cat([x[m] for x, m in zip(k.split(text), marks)]),
          torch.cat([x[m] for x, m in zip(v.split(text), marks)]))
    # one token each, several, and drafted ones
    for lengths, tree in ((None, None), (new, None), (new, [_tree(m, s) for s, m in enumerate(new)])):
        counts = lengths or [1] * 3
        depths = [[len(w) - 1 for w in _ways(t)] for t in tree] if tree else [list(range(m)) for m in counts]
        turns = [torch.tensor(d) + m for d, m in zip(depths, text)]
        kn, vn, q = (_normal(s, sum(counts), m, dim, dtype=dtype) for s, m in ((7, g), (8, g), (9, h)))
        more = torch.tensor(counts, device=dev)
        for cast in (torch.int32, torch.int64):
            got = fs.flagsparse_paged_append(
                kn.to(dev), vn.to(dev), (left + more).to(cast), lengths and _indptr(lengths, dev), prepared=to,
                q=q.to(dev), parents=torch.tensor(sum(tree, []), device=dev) if tree else None,
                text_lengths=(n + more).to(cast), **kw)
            ref.check("q", got, _turned(q, torch.cat(turns), cos, sin, interleaved))
            check(to, left + more, turns, kn, vn)
    # a position that the table does not hold, or before the text: not stored, and NaN
    before = _bits(to.k_pages).clone()
    for bad in (0, -7, 401, 2**40):
        wrong = torch.full((3,), bad, device=dev)
        q = _normal(9, 3, h, dim, dtype=dtype).to(dev)
        got = fs.flagsparse_paged_append(q[:, :g], q[:, :g], left + 1, prepared=to, q=q, text_lengths=wrong, **kw)
        assert torch.isnan(got).all() and torch.equal(_bits(to.k_pages), before)
    # without a rotation there is nothing to go by
    fs.flagsparse_paged_append(q[:, :g], q[:, :g], left + 1, prepared=to, text_lengths=wrong)
    here = _slots(to, 1, [int(left[1])])
    assert torch.equal(to.k_pages[here], q[1:2, :g])
    for bad in (n[:2], n.cpu(), n[None]):
        with pytest.raises(ValueError):
            fs.flagsparse_paged_append(q[:, :g], q[:, :g], left + 1, prepared=to, text_lengths=bad, **kw)
    with pytest.raises(TypeError):
        fs.flagsparse_paged_append(q[:, :g], q[:, :g], left + 1, prepared=to, text_lengths=n.float(), **kw)


def test_texts_as_long_as_the_cache_holds_are_the_call_without(dev):
    lengths = [70, 20]
    kv, _, _ = _cache(dev, lengths, 16, 2, 64, BF)
    cos, sin = (t.to(dev) for t in _table(80, 32))
    k, v, q = (_normal(s, 7, m, 64, dtype=BF).to(dev) for s, m in ((1, 2), (2, 2), (3, 4)))
    n, tokens = torch.tensor(lengths, dtype=torch.int32, device=dev), torch.tensor([0, 4, 7], device=dev)
    kw = {"prepared": kv, "q": q, "cos": cos, "sin": sin}
    for parents in (None, torch.tensor([-1, 0, 0, 1, -1, 0, 1], device=dev)):
        want = fs.flagsparse_paged_append(k, v, n, tokens, parents=parents, **kw)
        kept = _bits(kv.k_pages).clone()
        kv.k_pages.zero_()
        fs.flagsparse_paged_append(k, v, n, tokens, parents=parents, **kw)
        now = _bits(kv.k_pages).clone()
        kv.k_pages.zero_()
        got = fs.flagsparse_paged_append(k, v, n, tokens, parents=parents, text_lengths=n, **kw)
        assert torch.equal(got, want) and torch.equal(_bits(kv.k_pages), now)
        kv.k_pages.view(torch.int16).copy_(kept)


def test_copies_of_more_pages_than_one_launch_has(dev):
    n = 4_500_000
    x = torch.arange(2 * n, dtype=torch.int32, device=dev).view(torch.bfloat16).view(2 * n, 1, 1, 2)
    k = torch.cat([x] * 4, -1)
    v = k.view(torch.int16).bitwise_not().view(torch.bfloat16)
    want = [t.view(torch.int16)[n:].flip(0).clone() for t in (k, v)]
    at = torch.arange(n, dtype=torch.int32, device=dev)
    kv = fs.prepare_paged_kv(k, v, torch.zeros(1, dtype=torch.int32, device=dev), at[:0])
    fs.flagsparse_paged_copy(2 * n - 1 - at, at, prepared=kv)
    for t, w in zip((k, v), want):
        assert torch.equal(t.view(torch.int16)[:n], w) and torch.equal(t.view(torch.int16)[n:], w.flip(0))


def test_keep_of_more_tokens_than_one_launch_has(dev):
    # the same page for all places, here and there: as long as none but the last is dropped, places do not change
    page, times = 1 << 20, 1100
    kp, vp = (_normal(s, 1, page, 1, 8, dtype=BF).to(dev) for s in (1, 2))
    table = torch.zeros(times, dtype=torch.int32, device=dev)
    ends = torch.tensor([0, times], device=dev)
    kv = fs.prepare_paged_kv(kp, vp, ends, table)
    k2, v2 = torch.zeros_like(kp), torch.zeros_like(vp)
    to = fs.prepare_paged_kv(k2, v2, ends, table)
    n = torch.tensor([page * times], dtype=torch.int32, device=dev)
    got = fs.flagsparse_paged_keep(torch.tensor([True, True, False], device=dev), n, prepared=kv, into=to)
    assert got.tolist() == [page * times - 1]
    assert torch.equal(k2, kp) and torch.equal(v2, vp)
