"""Attention without a GPU: the work lists, the argument structs, the refusals that need no device, and
the 64-bit reference against autograd."""

import ctypes

import numpy as np
import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _abi, attention
from oracle import attention as ref


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("keys", [False, True])
@pytest.mark.parametrize("lengths", [([], []), ([5], [5]), ([0, 300, 64, 65], [7, 0, 64, 1000]),
                                     ([1] * 50, [3] * 50)])
def test_tiles_cover_every_row_once(lengths, keys, causal):
    q_len, k_len = (np.array(x, dtype=np.int64) for x in lengths)
    t = attention._tiles(q_len, k_len, 64, causal, keys)
    assert t.shape[1] == 8 and t.dtype == np.int32
    rows = k_len if keys else q_len
    seen = np.zeros(rows.sum(), dtype=int)
    begin = {False: np.cumsum(q_len) - q_len, True: np.cumsum(k_len) - k_len}
    work = []
    for first, n, at, q_begin, nq, k_begin, nk, zero in t.tolist():
        assert 1 <= n <= 64 and zero == 0
        seen[first:first + n] += 1
        b = [b for b in range(len(rows)) if rows[b] and
             begin[keys][b] <= first < begin[keys][b] + rows[b]][0]
        assert (q_begin, nq, k_begin, nk) == (begin[False][b], q_len[b], begin[True][b], k_len[b])
        assert first == begin[keys][b] + at and at + n <= rows[b]
        mask = ref.seen(nq, nk, causal, None)
        mask = mask[:, at:at + n] if keys else mask[at:at + n]
        work.append(int(mask.any(0 if not keys else 1).sum()))
    assert (seen == 1).all()
    assert work == sorted(work, reverse=True)


def test_exports_have_a_name_in_the_package():
    import flagsparse

    for name in fs.ATTENTION_EXPORTS:
        assert getattr(flagsparse, name) is getattr(fs, name)
        assert name not in fs.__all__  # the reference's list


def test_struct_sizes():
    # 8-byte fields, as in the header
    assert attention._CACHE.size == 8 * 17
    assert attention._APPEND.size + attention._APPEND_AT.size == 8 * 21
    assert attention._PAGED.size + attention._PAGED_AT.size == 8 * 17
    assert attention._PACKED.size + attention._PACKED_AT.size == 8 * (19 + 16 + 10)
    assert _abi.lib().fsp_attention_dim_cap() == attention._DIM_CAP


@pytest.mark.parametrize("pages", [[], [0], [8, 0, 9, 1], [320, 1, 8]])
def test_pieces_cover_the_rooms(pages):
    table, firsts, most = attention._pieces(np.array(pages, dtype=np.int64), 16, 128)
    at = 0
    assert most == max([1] + [-(-16 * n // 128) for n in pages])
    for b, n in enumerate(pages):
        first = at
        assert firsts[b] == first
        for i in range(max(1, -(-16 * n // 128))):
            assert table[at].tolist() == [b, 128 * i, first, sum(pages[:b]), 16 * n, 0, 0, 0]
            at += 1
    assert at == len(table)


def test_piece_sizes():
    L = _abi.lib()
    for tokens in (0, 1, 1000, 50000, 10**6, 2**31):
        for heads in (1, 8, 64):
            piece = L.fsp_attention_paged_piece(tokens, heads)
            assert 128 <= piece <= 1024 and piece % 128 == 0


def _packed(**kw):
    a = dict(dtype=2, heads=4, kv_heads=2, dim=64, q_tokens=8, k_tokens=8, q_longest=8, k_longest=8,
             causal=1, window=0, scale=0.125, q_tiles=16, n_q_tiles=1, q_halves=16, n_q_halves=2,
             k_tiles=16, n_k_tiles=1, k_halves=16, n_k_halves=2)
    for n in ("q", "k", "v", "out", "go", "gq", "gk", "gv"):
        a |= {n: 64, n + "_token": 256, n + "_head": 64}
    a |= {"lse": 16, "work": 16} | kw
    order = ["dtype", "heads", "kv_heads", "dim", "q_tokens", "k_tokens", "q_longest", "k_longest",
             "causal", "window", "scale", "q_tiles", "n_q_tiles", "q_halves", "n_q_halves", "k_tiles",
             "n_k_tiles", "k_halves", "n_k_halves"]
    eight = ("q", "k", "v", "out", "go", "gq", "gk", "gv")
    order += [n + e for n in eight for e in ("_token", "_head")]
    at = [*eight[:4], "lse", *eight[4:], "work"]
    return attention._PACKED.pack(*(a[n] for n in order)) + \
        attention._PACKED_AT.pack(*(a[n] for n in at))


@pytest.mark.parametrize("status,kw", [
    (-3, {"dtype": 0}), (-3, {"dim": 132}), (-3, {"dim": 12}), (-3, {"dim": 0}),
    (-1, {"heads": 3}), (-1, {"kv_heads": 0}), (-1, {"heads": 0}), (-1, {"q_tokens": -1}),
    (-1, {"n_q_tiles": 1 << 40}), (-1, {"window": -1}), (-1, {"window": 5, "causal": 0}),
    (-1, {"q": 0}), (-1, {"k": 0}), (-1, {"lse": 0}), (-1, {"q": 72}), (-1, {"k_token": 12}),
    (-1, {"v_head": 4}), (-1, {"out": 8}), (-1, {"q_tiles": 0})])
def test_packed_refusals_of_the_library(status, kw):
    L = _abi.lib()
    assert L.fsp_attention_packed(_packed(**kw), None) == status
    assert L.fsp_last_error()
    assert L.fsp_attention_packed_backward(_packed(**kw), None) == status
    assert L.fsp_attention_packed(None, None) == -1
    assert L.fsp_attention_packed_backward(None, None) == -1


@pytest.mark.parametrize("kw", [{"go": 0}, {"gq": 0}, {"gk": 0}, {"gv": 0}, {"work": 0}, {"go": 4},
                                {"gk_token": 3}, {"k_tiles": 0}])
def test_backward_refusals_of_the_library(kw):
    assert _abi.lib().fsp_attention_packed_backward(_packed(**kw), None) == -1


def _cache(**kw):
    a = dict(dtype=2, kv_heads=2, dim=64, page_size=16, n_pages=4, batch=2, table_len=3, k=64, kp=2048,
             ks=128, kh=64, v=64, vp=2048, vs=128, vh=64, indptr=16, indices=16) | kw
    return attention._CACHE.pack(*a.values())


_PAGED_ARGS = dict(pieces=16, first=16, n_pieces=3, piece=128, heads=4, window=0, scale=0.125, qt=256,
                   qh=64, ot=256, oh=64, q=64, out=64, lse=0, lengths=16, work=16, counts=16)
_APPEND_ARGS = dict(n_tokens=2, heads=4, half=32, rows=64, interleaved=0, kt=128, kh=64, vt=128, vh=64,
                    qt=256, qh=64, qot=256, qoh=64, k=64, v=64, q=64, qo=64, cos=16, sin=16, tokens=0,
                    lengths=16)


def _paged(**kw):
    a = list((_PAGED_ARGS | kw).values())
    return attention._PAGED.pack(*a[:11]) + attention._PAGED_AT.pack(*a[11:])


def _append(**kw):
    a = list((_APPEND_ARGS | kw).values())
    return attention._APPEND.pack(*a[:13]) + attention._APPEND_AT.pack(*a[13:])


@pytest.mark.parametrize("status,kw", [
    (-3, {"dtype": 1}), (-3, {"dim": 130}), (-1, {"page_size": 0}), (-1, {"batch": -1}),
    (-1, {"n_pages": 1 << 31}), (-1, {"table_len": 1 << 28}), (-1, {"k": 0}), (-1, {"v": 8}),
    (-1, {"kp": 4}), (-1, {"indptr": 0}), (-1, {"indices": 0})])
def test_cache_refusals_of_the_library(status, kw):
    L = _abi.lib()
    c = _cache(**kw)
    assert L.fsp_attention_paged(c + _paged(), None) == status
    assert L.fsp_paged_append(c + _append(), None) == status
    assert L.fsp_attention_paged(None, None) == -1 and L.fsp_paged_append(None, None) == -1


@pytest.mark.parametrize("kw", [{"heads": 3}, {"heads": 0}, {"window": -1}, {"q": 0}, {"out": 0},
                                {"lengths": 0}, {"q": 72}, {"oh": 2}, {"work": 0}, {"work": 8},
                                {"pieces": 0}, {"counts": 0, "first": 0}, {"n_pieces": 1}, {"n_pieces": 1 << 40},
                                {"piece": 0}, {"piece": 2048}, {"piece": 130}])
def test_paged_refusals_of_the_library(kw):
    L = _abi.lib()
    args = _cache() + _paged(**kw)
    assert L.fsp_attention_paged(args, None) == -1


@pytest.mark.parametrize("kw", [{"half": 33}, {"half": -1}, {"n_tokens": 3}, {"n_tokens": -1},
                                {"k": 0}, {"cos": 0}, {"qo": 0}, {"lengths": 0}, {"kt": 4},
                                {"rows": 1 << 32}])
def test_append_refusals_of_the_library(kw):
    L = _abi.lib()
    args = _cache() + _append(**kw)
    assert L.fsp_paged_append(args, None) == -1


def test_refusals_that_need_no_device():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    ip = torch.tensor([0, 4])
    with pytest.raises(ValueError):
        fs.flagsparse_attention_packed(q, q, q, ip)
    with pytest.raises(ValueError):
        fs.prepare_attention_packed(ip)
    with pytest.raises(ValueError):
        fs.prepare_paged_kv(q[None], q[None], ip, ip)
    with pytest.raises(TypeError):
        fs.flagsparse_attention_paged(q, ip, prepared=q)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_append(q, q, ip)


@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 3)])
def test_reference_is_the_gradient(causal, window):
    gen = torch.Generator().manual_seed(1)
    q, k, v, g = (torch.randn(9, 8, generator=gen).double() for _ in range(4))
    mask = ref.seen(9, 9, causal, window)
    r = ref.one(q, k, v, mask, 0.3, g)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    s = (leaves[0] @ leaves[1].T * 0.3).masked_fill(~mask, float("-inf"))
    out = torch.softmax(s, 1) @ leaves[2]
    out.backward(g)
    assert torch.allclose(out, r["out"], atol=1e-12)
    for t, n in zip(leaves, "qkv"):
        assert torch.allclose(t.grad, r[n], atol=1e-12)


def test_struct_of_bytes_reaches_the_library():
    # the structs go by address: a bytes object does
    assert isinstance(_packed(), bytes)
    assert ctypes.c_void_p in _abi.SIGNATURES["fsp_attention_packed"][1]


def _elements(t):
    i = sum(torch.arange(n).view(-1, *(1,) * (t.ndim - 1 - d)) * s
            for d, (n, s) in enumerate(zip(t.shape, t.stride())))
    return set((t.data_ptr() + t.element_size() * i).flatten().tolist())


def test_outputs_over_inputs_are_seen():
    # an output that shares an element with an input is not written by the kernel that reads it
    room = torch.zeros(4096, dtype=torch.float16)
    gen = torch.Generator().manual_seed(1)

    def some():
        n, h, d, s0, s1, at = (int(torch.randint(0, m, (1,), generator=gen)) for m in
                               (5, 4, 9, 6, 4, 200))
        return room.as_strided((n, h, 8 * (d % 2) + 8), (8 * [0, 1, 3, 8, 8, 9][s0], 8 * s1, 1), at)

    shared = 0
    for _ in range(3000):
        a, b = some(), some()
        if a.numel() and b.numel() and _elements(a) & _elements(b):
            assert attention._overlap(a, b) and attention._overlap(b, a)
            shared += 1
    assert shared > 300


def test_slices_side_by_side_do_not_overlap():
    fused = torch.zeros(7, 8, 16, dtype=torch.float16)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    for a, b in ((q, k), (k, q), (q, v), (k, v), (fused[:3], fused[3:]), (q, torch.zeros_like(q)),
                 (q, q[:0])):
        assert not attention._overlap(a, b)
    for a, b in ((q, q), (fused[:, 3:5], q), (q, fused[:, 3:5]), (fused[1:], fused[:-1]),
                 (q, fused[:, :, None].expand(7, 8, 2, 16)[:, 0, :1].expand(7, 4, 16)),
                 (q, fused.view(7, 2, 4, 16))):
        assert attention._overlap(a, b)


def test_a_graph_has_counts_of_its_own(monkeypatch):
    # of a stream with calls before: neither theirs, nor another graph's, nor kept for later calls
    class Cache:
        device, _counts = torch.device("cpu"), _abi.Calls()

    capturing = False
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    kept = attention._arrivals(Cache, 7, 5)
    assert attention._arrivals(Cache, 7, 5) is kept and attention._arrivals(Cache, 8, 5) is not kept
    before = dict(Cache._counts)
    capturing = True
    graphs = [attention._arrivals(Cache, 7, 5) for _ in range(2)]
    assert len({t.data_ptr() for t in (kept, *graphs)}) == 3
    for t in graphs:
        assert t.dtype == torch.int32 and t.shape == (5,) and not t.any()
    assert Cache._counts.keys() == before.keys()
    assert all(Cache._counts[n] is before[n] for n in before)


@pytest.mark.parametrize("tokens", [2**31 - 1023, 2**31 - 16, 2**31 - 1])
def test_lengths_that_a_step_would_pass_32_bits_from(tokens):
    # places up to a step (1024 tokens) past the last token are 32-bit numbers in the kernels
    L = _abi.lib()
    for kw in ({"q_tokens": tokens}, {"k_tokens": tokens}):
        assert L.fsp_attention_packed(_packed(**kw), None) == -1
        assert L.fsp_attention_packed_backward(_packed(**kw), None) == -1
    c = _cache(table_len=tokens, page_size=1)
    assert L.fsp_attention_paged(c + _paged(), None) == -1
    assert L.fsp_paged_append(c + _append(), None) == -1
    assert attention._TOKENS_CAP == 2**31 - 1024


@pytest.mark.parametrize("tokens,heads", [(1, 4), (5, 1), (1, 1), (5, 4)])
def test_rows_have_steps_that_the_kernels_take(tokens, heads):
    # whatever an axis of one element has as its step, which contiguous() keeps
    for room, s0, s1 in ((5000, 515, 64), (5000, 512, 67), (5000, 515, 67), (5000, 512, 64), (5000, 3, 5)):
        t = torch.zeros(room, dtype=torch.float16).as_strided((tokens, heads, 64), (s0, s1, 1))
        if t.data_ptr() % 16:
            continue
        r = attention._rows(t)
        s = attention._steps(r)
        assert torch.equal(r, t) and s[0] % 8 == 0 and s[1] % 8 == 0 and 64 <= s[0] <= 2**23
        if (tokens == 1 or s0 == 512) and (heads == 1 or s1 == 64):
            assert r is t  # no copy for a step that says nothing


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_scales_of_the_library_are_finite(scale):
    L = _abi.lib()
    assert L.fsp_attention_packed(_packed(scale=scale), None) == -1
    assert L.fsp_attention_packed_backward(_packed(scale=scale), None) == -1
    assert L.fsp_attention_paged(_cache() + _paged(scale=scale), None) == -1
    with pytest.raises(ValueError):
        attention._scale_of(scale, 64)


def test_tangents_are_seen():
    t = torch.zeros(3)
    assert not attention._has_tangent(t, None)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(t, torch.ones(3))
        assert attention._has_tangent(t, dual) and not attention._has_tangent(t, None)
        with torch.no_grad():
            assert attention._has_tangent(dual)
