"""Drafted trees, kept tokens and copied pages without a GPU: work lists, argument structs, the refusals of the
library, and which drafted tokens the tests' reference lets a row see."""

import numpy as np
import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _abi, attention
from tests import test_attention_cpu as base
from tests.test_gpu_tree import _masks, _ways

_TREE_ARGS = dict(pieces=16, first=16, n_pieces=3, piece=256, heads=4, window=0, scale=0.125, sinks=0, tokens=6,
                  longest=3, qt=256, qh=64, ot=256, oh=64, q=64, out=64, lse=0, lengths=16, indptr=16,
                  parents=16, work=16, counts=0)
_KEEP_ARGS = dict(other=0, tokens=6, each=3, n_pieces=3, piece=256, pieces=16, keep=3, indptr=16, lengths=16,
                  kept=16)


def _tree(**kw):
    a = list((_TREE_ARGS | kw).values())
    return attention._TREE.pack(*a[:14]) + attention._TREE_AT.pack(*a[14:])


def _keep(**kw):
    a = list((_KEEP_ARGS | kw).values())
    return attention._KEEP.pack(*a[:5]) + attention._KEEP_AT.pack(*a[5:])


def test_struct_sizes():
    assert attention._TREE.size + attention._TREE_AT.size == 8 * 22
    assert attention._KEEP.size + attention._KEEP_AT.size == 8 * 10
    assert _abi.lib().fsp_attention_tree_drafts() == 256


@pytest.mark.parametrize("kw", [
    {"heads": 3}, {"heads": 0}, {"window": -1}, {"window": 2**40}, {"sinks": 4}, {"sinks": -1, "window": 4},
    {"sinks": 2**31, "window": 4}, {"scale": float("nan")}, {"scale": 1e39}, {"piece": 0}, {"piece": 130},
    {"piece": 1 << 21}, {"n_pieces": 1}, {"n_pieces": 1 << 40}, {"tokens": -1}, {"tokens": 2**31},
    {"longest": 257}, {"longest": -1}, {"longest": 0}, {"indptr": 0, "tokens": 5}, {"q": 0}, {"q": 72},
    {"out": 0}, {"oh": 2}, {"qt": 12}, {"lengths": 0}, {"pieces": 0}, {"work": 0}, {"work": 8}, {"first": 0}])
def test_tree_refusals_of_the_library(kw):
    L = _abi.lib()
    assert L.fsp_attention_tree(base._cache() + _tree(**kw), None) == -1
    assert L.fsp_last_error()
    assert L.fsp_attention_tree(None, None) == -1


@pytest.mark.parametrize("kw", [{"tokens": -1}, {"tokens": 2**31}, {"each": -1}, {"each": 2, "indptr": 0},
                                {"keep": 0}, {"lengths": 0}, {"kept": 0}])
def test_keep_refusals_of_the_library(kw):
    L, c = _abi.lib(), base._cache()
    for other in (0, 1):
        assert L.fsp_paged_keep(c + c + _keep(**({"other": other} | kw)), None) == -1
    assert L.fsp_paged_keep(None, None) == -1


@pytest.mark.parametrize("kw", [{"dtype": 3}, {"kv_heads": 1}, {"dim": 72}, {"batch": 1}, {"k": 0},
                                {"page_size": 0}, {"kp": 4}])
def test_keep_refuses_another_kind_of_cache(kw):
    c = base._cache()
    assert _abi.lib().fsp_paged_keep(c + base._cache(**kw) + _keep(other=1), None) == -1


@pytest.mark.parametrize("kw", [{"pieces": 0}, {"n_pieces": 1}, {"n_pieces": 1 << 40}, {"piece": 0},
                                {"piece": 2048}, {"piece": 200}])
def test_keep_into_refuses_lists(kw):
    c = base._cache()
    assert _abi.lib().fsp_paged_keep(c + c + _keep(other=1, **kw), None) == -1


@pytest.mark.parametrize("status,kw", [
    (-3, {"dtype": 1}), (-3, {"dim": 130}), (-1, {"page_size": 0}), (-1, {"batch": -1}),
    (-1, {"n_pages": 1 << 31}), (-1, {"table_len": 1 << 28}), (-1, {"k": 0}), (-1, {"v": 8}),
    (-1, {"kp": 4}), (-1, {"indptr": 0}), (-1, {"indices": 0})])
def test_cache_refusals_of_the_library(status, kw):
    L, c = _abi.lib(), base._cache(**kw)
    assert L.fsp_attention_tree(c + _tree(), None) == status
    assert L.fsp_paged_keep(c + c + _keep(), None) == status
    assert L.fsp_paged_copy(c, 16, 16, 4, None) == status
    assert L.fsp_paged_append_drafts(c + base._append(), 16, None) == status


def test_copy_and_append_refusals_of_the_library():
    L, c = _abi.lib(), base._cache()
    for args in ((c, None, 16, 4), (c, 16, None, 4), (c, 16, 16, -1), (c, 16, 16, 1 << 40), (None, 16, 16, 4)):
        assert L.fsp_paged_copy(*args, None) == -1
    assert L.fsp_paged_copy(c, None, None, 0, None) == 0
    huge = base._cache(page_size=1 << 30, n_pages=1, table_len=1)
    assert L.fsp_paged_copy(huge, 16, 16, 1, None) == -1  # its rows are counted in 32 bits
    assert L.fsp_paged_append_drafts(c + base._append(), None, None) == -1
    assert L.fsp_paged_append_drafts(None, 16, None) == -1
    assert L.fsp_paged_append_drafts(c + base._append(half=33), 16, None) == -1


@pytest.mark.parametrize("pages", [[], [0], [8, 0, 9, 1], [320, 1, 8]])
@pytest.mark.parametrize("sight", [1, 100, 256, 257, 3000, 2**31 - 1024])
def test_pieces_under_a_window(pages, sight):
    # as many as ``sight`` tokens in a row can touch wherever they start, no more than the room takes
    table, firsts, most = attention._pieces(np.array(pages, dtype=np.int64), 16, 256, sight)
    at = 0
    for b, n in enumerate(pages):
        assert firsts[b] == at
        room = max(1, -(-16 * n // 256))
        need = max(len(set(range(s // 256, (s + min(sight, 6000) - 1) // 256 + 1))) for s in range(256))
        count = int((table[:, 0] == b).sum())
        assert min(room, need) <= count <= room
        for i in range(count):
            assert table[at].tolist() == [b, 256 * i, int(firsts[b]), sum(pages[:b]), 16 * n, 0, 0, 0]
            at += 1
    assert at == len(table) and most == max([1] + np.bincount(table[:, 0], minlength=1).tolist())


@pytest.mark.parametrize("rooms", [[], [0], [16], [30064] * 8, [2048, 0, 300, 16], [131072, 5], [1] * 900,
                                   [2**31 - 1024]])
@pytest.mark.parametrize("sight", [0, 1, 700, 100000])
def test_sizes_of_pieces(rooms, sight):
    rooms = np.array(rooms, dtype=np.int64)
    for each, slots, most, rows in ((1, 512, 8192, 128), (16, 512, 8192, 32), (8, 768, 1024, 16),
                                    (400, 512, 8192, 128)):
        piece = attention._piece_of(rooms, sight, each, slots, most, rows)
        assert 256 <= piece <= most and piece % 128 == 0


def test_pieces_fill_whole_rounds():
    # 8 sequences, 16 workgroups a piece: four even pieces each are one round of 512
    assert attention._piece_of(np.full(8, 30064), 0, 16, 512, 8192, 128) == 7552


def test_rows_of_a_tile():
    L = _abi.lib()
    assert L.fsp_attention_tree_rows(0, 4) == L.fsp_attention_tree_rows(4, 0) == 16
    for group, longest in ((1, 1), (4, 4), (4, 8), (23, 26), (1, 256), (64, 256)):
        assert L.fsp_attention_tree_rows(group, longest) in (16, 32, 128)


def test_ways_and_masks_of_the_reference():
    assert _ways([-1, 0, 0, 2, -1]) == [[0], [0, 1], [0, 2], [0, 2, 3], [4]]
    m = _masks([2], [[-1, 0, 0, 2]])[0]
    assert m.int().tolist() == [[1, 1, 1, 0, 0, 0], [1, 1, 1, 1, 0, 0], [1, 1, 1, 0, 1, 0], [1, 1, 1, 0, 1, 1]]
    m = _masks([2], [[-1, 0, 0, 2]], window=2, sinks=1)[0]
    # positions 2, 3, 3, 4
    assert m.int().tolist() == [[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 1, 0, 1, 0], [1, 0, 0, 0, 1, 1]]


def test_refusals_that_need_no_device():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    n = torch.tensor([4])
    with pytest.raises(TypeError):
        fs.flagsparse_attention_paged_tree(q, n, prepared=q)
    with pytest.raises(ValueError):
        fs.flagsparse_attention_paged_tree(q, n)
    with pytest.raises(TypeError):
        fs.flagsparse_paged_keep(n > 0, n, prepared=q)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_keep(n > 0, n)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_copy(n, n)
    with pytest.raises(TypeError):
        fs.flagsparse_paged_copy(n, n, prepared=q)
    with pytest.raises(ValueError):
        fs.flagsparse_paged_copy(n, n, k_pages=q[None], v_pages=q[None])


@pytest.mark.parametrize("kw,refusal", [
    ({"heads": 32, "longest": 256, "n_pieces": 262_143}, b"null pointer"),  # 2 x 32 tiles of 128 rows
    ({"heads": 32, "longest": 256, "n_pieces": 262_144}, b"out of range"),
    ({"heads": 4, "longest": 8, "n_pieces": 8_388_607}, b"null pointer"),  # 2 x 1 of 16
    ({"heads": 4, "longest": 8, "n_pieces": 8_388_608}, b"out of range")])
def test_pieces_of_a_launch(kw, refusal):
    # as many workgroups as a launch holds: a piece has one for every tile of rows and key head
    L = _abi.lib()
    assert L.fsp_attention_tree(base._cache() + _tree(tokens=8, q=0, **kw), None) == -1
    assert refusal in L.fsp_last_error()


@pytest.mark.parametrize("kw,refusal", [
    ({"n_pieces": 9000}, b"null pointer"),  # one each: nothing is joined
    ({"n_pieces": 9001}, b"out of range")])
def test_sequences_of_the_launch_that_joins(kw, refusal):
    L = _abi.lib()
    args = base._cache(batch=9000) + _tree(heads=64, longest=256, tokens=9000, q=0, **kw)
    assert L.fsp_attention_tree(args, None) == -1 and refusal in L.fsp_last_error()


def test_partial_sums_by_tokens():
    L = _abi.lib()
    # 64 sequences with room for 131072 tokens, 8 drafted ones each, no bound of them: rows of 128 + 2 numbers
    assert L.fsp_attention_tree_by_tokens_workspace(16, 512, 32, 128) == 16 * 512 * 32 * 130 * 4
    assert L.fsp_attention_tree_workspace(1024, 32, 128, 256) == 32 * 16 * 512 * 32 * 130 * 4
    assert L.fsp_attention_tree_by_tokens_workspace(-1, 512, 32, 128) == 0
    most = 2**31 - 1024
    assert L.fsp_attention_tree_by_tokens_workspace(2000, most, 64, 128) == 2000 * most * 64 * 520
    for most in (0, -1, 4):
        assert L.fsp_attention_tree_by_tokens(base._cache() + _tree(), most, None) == -1
    assert L.fsp_attention_tree_by_tokens(None, 1, None) == -1
    assert L.fsp_attention_tree_by_tokens(base._cache() + _tree(q=0), 2, None) == -1


def test_counted_keep_refusals_of_the_library():
    L, c = _abi.lib(), base._cache()
    call = L.fsp_paged_keep_counted
    assert call(None, 16, 16, None) == -1 and call(c + c + _keep(other=0), 16, 16, None) == -1
    for first, counts in ((None, 16), (16, None)):
        assert call(c + c + _keep(other=1), first, counts, None) == -1
    for kw in ({"tokens": -1}, {"keep": 0}, {"lengths": 0}, {"kept": 0}, {"pieces": 0}, {"n_pieces": 1},
               {"piece": 200}):
        assert call(c + c + _keep(**({"other": 1} | kw)), 16, 16, None) == -1


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 3), (8, 4), (1, 23), (1, 64), (3, 128)])
def test_ways_of_all_numbers_of_drafts(kv_heads, group):
    # what a call may look up, for any longest tree and any number of tokens, is among the ways
    L = _abi.lib()
    ways = attention._tree_ways(kv_heads, group)
    assert len(set(ways)) == len(ways) <= 10 + 4 * (2 * group).bit_length()
    for longest in (1, 2, 4, 5, 8, 9, 31, 100, 255, 256):
        rows = L.fsp_attention_tree_rows(group, longest)
        for tiles in range(1, -(-group * longest // rows) + 1):
            near = attention._near(tiles)
            assert abs(near - tiles) * 8 <= tiles and (tiles > 8 or near == tiles), (tiles, near)
            assert (kv_heads * near, rows) in ways


def test_sizes_of_pieces_of_several_ways():
    # those of each way alone, the soonest end by the rule written out
    rooms, slots, most = np.array([30064, 700, 0, 16, 9000, 4096], dtype=np.int64), 512, 8192
    ways = attention._tree_ways(4, 3) + ((600, 32),)

    def end_of(piece, each, rows):
        held = sorted((min(piece, n - at) for n in rooms for at in range(0, n, piece)), key=lambda n: (n < piece, -n))
        work = [n + 100 + 2 * rows for n in held for _ in range(each)]
        return sum(work[::slots]) + max(sum(work) / slots, work[0])

    sizes = attention._pieces_of(rooms, 0, ways, slots, most)
    for (each, rows), size in zip(ways, sizes):
        assert size == attention._piece_of(rooms, 0, each, slots, most, rows)
        assert all(end_of(size, each, rows) <= end_of(piece, each, rows) for piece in (256, 1024, 7552, 8192))


def test_copies_of_as_many_pages_as_there_are():
    L, c = _abi.lib(), base._cache(page_size=1, n_pages=2**31 - 1)
    assert L.fsp_paged_copy(c, None, 16, 2**31 - 1, None) == -1 and b"null pointer" in L.fsp_last_error()
    assert L.fsp_paged_copy(c, None, 16, 2**31, None) == -1 and b"out of range" in L.fsp_last_error()
