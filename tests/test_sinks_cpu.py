"""First tokens that stay visible under a window, without a GPU: refusals of the library and its sizes."""

import numpy as np
import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _abi, attention
from oracle import attention as ref
from tests import test_attention_cpu as base


@pytest.mark.parametrize("sinks,window,status", [(-1, 5, -1), (4, 0, -1), (2**31, 5, -1), (2**40, 5, -1)])
def test_refusals_of_the_library(sinks, window, status):
    L = _abi.lib()
    assert L.fsp_attention_packed_sinks(base._packed(window=window), sinks, None) == status
    assert L.fsp_attention_packed_sinks_backward(base._packed(window=window), sinks, 64, 1, None) == status
    assert L.fsp_attention_paged_sinks(base._cache() + base._paged(window=window), sinks, None) == status
    assert L.fsp_last_error()


def test_null_arguments():
    L = _abi.lib()
    assert L.fsp_attention_packed_sinks(None, 4, None) == -1
    assert L.fsp_attention_packed_sinks_backward(None, 4, None, 0, None) == -1
    assert L.fsp_attention_paged_sinks(None, 4, None) == -1
    for sequences, batch in ((None, 1), (64, 0), (64, -1), (64, 2**40)):
        assert L.fsp_attention_packed_sinks_backward(base._packed(window=5), 4, sequences, batch, None) == -1
    assert L.fsp_attention_packed_sinks_backward(base._packed(window=5, work=0), 4, 64, 1, None) == -1


@pytest.mark.parametrize("kw", [{"dtype": 0}, {"dim": 132}, {"heads": 3}, {"q": 72}, {"q_tokens": 2**31 - 1}])
def test_what_the_calls_without_refuse(kw):
    L = _abi.lib()
    kw = {"window": 5} | kw
    assert L.fsp_attention_packed_sinks(base._packed(**kw), 4, None) < 0
    assert L.fsp_attention_packed_sinks_backward(base._packed(**kw), 4, 64, 1, None) < 0


def test_jobs_that_a_launch_cannot_hold():
    # jobs of 32 first keys and 512 queries each, times the key heads, are workgroups of one launch
    many = base._packed(window=5, q_tokens=2**31 - 1024, k_tokens=2**31 - 1024, k_longest=2**31 - 1024)
    assert _abi.lib().fsp_attention_packed_sinks_backward(many, 2**31 - 1024, 64, 1, None) == -1


def test_first_keys_that_numbers_cannot_hold():
    # more than 2^30 vectors of four elements of their sums; and jobs of as many queries as there can be
    many = base._packed(window=5, heads=1, kv_heads=1, dim=128, k_tokens=2**25 - 1024, k_longest=2**25 - 1024)
    assert _abi.lib().fsp_attention_packed_sinks_backward(many, 2**25, 64, 1, None) == -1
    assert b"sinks of so many" in _abi.lib().fsp_last_error()
    sizes = (40, 8, 2, 64, 1000, 1000, 600, 3)
    assert _abi.lib().fsp_attention_packed_sinks_workspace(*sizes, 2**31 - 1, 4) == \
        _abi.lib().fsp_attention_packed_sinks_workspace(*sizes, 2**20, 4)


@pytest.mark.parametrize("q_len,chunk", [([0], 512), ([5, 0, 700, 512, 513], 512), ([1] * 900, 512),
                                         ([1024, 0, 0, 3], 640)])
def test_slots_of_jobs_are_apart(q_len, chunk):
    # slot q_begin / chunk + b + i for the i-th chunk of sequence b, fewer than q_tokens / chunk + batch
    begin = np.cumsum(q_len) - q_len
    taken = [int(q) // chunk + b + i for b, (q, n) in enumerate(zip(begin, q_len))
             for i in range(-(-n // chunk))]
    assert len(set(taken)) == len(taken)
    assert not taken or max(taken) < sum(q_len) // chunk + len(q_len)


def test_workspace_holds_the_jobs():
    L = _abi.lib()
    sizes = (40, 8, 2, 64, 1000, 1000)
    without = L.fsp_attention_packed_workspace(*sizes, 0)
    assert L.fsp_attention_packed_sinks_workspace(*sizes, 600, 3, 100, 0) == without
    rows = L.fsp_attention_packed_sinks_workspace(*sizes, 600, 3, 100, 4) - without
    # 1000 / 512 + 3 slots, two key heads, 64 rows of keys and of values, 32 bits, shares of 4 heads
    assert rows % (4 * 2 * 64 * 2 * 64 * 4) == 0 and rows // (4 * 2 * 64 * 2 * 64 * 4) in (1, 2, 4)
    assert L.fsp_attention_packed_sinks_workspace(*sizes, 600, 3, 100, 70) - without == 2 * rows
    # 600 of them, the longest sequence's, in jobs of 640 queries
    assert L.fsp_attention_packed_sinks_workspace(*sizes, 600, 3, 100, 2**30) - without == 10 * rows


def test_workspace_without_queries():
    # two slots, two key heads in one share, 64 rows of keys and of values, 32 bits
    assert _abi.lib().fsp_attention_packed_sinks_workspace(12, 2, 2, 64, 0, 709, 700, 2, 30, 7) == \
        2 * 2 * 64 * 2 * 64 * 4


def test_sinks_of():
    assert attention._sinks_of(None, 0) == 0 and attention._sinks_of(0, 0) == 0
    assert attention._sinks_of(3, 5) == 3 and attention._sinks_of(2**40, 5) == 2**31 - 1024
    for sinks, window in ((3, 0), (-1, 5)):
        with pytest.raises(ValueError):
            attention._sinks_of(sinks, window)


def test_windows_that_hide_nothing():
    for window, sinks, most, want in ((5, 3, 8, (0, 0)), (5, 3, 9, (5, 3)), (5, 0, 4, (5, 0)), (None, 0, 4, (0, 0)),
                                      (2**40, 2**40, 100, (0, 0)), (1, 7, 8, (0, 0)), (4, None, 2, (4, 0))):
        assert attention._sight_of(window, sinks, most) == want
    for window, sinks in ((None, 3), (5, -1), (0, 0), (-2, 0)):
        with pytest.raises(ValueError):
            attention._sight_of(window, sinks, 100)


def test_reference_sees_first_keys():
    m = ref.seen(4, 6, True, 2, 1)
    assert m.tolist() == [[True, True, True, False, False, False], [True, False, True, True, False, False],
                          [True, False, False, True, True, False], [True, False, False, False, True, True]]
    assert torch.equal(ref.seen(4, 6, True, 2, 0), ref.seen(4, 6, True, 2))


def test_refusals_that_need_no_device():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        fs.flagsparse_attention_packed(q, q, q, torch.tensor([0, 4]), window=2, sinks=1)


@pytest.mark.parametrize("heads,kv_heads,tokens", [(64, 8, 8_000_000), (32, 1, 4_000_000), (64, 1, 8_000_000),
                                                   (48, 16, 8_000_000)])
def test_tiles_of_several_heads_are_counted_as_workgroups(heads, kv_heads, tokens):
    # a tile of fewer tokens holds as many more heads: as many tokens as without first ones, refused here only for
    # the array that is missing
    L = _abi.lib()
    sizes = {"window": 5, "heads": heads, "kv_heads": kv_heads, "q_tokens": tokens, "k_tokens": tokens, "q": 0}
    tiles, halves = (-(-tokens // L.fsp_attention_packed_sinks_tile(which, heads // kv_heads)) for which in (0, 1))
    for n_tiles, n_halves, refusal in ((tiles, halves, b"null pointer"), (2**24, halves, b"out of range"),
                                       (tiles, 2**24, b"out of range")):
        args = base._packed(n_q_tiles=n_tiles, n_q_halves=n_halves, **sizes)
        assert L.fsp_attention_packed_sinks(args, 4, None) == -1 and refusal in L.fsp_last_error()
        assert L.fsp_attention_packed_sinks_backward(args, 4, 64, 1, None) == -1 and refusal in L.fsp_last_error()


@pytest.mark.parametrize("q_len,chunk", [([5, 0, 700, 512, 513], 512), ([1] * 900 + [513] + [2] * 900, 512),
                                         ([513] * 40, 512), ([1024, 0, 0, 641, 3, 640, 2000], 640),
                                         ([2**30, 2**30 - 2000, 976], 512), ([0, 0], 512), ([511, 1, 513], 512)])
def test_slots_by_twice_the_chunks_are_apart(q_len, chunk):
    # slot 2 * q_begin / chunk + i for the i-th chunk of a sequence of more than one, no more than twice
    # q_tokens / chunk + 1; the last sequence whose first slot is no later than a job's is the job's
    begin = [int(n) for n in np.cumsum(q_len) - q_len]
    first = [2 * q // chunk for q in begin]
    taken = []
    for b, (q, n) in enumerate(zip(begin, q_len)):
        for i in list(range(-(-n // chunk)))[:3] + [max(0, -(-n // chunk) - 1)] if n > chunk else ():
            assert max(x for x in range(len(first)) if first[x] <= first[b] + i) == b
        if n > chunk:
            taken.append((first[b], first[b] + -(-n // chunk)))
    assert all(a[1] <= b[0] for a, b in zip(taken, taken[1:]))
    assert not taken or taken[-1][1] <= 2 * (sum(q_len) // chunk + 1)


def test_workspace_of_short_sequences():
    L = _abi.lib()
    # 20000 sequences of 64 tokens have no job: the workspace of the call without first ones
    sizes = (20000, 32, 8, 128, 1_280_000, 1_280_000)
    assert L.fsp_attention_packed_sinks_chunk(32, 4, 64) == 512
    assert L.fsp_attention_packed_sinks_chunk(700, 4, 64) == 768 and L.fsp_attention_packed_sinks_chunk(0, 4, 64) == 0
    assert L.fsp_attention_packed_sinks_chunk(32, 900, 2000) == 1024
    # with one of 1000 beside them slots go by the queries, not by the sequences
    rows = L.fsp_attention_packed_sinks_workspace(*sizes, 1000, 20001, 32, 4) - \
        L.fsp_attention_packed_workspace(*sizes, 0)
    assert rows == 2 * (1_280_000 // 512 + 1) * 8 * 2 * 64 * 128 * 4
    # the library asks for no more: 58254 sequences were the most
    args = dict(window=32, heads=32, kv_heads=8, dim=128, q_tokens=10**7, k_tokens=10**7, q_longest=64, k_longest=64,
                go=0)
    assert L.fsp_attention_packed_sinks_backward(base._packed(**args), 4, 64, 10**6, None) == -1
    assert b"null pointer" in L.fsp_last_error()


@pytest.mark.parametrize("batch,q_longest", [(10**6, 64), (10**6, 5000), (200_000, 5000)])
def test_as_many_sequences_as_there_are(batch, q_longest):
    # with jobs and without: what is launched for the first keys' sums goes by the queries
    args = dict(window=32, heads=32, kv_heads=8, dim=128, q_tokens=2 * 10**7, k_tokens=2 * 10**7, go=0,
                q_longest=q_longest, k_longest=q_longest)
    assert _abi.lib().fsp_attention_packed_sinks_backward(base._packed(**args), 4, 64, batch, None) == -1
    assert b"null pointer" in _abi.lib().fsp_last_error()


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 130, 4096, 4097, 9000])
def test_search_for_the_sequence_of_a_slot(batch):
    # 64 at a look of the first slots, as the kernels do it
    rng = np.random.default_rng(batch)
    for twice in (False, True):
        q_len = rng.integers(0, 3, batch) * rng.integers(0, 900, batch)
        begin = np.cumsum(q_len) - q_len
        first = 2 * begin // 512 if twice else begin // 512 + np.arange(batch)
        for slot in {0, int(first[-1]), int(first[-1]) + 3, *rng.integers(0, first[-1] + 2, 40).tolist()}:
            b, n = 0, batch
            while n > 1:
                step = -(-n // 64)
                looks = [b + lane * step for lane in range(64) if lane * step < n]
                seen = [bool(first[i] <= slot) for i in looks]
                count = sum(seen)
                assert count >= 1 and all(seen[:count])
                b, n = b + (count - 1) * step, min(step, n - (count - 1) * step)
            assert b == int(np.nonzero(first <= slot)[0][-1])
