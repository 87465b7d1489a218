"""Attention over packed sequences and over a paged cache on gfx950.

Sequences of different lengths are rows of a CSR pattern: ``indptr`` over the tokens of a packed
batch, or over the pages that a cache holds of each sequence (``indices``: the pages).

* ``flagsparse_paged_append``: new keys and values, rotated by their positions, into the cache;
* ``flagsparse_paged_keep``: some of a sequence's last tokens stay and close up; ``flagsparse_paged_copy``:
  pages are copied;
* ``flagsparse_attention_paged``: one new query per sequence over all that the cache holds of it;
* ``flagsparse_attention_paged_tree``: the queries of a tree of drafted tokens, of which each sees its way;
* ``flagsparse_attention_packed`` and ``..._backward``: whole sequences, packed one after the other,
  causal, with a sliding window, or between two batches of sequences; with its gradient.

Queries, keys and values are [tokens, heads, dim] in bfloat16 or float16, ``dim`` a multiple of 8 up
to 128; the query heads are shared out evenly over the key heads.  Where query i sees the keys j,
S_ij = scale * q_i . k_j, lse_i = log(sum_j exp(S_ij)) and out_i = sum_j exp(S_ij - lse_i) v_j; a query that
sees no key has an output of zeros and an lse of minus infinity.  Everything is summed in 32 bits and
every sum has a fixed order: equal calls give equal results, bit for bit.

As with the sparse products, ``prepare_*`` checks index arrays once (the host waits for them) and
the calls with ``prepared=`` neither check them again nor wait: they can be captured in a graph.
"""

import functools
import struct

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _abi
from ._common import SUPPORTED_INDEX_DTYPES, _aligned
from ._csr_check import _capturing, csr_check

SUPPORTED_ATTENTION_DTYPES = (torch.bfloat16, torch.float16)

_CODES = {torch.bfloat16: _abi.FSP_BF16, torch.float16: _abi.FSP_F16}
_DIM_CAP = 128
_TOKENS_CAP = 2**31 - 1024  # a place past the last token by a step of any kernel is still an int32
_STEP_CAP = 2**23
_FLOAT_MAX = (2 - 2.0**-23) * 2.0**127

# The argument structs of include/flagsparse_hip.h: 8-byte fields, "d" the scale.  What a call's
# shapes, steps and types settle comes first, then the addresses of its arrays.
_CACHE = struct.Struct("17q")
_APPEND, _APPEND_AT = struct.Struct("13q"), struct.Struct("8q")
_PAGED, _PAGED_AT = struct.Struct("6qd4q"), struct.Struct("6q")
_PACKED, _PACKED_AT = struct.Struct("10qd24q"), struct.Struct("10q")
_KEEP, _KEEP_AT = struct.Struct("5q"), struct.Struct("5q")
_TREE, _TREE_AT = struct.Struct("6qd7q"), struct.Struct("8q")

# Where a text may have more marks than so many, they are counted by pieces before it is kept into other pages, by
# two more launches.  Without and with that, half of the tokens kept, us: 16 texts of 8192, 8 heads of 128 120 / 124,
# 16 of 16384 224 / 226, 8 of 32768 236 / 226, 4 of 131072 600 / 430; one head of 64, a text of 16384 12 / 19, of
# 32768 15 / 19, 8 of 16384 26 / 21, one of 131072 79 / 22, of 2^20 3482 / 112.
_COUNTED_FROM = 16384

# A prepared object keeps the first part for each layout of arrays that it has checked, so that the
# next call with such arrays is a look-up and a launch.  Of a cache it holds the pages' addresses, which
# the look-up goes by too: their storage is the caller's, and may move.
_KEPT_LAYOUTS = 64
_PLAIN = (type(None), bool, int, float)  # the settings a layout is kept with, by their values


_CONTIGUOUS = torch.contiguous_format


def _like(shape, dtype, device):
    """A pattern for new arrays: ``torch.empty_like(pattern, memory_format=_CONTIGUOUS)`` takes a third of
    the time of torch.empty with a shape, a type and a device.  One element of memory."""
    return torch.empty(1, dtype=dtype, device=device).expand(shape)


def _keep(calls, key, value):
    if len(calls) >= _KEPT_LAYOUTS:
        calls.clear()
    calls[key] = value


class _Streams:
    """The streams that a prepared object's arrays are marked as used on (see mark); a copy's arrays
    are other arrays, marked nowhere."""

    __slots__ = ("seen",)

    def __init__(self):
        self.seen = set()

    def __reduce__(self):
        return _Streams, ()

    def mark(self, stream, device, arrays):
        """Marks the arrays as used on ``stream``, the current one, once: calls do not wait, so
        without the mark the caching allocator could hand their memory out while a kernel of this
        stream still reads it.  Not while a graph is captured: nothing runs then, and keeping the
        prepared object for the replays is the caller's."""
        if torch.cuda.is_current_stream_capturing():
            return
        current = torch.cuda.current_stream(device)
        for t in arrays:
            t.record_stream(current)
        self.seen.add(stream)


def _check_tensor(t, name, dtype=None, device=None, heads=None, dim=None):
    if not torch.is_tensor(t):
        raise TypeError(f"{name} must be a tensor")
    if t.ndim != 3:
        raise ValueError(f"{name} must be a 3D tensor [tokens, heads, dim]")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in SUPPORTED_ATTENTION_DTYPES:
        raise TypeError(f"{name} dtype must be torch.bfloat16 or torch.float16")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} dtype must be {dtype}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if heads is not None and t.shape[1] != heads:
        raise ValueError(f"{name} must have {heads} heads, got {t.shape[1]}")
    if dim is not None and t.shape[2] != dim:
        raise ValueError(f"{name} must have dim {dim}, got {t.shape[2]}")
    if t.shape[0] > _TOKENS_CAP:
        raise ValueError(f"{name} must have at most 2^31 - 1024 tokens")


def _check_dim(dim):
    if dim < 8 or dim % 8 or dim > _DIM_CAP:
        raise NotImplementedError(
            f"dim {dim} has no gfx950 kernel in flagsparse_amd (multiples of 8 up to {_DIM_CAP})")


def _check_heads(heads, kv_heads):
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a multiple of key heads ({kv_heads})")


def _steps(t):
    """The steps of all axes but the last, as the kernels are given them: that of an axis of one element
    says nothing (contiguous() keeps it, whatever it is), so a row's takes its place."""
    return [s if n > 1 else t.shape[-1] for n, s in zip(t.shape[:-1], t.stride())]


def _rows(t):
    """``t`` itself where the kernels can read it (contiguous last axis, 16-byte rows, tokens that do
    not overlap and lie within 2^23 elements of each other), else a copy."""
    s = _steps(t)
    if t.stride(2) == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and t.data_ptr() % 16 == 0 and \
            t.shape[2] <= s[0] <= _STEP_CAP:
        return t
    return _aligned(t.contiguous())


def _scale_of(scale, dim):
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _FLOAT_MAX:
        raise ValueError("scale must be finite in float32")
    return scale


def _window_of(window):
    if window is None:
        return 0
    window = int(window)
    if window < 1:
        raise ValueError("window must be a positive number of tokens, or None")
    return min(window, _TOKENS_CAP)


def _sight_of(window, sinks, most):
    """(window, sinks) in numbers; (0, 0) where together they show all of ``most`` tokens."""
    window = _window_of(window)
    sinks = _sinks_of(sinks, window)
    return (0, 0) if sinks and window + sinks >= most else (window, sinks)


def _sinks_of(sinks, window):
    sinks = 0 if sinks is None else int(sinks)
    if sinks < 0:
        raise ValueError("sinks must be a number of tokens, 0 or more")
    if sinks and not window:
        raise ValueError("sinks need a window")
    return min(sinks, _TOKENS_CAP)


def _check_out(out, name, shape, dtype, device):
    if not torch.is_tensor(out) or tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} must be a tensor of shape {tuple(shape)}")
    if not out.is_cuda or out.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on {device}")
    if out.dtype != dtype:
        raise TypeError(f"{name} dtype must be {dtype}")


def _overlap(a, b):
    """Whether the arrays may share memory; slices side by side in the rows of one array do not."""
    if not a.numel() or not b.numel():
        return False
    size = a.element_size()
    row_a, row_b = (1 + sum((n - 1) * s for n, s in zip(t.shape[1:], t.stride()[1:])) for t in (a, b))
    step, gap = a.stride(0), b.data_ptr() - a.data_ptr()
    if gap >= size * (row_a + (a.shape[0] - 1) * step) or \
            -gap >= size * (row_b + (b.shape[0] - 1) * b.stride(0)):
        return False
    if step > 0 and step == b.stride(0):
        at = gap // size % step  # of b's rows in a's
        return at < row_a or at + row_b > step
    return True


def _result(out, name, shape, dtype, device, *inputs):
    """(the array the kernel writes, whether ``out`` is to be copied from it): a kernel reads its inputs
    while it writes, so it never writes over them."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device), False
    _check_out(out, name, shape, dtype, device)
    s = _steps(out)
    if out.stride(2) == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and out.data_ptr() % 16 == 0 and \
            all(s) and \
            not any(_overlap(out, t) for t in inputs):
        return out, False
    return torch.empty(shape, dtype=dtype, device=device), True


def _int32(t, name, length, device, least=-1):
    """A contiguous int32 device array of ``length``; what is less than ``least`` in 64 bits becomes it."""
    if not torch.is_tensor(t) or t.ndim != 1 or t.numel() != length:
        raise ValueError(f"{name} must be a 1D tensor of length {length}")
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on {device}")
    if t.dtype not in SUPPORTED_INDEX_DTYPES:
        raise TypeError(f"{name} dtype must be torch.int32 or torch.int64")
    if t.dtype == torch.int64:
        t = t.clamp(least, 2**31 - 1).to(torch.int32)
    return t.contiguous()


def _layouts(*tensors):
    """What of the arrays decides whether and how a call is made, their addresses apart."""
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.device)
                  if isinstance(t, torch.Tensor) else () for t in tensors])


# ---- the paged cache ----


class PreparedPagedKV:
    """A paged cache and its page table, checked once.

    ``k_pages`` / ``v_pages`` are the caller's own arrays, read and written in place.  The page table
    is a copy: a table that changes (another batch, more pages) is prepared anew.  ``room`` is the
    most tokens that the pages of one sequence hold."""

    __slots__ = ("k_pages", "v_pages", "dtype", "device", "indptr", "indices", "batch", "n_pages",
                 "page_size", "kv_heads", "dim", "room", "_piece", "_pieces", "_first", "_most", "_streams",
                 "_calls", "_counts", "_held", "_lists", "_sizes")

    def __init__(self, k_pages, v_pages, indptr, indices, pages):
        self.k_pages = k_pages
        self.v_pages = v_pages
        self.dtype = k_pages.dtype
        self.device = k_pages.device
        self.indptr = indptr
        self.indices = indices
        self.batch = indptr.numel() - 1
        self.n_pages, self.page_size, self.kv_heads, self.dim = (int(n) for n in k_pages.shape)
        rooms = pages * self.page_size
        self.room = int(rooms.max()) if len(rooms) else 0
        self._held = pages  # of each sequence, on the host
        self._lists, self._sizes = {}, {}  # pieces of other sizes, or under a window: see _list
        # the pieces that attention is cut into
        self._piece = int(_abi.lib().fsp_attention_paged_piece(int(rooms.sum()), self.kv_heads))
        self._pieces, self._first, self._most = _on_device(
            [(*_pieces(pages, self.page_size, self._piece), self._piece)], k_pages.device)[0]
        self._counts = _abi.Calls()  # the pieces' counts of arrivals, by stream and number
        self._streams = _Streams()
        self._calls = _abi.Calls()

    def _packed(self):
        k, v = self.k_pages, self.v_pages
        for t, name in ((k, "k_pages"), (v, "v_pages")):
            _check_pages(t, name)
            if t.dtype != self.dtype or t.device != self.device or \
                    t.shape != (self.n_pages, self.page_size, self.kv_heads, self.dim):
                raise ValueError(f"{name} are not what was prepared: prepare the cache anew")
        return _CACHE.pack(_CODES[k.dtype], self.kv_heads, self.dim, self.page_size, self.n_pages,
                           self.batch, self.indices.numel(), k.data_ptr(), *_steps(k), v.data_ptr(),
                           *_steps(v), self.indptr.data_ptr(), self.indices.data_ptr())

    def _on(self):
        """The current stream, on which the arrays are marked as used."""
        stream = _abi.raw_stream(self.device)
        if stream not in self._streams.seen:
            self._streams.mark(stream, self.device, (self.indptr, self.indices, self._pieces))
        return stream

    def _list(self, sight, slots, most, ways, way):
        """(tokens of a piece, pieces, first pieces, most of one sequence, streams that they are marked on):
        pieces of at most ``most`` tokens, of each sequence no more than ``sight`` tokens in a row can
        touch (0: all of its room), that go to ``way[0]`` workgroups of ``way[1]`` rows, of which ``slots`` run
        at a time.  The first call makes those of all ``ways`` that calls of its kind may go, and they are kept."""
        key = (sight, slots, most, ways)
        sizes = self._sizes.get(key)
        if sizes is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a call's first run with this window and these heads builds its work lists, "
                                   "which cannot be captured: make one such call before the capture")
            sizes = dict(zip(ways, _pieces_of(self._held * self.page_size, sight, ways, slots, most)))
            new = [piece for piece in sorted(set(sizes.values())) if (sight, piece) not in self._lists]
            tables = _on_device([(*_pieces(self._held, self.page_size, piece, sight), piece) for piece in new],
                                self.device)
            for piece, table in zip(new, tables):  # for good: captured graphs read it
                self._lists.setdefault((sight, piece), (piece, *table, _Streams()))
            torch.cuda.current_stream(self.device).synchronize()  # calls may come from other streams
            self._sizes[key] = sizes
        return self._lists[sight, sizes[way]]


@functools.lru_cache(maxsize=64)
def _tree_ways(kv_heads, group):
    """How the pieces of a tree call may be gone through, whatever its numbers of drafted tokens: (workgroups of a
    piece, rows of each)."""
    L = _abi.lib()
    tiles = {}
    for longest in range(1, int(L.fsp_attention_tree_drafts()) + 1):
        rows = int(L.fsp_attention_tree_rows(group, longest))
        tiles[rows] = max(tiles.get(rows, 1), -(-group * longest // rows))
    return tuple((kv_heads * n, rows) for rows, most in sorted(tiles.items())
                 for n in sorted({_near(n) for n in range(1, most + 1)}))


def _near(n):
    """A number of tiles or one close to it, by quarters of powers of two from 8 on.  By powers of two alone five tiles
    are sized as four: 4 sequences of 30000, 100 drafted tokens, 6 heads of 128 over 1 71 us, 58 so."""
    step = 1 << max(0, n.bit_length() - 3)
    return (n + step // 2) // step * step


def _piece_of(rooms, sight, each, slots, most, rows):
    """The size of a piece for one way: see _pieces_of."""
    return _pieces_of(rooms, sight, ((each, rows),), slots, most)[0]


def _pieces_of(rooms, sight, ways, slots, most):
    """For each of the ``ways``, (workgroups of a piece, rows of each), the tokens of a piece, from 256 to ``most``,
    by which the pieces of all sequences end soonest.  A workgroup takes as long as its tokens, and 100 + 2 * rows
    for what it does before and after them (its sums are written and read again); all of them take something
    between their sum over the ``slots`` and rounds of ``slots`` that wait for each other.  Mostly that gives whole
    rounds of even pieces: 8 sequences of 30064, 8 key heads, 256 rows beside each (16 workgroups a piece), pieces
    of 2048 / 3840 / 4096 / 5120 / 7552 (one round) / 10112 tokens 391 / 368 / 373 / 379 / 361 / 398 us; 96 ragged
    ones of up to 8000, 32 rows, of 256 / 512 / 1024 / 2048 / 4096 111 / 98 / 90 / 87 / 89 us, 128 rows 152 / 131 /
    116 / 112 / 142; 33 ragged ones under a window of 2047, 23 heads of 80, up to 26 tokens, of 128 / 256 / 512 /
    1024 35 / 28 / 32 / 40."""
    seen = np.minimum(rooms, sight) if sight else rooms
    longest, tokens = int(seen.max(initial=0)), int(seen.sum())
    best = [(float("inf"), 256)] * len(ways)
    n = max(1, -(-longest // most))
    while True:
        piece = max(256, -(-longest // n // 128) * 128)
        whole = seen // piece
        rest = seen - whole * piece
        rest = np.sort(rest[rest > 0])[::-1]
        wholes, rests, few = int(whole.sum()), len(rest), rest.tolist()
        for i, (each, rows) in enumerate(ways):
            around, count = 100 + 2 * rows, wholes * each
            starts = max(1, -(-(count + each * rests) // slots))  # rounds, and those that start with whole pieces
            full = min(starts, -(-count // slots)) if rests else starts
            first = piece if full else few[0]
            rounds = full * piece + starts * around
            if starts - full < 32:
                rounds += sum([few[(i * slots - count) // each] for i in range(full, starts)])
            else:
                rounds += int(rest[(np.arange(full, starts) * slots - count) // each].sum())
            total = each * (tokens + around * (wholes + rests))
            best[i] = min(best[i], (rounds + max(total / slots, float(first + around)), piece))
        if piece == 256:
            return [size for _, size in best]
        n += 1 + n // 8


def _on_device(lists, device):
    """Lists of _pieces and the tokens of a piece each, [(table, first pieces, most, piece)], on the device, in one
    array.  Long pieces first, for short ones to even out the end: 96 ragged sequences of up to 4096 tokens, 8
    heads of 128: 51 us, 55 in the sequences' order."""
    tables = [table[np.argsort(-np.minimum(piece, table[:, 4] - table[:, 1]), kind="stable")].ravel()
              for table, _, _, piece in lists]
    parts = tables + [first for _, first, _, _ in lists]
    if not parts:
        return []
    parts = torch.from_numpy(np.concatenate(parts)).to(device).split([len(part) for part in parts])
    return [(parts[i].view(-1, 8), parts[len(lists) + i], most) for i, (_, _, most, _) in enumerate(lists)]


def _pieces(pages, page_size, piece, sight=0):
    """(the pieces of ``piece`` tokens that sequences with so many pages may come to hold, the sequences'
    first ones, the most that one has), as the kernels read them; ``sight``: as many as so many tokens in a
    row can touch, counted from the first one that they do."""
    rooms = pages * page_size
    n = np.maximum(1, -(-rooms // piece))
    if sight:
        n = np.minimum(n, -(-sight // piece) + 1)
    slots = np.cumsum(n) - n
    seq = np.repeat(np.arange(len(rooms)), n)
    at = np.arange(len(seq)) - slots[seq]
    none = np.zeros_like(seq)
    table = np.stack([seq, at * piece, slots[seq], (np.cumsum(pages) - pages)[seq], rooms[seq],
                      none, none, none], axis=1)
    return table.astype(np.int32), slots.astype(np.int32), int(n.max(initial=1))


def _check_pages(t, name):
    if not torch.is_tensor(t):
        raise TypeError(f"{name} must be a tensor")
    if t.ndim != 4:
        raise ValueError(f"{name} must be a 4D tensor [pages, page_size, heads, dim]")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in SUPPORTED_ATTENTION_DTYPES:
        raise TypeError(f"{name} dtype must be torch.bfloat16 or torch.float16")
    if t.numel() and (t.stride(3) != 1 or t.data_ptr() % 16 or
                      any(s % 8 for n, s in zip(t.shape[:3], t.stride()) if n > 1)):
        raise ValueError(f"{name} must have a contiguous last axis and 16-byte aligned rows")


def prepare_paged_kv(k_pages, v_pages, indptr, indices):
    """Check a paged cache and its page table.

    ``k_pages``, ``v_pages``: [pages, page_size, kv_heads, dim], any order of the first three axes
    in memory.  Sequence b's tokens lie in pages ``indices[indptr[b]:indptr[b + 1]]``, in order; a
    sequence may own more pages than it fills yet, and sequences may share pages that they only
    read.  Returns a PreparedPagedKV for flagsparse_paged_append and flagsparse_attention_paged."""
    _check_pages(k_pages, "k_pages")
    _check_pages(v_pages, "v_pages")
    if k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must have the same shape")
    if k_pages.dtype != v_pages.dtype:
        raise TypeError("v_pages dtype must match k_pages dtype")
    if k_pages.device != v_pages.device:
        raise ValueError("k_pages and v_pages must be on the same CUDA device")
    n_pages, page_size, kv_heads, dim = k_pages.shape
    _check_dim(dim)
    if page_size < 1 or kv_heads < 1:
        raise ValueError("pages must hold at least one token and one head")
    if n_pages * page_size > 2**31 - 1:
        raise ValueError("the cache must hold fewer than 2^31 tokens")
    for t, name in ((indptr, "indptr"), (indices, "indices")):
        if not torch.is_tensor(t) or t.ndim != 1:
            raise ValueError(f"{name} must be a 1D tensor")
        if not t.is_cuda or t.device != k_pages.device:
            raise ValueError(f"{name} must be a CUDA tensor on {k_pages.device}")
        if t.dtype not in SUPPORTED_INDEX_DTYPES:
            raise TypeError(f"{name} dtype must be torch.int32 or torch.int64")
    if indptr.numel() < 1:
        raise ValueError("indptr must have at least one entry")
    if indices.numel() * page_size > _TOKENS_CAP:
        raise ValueError("the page table must hold at most 2^31 - 1024 tokens")
    (first, last, decreases, _, least, most), idx, ptr = csr_check(
        indices.contiguous(), indptr.contiguous(), 32)
    if first != 0:
        raise ValueError("indptr[0] must be 0")
    if last != indices.numel():
        raise ValueError(f"indptr[-1] must equal the number of indices {indices.numel()}")
    if decreases:
        raise ValueError("indptr must be nondecreasing")
    if indices.numel() and (least < 0 or most >= n_pages):
        raise IndexError("indices out of range for the cache's pages")
    # the prepared object's own: what the checks said of them stays true
    if idx.data_ptr() == indices.data_ptr():
        idx = idx.clone()
    if ptr.data_ptr() == indptr.data_ptr():
        ptr = ptr.clone()
    pages = np.diff(ptr.cpu().numpy().astype(np.int64))
    prepared = PreparedPagedKV(k_pages, v_pages, ptr, idx, pages)
    torch.cuda.current_stream(k_pages.device).synchronize()  # calls may come from other streams
    return prepared


def _paged_of(prepared, k_pages, v_pages, indptr, indices, lengths):
    """The prepared cache of a call; one that is made for the call has its lengths checked too."""
    if prepared is not None:
        if not isinstance(prepared, PreparedPagedKV):
            raise TypeError("prepared must be a PreparedPagedKV instance")
        return prepared, _int32(lengths, "lengths", prepared.batch, prepared.device)
    if any(t is None for t in (k_pages, v_pages, indptr, indices)):
        raise ValueError("k_pages, v_pages, indptr and indices are required when prepared is not "
                         "provided")
    kv = prepare_paged_kv(k_pages, v_pages, indptr, indices)
    n = _int32(lengths, "lengths", kv.batch, kv.device)
    if kv.batch:
        room = (kv.indptr[1:] - kv.indptr[:-1]) * kv.page_size
        if bool(((n < 0) | (n > room)).any()):
            raise ValueError("lengths must lie between 0 and what the sequences' pages hold")
    return kv, n


def flagsparse_paged_append(k, v, lengths, token_indptr=None, *, prepared=None, k_pages=None,
                            v_pages=None, indptr=None, indices=None, q=None, cos=None, sin=None,
                            interleaved=False, parents=None, text_lengths=None, out=None):
    """Write new keys and values into a paged cache, rotated by their positions on the way.

    ``k``, ``v``: [tokens, kv_heads, dim], the new tokens of each sequence one after the other:
    sequence b's are ``token_indptr[b]`` to ``token_indptr[b + 1]`` (None: one token per sequence).
    ``lengths[b]`` is what sequence b holds with them, so its last token has position
    ``lengths[b] - 1``.  ``cos``, ``sin``: float32 [positions, half]; the first 2 * half elements of
    every head of ``k`` and ``q`` are rotated by pairs, (a, b) -> (a cos - b sin, a sin + b cos):
    elements half apart, or neighbours with ``interleaved``.  Without them nothing is rotated.
    ``parents``: the new tokens are drafted ones, at most 256 a sequence, that form trees
    (flagsparse_attention_paged_tree): each is stored in its turn, but rotated by the position of its sequence's
    first new token plus the tokens before it on its way up the tree.
    ``text_lengths``: what the sequences' texts count with the new tokens, where that is more than the cache holds of
    them because some were given up (flagsparse_paged_keep leaves the others rotated as they are): new tokens are
    stored behind what is left, by ``lengths``, and rotated by their positions in the texts.

    Returns the rotated ``q`` [tokens, heads, dim] (written to ``out`` where given, which may be ``q``),
    or None without ``q``.  The pages that new tokens go to belong to one sequence each, and ``k``,
    ``v`` and ``q`` lie outside the cache.  With
    ``prepared`` nothing is waited for, so lengths are not checked: a token whose position is
    negative or past its sequence's pages, or whose parents do not come earlier, is not stored and its row of
    ``q`` comes back as NaN."""
    key = None
    if out is None and type(prepared) is PreparedPagedKV:
        key = _layouts(k, v, q, cos, sin, lengths, token_indptr, parents, text_lengths) + (
            bool(interleaved), prepared.k_pages.data_ptr(), prepared.v_pages.data_ptr())
        kept = prepared._calls.get(key)
        if kept is not None and not (k.data_ptr() | v.data_ptr()) % 16 and (
                q is None or q.data_ptr() % 16 == 0):
            head, like = kept
            res = None if q is None else torch.empty_like(like, memory_format=_CONTIGUOUS)
            _append(prepared, head, k, v, q, res, cos, sin, token_indptr, lengths, parents, text_lengths)
            return res
    kv, n = _paged_of(prepared, k_pages, v_pages, indptr, indices, lengths)
    dev, dt = kv.device, kv.dtype
    _check_tensor(k, "k", dt, dev, kv.kv_heads, kv.dim)
    _check_tensor(v, "v", dt, dev, kv.kv_heads, kv.dim)
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        raise ValueError(f"v must have {tokens} tokens, got {v.shape[0]}")
    given = (k, v, q, cos, sin, lengths, token_indptr, parents, text_lengths)
    if token_indptr is None:
        if tokens != kv.batch:
            raise ValueError(f"k must have one token for each of {kv.batch} sequences, got "
                             f"{tokens}; other numbers need token_indptr")
    else:
        token_indptr = _int32(token_indptr, "token_indptr", kv.batch + 1, dev)
    if parents is not None:
        parents = _int32(parents, "parents", tokens, dev, -2)
        if prepared is None:
            _check_drafts(kv, n, token_indptr, parents, tokens, 1 if token_indptr is None else
                          int(_abi.lib().fsp_attention_tree_drafts()))
    if text_lengths is not None:
        text_lengths = _int32(text_lengths, "text_lengths", kv.batch, dev)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    half = rows = 0
    if cos is not None:
        for t, name in ((cos, "cos"), (sin, "sin")):
            if not torch.is_tensor(t) or t.ndim != 2:
                raise ValueError(f"{name} must be a 2D tensor [positions, half]")
            if not t.is_cuda or t.device != dev:
                raise ValueError(f"{name} must be a CUDA tensor on {dev}")
            if t.dtype != torch.float32:
                raise TypeError(f"{name} dtype must be torch.float32")
        if cos.shape != sin.shape:
            raise ValueError("cos and sin must have the same shape")
        rows, half = (int(x) for x in cos.shape)
        if 2 * half > kv.dim:
            raise ValueError(f"cos and sin must have at most dim / 2 = {kv.dim // 2} columns")
        cos, sin = cos.contiguous(), sin.contiguous()
    heads, res, copied = 0, None, False
    if q is not None:
        _check_tensor(q, "q", dt, dev, None, kv.dim)
        if q.shape[0] != tokens:
            raise ValueError(f"q must have {tokens} tokens, got {q.shape[0]}")
        heads = q.shape[1]
        res, copied = _result(out, "out", q.shape, dt, dev, q, k, v)
        q = _rows(q)
    elif out is not None:
        raise ValueError("out is for the rotated q")
    if tokens and kv.batch:
        k, v = _rows(k), _rows(v)
        steps = (*_steps(q), *_steps(res)) if heads else (0, 0, 0, 0)
        head = kv._packed() + _APPEND.pack(tokens, heads, half, rows, bool(interleaved),
                                           *_steps(k), *_steps(v), *steps)
        _append(kv, head, k, v, q, res, cos, sin, token_indptr, n, parents, text_lengths)
        if key is not None and all(x is y for x, y in zip(
                (k, v, q, cos, sin, n, token_indptr, parents, text_lengths), given)):
            _keep(kv._calls, key, (head, None if q is None else _like(q.shape, dt, dev)))
    elif res is not None:  # tokens of no sequence
        res.fill_(float("nan"))
    if copied:
        out.copy_(res)
        res = out
    return res


def _at(t):
    return 0 if t is None else t.data_ptr()


def _append(kv, head, k, v, q, res, cos, sin, token_indptr, lengths, parents, text_lengths):
    args = head + _APPEND_AT.pack(k.data_ptr(), v.data_ptr(), _at(q), _at(res), _at(cos), _at(sin),
                                  _at(token_indptr), lengths.data_ptr())
    if text_lengths is not None:
        status = _abi.lib_on(kv.device).fsp_paged_append_at(args, _at(parents), text_lengths.data_ptr(), kv._on())
    elif parents is None:
        status = _abi.lib_on(kv.device).fsp_paged_append(args, kv._on())
    else:
        status = _abi.lib_on(kv.device).fsp_paged_append_drafts(args, parents.data_ptr(), kv._on())
    if status:
        _abi.check(status, "fsp_paged_append")


def flagsparse_paged_keep(keep, lengths, token_indptr=None, *, prepared=None, k_pages=None, v_pages=None,
                          indptr=None, indices=None, into=None):
    """Keep some of the last tokens of each sequence of a paged cache: drafted tokens that were accepted,
    or what is left of a text.

    ``keep``: [tokens], bool, the marks of the last tokens of each sequence one after the other: sequence
    b's are ``token_indptr[b]`` to ``token_indptr[b + 1]`` (None: as many for each), as many as it may have;
    ``lengths[b]`` is what sequence b holds.  The marked ones stay, in their order, and close up behind the
    tokens before them: in place, where the pages they move in belong to one sequence each (a chain of steps, made for
    drafted tokens: of a long text ``into`` takes a small part of the time), or in the pages of ``into``, another
    PreparedPagedKV with as many sequences, heads and dims, to which the tokens before them are copied too (pages
    that the call does not read; several may lie in the same arrays).  Keys stay rotated as they are: after a text
    whose tokens were given up go others by flagsparse_paged_append with ``text_lengths``.  A window of the
    attention, and its first tokens, go by places in the cache.

    Returns the new lengths, int32.  With ``prepared`` nothing is waited for, so lengths are not checked: where
    one is more than its pages hold or less than its marked tokens, or ``into`` has no room for
    what stays, nothing is moved and the new length is -1."""
    key = None
    if into is not None and not isinstance(into, PreparedPagedKV):
        raise TypeError("into must be a PreparedPagedKV instance")
    if into is not None and into is prepared:
        raise ValueError("into must be another table; in place needs none")
    if type(prepared) is PreparedPagedKV:
        key = _layouts(keep, lengths, token_indptr) + (
            "keep", prepared.k_pages.data_ptr(), prepared.v_pages.data_ptr())
        kept = prepared._calls.get(key)
        if kept is not None:
            return _keep_tokens(prepared, into, kept, keep, token_indptr, lengths)
    kv, n = _paged_of(prepared, k_pages, v_pages, indptr, indices, lengths)
    dev = kv.device
    if not torch.is_tensor(keep) or keep.ndim != 1:
        raise ValueError("keep must be a 1D tensor [tokens]")
    if not keep.is_cuda or keep.device != dev:
        raise ValueError(f"keep must be a CUDA tensor on {dev}")
    if keep.dtype != torch.bool:
        raise TypeError("keep dtype must be torch.bool")
    tokens = keep.numel()
    if tokens > _TOKENS_CAP:
        raise ValueError("keep must have at most 2^31 - 1024 tokens")
    given = (keep, n, token_indptr)
    each = 0
    if token_indptr is None:
        each = tokens // max(kv.batch, 1)
        if each * kv.batch != tokens:
            raise ValueError(f"keep must have as many tokens for each of {kv.batch} sequences, got "
                             f"{tokens}; other numbers need token_indptr")
    else:
        token_indptr = _int32(token_indptr, "token_indptr", kv.batch + 1, dev)
    if prepared is None:
        _check_drafts(kv, n, token_indptr, None, tokens, each if token_indptr is None else tokens)
    keep = keep.contiguous()
    head, sizes = kv._packed(), (tokens, each, kv._pieces.shape[0], kv._piece)
    counts = None  # of the pieces and the sequences
    if min(tokens, kv.room) > _COUNTED_FROM:
        counts = _like((kv._pieces.shape[0] + kv.batch,), torch.int32, dev)
    kept = (head, sizes, head + head + _KEEP.pack(0, *sizes), _like((kv.batch,), torch.int32, dev), counts)
    res = _keep_tokens(kv, into, kept, keep, token_indptr, n)
    if key is not None and all(x is y for x, y in zip((keep, lengths, token_indptr), given)):
        _keep(kv._calls, key, kept)
    return res


def _keep_tokens(kv, into, kept, keep, token_indptr, lengths):
    """The launch; returns the new lengths.  What ``into`` holds is looked up by every call: it is an
    argument, not a part of the prepared cache."""
    head, sizes, args, like, counts = kept
    stream = kv._on()
    if into is not None:
        if into.device != kv.device or into.dtype != kv.dtype:
            raise ValueError("into must be of the cache's type and on its device")
        if (into.batch, into.kv_heads, into.dim) != (kv.batch, kv.kv_heads, kv.dim):
            raise ValueError("into must have the cache's number of sequences, heads and dim")
        args = head + into._packed() + _KEEP.pack(1, *sizes)
        into._on()
    res = torch.empty_like(like, memory_format=_CONTIGUOUS)
    args += _KEEP_AT.pack(kv._pieces.data_ptr(), keep.data_ptr(), _at(token_indptr), lengths.data_ptr(),
                          res.data_ptr())
    if into is None or counts is None:
        status = _abi.lib_on(kv.device).fsp_paged_keep(args, stream)
    else:
        work = torch.empty_like(counts, memory_format=_CONTIGUOUS)
        status = _abi.lib_on(kv.device).fsp_paged_keep_counted(args, kv._first.data_ptr(), work.data_ptr(), stream)
    if status:
        _abi.check(status, "fsp_paged_keep")
    return res


def flagsparse_paged_copy(sources, targets, *, prepared=None, k_pages=None, v_pages=None):
    """Copy pages of a paged cache, keys and values: page ``sources[i]`` to page ``targets[i]``.

    A sequence that branches shares the pages that both only read by its page table, and has its last one
    copied.  ``sources``, ``targets``: [n], int32 or int64, numbers of the cache's pages; no page is the target
    of two, and none that is a target is another's source.  The cache is given by ``prepared``, for which any
    table of these pages does (it is not read, so that one prepared cache serves all branches), or by its pages;
    with ``prepared`` nothing is waited for, so numbers are not checked: a pair with one outside the cache copies
    nothing."""
    key = None
    if prepared is not None:
        if not isinstance(prepared, PreparedPagedKV):
            raise TypeError("prepared must be a PreparedPagedKV instance")
        kv = prepared
        key = _layouts(sources, targets) + ("copy", kv.k_pages.data_ptr(), kv.v_pages.data_ptr())
        kept = kv._calls.get(key)
        if kept is not None:
            _copy_pages(kv, kept, sources, targets)
            return
    else:
        if k_pages is None or v_pages is None:
            raise ValueError("k_pages and v_pages are required when prepared is not provided")
        none = torch.zeros(1, dtype=torch.int32, device=k_pages.device if torch.is_tensor(k_pages) else None)
        kv = prepare_paged_kv(k_pages, v_pages, none, none[:0])
    for t, name in ((sources, "sources"), (targets, "targets")):
        if not torch.is_tensor(t) or t.ndim != 1:
            raise ValueError(f"{name} must be a 1D tensor")
    n, given = sources.numel(), (sources, targets)
    sources = _int32(sources, "sources", n, kv.device)
    targets = _int32(targets, "targets", n, kv.device)
    if prepared is None and n:
        for t, name in ((sources, "sources"), (targets, "targets")):
            if int(t.min()) < 0 or int(t.max()) >= kv.n_pages:
                raise IndexError(f"{name} out of range for the cache's pages")
        if torch.unique(targets).numel() != n:
            raise ValueError("targets must be different pages")
        if bool((torch.isin(sources, targets) & (sources != targets)).any()):
            raise ValueError("a page cannot be a target and another one's source")
    kept = kv._packed(), n
    _copy_pages(kv, kept, sources, targets)
    if key is not None and sources is given[0] and targets is given[1]:
        _keep(kv._calls, key, kept)


def _copy_pages(kv, kept, sources, targets):
    status = _abi.lib_on(kv.device).fsp_paged_copy(kept[0], sources.data_ptr(), targets.data_ptr(), kept[1],
                                       _abi.raw_stream(kv.device))
    if status:
        _abi.check(status, "fsp_paged_copy")


def flagsparse_attention_paged(q, lengths, *, prepared=None, k_pages=None, v_pages=None,
                               indptr=None, indices=None, scale=None, window=None, sinks=0,
                               out=None, return_lse=False):
    """Attention of one query per sequence over what a paged cache holds of it.

    ``q``: [sequences, heads, dim]; ``lengths[b]``: the tokens that sequence b holds, the query's
    own among them (0: the sequence is empty, and its output is zeros).  ``window``: only the last
    ``window`` tokens are seen, and with ``sinks`` the first ``sinks`` too (the first call with such a window
    and as many heads builds a work list and cannot be captured).  ``scale``: dim ** -0.5 by default.  Returns
    [sequences, heads, dim], with the float32 log-sum-exp [sequences, heads] if ``return_lse``; neither is
    differentiable, nor is what flagsparse_paged_append gives.  With ``prepared`` nothing is waited for, so lengths
    are not checked: one that its sequence's pages cannot hold gives NaN."""
    key = None
    if out is None and type(prepared) is PreparedPagedKV and type(scale) in _PLAIN and \
            type(window) in _PLAIN and type(sinks) in _PLAIN:
        key = _layouts(q, lengths) + (scale, window, sinks, prepared.k_pages.data_ptr(),
                                      prepared.v_pages.data_ptr())
        kept = prepared._calls.get(key)
        if kept is not None and q.data_ptr() % 16 == 0:
            res = torch.empty_like(kept[1], memory_format=_CONTIGUOUS)
            lse = _attend(prepared, kept, q, res, lengths, return_lse)
            return (res, lse) if return_lse else res
    kv, n = _paged_of(prepared, k_pages, v_pages, indptr, indices, lengths)
    dev, dt = kv.device, kv.dtype
    _check_tensor(q, "q", dt, dev, None, kv.dim)
    if q.shape[0] != kv.batch:
        raise ValueError(f"q must have one token for each of {kv.batch} sequences, got "
                         f"{q.shape[0]}")
    heads = q.shape[1]
    _check_heads(heads, kv.kv_heads)
    factor, (past, first) = _scale_of(scale, kv.dim), _sight_of(window, sinks, kv.room)
    res, copied = _result(out, "out", q.shape, dt, dev, q, kv.k_pages, kv.v_pages)
    rows = _rows(q)
    # what such calls share: the arguments, patterns of their arrays, the counts of arrivals they need
    table, firsts, piece, most, marked = kv._pieces, kv._first, kv._piece, kv._most, None
    if first:
        tiles = -(-heads // kv.kv_heads // 16)
        way = (kv.kv_heads * tiles, 16)
        piece, table, firsts, most, marked = kv._list(min(past + first, _TOKENS_CAP), 768, 1024, (way,), way)
    pieces, need, room = table.shape[0], 0, None
    if pieces > kv.batch:
        need = int(_abi.lib().fsp_attention_paged_counts(pieces, most, kv.batch, heads, kv.kv_heads))
        room = _like((pieces * heads * (kv.dim + 2),), torch.float32, dev)
    kept = (kv._packed() + _PAGED.pack(
        table.data_ptr(), firsts.data_ptr(), pieces, piece, heads, past, factor,
        *_steps(rows), *_steps(res)), _like(q.shape, dt, dev),
        _like((kv.batch, heads), torch.float32, dev), room, need, first, (table, firsts), marked)
    lse = _attend(kv, kept, rows, res, n, return_lse)
    if key is not None and rows is q and n is lengths:
        _keep(kv._calls, key, kept)
    if copied:
        out.copy_(res)
        res = out
    return (res, lse) if return_lse else res


def _arrivals(kv, stream, need):
    """The counts that the pieces' arrivals are kept in, zeros between calls: one array a stream, whose
    calls follow each other.  A graph has its own, zeroed in each replay: it may run beside this
    stream's calls and beside other graphs that were captured here."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(need, dtype=torch.int32, device=kv.device)
    counts = kv._counts.get((stream, need))
    if counts is None:
        counts = kv._counts[stream, need] = torch.zeros(need, dtype=torch.int32, device=kv.device)
    return counts


def _attend(kv, kept, q, res, lengths, return_lse):
    """The launch; returns the log-sum-exp, if asked for."""
    head, _, like_lse, room, need, sinks, lists, marked = kept
    lse = torch.empty_like(like_lse, memory_format=_CONTIGUOUS) if return_lse else None
    if not kv.batch:
        return lse
    stream, work, counts = kv._on(), None, None
    if marked is not None and stream not in marked.seen:
        marked.mark(stream, kv.device, lists)
    if room is not None:
        work = torch.empty_like(room, memory_format=_CONTIGUOUS)
        if need:
            counts = _arrivals(kv, stream, need)
    args = head + _PAGED_AT.pack(q.data_ptr(), res.data_ptr(), _at(lse), lengths.data_ptr(),
                                 _at(work), _at(counts))
    if sinks:
        status = _abi.lib_on(kv.device).fsp_attention_paged_sinks(args, sinks, stream)
    else:
        status = _abi.lib_on(kv.device).fsp_attention_paged(args, stream)
    if status:
        _abi.check(status, "fsp_attention_paged")
    return lse


def flagsparse_attention_paged_tree(q, lengths, token_indptr=None, *, parents=None, longest=None,
                                    prepared=None, k_pages=None, v_pages=None, indptr=None,
                                    indices=None, scale=None, window=None, sinks=0, out=None,
                                    return_lse=False):
    """Attention of trees of drafted tokens over a paged cache that holds them, after the text that they
    go on from (flagsparse_paged_append).

    ``q``: [tokens, heads, dim], the drafted tokens of each sequence one after the other: sequence b's are
    ``token_indptr[b]`` to ``token_indptr[b + 1]`` (None: as many for each); ``lengths[b]`` is what
    sequence b holds with them.  ``parents``: [tokens], for each the place, among its sequence's
    drafted tokens, of the token before it, which comes earlier, or -1 where that is the text's last one
    (None: each follows the one before it).  A token sees the text, the drafted tokens on its way up
    the tree, and itself.  ``window`` and ``sinks`` go by positions, as in flagsparse_attention_paged: a
    drafted token's is the text's length plus the tokens before it on its way.  ``longest``: no
    sequence has more drafted tokens, at most 256 (by default 256; a smaller one saves work: each sequence has
    workgroups for so many).  Sums of long texts' pieces take tokens * heads * (dim + 2) * 4 bytes for every 256 to
    8192 tokens that the pages of one sequence hold, or less.

    Returns [tokens, heads, dim], with the float32 log-sum-exp [tokens, heads] if ``return_lse``; neither is
    differentiable.  With ``prepared`` nothing is waited for, so indices are not checked: rows of a
    sequence with more drafted tokens than ``longest``, or a length that its pages cannot hold or less than
    its drafted tokens, rows whose parents do not come earlier, and rows of no sequence are NaN.  What
    is not finite in a value that a row does not see, but another row of its sequence does, may reach it (a drafted
    token's off its way, or a token's of the text that only the windows of rows less deep hold: its weight is zero,
    and zero times it is NaN); in a key it does not.  The first call with its window, sinks and number
    of heads builds work lists and cannot be captured; others, whatever their numbers of tokens, use them."""
    key = None
    if out is None and type(prepared) is PreparedPagedKV and type(scale) in _PLAIN and \
            type(window) in _PLAIN and type(sinks) in _PLAIN and type(longest) in _PLAIN:
        key = _layouts(q, lengths, token_indptr, parents) + (
            "tree", scale, window, sinks, longest, prepared.k_pages.data_ptr(),
            prepared.v_pages.data_ptr())
        kept = prepared._calls.get(key)
        if kept is not None and q.data_ptr() % 16 == 0:
            res = torch.empty_like(kept[1], memory_format=_CONTIGUOUS)
            lse = _attend_tree(prepared, kept, q, res, lengths, token_indptr, parents, return_lse)
            return (res, lse) if return_lse else res
    kv, n = _paged_of(prepared, k_pages, v_pages, indptr, indices, lengths)
    dev, dt = kv.device, kv.dtype
    _check_tensor(q, "q", dt, dev, None, kv.dim)
    tokens, heads = q.shape[:2]
    _check_heads(heads, kv.kv_heads)
    given = (q, lengths, token_indptr, parents)
    most = int(_abi.lib().fsp_attention_tree_drafts())
    longest = most if longest is None else int(longest)
    if longest < 0 or longest > most:
        raise ValueError(f"longest must lie between 0 and {most}")
    if token_indptr is None:
        each = tokens // max(kv.batch, 1)
        if each * kv.batch != tokens:
            raise ValueError(f"q must have as many tokens for each of {kv.batch} sequences, got "
                             f"{tokens}; other numbers need token_indptr")
        if each > longest:
            raise ValueError(f"a sequence may have at most {longest} drafted tokens, got {each}")
        longest = each
    else:
        token_indptr = _int32(token_indptr, "token_indptr", kv.batch + 1, dev)
        longest = min(longest, tokens)
    if parents is not None:
        parents = _int32(parents, "parents", tokens, dev, -2)
    factor, (past, first) = _scale_of(scale, kv.dim), _sight_of(window, sinks, kv.room)
    res, copied = _result(out, "out", q.shape, dt, dev, q, kv.k_pages, kv.v_pages)
    rows = _rows(q)
    if prepared is None:
        _check_drafts(kv, n, token_indptr, parents, tokens, longest)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev) if return_lse else None
    if not kv.batch or not longest:  # tokens of no sequence, or none
        res.fill_(float("nan"))
        if return_lse:
            lse.fill_(float("nan"))
    else:
        # the same for all calls of a program, whatever numbers of tokens they have, and so are the lists
        sight = min(past + first + most, _TOKENS_CAP) if past else 0
        group = heads // kv.kv_heads
        of = int(_abi.lib().fsp_attention_tree_rows(group, longest))
        # tiles of an average sequence, as those of the longest trees are few
        tiles = min(-(-group * longest // of), 1 + group * tokens // (kv.batch * of))
        way = (kv.kv_heads * _near(tiles), of)
        piece, pieces, firsts, longest_list, marked = kv._list(
            sight, 512, 8192, (way,) if prepared is None else _tree_ways(kv.kv_heads, group), way)
        n_pieces, need, room, by_tokens = pieces.shape[0], 0, None, 0
        if n_pieces > kv.batch:
            need = int(_abi.lib().fsp_attention_tree_counts(n_pieces, longest_list, kv.batch, kv.kv_heads,
                                                            group, longest))
            size = int(_abi.lib().fsp_attention_tree_workspace(n_pieces, heads, kv.dim, longest))
            less = int(_abi.lib().fsp_attention_tree_by_tokens_workspace(longest_list, tokens, heads, kv.dim))
            if 2 * less < size:
                by_tokens, size = longest_list, less
            room = _like((size,), torch.uint8, dev)
        head = kv._packed() + _TREE.pack(
            pieces.data_ptr(), firsts.data_ptr(), n_pieces, piece, heads, past, factor, first, tokens,
            longest, *_steps(rows), *_steps(res))
        kept = (head, _like(q.shape, dt, dev), _like(q.shape[:2], torch.float32, dev), room, need,
                by_tokens, (pieces, firsts), marked)
        lse = _attend_tree(kv, kept, rows, res, n, token_indptr, parents, return_lse)
        if key is not None and all(x is y for x, y in zip((rows, n, token_indptr, parents), given)):
            _keep(kv._calls, key, kept)
    if copied:
        out.copy_(res)
        res = out
    return (res, lse) if return_lse else res


def _check_drafts(kv, lengths, token_indptr, parents, tokens, longest):
    """Of a call whose cache is not prepared: the host waits for it."""
    if token_indptr is None:
        count = torch.full((kv.batch,), longest, dtype=torch.int64, device=kv.device)
    else:
        p = token_indptr.to(torch.int64)
        count = p[1:] - p[:-1]
        if int(p[0]) != 0 or int(p[-1]) != tokens or bool((count < 0).any()):
            raise ValueError(f"token_indptr must lead from 0 to {tokens} without decreasing")
        if bool((count > longest).any()):
            raise ValueError(f"a sequence may have at most {longest} drafted tokens")
    if bool((count > lengths).any()):
        raise ValueError("lengths must count the drafted tokens")
    if parents is not None:
        place = torch.arange(tokens, device=kv.device) - torch.repeat_interleave(
            count.cumsum(0) - count, count)
        if bool(((parents < -1) | (parents >= place)).any()):
            raise ValueError("parents must come before their tokens, or be -1")


def _attend_tree(kv, kept, q, res, lengths, token_indptr, parents, return_lse):
    """The launch; returns the log-sum-exp, if asked for."""
    head, _, like_lse, room, need, by_tokens, lists, marked = kept
    lse = torch.empty_like(like_lse, memory_format=_CONTIGUOUS) if return_lse else None
    stream = kv._on()
    if stream not in marked.seen:
        marked.mark(stream, kv.device, lists)
    work = None if room is None else torch.empty_like(room, memory_format=_CONTIGUOUS)
    counts = _arrivals(kv, stream, need) if need else None
    args = head + _TREE_AT.pack(q.data_ptr(), res.data_ptr(), _at(lse), lengths.data_ptr(),
                                _at(token_indptr), _at(parents), _at(work), _at(counts))
    if by_tokens:
        status = _abi.lib_on(kv.device).fsp_attention_tree_by_tokens(args, by_tokens, stream)
    else:
        status = _abi.lib_on(kv.device).fsp_attention_tree(args, stream)
    if status:
        _abi.check(status, "fsp_attention_tree")
    return lse


# ---- packed sequences ----


class PreparedAttention:
    """The sequences of a packed batch, checked once, and the kernels' work lists over them: tiles of
    one sequence's rows, those with the most to do first, so that the last ones to finish are
    short."""

    __slots__ = ("batch", "q_tokens", "k_tokens", "device", "_longest", "_tiles", "_sequences", "_lengths",
                 "_grouped", "_streams", "_calls")

    def __init__(self, q_len, k_len, device):
        self.batch = len(q_len)
        self.q_tokens = int(q_len.sum())
        self.k_tokens = int(k_len.sum())
        self.device = device
        self._lengths = (q_len, k_len)
        self._grouped = {}  # lists of the queries' tiles under first keys, by the heads of a group
        self._longest = tuple(int(n.max(initial=0)) for n in (q_len, k_len))
        # (queries, queries in half tiles, keys, keys in half tiles; causal) -> the list
        names = [(which, causal) for which in range(4) for causal in (False, True)]
        lists = [_tiles(q_len, k_len, int(_abi.lib().fsp_attention_packed_tile(which)), causal,
                        which >= 2) for which, causal in names]
        sequences = np.zeros((self.batch, 8), dtype=np.int32)
        sequences[:, 3:7] = np.stack([np.cumsum(q_len) - q_len, q_len, np.cumsum(k_len) - k_len, k_len],
                                     axis=1)
        flat = torch.from_numpy(np.concatenate(lists + [sequences])).to(device)
        ends = np.cumsum([0] + [len(t) for t in lists])
        self._tiles = {name: flat[ends[i]:ends[i + 1]] for i, name in enumerate(names)}
        self._sequences = flat[ends[-1]:]
        self._streams = _Streams()
        self._calls = _abi.Calls()

    def _on(self):
        """The current stream, on which the work lists are marked as used."""
        stream = _abi.raw_stream(self.device)
        if stream not in self._streams.seen:
            self._streams.mark(stream, self.device, self._tiles.values())
        return stream

    def _query_tiles(self, sinks, group):
        """(tiles, half tiles, streams that they are marked on) of the queries; those under first keys depend on
        the heads of a group, and are made when first asked for and kept."""
        if not sinks:
            return self._tiles[0, True], self._tiles[1, True], self._streams
        kept = self._grouped.get(group)
        if kept is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first call with sinks builds its work list, which cannot be "
                                   "captured: make one such call before the capture")
            lists = [_tiles(*self._lengths, int(_abi.lib().fsp_attention_packed_sinks_tile(which, group)),
                            True, False) for which in (0, 1)]
            flat = torch.from_numpy(np.concatenate(lists)).to(self.device)
            torch.cuda.current_stream(self.device).synchronize()  # calls may come from other streams
            kept = (flat[:len(lists[0])], flat[len(lists[0]):], _Streams())
            kept = self._grouped.setdefault(group, kept)  # for good: captured graphs read them
        return kept


def _tiles(q_len, k_len, tile, causal, keys):
    """The tiles of ``tile`` query rows (or key rows) as the kernels read them, by falling work."""
    q_begin, k_begin = np.cumsum(q_len) - q_len, np.cumsum(k_len) - k_len
    length, begin = (k_len, k_begin) if keys else (q_len, q_begin)
    n = -(-length // tile)
    seq = np.repeat(np.arange(len(length)), n)
    at = (np.arange(len(seq)) - np.repeat(np.cumsum(n) - n, n)) * tile  # place in the sequence
    nq, nk = q_len[seq], k_len[seq]
    rows = np.minimum(tile, length[seq] - at)
    if not causal:
        work = nq if keys else nk
    elif keys:  # query i sees key j from i = j - nk + nq on
        work = np.clip(nq - np.clip(at - nk + nq, 0, None), 0, None)
    else:
        work = np.clip(at + rows + nk - nq, 0, nk)
    order = np.argsort(-work, kind="stable")
    table = np.stack([begin[seq] + at, rows, at, q_begin[seq], nq, k_begin[seq], nk,
                      np.zeros_like(at)], axis=1)
    return np.ascontiguousarray(table[order], dtype=np.int32)


def _host_lengths(indptr, name):
    if not torch.is_tensor(indptr) or indptr.ndim != 1 or indptr.numel() < 1:
        raise ValueError(f"{name} must be a 1D tensor with at least one entry")
    if not indptr.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if indptr.dtype not in SUPPORTED_INDEX_DTYPES:
        raise TypeError(f"{name} dtype must be torch.int32 or torch.int64")
    _capturing()
    p = indptr.cpu().numpy().astype(np.int64)
    if p[0] != 0:
        raise ValueError(f"{name}[0] must be 0")
    if (np.diff(p) < 0).any():
        raise ValueError(f"{name} must be nondecreasing")
    if p[-1] > _TOKENS_CAP:
        raise ValueError(f"{name} must count at most 2^31 - 1024 tokens")
    return np.diff(p)


def prepare_attention_packed(indptr, k_indptr=None):
    """Check the sequences of a packed batch: sequence b's queries are the tokens ``indptr[b]`` to
    ``indptr[b + 1]``, its keys ``k_indptr[b]`` to ``k_indptr[b + 1]`` (None: the same).  Returns a
    PreparedAttention for every call over these sequences: all layers, forward and backward."""
    q_len = _host_lengths(indptr, "indptr")
    k_len = q_len
    if k_indptr is not None:
        k_len = _host_lengths(k_indptr, "k_indptr")
        if len(k_len) != len(q_len):
            raise ValueError("indptr and k_indptr must have the same length")
        if k_indptr.device != indptr.device:
            raise ValueError("indptr and k_indptr must be on the same CUDA device")
    prepared = PreparedAttention(q_len, k_len, indptr.device)
    torch.cuda.current_stream(indptr.device).synchronize()  # calls may come from other streams
    return prepared


def _packed_inputs(q, k, v, indptr, k_indptr, prepared, causal, window, sinks):
    """(prepared, causal, window, sinks) of a call whose arrays are checked against each other; no window and
    sinks where together they show all keys."""
    _check_tensor(q, "q")
    _check_tensor(k, "k", q.dtype, q.device, None, q.shape[2])
    _check_tensor(v, "v", q.dtype, q.device, k.shape[1], q.shape[2])
    _check_heads(q.shape[1], k.shape[1])
    _check_dim(q.shape[2])
    if _window_of(window) and not causal:
        raise ValueError("window needs causal=True")
    _sinks_of(sinks, _window_of(window))
    if prepared is None:
        if indptr is None:
            raise ValueError("indptr is required when prepared is not provided")
        prepared = prepare_attention_packed(indptr, k_indptr)
    elif not isinstance(prepared, PreparedAttention):
        raise TypeError("prepared must be a PreparedAttention instance")
    if prepared.device != q.device:
        raise ValueError("q, k, v and the sequences must be on the same CUDA device")
    if q.shape[0] != prepared.q_tokens:
        raise ValueError(f"q must have {prepared.q_tokens} tokens, got {q.shape[0]}")
    if k.shape[0] != prepared.k_tokens or v.shape[0] != prepared.k_tokens:
        raise ValueError(f"k and v must have {prepared.k_tokens} tokens, got {k.shape[0]} and "
                         f"{v.shape[0]}")
    return prepared, bool(causal), *_sight_of(window, sinks, prepared._longest[1])


def _pack(prepared, q, k, v, causal, window, scale, out, grads=(), sinks=0):
    """A call's arguments up to the addresses; grads: grad_out, grad_q, grad_k, grad_v."""
    lists = [prepared._tiles[which, causal] for which in range(4)]
    if sinks:
        lists[:2] = prepared._query_tiles(sinks, q.shape[1] // k.shape[1])[:2]
    steps = [n for t in (q, k, v, out, *grads) for n in _steps(t)]
    steps += [0] * (16 - len(steps))
    return _PACKED.pack(_CODES[q.dtype], q.shape[1], k.shape[1], q.shape[2], q.shape[0],
                        k.shape[0], *prepared._longest, causal, window, scale,
                        *(n for i, t in enumerate(lists)
                          for n in (t.data_ptr(), t.shape[0] if i < 2 or grads else 0)), *steps)


def _tracked(t):
    return isinstance(t, torch.Tensor) and t.requires_grad


def _has_tangent(*tensors):
    """Whether one carries a tangent of forward-mode differentiation; no level open is the quick answer."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    return any(forward_ad.unpack_dual(t).tangent is not None for t in tensors
               if isinstance(t, torch.Tensor))


def _refuse_tangents(*tensors):
    if _has_tangent(*tensors):
        raise NotImplementedError("the gradient has no forward-mode derivative")


def _first_tiles(prepared, group):
    """Marks the lists of a call with sinks as used on the current stream."""
    *lists, marked = prepared._query_tiles(True, group)
    stream = _abi.raw_stream(prepared.device)
    if stream not in marked.seen:
        marked.mark(stream, prepared.device, lists)


def _run_forward(prepared, head, sinks, q, k, v, res, lse):
    if q.shape[0]:
        args = head + _PACKED_AT.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), res.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, 0)
        if sinks:
            _first_tiles(prepared, q.shape[1] // k.shape[1])
            status = _abi.lib_on(prepared.device).fsp_attention_packed_sinks(args, sinks, prepared._on())
        else:
            status = _abi.lib_on(prepared.device).fsp_attention_packed(args, prepared._on())
        if status:
            _abi.check(status, "fsp_attention_packed")


def _forward(prepared, q, k, v, causal, window, sinks, scale, out=None, key=None):
    res, copied = _result(out, "out", q.shape, q.dtype, q.device, q, k, v)
    rows = _rows(q), _rows(k), _rows(v)
    head = _pack(prepared, *rows, causal, window, scale, res, sinks=sinks)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    _run_forward(prepared, head, sinks, *rows, res, lse)
    if key is not None and rows[0] is q and rows[1] is k and rows[2] is v:
        _keep(prepared._calls, key, (head, sinks, _like(q.shape, q.dtype, q.device),
                                     _like(lse.shape, lse.dtype, lse.device)))
    if copied:
        out.copy_(res)
        res = out
    return res, lse


class _Differentiable(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, prepared, causal, window, sinks, scale):
        out, lse = _forward(prepared, q, k, v, causal, window, sinks, scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.rest = (prepared, causal, window, sinks, scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        q, k, v, out, lse = ctx.saved_tensors
        prepared, causal, window, sinks, scale = ctx.rest
        _refuse_tangents(grad, q, k, v)
        grads = _backward(prepared, grad, q, k, v, out, lse, causal, window, sinks, scale)
        return *grads, None, None, None, None, None


def flagsparse_attention_packed(q, k, v, indptr=None, k_indptr=None, *, prepared=None, causal=True,
                                window=None, sinks=0, scale=None, out=None, return_lse=False):
    """Attention over packed sequences.

    ``q``: [tokens, heads, dim]; ``k``, ``v``: [key tokens, kv_heads, dim]; the sequences are given
    by ``indptr`` / ``k_indptr`` (checked by this call, which waits for them) or by ``prepared``
    (prepare_attention_packed).  With ``causal`` query i of nq sees key j of nk if
    j <= i + nk - nq, the last query all of them; ``window``: only the last ``window`` of those, and with
    ``sinks`` the sequence's first ``sinks`` keys too (the first call with sinks that hide anything, and as many heads,
    builds a work list and cannot be captured).
    ``scale``: dim ** -0.5 by default.  Returns [tokens, heads, dim], with the float32 log-sum-exp
    [tokens, heads] if ``return_lse``.  The output is differentiable with respect to q, k and v where
    they require a gradient (the log-sum-exp is not); forward-mode tangents raise NotImplementedError.

    What is not finite in k reaches the rows that see it.  In v it reaches those, and may reach rows of
    the same sequence and block of 64 keys that do not (their weight is zero, and zero times it is
    NaN), as it does in a product of the weights' matrix; it never reaches another sequence."""
    key = None
    wanted = torch.is_grad_enabled() and (_tracked(q) or _tracked(k) or _tracked(v)) or \
        _has_tangent(q, k, v)  # which _Differentiable refuses
    if out is None and not wanted and type(prepared) is PreparedAttention and \
            type(scale) in _PLAIN and type(window) in _PLAIN and type(causal) in _PLAIN and \
            type(sinks) in _PLAIN:
        key = _layouts(q, k, v) + (causal, window, sinks, scale)
        kept = prepared._calls.get(key)
        if kept is not None and not (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
            head, first, like, like_lse = kept
            res = torch.empty_like(like, memory_format=_CONTIGUOUS)
            lse = torch.empty_like(like_lse, memory_format=_CONTIGUOUS)
            _run_forward(prepared, head, first, q, k, v, res, lse)
            return (res, lse) if return_lse else res
    prepared, causal, window, sinks = _packed_inputs(q, k, v, indptr, k_indptr, prepared, causal,
                                                     window, sinks)
    scale = _scale_of(scale, q.shape[2])
    if wanted:
        if out is not None:
            raise RuntimeError("out cannot be given where q, k or v require a gradient")
        res, lse = _Differentiable.apply(q, k, v, prepared, causal, window, sinks, scale)
    else:
        res, lse = _forward(prepared, q, k, v, causal, window, sinks, scale, out, key)
    return (res, lse) if return_lse else res


def _backward(prepared, grad_out, q, k, v, out, lse, causal, window, sinks, scale, key=None):
    rows = tuple(_rows(t) for t in (grad_out, q, k, v, out))
    flat = lse.contiguous()
    grads = tuple(torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v))
    head = _pack(prepared, *rows[1:4], causal, window, scale, rows[4], (rows[0], *grads), sinks)
    sizes = (prepared._tiles[2, causal].shape[0], q.shape[1], k.shape[1], q.shape[2], q.shape[0],
             k.shape[0])
    q_longest, k_longest = prepared._longest
    if sinks and q_longest > _abi.lib().fsp_attention_packed_sinks_chunk(window, sinks, k_longest):
        room = int(_abi.lib().fsp_attention_packed_sinks_workspace(
            *sizes, k_longest, prepared.batch, window, sinks))
    else:
        room = int(_abi.lib().fsp_attention_packed_workspace(*sizes, causal and not window))
    kept = (head, sinks, _like((room,), torch.uint8, q.device),
            tuple(_like(t.shape, t.dtype, t.device) for t in grads))
    _run_backward(prepared, kept, rows, flat, grads)
    if key is not None and flat is lse and all(
            x is y for x, y in zip(rows, (grad_out, q, k, v, out))):
        _keep(prepared._calls, key, kept)
    return grads


def _run_backward(prepared, kept, rows, lse, grads):
    """``kept``: the arguments up to the addresses, and a pattern of the workspace."""
    head, sinks, room, _ = kept
    grad_out, q, k, v, out = rows
    if q.shape[0] or k.shape[0]:
        work = torch.empty_like(room, memory_format=_CONTIGUOUS)
        args = head + _PACKED_AT.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            grad_out.data_ptr(), grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(),
            work.data_ptr())
        if sinks:
            _first_tiles(prepared, q.shape[1] // k.shape[1])
            status = _abi.lib_on(prepared.device).fsp_attention_packed_sinks_backward(
                args, sinks, prepared._sequences.data_ptr(), prepared.batch, prepared._on())
        else:
            status = _abi.lib_on(prepared.device).fsp_attention_packed_backward(args, prepared._on())
        if status:
            _abi.check(status, "fsp_attention_packed_backward")


def flagsparse_attention_packed_backward(grad_out, q, k, v, out, lse, indptr=None, k_indptr=None, *,
                                         prepared=None, causal=True, window=None, sinks=0, scale=None):
    """(grad_q, grad_k, grad_v) of flagsparse_attention_packed: ``grad_out`` is the gradient of its
    output, ``out`` and ``lse`` what it returned, the other arguments its own.  The gradients are not
    differentiable themselves.

    Sums are float32 and in a fixed order: equal calls give equal bits.  What is not finite may reach
    rows of the same sequence within 64 queries or keys of those that it belongs to, as in the
    forward pass; it never reaches another sequence."""
    key, rows = None, (grad_out, q, k, v, out)
    _refuse_tangents(*rows, lse)
    if type(prepared) is PreparedAttention and type(scale) in _PLAIN and \
            type(window) in _PLAIN and type(causal) in _PLAIN and type(sinks) in _PLAIN:
        key = _layouts(*rows, lse) + (causal, window, sinks, scale)
        kept = prepared._calls.get(key)
        if kept is not None and not (grad_out.data_ptr() | q.data_ptr() | k.data_ptr() |
                                     v.data_ptr() | out.data_ptr()) % 16:
            grads = tuple([torch.empty_like(t, memory_format=_CONTIGUOUS) for t in kept[3]])
            _run_backward(prepared, kept, rows, lse, grads)
            return grads
    prepared, causal, window, sinks = _packed_inputs(q, k, v, indptr, k_indptr, prepared, causal,
                                                     window, sinks)
    for t, name in ((grad_out, "grad_out"), (out, "out")):
        _check_tensor(t, name, q.dtype, q.device, q.shape[1], q.shape[2])
        if t.shape[0] != q.shape[0]:
            raise ValueError(f"{name} must have {q.shape[0]} tokens, got {t.shape[0]}")
    _check_out(lse, "lse", q.shape[:2], torch.float32, q.device)
    return _backward(prepared, grad_out, q, k, v, out, lse, causal, window, sinks,
                     _scale_of(scale, q.shape[2]), key)
