"""Attention over packed sequences and over a paged cache on gfx950.

Sequences of different lengths are rows of a CSR pattern: ``indptr`` over the tokens of a packed
batch, or over the pages that a cache holds of each sequence (``indices``: the pages).

* ``flagsparse_paged_append``: new keys and values, rotated by their positions, into the cache;
* ``flagsparse_attention_paged``: one new query per sequence over all that the cache holds of it;
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


def _int32(t, name, length, device):
    """A contiguous int32 device array of ``length``."""
    if not torch.is_tensor(t) or t.ndim != 1 or t.numel() != length:
        raise ValueError(f"{name} must be a 1D tensor of length {length}")
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on {device}")
    if t.dtype not in SUPPORTED_INDEX_DTYPES:
        raise TypeError(f"{name} dtype must be torch.int32 or torch.int64")
    if t.dtype == torch.int64:
        t = t.clamp(-1, 2**31 - 1).to(torch.int32)
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
                 "_calls", "_counts")

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
        # the pieces that attention is cut into
        self._piece = int(_abi.lib().fsp_attention_paged_piece(int(rooms.sum()), self.kv_heads))
        table, first, self._most = _pieces(pages, self.page_size, self._piece)
        # long pieces first, for short ones to even out the end: 96 ragged sequences of up to 4096 tokens,
        # 8 heads of 128: 51 us, 55 in the sequences' order
        held = np.minimum(self._piece, table[:, 4] - table[:, 1])
        table = table[np.argsort(-held, kind="stable")]
        both = torch.from_numpy(np.concatenate([table.ravel(), first])).to(k_pages.device)
        self._pieces, self._first = both[:table.size].view(-1, 8), both[table.size:]
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


def _pieces(pages, page_size, piece):
    """(the pieces of ``piece`` tokens that sequences with so many pages may come to hold, the sequences'
    first ones, the most that one has), as the kernels read them."""
    rooms = pages * page_size
    n = np.maximum(1, -(-rooms // piece))
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
                            interleaved=False, out=None):
    """Write new keys and values into a paged cache, rotated by their positions on the way.

    ``k``, ``v``: [tokens, kv_heads, dim], the new tokens of each sequence one after the other:
    sequence b's are ``token_indptr[b]`` to ``token_indptr[b + 1]`` (None: one token per sequence).
    ``lengths[b]`` is what sequence b holds with them, so its last token has position
    ``lengths[b] - 1``.  ``cos``, ``sin``: float32 [positions, half]; the first 2 * half elements of
    every head of ``k`` and ``q`` are rotated by pairs, (a, b) -> (a cos - b sin, a sin + b cos):
    elements half apart, or neighbours with ``interleaved``.  Without them nothing is rotated.

    Returns the rotated ``q`` [tokens, heads, dim] (written to ``out`` where given, which may be ``q``),
    or None without ``q``.  The pages that new tokens go to belong to one sequence each, and ``k``,
    ``v`` and ``q`` lie outside the cache.  With
    ``prepared`` nothing is waited for, so lengths are not checked: a token whose position is
    negative or past its sequence's pages is not stored and its row of ``q`` comes back as NaN."""
    key = None
    if out is None and type(prepared) is PreparedPagedKV:
        key = _layouts(k, v, q, cos, sin, lengths, token_indptr) + (
            bool(interleaved), prepared.k_pages.data_ptr(), prepared.v_pages.data_ptr())
        kept = prepared._calls.get(key)
        if kept is not None and not (k.data_ptr() | v.data_ptr()) % 16 and (
                q is None or q.data_ptr() % 16 == 0):
            head, like = kept
            res = None if q is None else torch.empty_like(like, memory_format=_CONTIGUOUS)
            _append(prepared, head, k, v, q, res, cos, sin, token_indptr, lengths)
            return res
    kv, n = _paged_of(prepared, k_pages, v_pages, indptr, indices, lengths)
    dev, dt = kv.device, kv.dtype
    _check_tensor(k, "k", dt, dev, kv.kv_heads, kv.dim)
    _check_tensor(v, "v", dt, dev, kv.kv_heads, kv.dim)
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        raise ValueError(f"v must have {tokens} tokens, got {v.shape[0]}")
    given = (k, v, q, cos, sin, lengths, token_indptr)
    if token_indptr is None:
        if tokens != kv.batch:
            raise ValueError(f"k must have one token for each of {kv.batch} sequences, got "
                             f"{tokens}; other numbers need token_indptr")
    else:
        token_indptr = _int32(token_indptr, "token_indptr", kv.batch + 1, dev)
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
        _append(kv, head, k, v, q, res, cos, sin, token_indptr, n)
        if key is not None and all(x is y for x, y in zip(
                (k, v, q, cos, sin, n, token_indptr), given)):
            _keep(kv._calls, key, (head, None if q is None else _like(q.shape, dt, dev)))
    elif res is not None:  # tokens of no sequence
        res.fill_(float("nan"))
    if copied:
        out.copy_(res)
        res = out
    return res


def _at(t):
    return 0 if t is None else t.data_ptr()


def _append(kv, head, k, v, q, res, cos, sin, token_indptr, lengths):
    args = head + _APPEND_AT.pack(k.data_ptr(), v.data_ptr(), _at(q), _at(res), _at(cos), _at(sin),
                                  _at(token_indptr), lengths.data_ptr())
    status = _abi.lib().fsp_paged_append(args, kv._on())
    if status:
        _abi.check(status, "fsp_paged_append")


def flagsparse_attention_paged(q, lengths, *, prepared=None, k_pages=None, v_pages=None,
                               indptr=None, indices=None, scale=None, window=None, out=None,
                               return_lse=False):
    """Attention of one query per sequence over what a paged cache holds of it.

    ``q``: [sequences, heads, dim]; ``lengths[b]``: the tokens that sequence b holds, the query's
    own among them (0: the sequence is empty, and its output is zeros).  ``window``: only the last
    ``window`` tokens are seen.  ``scale``: dim ** -0.5 by default.  Returns [sequences, heads, dim],
    with the float32 log-sum-exp [sequences, heads] if ``return_lse``; neither is differentiable, nor
    is what flagsparse_paged_append gives.  With ``prepared`` nothing is
    waited for, so lengths are not checked: one that its sequence's pages cannot hold gives NaN."""
    key = None
    if out is None and type(prepared) is PreparedPagedKV and type(scale) in _PLAIN and \
            type(window) in _PLAIN:
        key = _layouts(q, lengths) + (scale, window, prepared.k_pages.data_ptr(),
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
    factor, past = _scale_of(scale, kv.dim), _window_of(window)
    res, copied = _result(out, "out", q.shape, dt, dev, q, kv.k_pages, kv.v_pages)
    rows = _rows(q)
    # what such calls share: the arguments, patterns of their arrays, the counts of arrivals they need
    pieces, need, room = kv._pieces.shape[0], 0, None
    if pieces > kv.batch:
        need = int(_abi.lib().fsp_attention_paged_counts(pieces, kv._most, kv.batch, heads,
                                                         kv.kv_heads))
        room = _like((pieces * heads * (kv.dim + 2),), torch.float32, dev)
    kept = (kv._packed() + _PAGED.pack(
        kv._pieces.data_ptr(), kv._first.data_ptr(), pieces, kv._piece, heads, past, factor,
        *_steps(rows), *_steps(res)), _like(q.shape, dt, dev),
        _like((kv.batch, heads), torch.float32, dev), room, need)
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
    head, _, like_lse, room, need = kept
    lse = torch.empty_like(like_lse, memory_format=_CONTIGUOUS) if return_lse else None
    if not kv.batch:
        return lse
    stream, work, counts = kv._on(), None, None
    if room is not None:
        work = torch.empty_like(room, memory_format=_CONTIGUOUS)
        if need:
            counts = _arrivals(kv, stream, need)
    status = _abi.lib().fsp_attention_paged(head + _PAGED_AT.pack(
        q.data_ptr(), res.data_ptr(), _at(lse), lengths.data_ptr(), _at(work), _at(counts)), stream)
    if status:
        _abi.check(status, "fsp_attention_paged")
    return lse


# ---- packed sequences ----


class PreparedAttention:
    """The sequences of a packed batch, checked once, and the kernels' work lists over them: tiles of
    one sequence's rows, those with the most to do first, so that the last ones to finish are
    short."""

    __slots__ = ("batch", "q_tokens", "k_tokens", "device", "_longest", "_tiles", "_streams", "_calls")

    def __init__(self, q_len, k_len, device):
        self.batch = len(q_len)
        self.q_tokens = int(q_len.sum())
        self.k_tokens = int(k_len.sum())
        self.device = device
        self._longest = tuple(int(n.max(initial=0)) for n in (q_len, k_len))
        # (queries, queries in half tiles, keys, keys in half tiles; causal) -> the list
        names = [(which, causal) for which in range(4) for causal in (False, True)]
        lists = [_tiles(q_len, k_len, int(_abi.lib().fsp_attention_packed_tile(which)), causal,
                        which >= 2) for which, causal in names]
        flat = torch.from_numpy(np.concatenate(lists)).to(device)
        ends = np.cumsum([0] + [len(t) for t in lists])
        self._tiles = {name: flat[ends[i]:ends[i + 1]] for i, name in enumerate(names)}
        self._streams = _Streams()
        self._calls = _abi.Calls()

    def _on(self):
        """The current stream, on which the work lists are marked as used."""
        stream = _abi.raw_stream(self.device)
        if stream not in self._streams.seen:
            self._streams.mark(stream, self.device, self._tiles.values())
        return stream


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


def _packed_inputs(q, k, v, indptr, k_indptr, prepared, causal, window):
    """(prepared, causal, window) of a call whose arrays are checked against each other."""
    _check_tensor(q, "q")
    _check_tensor(k, "k", q.dtype, q.device, None, q.shape[2])
    _check_tensor(v, "v", q.dtype, q.device, k.shape[1], q.shape[2])
    _check_heads(q.shape[1], k.shape[1])
    _check_dim(q.shape[2])
    window = _window_of(window)
    if window and not causal:
        raise ValueError("window needs causal=True")
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
    return prepared, bool(causal), window


def _pack(prepared, q, k, v, causal, window, scale, out, grads=()):
    """A call's arguments up to the addresses; grads: grad_out, grad_q, grad_k, grad_v."""
    lists = [prepared._tiles[which, causal] for which in range(4)]
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


def _run_forward(prepared, head, q, k, v, res, lse):
    if q.shape[0]:
        status = _abi.lib().fsp_attention_packed(head + _PACKED_AT.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), res.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, 0),
            prepared._on())
        if status:
            _abi.check(status, "fsp_attention_packed")


def _forward(prepared, q, k, v, causal, window, scale, out=None, key=None):
    res, copied = _result(out, "out", q.shape, q.dtype, q.device, q, k, v)
    rows = _rows(q), _rows(k), _rows(v)
    head = _pack(prepared, *rows, causal, window, scale, res)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    _run_forward(prepared, head, *rows, res, lse)
    if key is not None and rows[0] is q and rows[1] is k and rows[2] is v:
        _keep(prepared._calls, key, (head, _like(q.shape, q.dtype, q.device),
                                     _like(lse.shape, lse.dtype, lse.device)))
    if copied:
        out.copy_(res)
        res = out
    return res, lse


class _Differentiable(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, prepared, causal, window, scale):
        out, lse = _forward(prepared, q, k, v, causal, window, scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.rest = (prepared, causal, window, scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        q, k, v, out, lse = ctx.saved_tensors
        prepared, causal, window, scale = ctx.rest
        _refuse_tangents(grad, q, k, v)
        grads = _backward(prepared, grad, q, k, v, out, lse, causal, window, scale)
        return *grads, None, None, None, None


def flagsparse_attention_packed(q, k, v, indptr=None, k_indptr=None, *, prepared=None, causal=True,
                                window=None, scale=None, out=None, return_lse=False):
    """Attention over packed sequences.

    ``q``: [tokens, heads, dim]; ``k``, ``v``: [key tokens, kv_heads, dim]; the sequences are given
    by ``indptr`` / ``k_indptr`` (checked by this call, which waits for them) or by ``prepared``
    (prepare_attention_packed).  With ``causal`` query i of nq sees key j of nk if
    j <= i + nk - nq, the last query all of them; ``window``: only the last ``window`` of those.
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
            type(scale) in _PLAIN and type(window) in _PLAIN and type(causal) in _PLAIN:
        key = _layouts(q, k, v) + (causal, window, scale)
        kept = prepared._calls.get(key)
        if kept is not None and not (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
            head, like, like_lse = kept
            res = torch.empty_like(like, memory_format=_CONTIGUOUS)
            lse = torch.empty_like(like_lse, memory_format=_CONTIGUOUS)
            _run_forward(prepared, head, q, k, v, res, lse)
            return (res, lse) if return_lse else res
    prepared, causal, window = _packed_inputs(q, k, v, indptr, k_indptr, prepared, causal, window)
    scale = _scale_of(scale, q.shape[2])
    if wanted:
        if out is not None:
            raise RuntimeError("out cannot be given where q, k or v require a gradient")
        res, lse = _Differentiable.apply(q, k, v, prepared, causal, window, scale)
    else:
        res, lse = _forward(prepared, q, k, v, causal, window, scale, out, key)
    return (res, lse) if return_lse else res


def _backward(prepared, grad_out, q, k, v, out, lse, causal, window, scale, key=None):
    rows = tuple(_rows(t) for t in (grad_out, q, k, v, out))
    flat = lse.contiguous()
    grads = tuple(torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v))
    head = _pack(prepared, *rows[1:4], causal, window, scale, rows[4], (rows[0], *grads))
    room = int(_abi.lib().fsp_attention_packed_workspace(
        prepared._tiles[2, causal].shape[0], q.shape[1], k.shape[1], q.shape[2], q.shape[0],
        k.shape[0], causal and not window))
    kept = (head, _like((room,), torch.uint8, q.device),
            tuple(_like(t.shape, t.dtype, t.device) for t in grads))
    _run_backward(prepared, kept, rows, flat, grads)
    if key is not None and flat is lse and all(
            x is y for x, y in zip(rows, (grad_out, q, k, v, out))):
        _keep(prepared._calls, key, kept)
    return grads


def _run_backward(prepared, kept, rows, lse, grads):
    """``kept``: the arguments up to the addresses, and a pattern of the workspace."""
    head, room, _ = kept
    grad_out, q, k, v, out = rows
    if q.shape[0] or k.shape[0]:
        work = torch.empty_like(room, memory_format=_CONTIGUOUS)
        status = _abi.lib().fsp_attention_packed_backward(head + _PACKED_AT.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            grad_out.data_ptr(), grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(),
            work.data_ptr()), prepared._on())
        if status:
            _abi.check(status, "fsp_attention_packed_backward")


def flagsparse_attention_packed_backward(grad_out, q, k, v, out, lse, indptr=None, k_indptr=None, *,
                                         prepared=None, causal=True, window=None, scale=None):
    """(grad_q, grad_k, grad_v) of flagsparse_attention_packed: ``grad_out`` is the gradient of its
    output, ``out`` and ``lse`` what it returned, the other arguments its own.  The gradients are not
    differentiable themselves.

    Sums are float32 and in a fixed order: equal calls give equal bits.  What is not finite may reach
    rows of the same sequence within 64 queries or keys of those that it belongs to, as in the
    forward pass; it never reaches another sequence."""
    key, rows = None, (grad_out, q, k, v, out)
    _refuse_tangents(*rows, lse)
    if type(prepared) is PreparedAttention and type(scale) in _PLAIN and \
            type(window) in _PLAIN and type(causal) in _PLAIN:
        key = _layouts(*rows, lse) + (causal, window, scale)
        kept = prepared._calls.get(key)
        if kept is not None and not (grad_out.data_ptr() | q.data_ptr() | k.data_ptr() |
                                     v.data_ptr() | out.data_ptr()) % 16:
            grads = tuple([torch.empty_like(t, memory_format=_CONTIGUOUS) for t in kept[2]])
            _run_backward(prepared, kept, rows, lse, grads)
            return grads
    prepared, causal, window = _packed_inputs(q, k, v, indptr, k_indptr, prepared, causal, window)
    for t, name in ((grad_out, "grad_out"), (out, "out")):
        _check_tensor(t, name, q.dtype, q.device, q.shape[1], q.shape[2])
        if t.shape[0] != q.shape[0]:
            raise ValueError(f"{name} must have {q.shape[0]} tokens, got {t.shape[0]}")
    _check_out(lse, "lse", q.shape[:2], torch.float32, q.device)
    return _backward(prepared, grad_out, q, k, v, out, lse, causal, window,
                     _scale_of(scale, q.shape[2]), key)
