"""Operators on CUDA tensors: one step of a batch of sequences over paged K/V.

* ``page_plan``        — block tables, slot map, positions and row offsets from request lengths
* ``kv_append``        — K and V rows into their slots of the pages (``KVPages``)
* ``prefix_attention`` — attention of sequences that share a prefix, the prefix read once for all
* ``token_logprobs``   — log probabilities of given tokens, entropy, the likeliest tokens

Tensors are torch CUDA tensors of one device.  Work runs on torch's current
stream of that device; a call returns without waiting for it and may be
captured into a CUDA graph (after a first call on the device).  Nothing is
kept between calls: outputs and workspaces come from torch's allocator.  What
is wrong with the arguments raises LayaError ("invalid"); what only the GPU
sees (page numbers, slots, lengths, token ids out of range) is skipped by the
kernels and reported by ``check_status``.  Forward only.  There is no
counterpart in the reference, which has no K/V cache.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib
from ._lib import E_INVALID, E_TIMEOUT, LayaError, check

PAGE = 64  # tokens per page
MAX_TOP = 64
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
STATUS_TIMEOUT, STATUS_PAGE, STATUS_TOKEN, STATUS_ROWS = 1, 2, 4, 8


_stream = torch._C._cuda_getCurrentRawStream  # of a device index, without making a Stream object
_current = torch._C._cuda_getDevice


def _refuse(message: str):
    raise LayaError(E_INVALID, message)


def _tensor(x, name: str, dim: int, dtype=None, device=None) -> None:
    # plain tests: a message is only put together when one fails (a call costs a few microseconds)
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        _refuse(f"{name} must be a CUDA tensor")
    if x.dim() != dim:
        _refuse(f"{name} must have {dim} dimension(s)")
    if dtype is not None and x.dtype is not dtype:
        _refuse(f"{name} must be {dtype}")
    if device is not None and x.device != device:
        _refuse(f"{name} is on another device")
    if x.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} requires a gradient; the operators are forward only")


def _flat(x, name: str, dtype, device) -> None:
    _tensor(x, name, 1, dtype, device)
    if not x.is_contiguous():
        _refuse(f"{name} must be contiguous")


def _rows(x, name: str) -> int:
    """Row stride of a tensor whose rows (everything past dimension 0) are contiguous."""
    shape, stride = x.shape, x.stride()
    width = 1
    for d in range(len(shape) - 1, 0, -1):
        if shape[d] != 1 and stride[d] != width:
            _refuse(f"the rows of {name} must be contiguous")
        width *= shape[d]
    return stride[0] if shape[0] > 1 else width


def _call(device, fn, *args):
    """Runs a library entry point with the tensors' device current, on its current stream."""
    index = device.index
    if _current() == index:
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(index))
    if rc < 0:
        check(rc)


def check_status(device: int = 0) -> None:
    """Waits for the device and raises LayaError if an operator met something
    out of range there since the last check (or a wait of its own ran out)."""
    bits = ctypes.c_uint32()
    check(_lib.lib().laya_device_status(device, ctypes.byref(bits)))
    if bits.value & STATUS_TIMEOUT:
        raise LayaError(E_TIMEOUT, "a device-side wait ran out of its budget")
    words = [w for b, w in ((STATUS_PAGE, "a page or slot outside the cache, or a length beyond its block table"),
                            (STATUS_TOKEN, "a token id outside the vocabulary"),
                            (STATUS_ROWS, "more query rows in a sequence than max_q, or offsets out of order"))
             if bits.value & b]
    if words:
        _refuse("; ".join(words))


class PagePlan(NamedTuple):
    """What page_plan computes, on the device (capacity c, n sequences)."""

    slots: torch.Tensor      # [c] int64: page * 64 + row, -1 without one
    positions: torch.Tensor  # [c] int32
    seqs: torch.Tensor       # [c] int32, -1 past the last sequence
    offsets: torch.Tensor    # [n + 1] int32: each sequence's first row
    lens: torch.Tensor       # [n] int32: past + count
    totals: torch.Tensor     # [2] int64: rows, pages taken from the free list (uncut)


def page_plan(past, count, free_pages, tables, capacity: int, base: int = 0) -> PagePlan:
    """Plans a step in which sequence i, holding past[i] tokens in the pages of
    tables[i], gets count[i] more.  Pages it lacks come from free_pages in
    sequence order and are written into tables ([n, width] int32, in place;
    other entries stay as they are).  Rows are numbered through the sequences;
    positions start at base + past[i].  past, count: [n] int32; n <= 8192."""
    _tensor(tables, "tables", 2, torch.int32)
    dev = tables.device
    n, width = tables.shape
    _flat(past, "past", torch.int32, dev)
    _flat(count, "count", torch.int32, dev)
    _flat(free_pages, "free_pages", torch.int32, dev)
    if past.shape[0] != n or count.shape[0] != n:
        _refuse("past, count and tables must have one row per sequence")
    if n and width > 1 and tables.stride(1) != 1:
        _refuse("the rows of tables must be contiguous")
    stride = tables.stride(0) if n > 1 else width
    if stride < width:
        _refuse("the rows of tables overlap")
    if not 0 <= capacity < 1 << 31:
        _refuse("capacity out of range")
    if not 0 <= base < 1 << 31:
        _refuse("base out of range")
    # the outputs share one allocation, each on 16 bytes
    a, c, m = -capacity % 4, 2 * (capacity % 2), (n + 1 + 3) // 4 * 4
    slots, _, positions, _, seqs, _, offsets, _, lens, _, totals = torch.split_with_sizes(
        tables.new_empty(4 * capacity + c + 2 * a + 2 * m + 4),
        (2 * capacity, c, capacity, a, capacity, a, n + 1, m - n - 1, n, m - n, 4))
    slots, totals = slots.view(torch.int64), totals.view(torch.int64)[:2]
    _call(dev, _lib.lib().laya_page_plan, past.data_ptr(), count.data_ptr(), n, free_pages.data_ptr(),
          free_pages.shape[0], base, tables.data_ptr(), stride, width, slots.data_ptr(), positions.data_ptr(),
          seqs.data_ptr(), capacity, offsets.data_ptr(), lens.data_ptr(), totals.data_ptr())
    return PagePlan(slots, positions, seqs, offsets, lens, totals)


class KVPages:
    """One layer's K and V pages, k and v [pages, kv_heads, 64, head_dim] F16 or
    BF16 with equal strides: the engine's layout, or a permuted view of pages
    held token by token ([pages, 64, kv_heads, head_dim].permute(0, 2, 1, 3))."""

    def __init__(self, k, v):
        _tensor(k, "k pages", 4)
        _tensor(v, "v pages", 4, k.dtype, k.device)
        if k.dtype not in (torch.float16, torch.bfloat16):
            _refuse("K/V pages must be F16 or BF16")
        if k.shape != v.shape:
            _refuse("k and v pages must have the same shape")
        pages, heads, rows, hd = k.shape
        if rows != PAGE:
            _refuse("a page holds 64 tokens")
        if hd not in (64, 128, 256):
            _refuse("head_dim must be 64, 128 or 256")
        if not pages or not heads:
            _refuse("empty K/V cache")
        if k.stride(3) != 1 or v.stride(3) != 1:
            _refuse("head vectors must be contiguous")
        # strides of dimensions of one element say nothing
        stride = [k.stride(d) if k.shape[d] > 1 else hd for d in range(3)]
        if any(v.stride(d) != stride[d] for d in range(3) if v.shape[d] > 1):
            _refuse("k and v pages must have the same strides")
        if any(s % 8 for s in stride) or (k.data_ptr() | v.data_ptr()) % 16:
            _refuse("K/V pages must be 16-byte aligned")
        last = 0
        for s, size in sorted((stride[d], k.shape[d]) for d in range(3)):  # each dimension past the one inside it
            if size > 1 and s < last + hd:
                _refuse("K/V pages overlap")
            last += s * (size - 1)
        self.k, self.v, self.device, self.dtype = k, v, k.device, k.dtype
        self.pages, self.kv_heads, self.head_dim = pages, heads, hd
        self._c = _lib.KvPages(k.data_ptr(), v.data_ptr(), stride[0], stride[1], stride[2], pages, heads, hd,
                               TYPES[k.dtype])
        self._ref = ctypes.byref(self._c)


def kv_append(pages: KVPages, k, v, slots) -> None:
    """Writes rows k, v ([rows, kv_heads, head_dim], the pages' type or F32, which
    is rounded once) to their slots ([rows] int64; -1: skipped; all others
    distinct)."""
    if not isinstance(pages, KVPages):
        _refuse("pages must be KVPages")
    _tensor(k, "k", 3, None, pages.device)
    _tensor(v, "v", 3, k.dtype, pages.device)
    _flat(slots, "slots", torch.int64, pages.device)
    if k.dtype not in (pages.dtype, torch.float32):
        _refuse("k and v must be of the pages' type or F32")
    if k.shape != v.shape or tuple(k.shape) != (slots.shape[0], pages.kv_heads, pages.head_dim):
        _refuse("k and v must be [rows, kv_heads, head_dim] with a slot per row")
    _call(pages.device, _lib.lib().laya_kv_append, pages._ref, TYPES[k.dtype], k.data_ptr(), v.data_ptr(),
          _rows(k, "k"), _rows(v, "v"), slots.data_ptr(), k.shape[0])


def prefix_attention(q, pages: KVPages, prefix_pages, prefix_len: int, tables, lens, offsets, max_q: int,
                     scale: float | None = None, out=None, lse=None):
    """Attention of sequences that share a prefix: row offsets[b] + j of q
    ([rows, heads, head_dim]) sees the prefix_len tokens in prefix_pages and,
    of its own lens[b] tokens in the pages of tables[b], those up to its own
    (its new rows are the last ones).  max_q: the most rows of a sequence.
    scale defaults to head_dim ** -0.5.  Returns out; rows of no sequence are
    left as they were (0 in an out made here), rows that see no key give 0.
    lse ([rows, heads] F32, optional) receives ln sum exp of the scores."""
    if not isinstance(pages, KVPages):
        _refuse("pages must be KVPages")
    dev = pages.device
    _tensor(q, "q", 3, pages.dtype, dev)
    rows, heads, hd = q.shape
    if hd != pages.head_dim:
        _refuse("q and the pages have different head_dim")
    if not heads or heads % pages.kv_heads:
        _refuse("heads must be a multiple of kv_heads")
    _flat(prefix_pages, "prefix_pages", torch.int32, dev)
    _flat(lens, "lens", torch.int32, dev)
    _flat(offsets, "offsets", torch.int32, dev)
    _tensor(tables, "tables", 2, torch.int32, dev)
    n, width = tables.shape
    if lens.shape[0] != n or offsets.shape[0] != n + 1:
        _refuse("lens, offsets and tables must fit the sequences")
    if n and width > 1 and tables.stride(1) != 1:
        _refuse("the rows of tables must be contiguous")
    if not 0 <= prefix_len <= prefix_pages.shape[0] * PAGE:
        _refuse("prefix_pages must hold prefix_len tokens")
    if not 0 <= max_q < 1 << 31:
        _refuse("max_q out of range")
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if out is None:
        out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    else:
        _tensor(out, "out", 3, pages.dtype, dev)
        if out.shape != q.shape:
            _refuse("out must have q's shape")
    if lse is not None:
        _tensor(lse, "lse", 2, torch.float32, dev)
        if tuple(lse.shape) != (rows, heads) or not lse.is_contiguous():
            _refuse("lse must be contiguous [rows, heads]")
    if _current() != dev.index:  # the workspace goes by the device that runs the call
        with torch.cuda.device(dev):
            return prefix_attention(q, pages, prefix_pages, prefix_len, tables, lens, offsets, max_q, scale, out, lse)
    L = _lib.lib()
    a = _lib.PrefixArgs(q.data_ptr(), _rows(q, "q"), rows, heads, offsets.data_ptr(), n, max_q,
                        prefix_pages.data_ptr(), prefix_len, width, tables.data_ptr(),
                        tables.stride(0) if n > 1 else width, lens.data_ptr(), scale, out.data_ptr(),
                        _rows(out, "out"), None if lse is None else lse.data_ptr(), None, 0)
    ref = ctypes.byref(a)
    a.workspace_bytes = size = L.laya_prefix_attention_workspace(pages._ref, ref)
    if size:
        work = q.new_empty(size, dtype=torch.uint8)
        a.workspace = work.data_ptr()
    _call(dev, L.laya_prefix_attention, pages._ref, ref)
    return out


class TokenLogprobs(NamedTuple):
    """What token_logprobs computes ([n] rows, c tokens, k alternatives)."""

    logprobs: torch.Tensor      # [n, c] F32; 0 for token -1
    entropy: torch.Tensor       # [n] F32, nats
    lse: torch.Tensor           # [n] F32
    top_ids: torch.Tensor       # [n, k] int32, likeliest first, equal ones by id; -1 where there are fewer
    top_logprobs: torch.Tensor  # [n, k] F32


def token_logprobs(logits, tokens, top: int = 0) -> TokenLogprobs:
    """Log probabilities of tokens ([n, c] int32) under the rows of logits ([n,
    vocab] F32, F16 or BF16), the rows' entropy and lse, and the `top` (at most
    64) likeliest tokens.  Logits of -inf are tokens that are not there."""
    _tensor(logits, "logits", 2)
    dev = logits.device
    if logits.dtype not in TYPES:
        _refuse("logits must be F32, F16 or BF16")
    n, vocab = logits.shape
    if not vocab:
        _refuse("empty vocabulary")
    _tensor(tokens, "tokens", 2, torch.int32, dev)
    if tokens.shape[0] != n:
        _refuse("tokens must have a row per row of logits")
    if not 0 <= top <= MAX_TOP:
        _refuse("top must be 0..64")
    c = tokens.shape[1]
    logprobs, entropy, lse, top_lp, ids = torch.split_with_sizes(
        logits.new_empty(n * (c + 2 + 2 * top), dtype=torch.float32), (n * c, n, n, n * top, n * top))
    logprobs, top_lp, ids = logprobs.view(n, c), top_lp.view(n, top), ids.view(torch.int32).view(n, top)
    _call(dev, _lib.lib().laya_token_logprobs, TYPES[logits.dtype], logits.data_ptr(), _rows(logits, "logits"), n,
          vocab, tokens.data_ptr(), _rows(tokens, "tokens") if c else 0, c, top, logprobs.data_ptr(),
          entropy.data_ptr(), lse.data_ptr(), ids.data_ptr(), top_lp.data_ptr())
    return TokenLogprobs(logprobs, entropy, lse, ids, top_lp)
