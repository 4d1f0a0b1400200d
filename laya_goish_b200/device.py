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
kernels and reported by ``check_status``.  Forward only: tensors that require a
gradient (while gradients are recorded) or have a tangent are refused.  There
is no counterpart in the reference, which has no K/V cache.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from ._lib import E_INVALID, E_TIMEOUT, LayaError, check

try:
    from . import _device
except ImportError as e:
    raise RuntimeError("_device.so is not built: run `python -m laya_goish_b200.build` (needs nvcc and g++)") from e

PAGE = 64  # tokens per page
MAX_TOP = 64
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
STATUS_TIMEOUT, STATUS_PAGE, STATUS_TOKEN, STATUS_ROWS = 1, 2, 4, 8


def _refuse(message: str):
    raise LayaError(E_INVALID, message)


def _pages(x, name: str) -> None:
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        _refuse(f"{name} must be a CUDA tensor")
    if x.dim() != 4:
        _refuse(f"{name} must have 4 dimensions")


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
    """What page_plan computes, on the device (capacity c, n sequences).  One
    allocation holds them all: who keeps one past the step (lens, say) keeps 24
    bytes per row of the capacity, or clones it."""

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
    return PagePlan(*_device.page_plan(past, count, free_pages, tables, capacity, base))


class KVPages:
    """One layer's K and V pages, k and v [pages, kv_heads, 64, head_dim] F16 or
    BF16 with equal strides: the engine's layout, or a permuted view of pages
    held token by token ([pages, 64, kv_heads, head_dim].permute(0, 2, 1, 3)).
    Tensors that are given other memory afterwards need a new one."""

    def __init__(self, k, v):
        _pages(k, "k pages")
        _pages(v, "v pages")
        if v.dtype != k.dtype or v.device != k.device:
            _refuse("k and v pages must have the same type and device")
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
        self._at = ctypes.addressof(self._c)
        self._device = k.get_device()


def kv_append(pages: KVPages, k, v, slots) -> None:
    """Writes rows k, v ([rows, kv_heads, head_dim], the pages' type or F32, which
    is rounded once) to their slots ([rows] int64; -1: skipped; all others
    distinct)."""
    if not isinstance(pages, KVPages):
        _refuse("pages must be KVPages")
    _device.kv_append(pages._at, pages._device, pages.k, pages.v, k, v, slots)


def prefix_attention(q, pages: KVPages, prefix_pages, prefix_len: int, tables, lens, offsets, max_q: int,
                     scale: float | None = None, out=None, lse=None):
    """Attention of sequences that share a prefix: row offsets[b] + j of q
    ([rows, heads, head_dim]) sees the prefix_len tokens in prefix_pages and,
    of its own lens[b] tokens in the pages of tables[b], those up to its own
    (its new rows are the last ones).  max_q: the most rows of a sequence.
    scale defaults to head_dim ** -0.5.  Returns out; rows of no sequence are
    left as they were (0 in an out made here), rows that see no key give 0.
    lse ([rows, heads] F32, optional) receives ln sum exp of the scores.  out
    and lse share no memory with each other or with what the call reads."""
    if not isinstance(pages, KVPages):
        _refuse("pages must be KVPages")
    return _device.prefix_attention(pages._at, pages._device, pages.k, pages.v, q, prefix_pages, prefix_len, tables,
                                    lens, offsets, max_q, scale, out, lse)


class TokenLogprobs(NamedTuple):
    """What token_logprobs computes ([n] rows, c tokens, k alternatives), in one
    allocation."""

    logprobs: torch.Tensor      # [n, c] F32; 0 for token -1
    entropy: torch.Tensor       # [n] F32, nats
    lse: torch.Tensor           # [n] F32
    top_ids: torch.Tensor       # [n, k] int32, likeliest first, equal ones by id; -1 where there are fewer
    top_logprobs: torch.Tensor  # [n, k] F32


def token_logprobs(logits, tokens, top: int = 0) -> TokenLogprobs:
    """Log probabilities of tokens ([n, c] int32) under the rows of logits ([n,
    vocab] F32, F16 or BF16), the rows' entropy and lse, and the `top` (at most
    64) likeliest tokens.  Logits of -inf are tokens that are not there."""
    return TokenLogprobs(*_device.token_logprobs(logits, tokens, top))
