"""Attention for a batch whose requests share a long prefix, computed once for all (``csrc/shared_prefix.cu``).

Requests come in groups; the requests of a group share a prefix (a system prompt, a document) whose keys and values are in
the cache once.  Every request brings its newest tokens, one or several (a last token and drafted ones), and each of
them attends over its group's prefix and over the request's own tokens up to itself.

All work goes to the current stream; nothing but scratch memory is kept between calls.
"""
from __future__ import annotations

import functools
import struct
import threading
from ctypes import c_char_p, c_longlong

import torch

from . import _Counter, _ok
from .build import load_library
from .quant_cache import _CODE, _at, _capturing, _device, _function, _of_device, _raw_stream

MAX_HEAD_DIM = 256
_ATTEND = struct.Struct("=29qd")
_LAUNCHES = {0: 3, -101: 1, -102: 2}    # what the entry point returns: how many kernels it launched
_int32 = torch.int32
_attend_functions: dict = {}


def supports(head_dim: int, heads: int, kv_heads: int) -> bool:
    """Whether the kernels take these heads."""
    return head_dim % 16 == 0 and 16 <= head_dim <= MAX_HEAD_DIM and kv_heads > 0 and heads > 0 and heads % kv_heads == 0


def _table(t, count, what, device):
    """(address, row stride, columns) of a table of pages."""
    shape, strides = t.shape, t.stride()
    if t.dtype is not _int32 or len(shape) != 2 or shape[0] != count or (strides[1] != 1 and shape[1] > 1):
        raise ValueError(f"{what} is int32 [{count}, pages], its columns side by side; got {t.dtype} {tuple(shape)}, strides "
                         f"{strides}")
    if count > 1 and strides[0] >= 1 << 31:
        raise ValueError(f"{what}'s rows are {strides[0]} entries apart: fewer than 2^31")
    return _at(t, device), strides[0] if count > 1 else 0, shape[1]


def _vector(t, count, what, device):
    if t.dtype is not _int32 or t.shape != (count,) or not t.is_contiguous():
        raise ValueError(f"{what} is int32 [{count}], contiguous; got {t.dtype} {tuple(t.shape)}")
    return _at(t, device)


# What a call's scratch depends on, in the order of the words that the library takes.
@functools.lru_cache(maxsize=1024)
def _scratch_bytes(hd, code, G, prefix_limit, B, limit, T, nh, nkv, sms, longest, page) -> int:
    f = load_library("shared_prefix", (f"GF_HEAD_DIM={hd}",)).gf_prefix_scratch
    f.argtypes, f.restype = [c_char_p], c_longlong
    return f(_ATTEND.pack(0, 0, code, 0, 0, 1, page, 0, 0, 0, G, prefix_limit, 0, 0, 0, B, limit, 0, 0, 0, T, nh, nkv, sms,
                          longest, 0, 0, 0, 0, 1.0))


_scratch: dict = {}
# Held from the choice of the scratch until the kernels that use it are in their stream: the foreign call lets other
# threads run, and another call on the stream between two of this one's kernels would overwrite its pieces.
_launching = threading.Lock()


def _scratch_for(size: int, device: int, stream: int) -> torch.Tensor:
    """A buffer that only this stream's calls use; a graph that is being captured keeps one of its own."""
    if _capturing():
        return torch.empty(size, dtype=torch.uint8, device=device)
    buf = _scratch.get((device, stream))
    if buf is None or buf.numel() < size:
        buf = _scratch[device, stream] = torch.empty(max(size, 1 << 20), dtype=torch.uint8, device=device)
    return buf


def attend(q: torch.Tensor, nh: int, pages, prefix_table: torch.Tensor, prefix_lens: torch.Tensor,
           block_table: torch.Tensor, lengths: torch.Tensor, scale: float, *, cu_groups=None, cu_seqlens_q=None,
           max_q_len: int | None = None, out=None) -> torch.Tensor:
    """Attention of the rows ``q [T, >= nh * head size]`` (bf16 or fp32, rotated) over shared prefixes and over each
    request's own tokens: ``[T, nh * head size]`` in ``q``'s type.

    ``pages``: the cache, ``[2, pages, page, kv heads, head size]`` or its two planes, keys and values rotated and written.
    ``prefix_table [G, P]``, ``prefix_lens [G]`` int32: the pages of every group's prefix in order and how many tokens it
    has (it may end inside a page).  ``block_table [B, W]``, ``lengths [B]`` int32: likewise of every request's own
    tokens, the new ones among them, counted from behind the prefix.  (Of tables that name all of a request's pages, with
    whole pages shared, these are ``table[first requests, :P]`` and ``table[:, P:]``; rows may have any stride.  How a call
    is carried out goes by the tables' widths: short sequences are fastest in narrow ones.)
    ``cu_groups [G + 1]`` int32: group ``g`` is the requests ``cu_groups[g] .. cu_groups[g + 1] - 1``, and a request of no
    group has no prefix; ``None``: one group of all requests.  ``cu_seqlens_q [B + 1]`` int32: request ``b`` has the rows
    ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1``; ``None``: row ``b`` alone.  ``max_q_len``: about how many rows a request
    has at most (a hint: the kernels' tiles go by it; ``None``: ``T / B``).

    The ``i``-th of a request's ``n`` rows sees the whole prefix and the own tokens ``0 .. length - n + i``; a row that
    sees nothing gives zeros.  What a row sees is finite (an infinity there leaves no number); what none sees may be
    anything.  Rows that belong to no request are not written: with ``out`` (``[T, nh * head size]``, contiguous, ``q``'s
    type) they stay as they were.  Entries of the tables behind a sequence's length are not read.  Starts rise or stay; of those
    that fall nothing but named rows is written, and a request whose rows lie in front of its group's first start does
    without the prefix there.  A wait inside that runs out leaves rows unwritten and is reported by
    ``gemm_bf16.check_errors``."""
    # (what follows is the host's time of a call: a plane of its own would be two tensors made, a helper a call)
    if torch.is_tensor(pages):
        shape, dtype = pages.shape, pages.dtype
        if len(shape) != 5 or shape[0] != 2 or not pages.is_contiguous():
            raise ValueError(f"the cache is [2, pages, page, kv heads, head size], contiguous; got {tuple(shape)}")
        _, count, page, nkv, hd = shape
        dev = _device(pages)
        k_at = pages.data_ptr()
        v_at = k_at + count * page * nkv * hd * pages.itemsize
    else:
        k, v = pages
        shape, dtype = k.shape, k.dtype
        if len(shape) != 4 or v.shape != shape or not k.is_contiguous() or not v.is_contiguous() or v.dtype != dtype:
            raise ValueError(f"the cache's planes are [pages, page, kv heads, head size], contiguous, of one shape and type; got "
                             f"{tuple(shape)}, {tuple(v.shape)}")
        count, page, nkv, hd = shape
        dev = _device(k)
        k_at, v_at = k.data_ptr(), _at(v, dev)
    code = _CODE.get(dtype)
    if code is None:
        raise TypeError(f"kernels take float32 or bfloat16 activations, not {dtype}")
    if not supports(hd, nh, nkv):
        raise ValueError(f"attention over shared prefixes takes head sizes that are a multiple of 16, at most "
                         f"{MAX_HEAD_DIM}, and a multiple of the kv heads; got head_dim={hd}, heads={nh}, kv_heads={nkv}")
    if count < 1 or page < 1 or count * page >= 1 << 31:
        raise ValueError(f"{count} pages of {page} tokens: a cache has at least one, and slots are 32-bit integers")
    width = nh * hd
    shape, strides = q.shape, q.stride()
    if len(shape) != 2 or q.dtype is not dtype or shape[1] < width or (strides[1] != 1 and shape[1] > 1):
        raise ValueError(f"q has rows of at least {width} channels without gaps in the cache's type {dtype}; got "
                         f"{q.dtype} {tuple(shape)}, strides {strides}")
    at, stride = _at(q, dev), strides[0]
    # (The kernels read 16 bytes at a time.  A clone: `contiguous` gives dense rows back as they are, wherever they start.)
    if (at | stride * q.itemsize) & 15 or not width <= stride < 1 << 31:
        q = q[:, :width].clone(memory_format=torch.contiguous_format)
        at, stride = q.data_ptr(), width
    T, B, G = shape[0], lengths.shape[0], prefix_lens.shape[0]
    prefix, prefix_stride, P = _table(prefix_table, G, "prefix_table", dev)
    table, table_stride, W = _table(block_table, B, "block_table", dev)
    prefix_tokens, own_tokens = _vector(prefix_lens, G, "prefix_lens", dev), _vector(lengths, B, "lengths", dev)
    groups = rows = 0
    if cu_groups is not None:
        groups = _vector(cu_groups, G + 1, "cu_groups", dev)
    elif G > 1:
        raise ValueError(f"{G} groups, and no cu_groups that says whose they are")
    if cu_seqlens_q is not None:
        rows = _vector(cu_seqlens_q, B + 1, "cu_seqlens_q", dev)
    elif T < B:
        raise ValueError(f"{T} rows for {B} requests of one row each")
    P, W = P * page, W * page
    if P >= 1 << 30 or W >= 1 << 30:
        raise ValueError(f"tables of {P} and {W} tokens: a sequence has fewer than 2^30")
    if max_q_len is not None and max_q_len < 0:
        raise ValueError(f"max_q_len is {max_q_len}")
    if not 0 < scale <= 1e38:                               # (in 32 bits, and times log2(e))
        raise ValueError(f"the scale of the scores is a positive number up to 1e38, not {scale}")
    if out is None:
        out = q.new_empty(T, width)
        out_at = out.data_ptr()
    else:
        if out.dtype is not dtype or out.shape != (T, width) or not out.is_contiguous():
            raise ValueError(f"out is {dtype} {(T, width)}, contiguous; got {out.dtype} {tuple(out.shape)}")
        out_at = _at(out, dev)
    if (k_at | v_at | out_at) & 15:
        raise ValueError("the cache's planes and out start at multiples of 16 bytes")
    if T == 0 or B == 0:
        return out
    sms, err = _of_device(dev)
    stream = _raw_stream(dev)
    longest = min(max_q_len or -(-T // B), T)
    size = _scratch_bytes(hd, code, G, P, B, W, T, nh, nkv, sms, longest, page)
    f = _attend_functions.get(hd)
    if f is None:
        f = _attend_functions[hd] = _function("shared_prefix", "gf_prefix_attend", (f"GF_HEAD_DIM={hd}",))
    with _launching:
        scratch = _scratch_for(size, dev, stream).data_ptr() if size else 0
        rc = f(_ATTEND.pack(at, stride, code, k_at, v_at, count, page, prefix, prefix_stride, prefix_tokens, G, P, table,
                            table_stride, own_tokens, B, W, groups, rows, out_at, T, nh, nkv, sms, longest, scratch, size, err,
                            stream, scale))
    if rc not in _LAUNCHES:
        _ok(rc, "shared_prefix.attend")
    _Counter.launches += _LAUNCHES[rc]
    return out
