"""A paged key-value cache of 8 bits (``csrc/quant_cache.cu``, ``csrc/quant_attention.cu``): writing a
step's keys and values, reading them back, and attention of single new tokens over it.

A *cache* is the pair ``(codes, scales)``: ``codes [pages, kv heads, 2, page, head size]`` in int8 or
float8_e4m3fn (keys, then values) and ``scales [pages, kv heads, page, 2]`` fp32, both contiguous.  A row
(the keys or the values of one token and head) has one scale:

    ``scale = max(amax |x| * (1/Q), 2^-126)``, ``code = round_to_even(x * (1/scale))``, ``value = code * scale``

with ``Q`` 127 or 448; a row with an infinity or a NaN reads back as NaN.  A token's *slot* is ``page number
* page + place in the page``; ``block_table [B, W]`` int32 names a request's pages in order (entries behind
its length are not read), ``lengths [B]`` int32 its tokens, the new one among them.

All work goes to the current stream; nothing is kept between calls.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

from . import _code, _fn, _ok, _p, _stream
from .gemm_bf16 import num_sms

KINDS = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_FP8 = {torch.int8: 0, torch.float8_e4m3fn: 1}
MAX_HEAD_DIM = 256


def supports(head_dim: int, heads: int, kv_heads: int) -> bool:
    """Whether the kernels take these heads."""
    return head_dim % 16 == 0 and 16 <= head_dim <= MAX_HEAD_DIM and kv_heads > 0 and heads % kv_heads == 0


def make_cache(kind: str, pages: int, kv_heads: int, page: int, head_dim: int, device="cuda"):
    """An empty cache: ``kind`` ``"int8"`` or ``"fp8"``."""
    if kind not in KINDS:
        raise ValueError(f"a cache of 8 bits is 'int8' or 'fp8', not {kind!r}")
    return (torch.zeros(pages, kv_heads, 2, page, head_dim, dtype=KINDS[kind], device=device),
            torch.zeros(pages, kv_heads, page, 2, dtype=torch.float32, device=device))


def _cache(cache):
    """The checked facts of a cache: codes, scales, kind, pages, kv heads, page, head size."""
    codes, scales = cache
    fp8 = _FP8.get(codes.dtype)
    if fp8 is None:
        raise TypeError(f"codes are int8 or float8_e4m3fn, not {codes.dtype}")
    if codes.dim() != 5 or codes.shape[2] != 2 or not codes.is_contiguous():
        raise ValueError("codes are [pages, kv heads, 2, page, head size], contiguous; got "
                         f"{tuple(codes.shape)}")
    pages, nkv, _, page, hd = codes.shape
    if scales.dtype != torch.float32 or scales.shape != (pages, nkv, page, 2) or not scales.is_contiguous():
        raise ValueError(f"the scales of codes {tuple(codes.shape)} are fp32 {(pages, nkv, page, 2)}, "
                         f"contiguous; got {scales.dtype} {tuple(scales.shape)}")
    if hd % 16 or not 16 <= hd <= MAX_HEAD_DIM:
        raise ValueError(f"a cache of 8 bits takes head sizes that are a multiple of 16, at most "
                         f"{MAX_HEAD_DIM}; got {hd}")
    if pages * page >= 1 << 31:
        raise ValueError(f"{pages} pages of {page} tokens: slots are 32-bit integers")
    return codes, scales, fp8, pages, nkv, page, hd


def _ints(t, shape, what):
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} is int32 {tuple(shape)}, contiguous; got {t.dtype} {tuple(t.shape)}")
    return _p(t)


def _rows(x, columns, what):
    if x.dim() != 2 or x.shape[1] < columns or x.stride(1) != 1:
        raise ValueError(f"{what} has rows of at least {columns} channels without gaps; got "
                         f"{tuple(x.shape)}, strides {tuple(x.stride())}")
    return _p(x), x.stride(0), _code(x.dtype)


def _angles(table, hd):
    """(address, rows, rotated channels) of a table of cosines and sines."""
    if table is None:
        return None, 0, 0
    rot = table.shape[-1]
    if (table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous() or rot % 2 or rot > hd
            or table.shape[0] < 1):
        raise ValueError(f"the table of angles is fp32 [positions, an even number up to {hd}], contiguous; "
                         f"got {table.dtype} {tuple(table.shape)}")
    return _p(table), table.shape[0], rot


def _heads(nh, nkv):
    if nh < 1 or nh % nkv:
        raise ValueError(f"{nh} query heads are not a multiple of {nkv} kv heads")


def write(qkv: torch.Tensor, nh: int, table, positions: torch.Tensor, slots: torch.Tensor, cache, *,
          neighbours: bool = False) -> torch.Tensor:
    """Rows ``qkv [T, (nh + 2 kv heads) * head size]`` (bf16 or fp32) of a step: q and k are rotated by
    their token's position, k and v are put into its slot.  Returns the rotated q ``[T, nh * head size]`` in
    ``qkv``'s type; ``qkv`` stays as it is.

    ``table [positions, rot]`` fp32: cosines, then sines, of the angles of ``rot / 2`` pairs; the first
    ``rot`` channels of a head turn in pairs ``(j, j + rot/2)``, or ``(2j, 2j + 1)`` with ``neighbours``.
    ``None``: nothing turns.  ``positions``, ``slots`` int32 ``[T]``: a token whose slot is negative (or
    beyond the cache) is not written; two tokens of one call have different slots."""
    codes, scales, fp8, pages, nkv, page, hd = _cache(cache)
    _heads(nh, nkv)
    x, stride, code = _rows(qkv, (nh + 2 * nkv) * hd, "qkv")
    T = qkv.shape[0]
    at, rows, rot = _angles(table, hd)
    q = torch.empty((T, nh * hd), dtype=qkv.dtype, device=qkv.device)
    f = _fn("quant_cache", "gf_quant_write",
            [c_void_p] + [c_int] * 6 + [c_void_p] + [c_int] * 3 + [c_void_p] * 4
            + [c_int, c_void_p, c_int, c_int, c_void_p])
    _ok(f(x, stride, code, T, nh, nkv, hd, at, rows, rot, int(neighbours), _ints(positions, (T,), "positions"),
          _ints(slots, (T,), "slots"), _p(q), _p(codes), fp8, _p(scales), page, pages * page, _stream()),
        "quant_cache.write")
    return q


_READ_ARGS = [c_void_p, c_int, c_void_p, c_void_p, c_int] + [c_void_p] * 3 + [c_int] * 6 + [c_void_p, c_int, c_void_p]


def read(cache, block_table: torch.Tensor, lengths: torch.Tensor, dtype: torch.dtype, first=None
         ) -> torch.Tensor:
    """``[2, B, W * page, kv heads, head size]`` in ``dtype`` (bf16 or fp32): the keys and values of the
    tokens ``first[b] <= c < lengths[b]`` (``first`` ``None``: from the first one), zeros elsewhere."""
    codes, scales, fp8, pages, nkv, page, hd = _cache(cache)
    B, W = block_table.shape
    out = torch.empty((2, B, W * page, nkv, hd), dtype=dtype, device=codes.device)
    f = _fn("quant_cache", "gf_quant_read", _READ_ARGS)
    _ok(f(_p(codes), fp8, _p(scales), _ints(block_table, (B, W), "block_table"), W,
          _ints(lengths, (B,), "lengths"), None if first is None else _ints(first, (B,), "first"), None,
          pages * page, B, W * page, nkv, hd, page, _p(out), _code(dtype), _stream()), "quant_cache.read")
    return out


def read_slots(cache, slots: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``[2, N, kv heads, head size]``: the keys and values in ``slots [N]``, zeros for a negative one."""
    codes, scales, fp8, pages, nkv, page, hd = _cache(cache)
    N = slots.shape[0]
    out = torch.empty((2, N, nkv, hd), dtype=dtype, device=codes.device)
    f = _fn("quant_cache", "gf_quant_read", _READ_ARGS)
    _ok(f(_p(codes), fp8, _p(scales), None, 0, None, None, _ints(slots, (N,), "slots"), pages * page, 1, N,
          nkv, hd, page, _p(out), _code(dtype), _stream()), "quant_cache.read_slots")
    return out


_DECODE_ARGS = ([c_void_p, c_int, c_int, c_void_p, c_int, c_void_p, c_void_p, c_int, c_int, c_void_p, c_int, c_void_p]
                + [c_int] * 5 + [c_float, c_int, c_void_p] + [c_int] * 4 + [c_void_p, c_longlong, c_void_p])
_F32 = {torch.float32: 1, torch.bfloat16: 0}
# Requests of at most this many visible tokens are one block's work a kv head and need no scratch (the kernel has the
# same line: kShortKeys).
_SHORT = 1024


def _decode(q, nh, facts, block_table, lengths, scale, span, fused=None):
    """``fused``: ``(address, rows, rotated channels)`` of the table of angles and ``neighbours``."""
    codes, scales, fp8, pages, nkv, page, hd = facts
    _heads(nh, nkv)
    x, stride, code = _rows(q, (nh if fused is None else nh + 2 * nkv) * hd, "q" if fused is None else "qkv")
    B, W = block_table.shape
    if q.shape[0] != B:
        raise ValueError(f"{q.shape[0]} queries for {B} requests")
    out = torch.empty((B, nh * hd), dtype=q.dtype, device=q.device)
    defines = (f"GF_HEAD_DIM={hd}",)
    sms = num_sms(q.device)
    scratch, words = None, 0
    if W * page > _SHORT:
        size = _fn("quant_attention", "gf_quant_decode_scratch", [c_int] * 4, defines, kernels=0, restype=c_longlong)
        words = size(B, nh, nkv, sms) // 4
        scratch = torch.empty(words, dtype=torch.float32, device=q.device)
    f = _fn("quant_attention", "gf_quant_decode", _DECODE_ARGS, defines)
    table, rows, rot, neighbours = (None, 0, 0, 0) if fused is None else fused
    f32 = _F32[q.dtype]
    _ok(f(x, stride, f32, _p(codes), fp8, _p(scales), _ints(block_table, (B, W), "block_table"), W, W,
          _ints(lengths, (B,), "lengths"), pages, _p(out), B, nh, nkv, page, int(span), float(scale),
          int(fused is not None), table, rows, rot, int(neighbours), sms, _p(scratch), 4 * words, _stream()),
        "quant_cache.decode")
    return out


def decode(q: torch.Tensor, nh: int, cache, block_table: torch.Tensor, lengths: torch.Tensor, scale: float,
           window: int = 0) -> torch.Tensor:
    """Attention of one new token a request, the last of its ``lengths[b]`` tokens, over its cache:
    ``[B, nh * head size]`` in ``q``'s type (bf16 or fp32).  ``q [B, >= nh * head size]`` is rotated and the
    new token's keys and values are in the cache already.  ``window``: the mask as ``ops.mask_span`` gives
    it.  A request without a token gets zeros."""
    return _decode(q, nh, _cache(cache), block_table, lengths, scale, window)


def step(qkv: torch.Tensor, nh: int, table, cache, block_table: torch.Tensor, lengths: torch.Tensor,
         scale: float, window: int = 0, *, neighbours: bool = False) -> torch.Tensor:
    """What a decode step does to a layer's cache: row ``b`` of ``qkv [B, (nh + 2 kv heads) * head size]`` is
    the last of request ``b``'s ``lengths[b]`` tokens; q and k are rotated, k and v written (as
    :func:`write` does), and the token attends over the cache, itself among the keys (as :func:`decode`)."""
    facts = _cache(cache)
    return _decode(qkv, nh, facts, block_table, lengths, scale, window, (*_angles(table, facts[6]), neighbours))
