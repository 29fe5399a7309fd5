"""Drafted tokens held against the target's probabilities (``csrc/drafts.cu``).

A request's step has the rows of its last token and of some drafted ones behind it; the target's logits of a row say what it
thinks of the next row's token.  :func:`verify` says how many of the drafts stay and draws the token behind them, so that
the tokens that a request gets are distributed as if the target alone had drawn them (``ops.sample``), one by one.

All work goes to the current stream; nothing but scratch memory is kept between calls.
"""
from __future__ import annotations

import struct

import torch

from . import _Counter, _ok
from .quant_cache import _at, _code, _device, _function, _of_device, _raw_stream
from .shared_prefix import _launching, _scratch_for

PIECE = 1024                   # the least logits of a piece of a row (the library has the same number)
_VERIFY = struct.Struct("=18q")


def _rows(x, rows, columns, what, device):
    """(address, row stride) of rows of logits."""
    strides = x.stride()
    if x.shape != (rows, columns) or (strides[1] != 1 and columns > 1):
        raise ValueError(f"{what} is [{rows}, {columns}], a row without gaps; got {tuple(x.shape)}, strides {strides}")
    return _at(x, device), strides[0]


def _vector(t, count, dtype, what, device):
    if t.dtype is not dtype or t.shape != (count,) or not t.is_contiguous():
        raise ValueError(f"{what} is {dtype} [{count}], contiguous; got {t.dtype} {tuple(t.shape)}")
    return _at(t, device)


def verify(logits: torch.Tensor, tokens: torch.Tensor, cu_rows: torch.Tensor, temperature: torch.Tensor,
           u: torch.Tensor, draft_logits=None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(accepted [B], next_token [B])``, both int32: how many of each request's drafted tokens stay, and the token that
    follows the last of them.

    ``logits [R, V]`` (fp32 or bf16; rows may have any stride): request ``b`` has the rows ``c0 = cu_rows[b] .. c1 - 1 =
    cu_rows[b + 1] - 1`` (``cu_rows [B + 1]`` int32).  ``tokens [R]`` int32: the token that each row was computed from, so that
    the drafts are ``tokens[c0 + 1 : c1]`` and row ``c0 + i`` judges the draft in ``c0 + i + 1``.  ``draft_logits [R, V]``
    of the same type: row ``c0 + i`` is what the drafter drew the draft in ``c0 + i + 1`` from (a request's last row is not
    read); ``None``: drafts of no distribution (a look-up), which the drafter is taken to have been sure of.
    ``temperature [B]`` fp32, also the drafter's.  ``u [R]`` fp32 in ``[0, 1)``: ``u[c0 + i]`` decides on the draft that row
    ``c0 + i`` judges, ``u[c1 - 1]`` draws the token behind.

    With ``p = softmax(logits / temperature)`` of the judging row and ``q`` the draft's likewise, a draft ``d`` stays if ``u
    q[d] < p[d]`` and all before it do; behind the first that does not the next token is drawn from ``max(p - q, 0)`` (from
    ``p`` without ``d`` for a look-up), behind the last draft from ``p``: the first ``j`` whose weight is above zero and at which the
    running sum reaches ``u`` times the whole.  A temperature of zero or below: a draft stays if it is the arg-max
    (the lowest index among equals), and the next token is the arg-max.

    A weight below ``2^-120`` of its row's largest counts as none, a ``u`` outside of ``[0, 1)`` as the nearest number in it
    (for the draw; a draft is compared with ``u`` as it is).  A NaN counts as ``-inf``, logits of ``+inf`` share all of a
    row's weight.  Where nothing is left of ``p - q`` the next token is drawn from ``p``, where nothing is left of that either it is
    the arg-max (0 in a row without a number).  A draft that is no index of the vocabulary does not stay.  A request without
    rows has ``(0, -1)``.  Starts rise or stay; where they do not, nothing but the results is written, and what these are is
    not said."""
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits are [rows, vocabulary]; got {tuple(logits.shape)}")
    (R, V), code = logits.shape, _code(logits.dtype)
    dev = _device(logits)
    B = temperature.shape[0]
    x, stride = _rows(logits, R, V, "logits", dev)
    y, draft_stride = 0, 0
    if draft_logits is not None:
        if draft_logits.dtype != logits.dtype:
            raise TypeError(f"the drafter's logits have the target's type {logits.dtype}, not {draft_logits.dtype}")
        y, draft_stride = _rows(draft_logits, R, V, "draft_logits", dev)
    if V >= 1 << 28 or R >= 1 << 30 or B >= 1 << 28:
        raise ValueError(f"{R} rows of {V} logits for {B} requests: fewer than 2^30 rows, 2^28 logits and requests")
    facts = (x, stride, code, y, draft_stride, _vector(tokens, R, torch.int32, "tokens", dev),
             _vector(cu_rows, B + 1, torch.int32, "cu_rows", dev),
             _vector(temperature, B, torch.float32, "temperature", dev), _vector(u, R, torch.float32, "u", dev))
    accepted, following = tokens.new_empty(B), tokens.new_empty(B)
    stream, size, sms = _raw_stream(dev), 16 * R * (V // PIECE + 2), _of_device(dev)[0]
    f = _function("drafts", "gf_verify")
    with _launching:
        scratch = _scratch_for(size, dev, stream)
        rc = f(_VERIFY.pack(*facts, accepted.data_ptr(), following.data_ptr(), R, V, B, scratch.data_ptr(), size, sms, stream))
    if rc:
        _ok(rc, "drafts.verify")
    _Counter.launches += (2 if R else 1) if B else 0
    return accepted, following
