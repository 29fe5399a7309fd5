"""A paged key-value cache of 8 bits (``csrc/quant_cache.cu``, ``csrc/quant_attention.cu``): writing a
step's keys and values, reading them back, and attention of single new tokens over it.

A *cache* is the pair ``(codes, scales)``: ``codes [pages, kv heads, 2, page, head size]`` in int8 or
float8_e4m3fn (keys, then values) and ``scales [pages, kv heads, page, 2]`` fp32, both contiguous.  A row
(the keys or the values of one token and head) has one scale:

    ``scale = max(amax |x| * (1/Q), 2^-126)``, ``code = round_to_even(x * (1/scale))``, ``value = code * scale``

with ``Q`` 127 or 448; a row with an infinity or a NaN reads back as NaN.  A token's *slot* is ``page number
* page + place in the page``; ``block_table [B, W]`` int32 names a request's pages in order (entries behind
its length are not read), ``lengths [B]`` int32 its tokens, the new one among them.

All work goes to the current stream; nothing but scratch memory (one buffer a stream) is kept between calls.  Threads
may share a stream: a call's kernels go out together (see ``_launching``).

A call's integers and addresses reach the library as one block of 64-bit words: a decode step makes a call a
layer, and converting two dozen arguments one by one costs more than the small kernels run.
"""
from __future__ import annotations

import functools
import struct
import threading
from ctypes import c_char_p, c_int

import torch

from . import _Counter, _ok
from .build import load_library
from .gemm_bf16 import error_word, num_sms

KINDS = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
MAX_HEAD_DIM = 256
_FP8 = {torch.int8: 0, torch.float8_e4m3fn: 1}
_CODE = {torch.float32: 0, torch.bfloat16: 1}
_WRITE, _READ, _DECODE = struct.Struct("=21q"), struct.Struct("=17q"), struct.Struct("=27qd")
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_capturing = torch.cuda.is_current_stream_capturing
_int32, _float32 = torch.int32, torch.float32


def supports(head_dim: int, heads: int, kv_heads: int) -> bool:
    """Whether the kernels take these heads."""
    return head_dim % 16 == 0 and 16 <= head_dim <= MAX_HEAD_DIM and kv_heads > 0 and heads % kv_heads == 0


def make_cache(kind: str, pages: int, kv_heads: int, page: int, head_dim: int, device="cuda"):
    """An empty cache: ``kind`` ``"int8"`` or ``"fp8"``."""
    if kind not in KINDS:
        raise ValueError(f"a cache of 8 bits is 'int8' or 'fp8', not {kind!r}")
    return (torch.zeros(pages, kv_heads, 2, page, head_dim, dtype=KINDS[kind], device=device),
            torch.zeros(pages, kv_heads, page, 2, dtype=torch.float32, device=device))


# ----------------------------------------------------------------------------- arguments
_functions: dict = {}


def _function(lib: str, name: str, defines=()):
    f = _functions.get((name, defines))
    if f is None:
        f = getattr(load_library(lib, defines), name)
        f.argtypes, f.restype = [c_char_p], c_int
        _functions[name, defines] = f
    return f


def _cache(cache):
    """The checked facts of a cache: codes, scales, kind, pages, kv heads, page, head size."""
    codes, scales = cache
    fp8 = _FP8.get(codes.dtype)
    if fp8 is None:
        raise TypeError(f"codes are int8 or float8_e4m3fn, not {codes.dtype}")
    shape = codes.shape
    if len(shape) != 5 or shape[2] != 2 or not codes.is_contiguous():
        raise ValueError(f"codes are [pages, kv heads, 2, page, head size], contiguous; got {tuple(shape)}")
    pages, nkv, _, page, hd = shape
    if scales.dtype is not _float32 or scales.shape != (pages, nkv, page, 2) or not scales.is_contiguous():
        raise ValueError(f"the scales of codes {tuple(shape)} are fp32 {(pages, nkv, page, 2)}, "
                         f"contiguous; got {scales.dtype} {tuple(scales.shape)}")
    if hd % 16 or not 16 <= hd <= MAX_HEAD_DIM:
        raise ValueError(f"a cache of 8 bits takes head sizes that are a multiple of 16, at most "
                         f"{MAX_HEAD_DIM}; got {hd}")
    if pages * page >= 1 << 31:
        raise ValueError(f"{pages} pages of {page} tokens: slots are 32-bit integers")
    return codes, scales, fp8, pages, nkv, page, hd


def _elsewhere(t):
    raise RuntimeError("ginfer_b200 kernels run on a CUDA device only, the current one, where all of a call's tensors "
                       f"are; got a tensor on {t.device}")


def _device(codes) -> int:
    """The number of the device that a call runs on."""
    device = codes.get_device()
    if device < 0 or device != _current_device():
        _elsewhere(codes)
    return device


_devices: dict = {}


def _of_device(device: int):
    """(SMs, the address of the word that kernels set when a bounded wait runs out)."""
    facts = _devices.get(device)
    if facts is None:
        facts = _devices[device] = num_sms(device), error_word(device).data_ptr()
    return facts


def _at(t, device: int):
    """The address of a tensor on the call's device."""
    if t.get_device() != device:
        _elsewhere(t)
    return t.data_ptr()


def _ints(t, shape, what, device):
    if t.dtype is not _int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} is int32 {tuple(shape)}, contiguous; got {t.dtype} {tuple(t.shape)}")
    return _at(t, device)


def _code(dtype):
    code = _CODE.get(dtype)
    if code is None:
        raise TypeError(f"kernels take float32 or bfloat16 activations, not {dtype}")
    return code


def _rows(x, columns, what, device):
    """(address, stride, type) of rows."""
    if x.dim() != 2 or x.shape[1] < columns or x.stride(1) != 1:
        raise ValueError(f"{what} has rows of at least {columns} channels without gaps; got "
                         f"{tuple(x.shape)}, strides {tuple(x.stride())}")
    return _at(x, device), x.stride(0), _code(x.dtype)


def _angles(table, hd, device):
    """(address, rows, rotated channels) of a table of cosines and sines."""
    if table is None:
        return 0, 0, 0
    rot = table.shape[-1]
    if (table.dtype is not _float32 or table.dim() != 2 or not table.is_contiguous() or rot % 2 or rot > hd
            or table.shape[0] < 1):
        raise ValueError(f"the table of angles is fp32 [positions, an even number up to {hd}], contiguous; "
                         f"got {table.dtype} {tuple(table.shape)}")
    return _at(table, device), table.shape[0], rot


def _heads(nh, nkv):
    if nh < 1 or nh % nkv:
        raise ValueError(f"{nh} query heads are not a multiple of {nkv} kv heads")


# ----------------------------------------------------------------------------- the operators
def write(qkv: torch.Tensor, nh: int, table, positions: torch.Tensor, slots: torch.Tensor, cache, *,
          neighbours: bool = False) -> torch.Tensor:
    """Rows ``qkv [T, (nh + 2 kv heads) * head size]`` (bf16 or fp32) of a step: q and k are rotated by
    their token's position, k and v are put into its slot.  Returns the rotated q ``[T, nh * head size]`` in
    ``qkv``'s type; ``qkv`` stays as it is.

    ``table [positions, rot]`` fp32: cosines, then sines, of the angles of ``rot / 2`` pairs; the first
    ``rot`` channels of a head turn in pairs ``(j, j + rot/2)``, or ``(2j, 2j + 1)`` with ``neighbours``.
    ``None``: nothing turns.  ``positions``, ``slots`` int32 ``[T]``: a token whose slot is negative (or
    beyond the cache) is not written; two tokens of one call have different slots.  A position beyond the
    table takes its last row."""
    codes, scales, fp8, pages, nkv, page, hd = _cache(cache)
    _heads(nh, nkv)
    dev = _device(codes)
    x, stride, code = _rows(qkv, (nh + 2 * nkv) * hd, "qkv", dev)
    T = qkv.shape[0]
    at, rows, rot = _angles(table, hd, dev)
    q = qkv.new_empty(T, nh * hd)
    f = _function("quant_cache", "gf_quant_write")
    rc = f(_WRITE.pack(x, stride, code, T, nh, nkv, hd, at, rows, rot, neighbours,
                       _ints(positions, (T,), "positions", dev), _ints(slots, (T,), "slots", dev), q.data_ptr(),
                       codes.data_ptr(), fp8, _at(scales, dev), page, pages, _raw_stream(dev), _of_device(dev)[0]))
    _Counter.launches += 1
    if rc:
        _ok(rc, "quant_cache.write")
    return q


def _read(facts, block_table, W, lengths, first, slots, B, S, dtype, dev):
    codes, scales, fp8, pages, nkv, page, hd = facts
    shape = (2, B, S, nkv, hd) if slots == 0 else (2, S, nkv, hd)
    out = scales.new_empty(*shape) if dtype is _float32 else scales.new_empty(shape, dtype=dtype)
    rc = _function("quant_cache", "gf_quant_read")(
        _READ.pack(codes.data_ptr(), fp8, _at(scales, dev), block_table, W, lengths, first, slots, pages, B, S,
                   nkv, hd, page, out.data_ptr(), _code(dtype), _raw_stream(dev)))
    _Counter.launches += 1
    if rc:
        _ok(rc, "quant_cache.read")
    return out


def read(cache, block_table: torch.Tensor, lengths: torch.Tensor, dtype: torch.dtype, first=None
         ) -> torch.Tensor:
    """``[2, B, W * page, kv heads, head size]`` in ``dtype`` (bf16 or fp32): the keys and values of the
    tokens ``first[b] <= c < lengths[b]`` (``first`` ``None``: from the first one), zeros elsewhere."""
    facts = _cache(cache)
    _code(dtype)
    dev = _device(facts[0])
    B, W = block_table.shape
    return _read(facts, _ints(block_table, (B, W), "block_table", dev), W, _ints(lengths, (B,), "lengths", dev),
                 0 if first is None else _ints(first, (B,), "first", dev), 0, B, W * facts[5], dtype, dev)


def read_slots(cache, slots: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``[2, N, kv heads, head size]``: the keys and values in ``slots [N]``, zeros for a negative one."""
    facts = _cache(cache)
    _code(dtype)
    dev = _device(facts[0])
    N = slots.shape[0]
    if N == 0:
        return torch.empty((2, 0, facts[4], facts[6]), dtype=dtype, device=slots.device)
    return _read(facts, 0, 0, 0, 0, _ints(slots, (N,), "slots", dev), 1, N, dtype, dev)


# Where tables hold at most this many tokens the kernel needs no scratch (it has the same line: kShortKeys).
_SHORT = 256
_TWO_LAUNCHES = -100      # what the attention's entry point returns when the joining kernel went out too
_scratch: dict = {}
# Held from the choice of the scratch until the kernels that use it are in their stream: the foreign call lets other
# threads run, and between the attention kernel and the joining one another call on the stream would overwrite the parts
# (or put a larger buffer in this one's place).
_launching = threading.Lock()


def _scratch_for(words: int, device: int, stream: int) -> torch.Tensor:
    """A buffer that only this stream's calls use; a graph that is being captured keeps one of its own."""
    if _capturing():
        return torch.empty(words, dtype=torch.float32, device=device)
    buf = _scratch.get((device, stream))
    if buf is None or buf.numel() < words:
        buf = _scratch[device, stream] = torch.empty(max(words, 1 << 18), dtype=torch.float32, device=device)
    return buf


def _decode(q, nh, facts, block_table, lengths, scale, span, fused=None, out=None):
    """``fused``: ``(table of angles, neighbours)``.  ``out``: where the result goes, if not into a tensor of its own."""
    codes, scales, fp8, pages, nkv, page, hd = facts
    _heads(nh, nkv)
    dev = _device(codes)
    x, stride, code = _rows(q, nh * hd, "q", dev) if fused is None else _rows(q, (nh + 2 * nkv) * hd, "qkv", dev)
    B, W = block_table.shape
    if q.shape[0] != B:
        raise ValueError(f"{q.shape[0]} queries for {B} requests")
    table, rows, rot = (0, 0, 0) if fused is None else _angles(fused[0], hd, dev)
    if out is None:
        out = q.new_empty(B, nh * hd)
    sms, err = _of_device(dev)
    stream = _raw_stream(dev)
    words = scratch_words(B, nh, nkv, hd, sms) if W * page > _SHORT else 0
    f = _function("quant_attention", "gf_quant_decode", (f"GF_HEAD_DIM={hd}",))
    with _launching:
        scratch = _scratch_for(words, dev, stream) if words else None
        rc = f(_DECODE.pack(x, stride, code == 0, codes.data_ptr(), fp8, _at(scales, dev),
                            _ints(block_table, (B, W), "block_table", dev), W, W, _ints(lengths, (B,), "lengths", dev),
                            pages, out.data_ptr(), B, nh, nkv, page, span, fused is not None, table, rows, rot,
                            fused is not None and fused[1], sms, 0 if scratch is None else scratch.data_ptr(), 4 * words,
                            stream, err, scale))
    _Counter.launches += 2 if rc == _TWO_LAUNCHES else 1
    if rc and rc != _TWO_LAUNCHES:
        _ok(rc, "quant_cache.decode" if fused is None else "quant_cache.step")
    return out


@functools.lru_cache(maxsize=1024)
def scratch_words(B: int, nh: int, nkv: int, hd: int, sms: int) -> int:
    """32-bit words that the attention kernels are content with: two parts of an item a block (at most 8 blocks an
    SM), a head's result with its maximum and sum, and two words an item (see ``csrc/quant_attention.cu``)."""
    G = nh // nkv
    chunks = (G + 15) // 16
    rows = -(-G // chunks)
    return sms * 8 * 2 * rows * (hd + 2) + 2 * B * nkv * chunks + 4


def decode(q: torch.Tensor, nh: int, cache, block_table: torch.Tensor, lengths: torch.Tensor, scale: float,
           window: int = 0) -> torch.Tensor:
    """Attention of one new token a request, the last of its ``lengths[b]`` tokens, over its cache:
    ``[B, nh * head size]`` in ``q``'s type (bf16 or fp32).  ``q [B, >= nh * head size]`` is rotated and the
    new token's keys and values are in the cache already.  ``window``: the mask as ``ops.mask_span`` gives
    it.  A request without a token gets zeros.

    The products on the tensor cores take q and a key's weight (its ``p`` times its values' scale) in 11 bits, with an
    fp32 q in 22; a weight that is small beside the heaviest is off by at most 2^-25 of it, whatever the scales.  Scores,
    maxima and sums are 32-bit; a key whose ``p`` is below 2^-119 counts as nothing."""
    return _decode(q, nh, _cache(cache), block_table, lengths, scale, window)


def step(qkv: torch.Tensor, nh: int, table, cache, block_table: torch.Tensor, lengths: torch.Tensor,
         scale: float, window: int = 0, *, neighbours: bool = False) -> torch.Tensor:
    """What a decode step does to a layer's cache, in one call: row ``b`` of ``qkv [B, (nh + 2 kv heads) *
    head size]`` is the last of request ``b``'s ``lengths[b]`` tokens; q and k are rotated, k and v written (as
    :func:`write` does: not where the table has no page of the cache for it, an entry outside the cache or a length beyond
    ``W * page``), and the token attends over the cache, itself among the keys (as :func:`decode`)."""
    return _decode(qkv, nh, _cache(cache), block_table, lengths, scale, window, (table, neighbours))


# ----------------------------------------------------------------------------- a layer's attention
# Tokens that a step's portions read back at a time: their requests are taken together while the longest of them times
# their number stays below this (a dense copy of 32,768 tokens of 4 heads of 128 takes 67 MB).
READ_AT_ONCE = 32768


def portion_pages(starts, counts, page: int, span: int, W: int, capturing: bool = False) -> list[int]:
    """Pages that the portions' tokens see, from the first one's first key (without a window: from the request's) to the
    last one: portion ``i`` is the tokens ``starts[i] .. starts[i] + counts[i] - 1``.  ``capturing``: the most that there are
    wherever the portions start, in tables of ``W`` pages."""
    if capturing:
        return [W if span <= 0 else min(W, (span + n - 3) // page + 2) for n in counts]
    return [-(-(s + n) // page) - (max(0, s - span + 1) // page if span > 0 else 0) for s, n in zip(starts, counts)]


def read_back_bytes(kv_heads: int, head_dim: int, itemsize: int, page: int, longest: int, portion: int, window: int = 0
                    ) -> int:
    """The most memory that a layer's portions take for keys and values read back (the next layer's take the same):
    requests of up to ``longest`` tokens, portions of up to ``portion``."""
    tokens = -(-longest // page) * page
    if window:
        tokens = min(tokens, portion_pages([0], [portion], page, window, tokens // page, capturing=True)[0] * page)
    return 2 * max(READ_AT_ONCE, tokens) * kv_heads * head_dim * itemsize


def portion_groups(pages_of: list[int], page: int) -> list[tuple[int, int]]:
    """Runs ``[i, j)`` of neighbouring requests whose dense copies (``pages_of`` pages each) fit READ_AT_ONCE together;
    a longer request is alone."""
    groups, i = [], 0
    while i < len(pages_of):
        j, widest = i + 1, pages_of[i]
        while j < len(pages_of) and (j + 1 - i) * max(widest, pages_of[j]) * page <= READ_AT_ONCE:
            widest = max(widest, pages_of[j])
            j += 1
        groups.append((i, j))
        i = j
    return groups


def attention(qkv: torch.Tensor, nh: int, table, cache, block_table: torch.Tensor, ctx, scale: float, span: int,
              slots) -> torch.Tensor:
    """A step's attention over a layer's cache: ``qkv [T, (nh + 2 kv heads) * head size]`` unrotated, ``slots [T]``
    where the new keys and values go (``None``: they are not written, the cache is another layer's).  Single tokens
    attend over the codes; prompt portions read what they see back and take the kernels of an unquantised cache, so a
    portion sees the keys and values that the tokens after it see: in fp32 the same numbers, in bf16 rounded to the 8 bits
    of that type, which the codes' values are not when single tokens read them.  Returns ``[T, nh * head size]``."""
    from . import attention_bf16, paged_attention_simt
    codes, page, hd = cache[0], cache[0].shape[3], cache[0].shape[4]
    nkv = codes.shape[1]
    if ctx.decode_only and slots is not None:
        return step(qkv, nh, table, cache, block_table, ctx.kv_lens, scale, span)
    q = write(qkv, nh, table, ctx.positions, torch.full_like(ctx.positions, -1) if slots is None else slots, cache)
    if ctx.decode_only:
        return decode(q, nh, cache, block_table, ctx.kv_lens, scale, span)
    # single tokens first (as the scheduler orders them), the portions behind them
    B, q_lens, q_starts, nd = ctx.num_seqs, ctx.q_lens_host, ctx.q_starts_host, 0
    while nd < B and q_lens[nd] == 1:
        nd += 1
    out = torch.empty_like(q)
    if nd:
        _decode(q[:nd], nh, _cache(cache), block_table[:nd], ctx.kv_lens[:nd], scale, span, out=out[:nd])
    cu, W = ctx.cu_seqlens_q, block_table.shape[1]
    # (a captured step is replayed with other starts)
    pages_of = portion_pages(q_starts[nd:], q_lens[nd:], page, span, W, ctx.capturing)
    # what the groups' calls take besides the cache is the same for all of the step's layers with this mask (a graph
    # works it out itself)
    same = ("read back", page, span, W, _capturing())
    groups = ctx.extras.get(same)
    if groups is None:
        groups = ctx.extras[same] = []
        first = below = None
        row = nd
        if span:
            # the first key that each portion's first token sees
            p = ctx.positions[cu[nd:B].long()]
            first = (p - (span - 1)).clamp(min=0) if span > 0 else p // -span * -span
        if span > 0:
            below = first // page            # pages that it does not see any more: nothing of them is read back
        for i, j in portion_groups(pages_of, page):
            wide, n, b0, b1 = max(pages_of[i:j]), j - i, nd + i, nd + j
            rows = sum(q_lens[b0:b1])
            at = torch.arange(wide, dtype=_int32, device=q.device)
            lens, low, columns, pos = ctx.kv_lens[b0:b1], None if first is None else first[i:j], None, None
            seq = ctx.seq_of_token[row:row + rows] - b0 if qkv.dtype is _float32 else None
            if seq is not None:
                pos = ctx.positions[row:row + rows]
            if below is not None:            # (positions are counted from the first page that is read back)
                gone = below[i:j] * page
                lens, low, columns = lens - gone, low - gone, (below[i:j, None] + at).clamp_(max=W - 1).long()
                pos = None if seq is None else pos - gone[seq.long()]
            own = torch.arange(n * wide, dtype=_int32, device=q.device).view(n, wide)
            groups.append((b0, b1, row, rows, wide, columns, lens, low, own, cu[b0:b1 + 1], seq, pos, max(q_lens[b0:b1])))
            row += rows
    for b0, b1, row, rows, wide, columns, lens, low, own, cu_own, seq, pos, most in groups:
        n = b1 - b0
        seen = block_table[b0:b1, :wide].contiguous() if columns is None else block_table[b0:b1].gather(1, columns)
        pages = read(cache, seen, lens, qkv.dtype, low).view(2, n * wide, page, nkv, hd)
        if qkv.dtype is _float32:
            out[row:row + rows] = paged_attention_simt(q[row:row + rows], pages, own, seq, pos, nh, nkv, hd, scale, span,
                                                       page)
        else:
            args = (q, pages, own, cu_own, lens, n, most, nh, nkv, hd, scale, span, page)
            if most < attention_bf16.TC_MIN_QUERY_ROWS or attention_bf16.prefill_tc(*args, out=out) is None:
                attention_bf16.prefill(*args, out=out)
            del args
        del pages                            # (the next group's take their place)
    return out
