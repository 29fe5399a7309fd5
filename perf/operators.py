"""A key-value cache of 8 bits: what writes it, what reads it back, and the attention on it.

A cached row (the keys or the values of one token and head) is held as 8-bit codes, integers or e4m3, and one
32-bit scale: ``scale = max(amax / Q, 2^-126)`` with ``Q`` 127 or 448, ``code = round(x / scale)``, and it
reads back as ``code * scale``.  ``codes [pages, kv heads, 2, page, dim]`` (keys, then values) and
``scales [pages, kv heads, page, 2]`` are paged: a request's ``c``-th token sits in page
``table[request, c // page]`` at place ``c % page``, and a slot is ``page number * page + place``.

``write``   a step's rows ``q | k | v``: q and k rotated by position (halves or neighbours, all of the head or
            its first channels), k and v put into their slots; gives the rotated q.
``read``    the tokens ``first .. length - 1`` of every request as a dense tensor, zeros elsewhere.
``decode``  one new token a request (the last of its length) over its cache, grouped heads, with or without
            a sliding window; a request without a token gives zeros.
``step``    all of that for a decode step: rotates, writes the new token and attends over the cache.

Here are the cases that these are measured on, in plain torch (32-bit, rounded once) and through the
framework's entry points, and their definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TINY = 2.0 ** -126
LIMIT = {"int8": 127.0, "fp8": 448.0}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ----------------------------------------------------------------------------- cases
def _case(op, kind, dtype, heads, kv_heads, dim, page, **more):
    return dict(op=op, kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, **more)


def listed():
    return [
        # one request's new token, where it is written by a call of its own
        dict(_case("write", "int8", "bf16", 14, 2, 64, 16, tokens=1, start=311, rot=64, neighbours=False),
             name="write-one-token"),
        # a whole step's budget of prompt tokens
        dict(_case("write", "fp8", "bf16", 28, 4, 128, 16, tokens=8192, start=0, rot=128, neighbours=False),
             name="write-prompt"),
        # the 32-bit path, a ragged portion, half of the head rotated in neighbouring pairs
        dict(_case("write", "int8", "f32", 12, 2, 128, 64, tokens=517, start=4001, rot=64, neighbours=True),
             name="write-f32-portion"),
        # short prompts read back for the attention of their next portions
        dict(_case("read", "int8", "bf16", 14, 2, 64, 16, batch=3, longest=701, window=0), name="read-short"),
        # everything a portion at the end of a long prompt attends to
        dict(_case("read", "fp8", "bf16", 28, 4, 128, 16, batch=2, longest=32768, window=0), name="read-long"),
        # a sliding window's tokens for the 32-bit path, heads of an odd size
        dict(_case("read", "fp8", "f32", 10, 5, 80, 32, batch=7, longest=3001, window=1024),
             name="read-window-f32"),
        # one chat at its beginning: latency
        dict(_case("decode", "int8", "bf16", 14, 2, 64, 16, batch=1, longest=300, window=0), name="decode-one"),
        # one request over a very long context
        dict(_case("decode", "int8", "bf16", 28, 4, 128, 16, batch=1, longest=131071, window=0),
             name="decode-long"),
        # a serving batch of ragged lengths, one request without a token (a padded row)
        dict(_case("decode", "fp8", "bf16", 28, 4, 128, 16, batch=64, longest=8192, window=0, empty=True),
             name="decode-batch"),
        # the 32-bit path with a sliding window
        dict(_case("decode", "int8", "f32", 14, 2, 64, 16, batch=8, longest=6001, window=2048),
             name="decode-f32-window"),
        # a decode step of one request
        dict(_case("step", "fp8", "bf16", 12, 2, 128, 16, batch=1, longest=1000, window=0, rot=128,
                   neighbours=False), name="step-one"),
        # a decode step of a full batch
        dict(_case("step", "int8", "bf16", 12, 2, 128, 16, batch=256, longest=4096, window=0, rot=128,
                   neighbours=False), name="step-batch"),
    ]


HEADS = ((14, 2, 64), (12, 2, 128), (28, 4, 128), (8, 8, 64), (9, 1, 80), (16, 4, 96), (40, 8, 128), (4, 2, 256),
         (20, 1, 64))


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("write", "read", "decode", "step"))
    heads, kv, dim = rng.choice(HEADS)
    kind, page = rng.choice(("int8", "fp8")), rng.choice((8, 16, 16, 24, 64))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    wide = 1 if dtype == "bf16" else 2
    rot = rng.choice((dim, dim, dim // 2, 0))
    if op == "write":
        row = (2 * heads + 4 * kv) * dim * wide
        return _case(op, kind, dtype, heads, kv, dim, page, tokens=_log(rng, 1, 8192 * 128 * 72 // row),
                     start=_log(rng, 1, 20000), rot=rot, neighbours=rng.random() < 0.5)
    row = kv * (2 * dim + 8)
    total = 120_000_000 // row // (1 if op != "read" else 2 * wide)           # cached tokens in all
    batch = min(_log(rng, 1, 256), total)
    longest = _log(rng, 1, max(1, min(131072, total // batch)))
    window = rng.choice((0, 0, _log(rng, 1, longest)))
    c = _case(op, kind, dtype, heads, kv, dim, page, batch=batch, longest=longest, window=window,
              empty=batch > 1 and rng.random() < 0.3)
    return dict(c, rot=rot, neighbours=rng.random() < 0.5) if op == "step" else c


def _lengths(case):
    """The requests' lengths: between a tenth of the longest and that, spread evenly."""
    n = [max(1, int(case["longest"] * (0.1 + 0.9 * ((1.0 - 0.6180339887498949 * b) % 1.0))))
         for b in range(case["batch"])]
    n[0] = case["longest"]
    if case.get("empty"):
        n[-1] = 0
    return n


def work(case):
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    es = DTYPES[case["dtype"]].itemsize
    if case["op"] == "write":
        T = case["tokens"]
        row = (nh + 2 * nkv) * hd * es + nh * hd * es + 2 * nkv * (hd + 4) + 2 * nkv * hd * es + 4 * case["rot"] + 8
        return {"bytes": T * row, "flops": T * (3 * (nh + nkv) * case["rot"] + 6 * nkv * hd)}
    n = [min(x, case["window"] or x) for x in _lengths(case)]
    keys, B, page = sum(n), case["batch"], case["page"]
    cache = keys * nkv * (2 * hd + 8) + 4 * sum(-(-x // page) for x in n)
    if case["op"] == "read":
        dense = B * -(-case["longest"] // page) * page
        return {"bytes": cache + 8 * B + 2 * dense * nkv * hd * es, "flops": 2 * keys * nkv * hd}
    rows = 2 * B * nh * hd * es + 4 * B
    if case["op"] == "step":
        rows += B * (2 * nkv * hd * es + 2 * nkv * (hd + 4) + 2 * nkv * hd * es + 4 * case["rot"])
    return {"bytes": cache + rows, "flops": 4 * keys * nh * hd}


# ----------------------------------------------------------------------------- inputs
def _table(case, positions):
    """Cosines, then sines, of every position's angles."""
    half = case["rot"] // 2
    if not half:
        return None
    f = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _rows(case, count, g):
    """Projections q | k | v as a layer leaves them: some channels of k stand out, tokens differ in size."""
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    x = torch.randn(count, nh + 2 * nkv, hd, generator=g, device=DEV)
    stand = 1.0 + 7.0 * (torch.rand(nkv, hd, generator=g, device=DEV) < 0.04)
    x[:, nh:nh + nkv] *= stand
    x[:, nh:] *= torch.exp(0.4 * torch.randn(count, 2 * nkv, 1, generator=g, device=DEV))
    return x.flatten(1).to(DTYPES[case["dtype"]])


@torch.no_grad()
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    nkv, hd, page = case["kv_heads"], case["dim"], case["page"]
    s = {"case": case}

    def ints(x):
        return torch.as_tensor(x, dtype=torch.int32, device=DEV)
    if case["op"] == "write":
        T = case["tokens"]
        pages = -(-T // page) + 3
        at = torch.arange(T, device=DEV)
        slots = torch.randperm(pages, generator=g, device=DEV)[at // page] * page + at % page
        if T > 8:
            slots[T // 2] = -1                                  # a row that pads the step
        s.update(qkv=_rows(case, T, g), table=_table(case, case["start"] + T), positions=ints(at + case["start"]),
                 slots=ints(slots), kept=torch.nonzero(slots >= 0)[:, 0],
                 codes=torch.zeros(pages, nkv, 2, page, hd, dtype=CODES[case["kind"]], device=DEV),
                 scales=torch.zeros(pages, nkv, page, 2, device=DEV))
        return s
    B, width = case["batch"], -(-case["longest"] // page)
    n = torch.tensor(_lengths(case), device=DEV)[torch.randperm(B, generator=g, device=DEV)]
    used = -(-n // page)
    total = int(used.sum())
    pages = total + 1
    table = torch.full((B, width), -1, dtype=torch.int64, device=DEV)
    here = torch.arange(width, device=DEV) < used[:, None]
    table[here] = torch.randperm(pages, generator=g, device=DEV)[:total]
    shape = (pages, nkv, 2, page, hd)
    if case["kind"] == "int8":
        # (in bytes from the start: the largest caches hold 300 million codes)
        codes = torch.randint(-48, 49, shape, generator=g, device=DEV, dtype=torch.int8)
        codes += torch.randint(-48, 49, shape, generator=g, device=DEV, dtype=torch.int8)
    else:
        codes = (100.0 * torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
                 ).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    unit = 1.0 / (40.0 if case["kind"] == "int8" else 100.0)
    scales = unit * torch.exp(0.5 * torch.randn(pages, nkv, page, 2, generator=g, device=DEV))
    s.update(codes=codes, scales=scales, table_of_pages=ints(table), lengths=ints(n))
    if case["op"] == "read":
        s["first"] = ints((n - case["window"]).clamp(min=0)) if case["window"] else None
    elif case["op"] == "decode":
        s["q"] = _rows(case, B, g)[:, :case["heads"] * hd].contiguous()
    else:
        last = (n - 1).clamp(min=0)
        slots = table.gather(1, (last // page)[:, None])[:, 0] * page + last % page
        s.update(qkv=_rows(case, B, g), table=_table(case, case["longest"]),
                 slots=ints(torch.where(n > 0, slots, -1)), kept=torch.nonzero(n > 0)[:, 0])
    return s


# ----------------------------------------------------------------------------- the plain form
def _rotated(x, angles, rot, neighbours):
    if not rot:
        return x
    c, s = angles[:, None, :rot // 2], angles[:, None, rot // 2:]
    if neighbours:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _quantised(x, kind):
    top = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    scale = (top * (1.0 / LIMIT[kind])).clamp(min=TINY)
    y = torch.where(fine, x * (1.0 / scale), 0.0).clamp(-LIMIT[kind], LIMIT[kind])
    codes = torch.round(y).to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)
    return codes, torch.where(fine, scale, math.nan)[..., 0]


def _put(s, k, v, kind):
    """k and v ``[tokens, kv heads, dim]`` into their slots."""
    page = s["codes"].shape[3]
    slots = s["slots"][s["kept"]].long()
    codes, scales = _quantised(torch.stack([k, v], 2)[s["kept"]], kind)
    s["codes"].view(torch.uint8)[slots // page, :, :, slots % page] = codes.view(torch.uint8)
    s["scales"][slots // page, :, slots % page] = scales


def _values(s, pages, places, seen):
    """The values kept at (pages, places) as ``[2, ..., kv heads, dim]`` in 32 bits, zeros where not seen."""
    codes = s["codes"].view(torch.uint8)[pages, :, :, places].view(s["codes"].dtype).float()
    x = codes * s["scales"][pages, :, places].unsqueeze(-1)
    return torch.where(seen[..., None, None, None], x, 0.0).movedim(-2, 0)


def _dense(s, first):
    page, table = s["codes"].shape[3], s["table_of_pages"].long().clamp(min=0)
    c = torch.arange(table.shape[1] * page, device=DEV)
    seen = (c < s["lengths"][:, None]) & (c >= first[:, None])
    return _values(s, table[:, c // page], (c % page).expand(table.shape[0], -1), seen), seen


def _attend(s, case, q):
    """q ``[batch, heads, dim]`` over its request's cache."""
    n = s["lengths"]
    first = (n - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(n)
    (k, v), seen = _dense(s, first)
    B, nkv = q.shape[0], k.shape[2]
    q = q.view(B, nkv, -1, q.shape[-1])
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * q.shape[-1] ** -0.5
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.transpose(1, 2))
    return torch.where(total > 0, out / total, 0.0).reshape(B, -1)


@torch.no_grad()
def run(s):
    case = s["case"]
    dtype, nh, op = DTYPES[case["dtype"]], case["heads"], case["op"]
    nkv, hd = case["kv_heads"], case["dim"]
    if own:
        from ginfer_b200.ops import quant_cache as qc
        cache = s["codes"], s["scales"]
        if op == "write":
            q = qc.write(s["qkv"], nh, s["table"], s["positions"], s["slots"], cache, neighbours=case["neighbours"])
            return q, qc.read_slots(cache, s["slots"], dtype)
        if op == "read":
            return qc.read(cache, s["table_of_pages"], s["lengths"], dtype, first=s["first"])
        if op == "decode":
            return qc.decode(s["q"], nh, cache, s["table_of_pages"], s["lengths"], hd ** -0.5, case["window"])
        out = qc.step(s["qkv"], nh, s["table"], cache, s["table_of_pages"], s["lengths"], hd ** -0.5,
                      case["window"], neighbours=case["neighbours"])
        return out, qc.read_slots(cache, s["slots"], dtype)
    page = s["codes"].shape[3]
    if op == "read":
        first = s["first"] if s["first"] is not None else torch.zeros_like(s["lengths"])
        return _dense(s, first)[0].to(dtype)
    if op == "decode":
        return _attend(s, case, s["q"].float().view(-1, nh, hd)).to(dtype)
    x = s["qkv"].float().view(-1, nh + 2 * nkv, hd)
    at = s["positions"] if op == "write" else (s["lengths"] - 1).clamp(min=0)
    angles = s["table"][at.long()] if case["rot"] else None
    q, k = (_rotated(t, angles, case["rot"], case["neighbours"]) for t in (x[:, :nh], x[:, nh:nh + nkv]))
    _put(s, k, x[:, nh + nkv:], case["kind"])
    slots = s["slots"].long().clamp(min=0)
    kept = _values(s, slots // page, slots % page, s["slots"] >= 0).to(dtype)
    return (q.flatten(1) if op == "write" else _attend(s, case, q)).to(dtype), kept


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _turn64(x, table, at, rot, neighbours):
    """x ``[tokens, heads, dim]`` as complex numbers, times ``cos + i sin``."""
    if not rot:
        return x
    turn = torch.complex(table[at, :rot // 2].double(), table[at, rot // 2:].double())[:, None]
    pairs = x[..., :rot].unflatten(-1, (rot // 2, 2) if neighbours else (2, rot // 2))
    pairs = pairs if neighbours else pairs.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z if neighbours else z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), x[..., rot:]], -1)


def _kept64(x, kind):
    """What a row in 64 bits reads back as."""
    unit = torch.clamp(x.abs().amax(-1, keepdim=True) / LIMIT[kind], min=TINY)
    y = x / unit
    if kind == "int8":
        return torch.round(y) * unit
    _, e = torch.frexp(y)                                # e4m3: four digits down to 2^-6, then steps of 2^-9
    grid = torch.exp2((e - 4).clamp(min=-9).double())
    return torch.round(y / grid) * grid * unit


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op, nh, nkv, hd, page = case["op"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    whole = (s["codes"], s["scales"])
    if op in ("write", "step"):
        x = s["qkv"].double().view(-1, nh + 2 * nkv, hd)
        at = s["positions"].long() if op == "write" else (s["lengths"].long() - 1).clamp(min=0)
        qk = _turn64(x[:, :nh + nkv], s["table"], at, case["rot"], case["neighbours"])
        new = _kept64(torch.stack([qk[:, nh:], x[:, nh + nkv:]]), case["kind"])
        new[:, s["slots"] < 0] = 0.0
        if op == "write":
            return qk[:, :nh].flatten(1), new
        q = qk[:, :nh]
    elif op == "decode":
        q = s["q"].double().view(-1, nh, hd)
    B, width = s["table_of_pages"].shape
    if op == "read":
        out = torch.zeros(2, B, width * page, nkv, hd, dtype=torch.float64, device=DEV)
    else:
        out = torch.zeros(B, nh * hd, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lengths"].tolist()):
        if not n:
            continue
        pages = s["table_of_pages"][b, :-(-n // page)].long()
        kv = whole[0].view(torch.uint8)[pages].view(whole[0].dtype).float().double()
        kv = kv * whole[1][pages].double().transpose(-1, -2).unsqueeze(-1)       # [pages, heads, 2, page, dim]
        kv = kv.permute(2, 0, 3, 1, 4).flatten(1, 2)[:, :n]
        low = max(0, n - case["window"]) if case["window"] else 0
        if op == "read":
            out[:, b, low:n] = kv[:, low:]
            continue
        if op == "step":
            kv[:, n - 1] = new[:, b]
        k, v = (t.repeat_interleave(nh // nkv, 1) for t in kv[:, low:])
        w = torch.softmax(torch.einsum("hd,chd->hc", q[b], k) * hd ** -0.5, -1)
        out[b] = torch.einsum("hc,chd->hd", w, v).flatten()
    return out if op != "step" else (out, new)
