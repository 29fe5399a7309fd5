"""The 8-bit key-value cache against its formulas in 64 bits: what a row is kept as, what reads it
back, and attention over it, at head layouts, page sizes, lengths and masks where it can go wrong.

Tolerances.  A kept value may differ from the formula's in 64 bits by one step of its grid, and only
where the 64-bit quotient lies within 2^-18 of the middle between two codes (the kernels' quotient is
rounded three times in 32 bits).  Attention in bfloat16: half a unit of the result (2^-8 of it where it
is a power of two), and 2^-10 of the largest value seen for weights rounded to 11 bits (2^-12 each) and scores off by 2^-12.
Attention in 32 bits: 2e-5 of the largest value seen, as the other 32-bit kernels."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LIMIT = {"int8": 127.0, "fp8": 448.0}
TYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
BF16, F32 = torch.bfloat16, torch.float32


def qc():
    from ginfer_b200.ops import quant_cache
    return quant_cache


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def angles(rot, rows=300):
    if not rot:
        return None
    f = 1e4 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
    a = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float().to(DEV)


def rotated(x, table, at, neighbours):
    """x [T, heads, hd] in 64 bits."""
    if table is None:
        return x
    rot = table.shape[1]
    c, s = table[at].double()[:, None].chunk(2, -1)
    out = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if neighbours else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, v = a * c - b * s, a * s + b * c
    if neighbours:
        out[..., 0:rot:2], out[..., 1:rot:2] = u, v
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = u, v
    return out


def grid(y, kind):
    """The distance between codes at y (64 bits, in units of the scale)."""
    if kind == "int8":
        return torch.ones_like(y)
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    return torch.exp2(e - 3)


def check_kept(got, x, kind, dtype):
    """Values read back in ``dtype`` against rows x (64 bits)."""
    unit = (x.abs().amax(-1, keepdim=True) / LIMIT[kind]).clamp(min=2.0 ** -126)
    y = x / unit
    g = grid(y, kind)
    want = torch.round(y / g) * g
    off = (y / g - torch.round(y / g)).abs()
    slack = 2.0 ** -20 if dtype == F32 else 2.0 ** -8
    fine = (got.double() - want * unit).abs() <= slack * (want * unit).abs() + 1e-37
    close = (off - 0.5).abs() < 2.0 ** -18 * (1 + (y / g).abs())
    near = (got.double() - want * unit).abs() <= g * unit * (1 + 2 * slack) + slack * (want * unit).abs()
    bad = ~(fine | (close & near))
    assert not bad.any(), (int(bad.sum()), x[bad][:4], got[bad][:4], (want * unit)[bad][:4])


def random_cache(kind, pages, nkv, page, hd, g):
    codes, scales = qc().make_cache(kind, pages, nkv, page, hd, DEV)
    raw = 40.0 * torch.randn(codes.shape, generator=g, device=DEV)
    codes.copy_(torch.round(raw.clamp(-127, 127)) if kind == "int8" else (2.5 * raw).clamp(-448, 448))
    scales.copy_(torch.exp(0.5 * torch.randn(scales.shape, generator=g, device=DEV)) / (40 if kind == "int8" else 100))
    return codes, scales


def tables(lens, page, g, spare=3):
    """Block table with -1 behind every length, pages in random order."""
    used = [-(-n // page) for n in lens]
    perm = torch.randperm(sum(used) + spare, generator=g, device=DEV)
    t = torch.full((len(lens), max(1, max(used))), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(used):
        t[b, :n] = perm[at:at + n].int()
        at += n
    return t, sum(used) + spare, perm[at:]


def kept_rows(cache, t, b, n):
    """Keys and values [2, n, nkv, hd] of request b in 64 bits."""
    codes, scales = cache
    page = codes.shape[3]
    pages = t[b, :-(-n // page)].long()
    c = codes.view(torch.uint8)[pages].view(codes.dtype).float().double()
    c = c * scales[pages].double().transpose(-1, -2).unsqueeze(-1)
    return c.permute(2, 0, 3, 1, 4).flatten(1, 2)[:, :n]


def first_key(n, span):
    p = n - 1
    return max(0, p - span + 1) if span > 0 else p // -span * -span if span < 0 else 0


def attend(cache, t, lens, q, nh, scale, span=0):
    """(out [B, nh * hd], the largest value that each row sees) in 64 bits."""
    hd = cache[0].shape[-1]
    nkv = cache[0].shape[1]
    out = torch.zeros(len(lens), nh * hd, dtype=torch.float64, device=DEV)
    top = torch.zeros(len(lens), 1, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        if n:
            k, v = kept_rows(cache, t, b, n)[:, first_key(n, span):].repeat_interleave(nh // nkv, 2)
            w = torch.softmax(torch.einsum("hd,chd->hc", q[b, :nh * hd].double().view(nh, hd), k) * scale, -1)
            out[b] = torch.einsum("hc,chd->hd", w, v).flatten()
            top[b] = v.abs().max()
    return out, top


def check_attention(got, want, top, dtype):
    d = (got.double() - want).abs()
    lim = 2.0 ** -8 * want.abs() + 2.0 ** -10 * top if dtype == BF16 else 2e-5 * top
    assert torch.isfinite(got).all()
    assert (d <= lim + 1e-30).all(), (float((d - lim).max()), float(d.max()), float(top.max()))


# ------------------------------------------------------------------------------------------- write
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("nh,nkv,hd,page,rot,neighbours,T", [
    (14, 2, 64, 16, 64, False, 1), (3, 3, 16, 1, 16, True, 7), (5, 1, 48, 5, 24, False, 33),
    (12, 2, 128, 16, 64, True, 100), (1, 1, 80, 24, 0, False, 19), (8, 4, 256, 64, 256, False, 130),
    (6, 2, 112, 8, 14, True, 65), (28, 4, 128, 16, 128, False, 700), (2, 2, 32, 3, 2, False, 11),
    (4, 2, 96, 16, 6, True, 12), (10, 5, 192, 7, 100, False, 21)])
def test_write(dtype, kind, nh, nkv, hd, page, rot, neighbours, T):
    g = torch.Generator(device=DEV).manual_seed(T + hd)
    x = torch.randn(T, (nh + 2 * nkv) * hd, generator=g, device=DEV)
    x *= torch.exp(2 * torch.randn(T, 1, generator=g, device=DEV))
    x = x.to(dtype)
    orig = x.clone()
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:T].int()
    if T > 4:
        slots[2], slots[3] = -1, pages * page                  # tokens that are not to be written
    at = torch.randint(0, 300, (T,), generator=g, device=DEV).int()
    table = angles(rot)
    codes, scales = qc().make_cache(kind, pages, nkv, page, hd, DEV)
    codes.view(torch.uint8).fill_(0x55)
    scales.fill_(-7.0)
    q = qc().write(x, nh, table, at, slots, (codes, scales), neighbours=neighbours)
    assert torch.equal(x, orig) and q.dtype == dtype and q.shape == (T, nh * hd)
    rows = x.double().view(T, nh + 2 * nkv, hd)
    qk = rotated(rows[:, :nh + nkv], table, at.long(), neighbours)
    tol = dict(atol=1e-6 * float(rows.abs().max()), rtol=1e-6) if dtype == F32 else dict(atol=1e-6, rtol=2.0 ** -8)
    torch.testing.assert_close(q.double(), qk[:, :nh].flatten(1), **tol)
    there = (slots >= 0) & (slots < pages * page)
    for out in (BF16, F32):
        got = qc().read_slots((codes, scales), slots.where(there, -1), out)
        assert not got[:, ~there].any()
        check_kept(got[:, there], torch.stack([qk[there][:, nh:], rows[there][:, nh + nkv:]]), kind, out)
    # nothing else was written
    free = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    free[slots[there].long()] = False
    flat = codes.view(torch.uint8).permute(0, 3, 1, 2, 4).reshape(pages * page, -1)
    assert (flat[free] == 0x55).all()
    assert (scales.permute(0, 2, 1, 3).reshape(pages * page, -1)[free] == -7.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_write_odd_rows(dtype, kind):
    """Rows of zeros, of the type's largest and smallest numbers, with infinities and NaN; views that start at an
    odd address and have an odd stride."""
    nh, nkv, hd, page, T = 2, 2, 64, 16, 9
    wide = torch.zeros(T, (nh + 2 * nkv) * hd + 3, device=DEV, dtype=dtype)
    x = wide[:, 1:1 + (nh + 2 * nkv) * hd]
    g = torch.Generator(device=DEV).manual_seed(3)
    x.copy_(torch.randn(x.shape, generator=g, device=DEV))
    big, small = torch.finfo(dtype).max, 2.0 ** -130
    k = x.unflatten(1, (-1, hd))[:, nh:]
    k[0] = 0.0
    k[1] = big
    k[1, :, ::2] = -big
    k[2] = small
    k[3, 1, 5] = math.inf
    k[4, 2, 63] = -math.inf
    k[5, 0, 0] = math.nan
    k[6, :, 7] = 3e4
    cache = qc().make_cache(kind, 2, nkv, page, hd, DEV)
    slots = i32(range(5, 5 + T))
    qc().write(x, nh, None, i32([0] * T), slots, cache)
    got = qc().read_slots(cache, slots, F32)
    rows = x.double().unflatten(1, (-1, hd))
    want = torch.stack([rows[:, nh:nh + nkv], rows[:, nh + nkv:]])
    fine = torch.isfinite(want).all(-1)
    assert fine.sum() == fine.numel() - 3
    assert got[~fine].isnan().all()
    check_kept(got[fine], want[fine], kind, F32)
    assert not got[:, 0].any()


# ------------------------------------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("nkv,hd,page,lens,first", [
    (2, 64, 16, (1,), None), (1, 16, 1, (5, 0, 3), None), (4, 128, 16, (100, 33, 700), (0, 5, 640)),
    (5, 80, 7, (50, 49, 7, 0), (49, 49, 8, 0)), (3, 256, 64, (64, 65), None), (2, 48, 5, (31,), (30,))])
def test_read(dtype, kind, nkv, hd, page, lens, first):
    g = torch.Generator(device=DEV).manual_seed(len(lens))
    t, pages, _ = tables(lens, page, g)
    cache = random_cache(kind, pages, nkv, page, hd, g)
    got = qc().read(cache, t, i32(lens), dtype, first=None if first is None else i32(first))
    assert got.shape == (2, len(lens), t.shape[1] * page, nkv, hd) and got.dtype == dtype
    for b, n in enumerate(lens):
        low = min(n, first[b]) if first else 0
        want = kept_rows(cache, t, b, n) if n else got.new_zeros(2, 0, nkv, hd).double()
        # one rounding of the product to 32 bits and one to the result's type
        torch.testing.assert_close(got[:, b, low:n].double(), want[:, low:], atol=0,
                                   rtol=2.0 ** -23 if dtype == F32 else 2.0 ** -8)
        assert not got[:, b, :low].any() and not got[:, b, n:].any()


# ------------------------------------------------------------------------------------------- attention
SHAPES = [  # heads, kv heads, head size, page, lengths
    (14, 2, 64, 16, (300,)), (7, 1, 64, 16, (1, 0, 2, 16, 17, 15)), (28, 4, 128, 16, (1000, 33, 0, 64)),
    (8, 8, 64, 8, (129, 5)), (9, 1, 80, 24, (77, 500)), (16, 4, 96, 5, (61, 4, 5)), (4, 2, 256, 64, (700, 64, 65)),
    (20, 1, 64, 16, (513, 100)), (40, 1, 128, 32, (99,)), (3, 1, 16, 1, (40, 3)), (6, 3, 48, 7, (100, 0)),
    (5, 5, 112, 16, (31, 200)), (12, 2, 192, 16, (130,)), (2, 1, 32, 128, (1000,)), (32, 2, 64, 4, (70, 71))]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("nh,nkv,hd,page,lens", SHAPES)
def test_decode(dtype, kind, nh, nkv, hd, page, lens):
    g = torch.Generator(device=DEV).manual_seed(nh)
    t, pages, free = tables(lens, page, g)
    cache = random_cache(kind, pages, nkv, page, hd, g)
    # what no request holds is no number: pages that nobody owns and places behind a length
    cache[0].view(torch.uint8)[free] = 0x7f if kind == "fp8" else 0x80
    cache[1][free] = math.nan
    for b, n in enumerate(lens):
        if n % page:
            cache[0].view(torch.uint8)[t[b, n // page].long(), :, :, n % page:] = 0xff
            cache[1][t[b, n // page].long(), :, n % page:] = math.inf
    q = (2.0 * torch.randn(len(lens), (nh + 2) * hd, generator=g, device=DEV)).to(dtype)
    for span in (0, 1, 13, 64, -48):
        got = qc().decode(q, nh, cache, t, i32(lens), hd ** -0.5, span)
        assert got.dtype == dtype and got.shape == (len(lens), nh * hd)
        want, top = attend(cache, t, lens, q, nh, hd ** -0.5, span)
        check_attention(got, want, top, dtype)
        assert torch.equal(got, qc().decode(q, nh, cache, t, i32(lens), hd ** -0.5, span))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("nh,nkv,hd,page,lens", [
    (14, 2, 64, 16, (20000,)), (28, 4, 128, 16, (9000, 10, 0, 3000, 1)), (8, 8, 64, 24, (4000, 7000)),
    (6, 1, 128, 8, tuple(range(1, 200, 3))), (20, 1, 80, 16, (5000, 1)), (2, 2, 128, 64, (30000, 29999)),
    (14, 2, 64, 16, tuple(64 + 37 * i % 900 for i in range(300)))])
def test_decode_long_and_ragged(dtype, kind, nh, nkv, hd, page, lens):
    g = torch.Generator(device=DEV).manual_seed(len(lens))
    t, pages, _ = tables(lens, page, g)
    cache = random_cache(kind, pages, nkv, page, hd, g)
    q = (2.0 * torch.randn(len(lens), nh * hd, generator=g, device=DEV)).to(dtype)
    for span in (0, 1000):
        got = qc().decode(q, nh, cache, t, i32(lens), hd ** -0.5, span)
        check_attention(got, *attend(cache, t, lens, q, nh, hd ** -0.5, span), dtype)
        assert torch.equal(got, qc().decode(q, nh, cache, t, i32(lens), hd ** -0.5, span))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("hd,n", [(64, 40), (128, 700)])
def test_decode_scales_of_every_size(dtype, kind, hd, n):
    """Values that are zero where the weight is (a row's scale is 2^-126 then), scales that differ by 2^40, queries
    of very different heads, scores far apart."""
    nh, nkv, page = 6, 2, 16
    g = torch.Generator(device=DEV).manual_seed(n)
    t, pages, _ = tables((n,), page, g)
    base = random_cache(kind, pages, nkv, page, hd, g)
    q = torch.randn(1, nh, hd, generator=g, device=DEV)
    q *= torch.tensor([1e-20, 1e-3, 1.0, 5.0, 40.0, 1.0], device=DEV)[None, :, None]
    q[:, 5] = 0.0
    q[:, 4, ::2] *= 1e-6
    q = q.flatten(1).to(dtype)
    lens = i32([n])
    cache = (base[0].clone(), base[1].clone())
    at = t[0].long()
    # the values of half of the tokens are zero, as the writer leaves them
    cache[0].view(torch.uint8)[at, :, 1, ::2] = 0
    cache[1][at, :, ::2, 1] = 2.0 ** -126
    got = qc().decode(q, nh, cache, t, lens, hd ** -0.5)
    want, top = attend(cache, t, (n,), q, nh, hd ** -0.5)
    check_attention(got, want, top, dtype)
    # value scales from 2^-60 to 2^-20 of one: each head's output is held against what that head's
    # weights give the largest value's neighbours, so small values beside large ones may vanish
    cache = (base[0].clone(), base[1].clone())
    e = torch.randint(-60, -20, cache[1][..., 1].shape, generator=g, device=DEV).double()
    cache[1][..., 1] = torch.exp2(e).float()
    got = qc().decode(q, nh, cache, t, lens, hd ** -0.5)
    want, top = attend(cache, t, (n,), q, nh, hd ** -0.5)
    check_attention(got, want, top, dtype)
    # all values small
    cache[1][..., 1] = 2.0 ** -100
    got = qc().decode(q, nh, cache, t, lens, hd ** -0.5)
    check_attention(got, *attend(cache, t, (n,), q, nh, hd ** -0.5), dtype)
    # all values large
    cache[1][..., 1] = 2.0 ** 90
    got = qc().decode(q, nh, cache, t, lens, hd ** -0.5)
    check_attention(got, *attend(cache, t, (n,), q, nh, hd ** -0.5), dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_decode_what_is_no_number(dtype, kind):
    """A key or value that is no number makes the heads that see it none, and no others."""
    nh, nkv, hd, page, lens = 4, 2, 64, 16, (100, 90, 80, 2000)
    g = torch.Generator(device=DEV).manual_seed(1)
    t, pages, _ = tables(lens, page, g)
    cache = random_cache(kind, pages, nkv, page, hd, g)
    q = torch.randn(4, nh * hd, generator=g, device=DEV).to(dtype)
    cache[1][t[0, 2].long(), 0, 3, 0] = math.nan         # a key of request 0's first kv head
    cache[1][t[1, 5].long(), 1, 9, 1] = math.nan         # a value of request 1's second
    cache[1][t[3, 0].long(), 1, 0, 1] = math.nan         # request 3's first value, out of the window
    got = qc().decode(q, nh, cache, t, i32(lens), hd ** -0.5, 1000).view(4, nkv, -1)
    assert got[0, 0].isnan().all() and got[1, 1].isnan().all()
    assert torch.isfinite(got[0, 1]).all() and torch.isfinite(got[1, 0]).all() and torch.isfinite(got[2:]).all()
    got = qc().decode(q, nh, cache, t, i32(lens), hd ** -0.5).view(4, nkv, -1)
    assert got[3, 1].isnan().all() and torch.isfinite(got[3, 0]).all()
    q[2, 5] = math.nan                                   # a query: its own head
    got = qc().decode(q, nh, cache, t, i32(lens), hd ** -0.5).view(4, nh, hd)
    assert got[2, 0].isnan().all() and torch.isfinite(got[2, 1:]).all()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_offsets_past_32_bits(kind):
    """Pages whose codes lie more than 4 GB into the cache."""
    nh, nkv, hd, page = 8, 8, 128, 64
    pages = (9 << 29) // (nkv * 2 * page * hd)
    g = torch.Generator(device=DEV).manual_seed(2)
    cache = qc().make_cache(kind, pages, nkv, page, hd, DEV)
    assert cache[0].numel() > 1 << 32
    t = i32([[pages - 1, 1, pages - 3], [0, pages - 2, -1]])
    lens = (3 * page - 5, page + 9)
    T = sum(lens)
    x = torch.randn(T, (nh + 2 * nkv) * hd, generator=g, device=DEV).to(BF16)
    pos = torch.cat([torch.arange(n, device=DEV) for n in lens])
    req = torch.cat([torch.full((n,), b, device=DEV) for b, n in enumerate(lens)])
    slots = (t[req, pos // page].long() * page + pos % page).int()
    q = qc().write(x, nh, None, pos.int(), slots, cache)
    rows = x.double().view(T, -1, hd)
    check_kept(qc().read_slots(cache, slots, F32), torch.stack([rows[:, nh:nh + nkv], rows[:, nh + nkv:]]), kind, F32)
    dense = qc().read(cache, t, i32(lens), F32)
    assert torch.equal(dense[:, 0, :lens[0]], qc().read_slots(cache, slots[:lens[0]], F32))
    last = q[[lens[0] - 1, T - 1]].contiguous()
    check_attention(qc().decode(last, nh, cache, t, i32(lens), hd ** -0.5),
                    *attend(cache, t, lens, last, nh, hd ** -0.5), BF16)


# ------------------------------------------------------------------------------------------- step
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("rot,neighbours,span", [(1.0, False, 0), (0.5, True, 0), (0, False, 40), (0.5, False, -64),
                                                 (1.0, True, 1)])
@pytest.mark.parametrize("nh,nkv,hd,page,lens", SHAPES + [(12, 2, 128, 16, (3000, 1, 0, 17, 16, 257))])
def test_step(dtype, kind, rot, neighbours, span, nh, nkv, hd, page, lens):
    rot = int(rot * hd) // 2 * 2
    g = torch.Generator(device=DEV).manual_seed(hd)
    t, pages, _ = tables(lens, page, g)
    cache = random_cache(kind, pages, nkv, page, hd, g)
    table = angles(rot, max(lens) + 1)
    x = (1.5 * torch.randn(len(lens), (nh + 2 * nkv) * hd, generator=g, device=DEV)).to(dtype)
    n = torch.tensor(lens, device=DEV)
    last = (n - 1).clamp(min=0)
    slots = t.long().gather(1, (last // page)[:, None])[:, 0] * page + last % page
    slots = torch.where(n > 0, slots, -1).int()
    apart = (cache[0].clone(), cache[1].clone())
    got = qc().step(x, nh, table, cache, t, i32(lens), hd ** -0.5, span, neighbours=neighbours)
    # the cache holds what the writer alone leaves there, bit for bit
    qc().write(x, nh, table, last.int(), slots, apart, neighbours=neighbours)
    assert torch.equal(cache[0].view(torch.uint8), apart[0].view(torch.uint8)) and torch.equal(cache[1], apart[1])
    q = rotated(x.double().view(len(lens), -1, hd)[:, :nh], table, last, neighbours).flatten(1)
    want, top = attend(apart, t, lens, q, nh, hd ** -0.5, span)
    assert got.dtype == dtype
    check_attention(got, want, top, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("nh,nkv,hd,page,lens", [
    (14, 2, 64, 16, (300, 0, 1, 2000)), (28, 4, 128, 16, (1000, 33, 0, 64)), (8, 8, 64, 24, (129, 5)),
    (9, 1, 80, 24, (77, 500)), (4, 2, 256, 64, (700, 64, 65)), (12, 2, 128, 16, tuple(range(0, 280, 7))),
    (40, 1, 128, 8, (99, 3000))])
def test_step_in_wide_tables(dtype, kind, nh, nkv, hd, page, lens):
    """Tables that are far wider than the lengths (the work is then shared out in equal runs)."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    t, pages, _ = tables(lens, page, g)
    wide = torch.full((len(lens), 40000 // page), -1, dtype=torch.int32, device=DEV)
    wide[:, :t.shape[1]] = t
    cache = random_cache(kind, pages, nkv, page, hd, g)
    table = angles(hd, max(lens) + 1)
    x = (1.5 * torch.randn(len(lens), (nh + 2 * nkv) * hd, generator=g, device=DEV)).to(dtype)
    last = (torch.tensor(lens, device=DEV) - 1).clamp(min=0)
    for span in (0, 100):
        got = qc().step(x, nh, table, cache, wide, i32(lens), hd ** -0.5, span)
        q = rotated(x.double().view(len(lens), -1, hd)[:, :nh], table, last, False).flatten(1)
        check_attention(got, *attend(cache, t, lens, q, nh, hd ** -0.5, span), dtype)
        assert torch.equal(got, qc().step(x, nh, table, cache, wide, i32(lens), hd ** -0.5, span))
    # a value that is no number, in the last request's first page: its first head's queries, and no others
    cache[1][t[-1, 0].long(), 0, 0, 1] = math.nan
    got = qc().step(x, nh, table, cache, wide, i32(lens), hd ** -0.5).view(len(lens), nkv, -1)
    assert got[-1, 0].isnan().all() and torch.isfinite(got[:-1]).all() and torch.isfinite(got[-1, 1:]).all()


# ------------------------------------------------------------------------------------------- use
def test_streams_and_graphs():
    """On a side stream, and replayed from a graph after the lengths, the queries and the cache have changed."""
    nh, nkv, hd, page, B, W = 14, 2, 64, 16, 5, 40
    g = torch.Generator(device=DEV).manual_seed(9)
    t = torch.randperm(B * W, generator=g, device=DEV).int().view(B, W)
    cache = random_cache("int8", B * W, nkv, page, hd, g)
    q = torch.randn(B, nh * hd, generator=g, device=DEV).to(BF16)
    n = i32([640, 1, 0, 77, 300])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qc().decode(q, nh, cache, t, n, hd ** -0.5)
    side.synchronize()
    check_attention(got, *attend(cache, t, n.tolist(), q, nh, hd ** -0.5), BF16)
    x = torch.randn(B, (nh + 2 * nkv) * hd, generator=g, device=DEV).to(BF16)
    table = angles(hd, W * page)
    qc().step(x, nh, table, cache, t, n, hd ** -0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qc().step(x, nh, table, cache, t, n, hd ** -0.5)
        dense = qc().read(cache, t, n, BF16)
    for lens in ([640, 1, 0, 77, 300], [2, 640, 333, 0, 16], [600, 601, 602, 603, 604]):
        x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        n.copy_(i32(lens))
        graph.replay()
        once = out.clone(), dense.clone()
        graph.replay()
        assert torch.equal(out, once[0]) and torch.equal(dense, once[1])
        last = (n.long() - 1).clamp(min=0)
        qr = rotated(x.double().view(B, -1, hd)[:, :nh], table, last, False).flatten(1)
        check_attention(out, *attend(cache, t, lens, qr, nh, hd ** -0.5), BF16)


def test_nothing_to_do():
    cache = qc().make_cache("fp8", 3, 2, 16, 64, DEV)
    none = i32([])
    assert qc().write(torch.zeros(0, 6 * 64, device=DEV), 2, None, none, none, cache).shape == (0, 128)
    assert qc().read(cache, torch.zeros(0, 4, dtype=torch.int32, device=DEV), none, F32).shape == (2, 0, 64, 2, 64)
    assert qc().read(cache, torch.zeros(2, 0, dtype=torch.int32, device=DEV), i32([0, 0]), BF16).numel() == 0
    assert qc().read_slots(cache, none, F32).shape == (2, 0, 2, 64)
    no_pages = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    q = torch.ones(2, 128, device=DEV)
    assert not qc().decode(q, 2, cache, no_pages, i32([0, 0]), 1.0).any()
    assert qc().decode(q[:0], 2, cache, no_pages[:0], none, 1.0).shape == (0, 128)
