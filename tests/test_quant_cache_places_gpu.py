"""A decode step whose new token has no place in the cache leaves the cache as it is, as the writer does."""
import pytest
import torch

from test_quant_cache_gpu import BF16, DEV, F32, angles, attend, check_attention, i32, qc, random_cache, rotated

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("nh,nkv,hd,page,W", [(14, 2, 64, 16, 4), (6, 1, 128, 8, 400), (9, 1, 80, 24, 9)])
@pytest.mark.parametrize("where", ["no page", "behind the cache", "far behind", "longer than the table"])
def test_tokens_without_a_place(dtype, kind, nh, nkv, hd, page, W, where):
    pages = W + 2
    g = torch.Generator(device=DEV).manual_seed(W)
    t = torch.arange(2, W + 2, device=DEV, dtype=torch.int32)[None].clone()       # (pages 0 and 1 are another's)
    n = (W - 1) * page + 3                                                        # in the table's last page
    if where == "longer than the table":
        n = W * page + 1
    else:
        t[0, W - 1] = {"no page": -1, "behind the cache": pages, "far behind": 2 ** 31 - 1}[where]
    cache = random_cache(kind, pages, nkv, page, hd, g)
    before = cache[0].view(torch.uint8).clone(), cache[1].clone()
    table = angles(hd, n)
    x = torch.randn(1, (nh + 2 * nkv) * hd, generator=g, device=DEV).to(dtype)
    got = qc().step(x, nh, table, cache, t, i32([n]), hd ** -0.5)
    assert torch.isfinite(got).all()
    assert torch.equal(cache[0].view(torch.uint8), before[0]) and torch.equal(cache[1], before[1])
    # the writer, told the same place
    slot = -1 if where == "no page" else pages * page + 2
    qc().write(x, nh, table, i32([n - 1]), i32([slot]), cache)
    assert torch.equal(cache[0].view(torch.uint8), before[0]) and torch.equal(cache[1], before[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_the_others_beside_it(dtype, kind):
    """Requests whose tokens have places are served and written; a full table's last place is one."""
    nh, nkv, hd, page, W = 12, 2, 128, 16, 40
    g = torch.Generator(device=DEV).manual_seed(5)
    t = torch.randperm(3 * W, generator=g, device=DEV).int().view(3, W)
    lens = [W * page, 333, 17]
    t[1, 333 // page] = -1
    cache = random_cache(kind, 3 * W, nkv, page, hd, g)
    apart = cache[0].clone(), cache[1].clone()
    table = angles(hd, W * page)
    x = torch.randn(3, (nh + 2 * nkv) * hd, generator=g, device=DEV).to(dtype)
    got = qc().step(x, nh, table, cache, t, i32(lens), hd ** -0.5)
    last = i32(lens).long() - 1
    slots = [int(t[b, (n - 1) // page]) * page + (n - 1) % page for b, n in enumerate(lens)]
    slots[1] = -1
    qc().write(x, nh, table, last.int(), i32(slots), apart)
    assert torch.equal(cache[0].view(torch.uint8), apart[0].view(torch.uint8)) and torch.equal(cache[1], apart[1])
    q = rotated(x.double().view(3, -1, hd)[:, :nh], table, last, False).flatten(1)
    want, top = attend(apart, t.clamp(min=0), lens, q, nh, hd ** -0.5)
    check_attention(got[::2], want[::2], top[::2], dtype)
