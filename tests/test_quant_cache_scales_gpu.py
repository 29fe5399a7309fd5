"""Attention over the 8-bit cache where one value row is far larger than all others and has next to no weight: the
result is the others', as exact as without that row.

Tolerances as in ``test_quant_cache_gpu.py``, with the large row left out of "the largest value seen": its score is 60
below the others', so that its share of the result is below 1e-8 of it up to a scale of 2^60 times the others'."""
import math

import pytest
import torch

from test_quant_cache_gpu import BF16, DEV, F32, attend, check_attention, i32, kept_rows, qc, random_cache, tables

pytestmark = pytest.mark.gpu


def loud_cache(kind, nh, nkv, page, hd, n, at, times, g):
    """A cache of one request and its q: channel 0 is what the scores of the row at ``at`` come from (the others have
    nothing there), and they are -60 for every head."""
    t, pages, _ = tables((n,), page, g)
    codes, scales = random_cache(kind, pages, nkv, page, hd, g)
    q = torch.randn(1, nh, hd, generator=g, device=DEV)
    q[..., 0] = 4.0
    pg, off = t[0, at // page].long(), at % page
    raw = codes.view(torch.uint8)
    raw[:, :, 0, :, 0] = 0
    raw[pg, :, 0, off] = 0
    codes[pg, :, 0, off, 0] = torch.tensor(-120.0, device=DEV).to(codes.dtype)      # (both kinds hold 120)
    scales[pg, :, off, 0] = 60.0 * math.sqrt(hd) / (4.0 * 120.0)
    scales[pg, :, off, 1] *= 2.0 ** times
    return t, (codes, scales), q.flatten(1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("times", [16, 20, 28, 60])
@pytest.mark.parametrize("nh,nkv,hd,n,at,span", [
    (6, 2, 64, 40, 0, 0), (6, 2, 64, 40, 39, 0), (14, 2, 128, 700, 0, 0), (14, 2, 128, 700, 333, 0),
    (14, 2, 128, 700, 31, 700 - 31),              # alone in the first tile that the window reaches
    (16, 1, 80, 500, 250, 0), (4, 1, 256, 300, 15, 300 - 15), (7, 1, 128, 9000, 4500, 0)])
def test_large_values_without_weight(dtype, kind, times, nh, nkv, hd, n, at, span):
    g = torch.Generator(device=DEV).manual_seed(n + at)
    t, cache, q = loud_cache(kind, nh, nkv, 16, hd, n, at, times, g)
    q = q.to(dtype)
    got = qc().decode(q, nh, cache, t, i32([n]), hd ** -0.5, span)
    want, _ = attend(cache, t, (n,), q, nh, hd ** -0.5, span)
    others = kept_rows(cache, t, 0, n)[1]
    others[at] = 0.0
    check_attention(got, want, others.abs().max().view(1, 1), dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("times", [20, 60])
@pytest.mark.parametrize("nh,nkv,hd,n,at", [(6, 2, 64, 40, 7), (14, 2, 128, 700, 0), (14, 2, 128, 700, 650), (16, 1, 80, 500, 250)])
def test_large_values_that_one_head_sees(dtype, kind, times, nh, nkv, hd, n, at):
    """Heads that share keys and values: to every other one the large row is all there is (its score is 60 above the
    others'), and the rest of them do as well as without it."""
    g = torch.Generator(device=DEV).manual_seed(n + at)
    t, cache, q = loud_cache(kind, nh, nkv, 16, hd, n, at, times, g)
    q = q.view(1, nh, hd)
    q[:, ::2, 0] = -4.0
    q = q.flatten(1).to(dtype)
    got = qc().decode(q, nh, cache, t, i32([n]), hd ** -0.5).view(1, nh, hd)
    want, _ = attend(cache, t, (n,), q, nh, hd ** -0.5)
    want = want.view(1, nh, hd)
    values = kept_rows(cache, t, 0, n)[1]
    check_attention(got[:, ::2], want[:, ::2], values[at].abs().max().view(1, 1, 1), dtype)
    values[at] = 0.0
    check_attention(got[:, 1::2], want[:, 1::2], values.abs().max().view(1, 1, 1), dtype)
