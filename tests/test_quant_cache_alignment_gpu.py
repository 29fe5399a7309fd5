"""Scales that start at 8 modulo 16 bytes: what lies in front of them and behind them is not theirs.

Tolerances: those of ``test_quant_cache_gpu.py``."""
import math

import pytest
import torch

from test_quant_cache_gpu import (BF16, DEV, F32, angles, attend, check_attention, i32, qc, random_cache, rotated)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("nh,nkv,hd,page,lens", [
    (14, 2, 64, 16, (300, 1)), (4, 2, 128, 16, (1,)), (9, 1, 80, 24, (77, 500)), (6, 3, 48, 7, (100, 9)),
    (4, 1, 256, 64, (700,)), (3, 1, 16, 1, (40, 3)), (7, 1, 128, 5, (9001, 2))])
def test_scales_at_eight_bytes(dtype, kind, nh, nkv, hd, page, lens):
    g = torch.Generator(device=DEV).manual_seed(hd)
    used = [-(-n // page) for n in lens]
    pages = sum(used)                              # every page of the cache is used, the first one first
    t = torch.full((len(lens), max(used)), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(used):
        t[b, :n] = torch.arange(n, device=DEV) + sum(used[:b])
    codes, plain = random_cache(kind, pages, nkv, page, hd, g)
    buf = torch.full((plain.numel() + 4,), math.nan, device=DEV)
    assert buf.data_ptr() % 16 == 0
    scales = buf[2:-2].view(plain.shape)
    scales.copy_(plain)
    cache = (codes, scales)
    q = (2.0 * torch.randn(len(lens), nh * hd, generator=g, device=DEV)).to(dtype)
    for span in (0, 13):
        got = qc().decode(q, nh, cache, t, i32(lens), hd ** -0.5, span)
        check_attention(got, *attend((codes, plain), t, lens, q, nh, hd ** -0.5, span), dtype)
    table = angles(hd, max(lens) + 1)
    x = (1.5 * torch.randn(len(lens), (nh + 2 * nkv) * hd, generator=g, device=DEV)).to(dtype)
    got = qc().step(x, nh, table, cache, t, i32(lens), hd ** -0.5)
    last = i32(lens).long() - 1
    qr = rotated(x.double().view(len(lens), -1, hd)[:, :nh], table, last, False).flatten(1)
    check_attention(got, *attend((codes, scales.clone()), t, lens, qr, nh, hd ** -0.5), dtype)
    dense = qc().read(cache, t, i32(lens), F32)
    assert torch.equal(dense, qc().read((codes, scales.clone()), t, i32(lens), F32))
    assert buf[:2].isnan().all() and buf[-2:].isnan().all()
