"""The writer on both sides of the line between one and two heads a group of lanes.  Every operation is rounded on its own, so
many tokens in one call leave the same bits as few at a time (which ``test_quant_cache_gpu.py`` holds against the
formulas)."""
import pytest
import torch

from test_quant_cache_gpu import BF16, DEV, F32, angles, qc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("nh,nkv,hd,page,rot,neighbours,T", [
    (28, 4, 128, 16, 128, False, 1052), (28, 4, 128, 16, 128, False, 1053), (14, 2, 64, 16, 32, True, 4300),
    (5, 1, 48, 5, 24, False, 11000), (7, 1, 80, 24, 0, False, 4500), (8, 4, 256, 64, 100, False, 1300),
    (2, 2, 32, 3, 2, False, 13000), (9, 3, 112, 8, 14, True, 2600)])
def test_many_tokens(dtype, kind, nh, nkv, hd, page, rot, neighbours, T):
    g = torch.Generator(device=DEV).manual_seed(T + hd)
    x = torch.randn(T, (nh + 2 * nkv) * hd, generator=g, device=DEV)
    x = (x * torch.exp(2 * torch.randn(T, 1, generator=g, device=DEV))).to(dtype)
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:T].int()
    slots[2], slots[3] = -1, pages * page                          # tokens that are not to be written
    at = torch.randint(0, 300, (T,), generator=g, device=DEV).int()
    table = angles(rot)
    whole, parts = (qc().make_cache(kind, pages, nkv, page, hd, DEV) for _ in range(2))
    q = qc().write(x, nh, table, at, slots, whole, neighbours=neighbours)
    few = [qc().write(x[i:i + 100], nh, table, at[i:i + 100], slots[i:i + 100], parts, neighbours=neighbours)
           for i in range(0, T, 100)]
    assert torch.equal(q, torch.cat(few))
    assert torch.equal(whole[0].view(torch.uint8), parts[0].view(torch.uint8)) and torch.equal(whole[1], parts[1])
