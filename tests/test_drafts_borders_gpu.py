"""``ops.drafts.verify`` where sums in 32 bits say the wrong thing, against the definition in 64 bits."""
import math

import pytest
import torch

import plain_shared_prefix as plain
from ginfer_b200.ops import drafts

pytestmark = pytest.mark.gpu
DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("draft", [3, 15, 1000])
def test_small_weights_beside_a_refused_draft(dtype, draft):
    """The draft is a look-up's and does not stay; in its part of the row lie weights that are lost beside its own, and a small u
    asks for one of them, not for the first large one behind."""
    x = torch.full((2, 6000), -float("inf"), device=DEV)
    x[:, 10:21] = 0.0
    x[:, draft] = 25.0
    x[:, 5000] = 24.0
    x = x.to(dtype)
    for u in (1e-13, 1e-11, 3e-11, 1e-10, 3e-10, 1e-9, 0.3):
        args = [x, i32([0, draft]), i32([0, 2]), torch.ones(1, device=DEV), torch.tensor([0.999, u], device=DEV)]
        accepted, following = drafts.verify(*args)
        assert ([0], following.tolist()) == (accepted.tolist(), plain.verify(*args)[1]), u


def test_the_largest_vocabulary():
    """A draft among 32 likely tokens and a flat tail of 2^28, with u a millionth below its probability and a millionth above.  (The
    likely ones stand in the first 32 pieces of the row, so that whoever adds pieces up, a lane every 32nd, adds small numbers.)"""
    V, high, n = (1 << 28) - 1, 13.0, 200
    if torch.cuda.mem_get_info()[0] < 4 << 30:
        pytest.skip("needs 4 GB")
    row = torch.zeros(V, device=DEV)
    row[777:32768:1024] = high
    high = float(row[777])
    temperature = torch.linspace(0.98, 1.02, n, device=DEV)
    p = torch.tensor([1.0 / (32.0 + (V - 32) * math.exp(-high / t)) for t in temperature.double().tolist()], dtype=torch.float64)
    assert 1e-3 < float(p.min()) and float(p.max()) < 3e-3
    tokens, cu = i32([0, 777] * n), i32(range(0, 2 * n + 1, 2))
    for off, stays in ((-1e-6, 1), (1e-6, 0)):
        u = torch.full((2 * n,), 0.0, device=DEV)
        u[::2] = (p * (1.0 + off)).float().to(DEV)
        accepted, _ = drafts.verify(row.expand(2 * n, V), tokens, cu, temperature, u)
        assert accepted.tolist() == [stays] * n, off
