"""``ops.drafts.verify`` where sums in 32 bits say the wrong thing, against the definition in 64 bits."""
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
