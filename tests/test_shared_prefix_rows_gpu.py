"""``ops.shared_prefix.attend`` with rows of q at any address (its tolerances: see ``test_shared_prefix_gpu``)."""
import pytest
import torch

from test_shared_prefix_gpu import BF16, DEV, F32, call, check, make, way  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("counts", [[2, 1, 1], [1]])
@pytest.mark.parametrize("heads", [(6, 2, 64), (6, 2, 96)])
def test_dense_rows_at_any_address(dtype, counts, heads):
    """Exactly the heads' channels, so that the rows are dense, and a single row; whatever they start at."""
    c = make(dtype, *heads, 16, [64], [40, 17, 33][:len(counts)], counts)
    width = heads[0] * heads[2]
    dense = c["q"][:, :width].clone()
    want = call(dict(c, q=dense))
    check(want, dict(c, q=dense))
    for offset in (1, 2, 3, 4, 5, 6, 7, 8):
        buf = torch.full((dense.numel() + 16,), float("nan"), dtype=dtype, device=DEV)
        q = buf[offset:offset + dense.numel()].view_as(dense)
        q.copy_(dense)
        assert q.is_contiguous() and torch.equal(call(dict(c, q=q)), want)
