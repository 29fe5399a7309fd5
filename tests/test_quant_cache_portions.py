"""What a step's portions read back of an 8-bit cache, without a GPU."""
import pytest

from ginfer_b200.ops import quant_cache as qc


@pytest.mark.parametrize("page", [1, 7, 16])
@pytest.mark.parametrize("span", [0, 1, 2, 16, 50, -48])
def test_portion_pages(page, span):
    W = 400 // page + 3
    for n in (1, 2, 15, 16, 17, 33, 64):
        most = 0
        for s in range(0, 300):
            low = max(0, s - span + 1) if span > 0 else 0
            (got,) = qc.portion_pages([s], [n], page, span, W)
            assert got == (s + n - 1) // page - low // page + 1
            most = max(most, got)
        (bound,) = qc.portion_pages([0], [n], page, span, W, capturing=True)
        assert bound >= most
        if span > 0:
            assert bound == most                   # (it is reached)
        else:
            assert bound == W
