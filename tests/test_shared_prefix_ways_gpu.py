"""``ops.shared_prefix.attend`` where requests are many and prefixes short."""
import pytest

from test_shared_prefix_gpu import BF16, F32, call, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(8, 2, 64), (40, 8, 128), (16, 4, 96)])
def test_many_rows_of_short_prefixes(dtype, heads):
    """A prefix of a tile or two with many rows, read once: its items are starts, mostly, and have SMs enough."""
    c = make(dtype, *heads, 16, [74], [5 + (b * 37) % 200 for b in range(200)], [1 + b % 5 for b in range(200)])
    check(call(c, max_q_len=5), c)
