"""Which way a call of ``ops.shared_prefix.attend`` goes where requests are many or prefixes short, by the launches that it counts, and
that its result is the definition's there."""
import pytest

from test_shared_prefix_gpu import BF16, F32, call, check, make
from ginfer_b200.ops import _Counter

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, heads, batch, prefix, own, launches", [
    (BF16, (14, 2, 64), 100, 60, 70, 1), (BF16, (14, 2, 64), 300, 60, 70, 2), (BF16, (28, 4, 128), 60, 100, 200, 1),
    (BF16, (28, 4, 128), 90, 100, 200, 2), (BF16, (40, 8, 128), 200, 50, 60, 2), (F32, (14, 2, 64), 100, 60, 70, 1),
    (F32, (14, 2, 64), 300, 60, 70, 2), (BF16, (28, 4, 128), 64, 400, 1000, 2), (BF16, (28, 4, 128), 64, 2000, 1000, 3),
    (BF16, (28, 4, 128), 4, 16000, 3000, 3), (BF16, (8, 4, 256), 16, 4000, 700, 3)])
def test_ways_by_size(dtype, heads, batch, prefix, own, launches):
    """One launch while a few blocks an SM do, runs behind that; a prefix read once where reading it for each is much."""
    c = make(dtype, *heads, 16, [prefix], [1 + (b * 131) % own for b in range(batch - 1)] + [own])
    before = _Counter.launches
    got = call(c)
    assert _Counter.launches - before == launches
    check(got, c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(8, 2, 64), (40, 8, 128), (16, 4, 96)])
def test_many_rows_of_short_prefixes(dtype, heads):
    """A prefix of a tile or two with many rows, read once: its items are starts, mostly, and have SMs enough."""
    c = make(dtype, *heads, 16, [74], [5 + (b * 37) % 200 for b in range(200)], [1 + b % 5 for b in range(200)])
    check(call(c, max_q_len=5), c)
