"""What ``ops.shared_prefix.attend`` hands to the library, without a GPU: rows of q start at multiples of 16 bytes, and the scale is a
number in 32 bits."""
import pytest
import torch

from test_shared_prefix_calls import calls, good, i32  # noqa: F401
from ginfer_b200.ops import shared_prefix


def handed_over(calls, q):
    """(address, row stride) of q as the library gets them."""
    B = q.shape[0]
    pages = torch.zeros(2, 9, 16, 2, 64).to(q.dtype)
    shared_prefix.attend(**good(q=q, pages=pages, block_table=i32(B, 4), lengths=i32(B)))
    return shared_prefix._ATTEND.unpack(calls[-1][2])[:2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("gap", [0, 1, 8, 64])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 4, 5, 8, 9])
def test_rows_of_q_are_aligned(calls, dtype, rows, gap, offset):  # noqa: F811
    """Dense rows and single ones, too, which are contiguous wherever they start."""
    buf = torch.zeros(rows * (256 + gap) + 16, dtype=dtype)
    q = buf[offset:].as_strided((rows, 256), (256 + gap, 1))
    at, stride = handed_over(calls, q)
    assert at % 16 == 0 and (rows == 1 or stride * q.itemsize % 16 == 0)
    if q.data_ptr() % 16 == 0 and q.stride(0) * q.itemsize % 16 == 0:
        assert (at, stride) == (q.data_ptr(), 256 + gap)                # (nothing is copied without need)


@pytest.mark.parametrize("scale", [1e39, 3e38, 1e300, float("inf"), -1.0])
def test_scales_that_32_bits_do_not_hold(calls, scale):  # noqa: F811
    """(Zero and NaN: with the other refusals.)"""
    with pytest.raises(ValueError, match="scale"):
        shared_prefix.attend(**good(scale=scale))
    assert not calls
    for fine in (1e38, 1e-30, 1):
        shared_prefix.attend(**good(scale=fine))
    assert len(calls) == 3
