"""``ops.shared_prefix.attend``: every key counts once, with the weight that its value is multiplied with."""
import pytest
import torch

from test_shared_prefix_gpu import BF16, DEV, F32, call, make, way  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128), (16, 4, 96), (4, 2, 256)])
@pytest.mark.parametrize("spread", [0.1, 2.0, 8.0, None])
def test_values_that_are_all_the_same(dtype, heads, spread):
    """The mean of equal values is that value, whatever the weights and their roundings are: what is summed has to be what is
    multiplied.  The prefix is so long that a piece of it has several tiles.  (Sums in 32 bits are off by far less than half a step of bfloat16; in 32 bits by 2e-5.)"""
    c = make(dtype, *heads, 16, [20000], [40, 300, 7, 129], [2, 1, 3, 1], spread=spread or 1.0)
    value = 2.0 ** (torch.arange(heads[2], device=DEV) % 5 - 2)
    value[1::2] *= -1
    c["pages"][1] = value.to(dtype)
    if spread is None:
        # one key in 128 counts, each 2^3a times as much as the one before, a from 1/2 to 3/2 by the row: where the reference of a tile's
        # weights follows the largest score late, the last one's weight is large and no power of two
        heads_q = c["q"][:, :heads[0] * heads[2]].zero_().view(len(c["q"]), heads[0], heads[2])
        heads_q[..., 0] = torch.linspace(0.5, 1.5, heads_q[..., 0].numel(), device=DEV).view(len(c["q"]), -1)
        c["pages"][0, ..., 0] = -1000.0
        for tile in range(20000 // 128):
            at = 128 * tile + 37 * tile % 128
            c["pages"][0, c["prefix_table"][0, at // 16].long(), at % 16, :, 0] = 3.0 * tile * heads[2] ** 0.5 / 1.442695
    want = value.repeat(heads[0]).expand(len(c["q"]), -1)
    for length in (20000,) if spread else range(19000, 20000, 128):          # (a piece ends at each of its tiles once)
        c["prefix_lens"].fill_(length)
        got = call(c).float()
        if dtype is BF16:
            assert torch.equal(got, want), float((got - want).abs().max())
        else:
            assert ((got - want).abs() <= 2e-5 * want.abs()).all()
