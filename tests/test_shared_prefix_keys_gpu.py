"""``ops.shared_prefix.attend``: no key is left out and none counts twice.

Tolerances.  Equal scores make every weight one, sums of them are whole numbers that 32 bits hold, and a channel that some keys
have at one and the others at zero says how many of them were seen: the result is a quotient of two whole numbers, rounded
to 32 bits and to bfloat16 (2^-8 of it).  Random scores: every weight is off by 2^-8 of itself for the product with the values
in bfloat16, their sum likewise, so the result by 2^-8 of sum_c w_c |V_c| + |result|, and by 2^-8 of itself for its own rounding; 2e-5 of the
largest value for what 32 bits leave."""
import pytest
import torch

import plain_shared_prefix as plain
from test_shared_prefix_gpu import BF16, DEV, F32, call, make, way  # noqa: F401

pytestmark = pytest.mark.gpu
HEADS = [(14, 2, 64), (28, 4, 128), (16, 4, 96), (9, 1, 80), (4, 2, 256), (6, 6, 16), (10, 2, 192)]


def mark(c, each):
    """Values: of token c of a sequence channel (c / each) modulo the head size is one, the others are zero."""
    _, _, page, nkv, hd = c["pages"].shape
    c["pages"][1] = 0.0
    c["q"].zero_()
    for table, lens in ((c["prefix_table"], c["prefix_lens"]), (c["block_table"], c["lengths"])):
        for row, n in zip(table, lens.tolist()):
            at = torch.arange(n, device=DEV)
            c["pages"][1, row[at // page].long(), at % page, :, at // each % hd] = 1.0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("prefix, page", [(77, 16), (1000, 24), (4099, 16), (9001, 8), (6016, 64)])
@pytest.mark.parametrize("each", [1, 16])
def test_every_key_counts_once(dtype, heads, prefix, page, each):
    """Runs of 16 keys, the smallest tile, and every hd-th key: a lost tile is a 16 hd-th part of the channels that it has."""
    c = make(dtype, *heads, page, [prefix, 300], [1, 300, 65, 9, 1100, 33], [1, 2, 1, 1, 5, 3], groups=[0, 4, 6])
    mark(c, each)
    want, _, known = plain.attend(c["q"], c["nh"], c["pages"], c["prefix_table"], c["prefix_lens"], c["block_table"],
                                  c["lengths"], c["scale"], c["cu_groups"], c["cu"])
    err = (call(c).double() - want).abs()[known]
    assert (err <= (2.0 ** -8 if dtype is BF16 else 2.0 ** -20) * want[known]).all()


def check(got, c):
    """Against the definition, with sum_c w_c |V_c| from the definition, too."""
    facts = (c["prefix_table"], c["prefix_lens"], c["block_table"], c["lengths"], c["scale"], c["cu_groups"], c["cu"])
    want, top, known = plain.attend(c["q"], c["nh"], c["pages"], *facts)
    size, _, _ = plain.attend(c["q"], c["nh"], (c["pages"][0], c["pages"][1].abs()), *facts)
    allowed = 2e-5 * top[known, None]
    if got.dtype is BF16:
        allowed = allowed + 2.0 ** -8 * (size + 2.0 * want.abs())[known]
    err = (got.double() - want).abs()[known]
    assert (err <= allowed).all(), float((err / allowed).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("prefix, page", [(131, 16), (1500, 24), (4099, 16), (9001, 64)])
def test_random_scores(dtype, heads, prefix, page):
    c = make(dtype, *heads, page, [prefix, 300], [1, 300, 65, 9, 1100, 33], [1, 2, 1, 1, 5, 3], groups=[0, 4, 6], spread=3.0)
    check(call(c), c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cu", [[3, 1, 8, 8], [6, 0, 7, 8], [7, 2, 0, 8], [4, 4, 2, 6], [5, 6, 7, 8], [-7, 2, 3, 1 << 30]])
@pytest.mark.parametrize("hd", [64, 128, 96])
def test_rows_of_starts_that_do_not_rise(dtype, cu, hd):
    """Rows that are nobody's stay as they were, and a request that begins behind its group's first start has its result."""
    c = make(dtype, 6, 2, hd, 16, [64], [40, 17, 33], [5, 1, 2])
    c["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    out = torch.full((8, 6 * hd), 7.0, dtype=dtype, device=DEV)
    call(c, out=out)
    cut = [min(max(s, 0), 8) for s in cu]
    named = torch.zeros(8, dtype=torch.bool, device=DEV)
    for b in range(3):
        named[cut[b]:max(cut[b], cut[b + 1])] = True
    assert (out[~named] == 7.0).all()
    for b in range(3):
        s, e = cut[b], cut[b + 1]
        if s < e and cut[0] <= s and e <= cut[3]:
            one = dict(c, q=c["q"][s:e], block_table=c["block_table"][b:b + 1], lengths=c["lengths"][b:b + 1],
                       cu=torch.tensor([0, e - s], dtype=torch.int32, device=DEV))
            check(out[s:e], one)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups", [[-5, 1 << 30], [9, -9], [7, 9], [2, 1]])
def test_groups_beyond_the_requests(dtype, groups):
    """Requests are a group's by its two numbers, whatever these are."""
    c = make(dtype, 6, 2, 64, 16, [64], [40, 17, 33], [2, 1, 1])
    c["cu_groups"] = torch.tensor(groups, dtype=torch.int32, device=DEV)
    check(call(c), c)
