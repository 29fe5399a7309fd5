"""What ``ops.shared_prefix.attend`` refuses and hands to the library, without a GPU."""
import pytest
import torch

from ginfer_b200.ops import shared_prefix


@pytest.fixture
def calls(monkeypatch):
    got = []

    def function(lib, name, defines=()):
        return lambda packed: got.append((lib, name, packed)) or 0
    monkeypatch.setattr(shared_prefix, "_function", function)
    monkeypatch.setattr(shared_prefix, "_device", lambda t: "cpu")
    monkeypatch.setattr(shared_prefix, "_at", lambda t, device: t.data_ptr())
    monkeypatch.setattr(shared_prefix, "_raw_stream", lambda device: 5)
    monkeypatch.setattr(shared_prefix, "_of_device", lambda device: (148, 0))
    monkeypatch.setattr(shared_prefix, "_scratch_bytes", lambda *sizes: 64)
    monkeypatch.setattr(shared_prefix, "_capturing", lambda: False)
    monkeypatch.setattr(shared_prefix, "_scratch", {})
    monkeypatch.setattr(shared_prefix, "_attend_functions", {})
    return got


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def good(**changed):
    c = dict(q=torch.zeros(3, 8 * 64), nh=4, pages=torch.zeros(2, 9, 16, 2, 64), prefix_table=i32(1, 5), prefix_lens=i32(1),
             block_table=i32(3, 4), lengths=i32(3), scale=0.125, cu_groups=None, cu_seqlens_q=None)
    return {**c, **changed}


def test_what_is_served(calls):
    q, pages = torch.zeros(3, 8 * 64), torch.zeros(2, 9, 16, 2, 64)
    for c in (good(), good(cu_seqlens_q=i32(4), q=torch.zeros(11, 256)), good(prefix_table=i32(2, 5), prefix_lens=i32(2), cu_groups=i32(3)),
              good(q=q.bfloat16(), pages=pages.bfloat16()), good(pages=(pages[0], pages[1].clone())),
              good(block_table=i32(3, 9)[:, 5:]), good(max_q_len=1), good(prefix_table=i32(0, 5), prefix_lens=i32(0))):
        assert shared_prefix.attend(**c).shape == (c["q"].shape[0], 256)
    assert len(calls) == 8
    out = torch.zeros(3, 256)
    assert shared_prefix.attend(**good(out=out)) is out


@pytest.mark.parametrize("changed,error", [
    (dict(pages=torch.zeros(2, 9, 16, 2, 72)), ValueError), (dict(pages=torch.zeros(2, 9, 16, 3, 64)), ValueError),
    (dict(pages=torch.zeros(2, 9, 16, 2, 272), q=torch.zeros(3, 8 * 272)), ValueError), (dict(pages=torch.zeros(2, 0, 16, 2, 64)), ValueError),
    (dict(pages=torch.zeros(2, 9, 16, 2, 64).transpose(1, 2)), ValueError), (dict(pages=torch.zeros(2, 9, 2, 64)), ValueError),
    (dict(pages=(torch.zeros(9, 16, 2, 64), torch.zeros(9, 16, 2, 32))), ValueError),
    (dict(pages=(torch.zeros(9, 16, 2, 64), torch.zeros(9, 16, 2, 64).bfloat16())), ValueError),
    (dict(q=torch.zeros(3, 255)), ValueError), (dict(q=torch.zeros(3, 512).bfloat16()), ValueError), (dict(q=torch.zeros(512, 3).t()), ValueError),
    (dict(q=torch.zeros(3, 512).half(), pages=torch.zeros(2, 9, 16, 2, 64).half()), TypeError), (dict(q=torch.zeros(2, 512)), ValueError),
    (dict(prefix_table=i32(2, 5)), ValueError), (dict(prefix_table=i32(5)), ValueError), (dict(prefix_table=i32(1, 5).long()), ValueError),
    (dict(prefix_table=i32(2, 5), prefix_lens=i32(2)), ValueError), (dict(prefix_lens=i32(1).long()), ValueError),
    (dict(block_table=i32(4, 3).t()), ValueError), (dict(block_table=i32(2, 4)), ValueError), (dict(lengths=i32(4)), ValueError),
    (dict(lengths=i32(6)[::2]), ValueError), (dict(cu_groups=i32(3)), ValueError), (dict(cu_seqlens_q=i32(3)), ValueError),
    (dict(cu_seqlens_q=i32(4).long()), ValueError), (dict(max_q_len=-1), ValueError), (dict(scale=0.0), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(out=torch.zeros(769)[1:].view(3, 256)), ValueError), (dict(pages=torch.zeros(2 * 9 * 16 * 128 + 1)[1:].view(2, 9, 16, 2, 64)), ValueError),
    (dict(out=torch.zeros(3, 257)), ValueError), (dict(out=torch.zeros(3, 256).bfloat16()), ValueError), (dict(out=torch.zeros(256, 3).t()), ValueError)])
def test_refusals(calls, changed, error):
    with pytest.raises(error):
        shared_prefix.attend(**good(**changed))
    assert not calls


def test_strides_beyond_32_bits(calls):
    """Tables' rows that far apart are refused, q's made dense; of a single row the stride says nothing."""
    far = torch.empty((1 << 32) + 512, device="meta")
    table = torch.empty((1 << 32) + 5, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        shared_prefix.attend(**good(block_table=table.as_strided((3, 4), (1 << 31, 1))))
    with pytest.raises(ValueError, match="2\\^31"):
        shared_prefix.attend(**good(prefix_table=table.as_strided((2, 5), (1 << 31, 1)), prefix_lens=i32(2), cu_groups=i32(3)))
    assert not calls
    shared_prefix.attend(**good(prefix_table=table.as_strided((1, 5), (1 << 32, 1))))
    assert shared_prefix._ATTEND.unpack(calls[-1][2])[8] == 0
    shared_prefix.attend(**good(q=far.as_strided((3, 256), (1 << 31, 1)), out=torch.zeros(3, 256)))
    assert shared_prefix._ATTEND.unpack(calls[-1][2])[1] == 256


def test_a_device_is_needed():
    with pytest.raises(RuntimeError, match="CUDA device"):
        shared_prefix.attend(**good())
