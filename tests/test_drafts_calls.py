"""What ``ops.drafts.verify`` refuses and hands to the library, without a GPU."""
import pytest
import torch

from ginfer_b200.ops import drafts


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(drafts, "_function", lambda lib, name: lambda packed: got.append((lib, name, packed)) or 0)
    monkeypatch.setattr(drafts, "_device", lambda t: "cpu")
    monkeypatch.setattr(drafts, "_at", lambda t, device: t.data_ptr())
    monkeypatch.setattr(drafts, "_raw_stream", lambda device: 5)
    monkeypatch.setattr(drafts, "_of_device", lambda device: (148, 0))
    monkeypatch.setattr(drafts, "_scratch_for", lambda size, device, stream: torch.empty(size, dtype=torch.uint8))
    return got


def good(**changed):
    c = dict(logits=torch.zeros(7, 50), tokens=torch.zeros(7, dtype=torch.int32), cu_rows=torch.tensor([0, 3, 7]).int(),
             temperature=torch.ones(2), u=torch.zeros(7), draft_logits=torch.zeros(7, 50))
    return {**c, **changed}


def test_what_is_served(calls):
    for c in (good(), good(draft_logits=None), good(logits=torch.zeros(7, 60)[:, 3:53]),
              good(logits=torch.zeros(7, 50).bfloat16(), draft_logits=torch.zeros(7, 50).bfloat16())):
        accepted, following = drafts.verify(**c)
        assert accepted.shape == following.shape == (2,) and accepted.dtype == following.dtype == torch.int32
    assert len(calls) == 4


@pytest.mark.parametrize("changed,error", [
    (dict(logits=torch.zeros(7)), ValueError), (dict(logits=torch.zeros(7, 0)), ValueError),
    (dict(logits=torch.zeros(7, 50).half()), TypeError), (dict(logits=torch.zeros(50, 7).t()), ValueError),
    (dict(tokens=torch.zeros(6, dtype=torch.int32)), ValueError), (dict(tokens=torch.zeros(7, dtype=torch.int64)), ValueError),
    (dict(tokens=torch.zeros(14, dtype=torch.int32)[::2]), ValueError), (dict(cu_rows=torch.tensor([0, 7]).int()), ValueError),
    (dict(cu_rows=torch.tensor([0, 3, 7])), ValueError), (dict(temperature=torch.ones(2).double()), ValueError),
    (dict(u=torch.zeros(6)), ValueError), (dict(u=torch.zeros(7).bfloat16()), ValueError),
    (dict(draft_logits=torch.zeros(5, 50)), ValueError), (dict(draft_logits=torch.zeros(7, 49)), ValueError),
    (dict(draft_logits=torch.zeros(7, 50).bfloat16()), TypeError), (dict(draft_logits=torch.zeros(50, 7).t()), ValueError)])
def test_refusals(calls, changed, error):
    with pytest.raises(error):
        drafts.verify(**good(**changed))
    assert not calls


def test_the_pieces_of_a_row():
    """Both sides of the call know how many there are."""
    import os
    import re
    from ginfer_b200.ops.build import CSRC_DIR
    with open(os.path.join(CSRC_DIR, "drafts.cu")) as f:
        assert int(re.search(r"\bkPiece = (\d+)", f.read())[1]) == drafts.PIECE


def test_a_device_is_needed():
    with pytest.raises(RuntimeError, match="CUDA device"):
        drafts.verify(**good())
