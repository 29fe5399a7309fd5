"""What ``ops.drafts.verify`` hands to the library, word by word, and the launches that both operators count, without a GPU."""
import pytest
import torch

import test_drafts_calls
import test_shared_prefix_calls
from ginfer_b200.ops import _Counter, drafts, shared_prefix

draft_calls, prefix_calls = test_drafts_calls.calls, test_shared_prefix_calls.calls


@pytest.mark.parametrize("dtype, code", [(torch.float32, 0), (torch.bfloat16, 1)])
@pytest.mark.parametrize("drafter", [False, True])
def test_the_words_of_a_verification(draft_calls, dtype, code, drafter):
    R, V, B = 7, 5000, 2
    x, y = torch.zeros(R, V + 11, dtype=dtype)[:, 3:3 + V], torch.zeros(R, V + 5, dtype=dtype)[:, :V]
    c = test_drafts_calls.good(logits=x, draft_logits=y if drafter else None)
    accepted, following = drafts.verify(**c)
    lib, name, packed = draft_calls[-1]
    w = drafts._VERIFY.unpack(packed)
    assert (lib, name) == ("drafts", "gf_verify")
    assert w[:5] == (x.data_ptr(), V + 11, code, y.data_ptr() if drafter else 0, V + 5 if drafter else 0)
    assert w[5:9] == tuple(c[n].data_ptr() for n in ("tokens", "cu_rows", "temperature", "u"))
    assert w[9:14] == (accepted.data_ptr(), following.data_ptr(), R, V, B)
    # two numbers of 32 bits for every piece of every row of both, however the row starts
    assert w[15] >= R * 2 * -(-(V + 16 // x.itemsize - 1) // (drafts.PIECE * 4 // x.itemsize)) * 8
    assert w[16:] == (148, 5)


def test_no_call_keeps_what_another_was_given(draft_calls, monkeypatch):
    """The library's function is looked up by every call: a stand-in of one test is not another's."""
    drafts.verify(**test_drafts_calls.good())
    assert len(draft_calls) == 1
    monkeypatch.setattr(drafts, "_function", lambda lib, name: lambda packed: draft_calls.append(None) or 0)
    drafts.verify(**test_drafts_calls.good())
    assert draft_calls[1] is None


def launched(module, monkeypatch, result, call):
    monkeypatch.setattr(module, "_function", lambda lib, name, defines=(): lambda packed: result)
    if module is shared_prefix:
        monkeypatch.setattr(module, "_attend_functions", {})
    before = _Counter.launches
    try:
        call()
    except RuntimeError:
        assert result not in (0, -101, -102)
    else:
        assert result in (0, -101, -102)
    return _Counter.launches - before


def test_launches_of_a_verification(draft_calls, monkeypatch):
    none = dict(logits=torch.zeros(0, 50), tokens=torch.zeros(0, dtype=torch.int32), u=torch.zeros(0), draft_logits=None)
    for changed, result, count in (({}, 0, 2), ({}, -5, 0), ({**none, "cu_rows": torch.zeros(3, dtype=torch.int32)}, 0, 1),
                                   ({**none, "cu_rows": torch.zeros(1, dtype=torch.int32), "temperature": torch.ones(0)}, 0, 0)):
        assert launched(drafts, monkeypatch, result, lambda: drafts.verify(**test_drafts_calls.good(**changed))) == count


@pytest.mark.parametrize("result, count", [(0, 3), (-101, 1), (-102, 2), (-5, 0), (-7, 0), (700, 0)])
def test_launches_of_attention(prefix_calls, monkeypatch, result, count):
    assert launched(shared_prefix, monkeypatch, result, lambda: shared_prefix.attend(**test_shared_prefix_calls.good())) == count
