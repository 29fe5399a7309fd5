"""What the 8-bit cache's entry points hand to the library, without a GPU."""
import pytest
import torch

from ginfer_b200.ops import quant_cache as qc


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("sms", [148, 132, 7])
def test_rules_follow_the_device(monkeypatch, sms):
    """Writer and attention choose their ways by the SMs of the device that they run on."""
    calls = {}

    def function(lib, name, defines=()):
        def f(packed):
            calls[name] = packed
            return 0
        return f
    monkeypatch.setattr(qc, "_function", function)
    monkeypatch.setattr(qc, "_device", lambda codes: "cpu")
    monkeypatch.setattr(qc, "_at", lambda t, device: t.data_ptr())
    monkeypatch.setattr(qc, "_raw_stream", lambda device: 5)
    monkeypatch.setattr(qc, "_capturing", lambda: False)
    monkeypatch.setattr(qc, "num_sms", lambda device: sms)
    monkeypatch.setattr(qc, "error_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(qc, "_scratch", {})
    monkeypatch.setattr(qc, "_devices", {})
    cache = qc.make_cache("int8", 4, 2, 16, 64, "cpu")
    qc.write(torch.zeros(3, 8 * 64), 4, None, i32(3), i32(3), cache)
    qc.decode(torch.zeros(1, 256), 4, cache, i32(1, 20), i32(1), 1.0)
    assert qc._WRITE.unpack(calls["gf_quant_write"])[-2:] == (5, sms)
    assert qc._DECODE.unpack(calls["gf_quant_decode"])[22] == sms


def test_the_line_of_short_tables():
    """Both sides of the call know from which width on the kernel needs scratch memory."""
    import os
    import re
    from ginfer_b200.ops.build import CSRC_DIR
    with open(os.path.join(CSRC_DIR, "quant_attention.cu")) as f:
        assert int(re.search(r"\bkShortKeys = (\d+)", f.read())[1]) == qc._SHORT


def test_bytes_that_the_benchmark_counts():
    import bench
    from ginfer_b200.cache.storage import GroupLayout
    cfg = bench.SHAPES["1.5b"]
    heads, width = cfg["num_key_value_heads"], cfg["head_dim"]
    for kept in ("auto", "int8", "fp8"):
        page = GroupLayout(((heads, width),) * 2, True, 0, (0,), 0, "" if kept == "auto" else kept).bytes_per_page(16, 2)
        assert bench.kv_bytes_per_token(cfg, 3, kept=kept) * 16 == 3 * page
