"""Calls of several threads on one stream, without a GPU: no call may choose or use the stream's scratch while another
one's kernels are on their way into the stream (the library's two launches are one call here, as slow as need be)."""
import struct
import threading
import time

import pytest
import torch

from ginfer_b200.ops import quant_cache as qc

SCRATCH = 23                       # words of the packed call in front of the scratch's address


class Library:
    """In place of the library: says who was inside when a call came."""

    def __init__(self, wait):
        self.wait, self.inside, self.meetings, self.calls = wait, {}, [], []

    def __call__(self, packed):
        call = qc._DECODE.unpack(packed)
        at, size = call[SCRATCH], call[SCRATCH + 1]
        me = threading.get_ident()
        self.meetings += [(at, other) for other in self.inside.values() if other]
        self.inside[me] = at
        time.sleep(self.wait)      # (lets the other threads run, as a foreign call does)
        self.inside[me] = 0
        self.calls.append((at, size))
        return qc._TWO_LAUNCHES


@pytest.fixture
def library(monkeypatch):
    lib = Library(0.01)
    monkeypatch.setattr(qc, "_function", lambda *a: lib)
    monkeypatch.setattr(qc, "_device", lambda codes: "cpu")
    monkeypatch.setattr(qc, "_at", lambda t, device: t.data_ptr())
    monkeypatch.setattr(qc, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(qc, "_capturing", lambda: False)
    monkeypatch.setattr(qc, "num_sms", lambda device: 148)
    monkeypatch.setattr(qc, "error_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(qc, "_scratch", {})
    monkeypatch.setattr(qc, "_devices", {})
    return lib


def test_place_of_the_scratch(library):
    cache = qc.make_cache("int8", 4, 2, 16, 64, "cpu")
    qc.decode(torch.zeros(1, 256), 4, cache, torch.zeros(1, 20, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1.0)
    buf = qc._scratch["cpu", 0]
    assert library.calls == [(buf.data_ptr(), 4 * qc.scratch_words(1, 4, 2, 64, 148))]
    assert struct.calcsize("=%dq" % SCRATCH) == 8 * SCRATCH
    # the shortest tables take none
    qc.decode(torch.zeros(1, 256), 4, cache, torch.zeros(1, 8, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1.0)
    assert library.calls[1] == (0, 0)


def test_calls_go_out_one_by_one(library):
    errors = []

    def work(heads):
        try:
            cache = qc.make_cache("int8", 4, heads, 16, 64, "cpu")
            for i in range(4):
                B = 1 + 300 * i            # (larger and larger: the buffer is replaced on the way)
                qc.decode(torch.zeros(B, 4 * heads * 64), 4 * heads, cache, torch.zeros(B, 20, dtype=torch.int32),
                          torch.zeros(B, dtype=torch.int32), 1.0)
        except Exception as e:             # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(h,)) for h in (1, 2, 8, 4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(library.calls) == 16
    assert not library.meetings            # (address, address of the call that was still under way)
