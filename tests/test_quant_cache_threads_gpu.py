"""Threads that share the default stream get the results that they get alone, bit for bit: calls of two launches each, over
tables of different widths, heads and sizes (their scratch is the same buffer)."""
import threading

import pytest
import torch

from test_quant_cache_gpu import BF16, DEV, F32, i32, qc, random_cache, tables

pytestmark = pytest.mark.gpu


def test_threads_on_one_stream():
    cases = []
    for nh, nkv, hd, lens, dtype, kind in ((14, 2, 64, (9000, 10, 3000), BF16, "int8"), (28, 4, 128, (20000,), F32, "fp8"),
                                           (16, 1, 80, (5000, 4000), BF16, "fp8"), (8, 8, 64, (12000, 1, 700, 90), BF16, "int8")):
        g = torch.Generator(device=DEV).manual_seed(nh)
        t, pages, _ = tables(lens, 16, g)
        cache = random_cache(kind, pages, nkv, 16, hd, g)
        q = torch.randn(len(lens), nh * hd, generator=g, device=DEV).to(dtype)
        args = (q, nh, cache, t, i32(lens), hd ** -0.5)
        cases.append((args, qc().decode(*args).clone()))
    torch.cuda.synchronize()
    wrong, errors = [], []

    def work(args, alone):
        try:
            with torch.cuda.device(0):
                got = [qc().decode(*args) for _ in range(100)]
                wrong.extend(i for i, o in enumerate(got) if not torch.equal(o, alone))
        except Exception as e:             # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong
