"""What the 8-bit cache's entry points refuse, without a GPU."""
import pytest
import torch

from ginfer_b200.ops import quant_cache as qc


def cache(kind="int8", pages=4, nkv=2, page=16, hd=64):
    return qc.make_cache(kind, pages, nkv, page, hd, "cpu")


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_make_cache():
    codes, scales = cache("fp8")
    assert codes.shape == (4, 2, 2, 16, 64) and codes.dtype == torch.float8_e4m3fn
    assert scales.shape == (4, 2, 16, 2) and scales.dtype == torch.float32
    with pytest.raises(ValueError, match="'int8' or 'fp8'"):
        cache("int4")


@pytest.mark.parametrize("change,error,text", [
    (lambda c, s: (c.float(), s), TypeError, "int8 or float8_e4m3fn"),
    (lambda c, s: (c[:, :, 0], s), ValueError, "codes are"),
    (lambda c, s: (c.transpose(3, 4), s), ValueError, "codes are"),
    (lambda c, s: (c, s.half()), ValueError, "scales"),
    (lambda c, s: (c, s[:, :, :8]), ValueError, "scales"),
    (lambda c, s: (c[..., :40].contiguous(), s), ValueError, "multiple of 16"),
    (lambda c, s: (c[..., :0].contiguous(), s), ValueError, "multiple of 16")])
def test_caches_that_do_not_fit(change, error, text):
    bad = change(*cache())
    calls = [lambda: qc.write(torch.zeros(1, 8 * 64), 4, None, i32(1), i32(1), bad),
             lambda: qc.read(bad, i32(1, 2), i32(1), torch.float32),
             lambda: qc.read_slots(bad, i32(1), torch.float32),
             lambda: qc.decode(torch.zeros(1, 256), 4, bad, i32(1, 2), i32(1), 1.0),
             lambda: qc.step(torch.zeros(1, 8 * 64), 4, None, bad, i32(1, 2), i32(1), 1.0)]
    for call in calls:
        with pytest.raises(error, match=text):
            call()


def test_tensors_on_the_host_are_refused():
    c = cache()
    for call in (lambda: qc.write(torch.zeros(1, 8 * 64), 4, None, i32(1), i32(1), c),
                 lambda: qc.read(c, i32(1, 2), i32(1), torch.float32),
                 lambda: qc.read_slots(c, i32(1), torch.float32),
                 lambda: qc.decode(torch.zeros(1, 256), 4, c, i32(1, 2), i32(1), 1.0),
                 lambda: qc.step(torch.zeros(1, 8 * 64), 4, None, c, i32(1, 2), i32(1), 1.0)):
        with pytest.raises(RuntimeError, match="CUDA device only"):
            call()


def test_heads():
    assert qc.supports(64, 14, 2) and qc.supports(256, 4, 4) and qc.supports(16, 1, 1)
    assert not qc.supports(72, 4, 2) and not qc.supports(272, 4, 2) and not qc.supports(64, 5, 2)
    with pytest.raises(ValueError, match="multiple of 2 kv heads"):
        qc.write(torch.zeros(1, 7 * 64), 3, None, i32(1), i32(1), cache())
    with pytest.raises(ValueError, match="multiple of 2 kv heads"):
        qc.decode(torch.zeros(1, 192), 3, cache(), i32(1, 2), i32(1), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("call,error,text", [
    (lambda c, z: qc.write(z(1, 7 * 64), 4, None, i32(1).cuda(), i32(1).cuda(), c), ValueError, "at least 512"),
    (lambda c, z: qc.write(z(1, 16 * 64)[:, ::2], 4, None, i32(1).cuda(), i32(1).cuda(), c), ValueError, "without gaps"),
    (lambda c, z: qc.write(z(1, 8 * 64).half(), 4, None, i32(1).cuda(), i32(1).cuda(), c), TypeError, "bfloat16"),
    (lambda c, z: qc.write(z(2, 8 * 64), 4, None, i32(1).cuda(), i32(2).cuda(), c), ValueError, "positions"),
    (lambda c, z: qc.write(z(2, 8 * 64), 4, None, i32(2).cuda(), i32(2).cuda().long(), c), ValueError, "slots"),
    (lambda c, z: qc.write(z(1, 8 * 64), 4, z(9, 66), i32(1).cuda(), i32(1).cuda(), c), ValueError, "table of angles"),
    (lambda c, z: qc.write(z(1, 8 * 64), 4, z(9, 31), i32(1).cuda(), i32(1).cuda(), c), ValueError, "table of angles"),
    (lambda c, z: qc.write(z(1, 8 * 64), 4, z(0, 64), i32(1).cuda(), i32(1).cuda(), c), ValueError, "table of angles"),
    (lambda c, z: qc.read(c, i32(2, 3).cuda(), i32(3).cuda(), torch.float32), ValueError, "lengths"),
    (lambda c, z: qc.read(c, i32(2, 6).cuda()[:, ::2], i32(2).cuda(), torch.float32), ValueError, "block_table"),
    (lambda c, z: qc.read(c, i32(2, 3).cuda(), i32(2).cuda(), torch.float16), TypeError, "bfloat16"),
    (lambda c, z: qc.decode(z(2, 256), 4, c, i32(3, 2).cuda(), i32(3).cuda(), 1.0), ValueError, "2 queries for 3"),
    (lambda c, z: qc.decode(z(3, 255), 4, c, i32(3, 2).cuda(), i32(3).cuda(), 1.0), ValueError, "at least 256"),
    (lambda c, z: qc.step(z(3, 511), 4, None, c, i32(3, 2).cuda(), i32(3).cuda(), 1.0), ValueError, "at least 512")])
def test_arguments_that_do_not_fit(call, error, text):
    with pytest.raises(error, match=text):
        call(qc.make_cache("int8", 4, 2, 16, 64, "cuda"), lambda *s: torch.zeros(*s, device="cuda"))
