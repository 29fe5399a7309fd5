"""``ops.quant_cache.attention``, a step's attention over a layer's 8-bit cache, against the formulas in 64 bits: single
tokens, portions of prompts and both together, with sliding windows and chunks, where the step writes the cache and where
it belongs to another layer.

Tolerances.  Single tokens: those of ``test_quant_cache_gpu.py``, with the q that the writer gives (rounded to the
activations' type) where portions stand beside them.  Portions see the rows as they read back in the activations' type.
In bfloat16: half a unit of the result, and weights rounded to 8 bits, 2^-9 of the largest value seen; twice that, since their
sum is of unrounded ones.  In 32 bits: 2e-5 of the largest value seen."""
import pytest
import torch

from test_quant_cache_gpu import BF16, DEV, F32, angles, check_attention, i32, kept_rows, qc, random_cache, rotated, tables

pytestmark = pytest.mark.gpu


def context(starts, counts, dtype, capturing=False):
    from ginfer_b200.parts.base import StepContext
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    T, B = cu[-1], len(counts)
    pos = [s + i for s, n in zip(starts, counts) for i in range(n)]
    req = [b for b, n in enumerate(counts) for _ in range(n)]
    lens = [s + n for s, n in zip(starts, counts)]
    return StepContext(num_tokens=T, num_seqs=B, dtype=dtype, device=torch.device(DEV), token_ids=i32([0] * T),
                       positions=i32(pos), seq_of_token=i32(req), cu_seqlens_q=i32(cu), kv_lens=i32(lens),
                       slot_ids=i32(range(B)), logit_rows=i32([]), q_lens_host=list(counts), q_starts_host=list(starts),
                       max_q_len=max(counts), max_kv_len=max(lens), decode_only=max(counts) == 1, capturing=capturing)


def attend_rows(q, k, v, starts, counts, span, scale):
    """q [T, heads, hd], k and v a request [n, kv heads, hd], all in 64 bits: (out, the largest value a row sees)."""
    out, top, at = torch.zeros_like(q), torch.zeros(len(q), 1, 1, dtype=torch.float64, device=DEV), 0
    for b, (s, n) in enumerate(zip(starts, counts)):
        p = torch.arange(s, s + n, device=DEV)[:, None]
        c = torch.arange(len(k[b]), device=DEV)
        seen = c <= p
        if span > 0:
            seen &= p - c < span
        elif span < 0:
            seen &= c >= p // -span * -span
        G = q.shape[1] // k[b].shape[1]
        scores = torch.einsum("thd,chd->thc", q[at:at + n], k[b].repeat_interleave(G, 1)) * scale
        w = torch.softmax(scores.masked_fill(~seen[:, None], float("-inf")), -1)
        out[at:at + n] = torch.einsum("thc,chd->thd", w, v[b].repeat_interleave(G, 1))
        top[at:at + n] = (v[b].abs().amax((1, 2)) * seen).amax(-1)[:, None, None]
        at += n
    return out.flatten(1), top[:, 0]


STEPS = [  # starts, tokens of the requests
    ((300, 0, 17, 64), (1, 1, 1, 1)), ((0, 40), (37, 100)), ((500, 31, 0, 200), (1, 1, 90, 70)), ((1000,), (129,)),
    ((0, 130, 700), (1, 5, 64)), ((15, 16, 33, 2), (1, 2, 3, 200))]


HEADS = [(14, 2, 64, 16), (28, 4, 128, 16), (9, 1, 80, 24), (4, 2, 64, 8)]       # heads, kv heads, head size, page
SPANS = [0, 1, 50, 300, -48]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("writes,capturing", [(True, False), (False, False), (True, True)])
@pytest.mark.parametrize("span", SPANS)
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attention(dtype, writes, capturing, span, step):
    starts, counts = STEPS[step]
    # (every step and mask with two of the head layouts or kinds, not with all)
    turn = step + SPANS.index(span)
    (nh, nkv, hd, page), kind = HEADS[(turn + capturing) % len(HEADS)], ("int8", "fp8")[(turn // 4 + writes) % 2]
    g = torch.Generator(device=DEV).manual_seed(sum(starts) + hd)
    lens = [s + n for s, n in zip(starts, counts)]
    t, pages, _ = tables(lens, page, g)
    t = torch.cat([t, torch.full((len(lens), 3), -1, dtype=torch.int32, device=DEV)], 1)       # (wider than the lengths)
    if span > 0:                                   # pages that no token of the step sees are another's by now
        for b, s in enumerate(starts):
            t[b, :max(0, s - span + 1) // page] = -1
    cache = random_cache(kind, pages, nkv, page, hd, g)
    table, scale = angles(hd, max(lens)), hd ** -0.5
    x = (1.5 * torch.randn(sum(counts), (nh + 2 * nkv) * hd, generator=g, device=DEV)).to(dtype)
    ctx = context(starts, counts, dtype, capturing)
    slots = (t[ctx.seq_of_token.long(), ctx.positions.long() // page].long() * page + ctx.positions % page).int()
    apart = cache[0].clone(), cache[1].clone()
    got = qc().attention(x, nh, table, cache, t, ctx, scale, span, slots if writes else None)
    q = qc().write(x, nh, table, ctx.positions, slots if writes else torch.full_like(slots, -1), apart)
    assert torch.equal(cache[0].view(torch.uint8), apart[0].view(torch.uint8)) and torch.equal(cache[1], apart[1])
    assert got.shape == (len(x), nh * hd) and got.dtype == dtype
    rows = [kept_rows(apart, t.clamp(min=0), b, n) for b, n in enumerate(lens)]
    if ctx.decode_only and writes:                 # (q rotated and not rounded to its type)
        q = rotated(x.double().view(len(x), -1, hd)[:, :nh], table, ctx.positions.long(), False)
    q = q.double().view(len(x), nh, hd)
    want, top = attend_rows(q, [r[0] for r in rows], [r[1] for r in rows], starts, counts, span, scale)
    seen = [r.float().to(dtype).double() for r in rows]
    read, read_top = attend_rows(q, [r[0] for r in seen], [r[1] for r in seen], starts, counts, span, scale)
    # (single tokens in front are read from the codes)
    front = 0
    while front < len(counts) and counts[front] == 1:
        front += 1
    check_attention(got[:front], want[:front], top[:front], dtype)
    lim = 2.0 ** -8 * (read.abs() + read_top) if dtype == BF16 else 2e-5 * read_top + 0 * read
    assert torch.isfinite(got).all() and ((got.double() - read).abs() <= lim)[front:].all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("capturing", [False, True])
def test_memory_of_a_window(dtype, capturing):
    """A portion far into a long prompt takes memory for what its window sees, not for the prompt."""
    nh, nkv, hd, page, start, n, span = 28, 4, 128, 16, 20000, 200, 1024
    g = torch.Generator(device=DEV).manual_seed(1)
    t, pages, _ = tables((start + n,), page, g)
    t[0, :(start - span + 1) // page] = -1
    cache = random_cache("int8", pages, nkv, page, hd, g)
    x = torch.randn(n, (nh + 2 * nkv) * hd, generator=g, device=DEV).to(dtype)
    ctx = context((start,), (n,), dtype, capturing)
    slots = (t[0, ctx.positions.long() // page].long() * page + ctx.positions % page).int()
    qc().attention(x, nh, None, cache, t, ctx, hd ** -0.5, span, slots)
    torch.cuda.synchronize()
    ctx.extras.clear()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    qc().attention(x, nh, None, cache, t, ctx, hd ** -0.5, span, slots)
    took = torch.cuda.max_memory_allocated() - before
    dense = 2 * (span + n + 2 * page) * nkv * hd * x.element_size()
    rows = 2 * n * nh * hd * x.element_size()                      # q, and the result
    assert took <= 2 * rows + dense + (1 << 20), (took, dense, rows)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_memory_of_several_groups(dtype):
    """Requests that are read back one by one take the memory of one."""
    nh, nkv, hd, page, starts, counts = 14, 2, 64, 16, (20000, 17000, 19000), (70, 70, 70)
    g = torch.Generator(device=DEV).manual_seed(2)
    lens = [s + n for s, n in zip(starts, counts)]
    t, pages, _ = tables(lens, page, g)
    cache = random_cache("fp8", pages, nkv, page, hd, g)
    x = torch.randn(sum(counts), (nh + 2 * nkv) * hd, generator=g, device=DEV).to(dtype)
    ctx = context(starts, counts, dtype)
    slots = (t[ctx.seq_of_token.long(), ctx.positions.long() // page].long() * page + ctx.positions % page).int()
    qc().attention(x, nh, None, cache, t, ctx, hd ** -0.5, 0, slots)
    torch.cuda.synchronize()
    ctx.extras.clear()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    qc().attention(x, nh, None, cache, t, ctx, hd ** -0.5, 0, slots)
    took = torch.cuda.max_memory_allocated() - before
    most = qc().read_back_bytes(nkv, hd, x.element_size(), page, max(lens), max(counts))
    rows = 2 * len(x) * nh * hd * x.element_size()                 # q, and the result
    assert took <= 2 * rows + most + (1 << 20), (took, most, rows)
