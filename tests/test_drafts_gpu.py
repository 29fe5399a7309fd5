"""``ops.drafts.verify`` against its definition in 64 bits: the numbers have to be the same."""
import pytest
import torch

import plain_shared_prefix as plain
from ginfer_b200 import ops
from ginfer_b200.ops import drafts

pytestmark = pytest.mark.gpu
DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def make(dtype, V, counts, drafter, heat=1.0, seed=0, flat=False):
    """counts: drafts a request; -1: a request without rows.  Drafts are likely ones, so that many stay."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = [n + 1 for n in counts]
    cu = [sum(rows[:b]) for b in range(len(rows) + 1)]
    R, B = cu[-1], len(rows)
    x = 2.0 * torch.randn(R, V, generator=g, device=DEV)
    if not flat:
        x.scatter_(1, torch.randint(V, (R, 5), generator=g, device=DEV), 9.0)
    x = x.to(dtype)
    tokens = torch.randint(V, (R,), generator=g, device=DEV)
    pos = torch.arange(1, R, device=DEV)
    sharp = torch.where(torch.rand(max(R - 1, 0), generator=g, device=DEV) < 0.7, x[:-1].float().argmax(1), tokens[1:])
    tokens[pos] = sharp
    y = None
    if drafter:
        y = (x.float() + 0.7 * torch.randn(x.shape, generator=g, device=DEV)).to(dtype)
    t = torch.full((B,), heat, device=DEV) * (0.7 + 0.6 * torch.rand(B, generator=g, device=DEV))
    return [x, tokens.int(), i32(cu), t, torch.rand(R, generator=g, device=DEV), y]


def check(args):
    got = drafts.verify(*args)
    want = plain.verify(*args)
    assert got[0].dtype == got[1].dtype == torch.int32
    assert got[0].tolist() == want[0], (got[0].tolist(), want[0])
    assert got[1].tolist() == want[1], (got[1].tolist(), want[1])


COUNTS = [[0], [1], [4], [8], [0, 3, 1, 5, 2], [4] * 16, [2, -1, 0, 3, -1], [40], [1] * 130]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("V", [1, 2, 7, 257, 4095, 32003])
def test_verify(dtype, drafter, counts, V):
    check(make(dtype, V, counts, drafter, seed=V + len(counts)))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("V", [151936, 152064, 262145])
@pytest.mark.parametrize("flat", [False, True])
def test_large_vocabularies(dtype, drafter, V, flat):
    for seed in range(3):
        check(make(dtype, V, [4, 0, 2, 7], drafter, seed=seed, flat=flat))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("heat", [1e-30, 1e-3, 0.3, 5.0, 1e6, 1e30, INF])
def test_temperatures(dtype, drafter, heat):
    check(make(dtype, 5003, [3, 5, 0, 1, 4, 4], drafter, heat, seed=5))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
def test_greedy(dtype, drafter):
    """Among sampled requests; equal logits: the lowest index."""
    args = make(dtype, 3001, [4, 2, 0, 5, 3, 8, 1], drafter, seed=2)
    args[3][::2] = torch.tensor([0.0, -1.0, -INF, NAN], device=DEV)
    check(args)
    x = args[0]
    best = x.float().argmax(1)
    at = torch.arange(len(x), device=DEV)
    x[at, (best + 11) % 3001] = x[at, best]
    check(args)
    args[1][1:] = torch.tensor([plain.best(r) for r in x[:-1]], device=DEV)
    check(args)
    assert (drafts.verify(*args)[0][0]) == 4


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
def test_random_numbers_at_their_ends(dtype, drafter):
    args = make(dtype, 2049, [3, 0, 5, 2], drafter, seed=3)
    for u in (0.0, 1.0 - 2.0 ** -24, 2.0 ** -149):
        args[4].fill_(u)
        check(args)
    args[0][:, :5] = -INF                    # (u of zero: the first token of any weight)
    args[4].zero_()
    check(args)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
def test_logits_that_are_no_numbers(dtype, drafter):
    """Masked tokens (-inf and the type's lowest value), NaN, rows of nothing, infinities."""
    args = make(dtype, 1500, [3] * 12, drafter, seed=4)
    x, y = args[0], args[5]
    low = torch.finfo(dtype).min
    for t in (x, y) if drafter else (x,):
        t[::3, 100:1400] = -INF
        t[1::5, ::2] = low
        t[2::7, ::3] = NAN
    x[4] = -INF
    x[9] = NAN
    x[12] = low
    x[16, 7] = x[16, 70] = INF
    x[21] = INF
    if drafter:
        y[3], y[8], y[14] = -INF, NAN, low
        y[20, 70] = INF
    check(args)
    args[3][::2] = 0.0
    check(args)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_drafter_that_thinks_as_the_target(dtype):
    """p = q: every draft stays."""
    args = make(dtype, 3000, [5, 3, 8], True, seed=6)
    x, cu = args[0], args[2].tolist()
    args[5] = x.clone()
    args[5][[c - 1 for c in cu[1:]]] = NAN                   # (rows that are not read)
    args[4].fill_(1.0 - 2.0 ** -24)
    check(args)
    assert drafts.verify(*args)[0].tolist() == [5, 3, 8]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
def test_drafts_outside_the_vocabulary(dtype, drafter):
    args = make(dtype, 500, [3, 2, 4], drafter, seed=7)
    args[1][2], args[1][5], args[1][8] = 500, -1, 2 ** 31 - 1
    check(args)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [3001, 3008])
def test_strides(dtype, V):
    """Rows of any distance, at any address."""
    args = make(dtype, V, [3, 1, 4], True, seed=8)
    want = [t.tolist() for t in drafts.verify(*args)]
    for gap, start in ((1, 0), (7, 3), (8, 8), (64, 1), (0, 5)):
        more = list(args)
        for i in (0, 5):
            buf = torch.full((args[i].shape[0] * (V + gap) + 16,), INF, dtype=dtype, device=DEV)
            more[i] = buf[start:].as_strided(args[i].shape, (V + gap, 1)).copy_(args[i])
        assert [t.tolist() for t in drafts.verify(*more)] == want
    check(args)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_starts_that_are_none(dtype):
    """Starts beyond the rows are cut; the others' numbers stay."""
    args = make(dtype, 500, [3, 2, 4], True, seed=9)
    want = drafts.verify(*args)
    for cu in ([0, 4, 7, 1 << 30], [-9, 4, 7, 12]):
        args[2] = i32(cu)
        got = drafts.verify(*args)
        assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()
    for cu in ([0, 12, 3, 12], [12, 7, 4, 0], [50, 60, 70, 80]):
        args[2] = i32(cu)
        drafts.verify(*args)
    torch.cuda.synchronize()


def test_as_single_tokens_are_sampled():
    """Without drafts the next token is ``ops.sample``'s, but for borders that 32-bit sums meet otherwise."""
    args = make(F32, 4000, [0] * 200, False, seed=10)
    got = drafts.verify(*args)[1]
    assert (got == ops.sample(args[0], args[3], args[4])).sum() >= 199
    args[3].zero_()
    assert torch.equal(drafts.verify(*args)[1], ops.argmax(args[0]))


@pytest.mark.parametrize("drafter", [False, True])
def test_tokens_are_distributed_as_the_target_alone_would(drafter):
    """The first token of many steps of the same two distributions, drafted by q and verified, is distributed as p: the
    largest of 8 counts' distances from 20,000 p, in standard deviations, is below 5 (chance: 5e-6)."""
    n, V = 20000, 8
    g = torch.Generator(device=DEV).manual_seed(11)
    p, q = torch.randn(2, V, generator=g, device=DEV)
    x = p.expand(2 * n, V).contiguous()
    y = q.expand(2 * n, V).contiguous() if drafter else None
    tokens = torch.zeros(2 * n, dtype=torch.int32, device=DEV)
    tokens[1::2] = torch.multinomial(torch.softmax(q if drafter else torch.zeros(V, device=DEV), 0), n, True, generator=g).int()
    a, t = drafts.verify(x, tokens, i32(range(0, 2 * n + 1, 2)), torch.ones(n, device=DEV),
                         torch.rand(2 * n, generator=g, device=DEV), y)
    first = torch.where(a > 0, tokens[1::2], t)
    p = torch.softmax(p.double(), 0)
    off = (torch.bincount(first.long(), minlength=V) - n * p) / (n * p * (1 - p)).sqrt()
    assert float(off.abs().max()) < 5, off


def test_streams_and_graphs():
    args, more = make(F32, 32003, [4, 2, 7, 0], True, seed=12), make(F32, 32003, [1, 6, 3, 3], True, seed=13)
    want = [[t.tolist() for t in drafts.verify(*x)] for x in (args, more)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = drafts.verify(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert [t.tolist() for t in got] == want[0]
    graphs = []
    for x in (args, more):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, drafts.verify(*x)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, (graph, out) in zip(streams, graphs):
            for t in out:
                t.fill_(-9)
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for (_, out), w in zip(graphs, want):
            assert [t.tolist() for t in out] == w
    args[0].copy_(args[0].flip(1))
    args[4].copy_(args[4].flip(0))
    graphs[0][0].replay()
    assert [t.tolist() for t in graphs[0][1]] == list(plain.verify(*args))


def test_a_step_of_attention_head_and_verification():
    """As a step of a batch with drafts runs: attention behind a shared prefix, the head's product, verification."""
    import test_shared_prefix_gpu as sp
    counts = [1, 5, 3, 2, 4, 1]
    c = sp.make(BF16, 12, 2, 128, 16, [700], [30, 200, 64, 17, 90, 1], counts)
    h = sp.call(c, max_q_len=5)
    sp.check(h, c)
    g = torch.Generator(device=DEV).manual_seed(14)
    head = ops.Linear((0.5 * torch.randn(4000, h.shape[1], generator=g, device=DEV)).to(BF16), out_dtype=F32)
    logits = head(h)
    tokens = torch.randint(4000, (sum(counts),), generator=g, device=DEV).int()
    tokens[1:] = torch.where(torch.rand(len(tokens) - 1, generator=g, device=DEV) < 0.6, logits[:-1].argmax(1).int(), tokens[1:])
    t = torch.tensor([0.0, 0.8, 1.0, 0.0, 0.5, 1.0], device=DEV)
    check([logits, tokens, c["cu"], t, torch.rand(len(tokens), generator=g, device=DEV), None])
