"""``ops.shared_prefix.attend`` against its definition in 64 bits.

Tolerances.  bfloat16: a weight is rounded to 8 bits for the product with the values (off by 2^-8 of itself at most, so the result by 2^-8 of the largest value
seen) and the result is rounded once (2^-8 of itself); scores and sums in 32 bits add 2e-5 of the largest value: scores of up to 32 are
off by a few 2^-24 of that.  32 bits: those 2e-5 alone."""
import threading

import pytest
import torch

import plain_shared_prefix as plain
from ginfer_b200.ops import _Counter, shared_prefix

pytestmark = pytest.mark.gpu
DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


WIDER = {"narrow": lambda c: (0, 0), "cluster": lambda c: (0, _some(c)), "own": lambda c: (0, 4096),
         "prefix": lambda c: (_columns(c), 0)}


def _some(c):
    """So many columns more that a head's keys, a quarter of a megabyte, look like some blocks' work."""
    return (250 << 10) // (c["pages"].shape[4] * c["pages"].itemsize * c["pages"].shape[2])


def _columns(c):
    """So many columns more that reading prefixes for each request looks expensive: 128 MB of them and a bit."""
    _, _, page, nkv, hd = c["pages"].shape
    return (130 << 20) // (max(1, len(c["lengths"])) * nkv * hd * 2 * c["pages"].itemsize * page) + 1


@pytest.fixture(params=WIDER, autouse=True)
def way(request, monkeypatch):
    """How a call goes depends on its sizes, the tables' widths among them: every test with tables as wide as they need to be,
    with somewhat wider ones of own tokens (clusters of blocks), with wide ones of them (runs over warps, joined) and with
    wide ones of prefixes (read once for a group)."""
    monkeypatch.setitem(globals(), "wider_by", WIDER[request.param])
    return request.param


def wider_by(c):
    return 0, 0


def widen(table, by):
    return torch.cat([table, table.new_full((table.shape[0], by), -1)], 1) if by else table


def make_tables(counts, page, free, wider=0):
    used = [-(-c // page) for c in counts]
    table = torch.full((len(counts), max([1] + used) + wider), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(used):
        table[b, :n] = free[:n]
        free = free[n:]
    return table, free


def make(dtype, nh, nkv, hd, page, prefix, own, new=None, groups=None, seed=0, wider=0, extra_rows=0, spread=1.0):
    """Everything a call takes.  new: rows a request (None: one, without starts); groups: first requests."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    total = sum(-(-c // page) for c in list(prefix) + list(own)) + 2
    free = torch.randperm(total, generator=g, device=DEV).int()
    prefix_table, free = make_tables(prefix, page, free, wider)
    table, free = make_tables(own, page, free, wider)
    pages = torch.randn(2, total, page, nkv, hd, generator=g, device=DEV).to(dtype)
    rows = (sum(new) if new is not None else len(own)) + extra_rows
    q = (spread * torch.randn(rows, (nh + 2 * nkv) * hd, generator=g, device=DEV)).to(dtype)
    cu = None
    if new is not None:
        cu = i32([sum(new[:b]) for b in range(len(new) + 1)])
    c = dict(q=q, nh=nh, pages=pages, prefix_table=prefix_table, prefix_lens=i32(prefix), block_table=table,
             lengths=i32(own), scale=hd ** -0.5, cu_groups=None if groups is None else i32(groups), cu=cu)
    for name, by in zip(("prefix_table", "block_table"), wider_by(c)):
        c[name] = widen(c[name], by)
    return c


def call(c, **more):
    return shared_prefix.attend(c["q"], c["nh"], c["pages"], c["prefix_table"], c["prefix_lens"], c["block_table"],
                                c["lengths"], c["scale"], cu_groups=c["cu_groups"], cu_seqlens_q=c["cu"], **more)


def check(got, c, pages=None):
    want, top, known = plain.attend(c["q"], c["nh"], c["pages"] if pages is None else pages, c["prefix_table"],
                                    c["prefix_lens"], c["block_table"], c["lengths"], c["scale"], c["cu_groups"], c["cu"])
    err = (got.double() - want).abs()[known]
    allowed = 2e-5 * top[known, None]
    if got.dtype is BF16:
        allowed = allowed + 2.0 ** -8 * (top[known, None] + want[known].abs())
    assert torch.isfinite(got[known]).all()
    assert (err <= allowed).all(), (float(err.max()), float(top.max()))


HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (8, 8, 64), (9, 1, 80), (16, 4, 96), (40, 8, 128), (4, 2, 256), (20, 1, 64),
         (6, 6, 16), (3, 1, 48), (150, 1, 64), (17, 1, 128), (10, 2, 192)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 24])
def test_heads(dtype, heads, page):
    c = make(dtype, *heads, page, [131], [1, 40, 77, 16, 130], [1, 3, 1, 2, 4])
    check(call(c), c)


PREFIXES = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4099]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (16, 4, 96)])
@pytest.mark.parametrize("prefix", PREFIXES)
def test_prefix_lengths(dtype, heads, prefix):
    c = make(dtype, *heads, 16, [prefix], [1, 33, 64, 2, 200, 0, 129], wider=prefix % 3)
    check(call(c), c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128, 112])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 64, 128, 256])
def test_pages(dtype, hd, page):
    c = make(dtype, 10, 2, hd, page, [301, 70], [1, 300, 65, 9, 128], [1, 2, 1, 1, 5], groups=[0, 3, 5])
    check(call(c), c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch,prefix,own,new", [
    (1, 700, 90, 1), (2, 300, 40, 1), (3, 2000, 1, 1), (33, 515, 70, 2), (64, 1024, 300, 1), (129, 260, 20, 3), (256, 900, 33, 1),
    (300, 100, 5, 1), (5, 4097, 600, 8), (2, 130, 90, 70), (1, 0, 500, 200)])
def test_batches(dtype, batch, prefix, own, new):
    counts = [1 + (b * 7) % new for b in range(batch)]
    counts[0] = new
    lens = [max(n, 1 + (b * 131) % own) for b, n in enumerate(counts)]
    c = make(dtype, 14, 2, 64, 16, [prefix], lens, counts)
    for hint in (None, new):
        check(call(c, max_q_len=hint), c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128, 80])
def test_groups(dtype, hd):
    """Prefixes of very different lengths, one of nothing, one of nobody, requests before and behind the groups."""
    own = [3, 100, 17, 64, 1, 250, 40, 31, 5]
    for groups in ([0, 2, 2, 5, 9], [1, 3, 4, 4, 7], [0, 0, 9, 9, 9]):
        c = make(dtype, 8, 2, hd, 16, [500, 33, 0, 2100], own, [1, 2, 1, 0, 1, 5, 1, 1, 3], groups=groups)
        check(call(c), c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 96])
def test_rows_without_keys_and_without_requests(dtype, hd):
    """No prefix and no token; more rows than tokens; requests without rows; rows behind the last."""
    c = make(dtype, 6, 2, hd, 8, [0], [0, 2, 0, 1, 9], [1, 4, 0, 1, 2], extra_rows=3)
    out = torch.full((c["q"].shape[0], 6 * hd), 7.0, dtype=dtype, device=DEV)
    assert call(c, out=out) is out
    check(out, c)
    assert (out[-3:] == 7.0).all() and (out[0] == 0).all() and (out[1:3] == 0).all() and (out[3] != 0).any()
    c = make(dtype, 6, 2, hd, 8, [40], [0, 2], [3, 5])                    # (nothing but the prefix for most)
    check(call(c), c)
    c = make(dtype, 6, 2, hd, 8, [40], [3, 2], extra_rows=2)             # (one row a request, more rows than requests)
    out = torch.full((4, 6 * hd), 7.0, dtype=dtype, device=DEV)
    check(call(c, out=out), c)
    assert (out[2:] == 7.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nothing_to_do(dtype):
    c = make(dtype, 4, 2, 64, 16, [20], [3, 4], [0, 0])
    assert call(c).shape == (0, 256)
    c = make(dtype, 4, 2, 64, 16, [20], [], [], extra_rows=2)
    out = torch.full((2, 256), 7.0, dtype=dtype, device=DEV)
    call(c, out=out)
    assert (out == 7.0).all()
    c = make(dtype, 4, 2, 64, 16, [], [3, 40], [1, 2], groups=[0])       # (no group at all)
    check(call(c), c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128, 48])
@pytest.mark.parametrize("batch", [2, 40])
def test_what_is_masked_counts_as_nothing(dtype, hd, batch):
    """Infinities and NaN behind a sequence's last token, in its last page and in pages that are nobody's."""
    own = [(7 * b) % 75 + 1 for b in range(batch)]
    c = make(dtype, 12, 2, hd, 16, [203], own, [1 + b % 2 for b in range(batch)])
    clean = c["pages"].clone()
    seen = torch.zeros(c["pages"].shape[1:3], dtype=torch.bool, device=DEV)
    for table, lens in ((c["prefix_table"], [203]), (c["block_table"], own)):
        for b, n in enumerate(lens):
            for at in range(n):
                seen[table[b, at // 16].long(), at % 16] = True
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV).to(dtype)
    fill = bad[torch.arange(hd, device=DEV) % 3].expand_as(c["pages"])
    c["pages"] = torch.where(seen[None, :, :, None, None], c["pages"], fill)
    check(call(c), c, clean)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128, 80])
def test_large_scores(dtype, hd):
    """Scores far apart: one key takes all; maxima that grow from tile to tile."""
    c = make(dtype, 4, 2, hd, 16, [400], [90, 3], [2, 1], spread=1.0)
    c["q"] = torch.ones_like(c["q"])
    ramp = torch.linspace(-3, 3, c["pages"].shape[1] * 16, device=DEV).view(-1, 16, 1, 1)
    c["pages"][0] = (ramp * 40 / hd ** 0.5).to(dtype)
    check(call(c), c)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(dtype):
    """Rows of q at any distance and at an odd address; tables cut out of wider ones; planes of their own; whole tables."""
    c = make(dtype, 6, 2, 64, 16, [64], [40, 17, 33], [2, 1, 1])
    want = call(c)
    wide = torch.randn(4, 700, device=DEV).to(dtype)
    for start in (0, 1, 3, 8):
        q = wide[:, start:start + 6 * 64 + 5]
        q[:, :6 * 64] = c["q"][:, :6 * 64]
        check(call(dict(c, q=q)), dict(c, q=q))
        assert torch.equal(call(dict(c, q=q)), want)
    P = c["prefix_table"].shape[1]
    table = torch.cat([c["prefix_table"].expand(3, -1), c["block_table"]], 1)
    pages = (c["pages"][0].clone(), c["pages"][1].clone())
    got = call(dict(c, pages=pages, prefix_table=table[:1, :P], block_table=table[:, P:]))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_entries_that_are_no_page(dtype):
    """Behind the lengths they are not read; within them the call stays inside the cache and the other requests' results stay."""
    c = make(dtype, 6, 2, 64, 16, [64], [40, 17, 33])
    want = call(c)
    c["block_table"][1, :3] = i32([1 << 30, -(1 << 30), 77])
    got = call(c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_numbers_that_are_none(dtype):
    """Lengths beyond the tables, starts beyond the rows, groups beyond the requests: cut, never followed."""
    c = make(dtype, 6, 2, 64, 16, [64], [40, 17, 33], [2, 1, 1])
    c["lengths"] = i32([1 << 30, -5, 33])
    c["prefix_lens"] = i32([1 << 30])
    assert torch.isfinite(call(c)).all()
    for cu in ([0, 1 << 30, 1, 4], [-7, 2, 3, 4], [3, 2, 1, 0], [5, 6, 7, 8]):
        call(dict(c, cu=i32(cu)), out=torch.zeros(4, 384, dtype=dtype, device=DEV))
    for groups in ([-5, 1 << 30], [9, -9], [7, 9]):
        call(dict(c, cu_groups=i32(groups)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_starts_that_do_not_rise(dtype, hd):
    """A group's later requests may have rows in front of its first one's: they are no piece's.  The request behind is served."""
    c = make(dtype, 6, 2, hd, 16, [64], [40, 17, 33], [5, 1, 2])
    for cu in ([3, 1, 8, 8], [6, 0, 7, 8], [7, 2, 0, 8]):
        out = torch.zeros(8, 6 * hd, dtype=dtype, device=DEV)
        call(dict(c, cu=i32(cu)), out=out)
    torch.cuda.synchronize()
    check(call(c), c)


def test_more_requests_than_a_grid_has_rows():
    """70,000 requests are one call; halves of them, another way each, say the same."""
    batch = 70000
    c = make(F32, 4, 2, 16, 4, [9], [1 + b % 7 for b in range(batch)])
    got = call(c)
    half = batch // 2
    for b in (0, half):
        part = dict(c, q=c["q"][b:b + half], block_table=c["block_table"][b:b + half], lengths=c["lengths"][b:b + half])
        assert (got[b:b + half] - call(part)).abs().max() <= 4e-5 * c["pages"].abs().max()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_streams_and_graphs(dtype):
    """Another stream than the tensors' own; a captured call replayed with other lengths; two graphs and a call between."""
    c = make(dtype, 28, 4, 128, 16, [700], [60, 300, 9, 128] * 4, [1, 3, 1, 2] * 4)
    want = call(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    d = make(dtype, 28, 4, 128, 16, [333], [200, 5] * 8, [2, 1] * 8, seed=3)
    other = call(d)
    graphs = []
    for x in (c, d):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call(x)))
    for _ in range(3):
        graphs[0][0].replay()
        assert torch.equal(call(d), other)
        graphs[1][0].replay()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], other)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):                                     # both at once
        for s, (graph, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], other)
    c["lengths"].copy_(i32([7, 31, 300, 4] * 4).clamp(max=c["block_table"].shape[1] * 16))
    c["lengths"].copy_(torch.minimum(c["lengths"], i32([60, 300, 9, 128] * 4)))
    c["prefix_lens"].fill_(129)
    graphs[0][0].replay()
    check(graphs[0][1], c)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_same_twice(dtype):
    c = make(dtype, 12, 2, 128, 16, [3000], [(37 * b) % 900 + 1 for b in range(32)], [1 + b % 5 for b in range(32)])
    first = call(c)
    for _ in range(5):
        assert torch.equal(call(c), first)


def test_far_into_a_large_cache():
    """Pages whose elements' numbers pass 32 bits."""
    nkv, hd, page = 4, 128, 64
    count = (1 << 31) // (page * nkv * hd) + 40
    pages = torch.empty(2, count, page, nkv, hd, dtype=BF16, device=DEV)
    c = make(BF16, 8, nkv, hd, page, [300], [70, 130], [1, 2])
    n = c["pages"].shape[1]
    pages[:, -n:] = c["pages"]
    for t in ("prefix_table", "block_table"):
        c[t] = torch.where(c[t] >= 0, c[t] + (count - n), c[t])
    small = call(dict(c, prefix_table=c["prefix_table"] - (count - n), block_table=c["block_table"] - (count - n)))
    c["pages"] = pages
    assert torch.equal(call(c), small)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_ways(dtype, hd, way):
    """One launch for short tables, two where every request reads its own prefix, three where groups read them together (in
    32 bits only for heads of at most 64)."""
    c = make(dtype, 8, 2, hd, 16, [77], [1, 30, 9], [1, 2, 1])
    call(c)
    before = _Counter.launches
    check(call(c), c)
    shared = 3 if dtype is BF16 or hd <= 64 else 2
    assert _Counter.launches - before == {"narrow": 1, "cluster": 1, "own": 2, "prefix": shared}[way]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 80])
def test_many_groups(dtype, hd):
    """More groups than a warp has lanes, more requests than a block has threads; groups of none, of one, of many."""
    sizes = [(g * 5) % 13 for g in range(70)]
    first = [2 + sum(sizes[:g]) for g in range(71)]
    batch = first[-1] + 3
    counts = [(b * 3) % 4 for b in range(batch)]
    c = make(dtype, 6, 2, hd, 16, [(g * 37) % 300 for g in range(70)], [(b * 11) % 90 for b in range(batch)], counts, groups=first)
    check(call(c), c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)])
def test_hints_that_are_wrong(dtype, heads):
    c = make(dtype, *heads, 16, [290], [40, 9, 100, 64], [1, 9, 30, 2])
    for hint in (0, 1, 2, 7, 100, 1 << 20):
        check(call(c, max_q_len=hint), c)


def test_threads_on_one_stream(way):
    """Scratch memory is a stream's: calls of several threads on it follow one another whole."""
    cs = [make(BF16, 28, 4, 128, 16, [1200 + 100 * i], [200 + i, 5] * 20, seed=i) for i in range(4)]
    want = [call(c) for c in cs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        for _ in range(50):
            if not torch.equal(call(cs[i]), want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
