"""What a step of requests behind shared prompts, with drafted tokens, needs beside the cache and the sampler.

``attend``  attention of every request's newest tokens (one, or one and some drafted ones) over a prefix that its
            group of requests shares and over its own tokens: for row ``t``, the ``i``-th of ``n`` rows of request ``b``,

                ``out[t, h] = sum_c softmax_c(scale <q[t, h], K_c>) V_c``

            over the prefix's tokens and the request's own ``0 .. length - n + i``; a row without a key gives zeros.
            Keys and values are in pages ``[2, pages, page, kv heads, dim]``; a table names the pages of every
            group's prefix in order, another one those of every request's own tokens.
``verify``  how many of a request's drafted tokens stay, and the token behind them: with ``p = softmax(logits /
            temperature)`` of the target and ``q`` the draft's likewise (without its logits: all of it on the drafted
            token), draft ``d`` stays while ``u q(d) < p(d)``; the token behind the last that stays is drawn from
            ``max(p - q, 0)``, or from ``p`` where all stay: the first index at which the running sum reaches ``u``
            times the whole.  A temperature of zero takes the arg-max on both counts.

Here are the cases that these are measured on, in plain torch and through the framework's entry points, and their
definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ----------------------------------------------------------------------------- cases
def _attend(dtype, heads, kv_heads, dim, page, batch, prefix, longest, queries=1, groups=1, empty=False):
    """``prefix``: tokens of the longest shared prefix; ``longest``: of a request's own ones, the new among them;
    ``queries``: new tokens of a request at most; ``empty``: the last request pads the batch and has none."""
    return dict(op="attend", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, batch=batch,
                prefix=prefix, longest=longest, queries=queries, groups=groups, empty=empty)


def _verify(dtype, batch, drafts, vocab, drafter, greedy=False, gap=0):
    """``drafter``: whether a model drafted (its logits stand beside the target's) or a look-up; ``greedy``: every third request has
    temperature zero; ``gap``: channels between one row of logits and the next."""
    return dict(op="verify", dtype=dtype, batch=batch, drafts=drafts, vocab=vocab, drafter=drafter, greedy=greedy,
                gap=gap)


def listed():
    return [
        # two chats that have just begun behind a short system prompt: latency
        dict(_attend("bf16", 14, 2, 64, 16, 2, 300, 40), name="attend-two"),
        # a serving batch behind a long system prompt
        dict(_attend("bf16", 28, 4, 128, 16, 64, 8192, 1024), name="attend-batch"),
        # a last token and up to four drafted ones a request; the prefix ends inside a page
        dict(_attend("bf16", 12, 2, 128, 16, 32, 4099, 2048, queries=5, empty=True), name="attend-drafts"),
        # many requests about one long document
        dict(_attend("bf16", 40, 8, 128, 16, 256, 32768, 512), name="attend-document"),
        # heads of another size, two prompts of unequal length, short drafts
        dict(_attend("bf16", 16, 4, 96, 8, 24, 3001, 700, queries=3, groups=2), name="attend-two-prompts"),
        # the 32-bit path; one of three groups has no prefix
        dict(_attend("f32", 14, 2, 64, 16, 12, 2000, 600, queries=2, groups=3), name="attend-f32"),
        # one request whose drafts came from a look-up: latency
        dict(_verify("f32", 1, 4, 151936, False), name="verify-one"),
        # a serving batch with a draft model
        dict(_verify("f32", 64, 4, 152064, True), name="verify-batch"),
        # a full batch, long drafts, heads that leave bfloat16 logits
        dict(_verify("bf16", 256, 7, 151936, True), name="verify-full"),
        # a small odd vocabulary out of padded rows, some requests greedy
        dict(_verify("f32", 33, 6, 32003, True, greedy=True, gap=61), name="verify-greedy"),
    ]


HEADS = ((14, 2, 64), (12, 2, 128), (28, 4, 128), (8, 8, 64), (9, 1, 80), (16, 4, 96), (40, 8, 128), (4, 2, 256),
         (20, 1, 64))


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if rng.random() < 0.4:
        vocab, drafts = _log(rng, 1000, 152064), rng.randint(0, 8)
        rows = 580_000_000 // (vocab * DTYPES[dtype].itemsize)            # of the target and the draft, in all
        batch = _log(rng, 1, max(1, min(256, rows // (2 * drafts + 1))))
        return _verify(dtype, batch, drafts, vocab, rng.random() < 0.6, rng.random() < 0.3,
                       rng.choice((0, 0, rng.randint(1, 200))))
    heads, kv, dim = rng.choice(HEADS)
    queries = rng.choice((1, 1, 1, rng.randint(2, 8)))
    wide = 1 if dtype == "bf16" else 2
    batch = _log(rng, 1, 256)
    # products of the prefix and bytes of the requests' own tokens stay below the largest listed case's
    work = 160_000_000_000 // (1 if dtype == "bf16" else 40)
    prefix = _log(rng, 32, max(32, min(32768, work // (4 * batch * queries * heads * dim))))
    longest = _log(rng, queries, max(queries, min(8192, 400_000_000 // (batch * 4 * kv * dim * wide))))
    return _attend(dtype, heads, kv, dim, rng.choice((8, 16, 16, 24, 64)), batch, prefix, longest, queries,
                   rng.choice((1, 1, rng.randint(1, min(5, batch)))), batch > 1 and rng.random() < 0.3)


def _spread(n, b):
    """A share of n for the b-th of many: evenly between a tenth and all of it."""
    return max(1, int(n * (0.1 + 0.9 * ((1.0 - 0.6180339887498949 * b) % 1.0))))


def _shape(case):
    """Every request's own tokens, its new ones among them, and the groups' prefixes and first requests."""
    B, G = case["batch"], case["groups"]
    new = [1 + (case["queries"] - 1) * (b % 3) // 2 for b in range(B)]
    new[0] = case["queries"]
    length = [max(n, _spread(case["longest"], b)) for b, n in enumerate(new)]
    if case["empty"]:
        new[-1] = length[-1] = 0
    prefix = [case["prefix"]] + [_spread(case["prefix"], g) for g in range(1, G)]
    if G > 2:
        prefix[-1] = 0
    return length, new, prefix, [B * g // G for g in range(G + 1)]


def work(case):
    if case["op"] == "verify":
        es, B = DTYPES[case["dtype"]].itemsize, case["batch"]
        drafts = sum(_drafted(case))
        rows = B + drafts + (drafts if case["drafter"] else 0)
        return {"bytes": rows * case["vocab"] * es + 8 * (B + drafts) + 12 * B, "flops": 4 * rows * case["vocab"]}
    length, new, prefix, first = _shape(case)
    nh, nkv, hd, es = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]].itemsize
    keys = 0
    for g, p in enumerate(prefix):
        for b in range(first[g], first[g + 1]):
            keys += new[b] * (p + length[b]) - new[b] * (new[b] - 1) // 2
    tables = 4 * sum(-(-x // case["page"]) for x in prefix + length)
    return {"bytes": 2 * sum(new) * nh * hd * es + 2 * (sum(prefix) + sum(length)) * nkv * hd * es + tables,
            "flops": 4 * keys * nh * hd}


# ----------------------------------------------------------------------------- inputs
def _ints(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _drafted(case):
    """How many tokens each request has drafted."""
    k = case["drafts"]
    return [k if b % 4 != 3 else k // 2 for b in range(case["batch"])]


def _places(starts, wide):
    """Row numbers ``[sequences, wide]`` and whether there is such a row."""
    at = torch.tensor(starts, device=DEV)
    rows = at[:-1, None] + torch.arange(wide, device=DEV)
    there = rows < at[1:, None]
    return torch.where(there, rows, 0), there


def _tables(counts, page, g, free):
    """A table of pages for every sequence of ``counts`` tokens, from the shuffled ``free`` ones, -1 behind them."""
    used = [-(-c // page) for c in counts]
    table = torch.full((len(counts), max(1, max(used))), -1, dtype=torch.int64, device=DEV)
    here = torch.arange(table.shape[1], device=DEV) < torch.tensor(used, device=DEV)[:, None]
    table[here] = free[:sum(used)]
    return _ints(table), free[sum(used):]


@torch.no_grad()
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, g)
    dtype, page = DTYPES[case["dtype"]], case["page"]
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    length, new, prefix, first = _shape(case)
    total = sum(-(-c // page) for c in length + prefix) + 1
    free = torch.randperm(total, generator=g, device=DEV)
    prefix_table, free = _tables(prefix, page, g, free)
    table, free = _tables(length, page, g, free)
    T, cu = sum(new), _starts(new)
    # some channels of k stand out, tokens differ in size, some queries are sure of what they look for
    pages = torch.randn(2, total, page, nkv, hd, generator=g, device=DEV, dtype=torch.bfloat16).to(dtype)
    pages[0] *= 1.0 + 3.0 * (torch.rand(nkv, hd, generator=g, device=DEV) < 0.04).to(dtype)
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, generator=g, device=DEV)
    qkv[:, :nh * hd] *= torch.exp(0.5 * torch.randn(T, nh, 1, generator=g, device=DEV)).expand(-1, -1, hd).flatten(1)
    # the groups' rows, padded to the longest
    rows, there = _places([cu[b] for b in first], max(cu[b1] - cu[b0] for b0, b1 in zip(first, first[1:])))
    own_rows, own_there = _places(cu, max(new))
    return {"case": case, "pages": pages, "q": qkv.to(dtype), "prefix_table": prefix_table,
            "prefix_lens": _ints(prefix), "table": table, "lengths": _ints(length), "cu": _ints(cu), "groups": _ints(first),
            "longest_new": max(new), "rows": rows, "there": there, "own_rows": own_rows, "own_there": own_there}


def _prepare_verify(case, g):
    B, V, dtype = case["batch"], case["vocab"], DTYPES[case["dtype"]]
    drafted = _drafted(case)
    cu = _starts([n + 1 for n in drafted])
    R, D = cu[-1], sum(drafted)

    def logits(x):
        """In rows with a gap between one and the next."""
        out = torch.empty(x.shape[0], V + case["gap"], dtype=dtype, device=DEV)[:, :V]
        return out.copy_(x)
    # a few tokens of every row stand far out of the others
    target = 2.0 * torch.randn(R, V, generator=g, device=DEV)
    likely = torch.randint(V, (R, 24), generator=g, device=DEV)
    target.scatter_(1, likely, 10.0 + 3.0 * torch.randn(R, 24, generator=g, device=DEV))
    temperature = 0.5 + torch.rand(B, generator=g, device=DEV)
    request = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(drafted, device=DEV) + 1)
    last = torch.zeros(R, dtype=torch.bool, device=DEV)
    last[torch.tensor(cu[1:], device=DEV) - 1] = True
    said = target[~last]                                              # the rows that drafts are held against
    draft = None
    if case["drafter"]:
        draft = target + 0.1 * torch.randn(R, V, generator=g, device=DEV)
        draft.scatter_add_(1, likely, 0.8 * torch.randn(R, 24, generator=g, device=DEV))
        said = draft[~last]
    if case["greedy"]:
        temperature[::3] = 0.0
    # drafts as the drafter draws them; a look-up finds a wrong one now and then
    t = temperature[request[~last], None].clamp(min=1e-3)
    noise = -torch.log(-torch.log(torch.rand(D, V, generator=g, device=DEV).clamp(1e-30, 1.0 - 1e-7)))
    guess = (said / t + noise).argmax(1) if D else torch.zeros(0, dtype=torch.int64, device=DEV)
    del noise
    if not case["drafter"]:
        wrong = torch.rand(D, generator=g, device=DEV) < 0.2
        guess = torch.where(wrong, torch.randint(V, (D,), generator=g, device=DEV), guess)
    first = torch.zeros(R, dtype=torch.bool, device=DEV)
    first[torch.tensor(cu[:-1], device=DEV)] = True
    tokens = torch.randint(V, (R,), generator=g, device=DEV)
    tokens[~first] = guess
    rows, there = _places(cu, max(drafted) + 1)
    return {"case": case, "logits": logits(target), "draft": logits(draft) if draft is not None else None,
            "tokens": _ints(tokens), "cu": _ints(cu), "temperature": temperature,
            "u": torch.rand(R, generator=g, device=DEV), "rows": rows, "there": there}


# ----------------------------------------------------------------------------- the plain form
def _dense(s, table):
    """Keys and values ``[2, sequences, tokens, kv heads, dim]`` of the tables' pages in 32 bits."""
    return s["pages"][:, table.long().clamp(min=0)].flatten(2, 3).float()


def _scores(q, k, seen, scale):
    """``q [n, rows, kv heads, heads of one, dim]``, ``k [n, tokens, kv heads, dim]`` -> ``[n, kv heads, rows * heads, tokens]``."""
    x = torch.matmul(q.permute(0, 2, 1, 3, 4).flatten(2, 3), k.permute(0, 2, 3, 1)) * scale
    return torch.where(seen, x, -math.inf)


def _part(q, kv, seen, scale):
    """Largest score, sum of weights and weighted values of some keys for padded rows."""
    x = _scores(q, kv[0], seen, scale)
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - top.clamp(min=-1e30))
    n, rows, nkv, each, hd = q.shape

    def back(y):
        return y.view(n, nkv, rows, each, -1).transpose(1, 2)
    return back(top), back(w.sum(-1, keepdim=True)), back(torch.matmul(w, kv[1].transpose(1, 2)))


def _plain_attend(s):
    case = s["case"]
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    q = s["q"][:, :nh * hd].float().view(-1, nkv, nh // nkv, hd)
    scale = hd ** -0.5
    # over the shared prefixes, group by group ...
    kv = _dense(s, s["prefix_table"])
    seen = (torch.arange(kv.shape[2], device=DEV) < s["prefix_lens"][:, None])[:, None, None]
    far = [x[s["there"]] for x in _part(q[s["rows"]], kv, seen, scale)]
    # ... over what is a request's own ...
    kv = _dense(s, s["table"])
    new = s["cu"][1:] - s["cu"][:-1]
    last = (s["lengths"] - new)[:, None] + torch.arange(s["own_rows"].shape[1], device=DEV)
    seen = torch.arange(kv.shape[2], device=DEV) <= last[..., None]
    seen = seen[:, None, :, None].expand(-1, -1, -1, nh // nkv, -1).flatten(2, 3)
    near = [x[s["own_there"]] for x in _part(q[s["own_rows"]], kv, seen, scale)]
    # ... and both together
    top = torch.maximum(far[0], near[0]).clamp(min=-1e30)
    a, b = torch.exp(far[0] - top), torch.exp(near[0] - top)
    total = a * far[1] + b * near[1]
    out = torch.where(total > 0, (a * far[2] + b * near[2]) / total, 0.0)
    return out.flatten(1).to(s["q"].dtype)


def _softmax(x, temperature):
    x = x.double() / temperature[:, None]
    w = torch.exp(x - x.amax(1, keepdim=True))
    return w / w.sum(1, keepdim=True)


def _plain_verify(s):
    """In 64 bits: a border between two tokens is met by 32 now and then."""
    rows, there, tokens, V = s["rows"], s["there"], s["tokens"].long(), s["logits"].shape[1]
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()
    B, wide = rows.shape
    every = torch.arange(B, device=DEV)
    count = there.sum(1) - 1                                            # drafts of a request
    of_row = torch.zeros(s["logits"].shape[0], dtype=torch.int64, device=DEV)
    of_row[rows[there]] = every[:, None].expand(-1, wide)[there]
    best = s["logits"].argmax(1)
    # the drafts: the i-th is the (i + 1)-th row's token, held against the i-th row
    guess, row = tokens[rows[:, 1:]], rows[:, :-1]
    p, q = _softmax(s["logits"], t[of_row]), None
    share = torch.ones(guess.shape, dtype=torch.float64, device=DEV)
    if s["draft"] is not None:
        q = _softmax(s["draft"], t[of_row])
        share = q[row, guess]
    stays = torch.where(greedy[:, None], best[row] == guess, s["u"][row].double() * share < p[row, guess])
    accepted = (stays & there[:, 1:]).long().cumprod(1).sum(1) if wide > 1 else torch.zeros_like(count)
    # the token behind them
    stop = rows.gather(1, accepted[:, None])[:, 0]
    w = p[stop]
    if wide > 1:
        refused = (accepted < count)[:, None]
        if q is not None:
            w = torch.where(refused, (w - q[stop]).clamp(min=0.0), w)
        else:
            w = torch.where(refused, w.scatter(1, guess.gather(1, accepted.clamp(max=wide - 2)[:, None]), 0.0), w)
    run_up = w.cumsum(1)
    u = s["u"][s["cu"][1:].long() - 1].double()
    hit = (run_up >= u[:, None] * run_up[:, -1:]) & (w > 0)
    drawn = hit.to(torch.uint8).argmax(1)
    return accepted.int(), torch.where(greedy, best[stop], drawn).int()


@torch.no_grad()
def run(s):
    case = s["case"]
    if own:
        if case["op"] == "verify":
            from ginfer_b200.ops import drafts
            return drafts.verify(s["logits"], s["tokens"], s["cu"], s["temperature"], s["u"], s["draft"])
        from ginfer_b200.ops import shared_prefix
        return shared_prefix.attend(s["q"], case["heads"], s["pages"], s["prefix_table"], s["prefix_lens"], s["table"],
                                    s["lengths"], case["dim"] ** -0.5, cu_groups=s["groups"], cu_seqlens_q=s["cu"],
                                    max_q_len=s["longest_new"])
    return _plain_verify(s) if case["op"] == "verify" else _plain_attend(s)


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _tokens64(s, table, n):
    """The first n keys and values that a row of a table names."""
    page = s["pages"].shape[2]
    kv = s["pages"][:, table[:-(-n // page)].long()].double()
    return kv.reshape(2, -1, *kv.shape[3:])[:, :n]


def _exact_attend(case, s):
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    length, new, prefix, first = _shape(case)
    q = s["q"][:, :nh * hd].double().view(-1, nkv, nh // nkv, hd)
    out = torch.zeros_like(q)
    cu = _starts(new)
    for g, n in enumerate(prefix):
        shared = _tokens64(s, s["prefix_table"][g], n)
        for b in range(first[g], first[g + 1]):
            mine = _tokens64(s, s["table"][b], length[b])
            for i in range(new[b]):
                keys, values = torch.cat([shared, mine[:, :length[b] - new[b] + i + 1]], 1)
                x = torch.einsum("kgd,ckd->kgc", q[cu[b] + i], keys) * hd ** -0.5
                if x.shape[-1]:
                    out[cu[b] + i] = torch.einsum("kgc,ckd->kgd", torch.softmax(x, -1), values)
    return out.reshape(-1, nh * hd)


def _exact_verify(case, s):
    cu, u = s["cu"].tolist(), s["u"].double().tolist()
    tokens, heat = s["tokens"].tolist(), s["temperature"].double().tolist()
    accepted, following = [], []
    for b, t in enumerate(heat):
        a, rest, row = 0, None, cu[b]
        for row in range(cu[b], cu[b + 1]):
            x = s["logits"][row].double()
            if t <= 0:
                rest = torch.nn.functional.one_hot(x.argmax(), x.numel()).double()
                stays = row + 1 < cu[b + 1] and float(rest[tokens[row + 1]]) > 0
            else:
                rest = torch.softmax(x / t, 0)
                if row + 1 == cu[b + 1]:
                    break
                d = tokens[row + 1]
                if s["draft"] is None:
                    other = torch.nn.functional.one_hot(torch.tensor(d, device=DEV), x.numel()).double()
                else:
                    other = torch.softmax(s["draft"][row].double() / t, 0)
                stays = u[row] * float(other[d]) < float(rest[d])
                if not stays:
                    rest = torch.relu(rest - other)
            if not stays:
                break
            a += 1
        heap = torch.cumsum(rest, 0)
        at = int(torch.searchsorted(heap, u[cu[b + 1] - 1] * heap[-1:])[0])
        while float(rest[at]) <= 0:                  # (u of zero: tokens of no weight stand first)
            at += 1
        accepted.append(a)
        following.append(at)
    return _ints(accepted), _ints(following)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_verify(case, s) if case["op"] == "verify" else _exact_attend(case, s)
