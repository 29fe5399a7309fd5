"""Attention over shared prefixes and the verification of drafted tokens from their definitions, in 64 bits."""
import torch


def tokens_of(plane, table, n):
    """The first n rows that a row of a table names: [n, kv heads, dim]."""
    page = plane.shape[1]
    used = -(-n // page)
    return plane[table[:used].long()].reshape(used * page, *plane.shape[2:])[:n].double()


def attend(q, nh, pages, prefix_table, prefix_lens, block_table, lengths, scale, cu_groups=None, cu=None):
    """(out [T, nh * dim], the largest value a row sees, rows that belong to a request), all in 64 bits."""
    nkv, hd = pages[0].shape[2:]
    T, G, B = q.shape[0], len(prefix_lens), len(lengths)
    x = q[:, :nh * hd].double().view(T, nkv, nh // nkv, hd)
    out, top = torch.zeros_like(x), torch.zeros(T, dtype=torch.float64, device=q.device)
    known = torch.zeros(T, dtype=torch.bool, device=q.device)
    first = list(range(B + 1)) if cu is None else cu.tolist()
    groups = [0, B] if cu_groups is None else cu_groups.tolist()
    own, shared = lengths.tolist(), prefix_lens.tolist()
    for b in range(B):
        n = first[b + 1] - first[b]
        g = next((g for g in range(G) if groups[g] <= b < groups[g + 1]), None)
        kv = []
        for plane in pages:
            far = tokens_of(plane, prefix_table[g], shared[g]) if g is not None else \
                torch.zeros(0, nkv, hd, dtype=torch.float64, device=q.device)
            kv.append(torch.cat([far, tokens_of(plane, block_table[b], own[b])]))
        far = len(kv[0]) - own[b]
        for i in range(n):
            row, see = first[b] + i, far + max(0, own[b] - n + i + 1)
            known[row] = True
            if see:
                w = torch.softmax(torch.einsum("kgd,ckd->kgc", x[row], kv[0][:see]) * scale, -1)
                out[row] = torch.einsum("kgc,ckd->kgd", w, kv[1][:see])
                top[row] = kv[1][:see].abs().max()
    return out.flatten(1), top, known


def weights(x, t):
    """A row's probabilities: NaN counts as -inf, infinities share all, None where there is no number."""
    x = torch.where(torch.isnan(x), -float("inf"), x.double())
    if (x == float("inf")).any():
        return (x == float("inf")).double() / (x == float("inf")).sum()
    if (x == -float("inf")).all():
        return torch.zeros_like(x)
    return torch.softmax(x / t, 0)


def best(x):
    x = torch.where(torch.isnan(x), -float("inf"), x.double())
    return int((x == x.max()).nonzero()[0])


def first_reaching(w, u):
    """The first index with a weight at which the running sum reaches u times the whole; None where there is no weight."""
    run = torch.cumsum(w, 0)
    if not float(run[-1]) > 0:
        return None
    hit = ((run >= u * run[-1]) & (w > 0)).nonzero()
    return int(hit[0]) if len(hit) else None


def verify(logits, tokens, cu_rows, temperature, u, draft=None):
    """(accepted, next tokens) as lists."""
    V, accepted, following = logits.shape[1], [], []
    rows, toks, us = cu_rows.tolist(), tokens.tolist(), u.double().tolist()
    for b, t in enumerate(temperature.double().tolist()):
        c0, c1 = rows[b], rows[b + 1]
        a, token = 0, -1
        for row in range(c0, c1):
            x, last = logits[row], row + 1 == c1
            d = -1 if last else toks[row + 1]
            if not t > 0:
                token = best(x)
                if last or d != token:
                    break
                a += 1
                continue
            p = weights(x, t)
            if last:
                q = torch.zeros_like(p)
            elif draft is None:
                q = torch.zeros_like(p)
                if 0 <= d < V:
                    q[d] = 1.0
            else:
                q = weights(draft[row], t)
            if not last and 0 <= d < V and us[row] * float(q[d]) < float(p[d]):
                a += 1
                continue
            token = first_reaching((p - q).clamp(min=0.0), us[c1 - 1])
            if token is None:
                token = first_reaching(p, us[c1 - 1])
            if token is None:
                token = best(x)
            break
        accepted.append(a)
        following.append(token)
    return accepted, following
