"""Plain implementations of the caption-serving operators on the host: paged attention and logits processing in
64 bits, the page pool's rules one row after the other."""
import math

import torch


def paged_attention(q, k_pages, v_pages, table, kv_lens, k=None, v=None, starts=None, offsets=None, max_rows=None,
                    scale=None, causal=True):
    """-> (out, bound terms (sum_j p_j |v_j|, sum_j |v_j|, max scale |q| . |k|) per row, k_pages, v_pages), all float64
    (the pages in their own type).  Rows without a visible key are 0."""
    packed = offsets is not None
    pages, kvh, ps, d = k_pages.shape
    heads = q.shape[-2]
    grp = heads // kvh
    n, width = table.shape
    scale = d ** -0.5 if scale is None else scale
    k_pages, v_pages = k_pages.clone(), v_pages.clone()
    out = torch.zeros(q.shape, dtype=torch.float64)
    aux = [torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64),
           torch.zeros(q.shape[:-1], dtype=torch.float64)]
    spans = []
    for s in range(n):
        if packed:
            r0, r1 = int(offsets[s]), int(offsets[s + 1])
            rows = r1 - r0 if max_rows is None else min(r1 - r0, max_rows)
            full = r1 - r0
        else:
            r0, rows = s, q.shape[1]
            full = rows
        kv = max(0, min(int(kv_lens[s]), width * ps))
        st = int(starts[s]) if starts is not None else int(kv_lens[s]) - full
        spans.append((s, r0, rows, kv, st))
        if k is not None:
            for i in range(rows):
                p = st + i
                if 0 <= p < kv and 0 <= int(table[s, p // ps]) < pages:
                    src_k, src_v = (k[r0 + i], v[r0 + i]) if packed else (k[s, i], v[s, i])
                    k_pages[table[s, p // ps], :, p % ps] = src_k
                    v_pages[table[s, p // ps], :, p % ps] = src_v
    for s, r0, rows, kv, st in spans:
        ok = [j for j in range(kv) if 0 <= int(table[s, j // ps]) < pages]
        if not ok:
            continue
        j = torch.tensor(ok)
        page = table[s, j // ps].long()
        K = k_pages[page, :, j % ps].double()  # (keys, kvh, d)
        V = v_pages[page, :, j % ps].double()
        for i in range(rows):
            see = j <= st + i if causal else torch.ones(len(ok), dtype=torch.bool)
            if not bool(see.any()):
                continue
            at = (r0 + i,) if packed else (s, i)
            x = q[at].double().view(kvh, grp, d)
            kk, vv = K[see].transpose(0, 1), V[see].transpose(0, 1)
            sc = torch.matmul(x, kk.transpose(1, 2)) * scale
            p = torch.softmax(sc, -1)
            out[at] = torch.matmul(p, vv).reshape(heads, d)
            aux[0][at] = torch.matmul(p, vv.abs()).reshape(heads, d)
            aux[1][at] = vv.abs().sum(1, keepdim=True).expand(kvh, grp, d).reshape(heads, d)
            aux[2][at] = (torch.matmul(x.abs(), kk.abs().transpose(1, 2)) * scale).amax(-1).reshape(heads)
    return out, aux, k_pages, v_pages


def pages_update(table, lens, refs, parents, new_lens, page_size, data=None):
    """Lists in, lists out: (table, lens, refs, short); data (a tensor) changed in place."""
    n, width, pages = len(lens), len(table[0]) if len(table) else 0, len(refs)
    cap = width * page_size
    up = lambda t: -(-t // page_size)  # noqa: E731
    lens_c = [min(max(v, 0), cap) for v in lens]
    keep, rows, want = [], [], []
    for s in range(n):
        p = s if parents is None else parents[s]
        base = lens_c[p] if 0 <= p < n else 0
        w = base if new_lens is None else min(max(new_lens[s], 0), cap)
        keep.append(min(base, w))
        want.append(w)
        rows.append([x if 0 <= x < pages else -1 for x in table[p][:up(keep[s])]] if keep[s] else [])
    r = list(refs)
    for s in range(n):
        for x in table[s][:up(lens_c[s])]:
            if 0 <= x < pages:
                r[x] -= 1
    for row in rows:
        for x in row:
            if x >= 0:
                r[x] += 1
    free = [x for x in range(pages) if r[x] == 0]
    # a copy for every growing row of a partial shared page but the highest, if no other row keeps the page
    asked, plan = 0, []
    sharers = {}
    for s in range(n):
        if want[s] > keep[s] and keep[s] % page_size and rows[s][-1] >= 0 and r[rows[s][-1]] > 1:
            sharers.setdefault(rows[s][-1], []).append(s)
    copies = {s for x, who in sharers.items() for s in (who[:-1] if len(who) == r[x] else who)}
    for s in range(n):
        cow = None
        if s in copies:
            cow, asked = asked, asked + 1
        fresh = list(range(asked, asked + up(want[s]) - len(rows[s])))
        asked += len(fresh)
        plan.append((cow, fresh))
    if asked > len(free):
        return [list(t) for t in table], list(lens), list(refs), asked - len(free)
    out = []
    for s, (cow, fresh) in enumerate(plan):
        row = list(rows[s])
        if cow is not None:
            used, old = keep[s] % page_size, row[-1]
            if data is not None:
                data[:, :, free[cow], :, :used] = data[:, :, old, :, :used]
            r[old] -= 1
            row[-1] = free[cow]
        row += [free[k] for k in fresh]
        out.append(row + [-1] * (width - len(row)))
    for k in range(asked):
        r[free[k]] = 1
    return out, want, r, 0


def pages_compact(table, refs, data=None):
    """(table, refs, remap, live); data changed in place."""
    live = sum(r > 0 for r in refs)
    holes = [x for x in range(live) if refs[x] <= 0]
    movers = [x for x in range(live, len(refs)) if refs[x] > 0]
    remap = [x if r > 0 else -1 for x, r in enumerate(refs)]
    out = [r if x < live and r > 0 else 0 for x, r in enumerate(refs)]
    for a, b in zip(movers, holes):
        remap[a], out[b] = b, refs[a]
        if data is not None:
            data[:, :, b] = data[:, :, a]
    return [[remap[x] if 0 <= x < len(refs) else -1 for x in row] for row in table], out, remap, live


def process_logits(logits, tokens=None, token_lens=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
                   allowed=None, states=None):
    """(values (n, vocab) float64, best, lse)"""
    n, vocab = logits.shape
    per_row = lambda x, i: float(x[i]) if isinstance(x, torch.Tensor) else x  # noqa: E731
    if allowed is not None and allowed.dtype == torch.int32:
        v = torch.arange(vocab)
        allowed = ((allowed.long().reshape(-1, allowed.shape[-1])[:, v // 32] >> (v % 32)) & 1) != 0
    elif allowed is not None:
        allowed = allowed.reshape(-1, vocab) != 0
    outs, best, lse = [], [], []
    for i in range(n):
        x = logits[i].double()
        if tokens is not None:
            t = tokens[i][:max(0, int(token_lens[i])) if token_lens is not None else None].long()
            t = t[(t >= 0) & (t < vocab)]
            c = torch.bincount(t, minlength=vocab)
            r = per_row(repetition, i)
            y = torch.where(x > 0, x / r, x * r) - per_row(presence, i) - per_row(frequency, i) * c
            x = torch.where(c > 0, y, x)
        if bias is not None:
            x = x + (bias[i] if bias.dim() == 2 else bias).double()
        if allowed is not None:
            row = int(states[i]) if states is not None else (0 if allowed.shape[0] == 1 else i)
            if 0 <= row < allowed.shape[0]:
                x = torch.where(allowed[row], x, -math.inf)
        outs.append(x)
        lse.append(torch.logsumexp(x, 0))
        nan = torch.isnan(x)
        top = torch.nonzero(nan)[0, 0] if bool(nan.any()) else torch.nonzero(x == x.max())[0, 0]
        best.append(-1 if bool((x == -math.inf).all()) else int(top))
    return torch.stack(outs), torch.tensor(best), torch.stack(lse)
