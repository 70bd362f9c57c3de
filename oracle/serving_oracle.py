"""64-bit CPU restatements of the serving operators (page plan, page write, attention over pages, token sampling), from
their definitions, one request, row or token at a time.  Used by the tests only.  No counterpart in the reference."""
import math

import torch


def page_plan(kv_lens, new_lens, finished, table, free_pages, free_count, page_size, rows):
    """Lists in, dict of lists out: kv_lens, table, free_pages, free_count, slots, cu_rows, granted."""
    kv = [max(0, k) for k in kv_lens]
    new = [max(0, n) for n in new_lens]
    table, free, top = [list(r) for r in table], list(free_pages), free_count
    width = len(table[0])
    pages = lambda n: -(-n // page_size)
    for b in range(len(kv)):
        if finished is not None and finished[b]:
            for c in range(pages(kv[b])):
                if top < len(free):
                    free[top] = table[b][c]
                    top += 1
            kv[b] = 0
    height, asked = top, 0
    slots, cu, granted = [-1] * rows, [0], []
    for b in range(len(kv)):
        cu.append(cu[-1] + new[b])
        held, want = pages(kv[b]), pages(kv[b] + new[b])
        ok = kv[b] + new[b] <= width * page_size and cu[-1] <= rows
        if ok:
            asked += want - held
            ok = want == held or asked <= height
        granted.append(ok)
        if not ok:
            continue
        for c in range(held, want):
            top -= 1
            table[b][c] = free[top]
        for i in range(new[b]):
            pos = kv[b] + i
            slots[cu[b] + i] = table[b][pos // page_size] * page_size + pos % page_size
        kv[b] += new[b]
    return dict(kv_lens=kv, table=table, free_pages=free, free_count=top, slots=slots, cu_rows=cu, granted=granted)


def page_attention(q, k_pages, v_pages, table, kv_lens, cu_rows, scale, window=0, sinks=0, causal=True):
    """-> (out [N][H][D] float64, sum_j p_j |v_j| of every output element: what relative errors of p and v multiply)."""
    n_pages, hk, ps, d = k_pages.shape
    h = q.shape[1]
    group = h // hk
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros(q.shape, dtype=torch.float64)
    kd, vd, qd = k_pages.double(), v_pages.double(), q.double()
    for b in range(len(kv_lens)):
        c0, n, kv = cu_rows[b], cu_rows[b + 1] - cu_rows[b], max(0, kv_lens[b])
        for i in range(n):
            p = kv - n + i
            seen = []
            for j in range(kv):
                if causal and j > p:
                    break
                if window and not (j > p - window or j < sinks):
                    continue
                page = int(table[b][j // ps])
                if 0 <= page < n_pages:
                    seen.append((page, j % ps))
            if not seen:
                continue
            pg = torch.tensor([s[0] for s in seen])
            sl = torch.tensor([s[1] for s in seen])
            for hh in range(h):
                kk, vv = kd[pg, hh // group, sl], vd[pg, hh // group, sl]
                w = torch.softmax(kk @ qd[c0 + i, hh] * scale, 0)
                out[c0 + i, hh] = w @ vv
                mag[c0 + i, hh] = w @ vv.abs()
    return out, mag


def sample_token(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row (a 1-d tensor of any float type) -> token, by sorting."""
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    n = x.numel()
    top = x.max()
    if top == -math.inf:
        return -1
    order = sorted(range(n), key=lambda i: (-x[i].item(), i))
    if not temperature > 0:
        return order[0]
    w = torch.exp((x - top) / temperature).tolist()
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        total, before, kept = math.fsum(w[i] for i in order), 0.0, []
        for i in order:
            if kept and not before < top_p * total:
                break
            kept.append(i)
            before += w[i]
        order = kept
    kept = sorted(i for i in order if w[i] >= min(min_p, 1.0) or x[i] == top)
    total = math.fsum(w[i] for i in kept)
    run = 0.0
    for i in kept:
        run += w[i]
        if run > u * total:
            return i
    return kept[-1]
