"""What is measured of the serving operators: the page plan, the page write, attention of a chunk over the pages and
token sampling, each with a plain form in elementary torch operations and a 64-bit definition.

`run(state)` is one pass as a serving program makes it: in plain form while `own` is false, through
`conformer_amd.ops` when it is true.  A cache is a pool of pages [page][kv head][slot of the page][head dim] for K and
one for V; a block table holds a request's page ids in order.
"""
import math
import random

import torch

own = False
DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 running requests: the smallest plan, pure latency
        dict(name="plan_step", op="plan", batch=64, prompts=0, max_new=1, finished=0, page=16, width=256),
        # a busy scheduler step: single tokens, whole prompts and rows that end, 256 requests
        dict(name="plan_mixed", op="plan", batch=256, prompts=32, max_new=4096, finished=9, page=16, width=2048),
        # the K/V rows of one decode step, 64 requests
        dict(name="write_step", op="write", rows=64, kv_heads=8, dim=64, dtype="bf16", page=16, packed=True),
        # the K/V rows of prompts, an odd count, cut out of a fused q|k|v projection
        dict(name="write_prompt", op="write", rows=16411, kv_heads=8, dim=128, dtype="bf16", page=64, packed=True),
        # streaming chunks of a speech encoder in fp32: 8 heads of 48, 4 frames a chunk that see each other, local
        # context 256 and the first 4 frames of the stream
        dict(name="attn_stream", op="attn", batch=8, mode="chunk", max_new=4, max_kv=1501, heads=8, kv_heads=8, dim=48,
             dtype="fp32", page=16, window=256, sinks=4, causal=False),
        # a decode step of a batch with ragged lengths, grouped heads
        dict(name="attn_step", op="attn", batch=64, mode="step", max_new=1, max_kv=8192, heads=32, kv_heads=8, dim=128,
             dtype="bf16", page=64, window=0, sinks=0, causal=True),
        # a decode step of two long contexts: few rows, a long axis
        dict(name="attn_step_long", op="attn", batch=2, mode="step", max_new=1, max_kv=131072, heads=32, kv_heads=4,
             dim=128, dtype="bf16", page=64, window=0, sinks=0, causal=True),
        # chunked prompts beside single tokens over a filled cache
        dict(name="attn_chunk", op="attn", batch=12, mode="mixed", max_new=512, max_kv=16384, heads=32, kv_heads=8,
             dim=128, dtype="bf16", page=32, window=0, sinks=0, causal=True),
        # whole prompts under a sliding window with sinks: the largest matrix work
        dict(name="attn_prompt", op="attn", batch=3, mode="prompt", max_new=8192, max_kv=8192, heads=32, kv_heads=8,
             dim=128, dtype="bf16", page=64, window=4096, sinks=4, causal=True),
        # the joint network's logits of 64 streams, 29 characters: the smallest draw
        dict(name="sample_chars", op="sample", rows=64, vocab=29, dtype="fp32", filters="temperature"),
        # one request, a word-piece vocabulary
        dict(name="sample_one", op="sample", rows=1, vocab=32001, dtype="fp32", filters="all"),
        # a full batch over a large vocabulary, each row with filters of its own
        dict(name="sample_batch", op="sample", rows=256, vocab=131072, dtype="bf16", filters="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    while True:
        case = _draw(rng)
        if case["op"] != "attn":
            return case
        w = work(case)
        # not above the largest listed attention cases in pairs or in cache
        if w["flops"] <= 1.2e12 and w["bytes"] <= 1.0e9:
            return case


def _draw(rng):
    op = rng.choice(["plan", "write", "attn", "attn", "attn", "sample", "sample"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        batch = _log(rng, 1, 256)
        return dict(op=op, batch=batch, prompts=rng.randint(0, min(batch, 32)), max_new=_log(rng, 1, 4096),
                    finished=rng.randint(0, batch // 8), page=page, width=_log(rng, 300, 2048))
    if op == "write":
        return dict(op=op, rows=_log(rng, 1, 16411), kv_heads=rng.choice([1, 2, 4, 5, 8]), dim=rng.choice([48, 64, 80, 128]),
                    dtype=rng.choice(["bf16", "bf16", "fp32"]), page=page, packed=rng.random() < 0.5)
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 29, 131072), dtype=rng.choice(["bf16", "fp32"]),
                    filters=rng.choice(["temperature", "all", "mixed"]))
    mode = rng.choice(["step", "chunk", "mixed", "prompt"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    window = rng.choice([0, 0, _log(rng, 64, 4096)])
    case = dict(op="attn", mode=mode, heads=heads, kv_heads=kv_heads, dim=rng.choice([48, 64, 64, 80, 96, 128, 128]),
                dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]), page=page, window=window,
                sinks=rng.choice([0, 1, 4, 64]) if window else 0, causal=rng.random() < 0.8)
    if mode == "step":
        batch = _log(rng, 1, 128)
        case.update(batch=batch, max_new=1, max_kv=_log(rng, 32, 131072 // batch + 2048))
    elif mode == "chunk":
        batch = _log(rng, 1, 64)
        case.update(batch=batch, max_new=_log(rng, 2, 64), max_kv=_log(rng, 128, 65536 // batch + 1024))
    elif mode == "mixed":
        case.update(batch=rng.randint(2, 24), max_new=_log(rng, 16, 512), max_kv=_log(rng, 1024, 16384))
    else:
        n = _log(rng, 100, 4096)
        case.update(batch=rng.randint(1, 4), max_new=n, max_kv=n)
    return case


# ------------------------------------------------------------------------------------------------
# sizes that a scheduler knows on the host
# ------------------------------------------------------------------------------------------------
def _case_rng(case):
    """Lengths belong to the case: every seed has the same ones, with other pages and values."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _attn_lengths(case):
    """(rows of the chunk, cache length with them) of every request."""
    rng = _case_rng(case)
    new, kv = [], []
    for b in range(case["batch"]):
        m = case["mode"]
        if m == "step":
            n = 1
        elif m == "chunk":
            n = case["max_new"]
        elif m == "mixed":
            n = 1 if b % 3 == 2 else (case["max_new"] if b == 0 else rng.randint(1, case["max_new"]))
        else:
            n = case["max_new"] if b == 0 else rng.randint(max(1, case["max_new"] // 2), case["max_new"])
        total = n if m == "prompt" else max(n, case["max_kv"] if b == 0 else rng.randint(case["max_kv"] // 4, case["max_kv"]))
        new.append(n)
        kv.append(total)
    return new, kv


def _visible(n, kv, window, sinks, causal):
    """(visible key-row pairs, keys that at least one row sees) of a chunk."""
    pairs = 0
    for i in range(n):
        p = kv - n + i
        hi = p if causal else kv - 1
        lo = max(0, p - window + 1) if window else 0
        pairs += hi - lo + 1 + min(sinks, lo)
    lo = max(0, kv - n - window + 1) if window else 0
    return pairs, kv - lo + min(sinks, lo)


def _plan_lengths(case):
    rng = _case_rng(case)
    b, cap = case["batch"], case["width"] * case["page"]
    new = [1] * b
    for i in rng.sample(range(b), case["prompts"]):
        new[i] = rng.randint(1, case["max_new"])
    kv = [rng.randint(0, cap - case["max_new"]) if cap > case["max_new"] else 0 for _ in range(b)]
    for i, n in enumerate(new):
        if n > 1:
            kv[i] = 0                       # a prompt starts an empty row
    fin = [False] * b
    for i in rng.sample(range(b), case["finished"]):
        fin[i], new[i] = True, 0
    return new, kv, fin


def work(case):
    if case["op"] == "plan":
        new, kv, fin = _plan_lengths(case)
        ps = case["page"]
        pages = sum(-(-(k + n) // ps) - -(-k // ps) for n, k, f in zip(new, kv, fin) if not f)
        freed = sum(-(-k // ps) for k, f in zip(kv, fin) if f)
        tables = sum(-(-(k + n) // ps) - k // ps for n, k in zip(new, kv) if n)
        b = case["batch"]
        return {"bytes": 9 * b + 8 * (pages + freed) + 4 * (tables - pages) + 8 * sum(new) + 9 * b + 12,
                "flops": 0}
    if case["op"] == "write":
        es = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": case["rows"] * (4 * case["kv_heads"] * case["dim"] * es + 8), "flops": 0}
    if case["op"] == "sample":
        es = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": case["rows"] * (case["vocab"] * es + 24), "flops": 4 * case["rows"] * case["vocab"]}
    es = 2 if case["dtype"] == "bf16" else 4
    new, kv = _attn_lengths(case)
    pairs = keys = 0
    for n, k in zip(new, kv):
        p, c = _visible(n, k, case["window"], case["sinks"], case["causal"])
        pairs, keys = pairs + p, keys + c
    return {"bytes": 2 * sum(new) * case["heads"] * case["dim"] * es + 2 * keys * case["kv_heads"] * case["dim"] * es
            + 4 * (keys // case["page"] + 3 * case["batch"]),
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _i32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def _tables(kv, page, width, pool, rng):
    """Block table with the pages of every request scattered over the pool, -1 past them, and the pages left."""
    order = list(range(pool))
    rng.shuffle(order)
    table, at = torch.full((len(kv), width), -1, dtype=torch.int32), 0
    for b, k in enumerate(kv):
        c = -(-k // page)
        table[b, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    return table.to(DEV), order[at:]


def prepare(case, seed):
    rng = random.Random(seed * 31 + 3)
    gen = torch.Generator(device=DEV).manual_seed(seed * 9973 + 17)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)

    st = dict(case=case)
    if case["op"] == "plan":
        new, kv, fin = _plan_lengths(case)
        ps = case["page"]
        need = sum(-(-(k + n) // ps) - -(-k // ps) for n, k, f in zip(new, kv, fin) if not f)
        pool = sum(-(-k // ps) for k in kv) + need + 64
        table, left = _tables(kv, ps, case["width"], pool, rng)
        free = torch.full((pool,), -1, dtype=torch.int32)
        free[:len(left)] = torch.tensor(left, dtype=torch.int32)
        counters = _i32(kv + [0] * (-len(kv) % 4) + [len(left)])    # lengths and the stack's height, restored at once
        st.update(counters0=counters, counters=counters.clone(), new=_i32(new), table=table, free=free.to(DEV),
                  finished=torch.tensor(fin).to(DEV), rows=sum(new), at=len(kv) + -len(kv) % 4)
    elif case["op"] == "write":
        h, d, ps, n, dt = case["kv_heads"], case["dim"], case["page"], case["rows"], _DT[case["dtype"]]
        pool = -(-n // ps) + 8
        if case["packed"]:       # k and v inside a fused projection with as many query columns
            qkv = randn(n, 3 * h * d, dtype=dt).view(n, 3 * h, d)
            k, v = qkv[:, h:2 * h], qkv[:, 2 * h:]
        else:
            k, v = randn(n, h, d, dtype=dt), randn(n, h, d, dtype=dt)
        # the rows of requests that hold neighbouring slots of scattered pages
        slots = torch.randperm(pool, generator=gen, device=DEV)[:, None] * ps + torch.arange(ps, device=DEV)
        slots = slots.reshape(-1)[:n].contiguous()
        if n > 7:
            slots[n // 2] = -1   # a request that got no page
        st.update(k=k, v=v, slots=slots, kp=randn(pool, h, ps, d, dtype=dt), vp=randn(pool, h, ps, d, dtype=dt))
    elif case["op"] == "attn":
        h, d, ps, dt = case["kv_heads"], case["dim"], case["page"], _DT[case["dtype"]]
        new, kv = _attn_lengths(case)
        width = -(-max(kv) // ps) + 3
        pool = sum(-(-k // ps) for k in kv) + 5
        table, _ = _tables(kv, ps, width, pool, rng)
        kp, vp = randn(pool, h, ps, d, dtype=dt), randn(pool, h, ps, d, dtype=dt)
        q = randn(sum(new), case["heads"], d, dtype=dt) * 1.5
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        st.update(q=q, kp=kp, vp=vp, table=table, kv_lens=_i32(kv), cu=_i32(cu), new=new, kv=kv, scale=d ** -0.5)
    else:
        r, v = case["rows"], case["vocab"]
        x = randn(r, v) * 2.2
        x += 4.0 * (torch.rand((r, v), generator=gen, device=DEV) < 20.0 / (v + 20)).float()     # a few likely tokens
        x = x.clamp(-15.0, 15.0).to(_DT[case["dtype"]])
        u = torch.rand((r,), generator=gen, device=DEV)
        temp = torch.tensor([rng.choice([0.6, 0.8, 1.0, 1.3]) for _ in range(r)]).to(DEV)
        top_k = top_p = min_p = None
        if case["filters"] == "all":
            top_k = _i32([rng.choice([20, 50, 200]) for _ in range(r)])
            top_p = torch.tensor([rng.choice([0.8, 0.9, 0.95]) for _ in range(r)]).to(DEV)
            min_p = torch.tensor([rng.choice([0.02, 0.05]) for _ in range(r)]).to(DEV)
        elif case["filters"] == "mixed":
            temp = torch.tensor([rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]) for _ in range(r)]).to(DEV)
            top_k = _i32([rng.choice([0, 0, 1, 40, 1000]) for _ in range(r)])
            top_p = torch.tensor([rng.choice([1.0, 0.5, 0.9, 0.98]) for _ in range(r)]).to(DEV)
            min_p = torch.tensor([rng.choice([0.0, 0.0, 0.03]) for _ in range(r)]).to(DEV)
        st.update(logits=x, u=u, temperature=temp, top_k=top_k, top_p=top_p, min_p=min_p)
    return st


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    return {"plan": _run_plan, "write": _run_write, "attn": _run_attn, "sample": _run_sample}[case["op"]](st, case)


def _run_plan(st, case):
    # the plan advances lengths and stack in place; a pass starts from the same state
    st["counters"].copy_(st["counters0"])
    b = case["batch"]
    kv_lens, free_count = st["counters"][:b], st["counters"][st["at"]:]
    fin = st["finished"] if case["finished"] else None
    if own:
        from conformer_amd import ops
        slots, cu, granted = ops.kv_page_plan_(kv_lens, st["new"], fin, st["table"], st["free"], free_count, case["page"],
                                               st["rows"])
    else:
        slots, cu, granted = _plain_plan(kv_lens, st["new"], fin, st["table"], st["free"], free_count, case["page"],
                                         st["rows"])
    return {"slots": slots, "cu_rows": cu, "granted": granted, "kv_lens": kv_lens, "free_count": free_count,
            "table": st["table"], "free_pages": st["free"]}


def _plain_plan(kv_lens, new, fin, table, free, free_count, ps, rows):
    dev, (b, width), pool = table.device, table.shape, free.numel()
    col = torch.arange(width, device=dev)
    row_of = torch.arange(b, device=dev)
    kv, n, top = kv_lens.long(), new.long(), free_count.long()
    if fin is not None:
        back = (col < ((kv + ps - 1) // ps)[:, None]) & fin[:, None]
        pages = table[back]
        free[(top + torch.arange(pages.numel(), device=dev))] = pages
        top = top + pages.numel()
        kv = torch.where(fin, 0, kv)
    held = (kv + ps - 1) // ps
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), n.cumsum(0)])
    fits = (kv + n <= width * ps) & (cu[1:] <= rows)
    need = torch.where(fits, (kv + n + ps - 1) // ps - held, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= top))
    need = torch.where(granted, need, 0)
    take = need.cumsum(0) - need
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    at = top - 1 - (take[:, None] + col - held[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, pool - 1)], table))
    owner = torch.repeat_interleave(row_of, n, output_size=rows)
    pos = kv[owner] + torch.arange(rows, device=dev) - cu[owner]
    slot = table[owner, (pos // ps).clamp(max=width - 1)].long() * ps + pos % ps
    slots = torch.where(granted[owner], slot, -1)
    kv_lens.copy_(kv + torch.where(granted, n, 0))
    free_count.copy_(top - need.sum())
    return slots, cu.int(), granted


def _run_write(st, case):
    if own:
        from conformer_amd import ops
        ops.kv_page_write_(st["k"], st["v"], st["kp"], st["vp"], st["slots"])
    else:
        ps = case["page"]
        keep = st["slots"] >= 0
        slots = st["slots"][keep]
        st["kp"][slots // ps, :, slots % ps] = st["k"][keep]
        st["vp"][slots // ps, :, slots % ps] = st["v"][keep]
    return {"k_pages": st["kp"], "v_pages": st["vp"]}


def _run_attn(st, case):
    if own:
        from conformer_amd import ops
        return ops.kv_page_attention(st["q"], st["kp"], st["vp"], st["table"], st["kv_lens"], st["cu"], st["scale"],
                                     case["window"], case["sinks"], case["causal"], max(st["new"]))
    out = torch.empty_like(st["q"])
    groups = {}                               # requests with as many rows go together, padded to the longest cache
    for b, n in enumerate(st["new"]):
        groups.setdefault(n, []).append(b)
    for n, members in groups.items():
        per = case["kv_heads"] * case["dim"] * max(st["kv"][b] for b in members)
        step = max(1, int(2 ** 29 // per))
        for i in range(0, len(members), step):
            _plain_attn(st, case, n, members[i:i + step], out)
    return out


def _plain_attn(st, case, n, members, out):
    hk, g, d, ps = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"], case["page"]
    m = len(members)
    pages = -(-max(st["kv"][b] for b in members) // ps)
    idx = torch.tensor(members, device=DEV)
    table = st["table"][idx, :pages].long().clamp(min=0)
    kv = st["kv_lens"][idx].long()
    k = st["kp"][table].permute(0, 2, 1, 3, 4).reshape(m, hk, pages * ps, d).float()
    v = st["vp"][table].permute(0, 2, 1, 3, 4).reshape(m, hk, pages * ps, d).float()
    j = torch.arange(pages * ps, device=DEV)
    v = torch.where((j < kv[:, None])[:, None, :, None], v, 0.0)
    start = st["cu"][idx].long()
    step = max(1, int(2 ** 28 // (m * hk * g * pages * ps)))
    for r0 in range(0, n, step):
        rows = min(step, n - r0)
        at = (start[:, None] + r0 + torch.arange(rows, device=DEV)).reshape(-1)
        q = st["q"][at].float().view(m, rows, hk, g, d).permute(0, 2, 3, 1, 4).reshape(m, hk, g * rows, d)
        p = (kv - n + r0)[:, None] + torch.arange(rows, device=DEV)
        see = _sees(j, p[:, :, None], kv[:, None, None], case)
        s = torch.matmul(q, k.transpose(2, 3).contiguous()) * st["scale"]
        s = s.view(m, hk, g, rows, -1).masked_fill(~see[:, None, None], float("-inf"))
        top = s.amax(-1, keepdim=True)
        e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
        z = e.sum(-1, keepdim=True)
        e = e / torch.where(z == 0, 1.0, z)
        o = torch.matmul(e.view(m, hk, g * rows, -1), v)
        o = o.view(m, hk, g, rows, d).permute(0, 3, 1, 2, 4).reshape(m * rows, hk * g, d)
        out[at] = o.to(out.dtype)


def _sees(j, p, kv, case):
    see = j < kv
    if case["causal"]:
        see = see & (j <= p)
    if case["window"]:
        see = see & ((j > p - case["window"]) | (j < case["sinks"]))
    return see


def _run_sample(st, case):
    if own:
        from conformer_amd import ops
        return ops.sample_tokens(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])
    return _plain_sample(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    """Weights and masses in 64 bits: a draw is a comparison of a sum with a border."""
    x = logits.float()
    rows, vocab = x.shape
    t = temperature.double()[:, None]
    order = torch.sort(x, dim=1, descending=True, stable=True)
    xs = order.values.double()
    z = torch.where(xs == xs[:, :1], 0.0, (xs - xs[:, :1]) / torch.where(t > 0, t, 1.0))
    w = torch.exp(z)
    rank = torch.arange(vocab, device=x.device)
    keep = torch.where(t > 0, rank >= 0, rank < 1)
    if top_k is not None:
        keep = keep & ((rank < top_k[:, None]) | (top_k[:, None] <= 0))
    wk = torch.where(keep, w, 0.0)
    if top_p is not None:
        before = wk.cumsum(1) - wk
        p = top_p.double()[:, None]
        keep = keep & ((before < p * wk.sum(1, keepdim=True)) | (p >= 1) | (rank == 0))
    if min_p is not None:
        keep = keep & (w >= min_p.double()[:, None].clamp(max=1.0))
    wi = torch.zeros_like(w).scatter_(1, order.indices, torch.where(keep, w, 0.0))
    mass = wi.cumsum(1)
    total = mass[:, -1:].contiguous()
    tok = torch.searchsorted(mass, u.double()[:, None] * total, right=True)[:, 0]
    return tok.clamp(max=vocab - 1).int()


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"plan": _exact_plan, "write": _exact_write, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](st, case)


def _exact_plan(st, case):
    ps, b, width = case["page"], case["batch"], case["width"]
    kv, new, fin = st["counters0"][:b].tolist(), st["new"].tolist(), st["finished"].tolist()
    table, free, top = st["table"].tolist(), st["free"].tolist(), int(st["counters0"][st["at"]])
    for i in range(b):
        if fin[i]:
            for c in range(-(-kv[i] // ps)):
                free[top] = table[i][c]
                top += 1
            kv[i] = 0
    slots, cu, granted, asked, height = [-1] * st["rows"], [0], [], 0, top
    for i in range(b):
        cu.append(cu[-1] + new[i])
        ok = kv[i] + new[i] <= width * ps and cu[-1] <= st["rows"]
        held, want = -(-kv[i] // ps), -(-(kv[i] + new[i]) // ps)
        if ok:
            asked += want - held
            ok = want == held or asked <= height
        granted.append(ok)
        if ok:
            for c in range(held, want):
                top -= 1
                table[i][c] = free[top]
            for j in range(new[i]):
                pos = kv[i] + j
                slots[cu[i] + j] = table[i][pos // ps] * ps + pos % ps
            kv[i] += new[i]
    return {"slots": torch.tensor(slots, dtype=torch.int64, device=DEV), "cu_rows": _i32(cu), "granted": torch.tensor(granted, device=DEV),
            "kv_lens": _i32(kv), "free_count": _i32([top]), "table": _i32(table), "free_pages": _i32(free)}


def _exact_write(st, case):
    ps = case["page"]
    kp, vp = st["kp"].double(), st["vp"].double()
    keep = torch.nonzero(st["slots"] >= 0).flatten()
    page, off = st["slots"][keep] // ps, st["slots"][keep] % ps
    for h in range(case["kv_heads"]):
        kp[:, h].index_put_((page, off), st["k"][keep, h].double())
        vp[:, h].index_put_((page, off), st["v"][keep, h].double())
    return {"k_pages": kp, "v_pages": vp}


def _exact_attn(st, case):
    if work(case)["flops"] > 2e12:
        return None
    hk, g, d, ps = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, kv) in enumerate(zip(st["new"], st["kv"])):
        pages = st["table"][b, :-(-kv // ps)].long()
        for h in range(hk):
            k = st["kp"][pages, h].reshape(-1, d)[:kv].double()
            v = st["vp"][pages, h].reshape(-1, d)[:kv].double()
            for r0 in range(0, n, 1024):
                r1 = min(n, r0 + 1024)
                pos = torch.arange(kv - n + r0, kv - n + r1, device=DEV)
                # keys that no row of this piece sees have no part in its sums
                lo = max(0, kv - n + r0 - case["window"] + 1) if case["window"] else 0
                key = torch.arange(kv, device=DEV)
                key = key[(key >= lo) | (key < case["sinks"])]
                see = torch.ones((r1 - r0, key.numel()), dtype=torch.bool, device=DEV)
                if case["causal"]:
                    see &= key <= pos[:, None]
                if case["window"]:
                    see &= (key + case["window"] > pos[:, None]) | (key < case["sinks"])
                kk, vv = k[key], v[key]
                for c in range(h * g, (h + 1) * g):
                    s = (st["q"][at + r0:at + r1, c].double() @ kk.t()) * st["scale"]
                    out[at + r0:at + r1, c] = torch.softmax(s.masked_fill(~see, -math.inf), 1) @ vv
        at += n
    return out


def _exact_sample(st, case):
    x = st["logits"].double().cpu()
    rows, vocab = x.shape
    par = {k: st[k].double().cpu().tolist() if st[k] is not None else None for k in ("u", "temperature", "top_k", "top_p", "min_p")}
    tokens = []
    for r in range(rows):
        t = par["temperature"][r]
        row = x[r]
        if not t > 0:
            tokens.append(int((row == row.max()).nonzero()[0]))
            continue
        w = torch.exp((row - row.max()) / t)
        order = torch.argsort(row, descending=True, stable=True)
        kept = order
        if par["top_k"] and par["top_k"][r] > 0:
            kept = kept[:int(par["top_k"][r])]
        if par["top_p"] and par["top_p"][r] < 1:
            mass = torch.cat([torch.zeros(1, dtype=torch.float64), w[kept].cumsum(0)])
            count = int((mass[:-1] < par["top_p"][r] * mass[-1]).sum())
            kept = kept[:max(1, count)]
        if par["min_p"] and par["min_p"][r] > 0:
            kept = kept[w[kept] >= min(par["min_p"][r], 1.0)]
        kept = torch.sort(kept).values
        mass = w[kept].cumsum(0)
        hit = int(torch.searchsorted(mass, par["u"][r] * mass[-1], right=True))
        tokens.append(int(kept[min(hit, kept.numel() - 1)]))
    return _i32(tokens)
