"""The serving operators on the GPU (page plan, page write, attention over pages, token sampling, the cache that joins
them) against the 64-bit oracle, at the lengths, masks and layouts where they can go wrong.

Tolerances.  One rounding is off by at most half a step (2^-8 relative for bf16, 2^-24 for fp32).  An attention output is
sum_j p_j v_j / sum_j p_j.  With mag = sum_j p_j |v_j| (normalised p): a relative error e of the p_j moves it by at most
2 e mag, the rounding of p to the storage type by half a step times mag, the sums over n keys by n 2^-24 mag each for
numerator and denominator, the last rounding by half a step of the value.  The error of p comes from the score: D products summed in fp32,
(D + 2) 2^-24 scale |q| |k| at most, and from exp2 of a number of size |s| log2(e): 2^-22 (|s| + 1)."""
import math

import pytest
import torch

from conformer_amd import KVPages, _native as N, ops
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _tables(kv_lens, page, width, pool, gen):
    """Pages scattered over the pool; entries past a request's pages are garbage that must not be followed."""
    perm = torch.randperm(pool, generator=gen).tolist()
    table, at = [], 0
    for k in kv_lens:
        c = -(-max(0, k) // page)
        table.append(perm[at:at + c] + [(-1, 10 ** 9, -2 ** 31)[len(table) % 3]] * (width - c))
        at += c
    return table


def _problem(dtype, h, hk, d, page, new, kv, seed, tail=0, extra_width=2):
    gen = torch.Generator().manual_seed(seed)
    pool = sum(-(-max(0, k) // page) for k in kv) + 3
    width = max(1, -(-max(kv) // page)) + extra_width
    table = _tables(kv, page, width, pool, gen)
    # every slot that no request holds is NaN: pages of nobody, slots behind a length
    kp = torch.full((pool, hk, page, d), math.nan)
    vp = torch.full((pool, hk, page, d), math.nan)
    for b, k in enumerate(kv):
        for j in range(0, max(0, k), page):
            n = min(page, k - j)
            pg = table[b][j // page]
            kp[pg, :, :n] = torch.randn(hk, n, d, generator=gen)
            vp[pg, :, :n] = torch.randn(hk, n, d, generator=gen)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + tail, h, d, generator=gen)
    return [t.to(dtype) for t in (q, kp, vp)] + [table, cu]


def _check(got, q, kp, vp, table, kv, cu, scale, dtype, **mask):
    fin = lambda t: torch.nan_to_num(t.float(), nan=0.0)
    want, mag = S.page_attention(q, kp, vp, table, kv, cu, scale, **mask)
    d = q.shape[2]
    qk = fin(q).norm(dim=2).max() * fin(kp).norm(dim=3).max() * scale
    p_err = (d + 2) * 2.0 ** -24 * qk + 2.0 ** -22 * (qk + 1)
    tol = mag * (2 * p_err + HALF[dtype] + 2 * max(kv) * 2.0 ** -24) + HALF[dtype] * want.abs() + 1e-30
    err = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    bad = err > tol
    assert not bad.any(), (bad.nonzero()[:4].tolist(), (err / tol).max().item())


def _run(q, kp, vp, table, kv, cu, scale, window=0, sinks=0, causal=True, max_rows=0):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    return ops.kv_page_attention(q.cuda(), kp.cuda(), vp.cuda(), i32(table), i32(kv), i32(cu), scale, window, sinks, causal, max_rows)


# lengths of (chunk, cache): nothing at all, one token, tokens at the borders of 16 / 32 / 64-token tiles and pages, a chunk
# that is the whole request, a chunk longer than what the request holds (rows in front of its start see nothing)
LENGTHS = [(0, 0), (1, 1), (1, 0), (2, 16), (1, 17), (0, 40), (3, 31), (5, 5), (1, 64), (4, 65), (7, 3), (33, 70), (1, 129)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h,hk,d,page", [(4, 4, 64, 16), (8, 2, 128, 32), (6, 2, 48, 16), (7, 1, 72, 64), (2, 2, 8, 16),
                                         (40, 1, 128, 128), (18, 1, 40, 16)])
@pytest.mark.parametrize("mask", [dict(), dict(causal=False), dict(window=20), dict(window=1), dict(window=9, sinks=3),
                                  dict(window=33, sinks=40, causal=False)])
def test_attention_mixed_batch(dtype, h, hk, d, page, mask):
    new, kv = [n for n, _ in LENGTHS], [k for _, k in LENGTHS]
    q, kp, vp, table, cu = _problem(dtype, h, hk, d, page, new, kv, 3, tail=2)
    got = _run(q, kp, vp, table, kv, cu, d ** -0.5, **mask)
    assert (got[cu[-1]:] == 0).all()                       # rows of nobody
    _check(got[:cu[-1]], q[:cu[-1]], kp, vp, table, kv, cu, d ** -0.5, dtype, **mask)
    assert torch.equal(got, _run(q, kp, vp, table, kv, cu, d ** -0.5, **mask))


@pytest.mark.parametrize("dtype,h,hk,d,new,kv,mask", [
    (torch.bfloat16, 4, 2, 128, [130, 1], [700, 300], dict()),                       # a long chunk beside a single token
    (torch.bfloat16, 4, 4, 64, [190], [190], dict(window=50, sinks=4)),              # a prompt
    (torch.float32, 2, 1, 64, [75], [333], dict(window=100, sinks=1)),
    (torch.float32, 3, 1, 128, [50, 9], [50, 411], dict(causal=False)),
    (torch.bfloat16, 8, 1, 96, [1], [4100], dict()),                                 # one row, a long axis: split and joined
    (torch.bfloat16, 2, 2, 64, [1, 1], [2500, 30], dict(window=2000, sinks=70)),
    (torch.float32, 8, 2, 128, [1], [3000], dict()),
    (torch.bfloat16, 2, 1, 128, [20], [2600], dict()),
    (torch.bfloat16, 16, 1, 64, [40], [1400], dict())])                              # a chunk whose axis is split
def test_attention_long(dtype, h, hk, d, new, kv, mask):
    q, kp, vp, table, cu = _problem(dtype, h, hk, d, 32, new, kv, 5, extra_width=40)
    _check(_run(q, kp, vp, table, kv, cu, d ** -0.5, **mask), q, kp, vp, table, kv, cu, d ** -0.5, dtype, **mask)


@pytest.mark.parametrize("max_rows", [1, 2, 40, 1000])
def test_attention_hint_changes_nothing_but_speed(max_rows):
    new, kv = [1, 40, 3], [90, 140, 3]
    q, kp, vp, table, cu = _problem(torch.bfloat16, 8, 2, 64, 16, new, kv, 7)
    got = _run(q, kp, vp, table, kv, cu, 0.2, max_rows=max_rows)
    _check(got, q, kp, vp, table, kv, cu, 0.2, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [8, 32, 56, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("mask", [dict(), dict(window=100, sinks=70), dict(causal=False)])
def test_attention_chunks_of_every_width(dtype, d, mask):
    """Whole tiles of 64 tokens between ragged ones, at head dims that fill a row of the padded width and that do not."""
    new, kv = [70, 33], [300, 257]
    q, kp, vp, table, cu = _problem(dtype, 4, 2, d, 64, new, kv, 23)
    _check(_run(q, kp, vp, table, kv, cu, d ** -0.5, **mask), q, kp, vp, table, kv, cu, d ** -0.5, dtype, **mask)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("extra_width", [40, 300])          # 24 pieces of the key axis at most, and 50
@pytest.mark.parametrize("mask", [dict(), dict(window=3000, sinks=33)])
def test_attention_pieces_by_length(dtype, extra_width, mask):
    """Chunks and single tokens, long requests whose key axis is cut and short ones whose is not, empty ones and rows of nobody, in
    one call."""
    new, kv = [40, 1, 0, 3, 60, 2, 33, 1], [5000, 4000, 900, 20, 60, 3000, 700, 1]
    q, kp, vp, table, cu = _problem(dtype, 8, 1, 64, 32, new, kv, 29, tail=3, extra_width=extra_width)
    got = _run(q, kp, vp, table, kv, cu, 0.125, **mask)
    assert (got[cu[-1]:] == 0).all()
    _check(got[:cu[-1]], q[:cu[-1]], kp, vp, table, kv, cu, 0.125, dtype, **mask)
    assert torch.equal(got, _run(q, kp, vp, table, kv, cu, 0.125, **mask))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("max_rows", [0, 40])
def test_attention_small_step_of_a_large_table(dtype, max_rows):
    """Few of many requests bring rows, short ones and chunks, all of them with a key axis that is cut."""
    new, kv = [0] * 200, [0] * 200
    for b, n, k in ((5, 1, 5000), (60, 40, 3000), (61, 2, 2000), (100, 4, 4100), (101, 5, 2500), (199, 1, 20)):
        new[b], kv[b] = n, k
    q, kp, vp, table, cu = _problem(dtype, 8, 1, 64, 32, new, kv, 37, tail=2, extra_width=100)
    got = _run(q, kp, vp, table, kv, cu, 0.125, max_rows=max_rows)
    assert (got[cu[-1]:] == 0).all()
    _check(got[:cu[-1]], q[:cu[-1]], kp, vp, table, kv, cu, 0.125, dtype)


@pytest.mark.parametrize("longest", [1, 40])
def test_attention_time_follows_the_rows_not_the_table(longest):
    """The same 64 rows in a table of 64 requests and in one of 16384, where workgroups for every request would take 20 ms."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    kp = torch.randn(64, 8, 64, 128, device="cuda").bfloat16()
    q = torch.randn(64, 32, 128, device="cuda").bfloat16()
    times = []
    for batch in (64, 16384):
        new, kv = [0] * batch, [0] * batch
        for i in range(64 - longest + 1):
            new[i], kv[i] = (longest, 2000) if i == 3 else (1, 500)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        args = q, kp, kp, torch.randint(0, 64, (batch, 512), dtype=torch.int32).cuda(), i32(kv), i32(cu), 0.09, 0, 0, True, longest
        marks = [torch.cuda.Event(enable_timing=True) for _ in range(8)]
        for m in marks:
            ops.kv_page_attention(*args)
            m.record()
        torch.cuda.synchronize()
        times.append(min(a.elapsed_time(b) for a, b in zip(marks, marks[1:])))
    assert times[1] < 5 * times[0] + 0.1, times


@pytest.mark.parametrize("h,hk,d", [(8, 2, 128), (4, 4, 64), (3, 1, 40), (32, 1, 96)])
@pytest.mark.parametrize("mask", [dict(), dict(window=30, sinks=3)])
def test_attention_of_single_tokens_keeps_the_probabilities(h, hk, d, mask):
    """Up to 32 rows times heads per kv head in bf16: the p_j are two bf16 numbers each, the first off by less than a whole step (2^-7),
    the second, that difference, by half a step of it: 2^-15 before the last rounding instead of 2^-8."""
    new, kv = [1, 1, 1, 1, 1], [2, 33, 70, 900, 2100]
    q, kp, vp, table, cu = _problem(torch.bfloat16, h, hk, d, 32, new, kv, 41)
    got = _run(q, kp, vp, table, kv, cu, d ** -0.5, **mask)
    fin = lambda t: torch.nan_to_num(t.float(), nan=0.0)
    want, mag = S.page_attention(q, kp, vp, table, kv, cu, d ** -0.5, **mask)
    qk = fin(q).norm(dim=2).max() * fin(kp).norm(dim=3).max() * d ** -0.5
    p_err = (d + 2) * 2.0 ** -24 * qk + 2.0 ** -22 * (qk + 1)
    tol = mag * (2 * p_err + 2.0 ** -15 + 2 * max(kv) * 2.0 ** -24) + 2.0 ** -8 * want.abs() + 1e-30
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), (err / tol).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv", [50, 2500])
def test_attention_of_single_tokens_keeps_infinite_values(dtype, kv):
    q, kp, vp, table, cu = _problem(dtype, 4, 2, 64, 32, [1], [kv], 43)
    want = _run(q, kp, vp, table, [kv], cu, 0.125)
    vp[table[0][1], 0, 2, 5], vp[table[0][0], 1, 7, 60] = math.inf, -math.inf
    want[0, :2, 5], want[0, 2:, 60] = math.inf, -math.inf
    assert torch.equal(_run(q, kp, vp, table, [kv], cu, 0.125), want)


def test_attention_extreme_windows_and_unit_dimensions():
    """A window of 2^31 - 1 tokens is none, also where rows in front of the request's start share a tile with others; strides of
    dimensions of one element are not looked at."""
    new, kv = [7, 50], [3, 41]
    q, kp, vp, table, cu = _problem(torch.bfloat16, 2, 1, 64, 16, new, kv, 19)
    want = _run(q, kp, vp, table, kv, cu, 0.125)
    for causal in (True, False):
        got = _run(q, kp, vp, table, kv, cu, 0.125, window=2 ** 31 - 1, sinks=2 ** 31 - 1, causal=causal)
        _check(got, q, kp, vp, table, kv, cu, 0.125, torch.bfloat16, causal=causal)
        assert torch.equal(got, want) or not causal
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    odd = lambda t: t.cuda().as_strided(t.shape, (t.stride(0), 3, t.stride(2), 1))           # one kv head
    one = q[:1, :1].cuda().as_strided((1, 1, 64), (5, 7, 1))                                   # one row, one head
    got = ops.kv_page_attention(one, odd(kp), odd(vp), i32(table[1:]), i32([41]), i32([0, 1]), 0.125)
    _check(got, q[:1, :1], kp, vp, table[1:], [41], [0, 1], 0.125, torch.bfloat16)
    k = torch.randn(1, 1, 64).bfloat16().cuda()
    kc, vc = kp.cuda(), vp.cuda()
    ops.kv_page_write_(k.as_strided((1, 1, 64), (1, 1, 1)), k, odd(kc), odd(vc), torch.tensor([16 * table[0][0] + 5]).cuda())


@pytest.mark.parametrize("many", [63, 64, 66, 70, 300, 4200, 4280])
def test_attention_many_requests(many):
    """The search for a tile's request over more than 64 and more than 4096 of them, with empty ones among them."""
    new = [(i * 7) % 3 if many < 1000 else int(i % 97 == 5 or many > 4200) for i in range(many)]
    kv = [n + (i * 5) % 20 for i, n in enumerate(new)]
    q, kp, vp, table, cu = _problem(torch.bfloat16, 2, 1, 16, 16, new, kv, 9)
    _check(_run(q, kp, vp, table, kv, cu, 0.25), q, kp, vp, table, kv, cu, 0.25, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 60])
def test_attention_bad_pages_are_not_seen(dtype, n):
    new, kv = [n, n], [200, 100]
    q, kp, vp, table, cu = _problem(dtype, 4, 2, 64, 16, new, kv, 11)
    table[0][2], table[0][7], table[1][0] = -1, kp.shape[0], 2 ** 31 - 1
    _check(_run(q, kp, vp, table, kv, cu, 0.125), q, kp, vp, table, kv, cu, 0.125, dtype)
    table[1] = [-5] * len(table[1])
    got = _run(q, kp, vp, table, kv, cu, 0.125)
    assert (got[n:] == 0).all()


@pytest.mark.parametrize("n", [1, 50])
def test_attention_non_finite_keys_that_nobody_sees(n):
    """Infinities and NaN in front of the window, and in the keys of later rows of the chunk, reach nobody."""
    kv = [300]
    q, kp, vp, table, cu = _problem(torch.bfloat16, 4, 2, 64, 16, [n], kv, 13)
    first_seen = 300 - n - 40 + 1
    for j in range(5, first_seen):
        kp[table[0][j // 16], :, j % 16] = (math.nan, math.inf, -math.inf)[j % 3]
        vp[table[0][j // 16], :, j % 16] = math.nan
    want = _run(q, kp, vp, table, kv, cu, 0.125, window=40, sinks=5)
    _check(want, q, kp, vp, table, kv, cu, 0.125, torch.bfloat16, window=40, sinks=5)
    if n > 1:
        kp[table[0][299 // 16], :, 299 % 16] = math.nan    # the last row's own key: NaN for that row alone
        got = _run(q, kp, vp, table, kv, cu, 0.125, window=40, sinks=5)
        assert torch.equal(got[:-1], want[:-1]) and torch.isnan(got[-1]).all()


def test_attention_visible_non_finite_values_show():
    q, kp, vp, table, cu = _problem(torch.bfloat16, 2, 2, 64, 16, [1, 1], [50, 2500], 15)
    kp[table[0][1], 0, 3] = math.nan                       # head 0 of request 0, and a split axis
    kp[table[1][100], 1, 0] = math.nan
    got = _run(q, kp, vp, table, [50, 2500], cu, 0.125).cpu()
    assert torch.isnan(got[0, 0]).all() and torch.isfinite(got[0, 1]).all()
    assert torch.isnan(got[1, 1]).all() and torch.isfinite(got[1, 0]).all()


@pytest.mark.parametrize("dtype,new", [(torch.bfloat16, [1, 3, 50]), (torch.float32, [2, 40, 1])])
def test_attention_strided_operands(dtype, new):
    """q inside a fused projection, pages whose slots lie token by token ([page][slot][head][dim]), a table with wider rows."""
    kv = [100, 37, 170]
    q, kp, vp, table, cu = _problem(dtype, 4, 2, 64, 16, new, kv, 17)
    n = q.shape[0]
    fused = torch.zeros(n, 8, 64, dtype=dtype)
    fused[:, 2:6] = q
    nhd = lambda t: t.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
    wide = torch.full((3, len(table[0]) + 5), 77, dtype=torch.int32)
    wide[:, :len(table[0])] = torch.tensor(table, dtype=torch.int32)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    got = ops.kv_page_attention(fused.cuda()[:, 2:6], nhd(kp), nhd(vp), wide.cuda()[:, :len(table[0])], i32(kv), i32(cu), 0.125)
    _check(got, q, kp, vp, table, kv, cu, 0.125, dtype)


def test_attention_and_write_past_32_bit_offsets():
    """A pool of more than 4 GiB per tensor: pages at its far end."""
    n_pages, ps, d = 290000, 64, 128
    kp = torch.empty(n_pages, 1, ps, d, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    assert kp.numel() * 2 > 2 ** 32
    g = torch.Generator().manual_seed(3)
    kv, pages = 150, [n_pages - 1, 3, n_pages - 2]
    k, v = (torch.randn(kv, 1, d, generator=g).bfloat16() for _ in range(2))
    slots = torch.tensor([pages[j // ps] * ps + j % ps for j in range(kv)])
    ops.kv_page_write_(k.cuda(), v.cuda(), kp, vp, slots.cuda())
    q = torch.randn(60, 4, d, generator=g).bfloat16()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    small = torch.zeros(3, 1, ps, d, dtype=torch.bfloat16), torch.zeros(3, 1, ps, d, dtype=torch.bfloat16)
    for t, src in zip(small, (k, v)):
        for j in range(kv):
            t[j // ps, 0, j % ps] = src[j, 0]
    for n in (2, 60):                                          # the kernels of short chunks and of long ones
        got = ops.kv_page_attention(q[:n].cuda(), kp, vp, i32([pages]), i32([kv]), i32([0, n]), 0.09)
        _check(got, q[:n], *small, [[0, 1, 2]], [kv], [0, n], 0.09, torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------
def _plan_state(seed, b, width, page, pool, new_max, with_finished):
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi, n=1: torch.randint(lo, hi + 1, (n,), generator=g).tolist()
    kv = [k if r(0, 3)[0] else 0 for k in r(0, width * page, b)]
    held = sum(-(-k // page) for k in kv)
    ids = torch.randperm(held + pool, generator=g).tolist()
    table, at = [], 0
    for k in kv:
        c = -(-k // page)
        table.append(ids[at:at + c] + [-1] * (width - c))
        at += c
    new = [n if r(0, 2)[0] else 0 for n in r(0, new_max, b)]
    fin = [r(0, 5)[0] == 0 for _ in range(b)] if with_finished else None
    free = ids[at:] + [-7] * held
    return kv, new, fin, table, free, pool


def _run_plan(kv, new, fin, table, free, count, page, rows):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    st = [i32(kv), i32(new), torch.tensor(fin).cuda() if fin is not None else None, i32(table), i32(free), i32([count])]
    slots, cu, granted = ops.kv_page_plan_(*st, page, rows)
    return dict(kv_lens=st[0].tolist(), table=st[3].tolist(), free_pages=st[4].tolist(), free_count=int(st[5]),
                slots=slots.tolist(), cu_rows=cu.tolist(), granted=granted.tolist())


@pytest.mark.parametrize("b,width,page,pool,new_max,fin", [
    (1, 4, 16, 5, 40, False), (7, 6, 16, 40, 30, True), (64, 5, 32, 90, 1, False), (64, 40, 16, 900, 300, True),
    (65, 8, 64, 20, 200, True), (300, 3, 128, 200, 60, True), (1024, 2, 16, 700, 2, True), (1500, 3, 16, 1200, 9, True),
    (130, 30, 16, 2500, 400, False), (20, 100, 1024, 60, 5000, True)])
@pytest.mark.parametrize("slack", [0, 37])
def test_plan(b, width, page, pool, new_max, fin, slack):
    for seed in (1, 2):
        kv, new, f, table, free, count = _plan_state(seed, b, width, page, pool, new_max, fin)
        rows = sum(new) + slack
        got, want = _run_plan(kv, new, f, table, free, count, page, rows), S.page_plan(kv, new, f, table, free, count, page, rows)
        for k in want:
            assert got[k] == want[k], k


def test_plan_limits():
    # more rows than the step has room for: the request that crosses the end is refused, and so are the later ones
    r = _run_plan([3, 0, 9], [5, 6, 2], None, [[0, -1], [-1, -1], [1, -1]], [5, 6, 7], 3, 16, 10)
    assert r == S.page_plan([3, 0, 9], [5, 6, 2], None, [[0, -1], [-1, -1], [1, -1]], [5, 6, 7], 3, 16, 10)
    assert r["granted"] == [True, False, False]
    # a later row is never served before an earlier one that waits, unless it needs nothing
    r = _run_plan([0, 0, 3, 0], [64, 10, 4, 1], None, [[-1] * 4, [-1] * 4, [9] + [-1] * 3, [-1] * 4], [1, 2], 2, 16, 79)
    assert r["granted"] == [False, False, True, False] and r["free_count"] == 2
    # negative lengths count as none, a length past the table refuses, an empty pool serves rows that need no page
    r = _run_plan([-4, 40, 5], [-1, 1, 3], None, [[-1, -1], [0, 1], [2, -1]], [3], 0, 16, 4)
    assert r["kv_lens"] == [0, 40, 8] and r["granted"] == [True, False, True] and r["cu_rows"] == [0, 0, 1, 4]
    assert r["slots"] == [-1, 37, 38, 39]
    # a stack that would pass the pool is cut off, never written past its end
    r = _run_plan([32, 32], [0, 0], [True, True], [[0, 1], [2, 3]], [7, 8, 9], 2, 16, 0)
    assert r["free_pages"] == [7, 8, 0] and r["free_count"] == 3 and r["slots"] == []


@pytest.mark.parametrize("dtype,h,d,page,n", [(torch.bfloat16, 8, 64, 16, 77), (torch.float32, 3, 48, 64, 130),
                                              (torch.bfloat16, 1, 8, 16, 1), (torch.float32, 5, 4, 32, 9), (torch.bfloat16, 2, 128, 256, 999)])
@pytest.mark.parametrize("packed", [False, True])
def test_write(dtype, h, d, page, n, packed):
    g = torch.Generator().manual_seed(n)
    pool = n // page + 3
    kp, vp = (torch.randn(pool, h, page, d, generator=g).to(dtype) for _ in range(2))
    qkv = torch.randn(n, 3 * h, d, generator=g).to(dtype).cuda()
    k, v = qkv[:, h:2 * h], qkv[:, 2 * h:]
    if not packed:
        k, v = k.contiguous(), v.contiguous()
    slots = torch.randperm(pool * page, generator=g)[:n]
    if n > 4:
        slots[1], slots[3], slots[4] = -1, pool * page, 2 ** 40          # nowhere
    got = kp.cuda(), vp.cuda()
    ops.kv_page_write_(k, v, *got, slots.cuda())
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < pool * page:
            kp[s // page, :, s % page], vp[s // page, :, s % page] = k[i].cpu(), v[i].cpu()
    assert torch.equal(got[0].cpu(), kp) and torch.equal(got[1].cpu(), vp)


# ---------------------------------------------------------------------------------------------------------------
def _sample(x, u, t=None, k=None, p=None, m=None):
    f = lambda v, dt: None if v is None else torch.tensor(v, dtype=dt).cuda()
    return ops.sample_tokens(x.cuda(), f(u, torch.float32), f(t, torch.float32), f(k, torch.int32), f(p, torch.float32),
                             f(m, torch.float32)).tolist()


def _want(x, u, t=None, k=None, p=None, m=None):
    f32 = lambda v: torch.tensor(v, dtype=torch.float32).double().tolist()
    at = lambda v, i, d: d if v is None else (f32(v)[i] if isinstance(v[i], float) else v[i])
    return [S.sample_token(x[i], f32(u)[i], at(t, i, 1.0), at(k, i, 0), at(p, i, 1.0), at(m, i, 0.0)) for i in range(len(u))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 29, 63, 512, 513, 1000, 4097, 9000])
@pytest.mark.parametrize("kind", ["flat", "peaked", "ties", "equal"])
def test_sampling(dtype, v, kind):
    g = torch.Generator().manual_seed(v)
    r = 12
    x = torch.randn(r, v, generator=g) * {"flat": 0.5, "peaked": 4.0, "ties": 2.0, "equal": 0.0}[kind]
    if kind == "ties":
        x = x.round()
    x = x.to(dtype)
    u = torch.rand(r, generator=g).tolist()
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    pick = lambda *o: [o[i] for i in torch.randint(0, len(o), (r,), generator=g).tolist()]
    for t, k, p, m in ((None, None, None, None), (pick(0.0, 0.5, 1.0, 2.0), None, None, None), (None, pick(1, 2, 5, 40, 500, 0, 10 ** 9), None, None),
                       (pick(0.7, 1.5), None, pick(0.0, 0.1, 0.5, 0.9, 0.999, 1.0), None), (None, None, None, pick(0.0, 0.02, 0.5, 1.0)),
                       (pick(0.8, 1.0), pick(3, 30, 300), pick(0.3, 0.8, 0.95), pick(0.0, 0.05))):
        assert _sample(x, u, t, k, p, m) == _want(x, u, t, k, p, m), (t, k, p, m)


def test_sampling_masked_and_non_finite_logits():
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    x = torch.tensor([[-inf, 1.0, -inf, 1.0, -inf], [nan, 0.0, nan, nan, 0.0], [-inf] * 5, [nan] * 5, [low] * 5, [low, 3.0, low, 3.0, low],
                      [inf, 0.0, inf, 1.0, -inf], [-0.0, 0.0, -0.0, -5.0, -inf]])
    u = [0.7] * 8
    assert _sample(x, u) == [3, 4, -1, -1, 3, 3, 2, 2] == _want(x, u)
    assert _sample(x, u, t=[0.0] * 8) == [1, 1, -1, -1, 0, 1, 0, 0]
    assert _sample(x, u, k=[2] * 8) == _want(x, u, k=[2] * 8) == [3, 4, -1, -1, 1, 3, 2, 1]
    assert _sample(x, u, k=[4] * 8, p=[0.9] * 8) == _want(x, u, k=[4] * 8, p=[0.9] * 8)
    b = torch.full((3, 70), torch.finfo(torch.bfloat16).min).bfloat16()
    b[1, 66] = 1.0
    b[2, :] = -inf
    assert _sample(b, [0.5] * 3) == [35, 66, -1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [8, 64, 700, 9001])
def test_sampling_when_top_k_reaches_masked_tokens(dtype, v):
    """Tokens masked with the type's lowest value or -inf, fewer others than k: the border lies at the far end of the keys
    (a range of keys that ends at the last one there is)."""
    g = torch.Generator().manual_seed(v)
    for fill in (torch.finfo(dtype).min, -math.inf, -1e4):
        for t in (0.1, 1.0):
            x = (torch.randn(6, v, generator=g) * 2.2).to(dtype)
            x[torch.rand(6, v, generator=g) < 0.4] = fill
            x[:, 0] = 1.0
            u, k = torch.rand(6, generator=g).tolist(), [max(1, v * 4 // 5)] * 6
            for m in (None, [0.01] * 6):
                assert _sample(x, u, [t] * 6, k, None, m) == _want(x, u, [t] * 6, k, None, m), (fill, t, m)


@pytest.mark.parametrize("v", [8192, 8193, 12345])
def test_sampling_long_bf16_rows_at_the_ends_of_the_value_range(v):
    """Values around 2^-30 and 2^7, zeros of both signs, large temperatures that give low values weight, filters that end
    inside equal values."""
    g = torch.Generator().manual_seed(v)
    r = 8
    u = torch.rand(r, generator=g).tolist()
    u[0] = 0.0
    rows = {"tiny": torch.randn(r, v, generator=g) * 2.0 ** -30, "huge": torch.randn(r, v, generator=g) * 60,
            "zeros": torch.where(torch.rand(r, v, generator=g) < 0.5, -0.0, 0.0), "below": -130 - torch.rand(r, v, generator=g),
            "low": torch.where(torch.rand(r, v, generator=g) < 0.3, -200.0, torch.randn(r, v, generator=g)),
            "edge": torch.tensor([127.5, -127.5, 2.0 ** -30, -2.0 ** -30, 0.0, 1.0, -1.0])[torch.randint(0, 7, (r, v), generator=g)],
            "steps": (torch.randn(r, v, generator=g) * 3).round()}
    for name, x in rows.items():
        x = x.bfloat16()
        for t, k, p, m in ((None, None, None, None), ([9.0] * r, None, [0.7] * r, None), (None, [v // 3] * r, [0.6] * r, [0.1] * r),
                           ([1.5] * r, [v - 1] * r, None, [1.0] * r), (None, None, [0.5, 0.05] * (r // 2), None)):
            assert _sample(x, u, t, k, p, m) == _want(x, u, t, k, p, m), (name, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [8192, 8193, 20000])
def test_sampling_at_u_zero_takes_a_token_of_any_weight(dtype, v):
    """u = 0 draws the first kept token whose weight is a number at all, also far below the units that sums are held in: logits at
    and below -2^7 in front of a long row."""
    x = torch.zeros(8, v)
    x[:, 0] = torch.tensor([-200.0, -128.0, -744.0, -760.0, -math.inf, -200.0, -200.0, -300.0])
    x[:, 1] = torch.tensor([0.0, 0.0, 0.0, -130.0, -700.0, 0.0, -150.0, -1.0])
    x = x.to(dtype)
    u = [0.0] * 8
    for t, k, p, m in ((None, None, None, None), ([0.5] * 8, None, None, None), ([0.1] * 8, None, None, None), ([math.inf] * 8, None, None, None),
                       (None, [v - 1] * 8, None, None), (None, None, [0.9] * 8, None), (None, None, None, [1e-30] * 8)):
        assert _sample(x, u, t, k, p, m) == _want(x, u, t, k, p, m), (t, k, p, m)
    assert _sample(x, u) == [0, 0, 0, 1, 1, 0, 0, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [50, 700, 9000])
def test_sampling_filters_that_are_nan_are_off(dtype, v):
    """In every form: few candidates and many, long rows and short ones."""
    g = torch.Generator().manual_seed(v)
    x = (torch.randn(8, v, generator=g) * 2).to(dtype)
    u, nan = torch.rand(8, generator=g).tolist(), [math.nan] * 8
    for k in (None, [40] * 8, [v // 2] * 8):
        assert _sample(x, u, None, k, nan, nan) == _sample(x, u, None, k) == _want(x, u, None, k), k
        assert _sample(x, u, nan, k) == _want(x, u, [0.0] * 8)           # a temperature that is not above 0: the first maximum


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("second,low,tops,lows,p", [(-0.5, -9.0, 35104, 11445, 0.9999597668647766), (-0.5, -11.0, 52562, 57777, 0.9999816417694092),
                                                    (-0.75, -9.0, 51295, 45541, 0.9998904466629028), (-1.5, -9.5, 48411, 14418, 0.999977707862854)])
def test_sampling_where_top_p_ends_at_a_rounded_sum(dtype, second, low, tops, lows, p):
    """`tops` logits of 0, one of `second`, `lows` of `low`: in units of 2^-46 the mass down to `second` passes 2^53, and p times the whole
    mass, as a double, equals that sum rounded up.  The last token that has any part in the kept mass is `second`'s (the first low one
    weighs less than 2^-24 of it)."""
    x = torch.full((1, 131072), -math.inf)
    x[0, :tops], x[0, tops], x[0, tops + 1:tops + 1 + lows] = 0.0, second, low
    assert _sample(x.to(dtype), [1 - 2.0 ** -24], None, None, [p]) == [tops]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampling_where_one_step_of_the_histogram_holds_too_many(dtype):
    """Thousands of equal logits, and thousands within one step: the candidate list does not fit."""
    n = 1 << 15
    x = torch.zeros(3, n)
    x[1] = torch.linspace(0, 1e-4, n)
    x[2, ::2] = 3.0
    x = x.to(dtype)
    u = [0.3, 0.6, 0.9]
    k, p = [20000, 25000, 9000], [0.7, 0.45, 0.99]
    for kk, pp in ((k, None), (None, p), (k, p)):
        got = _sample(x, u, None, kk, pp)
        # counted by hand: falling order, equal ones by index, weights 1 (rows 0, 2) or exp
        xd = x.double()
        for r in range(3):
            order = torch.argsort(xd[r], descending=True, stable=True)
            w = torch.exp(xd[r] - xd[r].max())
            kept = order[:kk[r]] if kk else order
            if pp:
                f = torch.tensor(pp[r], dtype=torch.float32).double()
                mass = w[kept].cumsum(0)
                kept = kept[:max(1, int((mass - w[kept] < f * mass[-1]).sum()))]
            kept = kept.sort().values
            run = w[kept].cumsum(0)
            uu = torch.tensor(u[r], dtype=torch.float32).double()
            assert got[r] == int(kept[int((run <= uu * run[-1]).sum())]), (r, kk, pp)


def test_sampling_under_a_transform():
    """A wrapped tensor goes through the dispatcher, which calls the operator slice by slice."""
    g = torch.Generator().manual_seed(8)
    x, u = torch.randn(3, 4, 50, generator=g).cuda(), torch.rand(4, generator=g).cuda()
    got = torch.func.vmap(lambda r: ops.sample_tokens(r, u))(x)
    assert torch.equal(got, torch.stack([ops.sample_tokens(r, u) for r in x]))


def test_lazily_negated_operands():
    """The imaginary part of a conjugate is a view whose memory holds the negative of its values."""
    u = torch.tensor([0.7j]).neg().cuda().conj().imag
    assert u.is_neg() and abs(float(u) - 0.7) < 1e-6
    row = torch.zeros(1, 10).cuda()
    # ten equal weights; 0.7 in fp32 is 0.69999999, and 7 > 6.9999999: the seventh
    assert ops.sample_tokens(row, u).tolist() == [6] == ops.sample_tokens.op(row, u).tolist()
    assert ops.sample_tokens(row, u, temperature=u, min_p=u).tolist() == [6]


def test_sampling_largest_vocabulary_and_strided_rows():
    n = 1 << 18
    assert _sample(torch.zeros(2, n), [0.5, 1 - 2.0 ** -24]) == [n // 2, n - 1]
    with pytest.raises(RuntimeError, match="vocabulary"):
        _sample(torch.zeros(1, n + 1), [0.5])
    g = torch.Generator().manual_seed(1)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(9, 1111, generator=g).to(dtype).cuda()
        x = wide[::2, 3:1004]                              # rows at every alignment of the type
        u = torch.rand(5, generator=g).tolist()
        assert ops.sample_tokens(x, torch.tensor(u).cuda(), None, torch.full((5,), 50, dtype=torch.int32).cuda()).tolist() == _want(x.cpu(), u, k=[50] * 5)


# ---------------------------------------------------------------------------------------------------------------
def _small_cache(pages=20, dtype=torch.float32):
    return KVPages(layers=2, pages=pages, kv_heads=2, head_dim=32, batch=4, max_tokens=80, page_size=16, dtype=dtype)


class _Model:
    """Two attention layers with a residual and a token head; every request's tokens kept on the host as well."""

    def __init__(self, vocab, h=4, hk=2, d=32, layers=2, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = h * d
        self.h, self.hk, self.d = h, hk, d
        self.emb = torch.randn(vocab, w, generator=g)
        self.qkv = [torch.randn(w, (h + 2 * hk) * d, generator=g) / w ** 0.5 for _ in range(layers)]
        self.out = [torch.randn(w, w, generator=g) / w ** 0.5 for _ in range(layers)]
        self.head = torch.randn(w, vocab, generator=g) / w ** 0.5

    def cuda(self):
        m = object.__new__(_Model)
        m.__dict__.update(self.__dict__, emb=self.emb.cuda(), qkv=[t.cuda() for t in self.qkv], out=[t.cuda() for t in self.out], head=self.head.cuda())
        return m

    def step(self, cache, tokens, **mask):
        x = self.emb[tokens]
        for i in range(len(self.qkv)):
            y = (x @ self.qkv[i]).view(x.shape[0], -1, self.d)
            cache.write(i, y[:, self.h:self.h + self.hk], y[:, self.h + self.hk:])
            x = x + cache.attend(i, y[:, :self.h], **mask).reshape(x.shape[0], -1) @ self.out[i]
        return x @ self.head

    def dense(self, tokens, window, sinks):
        """Logits of a whole token sequence in 64 bits."""
        n = len(tokens)
        x = self.emb[tokens].double()
        j = torch.arange(n)
        see = (j <= j[:, None]) & ((j > j[:, None] - window) | (j < sinks))
        for wq, wo in zip(self.qkv, self.out):
            y = (x @ wq.double()).view(n, -1, self.d).transpose(0, 1)
            g = self.h // self.hk
            q, k, v = y[:self.h], y[self.h:self.h + self.hk].repeat_interleave(g, 0), y[self.h + self.hk:].repeat_interleave(g, 0)
            s = (q @ k.transpose(1, 2) * self.d ** -0.5).masked_fill(~see, -math.inf).softmax(-1)
            x = x + (s @ v).transpose(0, 1).reshape(n, -1) @ wo.double()
        return x @ self.head.double()


def test_requests_come_and_go_through_the_cache():
    """Continuous batching: prompts and single tokens in one step, a request refused for want of pages and served later, rows
    reused; logits against a dense 64-bit model, tokens against the oracle's draw from the same logits."""
    vocab, mask = 61, dict(window=24, sinks=2)
    model = _Model(vocab)
    gpu, cache = model.cuda(), _small_cache(11)
    g = torch.Generator().manual_seed(5)
    text = [[], [], [], []]                                # tokens of each table row so far, the next one's input included
    # pages held after each step (16 tokens each, 11 in the pool): 2+2, 2+2+3, the same and 5 more wanted, 3+0+3+5, 2+0+3+5
    plans = [{0: 30, 1: 20}, {0: 1, 1: 1, 2: 40}, {0: 1, 1: 1, 2: 1, 3: 70}, {0: 1, 2: 1, 3: 70}, {0: 17, 2: 1, 3: 1}]
    finish = {3: [1], 4: [0]}                              # at 4 row 0 ends and a new request begins in it
    waiting = 0
    for t, plan in enumerate(plans):
        fin = [b in finish.get(t, ()) for b in range(4)]
        new = [plan.get(b, 0) for b in range(4)]
        for b in range(4):
            if fin[b]:
                text[b] = []
            if new[b] > 1 or (new[b] and not text[b]):     # a prompt
                text[b] = torch.randint(0, vocab, (new[b],), generator=g).tolist()
        rows = sum(new) + 3                                # capacity of the step
        held = cache.kv_lens.tolist()
        step = cache.plan(torch.tensor(new, dtype=torch.int32).cuda(), rows, torch.tensor(fin).cuda() if any(fin) else None)
        feed = []
        for b in range(4):
            feed += text[b][len(text[b]) - new[b]:]
        logits = gpu.step(cache, torch.tensor(feed + [0] * 3).cuda(), **mask)
        u = torch.rand(rows, generator=g)
        tokens = ops.sample_tokens(logits, u.cuda(), None, torch.full((rows,), 20, dtype=torch.int32).cuda(), torch.full((rows,), 0.9).cuda()).tolist()
        granted, cu = step.granted.tolist(), step.cu_rows.tolist()
        assert cache.kv_lens.tolist() == [(0 if fin[b] else held[b]) + (new[b] if granted[b] else 0) for b in range(4)]
        for b in range(4):
            if not new[b]:
                continue
            if not granted[b]:
                waiting += 1
                continue
            last = cu[b + 1] - 1
            want = model.dense(text[b], **mask)[-1]
            assert (logits[last].cpu().double() - want).abs().max() < 1e-4 * want.abs().max()
            assert tokens[last] == S.sample_token(logits[last].cpu(), float(u[last]), 1.0, 20, float(torch.tensor(0.9)))
            text[b].append(tokens[last])
    assert waiting == 1                                    # the prompt of 70 had to wait for the pages of a finished row
    assert sorted(cache.free_pages.tolist()[:int(cache.free_count)] + [p for b in range(4) for p in cache.block_table[b].tolist()[:-(-int(cache.kv_lens[b]) // 16)]]) == list(range(11))


def test_a_captured_step_advances_the_cache_on_every_replay():
    model = _Model(37, seed=2)
    gpu = model.cuda()
    caches = [_small_cache() for _ in range(2)]
    new = torch.ones(4, dtype=torch.int32).cuda()
    new[3] = 0
    last = [torch.tensor([5, 6, 7, 0]).cuda() for _ in caches]      # one input row per request, row 3 belongs to nobody
    u = torch.rand(40, 4, generator=torch.Generator().manual_seed(3)).cuda()
    u_now = [u[0].clone() for _ in caches]

    def step(i):
        caches[i].plan(new, 4)
        tok = ops.sample_tokens(gpu.step(caches[i], last[i]), u_now[i])
        last[i].copy_(tok.clamp(min=0).long())
        return tok

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for i in range(2):
            step(i)                                                  # eager, on a stream that is not the tensors' own
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(0)
    for t in range(1, 40):
        for w in u_now:
            w.copy_(u[t])
        graph.replay()
        want = step(1)
        noise = torch.randn(1 << 16, device="cuda").sum()            # the program's own work in between
        assert torch.equal(got, want), t
        assert torch.equal(caches[0].kv_lens, caches[1].kv_lens) and torch.equal(caches[0].block_table, caches[1].block_table)
        first = [c.k_pages[:, c.block_table[0, 0], :, :min(16, t + 1)] for c in caches]      # slots beyond were never written
        assert torch.equal(*first)
    assert caches[0].kv_lens.tolist() == [40, 40, 40, 0] and torch.isfinite(noise)


def test_two_graphs_do_not_share_a_workspace():
    """Split key axes need a workspace: two captured calls with other inputs, replayed in turn."""
    cases = []
    for seed in (1, 2):
        q, kp, vp, table, cu = _problem(torch.bfloat16, 4, 1, 64, 16, [1], [1500], seed)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
        cases.append([q.cuda(), kp.cuda(), vp.cuda(), i32(table), i32([1500]), i32(cu)])
    want = [ops.kv_page_attention(*c, 0.125) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.kv_page_attention(*c, 0.125))
        graphs.append(gr)
    for _ in range(3):
        for gr in graphs:
            gr.replay()
        torch.randn(1000, device="cuda").sum()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()                  # and two at once
    torch.cuda.synchronize()
    res = []
    for _ in range(4):
        for s, c in zip((a, b), cases):
            with torch.cuda.stream(s):
                res.append(ops.kv_page_attention(*c, 0.125))
    torch.cuda.synchronize()
    for i, r in enumerate(res):
        assert torch.equal(r, want[i % 2])


def test_a_captured_chunk_call_follows_its_lengths():
    """One captured call, replayed for batches in which the same requests bring single tokens, chunks, prompts or nothing: which kernel
    takes a request and how its key axis is cut is found on the device."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    most = [1500, 900, 700, 1100]
    q, kp, vp, table, _ = _problem(torch.bfloat16, 8, 2, 64, 32, [30, 30, 30, 30], most, 31)
    kv, cu = i32(most), i32([0, 30, 60, 90, 120])
    args = q.cuda(), kp.cuda(), vp.cuda(), i32(table), kv, cu, 0.125
    ops.kv_page_attention(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.kv_page_attention(*args)
    for new, lens in (([30, 30, 30, 30], most), ([1, 1, 1, 1], [1500, 1, 33, 1100]), ([90, 0, 1, 20], [90, 0, 700, 1100]),
                      ([0, 0, 0, 0], [0, 0, 0, 0]), ([2, 100, 3, 15], [1400, 900, 3, 15])):
        starts = [sum(new[:i]) for i in range(5)]
        kv.copy_(i32(lens))
        cu.copy_(i32(starts))
        graph.replay()
        assert torch.equal(got, ops.kv_page_attention(*args))
        assert (got[starts[-1]:] == 0).all()
        if starts[-1]:
            _check(got[:starts[-1]], q[:starts[-1]], kp, vp, table, lens, starts, 0.125, torch.bfloat16)


def test_refusals():
    q, kp, vp, table, cu = _problem(torch.bfloat16, 4, 2, 64, 16, [2, 1], [20, 30], 1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    a = dict(q=q.cuda(), k_pages=kp.cuda(), v_pages=vp.cuda(), block_table=i32(table), kv_lens=i32([20, 30]), cu_rows=i32(cu), scale=0.125)
    call = lambda **k: ops.kv_page_attention(**{**a, **k})
    call()
    for bad, exc in ((dict(q=a["q"].float()), TypeError), (dict(q=a["q"].half(), k_pages=a["k_pages"].half(), v_pages=a["v_pages"].half()), ValueError),
                     (dict(q=a["q"][..., :32]), ValueError), (dict(q=a["q"][0]), ValueError), (dict(v_pages=a["v_pages"][1:]), ValueError),
                     (dict(kv_lens=i32([20])), ValueError), (dict(cu_rows=i32([0, 3])), ValueError), (dict(kv_lens=a["kv_lens"].long()), TypeError),
                     (dict(block_table=a["block_table"].cpu()), RuntimeError), (dict(scale=0.0), RuntimeError), (dict(scale=math.nan), RuntimeError),
                     (dict(window=-1), RuntimeError), (dict(sinks=-2), RuntimeError), (dict(q=a["q"][:, :3]), RuntimeError),
                     (dict(q=a["q"].transpose(1, 2)), ValueError), (dict(k_pages=a["k_pages"][:, :, :10], v_pages=a["v_pages"][:, :, :10]), RuntimeError),
                     (dict(q=a["q"].clone().requires_grad_()), RuntimeError),
                     (dict(q=torch.zeros(3 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 4, 64)), RuntimeError)):
        with pytest.raises(exc):
            call(**bad)
    assert call(q=a["q"][:0], cu_rows=i32([0, 0, 0])).shape == (0, 4, 64)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    sl = torch.arange(3).cuda()
    for bad, exc in (((k.float(), k, a["k_pages"], a["v_pages"], sl), TypeError), ((k[:2], k, a["k_pages"], a["v_pages"], sl), ValueError),
                     ((k, k[:, :1], a["k_pages"], a["v_pages"], sl), ValueError), ((k, k, a["k_pages"], a["v_pages"], sl.int()), TypeError),
                     ((k, k, a["k_pages"], a["v_pages"], sl.cpu()), RuntimeError)):
        with pytest.raises(exc):
            ops.kv_page_write_(*bad)
    p = [i32([0, 0]), i32([1, 1]), None, i32([[-1] * 3] * 2), i32([0, 1]), i32([2])]
    for i, bad, exc in ((0, i32([0]), ValueError), (1, i32([1, 1, 1]), ValueError), (2, torch.zeros(1, dtype=torch.bool).cuda(), ValueError),
                        (2, i32([0, 0]), TypeError), (5, i32([2, 2]), ValueError), (3, i32([0]), ValueError), (4, i32([]), ValueError)):
        with pytest.raises(exc):
            ops.kv_page_plan_(*[bad if j == i else t for j, t in enumerate(p)], 16, 2)
    for page, rows in ((20, 2), (16, -1)):
        with pytest.raises((RuntimeError, ValueError)):
            ops.kv_page_plan_(*p, page, rows)
    x, u = torch.zeros(2, 9).cuda(), torch.zeros(2).cuda()
    for bad, exc in (((x.half(), u), ValueError), ((x, u[:1]), ValueError), ((x, u.double()), TypeError), ((x, u, u[:1]), ValueError),
                     ((x, u, None, u), TypeError), ((x[:, :0], u), ValueError), ((x.t(), torch.zeros(9).cuda()), ValueError),
                     ((x.clone().requires_grad_(), u), RuntimeError), ((x, u.cpu()), RuntimeError)):
        with pytest.raises(exc):
            ops.sample_tokens(*bad)
    assert ops.sample_tokens(x[:0], u[:0]).shape == (0,)
    with torch.no_grad():
        assert ops.sample_tokens(x.clone().requires_grad_(), u).tolist() == [0, 0]


def test_operands_that_require_a_gradient_are_refused_wherever_they_stand():
    x, u = torch.zeros(2, 9).cuda(), torch.full((2,), 0.5).cuda()
    t = torch.ones(2).cuda().requires_grad_()
    for call in (ops.sample_tokens, ops.sample_tokens.op):
        for args in ((x, t), (x, u, t), (x, u, None, None, t), (x, u, None, None, None, t), (x.clone().requires_grad_(), u)):
            with pytest.raises(RuntimeError, match="backward"):
                call(*args)
            with torch.no_grad():
                call(*args)
        assert call(x, u).tolist() == [4, 4]
    pages = torch.zeros(2, 1, 16, 8).cuda()
    k, slots = torch.ones(1, 1, 8).cuda(), torch.zeros(1, dtype=torch.int64).cuda()
    for call in (ops.kv_page_write_, ops.kv_page_write_.op):
        for args in ((k.clone().requires_grad_(), k, pages, pages, slots), (k, k, pages, pages.clone().requires_grad_(), slots)):
            with pytest.raises(RuntimeError, match="backward"):
                call(*args)
