"""CPU side of the serving operators: the 64-bit oracle against independent forms, refusals of the C entry points (which
return before any launch), operand refusals, shape functions."""
import ctypes as C
import math

import pytest
import torch

from conformer_amd import KVPages, _native as N, ops
from oracle import serving_oracle as S


def test_oracle_attention_is_softmax_attention():
    g = torch.Generator().manual_seed(1)
    hk, ps, d, kv = 2, 16, 8, 37
    kp, vp = torch.randn(5, hk, ps, d, generator=g), torch.randn(5, hk, ps, d, generator=g)
    table = [[3, 0, 4, -1]]
    q = torch.randn(kv, 4, d, generator=g)
    out, mag = S.page_attention(q, kp, vp, table, [kv], [0, kv], 0.4)
    k = kp[[3, 0, 4]].permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :kv].repeat_interleave(2, 0)
    v = vp[[3, 0, 4]].permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :kv].repeat_interleave(2, 0)
    s = torch.einsum("nhd,hjd->hnj", q.double(), k.double()) * 0.4
    s = s.masked_fill(torch.ones(kv, kv).triu(1).bool(), -math.inf).softmax(-1)
    want = torch.einsum("hnj,hjd->nhd", s, v.double())
    assert (out - want).abs().max() < 1e-12 and (mag >= out.abs() - 1e-12).all()
    # a window of one token and no sinks: every row returns its own value; nothing in a page outside the pool is seen
    out, _ = S.page_attention(q, kp, vp, table, [kv], [0, kv], 0.4, window=1)
    assert (out - v.double().permute(1, 0, 2)).abs().max() < 1e-12
    out, _ = S.page_attention(q[:1], kp, vp, [[5, 9, 4, -1]], [16], [0, 1], 0.4)
    assert (out == 0).all()


def test_oracle_plan_by_hand():
    r = S.page_plan([5, 16, 40], [11, 1, 1], [False, False, True], [[7, -1], [2, -1], [3, 1]], [9, 8, -1, -1], 2, 16, 13)
    # row 2 gives back 3, 1 and 40 is clipped to nothing; row 0 fits its page; row 1 takes page 1, row 2 page 3
    assert r["granted"] == [True, True, True] and r["kv_lens"] == [16, 17, 1]
    assert r["table"] == [[7, -1], [2, 1], [3, 1]] and r["free_count"] == 2 and r["free_pages"] == [9, 8, 3, 1]
    assert r["slots"] == [7 * 16 + i for i in range(5, 16)] + [16, 48] and r["cu_rows"] == [0, 11, 12, 13]


def test_oracle_sampling_by_hand():
    x = torch.log(torch.tensor([0.1, 0.4, 0.3, 0.2]))
    pick = lambda u, **k: S.sample_token(x, u, **k)
    assert [pick(u) for u in (0.0, 0.099, 0.101, 0.499, 0.51, 0.79, 0.81, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [pick(u, top_k=2) for u in (0.0, 0.56, 0.58)] == [1, 1, 2]
    assert [pick(u, top_p=0.5) for u in (0.0, 0.999)] == [1, 2] and pick(0.99, top_p=0.39) == 1
    assert pick(0.999, min_p=0.6) == 2 and pick(0.99, min_p=0.8) == 1 and pick(0.7, temperature=0.0) == 1
    assert S.sample_token(torch.tensor([2.0, 2.0, 2.0]), 0.99, top_k=2) == 1
    assert S.sample_token(torch.tensor([-math.inf, math.nan]), 0.5) == -1


def _err(rc):
    assert rc == -1
    return N.lib().fcenc_last_error().decode()


def test_c_entry_refusals_return_before_any_launch():
    lib, p = N.lib(), 4096                       # p: an aligned non-null address that nothing may touch
    plan = lambda **k: lib.fcenc_page_plan(*[{**dict(kv=p, new=p, fin=None, B=4, t=p, row=8, w=8, f=p, c=p, pool=9, ps=16,
                                                     slots=p, rows=4, cu=p, g=p, s=None), **k}[n]
                                             for n in ("kv", "new", "fin", "B", "t", "row", "w", "f", "c", "pool", "ps",
                                                       "slots", "rows", "cu", "g", "s")])
    assert "empty batch" in _err(plan(B=0)) and "empty batch" in _err(plan(pool=0)) and "empty batch" in _err(plan(rows=-1))
    for ps in (0, 8, 24, 2048, -16):
        assert "power of two" in _err(plan(ps=ps))
    assert "overlap" in _err(plan(row=7)) and "2^31" in _err(plan(w=1 << 28, row=1 << 28)) and "null" in _err(plan(new=None))

    def pages(**k):
        d = dict(k=p, v=p, k_page=2048, k_head=1024, k_slot=64, v_page=2048, v_head=1024, v_slot=64, n_pages=4, page_size=16,
                 kv_heads=2, head_dim=64)
        return N.Pages(**{**d, **k})

    write = lambda pg, dt=N.BF16, k=p, row=128, n=3: lib.fcenc_page_write(dt, C.byref(pg), k, p, row, 64, row, 64, p, n, None)
    assert "dtype" in _err(write(pages(), dt=2)) and "power of two" in _err(write(pages(page_size=17)))
    assert "16 bytes" in _err(write(pages(), row=100)) and "aligned" in _err(write(pages(), k=p + 2))
    assert "head" in _err(write(pages(head_dim=63))) and "no pages" in _err(write(pages(n_pages=0)))
    assert "null" in _err(write(pages(), k=None)) and "null pages" in _err(lib.fcenc_page_write(1, None, p, p, 1, 1, 1, 1, p, 1, None))
    assert write(pages(), n=0) == 0

    def rows(**k):
        d = dict(q=p, block_table=p, kv_lens=p, cu_rows=p, q_row=256, q_head=64, table_row=4, batch=2, rows=3, heads=4,
                 table_width=4, window=0, sinks=0, causal=1, max_rows=0, scale=0.1)
        return N.PageRows(**{**d, **k})

    def attn(pg, rw, dt=N.BF16, ws=None, nb=0, out=p):
        return lib.fcenc_page_attention(dt, C.byref(pg), C.byref(rw), out, ws, nb, None)

    assert "dtype" in _err(attn(pages(), rows(), dt=5)) and "heads over" in _err(attn(pages(), rows(heads=5)))
    for dim in (0, 12, 136):
        assert "head dim" in _err(attn(pages(head_dim=dim), rows()))
    assert "table" in _err(attn(pages(), rows(table_row=3))) and "negative" in _err(attn(pages(), rows(window=-1)))
    assert "negative" in _err(attn(pages(), rows(sinks=-1))) and "negative" in _err(attn(pages(), rows(max_rows=-1)))
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert "scale" in _err(attn(pages(), rows(scale=scale)))
    assert "16 bytes" in _err(attn(pages(k_head=1001), rows())) and "slots" in _err(attn(pages(k_slot=56), rows()))
    assert "slot strides" in _err(attn(pages(v_slot=-64), rows())) and "page strides" in _err(attn(pages(k_page=1 << 32), rows()))
    assert "page strides" in _err(attn(pages(v_page=-1024), rows())) and "2 GiB" in _err(attn(pages(k_slot=1 << 23, page_size=256), rows()))
    assert "null" in _err(attn(pages(), rows(q=None))) and "aligned" in _err(attn(pages(k=p + 8), rows()))
    big = rows(batch=1, rows=1, table_width=4096, table_row=4096)
    need = lib.fcenc_page_attention_workspace_bytes(N.BF16, C.byref(pages()), C.byref(big))
    assert need > 0 and "workspace" in _err(attn(pages(), big, ws=p, nb=need - 1))
    assert attn(pages(), rows(rows=0)) == 0

    sample = lambda dt=N.F32, x=p, stride=8, r=2, v=8, u=p, tok=p: lib.fcenc_sample_tokens(dt, x, stride, r, v, u, None, None, None, None, tok, None)
    assert "dtype" in _err(sample(dt=9)) and "vocabulary" in _err(sample(v=0)) and "vocabulary" in _err(sample(v=(1 << 18) + 1))
    assert "overlap" in _err(sample(stride=7)) and "null" in _err(sample(u=None)) and "aligned" in _err(sample(x=p + 2))
    assert sample(r=0) == 0


def test_operators_refuse_cpu_operands():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.kv_page_plan_(i32(2), i32(2), None, i32(2, 4), i32(9), i32(1), 16, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.kv_page_write_(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.kv_page_attention(torch.zeros(1, 2, 64), torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64), i32(1, 4), i32(1), i32(2), 0.1)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2))


@pytest.mark.parametrize("bad", [dict(page_size=48), dict(page_size=8), dict(head_dim=132), dict(head_dim=20), dict(layers=0),
                                 dict(dtype=torch.float16)])
def test_cache_refuses_sizes_it_has_no_kernels_for(bad):
    with pytest.raises(ValueError):
        KVPages(**{**dict(layers=1, pages=4, kv_heads=2, head_dim=64, batch=2, max_tokens=100, device="cpu"), **bad})


def test_cache_needs_an_open_step():
    c = KVPages(layers=1, pages=4, kv_heads=2, head_dim=64, batch=2, max_tokens=100, page_size=32, device="cpu")
    assert tuple(c.block_table.shape) == (2, 4) and int(c.free_count) == 4
    with pytest.raises(RuntimeError, match="plan"):
        c.write(0, torch.zeros(1, 2, 64), torch.zeros(1, 2, 64))


def test_shape_functions():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dt=torch.int32: torch.empty(s, dtype=dt, device="cuda")
        slots, cu, granted = ops.kv_page_plan_(e(3), e(3), None, e(3, 4), e(9), e(1), 16, 7)
        assert slots.shape == (7,) and slots.dtype == torch.int64 and cu.shape == (4,) and granted.dtype == torch.bool
        kp = e(9, 2, 16, 64, dt=torch.bfloat16)
        out = ops.kv_page_attention(e(7, 4, 64, dt=torch.bfloat16), kp, kp, e(3, 4), e(3), cu, 0.1)
        assert out.shape == (7, 4, 64) and out.dtype == torch.bfloat16
        assert ops.kv_page_write_(e(7, 2, 64, dt=torch.bfloat16), e(7, 2, 64, dt=torch.bfloat16), kp, kp, slots) is None
        tok = ops.sample_tokens(e(5, 100, dt=torch.float32), e(5, dt=torch.float32))
        assert tok.shape == (5,) and tok.dtype == torch.int32


def test_tracers_and_modes_see_the_operators():
    """Eager calls on plain tensors do not go through the dispatcher; calls that something traces or intercepts do."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    logits, u = torch.zeros(2, 8), torch.zeros(2)
    named = lambda gm: any("sample_tokens" in str(n.target) for n in gm.graph.nodes)
    assert named(make_fx(lambda x, y: ops.sample_tokens(x, u=y), tracing_mode="fake")(logits, u))

    seen = []

    class See(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return torch.zeros(2, dtype=torch.int32) if "sample_tokens" in str(func) else func(*args, **(kwargs or {}))

    with See():
        ops.sample_tokens(logits, u)
    assert any("sample_tokens" in s for s in seen)

    with FakeTensorMode() as mode:
        fake = torch.empty((2, 8)), torch.empty(2)
    assert ops.sample_tokens(*fake).shape == (2,)             # outside of the mode that made them

    graphs = []
    compiled = torch.compile(lambda x, y: ops.sample_tokens(x, y) + 1, fullgraph=True,
                             backend=lambda gm, _: graphs.append(gm) or gm.forward)
    with pytest.raises(RuntimeError, match="GPU"):            # traced whole, then refused where it runs: on the CPU
        compiled(logits, u)
    assert named(graphs[0])


def _stand_in(name, mutates=()):
    """An operator registered as the serving ones are, with a kernel that runs on the CPU and leaves nothing for a tracer to see."""
    def put(to, x):
        C.memmove(to.data_ptr(), (x.numpy(force=True) * 2).ctypes.data, 4 * x.numel())

    if mutates:
        def fn(x: torch.Tensor, y: torch.Tensor) -> None:
            ops._no_grad(x, y)
            put(y, x)
    else:
        def fn(x: torch.Tensor) -> torch.Tensor:
            ops._no_grad(x)
            y = x.new_empty(x.shape)
            put(y, x)
            return y
    fn.__name__ = name
    return ops._serving_op(mutates)(fn)


def test_a_torchscript_trace_records_the_operators():
    twice, twice_ = _stand_in("traced_twice"), _stand_in("traced_twice_", ("y",))
    x = torch.arange(4.0)

    def both(x):
        y = torch.zeros_like(x)
        twice_(x, y)
        return twice(x), y

    traced = torch.jit.trace(both, (x,), check_trace=False)
    for got in traced(x + 1):
        assert torch.equal(got, 2 * (x + 1))


def test_function_modes_and_profilers_see_the_operators():
    from torch.overrides import TorchFunctionMode
    twice, x, seen = _stand_in("seen_twice"), torch.arange(4.0), []

    class See(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with See():
        assert torch.equal(twice(x), 2 * x)
    assert any("seen_twice" in s for s in seen)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        twice(x)
    assert any("seen_twice" in e.key for e in prof.key_averages())


def test_derivatives_are_refused_not_dropped():
    """Forward mode, and the transforms, whose tensors the kernels never meet as tensors that require a gradient."""
    from torch.autograd import forward_ad
    x, y = torch.arange(4.0), torch.zeros(4)
    twice, twice_ = _stand_in("derived_twice"), _stand_in("derived_twice_", ("y",))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(4))
        for call in (lambda: twice(dual), lambda: twice.op(dual), lambda: twice_(dual, y), lambda: twice_(x, forward_ad.make_dual(y, x))):
            with pytest.raises(RuntimeError, match="derivative"):
                call()
        assert torch.equal(twice(x), 2 * x)                   # an operand without a tangent
    for call in (twice, twice.op):
        with pytest.raises(RuntimeError, match="derivative"):
            torch.func.jvp(call, (x,), (torch.ones(4),))
        with pytest.raises(RuntimeError, match="backward"):
            torch.func.grad(lambda x: call(x).sum())(x)
        with pytest.raises(RuntimeError, match="backward"):
            call(x.clone().requires_grad_())
        with torch.no_grad():
            assert torch.equal(call(x.clone().requires_grad_()), 2 * x)
        assert torch.equal(torch.func.vmap(call)(torch.stack([x, x + 1])), 2 * torch.stack([x, x + 1]))
        with torch.inference_mode():
            assert torch.equal(call(x + 1), 2 * (x + 1))
    # a transform over other operands
    assert torch.equal(torch.func.grad(lambda a: (a * twice(x)).sum())(x), 2 * x)


def test_integers_past_32_bits_are_refused():
    """They cross the C ABI as `int`: a window of 2^32 + 64 must not become one of 64."""
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    attn = lambda **k: ops.kv_page_attention(torch.zeros(1, 2, 64), torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64), i32(1, 4), i32(1), i32(2), 0.1, **k)
    for big in (2 ** 31, 2 ** 32, 2 ** 32 + 64, -2 ** 32 + 5):
        for name in ("window", "sinks", "max_rows"):
            with pytest.raises(ValueError, match="32 bits"):
                attn(**{name: big})
        with pytest.raises(ValueError, match="32 bits"):
            ops.kv_page_plan_(i32(2), i32(2), None, i32(2, 4), i32(9), i32(1), big + 16, 2)
        with pytest.raises(ValueError, match="32 bits"):
            ops.kv_page_plan_(i32(2), i32(2), None, i32(2, 4), i32(9), i32(1), 16, big + 2)
    with pytest.raises(RuntimeError, match="GPU"):            # the largest that fit
        attn(window=2 ** 31 - 1, sinks=2 ** 31 - 1, max_rows=2 ** 31 - 1)


@pytest.mark.parametrize("batch,rows,max_rows", [(1024, 16, 12), (4096, 40, 40), (100000, 64, 50), (40, 40, 0), (40, 400, 30), (1, 4000, 0), (2000, 4000, 100)])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (8, 8), (64, 1)])
def test_attention_workspace_follows_the_rows_of_the_step(batch, rows, max_rows, heads, kv_heads):
    """However long the table is: at most 256 pieces of the key axis of each (row, head), and no more than make 2560 workgroups of the
    rows' tiles; twice, as short requests and chunks may both be cut."""
    pages = N.Pages(4096, 4096, 64 * 128 * kv_heads, 64 * 128, 128, 64 * 128 * kv_heads, 64 * 128, 128, 1 << 20, 64, kv_heads, 128)
    r = N.PageRows(4096, 4096, 4096, 4096, heads * 128, 128, 2048, batch, rows, heads, 2048, 0, 0, 1, max_rows, 0.1)
    group = heads // kv_heads
    some = min(batch, rows)                              # one tile per request with rows at the least that can be supposed
    pieces = [min(256, max(1, 2560 // (n * kv_heads))) for n in (some, -(-rows * min(group, 128) // 128))]
    pair = 128 * 4 + 8
    need = N.lib().fcenc_page_attention_workspace_bytes(N.BF16, C.byref(pages), C.byref(r))
    assert need <= rows * heads * sum(pieces) * pair + 64


@pytest.mark.parametrize("rows", [0, 4, 6])
def test_cache_refuses_other_rows_than_the_step_has(rows):
    """With fewer, the rows of the last request would be taken for its last ones."""
    from conformer_amd.paging import Step
    c = KVPages(layers=1, pages=4, kv_heads=2, head_dim=64, batch=2, max_tokens=100, page_size=32, device="cpu")
    c.step = Step(torch.arange(5), torch.tensor([0, 2, 5], dtype=torch.int32), torch.tensor([True, True]))
    with pytest.raises(ValueError, match="rows"):
        c.attend(0, torch.zeros(rows, 4, 64))
