"""Calls of the paged cache beside one another: plans of one kernel instance with different shared memory, captured steps
that reuse their buffers, other streams, and what a bad value or a failed call leaves behind."""
import numpy as np
import pytest

import backburner_b200 as pa
from backburner_b200 import api
from test_cache_gpu import Seqs, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant,first,second", [(pa.F16, (8, 1), (8, 64)), (pa.Q8_0, (8, 1), (2, 1)), (pa.Q4_0, (8, 3), (2, 70))])
def test_plans_of_one_kernel_keep_their_shared_memory(ctx, quant, first, second):
    """two live plans of one split-K instance, the larger one made first: neither takes the other's launch away"""
    made = []
    ctx.set_kernel(1)
    for nkv, tok in (first, second):
        sq = Seqs(nkv + tok, [200, 77], 128, nkv, quant)
        made.append((sq, tok, pa.CachePlan(ctx, sq.cache, 2, tok, 1, sq.max_pages)))
    ctx.set_kernel(0)
    for i in (0, 1, 0, 1):
        sq, tok, plan = made[i]
        Qs = sq.q(tok, 1)
        out = plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
        ctx.status()
        _check(sq, Qs, out, tok, 1)
    for _, _, plan in made:
        plan.close()


@pytest.mark.parametrize("kernel,tok", [(1, 1), (1, 7), (2, 7), (2, 60), (3, 60)])
@pytest.mark.parametrize("captured", [False, True])
def test_steps_that_reuse_their_buffers(ctx, kernel, tok, captured):
    """append, then attention on the queries it has just written, over a table written just before: one set of buffers for
    every step, the steps back to back, each as if it were alone"""
    import torch
    S, hd, nkv, gqa, steps = 3, 128, 8, 5, 6
    g = torch.Generator(device="cuda")
    g.manual_seed(kernel + tok)
    c = pa.Cache(hd, nkv, pa.Q8_0, 1, 64, 64)
    tables = [torch.randperm(64, generator=g, device="cuda")[:S * 8].view(S, 8).int() for _ in range(steps)]
    xs = [[torch.randn(S, tok, n, hd, generator=g, device="cuda") for n in (nkv * gqa, nkv, nkv)] for _ in range(steps)]
    for p in (c.K, c.V):   # every row of the pool is finite
        p.copy_(pa.quantize_q8_0(torch.randn(64 * 64, nkv, hd, generator=g, device="cuda")).reshape(p.shape))
    pool = [p.clone() for p in (c.K, c.V)]
    start = torch.tensor([300, 0, 129], dtype=torch.int32, device="cuda")
    n = start + tok
    ctx.set_kernel(kernel)
    plan = pa.CachePlan(ctx, c, S, tok, gqa, 8)
    ctx.set_kernel(0)
    x, table = [t.clone() for t in xs[0]], tables[0].clone()
    Qs = torch.empty(S, nkv, gqa * tok, hd, dtype=torch.float16, device="cuda")
    out = torch.empty_like(Qs), torch.empty(S, nkv, gqa * tok, device="cuda")
    want = []
    for i in range(steps):   # each step alone
        for p, was in zip((c.K, c.V), pool):
            p.copy_(was)
        q = pa.cache_append(ctx, c, 0, *xs[i], tables[i], start, scale=hd ** -0.5)
        torch.cuda.synchronize()
        o = plan.reply(0, q, tables[i], n)
        torch.cuda.synchronize()
        want.append([t.clone() for t in (q, *o)])

    def step():
        pa.cache_append(ctx, c, 0, *x, table, start, scale=hd ** -0.5, out=Qs)
        plan.reply(0, Qs, table, n, out=out)

    run = step
    if captured:
        graph = torch.cuda.CUDAGraph()
        step()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            step()
        run = graph.replay
    got = []
    for i in range(steps):
        for p, was in zip((c.K, c.V), pool):
            p.copy_(was)
        for a, b in zip(x, xs[i]):
            a.copy_(b)
        table.copy_(tables[i])
        run()
        got.append([t.clone() for t in (Qs, *out)])
    torch.cuda.synchronize()
    ctx.status()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    plan.close()


@pytest.mark.parametrize("quant", [pa.F16, pa.Q8_0, pa.Q4_0])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_append_keeps_what_is_not_a_number(ctx, quant, dtype):
    """a NaN, an infinity of either sign and (fp32) a value whose block's d passes f16's range: the block reads as NaN, every
    other block as if it were not there; f16 rows keep each element. With a norm a NaN takes its head with it."""
    import torch
    nkv, hd, tok = 8, 128, 6
    bad = [float("nan"), float("inf"), -float("inf")] + ([1e7, -1e30] if dtype == "float32" else [])
    sq = Seqs(1, [0], hd, nkv, quant, 64, extra=tok)
    x = [torch.randn(1, tok, n, hd, generator=sq.g, device="cuda").to(getattr(torch, dtype)) for n in (nkv, nkv, nkv)]
    st = torch.tensor([0], dtype=torch.int32, device="cuda")
    pa.cache_append(ctx, sq.cache, 0, *x, sq.table, st)
    clean = [t.clone() for t in pa.cache_rows(ctx, sq.cache, 0, sq.table, st, tok)]
    y = [t.clone() for t in x]
    want = [t.clone() for t in clean]
    for i, b in enumerate(bad):
        for kv in range(2):
            h, d = (3 * i + kv) % nkv, (37 * i + 5 * kv) % hd   # (lanes, halves of a nibble pair and blocks of every kind)
            y[1 + kv][0, i, h, d] = b
            if quant == pa.F16:
                want[kv][0, i, h, d] = b   # 1e7 and -1e30 are infinities in f16
            else:
                want[kv][0, i, h, d // 32 * 32:d // 32 * 32 + 32] = float("nan")
    pa.cache_append(ctx, sq.cache, 0, *y, sq.table, st)
    got = pa.cache_rows(ctx, sq.cache, 0, sq.table, st, tok)
    ctx.status()
    for g, w in zip(got, want):
        assert torch.equal(torch.isnan(g), torch.isnan(w)) and torch.equal(torch.nan_to_num(g), torch.nan_to_num(w))
    w = torch.ones(hd, device="cuda")
    Qs = pa.cache_append(ctx, sq.cache, 0, *y, sq.table, st, wq=w, wk=w)
    K, _ = pa.cache_rows(ctx, sq.cache, 0, sq.table, st, tok)
    ctx.status()
    assert bool(torch.isnan(K[0, 0, 0]).all()) and not torch.isnan(K[0, 0, 1:]).any() and not torch.isnan(Qs).any()


@pytest.mark.parametrize("start,bad", [(-1, True), (-2 ** 31, True), (0, False), (64 * 5 - 3, False), (64 * 5 - 2, True), (2 ** 31 - 1, True)])
def test_append_without_positions_reports_keys_out_of_reach(ctx, start, bad):
    """a start before key 0, or one whose tokens pass the table, is reported whether the call gives positions or not"""
    import torch
    sq = Seqs(3, [0, 0], 128, 8, pa.Q8_0, 64, extra=64 * 4)   # (the table has an entry more, outside the pool)
    table = torch.arange(10, dtype=torch.int32, device="cuda").view(2, 5)
    x = [torch.randn(2, 3, n, 128, generator=sq.g, device="cuda") for n in (40, 8, 8)]
    st = torch.tensor([5, start], dtype=torch.int32, device="cuda")
    pos = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for kw in ({}, dict(pos=pos)):
        pa.cache_append(ctx, sq.cache, 0, *x, table, st, **kw)
        if bad:
            with pytest.raises(pa.PaCudaError) as e:
                ctx.status()
            assert e.value.code == api.EINVAL
        ctx.status()
    # padding is none of this, wherever its sequence starts
    pa.cache_append(ctx, sq.cache, 0, *x, table, st, pos=torch.tensor([[0, 0, 0], [-1, -1, -1]], dtype=torch.int32, device="cuda"))
    ctx.status()


def _inputs(sq, x, Qs):
    """inputs of every call on a cache that nothing else holds, in the order of _all_calls"""
    import torch
    table, n = sq.table, sq.n_keys
    i32 = dict(dtype=torch.int32, device="cuda")
    S = len(sq.lens)
    return [[Qs.clone(), table.clone(), n + 0], [Qs.clone(), table.clone(), n + 0], [*(t.clone() for t in x), table.clone(), n - 3],
            [table.clone(), n - 9], [table[0, :1].clone(), table[1, :1].clone()], [table.clone(), n - n],
            [table.clone(), n - 3, torch.tensor([[0, 2, 0]] * S, **i32), torch.tensor([2] * S, **i32)]]


def _all_calls(ctx, sq, plan, inputs, stream):
    """every call on a cache, on `stream`; a call's inputs are dropped when it returns, unless the caller holds them"""
    out = [*plan.reply(sq.layer, *inputs.pop(0), stream=stream)]
    out += plan.run(sq.layer, *inputs.pop(0), stream=stream)
    out += [pa.cache_append(ctx, sq.cache, 0, *inputs.pop(0), scale=0.5, stream=stream)]
    out += pa.cache_rows(ctx, sq.cache, sq.layer, *inputs.pop(0), 9, stream=stream)
    pa.cache_copy_pages(ctx, sq.cache, *inputs.pop(0), stream=stream)
    out += pa.cache_rows(ctx, sq.cache, sq.layer, *inputs.pop(0), 5, stream=stream)
    out += [pa.cache_compact(ctx, sq.cache, *inputs.pop(0), stream=stream)]
    return out


@pytest.mark.parametrize("as_handle", [False, True])
def test_calls_on_another_stream_own_what_they_use(ctx, as_handle):
    """`stream=` while the current stream is still reading memory that was given back, and (torch's streams) inputs dropped as
    soon as a call returns: outputs come from elsewhere, and the inputs' memory is not given out before the calls have run"""
    import torch
    S, tok, gqa = 2, 4, 5
    sq = Seqs(51, [300, 130], extra=8)
    plan = pa.CachePlan(ctx, sq.cache, S, tok, gqa, sq.max_pages)
    Qs = sq.q(tok, gqa)
    x = [torch.randn(S, 2, n, 128, generator=sq.g, device="cuda") for n in (40, 8, 8)]
    pool = [p.clone() for p in (sq.cache.K, sq.cache.V)]
    want = [t.clone() for t in _all_calls(ctx, sq, plan, _inputs(sq, x, Qs), None)]
    for p, was in zip((sq.cache.K, sq.cache.V), pool):
        p.copy_(was)
    side = torch.cuda.Stream()
    inputs = _inputs(sq, x, Qs)
    sizes = [t.numel() for i in inputs for t in i if t.dtype == torch.int32]
    seven = [torch.full_like(t, 7) for t in want]   # a block of every output's size
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)                  # (about 0.1 s)
    late = [t.clone() for t in seven]               # read late by the current stream, and given back at once
    del seven
    with torch.cuda.stream(side):
        torch.cuda._sleep(600_000_000)              # the calls run after everything below is queued
    held = [list(i) for i in inputs] if as_handle else None   # (of another's stream the caller keeps them)
    got = _all_calls(ctx, sq, plan, inputs, side.cuda_stream if as_handle else side)
    junk = [torch.full((n,), 2 ** 30, dtype=torch.int32, device="cuda") for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    ctx.status()
    assert all(bool((t == 7).all()) for t in late)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del junk, held
    plan.close()


@pytest.mark.parametrize("external", [False, True])
def test_a_stream_that_torch_does_not_own_may_end_before_the_tensors(ctx, external):
    """calls on a stream of the caller's, which is destroyed while the cache, the inputs and the outputs live on: freeing them
    later does not touch it"""
    import ctypes
    import torch
    with open("/proc/self/maps") as f:
        rt = ctypes.CDLL(next(line.split()[-1] for line in f if "libcudart" in line))
    sq = Seqs(53, [300, 130], extra=8)
    plan = pa.CachePlan(ctx, sq.cache, 2, 4, 5, sq.max_pages)
    Qs = sq.q(4, 5)
    x = [torch.randn(2, 2, n, 128, generator=sq.g, device="cuda") for n in (40, 8, 8)]
    inputs = _inputs(sq, x, Qs)
    held = [list(i) for i in inputs]
    # (no tensor has the stream on record, so that no free can meet it: looked at before the stream is destroyed)
    kept = []
    record, torch.Tensor.record_stream = torch.Tensor.record_stream, lambda t, s: kept.append(s)
    torch.cuda.synchronize()
    own = ctypes.c_void_p()
    assert rt.cudaStreamCreate(ctypes.byref(own)) == 0
    try:
        out = _all_calls(ctx, sq, plan, inputs, torch.cuda.ExternalStream(own.value) if external else own.value)
    finally:
        torch.Tensor.record_stream = record
        torch.cuda.synchronize()
        assert rt.cudaStreamDestroy(own) == 0
    ctx.status()
    assert own.value not in [s.cuda_stream for s in kept]
    want = plan.reply(sq.layer, held[0][0], sq.table, sq.n_keys)
    assert out[0].shape == want[0].shape
    del out, held, sq
    plan.close()


def test_a_stream_of_another_device_is_refused(ctx):
    import torch

    class Other(torch.cuda.Stream):   # (one GPU is enough to ask for it)
        device_index = 1

    sq = Seqs(52, [30, 10])
    plan = pa.CachePlan(ctx, sq.cache, 2, 1, 5, sq.max_pages)
    with pytest.raises(pa.PaCudaError) as e:
        plan.reply(0, sq.q(1, 5), sq.table, sq.n_keys, stream=Other())
    assert e.value.code == api.EINVAL
    plan.close()


def test_status_reports_a_wait_and_a_bad_argument(ctx):
    """a wait that ran out and an argument out of range, both since the last look: one after the other, then neither"""
    import torch
    sq = Seqs(61, [300, 80])
    x = [torch.randn(2, 1, n, 128, generator=sq.g, device="cuda") for n in (40, 8, 8)]
    ctx.set_kernel(1)
    plan = pa.CachePlan(ctx, sq.cache, 2, 1, 5, sq.max_pages)
    ctx.set_kernel(0)
    Qs = sq.q(1, 5)
    ctx.set_timeout_ns(20_000_000)
    ctx.set_stall_test(True)
    try:
        plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
        torch.cuda.synchronize()
    finally:
        ctx.set_stall_test(False)
        ctx.set_timeout_ns(2_000_000_000)
    pa.cache_append(ctx, sq.cache, 0, *x, sq.table, torch.tensor([-1, 0], dtype=torch.int32, device="cuda"))
    for code in (api.ETIMEOUT, api.EINVAL):
        with pytest.raises(pa.PaCudaError) as e:
            ctx.status()
        assert e.value.code == code
    ctx.status()
    out = plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
    ctx.status()
    _check(sq, Qs, out, 1, 5)
    plan.close()


def test_a_failed_launch_leaves_no_error_behind(ctx):
    """a launch that CUDA refuses (the legacy stream while a blocking stream captures) is the call's error and nobody else's"""
    import ctypes
    import torch
    sq = Seqs(71, [300, 80])
    plan = pa.CachePlan(ctx, sq.cache, 2, 1, 5, sq.max_pages)
    Qs = sq.q(1, 5)
    out = plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
    torch.cuda.synchronize()
    with open("/proc/self/maps") as f:
        rt = ctypes.CDLL(next(line.split()[-1] for line in f if "libcudart" in line))
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.cudaStreamCreate(ctypes.byref(stream)) == 0
    assert rt.cudaStreamBeginCapture(stream, 0) == 0
    try:
        with pytest.raises(pa.PaCudaError) as e:
            plan.reply(sq.layer, Qs, sq.table, sq.n_keys, out=out, stream=1)
        left = rt.cudaPeekAtLastError()
    finally:
        rt.cudaStreamEndCapture(stream, ctypes.byref(graph))   # (invalidated by the refused launch)
        rt.cudaGetLastError()
        rt.cudaStreamDestroy(stream)
    assert e.value.code == api.ECUDA and left == 0
    again = plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
    ctx.status()
    assert all(torch.equal(a, b) for a, b in zip(again, out))
    plan.close()


@pytest.mark.parametrize("kernel,quant,hd,nkv", [(1, pa.Q8_0, 128, 8), (1, pa.F16, 256, 4), (2, pa.Q8_0, 128, 8), (2, pa.Q4_0, 256, 4),
                                                 (3, pa.Q8_0, 128, 8)])
def test_scores_that_are_not_numbers_give_nan(ctx, kernel, quant, hd, nkv):
    """a query row with a NaN or an infinity, and a key with NaN that every token sees: NaN, not an empty row's zeros; the
    other rows and heads as they are, and a key outside the window changes nothing"""
    import torch
    tok, gqa, W = 5, 5, 700
    sq = Seqs(81, [2000, 900], hd, nkv, quant, 64)
    ctx.set_kernel(kernel)
    plan = pa.CachePlan(ctx, sq.cache, 2, tok, gqa, sq.max_pages, W, 3)
    ctx.set_kernel(0)
    Qs = sq.q(tok, gqa)
    clean = plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
    _check(sq, Qs, clean, tok, gqa, W, 3)
    bad = torch.zeros(2, nkv, gqa * tok, dtype=torch.bool, device="cuda")
    Qb = Qs.clone()
    for s, h, r, d, x in ((0, 0, 0, 0, float("nan")), (0, 1, 24, hd - 1, float("nan")), (1, nkv - 1, 7, 5, float("inf"))):
        Qb[s, h, r, d] = x
        bad[s, h, r] = True
    K = sq.cache.K[sq.layer].view(-1, sq.cache.rs)
    at = sq.rows(0, [1999 - 400])[0]
    K[at, 2 * sq.hb:2 * sq.hb + 2] = 0x7E   # f16 0x7e7e is NaN: d of head 2's first block, or its first value
    bad[0, 2] = True
    K[sq.rows(0, [1000])[0], :2] = 0x7E     # no token's
    Oh, lse = plan.reply(sq.layer, Qb, sq.table, sq.n_keys)
    O, m, l = plan.run(sq.layer, Qb, sq.table, sq.n_keys)
    ctx.status()
    for t in (lse, l, m):
        assert torch.equal(torch.isnan(t), bad)
    for t in (Oh, O):
        assert torch.equal(torch.isnan(t), bad[..., None].expand_as(t))
    assert bool(((Oh - clean[0]).abs()[~bad] <= 2.0 ** -10 * clean[0].abs().amax()).all())
    assert bool(((lse - clean[1]).abs()[~bad] <= 2.0 ** -18 * clean[1].abs().amax()).all())
    plan.close()
