"""The paged-cache operators on the GPU against plain implementations in 64 bits: windowed and tree attention, the append
(head norm, rotation, quantised rows), reading rows back, page copies, compaction, and a run of them together.

Tolerances of the attention: the kernels round P to f16 (half a step, 2^-11 of it; below 2^-14 half of f16's smallest step,
2^-25 against a reference maximum no larger than the row's) and sum in fp32, so with A = sum p|v| / l an output is off by at
most A * (2^-11 + 2 ds) + 2^-25 sum|v| / l, plus its own rounding to f16; ds = hd * 2^-23 * max_j sum_d |q_d k_jd| bounds a
score's error, and lse is off by ds, the exponentials' 2^-20 and the sum's n * 2^-24."""
import math

import numpy as np
import pytest

import backburner_b200 as pa
from backburner_b200 import api

pytestmark = pytest.mark.gpu

QUANTS = [pa.F16, pa.Q8_0, pa.Q4_0]


def _quantise(torch, x, quant):
    if quant == pa.F16:
        return x.to(torch.float16).view(torch.uint8)
    return (pa.quantize_q8_0 if quant == pa.Q8_0 else pa.quantize_q4_0)(x)


def _stored(torch, x, quant):
    """The bytes of float32 x [..., hd] on the CPU by the format's formula, each quotient rounded once (the package's quantisers
    multiply by the rounded 1 / d, which turns some ties the other way)."""
    if quant == pa.F16:
        return _quantise(torch, x, quant)
    top = 127 if quant == pa.Q8_0 else 7
    b = x.unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1, keepdim=True) / top).to(torch.float16)
    q = torch.where(d == 0, 0.0, torch.round(b / d.float())).clamp(-top, top)
    data = q.to(torch.int8).view(torch.uint8)
    if quant == pa.Q4_0:
        n = (q + 8).to(torch.uint8)
        data = n[..., :16] | n[..., 16:] << 4
    return torch.cat([d.view(torch.uint8), data], -1).flatten(-2)


def _value(torch, rows, quant, hd):
    """uint8 [..., head bytes] -> the f16 values as float64"""
    if quant == pa.F16:
        return rows.contiguous().view(torch.float16).double()
    return pa.dequantize(rows, quant, hd).to(torch.float16).double()   # f16 d times a small integer: exact in fp32


class Seqs:
    """A cache with sequences of the given lengths in shuffled pages; everything else in it is NaN patterns, and table
    entries no key needs are out of range."""

    def __init__(self, seed, lens, hd=128, nkv=8, quant=pa.Q8_0, page=64, layers=2, extra=0, pad_row=0):
        import torch
        self.torch, self.hd, self.nkv, self.quant, self.page, self.lens = torch, hd, nkv, quant, page, lens
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.g = g
        need = [-(-(n + extra) // page) for n in lens]
        total = sum(need) + 2
        hb = pa.head_bytes(quant, hd)
        self.hb = hb
        rs = (nkv * hb + 15) // 16 * 16 + pad_row
        K = torch.full((layers, total, page, rs), 0xFF, dtype=torch.uint8, device="cuda")
        self.cache = pa.Cache.of(K, K.clone(), hd=hd, nkv=nkv, quant=quant)
        order = torch.randperm(total, generator=g, device="cuda").tolist()
        self.max_pages = max(1, max(need)) + 1
        tab, at = np.full((len(lens), self.max_pages), -7, np.int32), 0
        for s, n in enumerate(need):
            tab[s, :n] = order[at:at + n]
            at += n
        self.tab = tab
        self.table = torch.from_numpy(tab).cuda()
        self.n_keys = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.layer = layers - 1
        self.kv = []
        for s, n in enumerate(lens):
            k = torch.randn(n, nkv, hd, generator=g, device="cuda")
            k[:, :, :3] *= 8
            v = torch.randn(n, nkv, hd, generator=g, device="cuda")
            self.put(s, 0, k, v)

    def rows(self, s, j):
        j = np.asarray(j)
        return self.torch.from_numpy(self.tab[s][j // self.page].astype(np.int64) * self.page + j % self.page).cuda()

    def put(self, s, j0, k, v):
        at = self.rows(s, np.arange(j0, j0 + len(k)))
        for pool, x in ((self.cache.K, k), (self.cache.V, v)):
            pool[self.layer].view(-1, self.cache.rs)[at, :self.nkv * self.hb] = _quantise(self.torch, x, self.quant).reshape(len(k), self.nkv * self.hb)

    def get(self, s, n):
        """K, V of keys 0 .. n-1 in float64 [n][nkv][hd]"""
        at = self.rows(s, np.arange(n))
        return [_value(self.torch, p[self.layer].view(-1, self.cache.rs)[at, :self.nkv * self.hb].reshape(n, self.nkv, self.hb),
                       self.quant, self.hd) for p in (self.cache.K, self.cache.V)]

    def q(self, tok, gqa):
        q = self.torch.randn(len(self.lens), self.nkv, gqa * tok, self.hd, generator=self.g, device="cuda")
        return (q * self.hd ** -0.5).to(self.torch.float16)


def _sees(torch, n, q0, tok, window, sinks, bits):
    """[tok][n] on the host, from the definition"""
    m = np.zeros((tok, n), bool)
    for t in range(tok):
        if bits is None:
            at, end, named = q0 + t, q0 + t + 1, []
        else:
            b = int(bits[t]) & (2 ** 64 - 1)
            if not b:
                continue
            at, end, named = q0 + bin(b).count("1") - 1, q0, [q0 + u for u in range(tok) if b >> u & 1]
        for j in range(max(0, min(end, n))):
            m[t, j] = not window or j > at - window or j < sinks
        for j in named:
            if 0 <= j < n:
                m[t, j] = True
    return m


def _check(sq, Qs, out, tok, gqa, window=0, sinks=0, q_pos=None, bits=None, lens=None, partial=None):
    """out = (Oh, lse) [and partial = (O, m, l)] against 64 bits"""
    torch = sq.torch
    Oh, lse = out
    for s, n in enumerate(lens if lens is not None else sq.lens):
        q0 = int(q_pos[s]) if q_pos is not None else n - tok
        see = torch.from_numpy(_sees(torch, n, q0, tok, window, sinks, None if bits is None else bits[s].tolist())).cuda()
        see = see.repeat(gqa, 1)
        K, V = sq.get(s, n)
        live = see.any(0)[:, None, None]
        K, V = torch.where(live, K, 0.0), torch.where(live, V, 0.0)
        for h in range(sq.nkv):
            q = Qs[s, h].double()
            x = torch.where(see, q @ K[:, h].T, -math.inf)
            z = torch.logsumexp(x, 1) if n else torch.full((len(q),), -math.inf, dtype=torch.float64, device="cuda")
            some = z > -math.inf
            assert torch.equal(lse[s, h] > -math.inf, some)
            assert not Oh[s, h][~some].any()
            if not some.any():
                continue
            p = torch.where(some[:, None], torch.exp(x - z.clamp(min=-1e300)[:, None]), 0.0)
            O = p @ V[:, h]
            ds = sq.hd * 2.0 ** -23 * float(torch.where(see, q.abs() @ K[:, h].abs().T, 0.0).max())
            pmax = p.max(1).values[:, None]
            tol = ((p @ V[:, h].abs()) * (2.0 ** -11 + 2 * ds + 2.0 ** -20) + 2.0 ** -25 * pmax * V[:, h].abs().sum(0) +
                   2.0 ** -11 * O.abs() + 2.0 ** -25)
            err = (Oh[s, h].double() - O).abs()
            assert bool((err <= tol)[some].all()), (s, h, float((err / tol)[some].max()))
            tl = ds + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -22 * z.abs()
            el = (lse[s, h].double() - z).abs()
            assert bool((el <= tl)[some].all()), (s, h, float((el / tl)[some].max()))
            if partial is not None:
                Of, m, l = (t[s, h].double() for t in partial)
                assert bool((m[~some] == -math.inf).all()) and not l[~some].any()
                top = x.max(1).values
                assert bool(((m - top).abs() <= ds)[some].all())
                assert bool(((Of / l.clamp(min=1e-30)[:, None] - O).abs() <= tol)[some].all())


def _tree(rng, sets, tok, pad=0.0):
    out = np.zeros((sets, tok), np.uint64)
    for s in range(sets):
        for t in range(tok):
            p = rng.integers(-1, t) if t else -1
            out[s, t] = np.uint64(1 << t) | (out[s, p] if p >= 0 else np.uint64(0))
        out[s, rng.random(tok) < pad] = 0
    return out.view(np.int64)


def _run(ctx, sq, tok, gqa, kernel, window=0, sinks=0, q_pos=None, bits=None):
    torch = sq.torch
    ctx.set_kernel(kernel)
    try:
        plan = pa.CachePlan(ctx, sq.cache, len(sq.lens), tok, gqa, sq.max_pages, window, sinks, bits is not None)
    finally:
        ctx.set_kernel(0)
    Qs = sq.q(tok, gqa)
    tb = None if bits is None else torch.from_numpy(bits).cuda()
    qp = None if q_pos is None else torch.tensor(q_pos, dtype=torch.int32, device="cuda")
    out = plan.reply(sq.layer, Qs, sq.table, sq.n_keys, qp, tb)
    part = plan.run(sq.layer, Qs, sq.table, sq.n_keys, qp, tb)
    ctx.status()
    _check(sq, Qs, out, tok, gqa, window, sinks, q_pos, None if bits is None else tb.cpu(), partial=part)
    plan.close()


KERNELS = [0, 1, 2, 3]
LENS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 129, 500, 1031]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("quant", QUANTS)
@pytest.mark.parametrize("hd,nkv,gqa,tok", [(128, 8, 5, 1), (256, 4, 6, 1), (128, 4, 3, 5), (256, 8, 4, 12), (128, 2, 7, 40)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 4), (100, 65), (700, 17)])
def test_window(ctx, kernel, quant, hd, nkv, gqa, tok, window, sinks):
    if kernel >= 2 and quant == pa.F16:
        pytest.skip("f16 rows run on the split-K kernel")
    sq = Seqs(11 * tok + window, LENS, hd, nkv, quant, 64 if hd == 128 else 128)
    _run(ctx, sq, tok, gqa, kernel, window, sinks)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("quant", QUANTS)
@pytest.mark.parametrize("hd,nkv,gqa,tok", [(128, 8, 5, 1), (256, 4, 6, 7), (128, 2, 8, 33), (128, 4, 1, 64), (256, 8, 1, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 70)])
def test_tree(ctx, kernel, quant, hd, nkv, gqa, tok, window, sinks):
    if kernel >= 2 and quant == pa.F16:
        pytest.skip("f16 rows run on the split-K kernel")
    sq = Seqs(13 * tok + hd, LENS, hd, nkv, quant, 64 if hd == 128 else 192)
    _run(ctx, sq, tok, gqa, kernel, window, sinks, bits=_tree(np.random.default_rng(tok), len(LENS), tok, 0.2))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3), (1 << 30, (1 << 32) - 1)])
def test_positions_of_the_queries(ctx, kernel, bits, window, sinks):
    """q_pos before, inside, right behind and far behind the keys held (an older position range), up to int32's ends"""
    tok, lens = 6, [200] * 9
    q_pos = [-2 ** 31, -3, 0, 100, 194, 200, 260, 2 ** 31 - 1, 199]
    sq = Seqs(5, lens)
    _run(ctx, sq, tok, 5, kernel, window, sinks, q_pos, _tree(np.random.default_rng(1), 9, tok, 0.1) if bits else None)


@pytest.mark.parametrize("kernel,quant", [(0, pa.Q8_0), (1, pa.Q4_0), (2, pa.Q8_0), (3, pa.Q8_0)])
def test_many_ragged_sequences(ctx, kernel, quant):
    """more units than a warp has lanes: their parts are found in rounds, and every length keeps its own"""
    rng = np.random.default_rng(5)
    sq = Seqs(6, [int(x) for x in np.exp(rng.uniform(0, np.log(900), 71))] + [0], 128, 2, quant, 64, layers=1)
    _run(ctx, sq, 3, 5, kernel)
    _run(ctx, sq, 30, 9, kernel, 50, 5)


@pytest.mark.parametrize("kernel", [1, 2])
def test_more_sequences_than_a_block_has_threads(ctx, kernel):
    """over 1,024 units: dealt out in several rounds, empty sequences and one long one among them"""
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(0, 90, 1040)]
    lens[700], lens[:3], lens[-1] = 3000, [0, 0, 0], 0
    _run(ctx, Seqs(8, lens, 128, 2, pa.Q8_0, 64, layers=1), 1, 1, kernel)


@pytest.mark.parametrize("kernel,quant", [(0, pa.Q8_0), (1, pa.Q4_0), (2, pa.Q4_0), (3, pa.Q4_0), (0, pa.F16)])
def test_many_rows_and_a_long_cache(ctx, kernel, quant):
    """several row tiles, several parts of a sequence, wide pages, rows with padding bytes"""
    sq = Seqs(3, [4097, 130, 2500], 128, 8, quant, 1024, pad_row=16)
    _run(ctx, sq, 75, 5, kernel, 333, 21)
    _run(ctx, sq, 110, 5, kernel, 333, 21)
    _run(ctx, sq, 60, 5, kernel, bits=_tree(np.random.default_rng(2), 3, 60))


@pytest.mark.parametrize("kernel", KERNELS)
def test_masked_rows_may_hold_anything(ctx, kernel):
    """NaN and infinite rows where no token looks: between the sinks and the window, a draft no mask names"""
    torch = __import__("torch")
    sq = Seqs(8, [700], 128, 8, pa.Q8_0, 64)
    nan = sq.rows(0, np.arange(5, 500))
    for pool in (sq.cache.K, sq.cache.V):
        pool[sq.layer].view(-1, sq.cache.rs)[nan] = 0xFF
    _run(ctx, sq, 4, 5, kernel, window=190, sinks=5)
    sq = Seqs(9, [300], 128, 8, pa.Q4_0, 64)
    for pool in (sq.cache.K, sq.cache.V):
        pool[sq.layer].view(-1, sq.cache.rs)[sq.rows(0, [297])] = 0xFF   # drafted token 2 of 5
    _run(ctx, sq, 5, 5, kernel, bits=np.array([[1, 3, 0, 9, 27]], np.int64))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("tok", [1, 9])
def test_captured_call_follows_lengths_tables_and_masks(ctx, kernel, tok):
    torch = __import__("torch")
    sq = Seqs(21, [900, 40, 333], extra=0)
    ctx.set_kernel(kernel)
    plan = pa.CachePlan(ctx, sq.cache, 3, tok, 5, sq.max_pages, tree=True)
    ctx.set_kernel(0)
    Qs = sq.q(tok, 5)
    bits = torch.from_numpy(_tree(np.random.default_rng(0), 3, tok)).cuda()
    n, table = sq.n_keys.clone(), sq.table.clone()
    out = (torch.empty_like(Qs), torch.empty(Qs.shape[:3], device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan.reply(0, Qs, table, n, tree=bits, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan.reply(sq.layer, Qs, table, n, tree=bits, out=out)
    for lens in ([900, 40, 333], [13, 40, 0], [899, 12, 1]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        bits.copy_(torch.from_numpy(_tree(np.random.default_rng(lens[0]), 3, tok, 0.3)))
        graph.replay()
        torch.cuda.synchronize()
        ctx.status()
        _check(sq, Qs, out, tok, 5, bits=bits.cpu(), lens=lens)
    del graph
    plan.close()


def test_partials_of_two_caches_merge_to_the_whole(ctx):
    """an older range here, the newest keys there: the partials fold to the attention over both"""
    torch = __import__("torch")
    sq = Seqs(31, [1000], page=64)
    tok, gqa, W, S = 3, 5, 400, 10
    Qs = sq.q(tok, gqa)
    whole = pa.CachePlan(ctx, sq.cache, 1, tok, gqa, sq.max_pages, W, S)
    ref = whole.run(sq.layer, Qs, sq.table, sq.n_keys)
    i32 = dict(dtype=torch.int32, device="cuda")
    a = whole.run(sq.layer, Qs, sq.table, torch.tensor([704], **i32), q_pos=torch.tensor([997], **i32))
    newer = pa.CachePlan(ctx, sq.cache, 1, tok, gqa, sq.max_pages - 11, W, 0)
    b = newer.run(sq.layer, Qs, sq.table[:, 11:].contiguous(), torch.tensor([296], **i32), q_pos=torch.tensor([293], **i32))
    O, m, l = pa.merge(ctx, 128, *(torch.stack([x.reshape(-1, *x.shape[3:]), y.reshape(-1, *y.shape[3:])]) for x, y in zip(a, b)))
    ctx.status()
    got, want = pa.normalize(ctx, 128, O, m, l), pa.normalize(ctx, 128, *(t.reshape(-1, *t.shape[3:]) for t in ref))
    assert float((got[0].double() - want[0].double()).abs().max()) <= 2.0 ** -9 * float(want[0].double().abs().max())
    assert float((got[1] - want[1]).abs().max()) <= 1e-4


def test_two_plans_on_two_streams(ctx):
    import torch
    sq = Seqs(41, [1500, 700, 30], page=64)
    streams = [torch.cuda.Stream() for _ in range(2)]
    plans = [pa.CachePlan(ctx, sq.cache, 3, tok, 5, sq.max_pages) for tok in (1, 9)]
    Qs = [sq.q(tok, 5) for tok in (1, 9)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(plans[i].reply(sq.layer, Qs[i], sq.table, sq.n_keys))
    torch.cuda.synchronize()
    ctx.status()
    for i, tok in enumerate((1, 9)):
        _check(sq, Qs[i], outs[i][0], tok, 5)
        for o in outs[i][1:]:   # and every call gives the same bits
            assert torch.equal(o[0], outs[i][0][0]) and torch.equal(o[1], outs[i][0][1])
        plans[i].close()


@pytest.mark.parametrize("kernel", [1, 2, 3])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(ctx, kernel):
    sq = Seqs(43, [300, 80], page=64)
    ctx.set_kernel(kernel)
    plan = pa.CachePlan(ctx, sq.cache, 2, 3, 5, sq.max_pages)
    ctx.set_kernel(0)
    Qs = sq.q(3, 5)
    ctx.set_timeout_ns(20_000_000)
    ctx.set_stall_test(True)
    try:
        plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
        with pytest.raises(pa.PaCudaError) as e:
            ctx.status()
        assert e.value.code == api.ETIMEOUT
    finally:
        ctx.set_stall_test(False)
        ctx.set_timeout_ns(2_000_000_000)
    out = plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
    ctx.status()
    _check(sq, Qs, out, 3, 5)
    plan.close()


@pytest.mark.parametrize("kernel", [1, 2, 3])
def test_pages_past_four_gigabytes(ctx, kernel):
    """row offsets that pass 32 bits: every call on the last pages of a layer of 4.6 GB"""
    import torch
    n_pages = 1040
    c = pa.Cache(128, 8, pa.Q8_0, 1, n_pages, 4096)
    assert n_pages * 4096 * c.rs > 1 << 32
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    i32 = dict(dtype=torch.int32, device="cuda")
    far, near = torch.tensor([[n_pages - 1]], **i32), torch.tensor([[2]], **i32)
    x = [torch.randn(1, 300, k, 128, generator=g, device="cuda") for k in (40, 8, 8)]
    start = torch.tensor([0], **i32)
    ctx.set_kernel(kernel)
    plan = pa.CachePlan(ctx, c, 1, 300, 5, 1)
    ctx.set_kernel(0)
    out = []
    for t in (far, near):
        Qs = pa.cache_append(ctx, c, 0, *x, t, start, scale=128 ** -0.5)
        out.append((*pa.cache_rows(ctx, c, 0, t, start, 300), *plan.reply(0, Qs, t, torch.tensor([300], **i32))))
    for a, b in zip(*out):
        assert torch.equal(a, b) and bool(a.float().abs().max() > 0)
    path = torch.zeros(1, 300, **i32)   # of 300 tokens every third is kept
    path[0, :100] = torch.arange(0, 300, 3)
    for t in (far, near):
        pa.cache_compact(ctx, c, t, start, path, torch.tensor([100], **i32))
    a, b = (pa.cache_rows(ctx, c, 0, t, start, 100) for t in (far, near))
    assert torch.equal(a[0], out[0][0][:, ::3]) and all(torch.equal(u, v) for u, v in zip(a, b))
    pa.cache_copy_pages(ctx, c, far[0], torch.tensor([5], **i32))
    ctx.status()
    assert torch.equal(c.K[0, 5], c.K[0, n_pages - 1]) and torch.equal(c.V[0, 5], c.V[0, n_pages - 1])
    plan.close()


# ------------------------------------------------------------------------------------------------- append
def _turned(torch, y, pos, freqs, inter):
    """float64 [S][T][H][hd], the first 2 * len(freqs) dims turned"""
    half = freqs.numel()
    a = pos.double()[:, :, None, None] * freqs
    y = y.clone()
    i = torch.arange(half, device=y.device)
    f, g = (2 * i, 2 * i + 1) if inter else (i, i + half)
    u, w = y[..., f].clone(), y[..., g].clone()
    y[..., f], y[..., g] = u * a.cos() - w * a.sin(), w * a.cos() + u * a.sin()
    return y


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("quant", QUANTS)
@pytest.mark.parametrize("hd,nkv,gqa,tok,rot,inter,view", [
    (128, 8, 5, 1, 128, False, "slice"), (256, 4, 6, 13, 64, True, "slice"), (128, 2, 1, 70, 20, False, "own"),
    (256, 8, 2, 3, 256, False, "odd"), (128, 4, 16, 5, 0, False, "odd"), (128, 8, 5, 300, 128, True, "slice")])
def test_append(ctx, dtype, quant, hd, nkv, gqa, tok, rot, inter, view):
    import torch
    dt, S = getattr(torch, dtype), 3
    start = [0, 61, 500]
    sq = Seqs(tok, [0, 0, 0], hd, nkv, quant, 64, extra=500 + tok, pad_row=32)
    nq = nkv * gqa
    if view == "own":
        q, k, v = (torch.randn(S, tok, n, hd, generator=sq.g, device="cuda").to(dt) for n in (nq, nkv, nkv))
    else:   # slices of one projection's output; "odd": starting one element into a row of an odd length
        o = 1 if view == "odd" else 0
        x = torch.randn(S, tok, (nq + 2 * nkv) * hd + o, generator=sq.g, device="cuda").to(dt)[:, :, o:]
        q, k, v = (x[:, :, a * hd:b * hd].unflatten(-1, (b - a, hd)) for a, b in
                   ((0, nq), (nq, nq + nkv), (nq + nkv, nq + 2 * nkv)))
    wdt = torch.float32 if tok % 2 else dt
    wq, wk = ((1 + 0.3 * torch.randn(hd, generator=sq.g, device="cuda")).to(wdt) for _ in range(2))
    freqs = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / max(1, rot))
    pos = torch.randint(0, 1 << 20, (S, tok), generator=sq.g, device="cuda", dtype=torch.int32)
    pos[2, tok // 2:] = -1 if tok > 1 else 7
    before = [p.clone() for p in (sq.cache.K, sq.cache.V)]
    st = torch.tensor(start, dtype=torch.int32, device="cuda")
    Qs = pa.cache_append(ctx, sq.cache, sq.layer, q, k, v, sq.table, st, pos=pos, wq=wq, wk=wk,
                         freqs=freqs if rot else None, eps=1e-5, scale=0.0883, interleaved=inter)
    got = pa.cache_rows(ctx, sq.cache, sq.layer, sq.table, st, tok)
    ctx.status()
    real = pos >= 0
    y = []
    for x, w in ((q, wq), (k, wk)):
        x = x.double()
        x = x / (x.square().mean(-1, keepdim=True) + float(np.float32(1e-5))).sqrt() * w.double()
        y.append(_turned(torch, x, pos, freqs, inter) if rot else x)
    # Qs: fp32 arithmetic (some 20 roundings of 2^-24 of the pair's size) and one rounding to f16
    want = torch.where(real[:, :, None, None], y[0] * float(np.float32(0.0883)), 0.0)
    size = y[0].abs().amax(-1, keepdim=True) * 0.0883
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -19 * size + 2.0 ** -25
    mine = Qs.view(S, nkv, gqa, tok, hd).permute(0, 3, 1, 2, 4).reshape(S, tok, nq, hd).double()
    assert bool(((mine - want).abs() <= tol).all())
    # rows: a value is at most half a step of its block from the exact one (d = amax / top, itself rounded to f16), plus f16's
    # rounding of d * q
    for got_x, x in zip(got, (y[1], v.double())):
        g = got_x.double()[real]
        x = x[real]
        size = x.abs().amax(-1, keepdim=True) * 2.0 ** -19
        if quant == pa.F16:
            t = 2.0 ** -11 * x.abs() + size
        else:
            top = 127 if quant == pa.Q8_0 else 7
            am = x.unflatten(-1, (hd // 32, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
            t = am / top * (0.5 + top * 2.0 ** -11 + 2.0 ** -10) + 2.0 ** -11 * (x.abs() + am / top) + size
        assert bool(((g - x).abs() <= t + 2.0 ** -24).all())
    # V takes no arithmetic: its rows are the formula's bytes (on the CPU: on the GPU torch divides by a
    # number as it multiplies by its rounded reciprocal, and max|x| * (1/7) is not always max|x| / 7); nothing else changed
    flat = [p[sq.layer].view(-1, sq.cache.rs) for p in (sq.cache.K, sq.cache.V)]
    touched = torch.zeros(flat[0].shape[0], dtype=torch.bool, device="cuda")
    for s in range(S):
        js = np.arange(start[s], start[s] + tok)[real[s].cpu().numpy()]
        at = sq.rows(s, js)
        touched[at] = True
        rows = _stored(torch, v[s][real[s]].float().cpu(), quant).reshape(len(js), nkv * sq.hb).cuda()
        assert torch.equal(flat[1][at, :nkv * sq.hb], rows)
        assert bool((flat[1][at, nkv * sq.hb:] == 0xFF).all()) and bool((flat[0][at, nkv * sq.hb:] == 0xFF).all())
    for i, p in enumerate((sq.cache.K, sq.cache.V)):
        assert torch.equal(p[0], before[i][0])
        assert torch.equal(flat[i][~touched], before[i][sq.layer].view(-1, sq.cache.rs)[~touched])


def test_append_without_norm_positions_or_rotation_and_far_positions(ctx):
    import torch
    sq = Seqs(2, [0], 128, 8, pa.F16, 64, extra=200)
    x = [torch.randn(1, 4, n, 128, generator=sq.g, device="cuda") for n in (8, 8, 8)]
    st = torch.tensor([100], dtype=torch.int32, device="cuda")
    Qs = pa.cache_append(ctx, sq.cache, 1, *x, sq.table, st)
    K, V = pa.cache_rows(ctx, sq.cache, 1, sq.table, st, 4)
    assert torch.equal(Qs, x[0].transpose(1, 2).half()) and torch.equal(K, x[1].half()) and torch.equal(V, x[2].half())
    freqs = torch.ones(64, dtype=torch.float64, device="cuda")   # a radian per position, two thousand million positions on
    pos = torch.tensor([[0, 1, 2 ** 31 - 1, 2 ** 30 + 7]], dtype=torch.int32, device="cuda")
    pa.cache_append(ctx, sq.cache, 1, *x, sq.table, st, pos=pos, freqs=freqs)
    K, _ = pa.cache_rows(ctx, sq.cache, 1, sq.table, st, 4)
    ctx.status()
    want = _turned(torch, x[1].double(), pos, freqs, False)
    # angle in turns to 2^-53 * 2^28.4 turns, so 2^-21 radians of a pair at most 8 long
    assert bool(((K.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -17).all())
    pa.cache_append(ctx, sq.cache, 1, *x, sq.table, st, freqs=freqs)   # positions: the key indexes
    K, _ = pa.cache_rows(ctx, sq.cache, 1, sq.table, st, 4)
    want = _turned(torch, x[1].double(), torch.arange(100, 104, device="cuda")[None], freqs, False)
    assert bool(((K.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -17).all())
    # nothing to do
    for shape in ((0, 4), (1, 0)):
        e = [t[:shape[0], :shape[1]] for t in x]
        assert pa.cache_append(ctx, sq.cache, 1, *e, sq.table[:shape[0]], st[:shape[0]]).numel() == 0
    ctx.status()


# ------------------------------------------------------------------------------------------------- row moves
@pytest.mark.parametrize("quant,hd,nkv,page,n", [(pa.Q8_0, 128, 8, 64, 5), (pa.Q4_0, 256, 4, 192, 17), (pa.F16, 128, 2, 64, 1)])
def test_copy_pages(ctx, quant, hd, nkv, page, n):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    c = pa.Cache(hd, nkv, quant, 3, 3 * n, page)
    for p in (c.K, c.V):
        p.copy_(torch.randint(0, 256, p.shape, dtype=torch.uint8, generator=g, device="cuda"))
    order = torch.randperm(3 * n, generator=g, device="cuda")
    src, dst = order[:n].clone(), order[n:2 * n].clone()
    src[n // 2] = src[0]                       # one page copied twice
    dst[0] = src[0] if n > 2 else dst[0]       # onto itself: nothing
    want = []
    for p in (c.K, c.V):
        w = p.clone()
        w[:, dst] = p[:, src]
        want.append(w)
    pa.cache_copy_pages(ctx, c, src.int(), dst.int())
    pa.cache_copy_pages(ctx, c, src[:0].int(), dst[:0].int())
    ctx.status()
    assert torch.equal(c.K, want[0]) and torch.equal(c.V, want[1])


@pytest.mark.parametrize("quant,hd,nkv,page,tok", [(pa.Q8_0, 128, 8, 64, 1), (pa.Q4_0, 128, 8, 64, 64), (pa.F16, 256, 4, 128, 37),
                                                   (pa.Q8_0, 256, 8, 64, 1024)])
def test_compact(ctx, quant, hd, nkv, page, tok):
    import torch
    rng = np.random.default_rng(tok)
    sq = Seqs(tok, [3, 60, 200, 64, 10], hd, nkv, quant, page, layers=3, extra=tok)
    S = 5
    for p in (sq.cache.K, sq.cache.V):
        p.copy_(torch.randint(0, 256, p.shape, dtype=torch.uint8, generator=sq.g, device="cuda"))
    count = np.array([0, tok, min(1, tok), (tok + 1) // 2, max(1, tok // 3)], np.int32)
    path = np.full((S, tok), -5, np.int32)     # entries past the count are not looked at
    for s in range(S):
        path[s, :count[s]] = np.sort(rng.choice(tok, count[s], replace=False))
    want = []
    for p in (sq.cache.K, sq.cache.V):
        w = p.clone().view(3, -1, sq.cache.rs)
        for s in range(S):
            a = sq.rows(s, sq.lens[s] + path[s, :count[s]])
            b = sq.rows(s, sq.lens[s] + np.arange(count[s]))
            w[:, b] = p.view(3, -1, sq.cache.rs)[:, a]
        want.append(w.view(p.shape))
    n = pa.cache_compact(ctx, sq.cache, sq.table, sq.n_keys, torch.from_numpy(path).cuda(), torch.from_numpy(count).cuda())
    ctx.status()
    assert torch.equal(sq.cache.K, want[0]) and torch.equal(sq.cache.V, want[1])
    assert n.tolist() == [a + int(b) for a, b in zip(sq.lens, count)]


# ------------------------------------------------------------------------------------------------- refusals
def _invalid(ctx):
    with pytest.raises(pa.PaCudaError) as e:
        ctx.status()
    assert e.value.code == api.EINVAL and "out of range" in str(e.value)
    ctx.status()   # cleared


def test_arguments_only_the_device_sees(ctx):
    """page ids, lengths and paths out of range are reported and do no harm"""
    import torch
    sq = Seqs(4, [100, 100], page=64, extra=100)
    total = sq.cache.n_pages
    keep = [p.clone() for p in (sq.cache.K, sq.cache.V)]
    Qs = sq.q(2, 5)
    i32 = dict(dtype=torch.int32, device="cuda")
    for kernel in KERNELS:
        ctx.set_kernel(kernel)
        plan = pa.CachePlan(ctx, sq.cache, 2, 2, 5, sq.max_pages)
        ctx.set_kernel(0)
        for bad in (-1, total, 2 ** 31 - 1, -2 ** 31):
            t = sq.table.clone()
            t[1, 1] = bad
            plan.reply(0, Qs, t, sq.n_keys)
            _invalid(ctx)
        for n in (-1, sq.max_pages * 64 + 1, 2 ** 31 - 1, -2 ** 31):
            plan.reply(0, Qs, torch.zeros_like(sq.table), torch.tensor([100, n], **i32))
            _invalid(ctx)
        # a call after a bad one is as good as any, whether the status was looked at or not
        bad = sq.table.clone()
        bad[0, 0] = total
        plan.reply(0, Qs, bad, sq.n_keys)
        out = plan.reply(sq.layer, Qs, sq.table, sq.n_keys)
        _invalid(ctx)
        _check(sq, Qs, out, 2, 5)
        plan.close()
    x = [torch.randn(2, 2, n, 128, generator=sq.g, device="cuda") for n in (40, 8, 8)]
    for start in ([-2, 5], [5, sq.max_pages * 64 - 1], [5, 2 ** 31 - 1], [5, 64 * (sq.max_pages - 1)]):
        pa.cache_append(ctx, sq.cache, 0, *x, sq.table, torch.tensor(start, **i32), pos=torch.zeros(2, 2, **i32))
        _invalid(ctx)
        pa.cache_rows(ctx, sq.cache, 0, sq.table, torch.tensor(start, **i32), 2)
        _invalid(ctx)
    sq.cache.K.copy_(keep[0])
    sq.cache.V.copy_(keep[1])
    for a, b in ((0, total), (-1, 0), (2 ** 31 - 1, -2 ** 31)):
        pa.cache_copy_pages(ctx, sq.cache, torch.tensor([a], **i32), torch.tensor([b], **i32))
        _invalid(ctx)
    one = [100, 100]
    for start, path, count in ((one, [[1, 0], [0, 1]], [2, 0]), (one, [[0, 2], [0, 1]], [2, 0]), (one, [[-1, 0], [0, 1]], [2, 0]),
                               (one, [[1, 1], [0, 1]], [2, 0]), (one, [[0, 1], [0, 1]], [3, 0]), (one, [[0, 1], [0, 1]], [-1, 0]),
                               ([-1, 100], [[0, 1], [0, 1]], [1, 0]), ([64 * sq.max_pages - 1, 100], [[0, 1], [0, 1]], [1, 0]),
                               ([2 ** 31 - 1, 100], [[0, 1], [0, 1]], [1, 0])):
        n = pa.cache_compact(ctx, sq.cache, sq.table, torch.tensor(start, **i32), torch.tensor(path, **i32), torch.tensor(count, **i32))
        assert n.tolist() == start
        _invalid(ctx)
    assert torch.equal(sq.cache.K, keep[0]) and torch.equal(sq.cache.V, keep[1])


def test_refusals(ctx):
    import torch
    c = pa.Cache(128, 8, pa.Q8_0, 2, 4, 64)

    def no(code, f, *a, **k):
        with pytest.raises(pa.PaCudaError) as e:
            f(*a, **k)
        assert e.value.code == code, str(e.value)

    P, U, I = pa.CachePlan, api.EUNSUPPORTED, api.EINVAL
    no(I, P, ctx, c, 0, 1, 5, 4)
    no(I, P, ctx, c, 1, 0, 5, 4)
    no(I, P, ctx, c, 1, 1, 0, 4)
    no(I, P, ctx, c, 1, 1, 5, 0)
    no(I, P, ctx, c, 1, 1, 5, (1 << 24) + 1)
    no(I, P, ctx, c, 1, 1, 5, 4, 0, 3)                 # sinks without a window
    no(I, P, ctx, c, 1, 1, 5, 4, (1 << 30) + 1)
    no(U, P, ctx, c, 1, 65, 5, 4, tree=True)
    no(U, P, ctx, c, 1, 9, 5, 4, 8, tree=True)
    no(U, P, ctx, c, 65536, 1, 5, 4)
    for k in (2, 3):
        ctx.set_kernel(k)
        no(U, P, ctx, pa.Cache(128, 8, pa.F16, 1, 4, 64), 1, 1, 5, 4)
        ctx.set_kernel(0)
    no(U, P, ctx, c, 65535, 1 << 14, 1, 4)
    no(U, P, ctx, pa.Cache(128, 8, pa.Q8_0, 1, 4, 96), 1, 1, 5, 4)
    no(U, P, ctx, pa.Cache(64, 8, pa.Q8_0, 1, 4, 64), 1, 1, 5, 4)
    no(I, P, ctx, pa.Cache(128, 8, pa.Q8_0, 1, 4, 64, rs=1024), 1, 1, 5, 4)
    no(U, P, ctx, pa.Cache(128, 8, pa.Q8_0, 1, 4, 64, rs=1096), 1, 1, 5, 4)
    ctx.set_qk_domain(pa.QK_INT8)
    no(U, P, ctx, c, 1, 1, 5, 4)
    ctx.set_qk_domain(pa.QK_F16)
    i32 = dict(dtype=torch.int32, device="cuda")
    plan = P(ctx, c, 1, 1, 5, 4)
    Q, t, n = torch.zeros(1, 8, 5, 128, dtype=torch.float16, device="cuda"), torch.zeros(1, 4, **i32), torch.ones(1, **i32)
    no(I, plan.reply, 2, Q, t, n)
    no(I, plan.reply, 0, Q.float(), t, n)
    no(I, plan.reply, 0, Q[:, :, :4], t, n)
    no(I, plan.reply, 0, Q, t.long(), n)
    no(I, plan.reply, 0, Q, t[:, :3], n)
    no(I, plan.reply, 0, Q, t, n.cpu())
    no(I, plan.reply, 0, Q, t, n, tree=torch.zeros(1, 1, dtype=torch.int64, device="cuda"))
    flat = torch.zeros(5 * 8 * 128 + 1, dtype=torch.float16, device="cuda")[1:]
    no(I, plan.reply, 0, flat.view(1, 8, 5, 128), t, n)   # 16-byte alignment
    no(I, plan.run, 0, Q, t, n, out=(Q, Q, Q))
    L, q, i, o, z = pa.lib(), Q.data_ptr(), t.data_ptr(), torch.zeros(1, 8, 5, device="cuda").data_ptr(), n.data_ptr()
    for a in ((q, i + 2, z, 0, 0, q, o), (q, i, z + 1, 0, 0, q, o), (q, i, z, z + 2, 0, q, o), (q, i, z, 0, 0, q + 8, o),
              (q, i, z, 0, 0, q, o + 2), (0, i, z, 0, 0, q, o), (q, 0, z, 0, 0, q, o), (q, i, z, 0, 0, 0, o)):
        assert L.pa_cuda_cache_attn_reply(plan._h, 0, *a, None) == api.EINVAL
    x = [torch.zeros(1, 1, k, 128, device="cuda") for k in (40, 8, 8)]
    no(I, pa.cache_append, ctx, c, 0, x[0][..., :64], x[1], x[2], t, n)
    no(I, pa.cache_append, ctx, c, 0, x[0][:, :, :39], x[1], x[2], t, n)
    no(I, pa.cache_append, ctx, c, 0, x[0], x[1].half(), x[2], t, n)
    no(I, pa.cache_append, ctx, c, 0, x[0].double(), x[1].double(), x[2].double(), t, n)
    no(I, pa.cache_append, ctx, c, 0, x[0].transpose(2, 3).contiguous().transpose(2, 3), x[1], x[2], t, n)
    no(I, pa.cache_append, ctx, c, 2, *x, t, n)
    no(I, pa.cache_append, ctx, c, 0, *x, t, n, freqs=torch.zeros(65, dtype=torch.float64, device="cuda"))
    no(I, pa.cache_append, ctx, c, 0, *x, t, n, freqs=torch.zeros(64, device="cuda"))
    no(U, pa.cache_append, ctx, c, 0, *x, t, n, wq=torch.zeros(128, dtype=torch.float16, device="cuda"))
    no(U, pa.cache_compact, ctx, c, t, n, torch.zeros(1, 1025, **i32), n)
    no(U, pa.cache_compact, ctx, c, t, n, torch.zeros(1, 0, **i32), n)
    plan.close()


def test_compact_does_not_write_the_lengths_over_an_input(ctx):
    """n_keys_out over start, count, path or table: blocks of a set read what another has written"""
    import torch
    c = pa.Cache(128, 8, pa.Q8_0, 1, 4, 64)
    buf = torch.zeros(16, dtype=torch.int32, device="cuda")
    start, count, path, table, out = buf[:2], buf[2:4], buf[4:10].view(2, 3), buf[10:14].view(2, 2), buf[14:]
    for bad in (start, count, buf[1:3], path.view(-1)[1:3], buf[9:11], buf[13:15]):
        with pytest.raises(pa.PaCudaError) as e:
            pa.cache_compact(ctx, c, table, start, path, count, out=bad)
        assert e.value.code == api.EINVAL
    assert pa.cache_compact(ctx, c, table, start, path, count, out=out).tolist() == [0, 0]


# ------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("quant", QUANTS)
def test_a_generation_with_drafts(ctx, quant):
    """prompt, then draft -> append -> verify -> keep an accepted path, on a side stream, against the same sequence kept as
    plain rows: what the cache holds and what the attention gives stay the sequence's own; then a fork"""
    import torch
    S, hd, nkv, gqa, T, W, sinks = 2, 128, 8, 2, 6, 64, 3
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g = torch.Generator(device="cuda")
        g.manual_seed(1)
        c = pa.Cache(hd, nkv, quant, 2, 16, 64)
        table = torch.tensor([[3, 7, 1, 15], [2, 9, 4, 0]], dtype=torch.int32, device="cuda")
        freqs = 1e4 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        wk = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
        n = torch.zeros(S, dtype=torch.int32, device="cuda")
        held = [[torch.empty(S, 0, nkv, hd, device="cuda", dtype=torch.float16) for _ in range(2)] for _ in range(2)]

        def new(tok):
            return [torch.randn(S, tok, k, hd, generator=g, device="cuda") for k in (nkv * gqa, nkv, nkv)]

        for layer in range(2):
            x = new(61)
            pa.cache_append(ctx, c, layer, *x, table, n, wq=wk, wk=wk, freqs=freqs)
            held[layer] = list(pa.cache_rows(ctx, c, layer, table, n, 61))
        n = n + 61
        plan = pa.CachePlan(ctx, c, S, T, gqa, 4, W, sinks, tree=True)
        rng = np.random.default_rng(3)
        for step in range(5):
            bits = _tree(rng, S, T)
            tb = torch.from_numpy(bits).cuda()
            depth = torch.tensor([[bin(int(b) & (2 ** 64 - 1)).count("1") - 1 for b in r] for r in bits], device="cuda")
            pos = (n[:, None] + depth).to(torch.int32)
            draft = []
            for layer in range(2):
                x = new(T)
                Qs = pa.cache_append(ctx, c, layer, *x, table, n, pos=pos, wq=wk, wk=wk, freqs=freqs, scale=hd ** -0.5)
                out = plan.reply(layer, Qs, table, n + T, tree=tb)
                draft.append(pa.cache_rows(ctx, c, layer, table, n, T))
                ctx.status()
                L = held[layer][0].shape[1]
                for s in range(S):
                    K, V = (torch.cat([a[s], b[s]]).double() for a, b in zip(held[layer], draft[layer]))
                    see = torch.from_numpy(_sees(torch, L + T, L, T, W, sinks, bits[s].tolist())).cuda().repeat(gqa, 1)
                    for h in range(nkv):
                        xs = torch.where(see, Qs[s, h].double() @ K[:, h].T, -math.inf)
                        O = torch.softmax(xs, 1) @ V[:, h]
                        A = torch.softmax(xs, 1) @ V[:, h].abs()
                        assert bool(((out[0][s, h].double() - O).abs() <= 2.0 ** -9 * A + 2.0 ** -24).all())
                        assert bool(((out[1][s, h] - torch.logsumexp(xs, 1)).abs() <= 1e-4).all())
            # the path of one token: its ancestors in order; the same number of tokens for both sequences
            last = [int(np.argmax(depth[s].cpu().numpy() == 1)) if (depth[s] == 1).any() else 0 for s in range(S)]
            path = [[t for t in range(T) if int(bits[s][last[s]]) >> t & 1] for s in range(S)]
            k = min(map(len, path))
            p = torch.tensor([(r[:k] + [0] * T)[:T] for r in path], dtype=torch.int32, device="cuda")
            n = pa.cache_compact(ctx, c, table, n, p, torch.full((S,), k, dtype=torch.int32, device="cuda"))
            for layer in range(2):
                for i in range(2):
                    kept = torch.stack([draft[layer][i][s][path[s][:k]] for s in range(S)])
                    held[layer][i] = torch.cat([held[layer][i], kept], 1)
                now = pa.cache_rows(ctx, c, layer, table, torch.zeros_like(n), held[layer][0].shape[1])
                assert torch.equal(now[0], held[layer][0]) and torch.equal(now[1], held[layer][1])
            assert n.tolist() == [held[0][0].shape[1]] * S
        # sequence 0 forked into sequence 1's place: the full first page shared, the second copied
        pa.cache_copy_pages(ctx, c, table[0, 1:2], table[1, 1:2])
        fork = torch.stack([table[0], torch.cat([table[0, :1], table[1, 1:]])])
        a, b = pa.cache_rows(ctx, c, 1, fork, torch.zeros_like(n), int(n[0]))[0]
        ctx.status()
        assert torch.equal(a, b)
        plan.close()
    side.synchronize()
