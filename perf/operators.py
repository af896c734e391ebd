"""The cache operators (attention over a paged cache with a sliding window and sinks, attention for a tree of drafted
tokens, head norm + rotation + append, row moves), as cases to run and measure.

own = False: run() is the operator's plain form in elementary torch operations; own = True: run() makes the calls a
program makes of this package. The cache has the package's layout: per layer and page, page_keys key positions of nkv
heads, each head hd/32 blocks of (f16 d, 32 x int8) for Q8_0, (f16 d, 16 bytes of two nibbles) for Q4_0, or hd f16; the
value a quantised element stands for is f16(d * q). Keys of sequence s are found through the page table."""
import math

import torch

own = False

F16, Q8_0, Q4_0 = 0, 1, 2
LEN_STEP = 7          # sequence lengths of a batch: nk, then down to about a quarter of it in LEN_STEP uneven steps
_CTX = {}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one generated token of one short conversation: latency
        dict(name="window token", op="window", sets=1, tok=1, nk=777, window=512, sinks=4, hd=128, nkv=8, gqa=5,
             quant=Q8_0, page=64, layers=2),
        # one generated token for each of 32 conversations of uneven length
        dict(name="window batch", op="window", sets=32, tok=1, nk=32749, window=4096, sinks=4, hd=256, nkv=4, gqa=6,
             quant=Q8_0, page=256, layers=1),
        # the same over f16 rows, a few tokens at once, a window that ends inside pages
        dict(name="window f16 rows", op="window", sets=6, tok=3, nk=9001, window=1000, sinks=17, hd=128, nkv=8, gqa=2,
             quant=F16, page=128, layers=1),
        # a prompt chunk of 512 tokens
        dict(name="window prompt chunk", op="window", sets=1, tok=512, nk=16384, window=4096, sinks=64, hd=128, nkv=8,
             gqa=5, quant=Q4_0, page=256, layers=1),
        # seven drafted tokens over a short cache
        dict(name="tree small", op="tree", sets=1, tok=7, nk=1003, window=0, sinks=0, hd=128, nkv=8, gqa=5, quant=Q8_0,
             page=64, layers=2),
        # a padded batch of draft trees
        dict(name="tree batch", op="tree", sets=8, tok=16, nk=16301, window=0, sinks=0, hd=256, nkv=4, gqa=6,
             quant=Q4_0, page=256, layers=1),
        # a large tree over the longest cache
        dict(name="tree long", op="tree", sets=1, tok=61, nk=131072, window=0, sinks=0, hd=128, nkv=8, gqa=5,
             quant=Q8_0, page=4096, layers=1),
        # the new token of a decode step
        dict(name="append token", op="append", sets=1, tok=1, nk=5000, hd=128, nkv=8, gqa=5, quant=Q8_0, page=64,
             layers=2, dtype="bfloat16", rot=128, inter=False),
        # the drafted tokens of a batch, partial rotation, f16 rows
        dict(name="append drafts", op="append", sets=16, tok=13, nk=100000, hd=256, nkv=4, gqa=6, quant=F16, page=256,
             layers=1, dtype="float16", rot=64, inter=True),
        # a long prompt
        dict(name="append prompt", op="append", sets=2, tok=8191, nk=65536, hd=128, nkv=8, gqa=5, quant=Q8_0, page=256,
             layers=1, dtype="bfloat16", rot=128, inter=False),
        # the accepted rows of every layer of a batch after a verify step
        dict(name="compact drafts", op="compact", sets=16, tok=32, nk=2048, hd=128, nkv=8, gqa=5, quant=Q8_0, page=64,
             layers=64),
        # the pages of a long prefix copied for another conversation, every layer
        dict(name="copy pages", op="copy", pages=301, hd=256, nkv=4, gqa=6, quant=Q4_0, page=256, layers=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _geometry(rng):
    hd, nkv, gqa = rng.choice([(128, 8, 5), (256, 4, 6), (128, 8, 2), (128, 4, 1), (256, 8, 4), (128, 2, 16)])
    return dict(hd=hd, nkv=nkv, gqa=gqa, page=rng.choice([64, 128, 256, 1024, 4096]))


def draw(rng):
    """One more case of the listed ranges; drawn again until it costs no more than the largest listed case of its kind
    (the plain form's score matrix and the cache's bytes are what it costs)."""
    while True:
        op = rng.choice(["window", "window", "tree", "tree", "append", "compact", "copy"])
        c = dict(op=op, **_geometry(rng))
        c["quant"] = rng.choice([F16, Q8_0, Q4_0])
        if op == "window":
            c.update(sets=_log(rng, 1, 32), tok=_log(rng, 1, 512), nk=_log(rng, 1, 65536), window=_log(rng, 1, 8192),
                     sinks=rng.choice([0, 1, 4, 17, 64, 130]), layers=rng.choice([1, 2, 3]))
        elif op == "tree":
            c.update(sets=_log(rng, 1, 16), tok=_log(rng, 1, 64), nk=_log(rng, 64, 131072), window=0, sinks=0,
                     layers=rng.choice([1, 2, 3]))
            if rng.random() < 0.3:
                c.update(window=_log(rng, 64, 8192), sinks=rng.choice([0, 4, 65]))
        elif op == "append":
            c.update(sets=_log(rng, 1, 64), tok=_log(rng, 1, 8192), nk=_log(rng, 8192, 1000000), layers=rng.choice([1, 2]),
                     dtype=rng.choice(["bfloat16", "float16", "float32"]), rot=rng.choice([c["hd"], c["hd"] // 2, 64]),
                     inter=rng.choice([False, True]))
            # (an element of Q4_0 is 1/7 of its block's largest value: where two correct computations round one of
            # millions of elements differently it stands out far more than an error would, so Q8_0 and f16 rows here)
            c["quant"] = rng.choice([F16, Q8_0])
        elif op == "compact":
            c.update(sets=_log(rng, 1, 64), tok=_log(rng, 1, 64), nk=_log(rng, 64, 4096), layers=_log(rng, 1, 64))
        else:
            c.update(pages=_log(rng, 1, 2000), layers=_log(rng, 1, 64))
        rows = c.get("sets", 1) * c["nkv"] * _row_bytes(c) // c["nkv"]
        if op in ("window", "tree"):
            ok = (c["sets"] * c["nkv"] * c["gqa"] * c["tok"] * c["nk"] <= 335000000 and
                  c["layers"] * rows * (c["nk"] + c["page"]) <= 320000000)
        elif op == "append":
            ok = (c["sets"] * c["tok"] * (c["nkv"] * (c["gqa"] + 2)) * c["hd"] <= 117000000)
        elif op == "compact":
            ok = c["layers"] * rows * (c["nk"] + c["page"] + c["tok"]) <= 2300000000
        else:
            ok = 2 * c["layers"] * c["pages"] * c["page"] * _row_bytes(c) <= 710000000
        if ok:
            return c


def _head_bytes(c):
    return c["hd"] * 2 if c["quant"] == F16 else c["hd"] // 32 * (34 if c["quant"] == Q8_0 else 18)


def _row_bytes(c):
    return -(-c["nkv"] * _head_bytes(c) // 16) * 16


def _lens(c):
    """Keys of each sequence."""
    return [max(1, c["nk"] - c["nk"] * 3 // 4 * (s % LEN_STEP) // LEN_STEP - s) for s in range(c["sets"])]


# ------------------------------------------------------------------------------------------------- inputs
def _quantise(x, quant):
    """float32 [..., hd] -> uint8 rows [..., head bytes]."""
    if quant == F16:
        return x.to(torch.float16).view(torch.uint8)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = 127 if quant == Q8_0 else 7
    d = (b.abs().amax(-1, keepdim=True) / top).to(torch.float16)
    q = torch.round(b / torch.where(d == 0, torch.ones_like(d), d).float()).clamp(-top, top)
    if quant == Q8_0:
        data = q.to(torch.int8).view(torch.uint8)
    else:
        n = (q + 8).to(torch.uint8)
        data = n[..., :16] | (n[..., 16:] << 4)
    return torch.cat([d.view(torch.uint8), data], -1).flatten(-2)


def _pages(c, lens, g, spare=0):
    """A shuffled page table [sets, max_pages] (-1: no page) and the number of pages in the pool."""
    need = [-(-n // c["page"]) for n in lens]
    total = sum(need) + spare + 1
    order = torch.randperm(total, generator=g, device="cuda")
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table, total


def _rows_of(c, s, lens, table):
    """Flat row index (page * page_keys + offset) of every key of sequence s."""
    j = torch.arange(lens[s], device="cuda")
    return table[s].long()[j // c["page"]] * c["page"] + j % c["page"]


def _normal_rows(c, n, g, wide):
    """n quantised rows of values as a model's keys (a few wide channels per head) or values have them."""
    x = torch.randn(n, c["nkv"], c["hd"], generator=g, device="cuda")
    if wide:
        x[:, :, torch.randperm(c["hd"], generator=g, device="cuda")[:4]] *= 8
    out = torch.zeros(n, _row_bytes(c), dtype=torch.uint8, device="cuda")
    out[:, :c["nkv"] * _head_bytes(c)] = _quantise(x, c["quant"]).reshape(n, -1)
    return out


def _pool(c, total, fill):
    """K or V of the whole cache; rows nothing was stored to yet hold whatever the memory held (here: NaN patterns)."""
    return torch.full((c["layers"], total, c["page"], _row_bytes(c)), fill, dtype=torch.uint8, device="cuda")


def _tree_bits(c, lens, g):
    """Ancestors of each drafted token, itself included, as 64-bit masks; from the third sequence on the last tokens are
    padding (no bit set)."""
    T = c["tok"]
    parent = (torch.rand(c["sets"], T, generator=g, device="cuda") * (torch.arange(T, device="cuda") + 1)).long() - 1
    par, bits = parent.tolist(), []
    for s in range(c["sets"]):
        b = []
        for t in range(T):
            b.append((1 << t) | (b[par[s][t]] if par[s][t] >= 0 else 0))
        live = T if s < 2 else max(0, T - s % (T + 1))
        bits.append([(x - (1 << 64) if x >= 1 << 63 else x) if t < live else 0 for t, x in enumerate(b)])
    return torch.tensor(bits, dtype=torch.int64, device="cuda")


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = dict(case=c, layer=c["layers"] - 1)
    if c["op"] == "copy":
        total = 2 * c["pages"]
        st["K"], st["V"] = (torch.randint(0, 256, (c["layers"], total, c["page"], _row_bytes(c)), dtype=torch.uint8,
                                          generator=g, device="cuda") for _ in range(2))
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        st["src"], st["dst"] = order[:c["pages"]].contiguous(), order[c["pages"]:].contiguous()
    elif c["op"] == "append":
        T, nq = c["tok"], c["nkv"] * c["gqa"]
        first = [max(0, n - T) for n in _lens(c)]
        cap = -(-T // c["page"]) + 1          # pages that the new tokens touch; the table starts at their first page
        start = [f % c["page"] for f in first]
        table, total = _pages(c, [cap * c["page"]] * c["sets"], g)
        st["K"], st["V"] = _pool(c, total, 0xFF), _pool(c, total, 0xFF)
        dt = getattr(torch, c["dtype"])
        x = torch.randn(c["sets"], T, nq + 2 * c["nkv"], c["hd"], generator=g, device="cuda")
        x *= torch.exp(torch.randn(x.shape[2], 1, generator=g, device="cuda"))
        x = x.to(dt)
        st["q"], st["k"], st["v"] = x[:, :, :nq], x[:, :, nq:nq + c["nkv"]], x[:, :, nq + c["nkv"]:]
        st["wq"], st["wk"] = ((1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda")).to(dt) for _ in range(2))
        st["freqs"] = 1e6 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
        pos = torch.tensor(first, device="cuda")[:, None] + torch.arange(T, device="cuda")
        pad = torch.arange(c["sets"], device="cuda")[:, None] * 3 % (T + 1)   # trailing padding tokens of each sequence
        st["pos"] = torch.where(torch.arange(T, device="cuda") < T - pad, pos, -1).to(torch.int32)
        st["start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
        st["table"], st["eps"], st["scale"] = table, 1e-6, c["hd"] ** -0.5
    else:
        lens = _lens(c)
        if c["op"] == "compact":   # the drafted rows follow the cached ones
            lens = [n + c["tok"] for n in lens]
        table, total = _pages(c, lens, g)
        st["K"], st["V"] = _pool(c, total, 0xFF), _pool(c, total, 0xFF)
        for s in range(c["sets"]):
            at = _rows_of(c, s, lens, table)
            if c["op"] == "compact":   # row moves do not look at what a row stands for
                for X in (st["K"], st["V"]):
                    X.view(c["layers"], -1, _row_bytes(c))[:, at] = torch.randint(
                        0, 256, (c["layers"], lens[s], _row_bytes(c)), dtype=torch.uint8, generator=g, device="cuda")
            else:
                st["K"][st["layer"]].view(-1, _row_bytes(c))[at] = _normal_rows(c, lens[s], g, True)
                st["V"][st["layer"]].view(-1, _row_bytes(c))[at] = _normal_rows(c, lens[s], g, False)
        st["table"] = table
        if c["op"] == "compact":
            T = c["tok"]
            st["start"] = torch.tensor([n - T for n in lens], dtype=torch.int32, device="cuda")
            count = 1 + torch.randint(0, max(1, T // 2), (c["sets"],), generator=g, device="cuda")
            rank = torch.rand(c["sets"], T, generator=g, device="cuda").argsort(-1)
            keep = rank < count[:, None]
            st["path"] = torch.where(keep, torch.arange(T, device="cuda"), T).sort(-1).values.clamp(max=T - 1).to(torch.int32)
            st["count"] = count.to(torch.int32)
        else:
            st["n_keys"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
            q = torch.randn(c["sets"], c["nkv"], c["gqa"] * c["tok"], c["hd"], generator=g, device="cuda")
            st["Qs"] = (q * c["hd"] ** -0.5).to(torch.float16)
            st["bits"] = _tree_bits(c, lens, g) if c["op"] == "tree" else None
    if own:
        import backburner_b200 as pa
        if "ctx" not in _CTX:
            _CTX["ctx"] = pa.Context(torch.cuda.current_device())
        st["ctx"] = _CTX["ctx"]
        st["cache"] = pa.Cache.of(st["K"], st["V"], hd=c["hd"], nkv=c["nkv"], quant=c["quant"])
        if c["op"] in ("window", "tree"):
            st["plan"] = pa.CachePlan(st["ctx"], st["cache"], n_sets=c["sets"], n_tok=c["tok"], gqa=c["gqa"],
                                      max_pages=st["table"].shape[1], window=c["window"], sinks=c["sinks"],
                                      tree=c["op"] == "tree")
    return st


# ------------------------------------------------------------------------------------------------- one pass
def run(st):
    op = st["case"]["op"]
    if own:
        return _own(st, op)
    if op in ("window", "tree"):
        return _plain_attention(st)
    if op == "append":
        return _plain_append(st)
    return _plain_compact(st) if op == "compact" else _plain_copy(st)


def _own(st, op):
    if op in ("window", "tree"):
        return st["plan"].reply(st["layer"], st["Qs"], st["table"], st["n_keys"], tree=st["bits"])
    import backburner_b200 as pa
    if op == "append":   # the queries for the attention call, and the stored rows read back as the values they stand for
        Qs = pa.cache_append(st["ctx"], st["cache"], st["layer"], st["q"], st["k"], st["v"], st["table"], st["start"],
                             pos=st["pos"], wq=st["wq"], wk=st["wk"], freqs=st["freqs"], eps=st["eps"],
                             scale=st["scale"], interleaved=st["case"]["inter"])
        return (Qs, *pa.cache_rows(st["ctx"], st["cache"], st["layer"], st["table"], st["start"], st["case"]["tok"]))
    if op == "compact":
        n_keys = pa.cache_compact(st["ctx"], st["cache"], st["table"], st["start"], st["path"], st["count"])
        return st["K"], st["V"], n_keys
    pa.cache_copy_pages(st["ctx"], st["cache"], st["src"], st["dst"])
    return st["K"], st["V"]


def _values(c, rows):
    """uint8 rows [..., row bytes] -> the values they stand for, f16(d * q), as float32 [..., nkv, hd]."""
    b = rows[..., :c["nkv"] * _head_bytes(c)]
    if c["quant"] == F16:
        return b.contiguous().view(torch.float16).unflatten(-1, (c["nkv"], c["hd"])).float()
    b = b.unflatten(-1, (c["nkv"], c["hd"] // 32, -1))
    d = b[..., :2].contiguous().view(torch.float16).float()
    if c["quant"] == Q8_0:
        q = b[..., 2:].contiguous().view(torch.int8).float()
    else:
        q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float() - 8
    return (d * q).to(torch.float16).float().flatten(-2)


def _visible(c, n_keys, bits, N):
    """Truth values [sets, tok, N]: token t's own key is key n_keys - tok + t. It sees the sinks and the last `window`
    keys up to itself (window 0: all of them); in a tree, the keys before the drafted ones (the window measured from its
    depth) and the drafted ones its mask names."""
    T, dev = c["tok"], n_keys.device
    j, t = torch.arange(N, device=dev), torch.arange(T, device=dev)
    q0 = n_keys.long() - T
    if bits is None:
        at = q0[:, None] + t
        last = at
    else:
        named = (bits[:, :, None] >> t) & 1 == 1
        at = q0[:, None] + named.sum(-1) - 1
        last = (q0[:, None] - 1).expand(-1, T)
    see = j <= last[:, :, None]
    if c["window"]:
        see &= (j > (at - c["window"])[:, :, None]) | (j < c["sinks"])
    if bits is not None:
        u = (j - q0[:, None])[:, None, :].expand(-1, T, -1)
        see |= (u >= 0) & (u < T) & named.gather(2, u.clamp(0, T - 1))
        see &= (bits != 0)[:, :, None]
    return see & (j < n_keys[:, None])[:, None, :]


def _plain_attention(st):
    c = st["case"]
    S, T, G, H, hd = c["sets"], c["tok"], c["gqa"], c["nkv"], c["hd"]
    at = st["table"].long().clamp(min=0)
    N = at.shape[1] * c["page"]
    K = _values(c, st["K"][st["layer"]][at].view(S, N, -1)).transpose(1, 2)   # [S, H, N, hd]
    V = _values(c, st["V"][st["layer"]][at].view(S, N, -1)).transpose(1, 2)
    see = _visible(c, st["n_keys"], st["bits"], N)
    live = see.any(1)[:, None, :, None]
    K, V = torch.where(live, K, 0.0), torch.where(live, V, 0.0)   # rows no token sees may hold anything
    s = (st["Qs"].float() @ K.transpose(2, 3)).view(S, H, G, T, N)
    s = torch.where(see[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    l = p.sum(-1, keepdim=True)
    O = (p.view(S, H, G * T, N) @ V).view(S, H, G, T, hd) / torch.where(l > 0, l, 1.0)
    lse = (m + torch.log(l)).view(S, H, G * T)
    return O.view(S, H, G * T, hd).to(torch.float16), lse


def _head_norm(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()


def _rotate(x, cos, sin, rot, inter):
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([r, rest], -1)


def _new_rows(st):
    """Flat row index of every new token, and whether it is one (not padding): [sets, tok]."""
    c = st["case"]
    j = st["start"].long()[:, None] + torch.arange(c["tok"], device="cuda")
    page = st["table"].long().gather(1, j // c["page"])
    return page * c["page"] + j % c["page"], st["pos"] >= 0


def _plain_append(st):
    c = st["case"]
    S, T, G, H, hd, rot = c["sets"], c["tok"], c["gqa"], c["nkv"], c["hd"], c["rot"]
    angle = (st["pos"].double()[..., None] * st["freqs"])[:, :, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotate(_head_norm(st["q"].float(), st["wq"], st["eps"]), cos, sin, rot, c["inter"]) * st["scale"]
    k = _rotate(_head_norm(st["k"].float(), st["wk"], st["eps"]), cos, sin, rot, c["inter"])
    at, real = _new_rows(st)
    q = torch.where(real[:, :, None, None], q, 0.0).to(torch.float16)
    Qs = q.view(S, T, H, G, hd).permute(0, 2, 3, 1, 4).reshape(S, H, G * T, hd)
    used = H * _head_bytes(c)
    out = []
    for pool, x in ((st["K"], k), (st["V"], st["v"].float())):
        rows = pool[st["layer"]].view(-1, _row_bytes(c))
        new = torch.where(real[..., None], _quantise(x, c["quant"]).flatten(-2), rows[at][..., :used])
        rows[at.flatten(), :used] = new.flatten(0, 1)
        out.append(_values(c, rows[at]).to(torch.float16))
    return Qs, out[0], out[1]


def _plain_compact(st):
    c = st["case"]
    T, tok = c["tok"], torch.arange(c["tok"], device="cuda")
    kept = tok < st["count"][:, None]
    src = st["start"].long()[:, None] + torch.where(kept, st["path"].long(), tok)
    dst = st["start"].long()[:, None] + tok
    a, b = (st["table"].long().gather(1, j // c["page"]) * c["page"] + j % c["page"] for j in (src, dst))
    for pool in (st["K"], st["V"]):
        rows = pool.view(c["layers"], -1, _row_bytes(c))
        rows[:, b.flatten()] = rows[:, a.flatten()]
    return st["K"], st["V"], (st["start"] + st["count"]).to(torch.int32)


def _plain_copy(st):
    for pool in (st["K"], st["V"]):
        pool[:, st["dst"].long()] = pool[:, st["src"].long()]
    return st["K"], st["V"]


# ------------------------------------------------------------------------------------------------- what it has to do
def work(case):
    c = case
    rb, G, H, hd = c["nkv"] * _head_bytes(c), c["gqa"], c["nkv"], c["hd"]
    if c["op"] == "copy":
        return {"bytes": 4 * c["layers"] * c["pages"] * c["page"] * _row_bytes(c), "flops": 0}
    S, T, lens = c["sets"], c["tok"], _lens(c)
    if c["op"] == "compact":   # about a quarter of the drafted rows is kept
        return {"bytes": 4 * c["layers"] * S * max(1, T // 4) * _row_bytes(c), "flops": 0}
    if c["op"] == "append":
        size = 4 if c["dtype"] == "float32" else 2
        n = S * T
        # inputs, queries, rows stored; then rows read and their values
        return {"bytes": n * (hd * H * ((G + 2) * size + G * 2) + 2 * rb + 2 * rb + 4 * hd * H), "flops": n * hd * H * (G + 2) * 8}
    keys = pairs = 0
    for n in lens:
        q0 = n - T
        for t in ((0, T - 1) if c["op"] == "tree" else range(T)):
            p = q0 + t if c["op"] == "window" else q0 - 1
            w = p + 1 if not c["window"] else min(p + 1, c["window"] + min(c["sinks"], max(0, p + 1 - c["window"])))
            pairs += max(0, w) * (T // 2 if c["op"] == "tree" and T > 1 else 1)
        first = max(0, q0 - c["window"] + 1) if c["window"] else 0
        keys += n - first + min(c["sinks"] if c["window"] else 0, first)
    return {"bytes": 2 * rb * keys + S * H * G * T * (4 * hd + 4), "flops": 4 * hd * H * G * pairs}


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """What run() returns, from the definitions in 64 bits, sequence by sequence and head by head."""
    c = case
    st = prepare(c, seed)
    if c["op"] in ("compact", "copy"):
        return None
    if c["op"] == "append":
        return _exact_append(c, st)
    if 4 * c["sets"] * c["nkv"] * c["gqa"] * c["tok"] * c["nk"] * c["hd"] > 6e11:
        return None
    S, T, G, H, hd = c["sets"], c["tok"], c["gqa"], c["nkv"], c["hd"]
    O = torch.zeros(S, H, G * T, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((S, H, G * T), -math.inf, dtype=torch.float64, device="cuda")
    for s in range(S):
        n = int(st["n_keys"][s])
        rows = _rows_of(c, s, [n] * S, st["table"])
        kv = []
        for pool in (st["K"], st["V"]):
            raw = pool[st["layer"]].reshape(-1, _row_bytes(c))[rows][:, :H * _head_bytes(c)]
            if c["quant"] == F16:
                kv.append(raw.contiguous().view(torch.float16).double().view(n, H, hd))
                continue
            blk = raw.reshape(n, H * hd // 32, -1)
            d = blk[:, :, :2].contiguous().view(torch.float16).double()
            if c["quant"] == Q8_0:
                e = blk[:, :, 2:].contiguous().view(torch.int8).double()
            else:
                e = torch.cat([blk[:, :, 2:].remainder(16), blk[:, :, 2:].div(16, rounding_mode="floor")], 2).double() - 8.0
            kv.append((d * e).half().double().reshape(n, H, hd))   # the product is exact in 64 bits: rounded once
        # which keys each token sees, token by token, as a list of key indices
        hide = torch.full((T, n), -math.inf, dtype=torch.float64, device="cuda")
        for t in range(T):
            own_key = n - T + t
            if st["bits"] is None:
                lo = max(0, own_key - c["window"] + 1) if c["window"] else 0
                hide[t, lo:max(0, own_key + 1)] = 0
                hide[t, :max(0, min(c["sinks"], own_key + 1))] = 0
            else:
                b = int(st["bits"][s, t]) & (2 ** 64 - 1)
                if b:
                    depth = bin(b).count("1") - 1
                    lo = max(0, n - T + depth - c["window"] + 1) if c["window"] else 0
                    end = max(0, n - T)
                    hide[t, min(lo, end):end] = 0
                    hide[t, :min(c["sinks"], end)] = 0
                    for u in range(T):
                        if b >> u & 1 and n - T + u >= 0:
                            hide[t, n - T + u] = 0
        for h in range(H):
            x = st["Qs"][s, h].double() @ kv[0][:, h].T + hide.repeat(G, 1)
            z = torch.logsumexp(x, 1)
            w = torch.where((z > -math.inf)[:, None], torch.exp(x - z[:, None].clamp(min=-1e300)), 0.0)
            O[s, h], lse[s, h] = w @ kv[1][:, h], z
    return O, lse


def _exact_append(c, st):
    S, T, G, H, hd, rot = c["sets"], c["tok"], c["gqa"], c["nkv"], c["hd"], c["rot"]
    half = rot // 2
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if c["inter"] else (i, i + half)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), st["pos"].double()[:, :, None, None] * st["freqs"])
    done = []
    for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
        y = x.double()
        y = y / (y.pow(2).sum(3, keepdim=True) / hd + st["eps"]).sqrt() * w.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        done.append(y)
    real = (st["pos"] >= 0)[:, :, None, None]
    q = torch.where(real, done[0] * st["scale"], 0.0)
    Qs = torch.empty(S, H, G, T, hd, dtype=torch.float64, device="cuda")
    for g in range(G):
        Qs[:, :, g] = q[:, :, torch.arange(H, device="cuda") * G + g].transpose(1, 2)
    out = [Qs.view(S, H, G * T, hd)]
    for x in (done[1], st["v"].double()):
        if c["quant"] == F16:
            y = x.half().double()
        else:
            b = x.reshape(S, T, H * hd // 32, 32)
            d = (b.abs().amax(3, keepdim=True) / 127).half().double()
            y = ((b / d.clamp(min=1e-30)).round().clamp(-127, 127) * d).half().double().reshape(S, T, H, hd)
        # the rows of padding tokens keep what they held: NaN patterns here
        held = -math.nan if c["quant"] == F16 else math.nan
        out.append(torch.where(real, y, held))
    return tuple(out)
