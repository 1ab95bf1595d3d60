"""Workloads of the prefill-side operators: page bookkeeping (pages), rotary
positions with the cache write (rotary) and attention of a chunk of new
tokens over the paged cache (chunk).

``run`` computes a case either through the package's entry points (``own``)
or in a plain form made of elementary torch operations; ``exact`` gives the
same outputs from the definitions in 64 bits.  Sizes are the serving
geometries of the benchmark: 32 query / 8 kv heads and 64 / 8 at head_dim
128, 8 / 2 at head_dim 64, 16-token pages, contexts up to 64K.
"""
import math
import random

import torch

own = False

PAGE = 16
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # one stream's next token, dense attention over its context: latency
        dict(name="chunk_one_token", op="chunk", dtype="bf16", n_kv=8, G=4,
             d=128, reqs=1, chunks=0, q_lo=1, q_hi=1, ctx_lo=4096,
             ctx_hi=4096, window=0, lse=False, lens=1),
        # a continuous batch: most requests bring one token, some a chunk
        dict(name="chunk_mixed", op="chunk", dtype="bf16", n_kv=8, G=4,
             d=128, reqs=32, chunks=4, q_lo=65, q_hi=512, ctx_lo=4096,
             ctx_hi=65536, window=0, lse=True, lens=2),
        # fresh prompts of odd lengths, nothing cached yet, 64 / 8 heads
        dict(name="chunk_prompts", op="chunk", dtype="bf16", n_kv=8, G=8,
             d=128, reqs=6, chunks=6, q_lo=333, q_hi=2047, ctx_lo=0,
             ctx_hi=0, window=0, lse=False, lens=3),
        # a long prompt's next chunk behind 64K cached tokens
        dict(name="chunk_long", op="chunk", dtype="bf16", n_kv=8, G=4,
             d=128, reqs=1, chunks=1, q_lo=2048, q_hi=2048, ctx_lo=65536,
             ctx_hi=65536, window=0, lse=False, lens=4),
        # the small geometry in fp16 with a sliding window
        dict(name="chunk_window", op="chunk", dtype="fp16", n_kv=2, G=4,
             d=64, reqs=5, chunks=4, q_lo=100, q_hi=1500, ctx_lo=17,
             ctx_hi=9000, window=1024, lse=True, lens=5),
        # the decode batch: one token of each of 64 requests
        dict(name="rotary_decode", op="rotary", dtype="bf16", n_kv=8, G=4,
             d=128, rot=128, layout="half", scaling="llama3", tokens=64,
             pos_hi=65536, pad=0),
        # a prefill step at far positions, extended context
        dict(name="rotary_prefill", op="rotary", dtype="bf16", n_kv=8, G=4,
             d=128, rot=128, layout="half", scaling="yarn", tokens=8192,
             pos_hi=131072, pad=0),
        # half of each head rotated in neighbouring pairs, a padded batch
        dict(name="rotary_part", op="rotary", dtype="fp16", n_kv=2, G=4,
             d=64, rot=32, layout="interleaved", scaling="linear",
             tokens=1777, pos_hi=9000, pad=15),
        # 64 decoding requests grow by a draft of 1..4 tokens, turned down
        dict(name="pages_draft", op="pages", reqs=64, new_lo=1, new_hi=4,
             ctx_lo=4096, ctx_hi=65536, max_pages=4128, spare=256,
             undo="truncate", lens=6),
        # a batch of prompts is admitted and, scored in one step, released
        dict(name="pages_prompts", op="pages", reqs=256, new_lo=1,
             new_hi=300, ctx_lo=0, ctx_hi=0, max_pages=256, spare=3,
             undo="release", lens=7),
        # slots and positions of an engine that keeps its own block table
        dict(name="pages_map", op="pages", reqs=37, new_lo=1, new_hi=777,
             ctx_lo=0, ctx_hi=30000, max_pages=2048, spare=0, undo="map",
             lens=8),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "rotary", "pages"])
    lens = rng.randrange(1 << 30)
    if op == "pages":
        undo = rng.choice(["truncate", "release", "map"])
        fresh = undo == "release"
        reqs = _log(rng, 1, 300)
        return dict(op=op, reqs=reqs,
                    new_lo=rng.choice([0, 1]) if reqs > 64 else 1,
                    new_hi=_log(rng, 1, 300),
                    ctx_lo=0 if fresh else rng.choice([0, 1, 500]),
                    ctx_hi=0 if fresh else _log(rng, 1000, 30000),
                    max_pages=rng.randrange(1920, 2100),
                    spare=rng.randrange(0, 300), undo=undo, lens=lens)
    n_kv, G, d = rng.choice([(8, 4, 128), (8, 8, 128), (2, 4, 64),
                             (1, 8, 128), (4, 1, 64), (2, 3, 128),
                             (1, 6, 64), (4, 2, 128)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rotary":
        rot = rng.choice([d, d, d // 2, 48, 20])
        return dict(op=op, dtype=dtype, n_kv=n_kv, G=G, d=d, rot=rot,
                    layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "llama3",
                                        "yarn"]),
                    tokens=_log(rng, 1, 8192 * 4 // max(4, G * n_kv // 8)),
                    pos_hi=_log(rng, 100, 131072),
                    pad=rng.choice([0, 0, 1, 33]))
    reqs = _log(rng, 1, 24)
    chunks = rng.randint(0, min(reqs, 4))
    return dict(op=op, dtype=dtype, n_kv=n_kv, G=G, d=d, reqs=reqs,
                chunks=chunks, q_lo=2, q_hi=_log(rng, 2, 1200), ctx_lo=0,
                ctx_hi=_log(rng, 16, 16384),
                window=rng.choice([0, 0, 0, 1, 100, 4096]),
                lse=rng.choice([False, True]), lens=lens)


# ----------------------------------------------------------------- lengths --
def _chunk_lengths(case):
    """(new tokens, tokens after the step) of every request."""
    rng = random.Random(case["lens"])
    out = []
    for r in range(case["reqs"]):
        new = rng.randint(case["q_lo"], case["q_hi"]) \
            if r < case["chunks"] else 1
        lo, hi = case["ctx_lo"], case["ctx_hi"]
        old = lo if lo == hi else _log(rng, lo + 1, hi + 1) - 1
        out.append((new, old + new))
    rng.shuffle(out)
    return out


def _pages_lengths(case):
    """(tokens before, new tokens) of every request."""
    rng = random.Random(case["lens"])
    out = []
    for _ in range(case["reqs"]):
        lo, hi = case["ctx_lo"], case["ctx_hi"]
        old = lo if lo == hi else _log(rng, lo + 1, hi + 1) - 1
        out.append((old, rng.randint(case["new_lo"], case["new_hi"])))
    return out


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _scaling(name):
    """The scaling of the frequencies, as a model's configuration gives it."""
    return {"none": None,
            "linear": dict(type="linear", factor=4.0),
            "ntk": dict(type="ntk", factor=4.0),
            "llama3": dict(type="llama3", factor=8.0, low_freq_factor=1.0,
                           high_freq_factor=4.0, original_max_position=8192),
            "yarn": dict(type="yarn", factor=16.0, beta_fast=32.0,
                         beta_slow=1.0, original_max_position=8192),
            }[name]


def _base(case):
    return 500000.0 if case["scaling"] == "llama3" else 10000.0


# ----------------------------------------------------------------- prepare --
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case, dev=dev)
    {"chunk": _prepare_chunk, "rotary": _prepare_rotary,
     "pages": _prepare_pages}[case["op"]](case, s, gen, dev)
    return s


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _prepare_chunk(case, s, gen, dev):
    n_kv, G, d, t = case["n_kv"], case["G"], case["d"], TYPES[case["dtype"]]
    lens = _chunk_lengths(case)
    npg = [_pages(n) for _, n in lens]
    MP, NB = max(npg), sum(npg) + 5
    perm = torch.randperm(NB, generator=gen, device=dev).to(torch.int32)
    bt = torch.zeros((len(lens), MP), dtype=torch.int32, device=dev)
    o = 0
    for r, n in enumerate(npg):
        bt[r, :n] = perm[o:o + n]
        o += n
    kv = torch.randn((NB, 2, PAGE, n_kv, d), generator=gen, device=dev,
                     dtype=torch.float32).to(t)
    # slots behind a request's last token were never written
    for r, (_, n) in enumerate(lens):
        if n % PAGE:
            kv[bt[r, n // PAGE].long(), :, n % PAGE:] = float("nan")
    starts = [0]
    for new, _ in lens:
        starts.append(starts[-1] + new)
    T = starts[-1]
    s.update(q=torch.randn((T, n_kv * G, d), generator=gen, device=dev,
                           dtype=torch.float32).to(t), kv=kv, bt=bt,
             lens=lens, starts=starts, sl=_i32([n for _, n in lens], dev),
             qsl=_i32(starts, dev), scale=d ** -0.5)
    if own:
        from amass_kv_b200.attention import ChunkBuffers
        s["buf"] = ChunkBuffers(dev, n_kv=n_kv, G=G, head_dim=d)
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros((T, n_kv * G), dtype=torch.float32,
                               device=dev) if case["lse"] else None


def _prepare_rotary(case, s, gen, dev):
    n_kv, G, d, t = case["n_kv"], case["G"], case["d"], TYPES[case["dtype"]]
    T, pad = case["tokens"], case["pad"]
    # one fused projection, as a model's attention layer makes it
    H = n_kv * G
    qkv = torch.randn((T + pad, H + 2 * n_kv, d), generator=gen, device=dev,
                      dtype=torch.float32).to(t)
    NB = _pages(T) + 3
    slots = torch.randperm(NB * PAGE, generator=gen, device=dev)[:T + pad]
    slots[T:] = -1
    pos = torch.randint(0, case["pos_hi"], (T + pad,), generator=gen,
                        device=dev)
    s.update(q=qkv[:, :H], k=qkv[:, H:H + n_kv], v=qkv[:, H + n_kv:],
             pos=pos, slots=slots,
             kv=torch.zeros((NB, 2, PAGE, n_kv, d), dtype=t, device=dev),
             q_out=torch.zeros((T + pad, H, d), dtype=t, device=dev))
    if own:
        from amass_kv_b200.rotary import Rotary
        s["rot"] = Rotary(dev, rotary_dim=case["rot"], base=_base(case),
                          layout=case["layout"],
                          scaling=_scaling(case["scaling"]))
    else:
        inv, m = _inv_freq_plain(case["rot"], _base(case),
                                 _scaling(case["scaling"]))
        s["inv"], s["mscale"] = inv.to(dev), m


def _prepare_pages(case, s, gen, dev):
    lens = _pages_lengths(case)
    R, MP = case["reqs"], case["max_pages"]
    old = [o for o, _ in lens]
    new = [n for _, n in lens]
    held = [_pages(o) for o in old]
    if case["undo"] == "map":
        held = [_pages(o + n) for o, n in lens]
    want = sum(_pages(o + n) for o, n in lens)
    NB = max(want, sum(held)) + case["spare"]
    if max(_pages(o + n) for o, n in lens) > MP:
        raise ValueError("a request outgrows its row of the block table")
    perm = torch.randperm(NB, generator=gen, device=dev).to(torch.int32)
    # row r owns the next held[r] blocks, the rest are free
    h = _i32(held, dev).long()
    first = torch.cumsum(h, 0) - h
    col = torch.arange(MP, device=dev)
    owned = col[None] < h[:, None]
    idx = torch.where(owned, first[:, None] + col[None], 0)
    bt = torch.where(owned, perm[idx], -1)
    used = int(sum(held))
    free = torch.full((NB,), -1, dtype=torch.int32, device=dev)
    free[:NB - used] = perm[used:]
    T = sum(new)
    s.update(T=T, NB=NB, new=_i32(new, dev))
    if case["undo"] == "map":
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s.update(bt=bt, sl=_i32([o + n for o, n in lens], dev),
                 qsl=_i32(starts, dev),
                 pos=torch.zeros((T,), dtype=torch.int64, device=dev),
                 slots=torch.zeros((T,), dtype=torch.int64, device=dev))
        return
    s["done"] = torch.ones((R,), dtype=torch.int32, device=dev)
    if own:
        from amass_kv_b200.paging import BlockPool
        p = BlockPool(dev, num_blocks=NB, max_reqs=R, max_pages=MP,
                      max_tokens=max(T, 1), page=PAGE)
        p.block_table.copy_(bt)
        p.seq_lens.copy_(_i32(old, dev))
        p.free_stack.copy_(free)
        p.free_top.fill_(NB - used)
        s["pool"] = p
    else:
        s.update(bt=bt, sl=_i32(old, dev), free=free,
                 top=_i32([NB - used], dev))


# --------------------------------------------------------------------- run --
def run(state):
    op = state["case"]["op"]
    if own:
        return {"chunk": _own_chunk, "rotary": _own_rotary,
                "pages": _own_pages}[op](state)
    return {"chunk": _plain_chunk, "rotary": _plain_rotary,
            "pages": _plain_pages}[op](state)


def _own_chunk(s):
    from amass_kv_b200.attention import paged_chunk_attention
    paged_chunk_attention(s["q"], s["kv"], s["bt"], s["sl"], s["qsl"],
                          s["out"], s["buf"], scale=s["scale"],
                          window=s["case"]["window"] or None, lse=s["lse"])
    return [s["out"]] if s["lse"] is None else [s["out"], s["lse"]]


def _own_rotary(s):
    from amass_kv_b200.rotary import rotary_write_kv
    rotary_write_kv(s["rot"], s["q"], s["k"], s["v"], s["pos"], s["kv"],
                    s["slots"], q_out=s["q_out"])
    return [s["q_out"], s["kv"]]


def _own_pages(s):
    if s["case"]["undo"] == "map":
        from amass_kv_b200.paging import build_slot_map
        build_slot_map(s["bt"], s["sl"], s["qsl"], s["pos"], s["slots"],
                       page=PAGE)
        return [s["pos"], s["slots"]]
    p, T = s["pool"], s["T"]
    p.begin_step(s["new"], n_tokens=T)
    if s["case"]["undo"] == "truncate":
        p.truncate(s["new"])
    else:
        p.release(s["done"])
    return [p.query_start_loc, p.positions[:T], p.slot_mapping[:T], p.status,
            p.seq_lens, p.block_table, p.free_stack, p.free_top]


# ------------------------------------------------------------- plain forms --
def _plain_chunk(s):
    """Per request and kv head: scores, mask, softmax, product, in fp32."""
    case, q = s["case"], s["q"]
    n_kv, G, d, w = case["n_kv"], case["G"], case["d"], case["window"]
    T, H, _ = q.shape
    out = torch.zeros((T, H, d), dtype=q.dtype, device=q.device)
    lse = torch.zeros((T, H), dtype=torch.float32, device=q.device)
    for r, (new, n) in enumerate(s["lens"]):
        blocks = s["bt"][r, :_pages(n)].long()
        k = s["kv"][blocks, 0].reshape(-1, n_kv, d)[:n]
        v = s["kv"][blocks, 1].reshape(-1, n_kv, d)[:n]
        t0 = s["starts"][r]
        p = torch.arange(n - new, n, device=q.device)
        j = torch.arange(n, device=q.device)
        hide = j[None] > p[:, None]
        if w:
            hide = hide | (j[None] <= p[:, None] - w)
        for h in range(n_kv):
            qh = q[t0:t0 + new, h * G:(h + 1) * G].float()
            sc = torch.matmul(qh.transpose(0, 1), k[:, h].float().t())
            sc = (sc * s["scale"]).masked_fill(hide[None], float("-inf"))
            m = sc.amax(-1, keepdim=True)
            e = torch.exp(sc - m)
            z = e.sum(-1, keepdim=True)
            o = torch.matmul(e, v[:, h].float()) / z
            out[t0:t0 + new, h * G:(h + 1) * G] = o.transpose(0, 1).to(q.dtype)
            lse[t0:t0 + new, h * G:(h + 1) * G] = \
                (m + torch.log(z)).squeeze(-1).t()
    return [out, lse] if case["lse"] else [out]


def _inv_freq_plain(rot, base, sc):
    """Frequencies (rot / 2,) in fp64 and the factor on cos and sin."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    if sc is None:
        return base ** (-i / rot), 1.0
    f, kind = sc["factor"], sc["type"]
    if kind == "linear":
        return base ** (-i / rot) / f, 1.0
    if kind == "ntk":
        return (base * f ** (rot / (rot - 2))) ** (-i / rot), 1.0
    inv = base ** (-i / rot)
    orig = sc["original_max_position"]
    if kind == "llama3":
        turns = orig * inv / (2 * math.pi)
        lo, hi = sc["low_freq_factor"], sc["high_freq_factor"]
        keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
        return keep * inv + (1 - keep) * inv / f, 1.0
    dim = [rot * math.log(orig / (b * 2 * math.pi)) / (2 * math.log(base))
           for b in (sc["beta_fast"], sc["beta_slow"])]
    lo, hi = max(math.floor(dim[0]), 0), min(math.ceil(dim[1]), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo)
            / max(hi - lo, 1e-3)).clamp(0, 1)
    return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0


def _turn_plain(x, c, sn, rot, layout):
    y = x.float()
    if layout == "half":
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        z = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        z = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    return torch.cat([z, y[..., rot:]], -1).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    T, rot, lay = case["tokens"], case["rot"], case["layout"]
    # a position of 1e5 at the highest frequency leaves fp32 two digits of
    # the angle: the angle is formed in 64 bits
    a = s["pos"].double()[:, None] * s["inv"][None]
    c = (torch.cos(a) * s["mscale"]).float()[:, None]
    sn = (torch.sin(a) * s["mscale"]).float()[:, None]
    q = _turn_plain(s["q"], c, sn, rot, lay)
    k = _turn_plain(s["k"], c, sn, rot, lay)
    slots = s["slots"][:T]
    s["kv"][slots // PAGE, 0, slots % PAGE] = k[:T]
    s["kv"][slots // PAGE, 1, slots % PAGE] = s["v"][:T]
    return [q, s["kv"]]


def _plain_pages(s):
    case, new, sl, dev = s["case"], s["new"].long(), s["sl"].long(), s["dev"]
    T = s["T"]
    t = torch.arange(T, device=dev)
    if case["undo"] == "map":
        qsl = s["qsl"].long()
        r = torch.searchsorted(qsl, t, right=True) - 1
        pos = sl[r] - (qsl[r + 1] - t)
        slots = s["bt"][r, pos // PAGE].long() * PAGE + pos % PAGE
        return [pos, slots]
    R, MP, top = case["reqs"], case["max_pages"], s["top"].long()
    old, end = sl, sl + new
    have, pages = (old + PAGE - 1) // PAGE, (end + PAGE - 1) // PAGE
    too_long = pages > MP
    need = torch.where(too_long, 0, pages - have)
    upto = torch.cumsum(need, 0)
    short = (need > 0) & (upto > top)
    status = torch.where(too_long, 2, torch.where(short, 1, 0))
    ok = status == 0
    qsl = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev),
                     torch.cumsum(new, 0)])
    # the new blocks of row r, popped from the top of the free stack
    col = torch.arange(MP, device=dev)
    k = (upto - need)[:, None] + col[None] - have[:, None]
    fresh = (col[None] >= have[:, None]) & (col[None] < pages[:, None]) \
        & ok[:, None]
    pick = torch.where(fresh, top - 1 - k, 0)
    bt = torch.where(fresh, s["free"][pick], s["bt"])
    r = torch.searchsorted(qsl, t, right=True) - 1
    pos = old[r] + t - qsl[r]
    slots = torch.where(ok[r], bt[r, (pos // PAGE).clamp(max=MP - 1)].long()
                        * PAGE + pos % PAGE, -1)
    top = top - torch.where(ok, need, 0).sum()
    # undo: pages of the dropped tokens go back, last request first
    now = torch.where(ok, end, old)
    drop = new if case["undo"] == "truncate" else now
    left = now - torch.minimum(drop, now)
    have, keep = (now + PAGE - 1) // PAGE, (left + PAGE - 1) // PAGE
    freed = have - keep
    after = freed.sum() - torch.cumsum(freed, 0)
    gone = (col[None] >= keep[:, None]) & (col[None] < have[:, None])
    at = top + after[:, None] + have[:, None] - 1 - col[None]
    free = torch.cat([s["free"], s["free"][:1]])       # one place to spare
    free[torch.where(gone, at, s["NB"])] = bt
    free = free[:-1]
    bt = torch.where(gone, -1, bt)
    i32 = torch.int32
    return [qsl.to(i32), pos, slots, status.to(i32), left.to(i32), bt, free,
            (top + freed.sum()).to(i32)]


# ---------------------------------------------------------------- one pass --
def work(case):
    if case["op"] == "chunk":
        n_kv, G, d, w = case["n_kv"], case["G"], case["d"], case["window"]
        pairs = rows = seen = pages = 0
        for new, n in _chunk_lengths(case):
            old = n - new
            if w:
                pairs += sum(min(p + 1, w) for p in range(old, n))
                seen += n - max(0, old - w + 1)
            else:
                pairs += new * old + new * (new + 1) // 2
                seen += n
            rows += new
            pages += _pages(n)
        return {"bytes": rows * n_kv * G * (4 * d + (4 if case["lse"] else 0))
                + seen * n_kv * d * 4 + 4 * pages + 12 * case["reqs"],
                "flops": 4 * d * n_kv * G * pairs}
    if case["op"] == "rotary":
        n_kv, G, d, T = case["n_kv"], case["G"], case["d"], case["tokens"]
        n = T + case["pad"]
        return {"bytes": (n * n_kv * G + 2 * T * n_kv) * d * 4 + 16 * n,
                "flops": 3 * n * n_kv * (G + 1) * case["rot"]}
    lens = _pages_lengths(case)
    T, R = sum(n for _, n in lens), case["reqs"]
    if case["undo"] == "map":
        pages = sum(_pages(o + n) - o // PAGE for o, n in lens if n)
        return {"bytes": 16 * T + 4 * pages + 8 * R, "flops": 0}
    grown = sum(_pages(o + n) - _pages(o) for o, n in lens)
    return {"bytes": 16 * T + 28 * R + 16 * grown, "flops": 0}


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    if case["op"] == "pages":
        return None                      # whole numbers throughout
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return (_exact_chunk if case["op"] == "chunk" else _exact_rotary)(case, s)


def _exact_chunk(case, s):
    """Row blocks of all heads at once; weights exp(score - lse)."""
    n_kv, G, d, w = case["n_kv"], case["G"], case["d"], case["window"]
    T = s["q"].shape[0]
    out = torch.zeros((T, n_kv, G, d), dtype=torch.float64, device=s["dev"])
    lse = torch.zeros((T, n_kv, G), dtype=torch.float64, device=s["dev"])
    q = s["q"].view(T, n_kv, G, d).double()
    for r, (new, n) in enumerate(s["lens"]):
        tok = torch.arange(n, device=s["dev"])
        where = s["bt"][r].long()[tok // PAGE] * PAGE + tok % PAGE
        keys = s["kv"][:, 0].reshape(-1, n_kv, d)[where].double()
        vals = s["kv"][:, 1].reshape(-1, n_kv, d)[where].double()
        step = max(1, (1 << 28) // (n * n_kv * G))
        for i in range(0, new, step):
            a = s["starts"][r] + i
            b = s["starts"][r] + min(new, i + step)
            p = torch.arange(n - new + i, n - new + i + b - a,
                             device=s["dev"])
            sees = (tok[None] <= p[:, None])
            if w:
                sees = sees & (tok[None] > p[:, None] - w)
            x = torch.einsum("thgd,jhd->thgj", q[a:b], keys) * s["scale"]
            x = torch.where(sees[:, None, None], x, float("-inf"))
            z = torch.logsumexp(x, -1)
            out[a:b] = torch.einsum("thgj,jhd->thgd",
                                    torch.exp(x - z[..., None]), vals)
            lse[a:b] = z
    out, lse = out.view(T, -1, d), lse.view(T, -1)
    return [out, lse] if case["lse"] else [out]


def _exact_freq(i, rot, base, sc):
    """Frequency of pair i, one number at a time."""
    f = math.exp(-2.0 * i / rot * math.log(base))
    if sc is None:
        return f
    s = sc["factor"]
    if sc["type"] == "linear":
        return f / s
    if sc["type"] == "ntk":
        return f * math.exp(-2.0 * i / (rot - 2) * math.log(s))
    wave, orig = 2.0 * math.pi / f, sc["original_max_position"]
    if sc["type"] == "llama3":
        if wave < orig / sc["high_freq_factor"]:
            return f
        if wave > orig / sc["low_freq_factor"]:
            return f / s
        t = (orig / wave - sc["low_freq_factor"]) / \
            (sc["high_freq_factor"] - sc["low_freq_factor"])
        return (1.0 - t) * f / s + t * f

    def at(turns):
        return rot / 2.0 * math.log(orig / (2.0 * math.pi * turns)) / \
            math.log(base)
    lo = max(0, math.floor(at(sc["beta_fast"])))
    hi = min(rot - 1, math.ceil(at(sc["beta_slow"])))
    t = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
    return f * (1.0 - t + t / s)


def _exact_rotary(case, s):
    """Each pair as a complex number times m * exp(i angle)."""
    rot, T = case["rot"], case["tokens"]
    sc = _scaling(case["scaling"])
    f = torch.tensor([_exact_freq(i, rot, _base(case), sc)
                      for i in range(rot // 2)], dtype=torch.float64,
                     device=s["dev"])
    m = 0.1 * math.log(sc["factor"]) + 1.0 if case["scaling"] == "yarn" \
        else 1.0
    ang = s["pos"].double()[:, None, None] * f
    z = torch.polar(torch.full_like(ang, m), ang)

    def turn(x):
        y = x.double().clone()
        if case["layout"] == "half":
            u = torch.complex(y[..., :rot // 2].contiguous(),
                              y[..., rot // 2:rot].contiguous()) * z
            y[..., :rot // 2], y[..., rot // 2:rot] = u.real, u.imag
        else:
            u = torch.complex(y[..., 0:rot:2].contiguous(),
                              y[..., 1:rot:2].contiguous()) * z
            y[..., 0:rot:2], y[..., 1:rot:2] = u.real, u.imag
        return y

    kv = s["kv"].double()
    at = s["slots"][:T]
    kv.view(-1, 2 * PAGE, *kv.shape[3:])[at // PAGE, at % PAGE] = \
        turn(s["k"])[:T]
    kv.view(-1, 2 * PAGE, *kv.shape[3:])[at // PAGE, PAGE + at % PAGE] = \
        s["v"].double()[:T]
    return [turn(s["q"]), kv]
