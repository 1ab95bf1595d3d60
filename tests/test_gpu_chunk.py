"""Attention of a chunk of new tokens over the paged cache against fp64."""
import pytest
import torch

from amass_kv_b200.attention import ChunkBuffers, paged_chunk_attention
from tests.chunk_ref import chunk_reference

pytestmark = pytest.mark.gpu
PAGE = 16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def make(dev, lens, *, n_kv=2, G=4, d=128, dtype=torch.bfloat16, seed=0,
         layout=0, lead=0, tail=3, kmul=1.0):
    """A batch with random block ids, NaN behind each request's last token,
    nonsense ids behind its last page, `lead` / `tail` rows of nobody."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    npg = [-(-n // PAGE) for _, n in lens]
    MP, NB = max(npg) + 2, sum(npg) + 3
    perm = torch.randperm(NB, generator=gen, device=dev).to(torch.int32)
    bt = torch.full((len(lens), MP), 2 ** 31 - 1, dtype=torch.int32,
                    device=dev)
    bt[:, -1] = -7
    o = 0
    for r, n in enumerate(npg):
        bt[r, :n] = perm[o:o + n]
        o += n
    shape = (NB, 2, PAGE, n_kv, d) if layout == 0 else (2, NB, PAGE, n_kv, d)
    kv = torch.randn(shape, generator=gen, device=dev)
    k, v = (kv[:, 0], kv[:, 1]) if layout == 0 else (kv[0], kv[1])
    k *= kmul
    for r, (_, n) in enumerate(lens):
        if n % PAGE:
            k[bt[r, n // PAGE].long(), n % PAGE:] = float("nan")
            v[bt[r, n // PAGE].long(), n % PAGE:] = float("inf")
    kv = kv.to(dtype)
    starts = [lead]
    for new, _ in lens:
        starts.append(starts[-1] + new)
    T = starts[-1] + tail
    q = torch.randn((T, n_kv * G, d), generator=gen, device=dev).to(dtype)
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(q=q, kv=kv, bt=bt, lens=lens, starts=starts,
                sl=torch.tensor([n for _, n in lens], **i32),
                qsl=torch.tensor(starts, **i32), n_kv=n_kv, G=G, d=d,
                layout=layout)


def check(c, dev, *, window=None, scale=None, buf=None, q=None, out=None):
    q = c["q"] if q is None else q
    buf = buf or ChunkBuffers(dev, n_kv=c["n_kv"], G=c["G"], head_dim=c["d"])
    out = torch.full_like(q, 7.0) if out is None else out
    out.fill_(7.0)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device=dev)
    scale = c["d"] ** -0.5 if scale is None else scale
    paged_chunk_attention(q, c["kv"], c["bt"], c["sl"], c["qsl"], out, buf,
                          scale=scale, window=window, lse=lse)
    buf.check()
    k, v = (c["kv"][:, 0], c["kv"][:, 1]) if c["layout"] == 0 else \
        (c["kv"][0], c["kv"][1])
    ref, tol, lref, tol_l, rows = chunk_reference(
        q, k, v, c["bt"], c["lens"], c["starts"], scale, window)
    assert (out[~rows] == 7.0).all() and (lse[~rows] == 7.0).all()
    err = (out.double() - ref).abs()[rows]
    assert bool((err <= tol[rows]).all()), \
        (float(err.max()), float((err / tol[rows]).max()))
    some = torch.isfinite(lref) & rows[:, None]
    assert bool((lse[rows[:, None] & ~some] == float("-inf")).all())
    le = (lse.double() - lref).abs()[some]
    assert bool((le <= tol_l[some]).all()), float(le.max())
    return out, lse


GEOMS = [(torch.bfloat16, 128, 2, 4), (torch.float16, 64, 2, 4),
         (torch.bfloat16, 128, 1, 8), (torch.float16, 128, 3, 1),
         (torch.bfloat16, 64, 2, 2), (torch.bfloat16, 128, 2, 3),
         (torch.float16, 64, 1, 5), (torch.bfloat16, 64, 1, 7)]


@pytest.mark.parametrize("dtype,d,n_kv,G", GEOMS)
def test_one_token(dev, dtype, d, n_kv, G):
    check(make(dev, [(1, 1)], dtype=dtype, d=d, n_kv=n_kv, G=G), dev)
    check(make(dev, [(1, 129)], dtype=dtype, d=d, n_kv=n_kv, G=G), dev)


@pytest.mark.parametrize("dtype,d,n_kv,G", GEOMS)
@pytest.mark.parametrize("lens", [
    [(1, 700), (1, 16), (1, 17), (1, 1), (1, 2000)],
    [(128, 128), (129, 129), (5, 400), (300, 301)],
    [(255, 1024), (1, 3), (33, 33), (64, 6000)]])
def test_mixed_lengths(dev, dtype, d, n_kv, G, lens):
    check(make(dev, lens, dtype=dtype, d=d, n_kv=n_kv, G=G, lead=2), dev)


@pytest.mark.parametrize("window", [1, 2, 16, 127, 128, 129, 1000])
@pytest.mark.parametrize("d", [64, 128])
def test_window(dev, window, d):
    check(make(dev, [(200, 777), (1, 1300), (40, 40), (130, 131)], d=d), dev,
          window=window)


@pytest.mark.parametrize("window,dtype,d,G", [
    (5, torch.bfloat16, 128, 4), (40, torch.float16, 64, 4),
    (129, torch.bfloat16, 64, 1), (300, torch.bfloat16, 128, 8)])
def test_before_the_window(dev, window, dtype, d, G):
    """Slots before every row's window hold anything (an engine has given
    their pages away): nothing of it reaches a row."""
    lens = [(1, 1000), (1, 17), (70, 900), (300, 1333), (3, 128), (1, 645),
            (33, 33), (2, 2500)]
    c = make(dev, lens, n_kv=2, G=G, d=d, dtype=dtype, seed=11)
    clean, lse = check(c, dev, window=window)
    for r, (new, n) in enumerate(lens):
        first = max(n - new - window + 1, 0)
        pos = torch.arange(first, device=dev)
        blk = c["bt"][r, pos // PAGE].long()
        c["kv"][blk, 0, pos % PAGE] = float("nan")
        c["kv"][blk, 1, pos % PAGE] = float("inf")
        if r % 2:                            # pages of nobody
            c["bt"][r, :first // PAGE] = -1
    buf = ChunkBuffers(dev, n_kv=2, G=G, head_dim=d)
    out, got = torch.full_like(clean, 7.0), torch.full_like(lse, 7.0)
    paged_chunk_attention(c["q"], c["kv"], c["bt"], c["sl"], c["qsl"], out,
                          buf, window=window, lse=got)
    buf.check()
    assert torch.equal(out, clean) and torch.equal(got, lse)


def test_empty_rows_and_requests(dev):
    """Requests without new tokens, with none at all, and with fewer tokens
    than rows (their first rows see nothing: 0 and -inf)."""
    lens = [(0, 50), (3, 0), (40, 9), (0, 0), (70, 70), (200, 1), (1, 1)]
    for w in (None, 4):
        check(make(dev, lens), dev, window=w)
    c = make(dev, [(0, 0)])
    out, _ = check(c, dev)
    assert bool((out == 7.0).all())


def test_windows_beyond_any_length(dev):
    """A window as long as the types hold is none, for rows before position 0
    too."""
    c = make(dev, [(40, 200), (9, 4), (1, 300), (5, 0)])
    want = check(c, dev)
    for window in (2 ** 30, 2 ** 31 - 1, 2 ** 40):
        got = check(c, dev, window=window)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_strides_and_layouts(dev):
    """q out of a fused projection, out into a wider row, both cache layouts,
    a block table with wider rows."""
    for layout in (0, 1):
        c = make(dev, [(70, 300), (1, 90)], layout=layout)
        T, H, d = c["q"].shape
        fused = torch.randn((T, H + 4, d), device=dev).to(torch.bfloat16)
        wide = torch.full((T, H + 1, d), 3.0, device=dev,
                          dtype=torch.bfloat16)
        bt = torch.full((2, c["bt"].shape[1] + 5), -1, dtype=torch.int32,
                        device=dev)
        bt[:, :c["bt"].shape[1]] = c["bt"]
        c["bt"] = bt[:, :c["bt"].shape[1]]
        check(c, dev, q=fused[:, 2:2 + H], out=wide[:, :H])
        assert bool((wide[:, H] == 3.0).all())


def test_one_row_of_any_stride(dev):
    """A single token's strides are not used, whatever they are."""
    c = make(dev, [(1, 77)], tail=0)
    q, out = (torch.zeros(1, 8 * 128 + 4, device=dev, dtype=torch.bfloat16)
              [:, :8 * 128].view(1, 8, 128) for _ in range(2))
    check(c, dev, q=q.copy_(c["q"]), out=out)


def test_heads_before_tokens(dev):
    """A cache stored (blocks, 2, heads, page, d), seen as (.., page, heads,
    d), and q in place."""
    c = make(dev, [(70, 300), (1, 90), (33, 33)])
    c["kv"] = c["kv"].permute(0, 1, 3, 2, 4).contiguous().permute(
        0, 1, 3, 2, 4)
    a, _ = check(c, dev)
    buf = ChunkBuffers(dev, n_kv=2, G=4, head_dim=128)
    q = c["q"].clone()
    paged_chunk_attention(q, c["kv"], c["bt"], c["sl"], c["qsl"], q, buf)
    n = c["starts"][-1]
    assert torch.equal(q[:n], a[:n]) and torch.equal(q[n:], c["q"][n:])


def test_padded_cache(dev):
    """Blocks and heads further apart than their contents."""
    c = make(dev, [(40, 200), (5, 5)], d=64)
    NB = c["kv"].shape[0]
    big = torch.full((NB + 1, 2, PAGE, 4, 64), float("nan"), device=dev,
                     dtype=torch.bfloat16)
    big[:NB, :, :, :2] = c["kv"]
    c["kv"] = big[:NB, :, :, :2]
    check(c, dev)


def test_nan_and_infinite_keys(dev):
    """A NaN or infinite key in reach: the rows that see it are NaN, all
    others what they are without it."""
    for bad in (float("nan"), float("inf")):
        c = make(dev, [(60, 300), (1, 200)], seed=4)
        clean, lse = check(c, dev)
        p = 270                              # seen by rows 30 .. 59
        c["kv"][c["bt"][0, p // PAGE].long(), 0, p % PAGE, 1] = bad
        buf = ChunkBuffers(dev, n_kv=2, G=4, head_dim=128)
        out, got = torch.zeros_like(clean), torch.zeros_like(lse)
        paged_chunk_attention(c["q"], c["kv"], c["bt"], c["sl"], c["qsl"],
                              out, buf, lse=got)
        n = c["starts"][-1]
        same = torch.ones(n, 8, dtype=torch.bool, device=dev)
        if bad != bad:
            same[30:60, 4:] = False
            assert bool(torch.isnan(out[30:60, 4:]).all())
            assert bool(torch.isnan(got[30:60, 4:]).all())
        else:                                # q k is NaN, +inf or -inf
            same[30:60, 4:] = ~torch.isnan(got[30:60, 4:])
        assert torch.equal(out[:n][same], clean[:n][same]) or bad == bad
        assert torch.equal(got[:n, :4], lse[:n, :4])
        assert torch.equal(out[:30], clean[:30])
        assert torch.equal(out[60:n], clean[60:n])


def test_two_streams(dev):
    """Two streams at once, each with buffers of its own."""
    cs = [make(dev, [(50, 3000), (1, 9000)], seed=s) for s in (1, 2)]
    want = [check(c, dev)[0] for c in cs]
    bufs = [ChunkBuffers(dev, n_kv=2, G=4, head_dim=128) for _ in cs]
    outs = [torch.full_like(c["q"], 7.0) for c in cs]
    streams = [torch.cuda.Stream(dev) for _ in cs]
    torch.cuda.synchronize(dev)
    for _ in range(5):
        for c, b, o, s in zip(cs, bufs, outs, streams):
            with torch.cuda.stream(s):
                paged_chunk_attention(c["q"], c["kv"], c["bt"], c["sl"],
                                      c["qsl"], o, b)
    torch.cuda.synchronize(dev)
    for b, o, w in zip(bufs, outs, want):
        b.check()
        assert torch.equal(o, w)


def test_large_scores(dev):
    """Scores of hundreds: every tile moves the maximum, the rescale path and
    weights far below 1."""
    check(make(dev, [(100, 1500), (1, 3000)], kmul=12.0, seed=3), dev,
          scale=1.0)


def test_batch_of_many(dev):
    lens = [(1, 1 + (37 * i) % 500) for i in range(700)]
    check(make(dev, lens, n_kv=1, G=4, d=64), dev)


@pytest.mark.parametrize("window", [None, 70])
def test_many_items_of_a_request(dev, window):
    """Runs that start deep inside a request: more items than a warp has
    lanes, with one item a CTA and with several."""
    for G, new, more in ((8, 2600, 0), (8, 1100, 900), (1, 9000, 0)):
        c = make(dev, [(new, new + more), (40, 60)], n_kv=1, G=G, d=64)
        check(c, dev, window=window)


def test_long_context_few_rows(dev):
    """One item over all SMs: its partials come from every CTA."""
    check(make(dev, [(2, 40000)], n_kv=1, G=8), dev)
    check(make(dev, [(17, 20011)], n_kv=2, G=1, d=64), dev)


def test_repeatable(dev):
    """Same call, same bits; buffers hold the last call's partials."""
    c = make(dev, [(33, 5000), (1, 8000)])
    buf = ChunkBuffers(dev, n_kv=2, G=4, head_dim=128)
    a = check(c, dev, buf=buf)
    check(make(dev, [(300, 700)], seed=9), dev, buf=buf)
    b = check(c, dev, buf=buf)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_and_other_stream(dev):
    """A graph on a side stream, replayed with other lengths and an eager
    call with its own buffers in between."""
    c = make(dev, [(33, 500), (1, 800)])
    buf = ChunkBuffers(dev, n_kv=2, G=4, head_dim=128)
    out = torch.zeros_like(c["q"])
    args = (c["q"], c["kv"], c["bt"], c["sl"], c["qsl"], out, buf)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        paged_chunk_attention(*args)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        paged_chunk_attention(*args)
    c["sl"].copy_(torch.tensor([450, 640], dtype=torch.int32))
    c["lens"] = [(33, 450), (1, 640)]
    want, _ = check(c, dev)
    out.fill_(7.0)
    torch.cuda.synchronize(dev)
    g.replay()
    torch.cuda.synchronize(dev)
    assert torch.equal(out, want)
