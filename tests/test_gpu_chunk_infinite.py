"""Infinite keys in reach: a score of +inf makes the row NaN, one of -inf drops
the key, and no other row or head changes."""
import pytest
import torch

from amass_kv_b200.attention import ChunkBuffers, paged_chunk_attention
from tests.chunk_ref import chunk_reference
from tests.test_gpu_chunk import PAGE, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
@pytest.mark.parametrize("new,n,p", [(60, 300, 270), (1, 300, 100),
                                     (200, 900, 5), (3, 128, 126)])
def test_one_element_of_a_key(dev, bad, new, n, p):
    """One element of one key of the second kv head: the sign of the query's
    element there decides."""
    c = make(dev, [(new, n), (40, 200)], seed=4)
    clean, lse = check(c, dev)
    e, first = 17, max(p - (n - new), 0)     # rows from `first` on see it
    c["kv"][c["bt"][0, p // PAGE].long(), 0, p % PAGE, 1, e] = bad
    buf = ChunkBuffers(dev, n_kv=2, G=4, head_dim=128)
    out, got = torch.full_like(clean, 7.0), torch.full_like(lse, 7.0)
    paged_chunk_attention(c["q"], c["kv"], c["bt"], c["sl"], c["qsl"], out,
                          buf, lse=got)
    buf.check()
    up = torch.zeros_like(lse, dtype=torch.bool)
    down = torch.zeros_like(up)
    up[first:new, 4:] = c["q"][first:new, 4:, e] * bad > 0
    down[first:new, 4:] = c["q"][first:new, 4:, e] * bad < 0
    assert bool(up.any()) and bool(down.any())
    assert bool(torch.isnan(out[up]).all()) and bool(
        torch.isnan(got[up]).all())
    rest = ~(up | down)
    assert torch.equal(out[rest], clean[rest])
    assert torch.equal(got[rest], lse[rest])
    # the other rows: the same request without that key
    tok = torch.arange(n, device=dev)
    tok = tok[tok != p]
    kv = c["kv"][c["bt"][0, tok // PAGE].long(), :, tok % PAGE]
    flat = torch.zeros((-(-n // PAGE) * PAGE, 2, 2, 128), device=dev,
                       dtype=kv.dtype)
    flat[:n - 1] = kv
    k, v = (x.reshape(-1, PAGE, 2, 128) for x in (flat[:, 0], flat[:, 1]))
    bt = torch.arange(k.shape[0], device=dev)[None]
    ref, tol, lref, tol_l, _ = chunk_reference(
        c["q"][first:new], k, v, bt, [(new - first, n - 1)], [0],
        128 ** -0.5)
    at = down[first:new]
    err = (out[first:new].double() - ref).abs()
    assert bool((err <= tol)[at].all())
    assert bool(((got[first:new].double() - lref).abs() <= tol_l)[at].all())
