"""Chunk attention with keys from a K-only cache and values from a tensor of
their own."""
import pytest
import torch

from amass_kv_b200.attention import ChunkBuffers, paged_chunk_attention
from tests.test_gpu_chunk import PAGE, check, make

pytestmark = pytest.mark.gpu


class Source:
    def __init__(self, v):
        self.v = v

    def args(self):
        return (self.v, *self.v.stride()[:3])


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


@pytest.mark.parametrize("dtype,n_kv,G,d,window", [
    (torch.bfloat16, 2, 4, 128, None), (torch.float16, 3, 2, 64, 90),
    (torch.bfloat16, 1, 8, 128, None)])
@pytest.mark.parametrize("wide", [0, 64])
def test_values_apart(dev, dtype, n_kv, G, d, window, wide):
    """The same bits as with both halves in one cache, whatever the values'
    own strides and whatever V half the cache has."""
    lens = [(70, 300), (1, 900), (33, 33), (3, 1), (0, 20)]
    c = make(dev, lens, n_kv=n_kv, G=G, d=d, dtype=dtype, seed=2)
    want, lse = check(c, dev, window=window)
    NB = c["kv"].shape[0]
    raw = torch.full((NB, PAGE, n_kv, d + wide), float("nan"), device=dev,
                     dtype=dtype)
    v = raw[..., :d]
    v.copy_(c["kv"][:, 1])
    konly = c["kv"][:, :1].contiguous()
    both = torch.stack([c["kv"][:, 0], torch.full_like(v, float("nan"))])
    buf = ChunkBuffers(dev, n_kv=n_kv, G=G, head_dim=d)
    for cache in (konly, both):
        out, got = torch.full_like(want, 7.0), torch.full_like(lse, 7.0)
        paged_chunk_attention(c["q"], cache, c["bt"], c["sl"], c["qsl"], out,
                              buf, window=window, lse=got,
                              vsource=Source(v))
        buf.check()
        assert torch.equal(out, want) and torch.equal(got, lse)


def test_refused_values(dev):
    """Other shapes, types and block strides than the keys'."""
    c = make(dev, [(5, 40)])
    konly, v = c["kv"][:, :1].contiguous(), c["kv"][:, 1].contiguous()
    buf = ChunkBuffers(dev, n_kv=2, G=4, head_dim=128)
    for bad, match in ((v[:-1], "does not match K"),
                       (v.half(), "does not match K"),
                       (v.cpu(), "does not match K"),
                       (c["kv"][:, 1], "block strides")):
        with pytest.raises(ValueError, match=match):
            paged_chunk_attention(c["q"], konly, c["bt"], c["sl"], c["qsl"],
                                  torch.zeros_like(c["q"]), buf,
                                  vsource=Source(bad))
