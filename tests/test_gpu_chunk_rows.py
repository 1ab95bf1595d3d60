"""Chunk attention where a step's rows, start offsets and lengths do not go
together one to one."""
import pytest
import torch

from amass_kv_b200.attention import ChunkBuffers, paged_chunk_attention
from tests.chunk_ref import chunk_reference
from tests.test_gpu_chunk import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


@pytest.mark.parametrize("T,window", [(75, None), (75, 20), (71, None),
                                      (70, None), (30, 50), (1, None)])
def test_requests_cut_by_the_rows(dev, T, window):
    """q holds the first T of the step's 110 tokens (an n_tokens that was too
    small): its rows keep their positions, nothing need ever have been written
    for the tokens that are not there, and a request without a row does
    nothing."""
    c = make(dev, [(70, 300), (33, 60), (7, 7)], tail=0, seed=5)
    lens = []
    for r, (new, n) in enumerate(c["lens"]):
        gone = min(max(c["starts"][r + 1] - T, 0), new)
        at = torch.arange(n - gone, n, device=dev)
        c["kv"][c["bt"][r, at // 16].long(), :, at % 16] = float("nan")
        lens.append((new - gone, n - gone))
    q = c["q"][:T].contiguous()
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device=dev)
    buf = ChunkBuffers(dev, n_kv=2, G=4, head_dim=128)
    paged_chunk_attention(q, c["kv"], c["bt"], c["sl"], c["qsl"], out, buf,
                          lse=lse, window=window)
    buf.check()
    ref, tol, lref, tol_l, _ = chunk_reference(
        q, c["kv"][:, 0], c["kv"][:, 1], c["bt"], lens, c["starts"],
        128 ** -0.5, window)
    assert bool(((out.double() - ref).abs() <= tol).all())
    assert bool(((lse.double() - lref).abs() <= tol_l).all())
