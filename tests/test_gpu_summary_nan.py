"""Page summaries of pages that hold keys nobody has written yet (NaN): the
builders pad their block lists with a request's first page, complete or not.
The other pages' summaries stay what they are without such pages."""
import pytest
import torch

from amass_kv_b200 import selection as S
from amass_kv_b200 import summaries as SM

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,rank,v_bits", [(128, 2, 4), (64, 8, 8),
                                           (128, 8, 4), (64, 1, 8)])
def test_nan_pages(d, rank, v_bits):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    dev = torch.device("cuda", 0)
    NB, n_kv = 12, 2
    gen = torch.Generator(device=dev).manual_seed(5)
    k = torch.randn((NB, 16, n_kv, d), generator=gen, device=dev).to(
        torch.bfloat16)
    bad = k.clone()
    bad[3] = float("nan")                    # nothing written
    bad[5, 7:] = float("nan")                # seven tokens written
    bad[8, 2, 1, 3] = float("nan")           # one value, one head

    def build(keys):
        st = S.QuadState(dev, num_layers=1, num_blocks=NB, n_kv=n_kv, G=4,
                         head_dim=d, page=16, max_reqs=1, max_pages=NB,
                         rank=rank, v_bits=v_bits)
        SM.summarize_pages(st, [keys], torch.arange(
            NB, dtype=torch.int32, device=dev))
        torch.cuda.synchronize(dev)
        return st
    a, b = build(k), build(bad)
    ok = torch.ones(NB, n_kv, dtype=torch.bool, device=dev)
    ok[3] = ok[5] = False
    ok[8, 1] = False
    for n in ("quad_mu", "mu_scale", "quad_V", "V_scale", "quad_sig2"):
        x, y = getattr(a, n)[0], getattr(b, n)[0]
        assert torch.equal(x[ok], y[ok]), n
        assert bool(torch.isfinite(y.float()).all()), n
