"""Which tensors cache_layout takes for a paged cache (no GPU needed)."""
import pytest
import torch

from amass_kv_b200.attention import (cache_layout, paged_chunk_attention,
                                     split_kv)
from amass_kv_b200.rotary import Rotary, rotary_write_kv
from tests.test_prefill_refusals import chunk_args

BF = torch.bfloat16


@pytest.mark.parametrize("shape", [
    (4, 2, 16, 2, 64), (2, 4, 16, 2, 64), (4, 1, 16, 2, 64),
    (1, 2, 16, 2, 64), (1, 1, 16, 2, 64), (2, 2, 16, 2, 64),
    (2, 16, 2, 3, 64), (5, 2, 1, 1, 8)])
def test_layouts_are_those_of_split_kv(shape):
    kv = torch.zeros(shape, dtype=BF)
    k, v = split_kv(kv)
    nb, page, n_kv, d, st, ka, va = cache_layout(kv)
    assert (nb, page, n_kv, d) == tuple(k.shape) and st == k.stride()[:3]
    assert ka == k.data_ptr() and va == (0 if v is None else v.data_ptr())


@pytest.mark.parametrize("shape,match", [
    ((4, 3, 16, 2, 64), "kv_cache must be"),     # three halves
    ((4, 16, 2, 2, 64), "kv_cache must be"),     # the page before K and V
    ((3, 4, 16, 2, 64), "kv_cache must be"),
    ((4, 0, 16, 2, 64), "kv_cache must be"),
    ((0, 2, 16, 2, 64), "empty"), ((2, 0, 16, 2, 64), "empty"),
    ((4, 2, 0, 2, 64), "empty"), ((4, 2, 16, 0, 64), "empty"),
    ((4, 2, 16, 2, 0), "empty"),
    ((2, 1, 16, 2, 64), "two blocks of keys"),   # or one of keys and values
    ((4, 2, 16, 64), "kv_cache must be")])
def test_other_shapes_are_refused(shape, match):
    kv = torch.zeros(shape, dtype=BF)
    with pytest.raises(ValueError, match=match):
        cache_layout(kv)
    with pytest.raises(ValueError, match=match):
        paged_chunk_attention(**chunk_args(kv_cache=kv))
    k = torch.zeros(5, 2, 64, dtype=BF)
    for v in (k, None):
        with pytest.raises(ValueError, match=match):
            rotary_write_kv(Rotary("cpu", rotary_dim=64), None, k, v,
                            torch.arange(5), kv, torch.arange(5))
