"""Rotary positions and the cache write against fp64."""
import copy
import math

import pytest
import torch

from amass_kv_b200.rotary import (Rotary, rotary_embed, rotary_frequencies,
                                  rotary_write_kv)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def turned(rot, x, pos):
    """fp64 rotation and the bound on the kernel's error: the frequency in
    fp64 is off by 2^-53 of itself on either side, so the angle by
    2^-51 |position|; the fraction of a turn rounds to 24 bits and sincospi
    to 2 ulp: 2^-21 absolute on cos and sin; two products and a sum in fp32;
    one rounding of the result to the 16-bit type."""
    r = rot.rotary_dim
    a = pos.double()[:, None, None] * rot.inv_freq.to(x.device)
    c, s = torch.cos(a) * rot.mscale, torch.sin(a) * rot.mscale
    y = x.double().clone()
    if rot.layout == "half":
        i, j = slice(0, r // 2), slice(r // 2, r)
    else:
        i, j = slice(0, r, 2), slice(1, r, 2)
    x0, x1 = x.double()[..., i], x.double()[..., j]
    y[..., i], y[..., j] = x0 * c - x1 * s, x1 * c + x0 * s
    u = torch.finfo(x.dtype).eps / 2
    near = torch.zeros_like(y)
    near[..., i] = near[..., j] = (x0.abs() + x1.abs()) * rot.mscale * (
        2.0 ** -20 + 2.0 ** -50 * pos.double().abs()[:, None, None])
    tol = u * y.abs() + near + torch.finfo(x.dtype).tiny * u
    tol[..., r:] = 0                                  # copied bit by bit
    return y, tol


def close(got, want):
    y, tol = want
    err = (got.double() - y).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def make(dev, T, H, n_kv, d, dtype, seed=0, nb=None, layout=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    qkv = torch.randn((T, H + 2 * n_kv, d), generator=gen,
                      device=dev).to(dtype)
    nb = nb or -(-T // 16) + 2
    shape = (nb, 2, 16, n_kv, d) if layout == 0 else (2, nb, 16, n_kv, d)
    kv = torch.full(shape, 5.0, device=dev, dtype=dtype)
    slots = torch.randperm(nb * 16, generator=gen, device=dev)[:T]
    return qkv[:, :H], qkv[:, H:H + n_kv], qkv[:, H + n_kv:], kv, slots


SCALINGS = [None, dict(type="linear", factor=4.0),
            dict(type="ntk", factor=8.0),
            dict(type="llama3", factor=8.0, low_freq_factor=1.0,
                 high_freq_factor=4.0, original_max_position=8192),
            dict(type="yarn", factor=16.0, original_max_position=4096)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,r,H,n_kv", [
    (128, 128, 32, 8), (64, 64, 8, 2), (128, 64, 4, 4), (128, 96, 7, 1),
    (64, 20, 3, 1), (128, 2, 2, 2), (80, 80, 2, 1), (256, 256, 1, 1),
    (6, 4, 2, 1)])
def test_write(dev, layout, dtype, d, r, H, n_kv):
    for T, sc in ((1, None), (9, SCALINGS[3]), (301, SCALINGS[4])):
        rot = Rotary(dev, rotary_dim=r, layout=layout, scaling=sc)
        q, k, v, kv, slots = make(dev, T, H, n_kv, d, dtype, seed=T)
        slots[T // 2] = -1
        if T > 5:
            slots[1] = kv.shape[0] * 16               # behind the cache
        pos = torch.randint(0, 100000, (T,), device=dev)
        q_out = torch.zeros((T, H, d), dtype=dtype, device=dev)
        k0, v0 = k.clone(), v.clone()
        rotary_write_kv(rot, q, k, v, pos, kv, slots, q_out=q_out)
        close(q_out, turned(rot, q, pos))
        ok = (slots >= 0) & (slots < kv.shape[0] * 16)
        at = slots[ok]
        y, tol = turned(rot, k, pos)
        close(kv[at // 16, 0, at % 16], (y[ok], tol[ok]))
        assert torch.equal(kv[at // 16, 1, at % 16], v[ok])
        rest = torch.ones(kv.shape[0] * 16, dtype=torch.bool, device=dev)
        rest[at] = False
        rest = rest.nonzero()[:, 0]
        assert bool((kv[rest // 16, :, rest % 16] == 5.0).all())
        assert torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.parametrize("scaling", SCALINGS)
def test_far_positions(dev, scaling):
    """Positions to 2^40, negative ones, both index types."""
    rot = Rotary(dev, rotary_dim=64, base=500000.0, scaling=scaling)
    pos = torch.tensor([0, 1, 2 ** 20 + 1, 2 ** 31 - 1, -3, 2 ** 33 + 12345,
                        2 ** 40 - 1], device=dev)
    for p in (pos, pos[:5].to(torch.int32)):
        q, k, v, kv, slots = make(dev, p.shape[0], 4, 2, 64, torch.bfloat16)
        q_out = torch.zeros_like(q)
        rotary_write_kv(rot, q, k, v, p, kv, slots, q_out=q_out)
        close(q_out, turned(rot, q, p))


def test_frequencies():
    """The scalings at the points where their definitions fix them."""
    r, b = 128, 10000.0
    f, m = rotary_frequencies(r, b)
    assert m == 1.0 and f[0] == 1.0 and math.isclose(float(f[-1]),
                                                     b ** (-126 / 128))
    assert torch.allclose(rotary_frequencies(r, b, SCALINGS[1])[0], f / 4)
    n = rotary_frequencies(r, b, SCALINGS[2])[0]
    assert n[0] == 1.0 and math.isclose(float(n[-1]), float(f[-1]) / 8,
                                        rel_tol=1e-12)
    g = rotary_frequencies(r, b, SCALINGS[3])[0]
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 4], f[turns >= 4])
    assert torch.equal(g[turns <= 1], f[turns <= 1] / 8)
    assert bool(((g <= f) & (g >= f / 8)).all())
    y, m = rotary_frequencies(r, b, SCALINGS[4])
    assert math.isclose(m, 0.1 * math.log(16) + 1)
    assert y[0] == f[0] and y[-1] == f[-1] / 16


def test_in_place_and_k_only(dev):
    rot = Rotary(dev, rotary_dim=32, layout="interleaved")
    q, k, v, kv, slots = make(dev, 70, 4, 2, 64, torch.bfloat16)
    pos = torch.arange(70, device=dev)
    wq, wk = turned(rot, q, pos), turned(rot, k, pos)
    konly = kv[:, :1].contiguous()
    rotary_write_kv(rot, q, k, None, pos, konly, slots)      # q in place
    close(q, wq)
    close(konly[slots // 16, 0, slots % 16], wk)
    k1 = k.clone()
    rotary_embed(rot, None, k1, pos)
    close(k1, wk)
    k2 = torch.zeros_like(k1)
    rotary_embed(rot, None, k, pos, k_out=k2, n_tokens=33)
    assert torch.equal(k2[:33], k1[:33]) and bool((k2[33:] == 0).all())
    rotary_write_kv(rot, None, k, v, pos, kv, slots, n_tokens=0)
    assert bool((kv == 5.0).all())


def test_odd_strides_and_alignment(dev):
    """A head stride and a base that 16-byte words cannot take, and the
    cache layout with K and V apart."""
    rot = Rotary(dev, rotary_dim=64)
    q, k, v, kv, slots = make(dev, 40, 4, 2, 64, torch.float16, layout=1)
    pos = torch.arange(40, device=dev) * 1001
    want = turned(rot, q, pos)
    raw = torch.zeros(40 * 4 * 67 + 1, dtype=torch.float16, device=dev)
    odd = raw[1:].view(40, 4, 67)[..., :64]
    rotary_write_kv(rot, q, k, v, pos, kv, slots, q_out=odd)
    close(odd, want)
    close(kv[0, slots // 16, slots % 16], turned(rot, k, pos))
    assert torch.equal(kv[1, slots // 16, slots % 16], v)


def test_copied_rotary(dev):
    """A copy has frequencies of its own."""
    rot = Rotary(dev, rotary_dim=64)
    k = torch.randn(9, 2, 64, device=dev).to(torch.bfloat16)
    at, other = torch.arange(9, device=dev), copy.deepcopy(rot)
    a, b = k.clone(), k.clone()
    rotary_embed(rot, None, a, at)
    rot.freq.zero_()
    rotary_embed(other, None, b, at)
    assert torch.equal(a, b)


def test_captured_padded_batch(dev):
    """A graph of a padded batch: padding rows have slot -1."""
    rot = Rotary(dev, rotary_dim=128)
    q, k, v, kv, slots = make(dev, 24, 8, 2, 128, torch.bfloat16)
    pos = torch.zeros(24, dtype=torch.int64, device=dev)
    q_out = torch.zeros_like(q)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        rotary_write_kv(rot, q, k, v, pos, kv, slots, q_out=q_out)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rotary_write_kv(rot, q, k, v, pos, kv, slots, q_out=q_out)
    kv.fill_(5.0)
    pos.copy_(torch.arange(24) + 4000)
    slots[10:] = -1
    g.replay()
    close(q_out, turned(rot, q, pos))
    at = slots[:10]
    y, tol = turned(rot, k, pos)
    close(kv[at // 16, 0, at % 16], (y[:10], tol[:10]))
    assert int((kv != 5.0).any(-1).any(-1).sum()) == 20
