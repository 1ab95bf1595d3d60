"""Rotary positions of the new tokens' q and k, and the write of k and v into
the paged cache, in one launch.

  Rotary            frequencies of one rotary embedding: part of the head,
                    either pairing, the usual long-context scalings
  rotary_write_kv   turn q, turn k into the K cache, copy v into the V cache
                    at the step's slot mapping
  rotary_write_pools  the same into K and V pools apart (the tier's staging)
  rotary_embed      turn q and k only

Angles are formed in the kernel from 64-bit fixed-point frequencies (turns per
token), so there is no cos / sin table and no largest position.
"""
from __future__ import annotations

import decimal
import math

import torch

from . import _lib
from .attention import DTYPES, cache_layout

LAYOUTS = {"half": 0, "interleaved": 1}
# frequencies are formed as integers of 2^-256 from one power in 42 digits: fp64
# ones would leave an angle off by some 2^-55 turns a token, the 64-bit
# fractions can hold 2^-65
_LONG = decimal.Context(prec=42)
_ONE = 1 << 256
_TAU = 6283185307179586476925286766559005768394338798750 * _ONE // 10 ** 48


def rotary_frequencies(rotary_dim: int, base: float, scaling=None):
    """(f (rotary_dim / 2,) fp64 in radians per token, factor on cos / sin).

    f_i = base^(-2 i / rotary_dim), then by ``scaling["type"]``, s = factor:
      linear  f_i / s (positions interpolated)
      ntk     base times s^(r / (r - 2)): the lowest frequency becomes f / s
      llama3  by turns within original_max_position: f / s below
              low_freq_factor, f above high_freq_factor, linear in between
      yarn    by dimension, ramp between the dimensions that turn beta_fast
              and beta_slow times within original_max_position; cos and sin
              times ``attention_factor`` (default 0.1 ln(s) + 1)
    """
    f, m = _frequencies(rotary_dim, base, scaling)
    return torch.tensor([x / _ONE for x in f], dtype=torch.float64), m


def _fixed(x: float) -> int:
    n, d = x.as_integer_ratio()
    return n * _ONE // d


def _powers(r, log_base):
    """exp(-2 i log_base / r) in units of 2^-256, i < r / 2."""
    n, d = _LONG.exp(_LONG.multiply(log_base, _LONG.divide(
        decimal.Decimal(-2), decimal.Decimal(r)))).as_integer_ratio()
    q, f = n * _ONE // d, [_ONE]
    for _ in range(r // 2 - 1):
        f.append(f[-1] * q >> 256)
    return f


def _frequencies(r, base, scaling):
    """``rotary_frequencies`` in units of 2^-256."""
    r, log_base = int(r), _LONG.ln(decimal.Decimal(float(base)))
    if scaling is None:
        return _powers(r, log_base), 1.0
    sc = dict(scaling)
    kind = sc.pop("type", None)
    needs = {"linear": ("factor",), "ntk": ("factor",),
             "llama3": ("factor", "low_freq_factor", "high_freq_factor",
                        "original_max_position"),
             "yarn": ("factor", "original_max_position")}
    if kind not in needs:
        raise ValueError(f"scaling type must be one of {sorted(needs)}, got "
                         f"{kind!r}")
    optional = {"yarn": ("beta_fast", "beta_slow",
                         "attention_factor")}.get(kind, ())
    if kind == "yarn" and ("mscale" in sc or "mscale_all_dim" in sc):
        raise ValueError("mscale and mscale_all_dim are arguments of a formula "
                         "for the factor on cos and sin: give that factor as "
                         "attention_factor")
    missing = [k for k in needs[kind] if k not in sc]
    extra = [k for k in sc if k not in needs[kind] + optional]
    if missing or extra:
        raise ValueError(f"{kind} scaling: missing {missing}, unknown {extra}")
    s = float(sc["factor"])
    if not 1.0 <= s < float("inf"):
        raise ValueError(f"scaling factor must be at least 1, got {s}")
    if kind == "ntk":
        if r <= 2:
            raise ValueError("ntk scaling needs rotary_dim > 2")
        return _powers(r, _LONG.add(log_base, _LONG.multiply(
            _LONG.ln(decimal.Decimal(s)), _LONG.divide(
                decimal.Decimal(r), decimal.Decimal(r - 2))))), 1.0
    f = _powers(r, log_base)
    num, den = s.as_integer_ratio()
    if kind == "linear":
        return [x * den // num for x in f], 1.0

    def blend(keep):                         # f where keep is 1, f / s where 0
        return [(x * den // num * (_ONE - k) + x * k) >> 256 for x, k in
                ((x, min(max(k, 0), _ONE)) for x, k in zip(f, keep))]
    orig = float(sc["original_max_position"])
    if not 0 < orig < float("inf"):
        raise ValueError("original_max_position must be positive")
    if kind == "llama3":
        lo, hi = float(sc["low_freq_factor"]), float(sc["high_freq_factor"])
        if not 0 < lo < hi < float("inf"):
            raise ValueError("llama3 scaling needs 0 < low_freq_factor < "
                             "high_freq_factor")
        o, low, width = _fixed(orig), _fixed(lo), _fixed(hi) - _fixed(lo)
        return blend([(o * x // _TAU - low) * _ONE // width for x in f]), 1.0
    fast = float(sc.get("beta_fast", 32.0))
    slow = float(sc.get("beta_slow", 1.0))
    if not 0 < slow < fast:
        raise ValueError("yarn scaling needs 0 < beta_slow < beta_fast")

    def dim_of(turns):
        return r * math.log(orig / (turns * 2 * math.pi)) / \
            (2 * math.log(float(base)))
    lo = max(math.floor(dim_of(fast)), 0)
    hi = min(math.ceil(dim_of(slow)), r - 1)
    m = sc.get("attention_factor")
    m = 0.1 * math.log(s) + 1.0 if m is None else float(m)
    if not 0 < m < float("inf"):
        raise ValueError(f"attention_factor must be positive, got {m}")
    width = max(_fixed(float(hi - lo)), _ONE // 1000)
    return blend([_ONE - (i - lo) * _ONE * _ONE // width
                  for i in range(r // 2)]), m


class Rotary:
    """One rotary embedding: ``rotary_dim`` leading elements of each head in
    pairs (i, i + rotary_dim / 2) (``layout="half"``) or (2i, 2i + 1)
    (``"interleaved"``), frequencies by ``base`` and ``scaling`` (see
    ``rotary_frequencies``).  Holds the frequencies only; shared by all
    layers and streams."""

    def __init__(self, device, *, rotary_dim: int, base: float = 10000.0,
                 layout: str = "half", scaling=None):
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(LAYOUTS)}, got "
                             f"{layout!r}")
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > 256:
            raise ValueError(f"rotary_dim must be even and 2 .. 256, got "
                             f"{rotary_dim}")
        if not 1.0 < base < float("inf"):
            raise ValueError(f"base must be above 1, got {base}")
        dev = _lib.device_of(device)
        self.index = -1 if dev.index is None else dev.index
        self.device, self.rotary_dim, self.layout = dev, rotary_dim, layout
        f, self.mscale = _frequencies(rotary_dim, base, scaling)
        self.inv_freq = torch.tensor([x / _ONE for x in f],
                                     dtype=torch.float64)
        # turns per token as 64-bit binary fractions (f <= 1 rad < 1/6 turn)
        turns = [((x << 65) + _TAU) // (2 * _TAU) for x in f]
        self.freq = torch.tensor(turns, dtype=torch.int64, device=dev)


_NONE = (0, 0, 0, 0)                     # pointer, token / head stride, heads


def _rows(index, name, t, dtype, T, d):
    """(address, token stride, head stride, heads) of (>= T, heads, d)."""
    shape, s = t.shape, t.stride()
    if len(shape) != 3 or shape[0] < T or shape[2] != d or s[2] != 1 or \
            t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{name} must be (>= {T} tokens, heads, {d}) {dtype} "
                         f"on GPU {index} with a contiguous head_dim, got "
                         f"{tuple(shape)} {t.dtype} on {t.device}")
    return t.data_ptr(), s[0], s[1], shape[1]


def _vector(index, name, t, T, dtypes):
    """(address, its place in dtypes) of a vector of >= T tokens."""
    dtype = t.dtype
    if dtype not in dtypes or t.get_device() != index or t.dim() != 1 or \
            t.numel() < T or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of at least "
                         f"{T} tokens, {' or '.join(map(str, dtypes))}, on "
                         f"GPU {index}")
    return t.data_ptr(), dtypes.index(dtype)


_SLOTS, _INDEX = (torch.int64,), (torch.int32, torch.int64)


def _launch(rot, x, q, q_out, k, v, k_dst, kd, v_dst, vd, slots, nb, page,
            positions, T):
    dtype, shape, index, r = x.dtype, x.shape, rot.index, rot.rotary_dim
    type_id = DTYPES.get(dtype)
    if type_id is None:
        raise ValueError(f"q, k and v must be bf16 or fp16, got {dtype}")
    if len(shape) != 3 or not 0 <= T <= shape[0]:
        raise ValueError(f"n_tokens {T} outside the tokens of {tuple(shape)}")
    d = shape[2]
    if r > d or d > 256 or d % 2:
        raise ValueError(f"no kernel for head_dim {d} with rotary_dim {r}")
    qp, q_st, q_sh, H = o = _NONE if q is None else \
        _rows(index, "q", q, dtype, T, d)
    if q_out is not q:
        o = _rows(index, "q_out", q_out, dtype, T, d)
    op, o_st, o_sh, o_h = o
    if o_h != H:
        raise ValueError("q_out must have q's heads")
    if (op and not (o_st and o_sh)) or (v is not None and 0 in vd) or \
            (k is not None and 0 in (kd if slots else kd[::2])):
        raise ValueError("q_out, k_out and the caches must not be expanded")
    kp, k_st, k_sh, n_kv = _NONE if k is None else \
        _rows(index, "k", k, dtype, T, d)
    vp, v_st, v_sh, nv = _NONE if v is None else \
        _rows(index, "v", v, dtype, T, d)
    if v is not None and nv != n_kv:
        raise ValueError("v must have k's heads")
    pos, pos64 = _vector(index, "positions", positions, T, _INDEX)
    if T == 0:
        return
    _lib.launch(index, "amass_rotary_write", _lib.ROTARY.pack(
        qp, op, kp, vp, k_dst, v_dst, slots, pos, rot.freq.data_ptr(), q_st,
        q_sh, o_st, o_sh, k_st, k_sh, v_st, v_sh, *kd, *vd, rot.mscale, nb,
        page, pos64, LAYOUTS[rot.layout], r, T, H, n_kv, d, type_id, 0))


def rotary_embed(rot, q, k, positions, *, q_out=None, k_out=None,
                 n_tokens=None) -> None:
    """Turn q (T, H, d) into ``q_out`` and k (T, n_kv, d) into ``k_out``
    (defaults: in place) for the first ``n_tokens`` tokens (default: all).
    Either of q and k may be None.  An output may be its input itself, but
    must not overlap it in another way."""
    x = q if q is not None else k
    if x is None or (q is None and q_out is not None) or \
            (k is None and k_out is not None):
        raise ValueError("an output needs its input, and q or k must be given")
    T = x.shape[0] if n_tokens is None else int(n_tokens)
    kd, dst = (0, 0, 0), 0
    if k is not None:
        k_out = k if k_out is None else k_out
        dst, st, sh, heads = _rows(rot.index, "k_out", k_out, x.dtype, T,
                                   x.shape[-1])
        if heads != k.shape[1]:
            raise ValueError("k_out must have k's heads")
        kd = (st, 0, sh)                 # one token a block, no slot mapping
    _launch(rot, x, q, q if q_out is None else q_out, k, None, dst, kd, 0,
            (0, 0, 0), 0, 1, 1, positions, T)


def rotary_write_kv(rot, q, k, v, positions, kv_cache, slot_mapping, *,
                    q_out=None, n_tokens=None) -> None:
    """One layer's step before attention: turn q (T, H, d) into ``q_out``
    (default: in place; q may be None), turn k (T, n_kv, d) into the K half
    and copy v into the V half of ``kv_cache`` (either layout of
    ``attention.split_kv``; a K-only cache takes ``v=None``) at
    ``slot_mapping`` (int64, block * page + offset; slots outside the cache
    are skipped) for the first ``n_tokens`` tokens (default: all of k).  k
    itself is left as it is.  Two tokens must not share a slot.  bf16 or
    fp16, the cache's type."""
    if k is None:
        raise ValueError("rotary_write_kv needs k")
    nb, page, n_kv, d, st, kc, vc = cache_layout(kv_cache)
    if (v is None) != (not vc):
        raise ValueError("v and the cache's V half go together")
    shape = k.shape
    if kv_cache.dtype is not k.dtype or kv_cache.get_device() != rot.index or \
            len(shape) != 3 or shape[1] != n_kv or shape[2] != d:
        raise ValueError(f"k {tuple(shape)} {k.dtype} does not fit the "
                         f"cache {tuple(kv_cache.shape)} {kv_cache.dtype}")
    if q is None and q_out is not None:
        raise ValueError("q_out without q")
    T = shape[0] if n_tokens is None else int(n_tokens)
    slots, _ = _vector(rot.index, "slot_mapping", slot_mapping, T,
                       _SLOTS)
    _launch(rot, k, q, q if q_out is None else q_out, k, v, kc, st, vc,
            st if vc else (0, 0, 0), slots, nb, page, positions, T)


def rotary_write_pools(rot, q, k, v, positions, k_pool, v_pool, slot_mapping,
                       *, q_out=None, n_tokens=None) -> None:
    """``rotary_write_kv`` into K and V pools that are tensors of their own,
    (num_blocks, page, n_kv, d) each (the tier's staging pools); v and
    ``v_pool`` may be None."""
    if k is None or (q is None and q_out is not None) or \
            (v is None) != (v_pool is None):
        raise ValueError("rotary_write_pools needs k, q for q_out, and v and "
                         "v_pool together")
    strides = [(0, 0, 0), (0, 0, 0)]
    for i, (name, t) in enumerate((("k_pool", k_pool), ("v_pool", v_pool))):
        if t is None:
            continue
        if t.dim() != 4 or t.dtype != k.dtype or \
                t.get_device() != rot.index or t.stride(3) != 1 or \
                t.shape[2:] != k.shape[1:] or t.shape[:2] != k_pool.shape[:2]:
            raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not fit "
                             f"{name} {tuple(t.shape)} {t.dtype}")
        strides[i] = t.stride()[:3]
    T = k.shape[0] if n_tokens is None else int(n_tokens)
    slots, _ = _vector(rot.index, "slot_mapping", slot_mapping, T,
                       _SLOTS)
    _launch(rot, k, q, q if q_out is None else q_out, k, v,
            k_pool.data_ptr(), strides[0],
            0 if v_pool is None else v_pool.data_ptr(), strides[1], slots,
            k_pool.shape[0], k_pool.shape[1], positions, T)


__all__ = ["Rotary", "rotary_embed", "rotary_write_kv", "rotary_write_pools",
           "rotary_frequencies"]
