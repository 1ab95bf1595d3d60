"""Rotary positions of the new tokens' q and k, and the write of k and v into
the paged cache, in one launch.

  Rotary            frequencies of one rotary embedding: part of the head,
                    either pairing, the usual long-context scalings
  rotary_write_kv   turn q, turn k into the K cache, copy v into the V cache
                    at the step's slot mapping
  rotary_embed      turn q and k only

Angles are formed in the kernel from 64-bit fixed-point frequencies (turns per
token), so there is no cos / sin table and no largest position.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from ._lib import ptr
from .attention import DTYPES, split_kv

LAYOUTS = {"half": 0, "interleaved": 1}


def rotary_frequencies(rotary_dim: int, base: float, scaling=None):
    """(f (rotary_dim / 2,) fp64 in radians per token, factor on cos / sin).

    f_i = base^(-2 i / rotary_dim), then by ``scaling["type"]``, s = factor:
      linear  f_i / s (positions interpolated)
      ntk     base times s^(r / (r - 2)): the lowest frequency becomes f / s
      llama3  by turns within original_max_position: f / s below
              low_freq_factor, f above high_freq_factor, linear in between
      yarn    by dimension, ramp between the dimensions that turn beta_fast
              and beta_slow times within original_max_position; cos and sin
              times 0.1 ln(s) + 1 (or ``mscale``)
    """
    r = rotary_dim
    f = torch.tensor([float(base) ** (-2.0 * i / r) for i in range(r // 2)],
                     dtype=torch.float64)
    if scaling is None:
        return f, 1.0
    sc = dict(scaling)
    kind = sc.pop("type", None)
    needs = {"linear": ("factor",), "ntk": ("factor",),
             "llama3": ("factor", "low_freq_factor", "high_freq_factor",
                        "original_max_position"),
             "yarn": ("factor", "original_max_position")}
    if kind not in needs:
        raise ValueError(f"scaling type must be one of {sorted(needs)}, got "
                         f"{kind!r}")
    optional = {"yarn": ("beta_fast", "beta_slow", "mscale")}.get(kind, ())
    missing = [k for k in needs[kind] if k not in sc]
    extra = [k for k in sc if k not in needs[kind] + optional]
    if missing or extra:
        raise ValueError(f"{kind} scaling: missing {missing}, unknown {extra}")
    s = float(sc["factor"])
    if not 1.0 <= s < float("inf"):
        raise ValueError(f"scaling factor must be at least 1, got {s}")
    if kind == "linear":
        return f / s, 1.0
    if kind == "ntk":
        if r <= 2:
            raise ValueError("ntk scaling needs rotary_dim > 2")
        b = float(base) * s ** (r / (r - 2.0))
        return torch.tensor([b ** (-2.0 * i / r) for i in range(r // 2)],
                            dtype=torch.float64), 1.0
    orig = float(sc["original_max_position"])
    if orig <= 0:
        raise ValueError("original_max_position must be positive")
    if kind == "llama3":
        lo, hi = float(sc["low_freq_factor"]), float(sc["high_freq_factor"])
        if not 0 < lo < hi:
            raise ValueError("llama3 scaling needs 0 < low_freq_factor < "
                             "high_freq_factor")
        keep = ((orig * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        return f / s * (1 - keep) + f * keep, 1.0
    fast = float(sc.get("beta_fast", 32.0))
    slow = float(sc.get("beta_slow", 1.0))
    if not 0 < slow < fast:
        raise ValueError("yarn scaling needs 0 < beta_slow < beta_fast")

    def dim_of(turns):
        return r * math.log(orig / (turns * 2 * math.pi)) / \
            (2 * math.log(float(base)))
    lo = max(math.floor(dim_of(fast)), 0)
    hi = min(math.ceil(dim_of(slow)), r - 1)
    ramp = ((torch.arange(r // 2, dtype=torch.float64) - lo)
            / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
    m = sc.get("mscale")
    m = 0.1 * math.log(s) + 1.0 if m is None else float(m)
    return f / s * ramp + f * (1 - ramp), m


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
        dev = torch.device(device)
        if dev.index is None and dev.type == "cuda":
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device, self.rotary_dim, self.layout = dev, rotary_dim, layout
        self.inv_freq, self.mscale = rotary_frequencies(rotary_dim, base,
                                                        scaling)
        # turns per token as 64-bit binary fractions (f <= 1 rad < 1/6 turn)
        turns = [round(x / (2 * math.pi) * 2.0 ** 64)
                 for x in self.inv_freq.tolist()]
        self.freq = torch.tensor(turns, dtype=torch.int64, device=dev)


def _rows(name, t, dev, dtype, T, d):
    if t.dim() != 3 or t.shape[0] < T or t.shape[2] != d:
        raise ValueError(f"{name} must be (>= {T} tokens, heads, {d}), got "
                         f"{tuple(t.shape)}")
    if t.dtype != dtype or t.device != dev:
        raise ValueError(f"{name} must be {dtype} on {dev}, got {t.dtype} on "
                         f"{t.device}")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must have a contiguous head_dim")


def _launch(rot, q, q_out, k, v, k_dst, v_dst, slot_mapping, nb, page,
            positions, n_tokens):
    dev = rot.device
    x = q if q is not None else k
    if x is None:
        raise ValueError("nothing to turn: q and k are both None")
    if x.dim() != 3:
        raise ValueError(f"q and k must be (T, heads, d), got "
                         f"{tuple(x.shape)}")
    T = x.shape[0] if n_tokens is None else int(n_tokens)
    d = x.shape[2]
    if x.dtype not in DTYPES:
        raise ValueError(f"q, k and v must be bf16 or fp16, got {x.dtype}")
    if T < 0 or T > x.shape[0]:
        raise ValueError(f"n_tokens {T} outside 0 .. {x.shape[0]}")
    if rot.rotary_dim > d or d > 256 or d % 2:
        raise ValueError(f"no kernel for head_dim {d} with rotary_dim "
                         f"{rot.rotary_dim}")
    for name, t in (("q", q), ("q_out", q_out), ("k", k), ("v", v)):
        if t is not None:
            _rows(name, t, dev, x.dtype, T, d)
    if q is not None and q_out.shape[1] != q.shape[1]:
        raise ValueError("q_out must have q's heads")
    if v is not None and v.shape[1] != k.shape[1]:
        raise ValueError("v must have k's heads")
    if positions.dtype not in (torch.int32, torch.int64) or \
            positions.device != dev or positions.dim() != 1 or \
            positions.shape[0] < T or \
            (positions.shape[0] > 1 and positions.stride(0) != 1):
        raise ValueError(f"positions must be a contiguous int32 or int64 "
                         f"vector of at least {T} tokens on {dev}")

    def st(t, n):
        return [0] * n if t is None else list(t.stride()[:n])
    with torch.cuda.device(dev):
        _lib.call("amass_rotary_write", ptr(q), *st(q, 2), ptr(q_out),
                  *st(q_out, 2), ptr(k), *st(k, 2), ptr(v), *st(v, 2),
                  ptr(k_dst), *(st(k_dst, 3) if slot_mapping is not None
                                else _token_major(k_dst)),
                  ptr(v_dst), *st(v_dst, 3), ptr(slot_mapping), int(nb),
                  int(page), ptr(positions),
                  1 if positions.dtype == torch.int64 else 0, ptr(rot.freq),
                  float(rot.mscale), LAYOUTS[rot.layout], rot.rotary_dim,
                  int(T), int(q.shape[1]) if q is not None else 0,
                  int(k.shape[1]) if k is not None else 0, int(d),
                  DTYPES[x.dtype], _lib.stream_of(dev))


def _token_major(t):
    return [0, 0, 0] if t is None else [t.stride(0), 0, t.stride(1)]


def rotary_embed(rot, q, k, positions, *, q_out=None, k_out=None,
                 n_tokens=None) -> None:
    """Turn q (T, H, d) into ``q_out`` and k (T, n_kv, d) into ``k_out``
    (defaults: in place) for the first ``n_tokens`` tokens (default: all).
    Either of q and k may be None."""
    if q is None and q_out is not None or k is None and k_out is not None:
        raise ValueError("an output without its input")
    if q is not None and q_out is None:
        q_out = q
    if k is not None:
        if k_out is None:
            k_out = k
        if k_out.shape != k.shape or k_out.dtype != k.dtype or \
                k_out.device != k.device or k_out.stride(-1) != 1:
            raise ValueError("k_out must match k")
    _launch(rot, q, q_out, k, None, k_out, None, None, 1, 1, positions,
            n_tokens)


def rotary_write_kv(rot, q, k, v, positions, kv_cache, slot_mapping, *,
                    q_out=None, n_tokens=None) -> None:
    """One layer's step before attention: turn q (T, H, d) into ``q_out``
    (default: in place; q may be None), turn k (T, n_kv, d) into the K half
    and copy v into the V half of ``kv_cache`` (either layout of
    ``attention.split_kv``; a K-only cache takes ``v=None``) at
    ``slot_mapping`` (int64, block * page + offset; slots outside the cache
    are skipped).  k itself is left as it is.  Two tokens must not share a
    slot.  bf16 or fp16, the cache's type."""
    kc, vc = split_kv(kv_cache)
    if k is None:
        raise ValueError("rotary_write_kv needs k")
    if (v is None) != (vc is None):
        raise ValueError("v and the cache's V half go together")
    if kc.dtype != k.dtype or kc.device != rot.device or \
            kc.stride(3) != 1 or kc.shape[2] != k.shape[1] or \
            kc.shape[3] != k.shape[2]:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not fit the "
                         f"cache {tuple(kv_cache.shape)} {kv_cache.dtype}")
    if q is not None and q_out is None:
        q_out = q
    if q is None and q_out is not None:
        raise ValueError("q_out without q")
    T = k.shape[0] if n_tokens is None else int(n_tokens)
    if slot_mapping.dtype != torch.int64 or \
            slot_mapping.device != rot.device or slot_mapping.dim() != 1 or \
            slot_mapping.shape[0] < T or \
            (slot_mapping.shape[0] > 1 and slot_mapping.stride(0) != 1):
        raise ValueError(f"slot_mapping must be a contiguous int64 vector of "
                         f"at least {T} tokens on {rot.device}")
    _launch(rot, q, q_out, k, v, kc, vc, slot_mapping, kc.shape[0],
            kc.shape[1], positions, T)


__all__ = ["Rotary", "rotary_embed", "rotary_write_kv", "rotary_frequencies"]
