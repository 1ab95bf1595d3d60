"""Calls the prefill-side entry points refuse, checked before any launch (no
GPU needed)."""
import copy
import ctypes

import pytest
import torch

from amass_kv_b200 import _lib
from amass_kv_b200.attention import paged_chunk_attention
from amass_kv_b200.paging import BlockPool, build_slot_map
from amass_kv_b200.rotary import (Rotary, rotary_embed, rotary_write_kv,
                                  rotary_write_pools)
from amass_kv_b200.serving import MemSession

CPU = torch.device("cpu")


class Buf:
    """What paged_chunk_attention reads of its buffers."""
    index, n_kv, G, d = -1, 2, 4, 64


def chunk_args(**kw):
    a = dict(q=torch.zeros(5, 8, 64, dtype=torch.bfloat16),
             kv_cache=torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16),
             block_table=torch.zeros(2, 3, dtype=torch.int32),
             seq_lens=torch.ones(2, dtype=torch.int32),
             query_start_loc=torch.zeros(3, dtype=torch.int32),
             out=torch.zeros(5, 8, 64, dtype=torch.bfloat16), buf=Buf())
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(5, 8, 64)), "bf16 or all fp16"),
    (dict(out=torch.zeros(5, 8, 64, dtype=torch.float16)), "bf16 or all"),
    (dict(out=torch.zeros(4, 8, 64, dtype=torch.bfloat16)), "same shape"),
    (dict(kv_cache=torch.zeros(4, 1, 16, 2, 64, dtype=torch.bfloat16)),
     "no V source"),
    (dict(kv_cache=torch.zeros(4, 2, 16, 4, 64, dtype=torch.bfloat16)),
     "do not fit"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int64)), "int32"),
    (dict(seq_lens=torch.ones(3, dtype=torch.int32)), "cover"),
    (dict(query_start_loc=torch.zeros(2, dtype=torch.int32)), "cover"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).t()),
     "contiguous in the last"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), "cover"),
    (dict(kv_cache=torch.zeros(20000, dtype=torch.bfloat16).as_strided(
        (4, 2, 16, 2, 64), (4104, 2048, 128, 64, 1))), "block strides"),
    (dict(window=0), "window"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(lse=torch.zeros(5, 4)), "lse"),
    (dict(q=torch.zeros(5, 8, 65, dtype=torch.bfloat16)[..., 1:]),
     "16-byte"),
    (dict(q=torch.zeros(5, 8, 128, dtype=torch.bfloat16)[..., ::2]),
     "contiguous head_dim"),
])
def test_chunk_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        paged_chunk_attention(**chunk_args(**kw))


def test_chunk_c_entry_refuses():
    lib = _lib.load()

    def call(**kw):
        a = dict(q=64, k=64, page=16, d=128, G=4, T=4, R=1, scale=0.1,
                 window=0, dtype=0, ksh=128, nb=3, mp=4, fault=64)
        a.update(kw)
        return lib.amass_paged_chunk(_lib.CHUNK.pack(
            a["q"], a["k"], 64, 64, 64, 64, 64, 64, 64, a["fault"], 64, 0,
            1024, 128, 4096, 256, a["ksh"], 4096, 256, 128, 4, 1024, 128,
            a["scale"], a["nb"], 8, a["window"], a["T"], a["R"], 2, a["G"],
            a["d"], a["page"], a["mp"], a["dtype"]), None)
    assert lib.amass_paged_chunk(None, None) == 1
    assert lib.amass_rotary_write(None, None) == 1
    assert call(T=0) == 0 and call(R=0) == 0
    for kw in (dict(q=0), dict(fault=0), dict(T=-1), dict(scale=0.0),
               dict(scale=float("nan")), dict(window=-1), dict(dtype=2),
               dict(ksh=100), dict(ksh=-128), dict(nb=0), dict(mp=0),
               dict(k=24)):
        assert call(**kw) == 1, kw
    for kw in (dict(d=96), dict(G=9), dict(page=32), dict(R=4097)):
        assert call(**kw) == 2, kw


def test_pool_refuses():
    for kw in (dict(num_blocks=0), dict(max_reqs=0), dict(max_reqs=4097),
               dict(max_pages=0), dict(max_tokens=0), dict(page=0),
               dict(max_pages=1 << 28)):
        a = dict(num_blocks=4, max_reqs=2, max_pages=3, max_tokens=9)
        a.update(kw)
        with pytest.raises(ValueError):
            BlockPool(CPU, **a)
    p = BlockPool(CPU, num_blocks=4, max_reqs=2, max_pages=3, max_tokens=9)
    one = torch.ones(2, dtype=torch.int32)
    for bad in (torch.ones(2), torch.ones(3, dtype=torch.int32),
                torch.ones(2, 1, dtype=torch.int32),
                torch.ones(4, dtype=torch.int32)[::2]):
        for f in (p.begin_step, p.truncate, p.release):
            with pytest.raises(ValueError):
                f(bad)
    for n in (-1, 10):
        with pytest.raises(ValueError):
            p.begin_step(one, n_tokens=n)
    p.check()
    p.overflow.fill_(6)
    with pytest.raises(RuntimeError, match="outgrew.*n_tokens"):
        p.check()
    lib = _lib.load()
    assert lib.amass_pages_begin(None, None, 0, 0, None) == 1
    assert lib.amass_pages_trim(None, None, 0, 0, None) == 1
    assert lib.amass_pages_trim(p._pool, None, 0, 0, None) == 0
    assert lib.amass_pages_trim(p._pool, None, 1, 0, None) == 1
    assert lib.amass_pages_begin(p._pool, ctypes.c_void_p(8), 3, 0, None) == 1
    assert lib.amass_pages_begin(p._pool, None, 0, 10, None) == 1
    with pytest.raises(AttributeError, match="fixed"):
        p.block_table = torch.zeros(2, 3, dtype=torch.int32)


def test_slot_map_refuses():
    i32, i64 = torch.int32, torch.int64
    a = dict(block_table=torch.zeros(2, 3, dtype=i32),
             seq_lens=torch.ones(2, dtype=i32),
             query_start_loc=torch.zeros(3, dtype=i32),
             positions=torch.zeros(9, dtype=i64),
             slot_mapping=torch.zeros(9, dtype=i64))
    for kw in (dict(positions=torch.zeros(9, dtype=i32)),
               dict(positions=torch.zeros(8, dtype=i64)),
               dict(slot_mapping=torch.zeros(18, dtype=i64)[::2]),
               dict(seq_lens=torch.ones(3, dtype=i32)), dict(page=0),
               dict(seq_lens=torch.ones(2)), dict(n_tokens=10)):
        with pytest.raises(ValueError):
            build_slot_map(**{**a, **kw})


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=258),
    dict(layout="pairs"), dict(base=1.0), dict(scaling=dict(factor=2.0)),
    dict(scaling=dict(type="linear")),
    dict(scaling=dict(type="linear", factor=0.5)),
    dict(scaling=dict(type="linear", factor=2.0, beta_fast=3)),
    dict(scaling=dict(type="yarn", factor=2.0)),
    dict(scaling=dict(type="yarn", factor=2.0, original_max_position=100,
                      beta_fast=1, beta_slow=2)),
    dict(scaling=dict(type="llama3", factor=2.0, low_freq_factor=4,
                      high_freq_factor=1, original_max_position=100)),
])
def test_rotary_refuses(kw):
    with pytest.raises(ValueError):
        Rotary(CPU, **{**dict(rotary_dim=64), **kw})


def test_rotary_calls_refuse():
    rot = Rotary(CPU, rotary_dim=64)
    bf = torch.bfloat16
    a = dict(q=torch.zeros(5, 8, 64, dtype=bf),
             k=torch.zeros(5, 2, 64, dtype=bf),
             v=torch.zeros(5, 2, 64, dtype=bf), positions=torch.arange(5),
             kv_cache=torch.zeros(4, 2, 16, 2, 64, dtype=bf),
             slot_mapping=torch.arange(5))
    for kw in (dict(q=torch.zeros(5, 8, 64)), dict(k=None), dict(v=None),
               dict(q=None, q_out=a["q"]),
               dict(positions=torch.arange(4)),
               dict(positions=torch.arange(5.0)),
               dict(slot_mapping=torch.arange(4)),
               dict(slot_mapping=torch.arange(5, dtype=torch.int32)),
               dict(slot_mapping=torch.arange(10)[::2]),
               dict(kv_cache=torch.zeros(4, 2, 16, 2, 128, dtype=bf)),
               dict(kv_cache=torch.zeros(4, 1, 16, 2, 64, dtype=bf)),
               dict(q_out=torch.zeros(5, 4, 64, dtype=bf)),
               dict(q_out=torch.zeros(4, 8, 64, dtype=bf)),
               dict(k=torch.zeros(5, 4, 64, dtype=bf)),
               dict(q=torch.zeros(5, 8, 32, dtype=bf)), dict(n_tokens=6),
               dict(n_tokens=-1)):
        with pytest.raises(ValueError):
            rotary_write_kv(rot, **{**a, **kw})
    with pytest.raises(ValueError):
        rotary_embed(rot, None, None, torch.arange(5))
    with pytest.raises(ValueError):
        rotary_embed(rot, a["q"], None, torch.arange(5), k_out=a["k"])
    with pytest.raises(ValueError):
        rotary_embed(rot, a["q"][..., :32], None, torch.arange(5))


def test_host_tensors_are_refused():
    """Arguments that fit in all but the device never reach a launch."""
    i32, bf = torch.int32, torch.bfloat16
    p = BlockPool(CPU, num_blocks=4, max_reqs=2, max_pages=3, max_tokens=9)
    rot = Rotary(CPU, rotary_dim=64)
    one = torch.ones(2, dtype=i32)
    q, at = torch.zeros(5, 8, 64, dtype=bf), torch.arange(5)

    class Whole(Buf):
        n_ctas, scratch = 1, (64, 64, 64, 64)
    for call in (
            lambda: p.begin_step(one), lambda: p.truncate(one),
            lambda: p.release(one),
            lambda: build_slot_map(p.block_table, one, torch.zeros(3, dtype=i32),
                                   p.positions, p.slot_mapping),
            lambda: rotary_embed(rot, q, None, at),
            lambda: rotary_embed(rot, None, q, at),
            lambda: rotary_write_kv(
                rot, q, q[:, :2], q[:, :2], at,
                torch.zeros(4, 2, 16, 2, 64, dtype=bf), at),
            lambda: paged_chunk_attention(**chunk_args(buf=Whole()))):
        with pytest.raises(ValueError, match="on a GPU"):
            call()


def test_expanded_outputs_are_refused():
    """One place for two heads, tokens or pages has no one answer."""
    rot, bf = Rotary(CPU, rotary_dim=64), torch.bfloat16
    at, q = torch.arange(5), torch.zeros(5, 8, 64, dtype=bf)
    one, k = torch.zeros(5, 1, 64, dtype=bf), q[:, :2]
    wide = one.expand(5, 8, 64)
    for call in (
            lambda: rotary_embed(rot, wide, None, at),
            lambda: rotary_embed(rot, q, None, at, q_out=wide),
            lambda: rotary_embed(rot, None, wide, at),
            lambda: rotary_embed(rot, None, q, at, k_out=wide),
            lambda: rotary_write_kv(
                rot, q, k, k, at, torch.zeros(1, 2, 16, 2, 64, dtype=bf)
                .expand(4, 2, 16, 2, 64), at),
            lambda: rotary_write_pools(
                rot, None, k, k, at, torch.zeros(4, 16, 2, 64, dtype=bf),
                torch.zeros(4, 1, 2, 64, dtype=bf).expand(4, 16, 2, 64), at)):
        with pytest.raises(ValueError, match="expanded"):
            call()


def test_buffers_are_not_copied():
    """Copies would keep the addresses of the buffers they were taken from."""
    p = BlockPool(CPU, num_blocks=4, max_reqs=2, max_pages=3, max_tokens=9)
    for f in (copy.copy, copy.deepcopy):
        with pytest.raises(TypeError, match="not copied"):
            f(p)
    assert copy.deepcopy(Rotary(CPU, rotary_dim=8)).freq.numel() == 4


def test_write_kv_refuses_half_a_rotary():
    rot, at = Rotary(CPU, rotary_dim=64), torch.arange(5)
    q = torch.zeros(5, 8, 64, dtype=torch.bfloat16)
    for kw in (dict(rotary=rot), dict(positions=at), dict(query=q),
               dict(rotary=rot, query=q), dict(positions=at, query=q)):
        with pytest.raises(ValueError, match="go together"):
            MemSession.write_kv(None, 0, q, q, at, 5, **kw)
