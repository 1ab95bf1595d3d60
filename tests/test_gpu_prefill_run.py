"""The prefill side as it is used: page bookkeeping, rotary positions with the
cache write and chunk attention over several steps and layers, then the
selection and sparse decode on the cache they filled."""
import numpy as np
import pytest
import torch

from amass_kv_b200 import attention as A
from amass_kv_b200 import selection as S
from amass_kv_b200 import summaries as SM
from amass_kv_b200.paging import BlockPool, build_slot_map
from amass_kv_b200.rotary import Rotary, rotary_embed, rotary_write_kv
from amass_kv_b200.serving import MemSession
from tests.chunk_ref import chunk_reference

pytestmark = pytest.mark.gpu
PAGE = 16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


@pytest.mark.parametrize("n_kv,G,d", [(2, 4, 128), (2, 4, 64)])
def test_steps(dev, n_kv, G, d):
    """Chunks, decode steps, a draft turned down, a request replaced: every
    step's attention equals the fp64 one over the rotated keys so far, and a
    decode step's equals the sparse decode of all pages."""
    L, R, MP = 2, 3, 40
    H = n_kv * G
    gen = torch.Generator(device=dev).manual_seed(11)
    pool = BlockPool(dev, num_blocks=R * MP - 20, max_reqs=R, max_pages=MP,
                     max_tokens=600)
    rot = Rotary(dev, rotary_dim=d, base=500000.0, scaling=dict(
        type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
        original_max_position=8192))
    kv = [torch.full((pool.NB, 2, PAGE, n_kv, d), float("nan"), device=dev,
                     dtype=torch.bfloat16) for _ in range(L)]
    buf = A.ChunkBuffers(dev, n_kv=n_kv, G=G, head_dim=d)
    st = S.QuadState(dev, num_layers=L, num_blocks=pool.NB, n_kv=n_kv, G=G,
                     head_dim=d, page=PAGE, max_reqs=R, max_pages=MP,
                     budget=1.0)
    A.ensure_stage_b_buffers(st, dev)
    # the model: rotated keys and values per layer and request, in order
    hist = [[[torch.empty(0, n_kv, d, device=dev, dtype=torch.bfloat16)
              for _ in range(2)] for _ in range(R)] for _ in range(L)]
    lens = np.zeros(R, np.int64)
    steps = [[70, 0, 33], [130, 5, 1], [1, 1, 1], [4, 3, 1], "draft",
             [1, 1, 1], "replace", [1, 200, 1], [1, 1, 1]]
    for step in steps:
        if step == "draft":
            drop = [3, 1, 0]
            pool.truncate(torch.tensor(drop, dtype=torch.int32, device=dev))
            lens -= drop
            for l in range(L):
                for r in range(R):
                    hist[l][r] = [x[:lens[r]] for x in hist[l][r]]
            continue
        if step == "replace":
            pool.release(torch.tensor([0, 1, 0], dtype=torch.int32,
                                      device=dev))
            lens[1] = 0
            for l in range(L):
                hist[l][1] = [x[:0] for x in hist[l][1]]
            continue
        new = np.array(step)
        T, pad = int(new.sum()), 7
        pool.begin_step(torch.tensor(step, dtype=torch.int32, device=dev),
                        n_tokens=T + pad)
        lens += new
        starts = np.concatenate([[0], np.cumsum(new)]).tolist()
        assert pool.seq_lens.tolist() == lens.tolist()
        pool.check()
        # an engine's own slot map from the same table
        pos = torch.empty_like(pool.positions)
        slot = torch.empty_like(pool.slot_mapping)
        build_slot_map(pool.block_table, pool.seq_lens, pool.query_start_loc,
                       pos, slot, n_tokens=T + pad)
        assert torch.equal(pos[:T + pad], pool.positions[:T + pad])
        assert torch.equal(slot[:T + pad], pool.slot_mapping[:T + pad])
        for l in range(L):
            qkv = torch.randn((T + pad, H + 2 * n_kv, d), generator=gen,
                              device=dev).to(torch.bfloat16)
            q, k, v = qkv[:, :H], qkv[:, H:H + n_kv], qkv[:, H + n_kv:]
            kr = k.clone()
            rotary_embed(rot, None, kr, pool.positions[:T + pad])
            rotary_write_kv(rot, q, k, v, pool.positions, kv[l],
                            pool.slot_mapping, n_tokens=T + pad)
            out = torch.full_like(q, 7.0)
            A.paged_chunk_attention(q, kv[l], pool.block_table,
                                    pool.seq_lens, pool.query_start_loc, out,
                                    buf)
            for r in range(R):
                a, b = starts[r], starts[r + 1]
                hist[l][r] = [torch.cat([hist[l][r][0], kr[a:b]]),
                              torch.cat([hist[l][r][1], v[a:b]])]
                n = int(lens[r])
                tok = torch.arange(n, device=dev)
                blk = pool.block_table[r, tok // PAGE].long()
                assert torch.equal(kv[l][blk, 0, tok % PAGE], hist[l][r][0])
                assert torch.equal(kv[l][blk, 1, tok % PAGE], hist[l][r][1])
            ref, tol, _, _, rows = chunk_reference(
                q, kv[l][:, 0], kv[l][:, 1], pool.block_table,
                list(zip(new.tolist(), lens.tolist())), starts, d ** -0.5)
            assert bool(((out.double() - ref).abs() <= tol)[rows].all())
            assert bool((out[T:] == 7.0).all())
            if new.max() != 1 or new.min() != 1:
                continue
            S.derive_page_params(st, pool.seq_lens, R)
            # budget 1: every page of every request
            SM.quad_build_bulk(st, [c[:, 0] for c in kv], pool.block_table,
                               pool.seq_lens, R, MP)
            S.select_pages_quad(st, l, q, pool.block_table, pool.seq_lens, R,
                                d ** -0.5)
            assert st.page_cnt.tolist() == [
                [-(-int(n) // PAGE)] * n_kv for n in lens]
            sp = torch.zeros_like(q[:R].contiguous())
            A.sparse_paged_decode_batched_cuda(
                q[:R], kv[l], pool.block_table, pool.seq_lens, st, sp,
                scale=d ** -0.5)
            assert bool(((sp.double() - ref[:R]).abs()
                         <= 2e-2 + 1e-2 * ref[:R].abs()).all())
    buf.check()


@pytest.mark.parametrize("offload_k", [False, True])
def test_mem_session_turns_keys(dev, offload_k):
    """MemSession.write_kv with a rotary leaves the caches as with keys turned
    beforehand, and turns the query in place."""
    L, R, MP, n_kv, G, d = 1, 2, 8, 2, 4, 128
    NB = R * MP + 3
    rot = Rotary(dev, rotary_dim=64, layout="interleaved")
    kw = dict(num_layers=L, num_blocks=NB, n_kv=n_kv, G=G, head_dim=d,
              max_reqs=R, max_pages=MP, max_tokens=64, hot_slots=8,
              budget=0.5, offload_k=offload_k, device=dev)
    one, two = MemSession(**kw), MemSession(**kw)
    bt = torch.randperm(NB, device=dev)[:R * MP].to(torch.int32).view(R, MP)
    sl = torch.tensor([37, 20], dtype=torch.int32, device=dev)
    qsl = torch.tensor([0, 37, 57], dtype=torch.int32, device=dev)
    pos = torch.zeros(57, dtype=torch.int64, device=dev)
    slot = torch.zeros(57, dtype=torch.int64, device=dev)
    build_slot_map(bt, sl, qsl, pos, slot)
    q = torch.randn((57, n_kv * G, d), device=dev).to(torch.bfloat16)
    k = torch.randn((57, n_kv, d), device=dev).to(torch.bfloat16)
    v = torch.randn((57, n_kv, d), device=dev).to(torch.bfloat16)
    q1, q2, k2 = q.clone(), q.clone(), k.clone()
    rotary_embed(rot, q2, k2, pos)
    for s in (one, two):
        s.begin_step(bt, sl, qsl, 37, 57)
    one.write_kv(0, k, v, slot, 57, rotary=rot, positions=pos, query=q1)
    two.write_kv(0, k2, v, slot, 57)
    assert torch.equal(q1, q2) and not torch.equal(k, k2)
    assert torch.equal(one.k_cache, two.k_cache)
    a, b = one.tier.staging, two.tier.staging
    assert torch.equal(a.v_pool, b.v_pool)
    if offload_k:
        assert torch.equal(a.k_pool, b.k_pool)


def test_blocks_past_32_bit_offsets(dev):
    """A cache of 4.6e9 elements: its last blocks are written and read where
    they are."""
    NB, n_kv, G, d = 140000, 8, 4, 128
    if torch.cuda.mem_get_info(dev)[0] < 20 << 30:
        pytest.skip("needs 10 GB")
    kv = torch.empty((NB, 2, PAGE, n_kv, d), dtype=torch.bfloat16, device=dev)
    lens, T = [(40, 40), (1, 1)], 41
    bt = torch.tensor([[NB - 1, 0, NB - 3], [NB - 2, -1, -1]],
                      dtype=torch.int32, device=dev)
    kv[[0, NB - 3, NB - 2, NB - 1]] = float("nan")
    sl = torch.tensor([40, 1], dtype=torch.int32, device=dev)
    qsl = torch.tensor([0, 40, 41], dtype=torch.int32, device=dev)
    pos = torch.empty(T, dtype=torch.int64, device=dev)
    slot = torch.empty_like(pos)
    build_slot_map(bt, sl, qsl, pos, slot)
    assert int(slot.max()) == (NB - 1) * PAGE + PAGE - 1
    gen = torch.Generator(device=dev).manual_seed(3)
    q, k, v = (torch.randn((T, h, d), generator=gen, device=dev)
               .to(torch.bfloat16) for h in (n_kv * G, n_kv, n_kv))
    rot = Rotary(dev, rotary_dim=d)
    kr = k.clone()
    rotary_embed(rot, None, kr, pos)
    rotary_write_kv(rot, q, k, v, pos, kv, slot)
    assert torch.equal(kv[slot // PAGE, 0, slot % PAGE], kr)
    assert torch.equal(kv[slot // PAGE, 1, slot % PAGE], v)
    out = torch.empty_like(q)
    buf = A.ChunkBuffers(dev, n_kv=n_kv, G=G, head_dim=d)
    A.paged_chunk_attention(q, kv, bt, sl, qsl, out, buf)
    buf.check()
    ref, tol, _, _, _ = chunk_reference(q, kv[:, 0], kv[:, 1], bt, lens,
                                        [0, 40, 41], d ** -0.5)
    assert bool(((out.double() - ref).abs() <= tol).all())
