"""A step that the block pool refuses in part, taken on to the attention."""
import pytest
import torch

from amass_kv_b200.attention import ChunkBuffers, paged_chunk_attention
from amass_kv_b200.paging import BlockPool
from amass_kv_b200.rotary import Rotary, rotary_write_kv
from tests.chunk_ref import chunk_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


@pytest.mark.parametrize("window", [None, 24])
@pytest.mark.parametrize("captured", [False, True])
def test_refused_rows(dev, window, captured):
    """Rows refused for want of blocks and for their length are 0 and -inf;
    the granted ones, one that needs no block among them, are what they are
    over their own tokens."""
    n_kv, G, d, R = 2, 4, 128, 5
    gen = torch.Generator(device=dev).manual_seed(8)
    pool = BlockPool(dev, num_blocks=12, max_reqs=R, max_pages=6,
                     max_tokens=200)
    rot = Rotary(dev, rotary_dim=d)
    kv = torch.full((pool.NB, 2, 16, n_kv, d), float("nan"), device=dev,
                    dtype=torch.bfloat16)
    buf = ChunkBuffers(dev, n_kv=n_kv, G=G, head_dim=d)
    new = torch.zeros(R, dtype=torch.int32, device=dev)
    q = torch.zeros((200, n_kv * G, d), device=dev, dtype=torch.bfloat16)
    k, v = (torch.zeros((200, n_kv, d), device=dev, dtype=torch.bfloat16)
            for _ in range(2))
    out = torch.zeros_like(q)
    lse = torch.zeros(200, n_kv * G, device=dev)

    def step():
        pool.begin_step(new)
        rotary_write_kv(rot, q, k, v, pool.positions, kv, pool.slot_mapping,
                        q_out=q)
        paged_chunk_attention(q, kv, pool.block_table, pool.seq_lens,
                              pool.query_start_loc, out, buf, window=window,
                              lse=lse, status=pool.status)
    run = step
    if captured:
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step()                           # nothing new: changes nothing
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            step()
        run = g.replay
    old = [0] * R
    for grow, status in (
            ([40, 20, 0, 17, 30], [0, 0, 0, 0, 0]),     # 9 of 12 blocks
            ([30, 33, 20, 5, 2], [0, 1, 1, 0, 0]),      # 2, no 2 and 2 of 1
            ([1, 100, 3, 1, 1], [0, 2, 0, 0, 1])):      # 1, then none left
        n = sum(grow)
        new.copy_(torch.tensor(grow, dtype=torch.int32))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device=dev))
        out.fill_(7.0)
        lse.fill_(7.0)
        run()
        buf.check()
        assert pool.status.tolist() == status
        lens, starts = [], [0]
        for r, x in enumerate(grow):
            old[r] += 0 if status[r] else x
            # a refused row's tokens are nobody's
            lens.append((0 if status[r] else x, old[r]))
            starts.append(starts[-1] + x)
        assert pool.seq_lens.tolist() == old
        ref, tol, lref, tol_l, rows = chunk_reference(
            q, kv[:, 0], kv[:, 1], pool.block_table, lens, starts,
            d ** -0.5, window)
        assert bool(((out.double() - ref).abs() <= tol)[rows].all())
        assert bool(((lse.double() - lref).abs() <= tol_l)[rows].all())
        refused = torch.zeros_like(rows)
        for r in range(R):
            if status[r]:
                refused[starts[r]:starts[r + 1]] = True
        assert bool((out[refused] == 0).all())
        assert bool((lse[refused] == float("-inf")).all())
        assert bool((out[n:] == 7.0).all()) and bool((lse[n:] == 7.0).all())


def test_status_that_does_not_fit(dev):
    buf = ChunkBuffers(dev, n_kv=2, G=4, head_dim=64)
    bf = dict(dtype=torch.bfloat16, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    for bad in (torch.zeros(1, **i32), torch.zeros(2, device=dev),
                torch.zeros(2, dtype=torch.int32),
                torch.zeros(2, 1, **i32), torch.zeros(4, **i32)[::2]):
        with pytest.raises(ValueError, match="status"):
            paged_chunk_attention(
                torch.zeros(5, 8, 64, **bf), torch.zeros(4, 2, 16, 2, 64, **bf),
                torch.zeros(2, 3, **i32), torch.ones(2, **i32),
                torch.zeros(3, **i32), torch.zeros(5, 8, 64, **bf), buf,
                status=bad)
