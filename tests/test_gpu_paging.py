"""Page bookkeeping on the GPU against a sequential model on the host."""
import numpy as np
import pytest
import torch

from amass_kv_b200.paging import BlockPool, build_slot_map

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


class Model:
    """The same bookkeeping, one request and one page at a time."""

    def __init__(self, p):
        self.page, self.MP, self.R = p.page, p.MP, p.R
        self.stack = p.free_stack[:int(p.free_top)].tolist()
        self.table = [[] for _ in range(p.R)]
        self.len = [0] * p.R

    def pages(self, n):
        return -(-n // self.page)

    def begin(self, new, n_tokens):
        status, qsl, pos, slot, asked = [], [0], [], [], 0
        room = len(self.stack)
        for r, x in enumerate(new):
            x = max(x, 0)
            old, want = self.len[r], self.len[r] + x
            need = self.pages(want) - self.pages(old)
            if self.pages(want) > self.MP:
                st = 2
            else:
                asked += need
                st = 1 if need and asked > room else 0
            if st == 0:
                self.table[r] += [self.stack.pop() for _ in range(need)]
                self.len[r] = want
            for i in range(x):
                p = old + i
                pos.append(p)
                slot.append(-1 if st else self.table[r][p // self.page]
                            * self.page + p % self.page)
            status.append(st)
            qsl.append(qsl[-1] + x)
        k = max(0, n_tokens - len(pos))
        return status, qsl, (pos + [0] * k)[:n_tokens], \
            (slot + [-1] * k)[:n_tokens]

    def drop(self, n):
        for r in reversed(range(len(n))):
            x = min(max(n[r], 0), self.len[r])
            self.len[r] -= x
            while len(self.table[r]) > self.pages(self.len[r]):
                self.stack.append(self.table[r].pop())

    def same(self, p):
        top = int(p.free_top)
        assert p.free_stack[:top].tolist() == self.stack
        assert p.seq_lens.tolist() == self.len
        bt = p.block_table.tolist()
        for r in range(self.R):
            assert bt[r] == self.table[r] + [-1] * (self.MP -
                                                    len(self.table[r]))


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("R,page,big", [(1, 16, 40), (3, 16, 1), (17, 4, 9),
                                        (700, 16, 5), (64, 16, 300),
                                        (4096, 16, 2), (5, 1, 3)])
def test_random_steps(dev, R, page, big):
    """Growth, drafts dropped, requests released, until blocks run out."""
    rng = np.random.default_rng(R * 31 + page)
    MP = 4 + big
    NB = max(2, R * 3 // 2 + big * R // (2 * page))
    p = BlockPool(dev, num_blocks=NB, max_reqs=R, max_pages=MP,
                  max_tokens=R * big + 40, page=page)
    m = Model(p)
    seen = set()
    for step in range(14):
        n = int(rng.integers(1, R + 1)) if step % 3 else R
        new = rng.integers(-1, big + 1, n).tolist()
        nt = min(p.max_tokens, max(0, sum(max(x, 0) for x in new)
                                   + int(rng.integers(-2, 9))))
        p.begin_step(i32(new, dev), n_tokens=nt)
        st, qsl, pos, slot = m.begin(new, nt)
        assert p.status[:n].tolist() == st
        assert p.query_start_loc[:n + 1].tolist() == qsl
        assert p.positions[:nt].tolist() == pos
        assert p.slot_mapping[:nt].tolist() == slot
        m.same(p)
        seen |= set(st)
        if step % 4 == 1:
            drop = rng.integers(-1, big + 2, n).tolist()
            p.truncate(i32(drop, dev))
            m.drop(drop)
        elif step % 4 == 3:
            done = (rng.random(n) < 0.4).astype(int).tolist()
            p.release(i32(done, dev))
            m.drop([m.len[r] if d else 0 for r, d in enumerate(done)])
        m.same(p)
    assert 0 in seen and int(p.ticket) == 0
    assert (int(p.overflow) & 1 != 0) == (1 in seen)
    assert (int(p.overflow) & 2 != 0) == (2 in seen)


def test_undo_restores_the_stack(dev):
    p = BlockPool(dev, num_blocks=500, max_reqs=9, max_pages=60,
                  max_tokens=2000)
    p.free_stack.copy_(torch.randperm(500, device=dev).to(torch.int32))
    p.begin_step(i32([5, 0, 100, 33, 16, 1, 48, 90, 17], dev))
    before = [p.free_stack.clone(), p.free_top.clone(), p.seq_lens.clone(),
              p.block_table.clone()]
    new = i32([30, 200, 1, 0, 16, 15, 3, 300, 7], dev)
    p.begin_step(new)
    p.truncate(new)
    for a, b in zip(before, (p.free_stack, p.free_top, p.seq_lens,
                             p.block_table)):
        assert torch.equal(a, b)


def test_refusals_on_the_device(dev):
    """Too few blocks, a row too long, more tokens than the maps hold."""
    p = BlockPool(dev, num_blocks=4, max_reqs=4, max_pages=3, max_tokens=100)
    p.begin_step(i32([33, 49, 20, 0], dev))
    # 3 pages fit, the row of 4 pages is too long, 2 more pages do not fit
    assert p.status.tolist() == [0, 2, 1, 0]
    assert p.seq_lens.tolist() == [33, 0, 0, 0]
    assert int(p.overflow) == 1 + 2 + 4      # 33 + 49 + 20 > 100 tokens too
    assert p.slot_mapping[33:].tolist() == [-1] * 67
    assert p.positions[33:40].tolist() == list(range(7))
    with pytest.raises(RuntimeError, match="ran out, a row outgrew"):
        p.check()
    p.overflow.zero_()
    p.begin_step(i32([5], dev), n_tokens=3)
    assert int(p.overflow) == 4 and p.seq_lens.tolist()[0] == 38
    p.begin_step(torch.empty(0, dtype=torch.int32, device=dev), n_tokens=2)
    assert p.slot_mapping[:2].tolist() == [-1, -1]
    assert p.query_start_loc.tolist()[0] == 0


def test_counts_past_any_step(dev):
    """New tokens whose sum passes 32 bits: those rows and the later ones are
    refused, nothing wraps, a row that asks for none stays granted."""
    big, end = 2 ** 31 - 1, 2 ** 30
    p = BlockPool(dev, num_blocks=9, max_reqs=6, max_pages=3, max_tokens=40)
    p.begin_step(i32([5, big, big, 7, 0, big], dev), n_tokens=30)
    assert p.status.tolist() == [0, 2, 2, 2, 0, 2]
    assert p.seq_lens.tolist() == [5, 0, 0, 0, 0, 0]
    assert p.query_start_loc.tolist() == [0, 5] + [end] * 5
    assert int(p.free_top) == 8 and int(p.overflow) == 2 + 4
    assert p.block_table[1:].max() == -1 and p.block_table[0, 1:].max() == -1
    assert p.slot_mapping[:30].tolist() == list(range(5)) + [-1] * 25
    p.begin_step(i32([30, 30, 3, 0, 16, 16], dev))
    assert p.seq_lens.tolist() == [35, 30, 3, 0, 16, 16]
    assert int(p.free_top) == 9 - 3 - 2 - 1 - 1 - 1


def test_captured(dev):
    """One graph serves steps of other counts, padded to its size."""
    p = BlockPool(dev, num_blocks=300, max_reqs=8, max_pages=40,
                  max_tokens=256)
    m = Model(p)
    new = i32([1] * 8, dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        p.begin_step(new, n_tokens=128)
    side.synchronize()
    m.begin([1] * 8, 128)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.begin_step(new, n_tokens=128)
    for v in ([1, 2, 3, 4, 5, 6, 7, 8], [0] * 8, [16, 0, 30, 1, 1, 1, 1, 40]):
        new.copy_(i32(v, dev))
        g.replay()
        _, _, pos, slot = m.begin(v, 128)
        assert p.positions[:128].tolist() == pos
        assert p.slot_mapping[:128].tolist() == slot
        m.same(p)


@pytest.mark.parametrize("R", [1, 5, 300, 4096])
def test_slot_map(dev, R):
    rng = np.random.default_rng(R)
    MP, page = 12, 16
    new = rng.integers(0, 40, R)
    sl = new + rng.integers(0, MP * page - 39, R)
    sl[0] = new[0] - 3 if new[0] > 3 else sl[0]       # first rows below 0
    bt = rng.integers(0, 10 ** 6, (R, MP + 2)).astype(np.int32)
    bt[R // 2, 2] = -1
    qsl = np.concatenate([[2], 2 + np.cumsum(new)])
    T = int(qsl[-1]) + 5
    pos = torch.full((T,), 99, dtype=torch.int64, device=dev)
    slot = torch.full((T,), 99, dtype=torch.int64, device=dev)
    table = torch.from_numpy(bt).to(dev)[:, :MP]
    build_slot_map(table, i32(sl, dev), i32(qsl, dev), pos, slot)
    wp, ws = [0] * T, [-1] * T
    for r in range(R):
        for i in range(new[r]):
            p = int(sl[r] - new[r] + i)
            t = int(qsl[r]) + i
            wp[t] = p
            if 0 <= p < MP * page and bt[r, p // page] >= 0:
                ws[t] = int(bt[r, p // page]) * page + p % page
    assert pos.tolist() == wp and slot.tolist() == ws
    slot.fill_(99)
    build_slot_map(table, i32(sl, dev), i32(qsl, dev), pos, slot, n_tokens=1)
    assert slot.tolist() == [-1] + [99] * (T - 1)
