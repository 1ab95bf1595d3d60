"""The first chunk attention of a process from several host threads at once."""
import subprocess
import sys

import pytest
import torch

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import threading
import torch
from amass_kv_b200.attention import ChunkBuffers, paged_chunk_attention
dev, n = torch.device("cuda", 0), 6
gen = torch.Generator(device=dev).manual_seed(1)
q = torch.randn(40, 8, 128, generator=gen, device=dev).to(torch.bfloat16)
kv = torch.randn(9, 2, 16, 2, 128, generator=gen, device=dev).to(
    torch.bfloat16)
i32 = dict(dtype=torch.int32, device=dev)
bt = torch.arange(9, **i32)[None]
sl, qsl = torch.tensor([130], **i32), torch.tensor([0, 40], **i32)
bufs = [ChunkBuffers(dev, n_kv=2, G=4, head_dim=128) for _ in range(n)]
outs = [torch.zeros_like(q) for _ in range(n)]
streams = [torch.cuda.Stream(dev) for _ in range(n)]
torch.cuda.synchronize()
gate, errors = threading.Barrier(n), []


def one(i):
    try:
        with torch.cuda.stream(streams[i]):
            gate.wait()
            paged_chunk_attention(q, kv, bt, sl, qsl, outs[i], bufs[i])
    except Exception as e:
        errors.append(e)


threads = [threading.Thread(target=one, args=(i,)) for i in range(n)]
for t in threads:
    t.start()
for t in threads:
    t.join()
torch.cuda.synchronize()
assert not errors, errors
assert bool((outs[0] != 0).any())
assert all(torch.equal(o, outs[0]) for o in outs)
for b in bufs:
    b.check()
"""


def test_threads():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
