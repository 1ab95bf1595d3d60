"""Stage B (sparse paged decode) -- host side of the sm_100a kernels.

Mirrors the reference's ``amass.attention`` surface for the hot path:

  ResidentVSource                   attention/decode.py:71-100
  ensure_stage_b_buffers(st, ...)   attention/decode.py:98-114
  sparse_paged_decode_batched_cuda  attention/decode_cuda.py:1376-1465

The split-K partials keep the reference layout (R, n_kv, split, G[, d]).
How a unit's pages are cut into partials is the kernel's own choice (equal
runs of the flat page list, one per warp of the grid, so ragged batches
balance); the reference's chunk rule pps = max(ceil(cnt/split), PPS_MIN)
(decode.py:154-160) is another cut of the same exact softmax re-association.
``pps_min`` here is the floor on pages per run.

``paged_chunk_attention`` is the prefill side: dense attention of a step's new
tokens (chunks, single tokens, mixtures) over the same cache.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import ptr

DEFAULT_SPLIT = 128


def split_kv(kv_cache: torch.Tensor):
    """(K, V) views (num_blocks, page, n_kv, d) for the vLLM cache layouts
    (nb, 2, page, n_kv, d) and (2, nb, page, n_kv, d); V is None for a K-only
    (nb, 1, ...) cache (reference attention/decode.py:59-68)."""
    if kv_cache.shape[0] == 2:
        return kv_cache[0], kv_cache[1]
    if kv_cache.shape[1] == 1:
        return kv_cache.select(1, 0), None
    return kv_cache.select(1, 0), kv_cache.select(1, 1)


class ResidentVSource:
    """AMASS-fast V source: the resident V half of the paged cache."""

    SRC_ID = 0

    def __init__(self, kv_cache: torch.Tensor):
        _, v = split_kv(kv_cache)
        if v is None:
            raise ValueError("ResidentVSource needs a resident V half; this "
                             "cache is K-only -- use a tier V source")
        self._v = v

    def args(self):
        v = self._v
        return v, v.stride(0), v.stride(1), v.stride(2)


def ensure_stage_b_buffers(st, device, split: int = DEFAULT_SPLIT) -> None:
    """Allocate the split-K partials once (outside any graph)."""
    if getattr(st, "m_part", None) is not None:
        st.split = getattr(st, "split", split)
        return
    R, n_kv, G = st.max_reqs, st.n_kv, st.G
    D = getattr(st, "D", None) or st.d
    f32 = torch.float32
    st.split = split
    st.m_part = torch.empty(R, n_kv, split, G, device=device, dtype=f32)
    st.l_part = torch.empty(R, n_kv, split, G, device=device, dtype=f32)
    st.acc_part = torch.empty(R, n_kv, split, G, D, device=device, dtype=f32)


def pps_min_for(n_req: int) -> int:
    """Floor on the pages of one warp run (the run length is otherwise the
    balanced share of the batch's selected pages).  4 for 2..16 requests
    (B200, 8 requests per GPU: 35.1 -> 34.1 us per layer-step), else 8
    (batch 1 and the 64-request batch are unchanged by it)."""
    return 4 if 2 <= n_req <= 16 else 8


def sparse_paged_decode_batched_cuda(q, kv_cache, block_table, seq_lens, st,
                                     out, vsource=None, *, scale=None,
                                     pps_min=None) -> None:
    """Stage B: split-K decode over ``st.page_table``/``st.page_cnt`` and the
    LSE merge into ``out[:n_req]`` (bf16, in place).  Same contract as the
    reference function; ``n_req = seq_lens.shape[0]``."""
    if scale is None:
        # the state's softmax scale, else 1/sqrt(head_dim)
        scale = getattr(st, "scale", None) or q.shape[-1] ** -0.5
    n_req = seq_lens.shape[0]
    k, v = split_kv(kv_cache)
    if vsource is not None:
        v = vsource.args()[0]
    if v is None:
        raise ValueError("no V source")
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or \
            out.dtype != torch.bfloat16:
        raise ValueError("q, kv_cache and out must be bf16")
    if getattr(st, "m_part", None) is None:
        raise RuntimeError("ensure_stage_b_buffers(st, ...) was not called")
    _, page, n_kv, d = k.shape
    if pps_min is None:
        pps_min = pps_min_for(n_req)
    _lib.call("amass_sparse_decode", ptr(q), q.stride(0), q.stride(1),
              ptr(k), k.stride(0), k.stride(1), k.stride(2),
              ptr(v), v.stride(0), v.stride(1), v.stride(2),
              ptr(block_table), block_table.stride(0), ptr(st.page_table),
              ptr(st.page_cnt), ptr(seq_lens), ptr(st.m_part),
              ptr(st.l_part), ptr(st.acc_part), int(st.split), int(pps_min),
              ptr(out), out.stride(0), out.stride(1), float(scale),
              int(n_req), int(n_kv), int(st.G), int(d), int(page),
              int(st.max_pages), _lib.stream_of(q.device))


sparse_paged_decode_batched = sparse_paged_decode_batched_cuda


# --------------------------------------------------------------------------- #
# attention of a chunk of new tokens (prefill, mixed batches)                 #
# --------------------------------------------------------------------------- #
DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def check_i32(index: int, name: str, t, dim: int):
    """The shape of an int32 tensor of ``dim`` dimensions on GPU ``index``
    (-1: the host) with a contiguous last one."""
    shape = t.shape
    if t.dtype is not torch.int32 or t.get_device() != index or \
            len(shape) != dim or (t.stride()[-1] != 1 and shape[-1] > 1):
        raise ValueError(f"{name} must be int32, of {dim} dimensions, on GPU "
                         f"{index} and contiguous in the last dimension; got "
                         f"{t.dtype} {tuple(shape)} on {t.device}")
    return shape


def cache_layout(kv_cache):
    """(num_blocks, page, n_kv, d, (block, token, head stride), K address, V
    address or 0) of the cache layouts of ``split_kv``, without making views;
    ValueError when it is none of them.

    A first dimension of 2 is K and V apart, as ``split_kv`` takes it: a cache
    of two blocks of both halves cannot be told from it and has to come as
    (2, 2, ...) with K first.  (2, 1, ...) could be two blocks of keys only or
    one block of both, and is refused."""
    shape, s = kv_cache.shape, kv_cache.stride()
    if len(shape) != 5 or (s[4] != 1 and shape[4] > 1) or \
            (shape[0] != 2 and not 1 <= shape[1] <= 2):
        raise ValueError("kv_cache must be (blocks, 1 or 2, page, n_kv, d) or "
                         "(2, blocks, page, n_kv, d) with a contiguous "
                         f"head_dim, got {tuple(shape)}")
    n0, n1, page, n_kv, d = shape
    s0, s1, st, sh, _ = s
    if not (n0 and n1 and page and n_kv and d):
        raise ValueError(f"kv_cache {tuple(shape)} is empty")
    p = kv_cache.data_ptr()
    if n0 != 2:
        v = 0 if n1 == 1 else p + s1 * kv_cache.element_size()
        return n0, page, n_kv, d, (s0, st, sh), p, v
    if n1 == 1:
        raise ValueError(f"kv_cache {tuple(shape)} may be two blocks of keys "
                         "or one block of keys and values: give it another "
                         "block")
    return (n1, page, n_kv, d, (s1, st, sh), p,
            p + s0 * kv_cache.element_size())


class ChunkBuffers(_lib.FixedBuffers):
    """Scratch of ``paged_chunk_attention`` for one head geometry, allocated
    once (outside any graph): the fp32 partials of the rows that two or more
    SMs share.  Calls that may overlap on the GPU -- other streams, two
    captured graphs replayed at once -- need a ``ChunkBuffers`` each.

    ``fault`` (1,) int32 latches 1 when a kernel gave up a bounded wait;
    ``check()`` reads it (synchronises) and raises: the buffers are then to be
    replaced."""

    def __init__(self, device, *, n_kv: int, G: int, head_dim: int):
        if head_dim not in (64, 128) or not 1 <= G <= 8 or n_kv < 1:
            raise ValueError(f"no kernel for head_dim {head_dim}, G {G}, "
                             f"n_kv {n_kv}")
        dev = _lib.device_of(device)
        self.device, self.n_kv, self.G, self.d = dev, n_kv, G, head_dim
        self.index = dev.index
        n = torch.cuda.get_device_properties(dev).multi_processor_count
        self.n_ctas = n
        f32 = torch.float32
        self.acc_part = torch.empty(n, 2, head_dim // 4, 256, 4, device=dev,
                                    dtype=f32)
        self.ml_part = torch.empty(n, 2, 256, 2, device=dev, dtype=f32)
        self.tickets = torch.zeros(n, 8, device=dev, dtype=torch.int32)
        self.fault = torch.zeros(1, device=dev, dtype=torch.int32)
        self.scratch = (ptr(self.acc_part), ptr(self.ml_part),
                        ptr(self.tickets), ptr(self.fault))
        self._fixed = True

    def check(self) -> None:
        if int(self.fault.item()):
            raise RuntimeError("paged_chunk_attention: a kernel gave up a "
                               "bounded wait; its outputs are incomplete")


def paged_chunk_attention(q, kv_cache, block_table, seq_lens, query_start_loc,
                          out, buf, *, scale=None, window=None, lse=None,
                          vsource=None, status=None) -> None:
    """Dense attention of the step's new tokens over the paged cache, which
    already holds their keys and values.

    q, out (T, H, d) bf16 or fp16 (the cache's type), H = n_kv * G; rows
    query_start_loc[r] .. query_start_loc[r + 1] - 1 are the last tokens of
    request r's ``seq_lens[r]``; a row at position p sees the keys
    max(0, p - window + 1) .. p (``window=None``: from 0).  Rows without a
    key (or with nothing but scores of -inf) become 0, rows outside every
    request are left as they are; a request's tokens from the T-th row of the
    step on count as not there.  ``lse`` (T, H) fp32, contiguous, receives
    the rows' natural log-sum-exp (-inf without a key).
    ``n_req = seq_lens.shape[0]``; ``buf`` is a ``ChunkBuffers``; ``out`` may
    be ``q``.

    ``status``: that of a ``BlockPool`` whose step may have been refused in
    part.  A refused request's length is without its new tokens, so they would
    be taken for its last old ones; with ``status`` they become 0 (lse -inf).

    Cache slots behind a request's last token, or before the windows of all
    its rows, may hold anything.  Between the two, a score of NaN or +inf (a
    NaN or infinite key) makes its row NaN, one of -inf drops the key from its
    row; a NaN or infinite value reaches the rows that see it, and may make
    other rows of the same request NaN.  Block ids outside the cache read as
    zeros.  One launch, no allocation, no synchronisation."""
    nb, page, n_kv, d, strides, k, v = cache_layout(kv_cache)
    k_sb, k_st, k_sh = v_sb, v_st, v_sh = strides
    dtype, dev = q.dtype, buf.index
    if vsource is not None:
        vt = vsource.args()[0]
        if tuple(vt.shape) != (nb, page, n_kv, d) or vt.dtype != dtype or \
                vt.get_device() != dev or vt.stride(3) != 1:
            raise ValueError(f"the V source's {tuple(vt.shape)} {vt.dtype} "
                             "does not match K")
        v, (v_sb, v_st, v_sh, _) = vt.data_ptr(), vt.stride()
        strides += (v_sb, v_st, v_sh)
    if not v:
        raise ValueError("no V source")
    shape = q.shape
    if len(shape) != 3 or out.shape != shape:
        raise ValueError("q and out must be (T, H, d) of the same shape")
    type_id = DTYPES.get(dtype)
    if type_id is None or kv_cache.dtype is not dtype or \
            out.dtype is not dtype:
        raise ValueError("q, kv_cache and out must all be bf16 or all fp16")
    T, H, dq = shape
    if dq != d or H != n_kv * buf.G or d != buf.d or n_kv != buf.n_kv:
        raise ValueError(f"q {tuple(shape)} and a cache of {n_kv} heads of "
                         f"{d} do not fit buffers for {buf.n_kv} x {buf.G} "
                         f"heads of {buf.d}")
    q_st, q_sh, q_sd = q.stride()
    o_st, o_sh, o_sd = out.stride()
    if q_sd != 1 or o_sd != 1:
        raise ValueError("q and out must have a contiguous head_dim")
    if q.get_device() != dev or out.get_device() != dev or \
            kv_cache.get_device() != dev:
        raise ValueError(f"q, kv_cache and out must be on GPU {dev}")
    qp, op = q.data_ptr(), out.data_ptr()
    if T > 1:
        strides += (q_st, o_st)
    if H > 1:
        strides += (q_sh, o_sh)
    every = 0
    for s in strides:
        every |= s if s > 0 else 1
    if (qp | op | k | v) & 15 or every & 7:
        raise ValueError("q, kv_cache and out must be 16-byte aligned, with "
                         "strides that are positive multiples of 8 elements")
    if n_kv > 1 and nb > 1 and (
            k_sb % k_sh or v_sb % v_sh or k_sb // k_sh != v_sb // v_sh or
            k_sb < n_kv * k_sh):
        raise ValueError("kv_cache needs block strides that are multiples of "
                         "the head strides, the same for K and V")
    rows, max_pages = check_i32(dev, "block_table", block_table, 2)
    n_req, = check_i32(dev, "seq_lens", seq_lens, 1)
    starts, = check_i32(dev, "query_start_loc", query_start_loc, 1)
    if rows < n_req or starts <= n_req or max_pages < 1:
        raise ValueError(f"block_table {(rows, max_pages)} and "
                         f"query_start_loc {tuple(query_start_loc.shape)} do "
                         f"not cover {n_req} requests")
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if lse is not None and (lse.dtype != torch.float32 or
                            lse.get_device() != dev or
                            tuple(lse.shape) != (T, H) or
                            not lse.is_contiguous()):
        raise ValueError(f"lse must be a contiguous fp32 ({T}, {H}) tensor")
    if status is not None and \
            check_i32(dev, "status", status, 1)[0] < n_req:
        raise ValueError(f"status {tuple(status.shape)} does not cover "
                         f"{n_req} requests")
    if scale is None:
        scale = d ** -0.5
    if not 0 < scale < float("inf"):
        raise ValueError(f"scale must be positive, got {scale}")
    if T == 0 or n_req == 0:
        return
    args = _lib.CHUNK.pack(
        qp, k, v, block_table.data_ptr(), seq_lens.data_ptr(),
        query_start_loc.data_ptr(), *buf.scratch, op,
        0 if lse is None else lse.data_ptr(), q_st, q_sh, k_sb, k_st, k_sh,
        v_sb, v_st, v_sh, block_table.stride(0), o_st, o_sh, scale, nb,
        buf.n_ctas, min(window, 0x7fffffff) if window else 0, T, n_req, n_kv,
        buf.G, d, page, max_pages, type_id)
    if status is None:
        _lib.launch(dev, "amass_paged_chunk", args)
    else:
        _lib.launch(dev, "amass_paged_chunk_granted", args,
                    status.data_ptr())
