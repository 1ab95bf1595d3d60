"""fp64 reference of the chunk attention and its error bound."""
import torch


def chunk_reference(q, k, v, block_table, lens, starts, scale, window=None):
    """out, lse in fp64 and the per-element bound on the kernel's error.

    Bound of out.  u = half a step of the 16-bit type, e = 2^-24.  The
    softmax weights P (relative to the running maximum) are rounded once:
    u sum w|v|.  A score is an fp32 sum of d exact products: off by at most
    d e sum|q k| scale (absolute, so relative in the weight, numerator and
    denominator: twice); the exponential adds 2^-21 (2^-22 and its argument's
    rounding at |x| <= 64), fp32 sums over n keys at most n e.  The result is
    rounded once: u |o|.  Weights below the type's normal range (fp16) lose
    at most 2^-25 each: n 2^-25 max|v|."""
    T, H, d = q.shape
    n_kv = k.shape[2]
    G = H // n_kv
    page = k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    e = 2.0 ** -24
    out = torch.zeros(T, H, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((T, H), float("-inf"), dtype=torch.float64,
                     device=q.device)
    tol_l = torch.zeros_like(lse)
    rows = torch.zeros(T, dtype=torch.bool, device=q.device)
    for r, (new, n) in enumerate(lens):
        t0 = starts[r]
        rows[t0:t0 + new] = True
        if n <= 0 or new <= 0:
            continue
        tok = torch.arange(n, device=q.device)
        blk = block_table[r, tok // page].long()
        kk = k[blk, tok % page].double()                  # (n, n_kv, d)
        vv = v[blk, tok % page].double()
        p = torch.arange(n - new, n, device=q.device)
        see = tok[None] <= p[:, None]
        if window:
            see = see & (tok[None] > p[:, None] - window)
        for h in range(H):
            qh, kh, vh = q[t0:t0 + new, h].double(), kk[:, h // G], \
                vv[:, h // G]
            s = (qh @ kh.t() * scale).masked_fill(~see, float("-inf"))
            z = torch.logsumexp(s, -1)
            w = torch.exp(s - z[:, None]).nan_to_num(0.0)  # empty rows
            o = w @ vh
            a = w @ vh.abs()
            ds = d * e * scale * (qh.abs() @ kh.abs().t()).masked_fill(
                ~see, 0.0).amax(-1, keepdim=True)
            err = u * a + (2 * ds + 2.0 ** -20 + 2 * n * e) * a + u * o.abs()
            if q.dtype == torch.float16:
                err = err + n * 2.0 ** -25 * vh.abs().amax()
            out[t0:t0 + new, h] = o
            tol[t0:t0 + new, h] = err + 1e-30
            lse[t0:t0 + new, h] = z
            tol_l[t0:t0 + new, h] = (ds[:, 0] + 2.0 ** -20 + n * e
                                     + 4 * e * z.abs().nan_to_num(
                                         posinf=0.0))
    return out, tol, lse, tol_l, rows
