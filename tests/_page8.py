"""Inputs of the 8-bit page tests: pools of random bytes, tables, and what a result may be off by."""
import numpy as np
import torch

from oracle import page8


def pool_bytes(rng, pages, heads, page, dim, spread=2):
    """A pool of random E4M3 bytes (no NaN) with exponents around 2^-8, as uint8 arrays."""
    def block(*shape):
        x = rng.integers(0, 256, shape, dtype=np.uint8)
        x[(x & 127) == 127] = 0x33
        return x
    exps = lambda: rng.integers(119 - spread, 119 + spread + 1, (pages, heads), dtype=np.uint8)
    return block(pages, heads, page, dim), block(pages, heads, dim, page), exps(), exps()


def gpu_raw(raw):
    """The pool on the GPU, in the interleaved buffers of pool.Page8Pool."""
    from xtier_amd.pool import Page8Pool
    k, vt, ke, ve = raw
    pool = Page8Pool(k.shape[0], k.shape[2], k.shape[1], k.shape[3])
    for t, x in zip(pool.raw, raw):
        t.copy_(torch.from_numpy(x))
    return pool


def table_for(rng, lens, page, pages, width=None):
    """Every request's pages, distinct, in random order."""
    width = width or max(1, max(-(-x // page) for x in lens))
    table = np.full((len(lens), width), -1, dtype=np.int32)
    order = rng.permutation(pages)
    at = 0
    for b, x in enumerate(lens):
        n = -(-x // page)
        table[b, :n] = order[at:at + n]
        at += n
    return table


def bf16(x):
    """float64 values rounded to BF16."""
    return torch.from_numpy(np.asarray(x, dtype=np.float32)).to(torch.bfloat16)


def attention_tolerance(ref, lse, spread, score, raw, keys, dim, eps):
    """What an attention output may be off by, for every element, and its lse.

    A score is a sum of dim exact products in FP32, times a factor: off by at most (dim + 2) 2^-24 of the sum of the
    products' magnitudes; the exponential adds 2^-22 and the running sums and rescalings one rounding for each key. Each
    probability, at most 1 beside a sum of at least 1, is then rounded to FP16 (2^-11 of itself, or 2^-25), and V, at most
    448 of its scale, to steps of 2^-24 of the largest scale where its own is far smaller. The output's own rounding is half of eps."""
    delta = (dim + 4) * 2.0 ** -24 * score + 2.0 ** -22
    weight = 2 * delta + (2 * keys + 64) * 2.0 ** -24
    v_scale = 2.0 ** (float(raw[3].max()) - 127)
    tol = eps / 2 * np.abs(ref) + spread * (weight[..., None] * 1.01 + 2.0 ** -11) \
        + keys * 2.0 ** -25 * 448 * v_scale + 2.0 ** -25 * v_scale
    lse_tol = delta + (keys + 64) * 2.0 ** -24 + np.abs(np.where(np.isfinite(lse), lse, 0)) * 2.0 ** -22
    return tol, lse_tol


def attention_on_gpu(q, raw, table, page, lens, scale, cu, window=0, sinks=0):
    """The same definition as oracle.page8.attention in plain float64 torch operations on the GPU, for sizes that are too
    long on the CPU: (out, lse, spread, score) as numpy arrays. Every page is taken to exist."""
    k8, vt8, ke, ve = (torch.from_numpy(x).cuda() for x in raw)
    two_to = lambda e: ((e.long() - 127 + 1023) << 52).view(torch.float64)
    q = q.cuda().double()
    group = q.shape[1] // k8.shape[1]
    out, spread = torch.empty_like(q), torch.empty_like(q)
    lse, score = (torch.empty(q.shape[:2], dtype=torch.float64, device='cuda') for _ in range(2))
    for b, length in enumerate(lens.tolist()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        if length <= 0:
            out[lo:hi] = spread[lo:hi] = score[lo:hi] = 0
            lse[lo:hi] = -np.inf
            continue
        ids = torch.from_numpy(table[b, :-(-length // page)].astype(np.int64)).cuda()
        p = torch.arange(length - (hi - lo), length, device='cuda')
        for h in range(k8.shape[1]):
            k = (k8[ids, h].view(torch.float8_e4m3fn).double() * two_to(ke[ids, h])[:, None, None]).flatten(0, 1)[:length]
            v = (vt8[ids, h].view(torch.float8_e4m3fn).double() * two_to(ve[ids, h])[:, None, None])
            v = v.transpose(1, 2).flatten(0, 1)[:length].contiguous()
            j = torch.arange(length, device='cuda')
            seen = j <= p[:, None]
            if window:
                seen &= (j > p[:, None] - window) | (j < sinks)
            for g in range(h * group, (h + 1) * group):
                qq = q[lo:hi, g]
                z = (qq @ k.t() * scale).masked_fill(~seen, -np.inf)
                lse[lo:hi, g] = torch.logsumexp(z, 1)
                w = torch.exp(z - lse[lo:hi, g, None]).masked_fill(~seen, 0)       # (a row may see nothing)
                out[lo:hi, g], spread[lo:hi, g] = w @ v, w @ v.abs()
                score[lo:hi, g] = (qq.abs() @ k.abs().t()).masked_fill(~seen, 0).amax(1) * scale
    return tuple(x.cpu().numpy() for x in (out, lse, spread, score))


__all__ = ['attention_on_gpu', 'attention_tolerance', 'bf16', 'gpu_raw', 'page8', 'pool_bytes', 'table_for']
