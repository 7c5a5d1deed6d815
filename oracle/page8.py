"""The 8-bit paged cache and its page tables, restated on the CPU in 64 bits: E4M3 blocks with one power-of-two scale for
each page and head, attention over them, and the bookkeeping of pages. numpy, one step at a time."""
import math

import numpy as np

E_MIN, E_MAX = 63, 246


def e4m3_values():
    """The 256 E4M3 (fn) values; 0x7F and 0xFF are NaN."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    mag = np.where(e > 0, 2.0 ** (e - 7.0) * (1 + m / 8), m * 2.0 ** -9)
    mag[(b & 127) == 127] = np.nan
    return np.where(b & 128, -mag, mag)


def e4m3_bytes(x):
    """Bytes of the nearest E4M3 values (ties to the even mantissa); beyond 448 the largest, NaN as 0x7F."""
    x = np.asarray(x, dtype=np.float64)
    mag = np.minimum(np.abs(x), 448.0)
    with np.errstate(invalid='ignore', divide='ignore'):
        e = np.floor(np.log2(np.where(mag > 0, mag, 1.0)))
    e = np.maximum(np.where(mag >= 2.0 ** (e + 1), e + 1, np.where(mag < 2.0 ** e, e - 1, e)), -6)
    step = 2.0 ** (e - 3)
    mag = np.rint(np.where(np.isnan(mag), 0, mag) / step) * step       # rint: halves to even
    grid = e4m3_values()[:127]
    code = np.searchsorted(grid, mag).astype(np.uint8)
    code = np.where(np.isnan(x), 127, code).astype(np.uint8)
    return code | np.where(np.signbit(x), 128, 0).astype(np.uint8)


def exponent_for(amax):
    """The smallest e with amax <= 448 * 2^(e - 127), within 63..246."""
    e = E_MIN
    while e < E_MAX and amax > 448.0 * 2.0 ** (e - 127):
        e += 1
    return e


def append(k, v, raw, table, page_size, seq_lens, cu=None):
    """xt_page8_append on float64 copies of the rows and uint8 arrays k [pages, heads, page, dim], vt [pages, heads, dim,
    page], k_exp, v_exp [pages, heads], changed in place."""
    vals = e4m3_values()
    blocks = (raw[0], raw[1].transpose(0, 1, 3, 2))     # the V block by token, a view
    batch, width = table.shape
    cu = np.arange(batch + 1) if cu is None else cu
    for b in range(batch):
        n = int(cu[b + 1] - cu[b])
        start = max(int(seq_lens[b]), 0) - n
        for col in range(max(start, 0) // page_size, -(-max(int(seq_lens[b]), 0) // page_size)):
            lo, hi = max(start, 0, col * page_size), min(int(seq_lens[b]), (col + 1) * page_size)
            if col >= width or lo >= hi or not 0 <= table[b, col] < raw[0].shape[0]:
                continue
            page, t0 = int(table[b, col]), lo - col * page_size
            rows = slice(int(cu[b]) + lo - start, int(cu[b]) + hi - start)
            for x, block, exps in ((k, blocks[0], raw[2]), (v, blocks[1], raw[3])):
                for h in range(x.shape[1]):
                    new = np.asarray(x[rows, h], dtype=np.float64)
                    finite = np.abs(new[np.isfinite(new)])
                    e0 = int(exps[page, h]) if t0 else 0
                    e = max(exponent_for(finite.max() if finite.size else 0.0), e0)
                    if t0 and e > e0:
                        block[page, h, :t0] = e4m3_bytes(vals[block[page, h, :t0]] * 2.0 ** (e0 - e))
                    block[page, h, t0:t0 + hi - lo] = e4m3_bytes(new * 2.0 ** (127 - e))
                    exps[page, h] = e


def visible(j, p, window, sinks):
    return j <= p and (window <= 0 or j > p - window or j < sinks)


def attention(q, raw, table, page_size, seq_lens, scale, cu=None, window=0, sinks=0):
    """xt_page8_attention in float64: (out [rows, q_heads, dim], lse [rows, q_heads], spread) with spread [rows, q_heads,
    dim] = sum_j p_j |v_j| and score [rows, q_heads] = max_j sum_d |q_d k_jd| * scale over the visible keys, for
    tolerances. Rows of no request are NaN."""
    vals = e4m3_values()
    k8, vt8, k_exp, v_exp = raw
    rows, q_heads, dim = q.shape
    group = q_heads // k8.shape[1]
    batch, width = table.shape
    cu = np.arange(batch + 1) if cu is None else cu
    out, spread = np.full(q.shape, np.nan), np.zeros(q.shape)
    lse, score = np.full((rows, q_heads), np.nan), np.zeros((rows, q_heads))
    for b in range(batch):
        n = int(cu[b + 1] - cu[b])
        start = max(int(seq_lens[b]), 0) - n
        for i in range(n):
            p = start + i
            keys = [j for j in range(min(p + 1, width * page_size)) if visible(j, p, window, sinks)
                    and 0 <= table[b, j // page_size] < k8.shape[0]]
            r = int(cu[b]) + i
            if not keys:
                out[r], lse[r] = 0.0, -np.inf
                continue
            keys = np.array(keys)
            page, t = table[b, keys // page_size], keys % page_size
            for h in range(q_heads):
                g = h // group
                ks = vals[k8[page, g, t]] * 2.0 ** (k_exp[page, g].astype(np.float64) - 127)[:, None]
                vs = vals[vt8[page, g, :, t]] * 2.0 ** (v_exp[page, g].astype(np.float64) - 127)[:, None]
                z = ks @ q[r, h] * scale
                top = z.max()
                w = np.exp(z - top)
                out[r, h] = w @ vs / w.sum()
                lse[r, h] = top + math.log(w.sum()) if np.isfinite(top) else np.nan
                spread[r, h] = w @ np.abs(vs) / w.sum()
                score[r, h] = (np.abs(ks) @ np.abs(q[r, h])).max() * scale
    return out, lse, spread, score


# --- pages ----------------------------------------------------------------------------------------------------------

def _free(refs):
    return [p for p in range(len(refs)) if refs[p] == 0]


def extend(refs, table, lens, add, page_size):
    free, asked = _free(refs), 0
    granted = np.zeros(len(lens), dtype=bool)
    for b in range(len(lens)):
        c0, c1 = -(-int(lens[b]) // page_size), -(-(int(lens[b]) + int(add[b])) // page_size)
        if add[b] < 0 or lens[b] < 0 or c1 > table.shape[1]:
            continue
        need, asked = c1 - c0, asked + c1 - c0
        if need and asked > len(free):
            continue
        for c in range(c0, c1):
            p = free[asked - need + c - c0]
            table[b, c], refs[p] = p, 1
        lens[b] += add[b]
        granted[b] = True
    return granted


def fork(refs, table, lens, parents, children, page_size):
    rows, width = table.shape
    free, before, old = _free(refs), lens.copy(), table.copy()
    moves = np.full((2, len(parents)), -1, dtype=np.int32)
    taken, seen = 0, set()
    for i, (p, c) in enumerate(zip(parents.tolist(), children.tolist())):
        first = c not in seen
        seen.add(c)
        if not (0 <= p < rows and 0 <= c < rows) or before[c] != 0 or not first:
            continue
        full, rest = divmod(int(before[p]), page_size)
        table[c] = -1
        table[c, :full] = old[p, :full]
        for x in old[p, :full]:
            if 0 <= x < len(refs):
                refs[x] += 1
        lens[c] = before[p]
        if rest:
            if taken < len(free):
                moves[:, i] = old[p, full], free[taken]
                table[c, full], refs[free[taken]] = free[taken], 1
            else:
                lens[c] = full * page_size
            taken += 1
    return moves


def free(refs, table, lens, rows):
    for r in sorted(set(rows.tolist())):
        if 0 <= r < len(lens):
            for p in table[r]:
                if 0 <= p < len(refs):
                    refs[p] -= 1
            table[r], lens[r] = -1, 0


def compact(refs, table):
    n = len(refs)
    live = int((refs > 0).sum())
    src = [p for p in range(live, n) if refs[p] > 0]
    dst = [p for p in range(live) if refs[p] <= 0]
    moves = np.full((2, n // 2), -1, dtype=np.int32)
    moves[0, :len(src)], moves[1, :len(dst)] = src, dst
    to = dict(zip(src, dst))
    for cell in np.ndindex(table.shape):
        table[cell] = to.get(int(table[cell]), int(table[cell]))
    for a, b in to.items():
        refs[b], refs[a] = refs[a], 0
    return moves, len(src)
