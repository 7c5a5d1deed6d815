"""The 8-bit paged cache as timed cases: the append that quantizes new keys and values with one power-of-two scale for
each page and head, the attention that reads such pages (decode, verification, prompt chunks; whole contexts, or a
sliding window with a few first tokens that stay visible), and the operators that keep the pages of every layer
(growing, forking, freeing, compacting and copying them).

Heads, dims, contexts and page sizes are those of the package's workloads (xtier_amd/workloads.py, bench.py), with
smaller, ragged and odd ones among the drawn cases. prepare() builds what a serving program holds before a call: the
pools, page tables, lengths and activations. run() is one pass, in plain torch operations or, where `own` is true,
through xtier_amd.ops. exact() is the definition in 64 bits.
"""
import math

import torch

own = False

DEV = 'cuda'
E_MIN, E_MAX = 63, 246       # the scale exponents an append writes (biased by 127)


def listed():
    return [
        # every layer of every decode step: one new token of each of 32 requests
        {'name': 'append_decode', 'path': 'append', 'batch': 32, 'rows': 1, 'ctx': 4096, 'kv_heads': 4, 'dim': 128,
         'page': 64, 'ragged': False},
        # prompts of differing lengths in one step, small pages, wide heads
        {'name': 'append_ragged', 'path': 'append', 'batch': 24, 'rows': 300, 'ctx': 2500, 'kv_heads': 2, 'dim': 256,
         'page': 16, 'ragged': True},
        # a chunk of a long prompt
        {'name': 'append_chunk', 'path': 'append', 'batch': 1, 'rows': 4096, 'ctx': 32768, 'kv_heads': 4, 'dim': 128,
         'page': 64, 'ragged': False},
        # one chat request: the latency of every layer of every token
        {'name': 'decode_one', 'path': 'attend', 'batch': 1, 'rows': 1, 'ctx': 4099, 'q_heads': 16, 'kv_heads': 2,
         'dim': 256, 'page': 16, 'window': 0, 'sinks': 0, 'ragged': False},
        # a full decode batch at 32K context
        {'name': 'decode_batch', 'path': 'attend', 'batch': 32, 'rows': 1, 'ctx': 32768, 'q_heads': 32, 'kv_heads': 4,
         'dim': 128, 'page': 64, 'window': 0, 'sinks': 0, 'ragged': False},
        # two documents of half a million tokens, of differing lengths
        {'name': 'decode_long', 'path': 'attend', 'batch': 2, 'rows': 1, 'ctx': 524288, 'q_heads': 32, 'kv_heads': 4,
         'dim': 128, 'page': 64, 'window': 0, 'sinks': 0, 'ragged': True},
        # a layer with a sliding window: 64 requests of differing lengths, pages behind the window already freed
        {'name': 'decode_window', 'path': 'attend', 'batch': 64, 'rows': 1, 'ctx': 32768, 'q_heads': 40, 'kv_heads': 8,
         'dim': 128, 'page': 32, 'window': 4096, 'sinks': 4, 'ragged': True},
        # verification of four drafted tokens of each request
        {'name': 'verify', 'path': 'attend', 'batch': 16, 'rows': 4, 'ctx': 16384, 'q_heads': 64, 'kv_heads': 4,
         'dim': 128, 'page': 64, 'window': 0, 'sinks': 0, 'ragged': False},
        # a chunk of a long prompt
        {'name': 'prefill_chunk', 'path': 'attend', 'batch': 1, 'rows': 4096, 'ctx': 32768, 'q_heads': 32,
         'kv_heads': 4, 'dim': 128, 'page': 64, 'window': 0, 'sinks': 0, 'ragged': False},
        # several prompts through a layer with a sliding window
        {'name': 'prefill_window', 'path': 'attend', 'batch': 5, 'rows': 2048, 'ctx': 8192, 'q_heads': 16,
         'kv_heads': 4, 'dim': 64, 'page': 64, 'window': 1000, 'sinks': 16, 'ragged': True},
        # a search step: every beam forked, its unfinished page copied in every layer, the losers freed
        {'name': 'pages_fork', 'path': 'fork', 'rows': 64, 'forks': 32, 'ctx': 4096, 'page': 64, 'pages': 2048,
         'layers': 12, 'bytes': 65536},
        # the end of a busy minute: half the requests freed, the rest grown, the pool compacted in every layer
        {'name': 'pages_compact', 'path': 'compact', 'rows': 96, 'ctx': 2048, 'page': 64, 'pages': 2500, 'layers': 8,
         'bytes': 65536},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    path = rng.choice(['append', 'append', 'attend', 'attend', 'attend', 'attend', 'fork', 'compact'])
    if path == 'append':
        rows = rng.choice([1, 1, _spread(rng, 2, 4096)])
        batch = _spread(rng, 1, 64 if rows == 1 else max(1, 4096 // rows))
        return {'path': path, 'batch': batch, 'rows': rows, 'ctx': rows + _spread(rng, 1, 4096),
                'kv_heads': rng.choice([1, 2, 4, 8]), 'dim': rng.choice([64, 128, 256]),
                'page': rng.choice([16, 32, 64, 128]), 'ragged': rng.random() < 0.7}
    if path == 'attend':
        q_heads, kv_heads, dim = rng.choice([(32, 4, 128), (8, 1, 128), (16, 2, 256), (32, 2, 256), (16, 4, 64),
                                             (40, 8, 128), (64, 4, 128), (4, 4, 128)])
        kind = rng.choice(['decode', 'decode', 'verify', 'prefill'])
        if kind == 'prefill':
            rows = _spread(rng, 40, 4096)
            batch = _spread(rng, 1, max(1, 4096 // rows))
            ctx = rows + _spread(rng, 1, 28672 * 4096 // max(4096, q_heads * dim) // batch)
        else:
            rows = 1 if kind == 'decode' else rng.randint(2, 8)
            batch = _spread(rng, 1, 64)
            ctx = rows + _spread(rng, 1, min(200000, (1 << 19) // batch))
        window = rng.choice([0, 0, _spread(rng, 100, 8192)])
        return {'path': path, 'batch': batch, 'rows': rows, 'ctx': ctx, 'q_heads': q_heads, 'kv_heads': kv_heads,
                'dim': dim, 'page': rng.choice([16, 32, 64, 128]), 'window': window,
                'sinks': rng.choice([0, 1, 4, 70]) if window else 0, 'ragged': rng.random() < 0.7}
    page = rng.choice([16, 32, 64, 128])
    ctx = _spread(rng, 100, 4096)
    rows = _spread(rng, 6, 64)
    pages = rows * -(-ctx // page) + 64
    case = {'path': path, 'rows': rows, 'ctx': ctx, 'page': page, 'pages': pages, 'layers': rng.randint(1, 12),
            'bytes': page * rng.choice([256, 512, 1024])}
    case['layers'] = max(1, min(case['layers'], (1 << 30) // (pages * case['bytes'])))
    if path == 'fork':
        case['forks'] = rng.randint(1, rows // 2)
    return case


# --- inputs ---------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _exponent(amax):
    """The biased exponent of the smallest power of two s with amax / s <= 448, kept within the written range."""
    m, e = torch.frexp(amax)                        # amax = m * 2^e, m in [0.5, 1)
    byte = e - 9 + (m > 0.875).to(e.dtype) + 127    # 448 = 0.875 * 2^9
    return torch.where(amax > 0, byte, torch.zeros_like(byte)).clamp(E_MIN, E_MAX)


def _to_e4m3(x):
    """E4M3 bytes of FP32 values, to nearest even; above 448 the largest value, NaN kept."""
    return torch.where(x.abs() > 448, torch.sign(x) * 448, x).to(torch.float8_e4m3fn).view(torch.uint8)


def _pow2(byte):
    return (byte.to(torch.int32).clamp(0, 254) << 23).view(torch.float32)


def _activations(shape, channels, g):
    """Normal values, with one channel in a hundred (along the axis `channels`) eight times as large."""
    x = torch.randn(*shape, generator=g, device=DEV)
    n = shape[channels]
    big = torch.where(torch.rand(n, generator=g, device=DEV) < 0.01, 8.0, 1.0)
    return x.mul_(big.view([-1 if i == channels % len(shape) else 1 for i in range(len(shape))])).to(torch.bfloat16)


def _pool(pages, heads, page, dim, g):
    """One layer's pool: per page and head the K block [page, dim] and the transposed V block [dim, page], E4M3 bytes,
    with the exponents of their scales."""
    buf = torch.empty(pages, heads, 2, page * dim, dtype=torch.uint8, device=DEV)
    exps = torch.empty(pages, heads, 2, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // (heads * page * dim))
    for lo in range(0, pages, step):
        n = min(step, pages - lo)
        for which, shape, channels in ((0, (n, heads, page, dim), 3), (1, (n, heads, dim, page), 2)):
            x = _activations(shape, channels, g).float()
            e = _exponent(x.abs().amax((2, 3)))
            buf[lo:lo + n, :, which] = _to_e4m3(x / _pow2(e)[:, :, None, None]).flatten(2)
            exps[lo:lo + n, :, which] = e.to(torch.uint8)
    k = buf[:, :, 0].unflatten(2, (page, dim))
    vt = buf[:, :, 1].unflatten(2, (dim, page))
    return k, vt, exps[..., 0], exps[..., 1]


def _lengths(case, seed):
    """(context lengths with the new rows, new rows) of each request, as host lists: the seed orders the requests of
    one set of lengths, so that every seed has the same number of rows and pages."""
    g = torch.Generator().manual_seed(case['ctx'])
    b, rows, ctx = case['batch'], case['rows'], case['ctx']
    if not case['ragged']:
        return [ctx] * b, [rows] * b
    n = [max(1, int(rows * (0.1 + 0.9 * f))) for f in torch.rand(b, generator=g).tolist()]
    old = [int((ctx - rows) * f) for f in torch.rand(b, generator=g).tolist()]
    if b == 1:
        old = [ctx - rows]
    order = torch.randperm(b, generator=torch.Generator().manual_seed(seed + 1)).tolist()
    return [old[i] + n[i] for i in order], [n[i] for i in order]


def _visible_from(case, length, n):
    """The lowest position of the window of a request's first new row (0 without a window)."""
    return max(0, length - n - case['window'] + 1) if case['window'] else 0


def prepare(case, seed):
    g = _gen(seed)
    if case['path'] in ('fork', 'compact'):
        return _prepare_pages(case, seed, g)
    lens, n = _lengths(case, seed)
    page, heads, dim = case['page'], case['kv_heads'], case['dim']
    width = max(-(-x // page) for x in lens)
    # the table: pages in random order; what a window has left behind is freed (-1)
    held = torch.zeros(len(lens), width, dtype=torch.bool)
    for b, (x, m) in enumerate(zip(lens, n)):
        held[b, :-(-x // page)] = True
        if case.get('window'):
            held[b, -(-case['sinks'] // page):_visible_from(case, x, m) // page] = False
    pages = int(held.sum()) + 3
    table = torch.full(held.shape, -1, dtype=torch.int32)
    table[held] = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 2))[:int(held.sum())].int()
    cu = [0]
    for m in n:
        cu.append(cu[-1] + m)
    state = {'case': case, 'lens_host': lens, 'rows_host': n, 'raw': _pool(pages, heads, page, dim, g),
             'table': table.to(DEV), 'lens': torch.tensor(lens, dtype=torch.int32, device=DEV),
             'cu': torch.tensor(cu, dtype=torch.int32, device=DEV) if max(n) > 1 else None}
    if case['path'] == 'append':
        state['k'] = _activations((cu[-1], heads, dim), 2, g)
        state['v'] = _activations((cu[-1], heads, dim), 2, g)
    else:
        state['q'] = (torch.randn(cu[-1], case['q_heads'], dim, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
        state['scale'] = 1 / math.sqrt(dim)
    return state


def _prepare_pages(case, seed, g):
    """Reference counts, a page table with random contexts in half (fork) or most of its rows, and the page buffers of
    every layer."""
    rows, page, pages = case['rows'], case['page'], case['pages']
    h = torch.Generator().manual_seed(seed + 1)
    width = -(-case['ctx'] // page) + 2
    live = rows // 2 if case['path'] == 'fork' else rows - rows // 8
    lens = torch.zeros(rows, dtype=torch.int32)
    lens[:live] = (case['ctx'] * (0.1 + 0.9 * torch.rand(live, generator=h))).int()
    used = -(-lens // page)
    order = torch.randperm(pages, generator=h).int()
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for b in range(live):
        table[b, :used[b]] = order[at:at + int(used[b])]
        at += int(used[b])
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    state = {'case': case, 'lens': lens.to(DEV), 'table': table.to(DEV), 'refs': refs.to(DEV),
             'data': torch.randint(0, 256, (case['layers'], pages, case['bytes']), generator=g, device=DEV,
                                   dtype=torch.uint8)}
    if own:
        from xtier_amd import ops
        state['buffers'] = ops.PageBuffers(list(state['data']))      # a server makes this once
    if case['path'] == 'fork':
        state['parents'] = torch.randint(0, live, (case['forks'],), generator=h, dtype=torch.int32).to(DEV)
        state['children'] = (live + torch.randperm(rows - live, generator=h)[:case['forks']]).int().to(DEV)
    else:
        state['ended'] = torch.randperm(live, generator=h)[:live // 2].int().to(DEV)
        add = torch.randint(0, page + 1, (rows,), generator=h, dtype=torch.int32)
        add[lens == 0] = 0
        state['add'] = add.to(DEV)
        state['start'] = {x: state[x].clone() for x in ('refs', 'table', 'lens')}
    return state


# --- the operators --------------------------------------------------------------------------------------------------

def run(state):
    return {'append': _run_append, 'attend': _run_attend, 'fork': _run_fork,
            'compact': _run_compact}[state['case']['path']](state)


def _run_append(s):
    if own:
        from xtier_amd import ops
        ops.page8_append(s['k'], s['v'], s['raw'], s['table'], s['lens'], s['cu'])
    else:
        _plain_append(s['k'], s['v'], s['raw'], s['table'], s['lens'], s['cu'], max(s['rows_host']))
    k, vt, ke, ve = s['raw']
    return [k.view(torch.float8_e4m3fn), vt.view(torch.float8_e4m3fn), ke, ve]


def _run_attend(s):
    c = s['case']
    if own:
        from xtier_amd import ops
        lse = torch.empty(s['q'].shape[:2], dtype=torch.float32, device=s['q'].device)
        out = ops.page8_attention(s['q'], s['raw'], s['table'], s['lens'], s['scale'], cu_q=s['cu'],
                                  window=c['window'], sinks=c['sinks'], lse=lse)
        return [out, lse]
    return _plain_attend(s)


def _run_fork(s):
    c = s['case']
    if own:
        from xtier_amd import ops
        moves = ops.pages_fork(s['refs'], s['table'], s['lens'], s['parents'], s['children'], c['page'])
        ops.pages_copy(s['buffers'], moves)
        forked = s['table'][s['children'].long()]
        ops.pages_free(s['refs'], s['table'], s['lens'], s['children'])
    else:
        moves = _plain_fork(s['refs'], s['table'], s['lens'], s['parents'], s['children'], c['page'])
        _plain_copy(s['data'], moves)
        forked = s['table'][s['children'].long()]
        _plain_free(s['refs'], s['table'], s['lens'], s['children'])
    return [moves, forked, s['refs'], s['table'], s['lens'], s['data']]


def _run_compact(s):
    c = s['case']
    for x, t in s['start'].items():      # every pass finds the same busy pool
        s[x].copy_(t)
    if own:
        from xtier_amd import ops
        ops.pages_free(s['refs'], s['table'], s['lens'], s['ended'])
        granted = ops.pages_extend(s['refs'], s['table'], s['lens'], s['add'], c['page'])
        moves, count = ops.pages_compact(s['refs'], s['table'])
        ops.pages_copy(s['buffers'], moves, count)
    else:
        _plain_free(s['refs'], s['table'], s['lens'], s['ended'])
        granted = _plain_extend(s['refs'], s['table'], s['lens'], s['add'], c['page'])
        moves, count = _plain_compact(s['refs'], s['table'])
        _plain_copy(s['data'], moves)
    return [granted, moves, count, s['refs'], s['table'], s['lens'], s['data']]


# --- plain forms ----------------------------------------------------------------------------------------------------

def _plain_append(k, v, raw, table, lens, cu, most):
    """Row i of request b goes to position lens[b] - n_b + i. A page and head that takes rows keeps its scale where
    that covers them, else its exponent grows and its earlier rows are rounded again; a page that takes its first row
    starts anew."""
    pages, heads, page, dim = raw[0].shape
    batch, width = table.shape
    if cu is None:
        cu = torch.arange(batch + 1, device=k.device)
    n = cu[1:] - cu[:-1]
    first = lens - n
    cols = first[:, None] // page + torch.arange(-(-most // page) + 1, device=k.device)       # [batch, touched pages]
    pos = cols[..., None] * page + torch.arange(page, device=k.device)                        # [batch, touched, page]
    new = (pos >= first[:, None, None]) & (pos < lens[:, None, None])
    take = new.any(-1) & (cols < width)
    row = (cu[:-1, None, None] + pos - first[:, None, None])[take].clamp(0, k.shape[0] - 1)   # [m, page]
    ids = table.gather(1, cols.clamp(0, width - 1).long())[take].long()
    new = new[take]                                                                           # [m, page]
    began = new[:, 0]
    t0 = new.int().argmax(-1)
    old = torch.arange(page, device=k.device) < t0[:, None]
    for x, blocks, exps, transposed in ((k, raw[0], raw[2], False), (v, raw[1], raw[3], True)):
        val = x[row].float().transpose(1, 2)                                                  # [m, heads, page, dim]
        here = new[:, None, :, None]
        mag = torch.where(here & torch.isfinite(val), val.abs(), torch.zeros_like(val)).amax((2, 3))
        e0 = torch.where(began[:, None], 0, exps[ids].int())
        e = torch.maximum(_exponent(mag), e0)
        was = blocks[ids].transpose(2, 3) if transposed else blocks[ids]
        fresh = _to_e4m3(val / _pow2(e)[:, :, None, None])
        again = _to_e4m3(was.view(torch.float8_e4m3fn).float() * _pow2(e0 - e + 127)[:, :, None, None])
        grown = (e > e0)[:, :, None, None] & old[:, None, :, None]
        now = torch.where(here, fresh, torch.where(grown, again, was))
        blocks[ids] = now.transpose(2, 3) if transposed else now
        exps[ids] = e.to(torch.uint8)


def _plain_attend(s):
    c, q, (k, vt, ke, ve), table = s['case'], s['q'], s['raw'], s['table']
    page, heads, dim = c['page'], c['kv_heads'], c['dim']
    group = c['q_heads'] // heads
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    at = 0
    for b, (length, n) in enumerate(zip(s['lens_host'], s['rows_host'])):
        lo = _visible_from(c, length, n)
        pos = torch.arange(length, device=q.device)
        if lo > c['sinks']:
            pos = torch.cat([pos[:c['sinks']], pos[lo:]])
        ids, off = table[b][pos // page].long(), pos % page
        kk = (k[ids, :, off].view(torch.float8_e4m3fn).float() * _pow2(ke[ids])[..., None]).transpose(0, 1)
        vv = (vt[ids, :, :, off].view(torch.float8_e4m3fn).float() * _pow2(ve[ids])[..., None]).transpose(0, 1)
        kk, vv = kk.transpose(1, 2).contiguous(), vv.contiguous()
        step = max(1, (1 << 28) // (c['q_heads'] * len(pos)))
        for i in range(0, n, step):
            m = min(step, n - i)
            here = slice(at + i, at + i + m)
            qq = q[here].float().view(m, heads, group, dim).permute(1, 2, 0, 3).reshape(heads, group * m, dim)
            z = (qq @ kk).view(heads, group, m, len(pos)) * s['scale']
            p = length - n + i + torch.arange(m, device=q.device)[:, None]
            seen = pos <= p
            if c['window']:
                seen &= (pos > p - c['window']) | (pos < c['sinks'])
            z = z.masked_fill(~seen, -math.inf)
            top = z.amax(-1, keepdim=True)
            w = torch.exp(z - top)
            total = w.sum(-1, keepdim=True)
            o = ((w / total).view(heads, group * m, len(pos)) @ vv).view(heads, group, m, dim)
            out[here] = o.permute(2, 0, 1, 3).reshape(m, heads * group, dim).to(q.dtype)
            lse[here] = (top + total.log())[..., 0].permute(2, 0, 1).reshape(m, heads * group)
        at += n
    return [out, lse]


def _free_list(refs):
    """(the free pages in ascending order, -1 behind them; how many)."""
    n = refs.numel()
    free = refs == 0
    rank = free.cumsum(0) - 1
    ids = torch.full((n + 1,), -1, dtype=torch.int32, device=refs.device)
    ids.scatter_(0, torch.where(free, rank, n), torch.arange(n, dtype=torch.int32, device=refs.device))
    ids[n] = -1
    return ids, free.sum()


def _count(refs, ids, by):
    """refs[ids] += by where ids are pages."""
    ok = (ids >= 0) & (ids < refs.numel())
    refs.scatter_add_(0, torch.where(ok, ids, 0).long().flatten(), torch.where(ok, by, 0).int().flatten())


def _plain_extend(refs, table, lens, add, page):
    rows, width = table.shape
    c0, c1 = -(-lens // page), -(-(lens + add) // page)
    fits = (add >= 0) & (c1 <= width)
    need = torch.where(fits, c1 - c0, 0)
    upto = need.cumsum(0)
    ids, n_free = _free_list(refs)
    granted = fits & ((need == 0) | (upto <= n_free))
    col = torch.arange(width, device=table.device)
    new = granted[:, None] & (col >= c0[:, None]) & (col < c1[:, None])
    got = ids[torch.where(new, (upto - need)[:, None] + col - c0[:, None], refs.numel())]
    table.copy_(torch.where(new, got, table))
    _count(refs, got, torch.ones_like(got))
    lens.copy_(torch.where(granted, lens + add, lens))
    return granted


def _plain_fork(refs, table, lens, parents, children, page):
    rows, width = table.shape
    n = parents.numel()
    ok = (parents >= 0) & (parents < rows) & (children >= 0) & (children < rows)
    p, ch = torch.where(ok, parents, 0).long(), torch.where(ok, children, 0).long()
    i = torch.arange(n, device=table.device)
    again = ((children[None, :] == children[:, None]) & (i[None, :] < i[:, None])).any(1)
    ok = ok & (lens[ch] == 0) & ~again
    length = lens[p]
    full = length // page
    need = ok & (length % page > 0)
    ids, n_free = _free_list(refs)
    rank = need.cumsum(0) - 1
    dst = torch.where(need & (rank < n_free), ids[torch.where(need, rank, refs.numel()).clamp(max=refs.numel())], -1)
    src = torch.where(dst >= 0, table[p].gather(1, full.clamp(max=width - 1)[:, None].long())[:, 0], -1)
    col = torch.arange(width, device=table.device)
    shared = torch.where(col < full[:, None], table[p], -1)
    row = torch.where((col == full[:, None]) & (dst >= 0)[:, None], dst[:, None], shared)
    _count(refs, torch.where(ok[:, None], shared, -1), torch.ones_like(shared))
    _count(refs, dst, torch.ones_like(dst))
    at = torch.where(ok, ch, rows)
    table.copy_(torch.cat([table, table[:1]]).scatter(0, at[:, None].expand(n, width), row)[:rows])
    kept = torch.where(need & (dst < 0), full * page, length)
    lens.copy_(torch.cat([lens, lens[:1]]).scatter(0, at, kept)[:rows])
    return torch.stack([src, dst])


def _plain_free(refs, table, lens, rows):
    end = torch.zeros(table.shape[0] + 1, dtype=torch.bool, device=table.device)
    end[torch.where((rows >= 0) & (rows < table.shape[0]), rows, table.shape[0]).long()] = True
    end = end[:-1]
    gone = torch.where(end[:, None], table, -1)
    _count(refs, gone, torch.full_like(gone, -1))
    table.copy_(torch.where(end[:, None], -1, table))
    lens.copy_(torch.where(end, 0, lens))


def _plain_compact(refs, table):
    """The pages in use at or above their number move, in ascending order, to the free ones below it."""
    n = refs.numel()
    page = torch.arange(n, device=refs.device)
    used = refs > 0
    live = used.sum()
    src, dst = used & (page >= live), ~used & (page < live)
    half = n // 2
    moves = torch.full((2, half + 1), -1, dtype=torch.int32, device=refs.device)
    for x, mask in ((0, src), (1, dst)):
        moves[x].scatter_(0, torch.where(mask, mask.cumsum(0) - 1, half), page.int())
    moves = moves[:, :half].contiguous()
    ok = moves[0] >= 0
    # (entries past the moves go through a spare element)
    to = torch.cat([page, page[:1]]).int().scatter(0, torch.where(ok, moves[0], n).long(), moves[1])
    held = (table >= 0) & (table < n)
    table.copy_(torch.where(held, to[torch.where(held, table, 0).long()], table))
    spare = torch.cat([refs, refs[:1]])
    moved = spare[torch.where(ok, moves[0], n).long()]
    spare.scatter_(0, torch.where(ok, moves[1], n).long(), moved)
    spare.scatter_(0, torch.where(ok, moves[0], n).long(), torch.zeros_like(moved))
    refs.copy_(spare[:n])
    return moves, src.sum().int().reshape(1)


def _plain_copy(data, moves):
    src, dst = moves[0].long(), moves[1].long()
    ok = (src >= 0) & (dst >= 0)
    src, dst = src[ok], dst[ok]
    data[:, dst] = data[:, src]


# --- the work of a pass and its exact outputs -----------------------------------------------------------------------

def work(case):
    """Inputs read once and outputs written once; products of queries with the keys that they see."""
    if case['path'] == 'append':
        values = sum(_lengths(case, 0)[1]) * case['kv_heads'] * case['dim'] * 2
        return {'bytes': values * 3, 'flops': values * 2}
    if case['path'] == 'attend':
        keys = pairs = 0
        for length, n in zip(*_lengths(case, 0)):
            lo = _visible_from(case, length, n)
            keys += length - lo + min(lo, case['sinks'])
            for p in range(length - n, length):
                lo = max(0, p - case['window'] + 1) if case['window'] else 0
                pairs += p + 1 - lo + min(lo, case['sinks'])
        q_bytes = sum(_lengths(case, 0)[1]) * case['q_heads'] * (case['dim'] * 4 + 4)
        return {'bytes': keys * case['kv_heads'] * case['dim'] * 2 + q_bytes,
                'flops': pairs * case['q_heads'] * case['dim'] * 4}
    table = case['rows'] * (-(-case['ctx'] // case['page']) + 2) * 4
    if case['path'] == 'fork':
        moved = case['forks']
    else:       # about half of the requests' pages are in use, half of those in the upper half of that span
        used = case['rows'] * 0.875 * 0.5 * 0.55 * case['ctx'] / case['page']
        moved = used * max(0.0, 1 - used / case['pages'])
    return {'bytes': moved * case['layers'] * case['bytes'] * 2 + 2 * (table + 4 * case['pages']),
            'flops': case['pages'] + table // 4}


def exact(case, seed):
    if case['path'] == 'attend':
        return _exact_attend(prepare(case, seed))
    if case['path'] == 'append':
        return _exact_append(prepare(case, seed))
    return None


def _two_to(e):
    """2^e in FP64, from its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _round_e4m3(x):
    """FP64 values to the nearest E4M3 value, ties to even, at most 448 in magnitude."""
    e = torch.frexp(x)[1].clamp(min=-5)            # the step of [2^(e-1), 2^e) is 2^(e-4); below 2^-6 it stays 2^-9
    step = _two_to(e - 4)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_append(s):
    (k8, v8, ke, ve), table = s['raw'], s['table'].cpu()
    page = s['case']['page']
    outs = [k8.view(torch.float8_e4m3fn).double(), v8.view(torch.float8_e4m3fn).double()]
    at = 0
    for b, (length, n) in enumerate(zip(s['lens_host'], s['rows_host'])):
        first = length - n
        for col in range(first // page, -(-length // page)):
            lo, hi = max(first, col * page), min(length, (col + 1) * page)
            p, t0, t1 = int(table[b, col]), lo - col * page, hi - col * page
            for x, o, exps in ((s['k'], outs[0], ke), (s['v'], outs[1], ve)):
                block = o[p] if o is outs[0] else o[p].transpose(1, 2)          # [heads, page, dim]
                val = x[at + lo - first:at + hi - first].double().transpose(0, 1)
                need = torch.ceil(torch.log2(val.abs().amax((1, 2)).clamp(min=2.0 ** -90) / 448) - 1e-9) + 127
                need = need.clamp(E_MIN, E_MAX)
                had = exps[p].double() if t0 else torch.zeros_like(need)
                e = torch.maximum(need, had)
                scale = _two_to(e - 127)[:, None, None]
                if t0:
                    shrink = _two_to(had - e)[:, None, None]
                    block[:, :t0] = torch.where(shrink < 1, _round_e4m3(block[:, :t0] * shrink), block[:, :t0])
                block[:, t0:t1] = _round_e4m3(val / scale)
        at += n
    return [outs[0], outs[1], None, None]


def _exact_attend(s):
    c, (k8, v8, ke, ve) = s['case'], s['raw']
    group, at = c['q_heads'] // c['kv_heads'], 0
    out = torch.empty(s['q'].shape, dtype=torch.float64, device=DEV)
    lse = torch.empty(s['q'].shape[:2], dtype=torch.float64, device=DEV)
    for b, (length, n) in enumerate(zip(s['lens_host'], s['rows_host'])):
        ids = s['table'][b, :-(-length // c['page'])].long()
        gone = ids < 0
        ids = torch.where(gone, 0, ids)
        for h in range(c['kv_heads']):
            keys = k8[ids, h].view(torch.float8_e4m3fn).double()
            keys = (keys * _two_to(ke[ids, h].int() - 127)[:, None, None]).flatten(0, 1)[:length]
            vals = v8[ids, h].view(torch.float8_e4m3fn).double()
            vals = (vals * _two_to(ve[ids, h].int() - 127)[:, None, None]).transpose(1, 2).flatten(0, 1)[:length]
            step = max(1, (1 << 27) // (length * group))
            for i in range(0, n, step):
                m = min(step, n - i)
                qq = s['q'][at + i:at + i + m, h * group:(h + 1) * group].double().flatten(0, 1)
                z = qq @ keys.t() * s['scale']
                j = torch.arange(length, device=DEV)[None]
                p = (length - n + i + torch.arange(m, device=DEV)).repeat_interleave(group)[:, None]
                hidden = j > p
                if c['window']:
                    hidden = hidden | ((j <= p - c['window']) & (j >= c['sinks']))
                z[hidden] = -math.inf
                total = torch.logsumexp(z, 1)
                o = torch.exp(z - total[:, None]) @ vals
                out[at + i:at + i + m, h * group:(h + 1) * group] = o.unflatten(0, (m, group))
                lse[at + i:at + i + m, h * group:(h + 1) * group] = total.unflatten(0, (m, group))
        at += n
    return [out, lse]
