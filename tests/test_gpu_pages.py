"""Page bookkeeping on the GPU against the CPU restatement: growing, forking, freeing, compacting and copying, alone and
in long random runs, with the caches that live in the pages."""
import numpy as np
import pytest
import torch

from tests._page8 import bf16, page8
from xtier_amd import ops
from xtier_amd.pool import KVPool, LatentPool, Page8Pool, PageTable

pytestmark = pytest.mark.gpu


class Pair:
    """A PageTable and its restatement, compared after every step."""

    def __init__(self, rows, width, pages, page):
        self.gpu = PageTable(rows, width, pages, page)
        self.page = page
        self.refs, self.table, self.lens = (x.cpu().numpy().copy() for x in
                                            (self.gpu.refs, self.gpu.table, self.gpu.lens))

    def same(self):
        for got, want in ((self.gpu.refs, self.refs), (self.gpu.table, self.table), (self.gpu.lens, self.lens)):
            assert np.array_equal(got.cpu().numpy(), want)

    def extend(self, add):
        add = np.asarray(add, np.int32)
        got = self.gpu.extend(torch.from_numpy(add).cuda())
        want = page8.extend(self.refs, self.table, self.lens, add, self.page)
        assert np.array_equal(got.cpu().numpy(), want)
        self.same()
        return want

    def fork(self, parents, children):
        p, c = np.asarray(parents, np.int32), np.asarray(children, np.int32)
        got = self.gpu.fork(torch.from_numpy(p).cuda(), torch.from_numpy(c).cuda())
        want = page8.fork(self.refs, self.table, self.lens, p, c, self.page)
        assert np.array_equal(got.cpu().numpy(), want)
        self.same()
        return got

    def free(self, rows):
        rows = np.asarray(rows, np.int32)
        self.gpu.free(torch.from_numpy(rows).cuda())
        page8.free(self.refs, self.table, self.lens, rows)
        self.same()

    def compact(self):
        moves, count = self.gpu.compact()
        want, n = page8.compact(self.refs, self.table)
        assert np.array_equal(moves.cpu().numpy(), want) and count.item() == n
        self.same()
        return moves, count


def test_extend_orders_and_refusals():
    t = Pair(6, 4, 10, 16)
    assert t.extend([0, 1, 16, 17, 64, 65]).tolist() == [True, True, True, True, True, False]    # 65: too wide
    assert t.extend([0, 15, 1, 0, 0, 33]).tolist() == [True, True, True, True, True, False]      # 2 pages left, 3 asked
    assert t.extend([16, 0, 0, -1, 0, 16]).tolist() == [True, True, True, False, True, False]    # the last page went first
    t.extend([0] * 6)


def test_extend_many_rows():
    """More rows than threads, many pages a row, the pool running out in the middle."""
    rng = np.random.default_rng(1)
    t = Pair(2500, 9, 5000, 32)
    for _ in range(3):
        t.extend(rng.integers(0, 90, 2500))
    t.free(rng.permutation(2500)[:900])
    t.extend(rng.integers(-3, 200, 2500))


def test_fork_shares_full_pages():
    t = Pair(8, 5, 12, 16)
    t.extend([40, 32, 7, 0, 0, 0, 0, 0])
    moves = t.fork([0, 1, 0, 2], [3, 4, 5, 6])
    assert moves.cpu().tolist()[0] == [2, -1, 2, 5]
    t.fork([0, 3], [7, 7])                          # the second is skipped: the child is taken
    t.free([0, 0, 4])                               # a row named twice


def test_fork_skips_and_runs_out():
    t = Pair(10, 5, 6, 16)
    t.extend([20, 30, 16, 0, 0, 0, 0, 0, 0, 0])
    t.fork([0, 1, 2, 0, -1, 10, 0, 3], [1, 4, 5, 11, 6, 6, -2, 6])     # a taken child, ids outside, an empty parent
    t.fork([0, 1], [7, 8])                                              # no free page: full pages only
    assert t.lens.tolist()[7:9] == [16, 16]


def test_fork_many():
    rng = np.random.default_rng(2)
    t = Pair(1400, 70, 30000, 16)
    t.extend(np.where(np.arange(1400) < 300, rng.integers(0, 1100, 1400), 0))
    t.fork(rng.integers(0, 300, 1024), 300 + rng.permutation(1100)[:1024])


def test_free_ignores_rows_outside():
    t = Pair(3, 3, 5, 16)
    t.extend([20, 20, 1])
    t.free([-1, 3, 1, 1 << 30])
    t.free([])


@pytest.mark.parametrize('pages', [1, 2, 7, 1023, 1025, 4100, 70001])
def test_compact_sizes(pages):
    rng = np.random.default_rng(pages)
    t = Pair(40, 60, pages, 16)
    t.extend(np.minimum(rng.integers(0, 950, 40), max(0, pages - 1) * 16 // 40 + 16))
    t.free(rng.permutation(40)[:25])
    t.compact()
    moves, count = t.compact()
    assert count.item() == 0 and (moves == -1).all()


def test_compact_high_pages():
    """Pages scattered over the whole pool, shared ones among them, and every page in use."""
    rng = np.random.default_rng(3)
    t = Pair(20, 30, 900, 16)
    t.extend([400] * 20)
    t.fork([1, 2, 3], [4, 5, 6])                    # children hold tokens: skipped
    t.free(np.arange(4, 15))
    t.fork([1, 1, 19], [4, 5, 6])
    t.free([0, 1, 16])
    t.compact()
    full = Pair(4, 2, 8, 16)
    full.extend([32] * 4)
    full.compact()


def test_random_runs():
    for seed in range(6):
        rng = np.random.default_rng(seed)
        rows, page = int(rng.integers(3, 70)), int(rng.choice([1, 16, 64]))
        t = Pair(rows, 12, int(rng.integers(10, 400)), page)
        for _ in range(25):
            op = rng.integers(0, 4)
            if op == 0:
                t.extend(rng.integers(0, 3 * page + 1, rows))
            elif op == 1:
                n = int(rng.integers(1, rows + 1))
                t.fork(rng.integers(0, rows, n), rng.integers(0, rows, n))
            elif op == 2:
                t.free(rng.integers(0, rows, int(rng.integers(1, max(2, rows // 3)))))
            else:
                t.compact()
            held = t.table[t.table >= 0]
            assert np.array_equal(np.bincount(held, minlength=len(t.refs)), t.refs)     # counts are the entries


def test_strided_tables():
    wide = torch.full((6, 20), -1, dtype=torch.int32, device='cuda')
    refs, lens = torch.zeros(30, dtype=torch.int32, device='cuda'), torch.zeros(6, dtype=torch.int32, device='cuda')
    table = wide[:, 4:9]
    ops.pages_extend(refs, table, lens, torch.tensor([40, 0, 0, 70, 0, 0], device='cuda'), 16)
    ops.pages_fork(refs, table, lens, torch.tensor([0, 3], device='cuda'), torch.tensor([1, 2], device='cuda'), 16)
    ops.pages_free(refs, table, lens, torch.tensor([0], device='cuda'))
    ops.pages_compact(refs, table)
    want = [np.zeros(30, np.int32), np.full((6, 5), -1, np.int32), np.zeros(6, np.int32)]
    page8.extend(*want, np.array([40, 0, 0, 70, 0, 0]), 16)
    page8.fork(*want, np.array([0, 3]), np.array([1, 2]), 16)
    page8.free(*want, np.array([0]))
    page8.compact(want[0], want[1])
    for got, x in zip((refs, table, lens), want):
        assert np.array_equal(got.cpu().numpy(), x)
    assert (wide[:, :4] == -1).all() and (wide[:, 9:] == -1).all()


@pytest.mark.parametrize('shape,dtype', [((7, 4, 2), torch.uint8), ((9, 3), torch.uint8), ((9, 16, 33), torch.uint8),
                                         ((40, 65536), torch.uint8), ((12, 5, 20), torch.bfloat16),
                                         ((11, 100001), torch.uint8)])
def test_copy_sizes(shape, dtype):
    gen = torch.Generator(device='cuda').manual_seed(4)
    x = torch.randint(0, 256, (*shape[:-1], shape[-1] * dtype.itemsize), generator=gen, device='cuda',
                      dtype=torch.uint8).view(dtype)
    moves = torch.tensor([[1, 3, -1, 2, shape[0], 0], [5, 4, 6, -1, 6, -7]], dtype=torch.int32, device='cuda')
    want = x.clone()
    want[5], want[4] = x[1], x[3]
    ops.pages_copy([x], moves)
    assert torch.equal(x.view(torch.uint8), want.view(torch.uint8))
    more = torch.tensor([[1, 4], [0, 2]], dtype=torch.int32, device='cuda')
    want[0] = want[1]
    ops.pages_copy([x], more, torch.tensor([1], dtype=torch.int32, device='cuda'))
    assert torch.equal(x.view(torch.uint8), want.view(torch.uint8))


def test_copy_many_buffers_and_strides():
    """More buffers than one launch takes, of differing sizes, strides and page counts."""
    gen = torch.Generator(device='cuda').manual_seed(5)
    base = [torch.randint(0, 256, (10 + i % 3, 100 + 16 * i), generator=gen, device='cuda', dtype=torch.uint8)
            for i in range(70)]
    views = [t[:, i % 5: 60 + i] for i, t in enumerate(base)]
    want = [t.clone() for t in base]
    moves = torch.tensor([[0, 9, 11], [8, 2, 1]], dtype=torch.int32, device='cuda')
    for i, t in enumerate(want):
        v = t[:, i % 5: 60 + i]
        v[8], v[2] = v[0].clone(), v[9].clone()
        if v.shape[0] > 11:
            v[1] = v[11].clone()
    ops.pages_copy(ops.PageBuffers(views), moves)
    assert all(torch.equal(a, b) for a, b in zip(base, want))


def test_caches_move_with_their_pages():
    """Every cache of the package through a fork and a compaction: each row still reads its own tokens."""
    page, pages, rows = 16, 32, 8
    t = PageTable(rows, 6, pages, page)
    pools = [KVPool(pages * page, 2, 64), KVPool(pages * page, 2, 64, layout='split'), LatentPool(pages * page),
             LatentPool(pages * page, layout='split'), Page8Pool(pages, page, 2, 64)]
    buffers = ops.PageBuffers([b for p in pools for b in (p.page_buffers() if isinstance(p, Page8Pool)
                                                          else p.page_buffers(page))])
    gen = torch.Generator(device='cuda').manual_seed(6)
    for b in buffers.tensors:
        b.view(torch.uint8).random_(0, 256, generator=gen)
    rng = np.random.default_rng(7)
    t.extend(torch.tensor([40, 33, 0, 80, 16, 5, 0, 0], device='cuda'))

    def rows_of(row):
        n = int(t.lens[row])
        pos = torch.arange(n, device='cuda')
        slots = t.table[row][pos // page].long() * page + pos % page
        token_major = [x[slots] for p in pools[:4] for x in p.raw if x.dim() > 1]
        k, vt = pools[4].k, pools[4].vt
        ids = t.table[row][pos // page].long()
        return [x.clone() for x in (*token_major, k[ids, :, pos % page], vt[ids, :, :, pos % page],
                                    pools[4].k_exp[ids], pools[4].v_exp[ids])]

    def equal(a, b):
        return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))

    before = {r: rows_of(r) for r in (0, 1, 3, 4, 5)}
    moves = t.fork(torch.tensor([0, 3, 0], device='cuda'), torch.tensor([2, 6, 7], device='cuda'))
    ops.pages_copy(buffers, moves)
    before |= {2: before[0], 6: before[3], 7: before[0]}
    for r, want in before.items():
        assert equal(rows_of(r), want), r
    t.free(torch.tensor([0, 4, 1], device='cuda'))
    moves, count = t.compact()
    ops.pages_copy(buffers, moves, count)
    assert count.item() > 0
    for r in (2, 3, 5, 6, 7):
        assert equal(rows_of(r), before[r]), r


def test_beams_of_a_server():
    """Prompt, forks, decode steps of the beams, losers freed, compaction, more decode: the beams' attention equals that of
    a cache in which every beam has its own pages throughout."""
    page, heads, group, dim = 16, 2, 4, 64
    rng = np.random.default_rng(8)
    beams = PageTable(6, 8, 40, page)
    pool = Page8Pool(40, page, heads, dim)
    alone = Page8Pool(64, page, heads, dim)
    own_table = torch.arange(48, dtype=torch.int32, device='cuda').view(6, 8)
    buffers = ops.PageBuffers(pool.page_buffers())
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device='cuda')
    rows = lambda n, h: bf16(rng.standard_normal((n, h, dim))).cuda()

    def step(ids, k, v, q):
        n = k.shape[0] // len(ids)
        add = [0] * 6
        for i in ids:
            add[i] = n
        assert beams.extend(dev(add)).all()
        cu, sel = dev([n * i for i in range(len(ids) + 1)]), dev(ids).long()
        lens = beams.lens[sel].contiguous()
        outs = []
        for p, table in ((pool, beams.table[sel]), (alone, own_table[sel])):
            p.append(k, v, table.contiguous(), lens, cu)
            outs.append(p.attend(q, table.contiguous(), lens, 0.1, cu, window=60, sinks=4))
        assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0]).all()

    step([0], rows(37, heads), rows(37, heads), rows(37, heads * group))
    ops.pages_copy(buffers, beams.fork(dev([0, 0, 0]), dev([1, 2, 3])))
    for r in (1, 2, 3):
        for b in alone.page_buffers():
            b[8 * r:8 * r + 8] = b[0:8]
    for _ in range(20):
        step([0, 1, 2, 3], rows(4, heads), rows(4, heads), rows(4, heads * group))
    beams.free(dev([0, 2]))
    moves, count = beams.compact()
    ops.pages_copy(buffers, moves, count)
    for _ in range(10):
        step([1, 3], rows(2, heads), rows(2, heads), rows(2, heads * group))


def test_replays_of_a_captured_step():
    """Fork, copy, extend, free and compact captured once; every replay agrees with the same steps run eagerly."""
    page = 16
    data = torch.arange(60 * 64, dtype=torch.int32, device='cuda').view(60, 64)
    t = PageTable(12, 8, 60, page)
    t.extend(torch.tensor([40, 20, 100, 7] + [0] * 8, device='cuda'))
    parents, children = (torch.tensor(x, dtype=torch.int32, device='cuda') for x in ([0, 2, 3], [4, 5, 6]))
    add, gone = torch.ones(12, dtype=torch.int32, device='cuda'), torch.tensor([4, 1], dtype=torch.int32, device='cuda')
    buffers = ops.PageBuffers([data])

    def step():
        ops.pages_copy(buffers, t.fork(parents, children))
        t.extend(add)
        t.free(gone)
        ops.pages_copy(buffers, *t.compact())

    state = (t.refs, t.table, t.lens, data)
    saved = [x.clone() for x in state]
    step()
    runs = [[x.clone() for x in state]]
    step()
    runs.append([x.clone() for x in state])
    for x, y in zip(state, saved):
        x.copy_(y)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for x, y in zip(state, saved):
        x.copy_(y)
    for want in runs:
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(state, want))
