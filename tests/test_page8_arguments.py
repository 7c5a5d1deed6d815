"""What the 8-bit pages and the page operators refuse, on the host, without a GPU."""
import ctypes

import pytest
import torch

from xtier_amd import _lib, ops
from xtier_amd.pool import KVPool, LatentPool, Page8Pool, PageTable

P = 1 << 20                     # an aligned stand-in address, never dereferenced on the host


@pytest.fixture(scope='module')
def lib():
    return _lib.lib()


def _append(lib, **kw):
    args = dict(k=P, k_rs=512, k_hs=128, v=P, v_rs=512, v_hs=128, rows=0, kp=P, vp=P, ke=P, ve=P, pages=8, heads=4,
                dim=128, page=64, ps=0, hs=0, eps=0, ehs=0, table=P, ts=4, width=4, lens=P, cu=P, batch=2, stream=None)
    args.update(kw)
    return lib.xt_page8_append(*args.values())


def _attend(lib, **kw):
    args = dict(q=P, q_rs=4096, q_hs=128, kp=P, vp=P, ke=P, ve=P, pages=8, heads=4, q_heads=32, dim=128, page=64, ps=0,
                hs=0, eps=0, ehs=0, table=P, ts=4, width=4, lens=P, cu=None, batch=0, rows=0, window=0, sinks=0,
                scale=0.1, out=P, o_rs=4096, o_hs=128, out_dtype=0, lse=None, ws=P, ws_bytes=1 << 40, stream=None)
    args.update(kw)
    return lib.xt_page8_attention(*args.values())


@pytest.mark.parametrize('call', [_append, _attend])
def test_pools(lib, call):
    assert call(lib) == _lib.XT_OK                                  # nothing to do
    for bad in (dict(dim=96), dict(dim=512), dict(page=8), dict(page=48), dict(page=256), dict(page=0)):
        assert call(lib, **bad) == _lib.XT_EUNSUPPORTED, bad
    for bad in (dict(kp=None), dict(ve=None), dict(kp=P + 8), dict(vp=P + 4), dict(pages=0), dict(pages=1 << 32),
                dict(heads=0), dict(hs=64 * 128 - 16), dict(hs=64 * 128 + 8), dict(ps=4096), dict(ps=64 * 128 * 4 + 4),
                dict(rows=-1), dict(batch=-1)):
        assert call(lib, **bad) == _lib.XT_EINVAL, bad


def test_append(lib):
    for bad in (dict(k=None), dict(v=P + 2), dict(k_rs=511), dict(v_hs=4), dict(table=None), dict(lens=None),
                dict(width=0), dict(ts=3), dict(cu=None)):
        assert _append(lib, rows=5, **bad) == _lib.XT_EINVAL, bad
    assert b'without row offsets' in lib.xt_last_error()


def test_attention(lib):
    for bad in (dict(window=-1), dict(sinks=-1), dict(q_heads=30), dict(q_heads=2), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float('inf')), dict(scale=float('nan')), dict(out_dtype=2)):
        assert _attend(lib, **bad) == _lib.XT_EINVAL, bad
    assert _attend(lib, q_heads=129, heads=1) == _lib.XT_EUNSUPPORTED
    for bad in (dict(width=1 << 25, ts=1 << 25), dict(heads=8200, q_heads=8200, rows=2), dict(ps=1 << 33)):
        assert _attend(lib, **{'rows': 2, 'batch': 2, **bad}) == _lib.XT_EUNSUPPORTED, bad
    for bad in (dict(q=None), dict(q=P + 8), dict(q_rs=4097), dict(out=P + 4), dict(o_hs=126), dict(width=0),
                dict(ts=1), dict(rows=3)):
        assert _attend(lib, **{'rows': 2, 'batch': 2, **bad}) == _lib.XT_EINVAL, bad
    need = lib.xt_page8_attention_workspace_bytes(2, 2, 32, 4, 128)
    assert need > 0
    for bad in (dict(ws=None), dict(ws=P + 128), dict(ws_bytes=need - 1)):
        assert _attend(lib, rows=2, batch=2, **bad) == _lib.XT_EWORKSPACE, bad
    assert lib.xt_page8_attention_workspace_bytes(-1, 2, 32, 4, 128) == 0
    assert lib.xt_page8_attention_workspace_bytes(1, 2, 30, 4, 128) == 0


def test_calls_too_large_for_one_launch(lib):
    assert _append(lib, rows=1 << 30, cu=P) == _lib.XT_EUNSUPPORTED
    assert _append(lib, rows=1 << 27, cu=None, batch=1 << 27) == _lib.XT_EUNSUPPORTED
    assert _attend(lib, rows=1 << 21, batch=1 << 21) == _lib.XT_EUNSUPPORTED
    assert b'row tiles of 4 KV heads' in lib.xt_last_error()
    assert lib.xt_pages_free(P, 100, P, 9, 9, P, 3, P, 1 << 24, None) == _lib.XT_EUNSUPPORTED
    # a large batch's workspace holds its plan too
    one, many = (lib.xt_page8_attention_workspace_bytes(n, n, 32, 4, 128) for n in (40, 4000))
    assert many > one + 4000 * 32
    assert _attend(lib, rows=4000, batch=4000, ws_bytes=many - 1) in (_lib.XT_EWORKSPACE, _lib.XT_ELAUNCH)
    assert _attend(lib, rows=4000, batch=4000, ws_bytes=one) == _lib.XT_EWORKSPACE


def test_page_operators(lib):
    ok, bad, small, far = _lib.XT_OK, _lib.XT_EINVAL, _lib.XT_EWORKSPACE, _lib.XT_EUNSUPPORTED
    assert lib.xt_pages_workspace_bytes(100) == 400 and lib.xt_pages_workspace_bytes(-1) == 0
    extend = lambda refs=P, pages=100, table=P, ts=9, w=9, lens=P, add=P, rows=3, page=16, g=P, ws=P, n=400: \
        lib.xt_pages_extend(refs, pages, table, ts, w, lens, add, rows, page, g, ws, n, None)
    assert extend(rows=0) == ok
    for kw in (dict(refs=None), dict(table=None), dict(lens=None), dict(add=None), dict(g=None), dict(pages=0),
               dict(w=0), dict(ts=8), dict(rows=-1), dict(page=0), dict(page=12), dict(page=-16)):
        assert extend(**kw) == bad, kw
    assert extend(ws=None) == small and extend(n=399) == small
    fork = lambda forks=7, p=P, c=P, moves=P, ms=7, n=0, page=16, w=9: \
        lib.xt_pages_fork(P, 100, P, w, w, P, 3, page, p, c, forks, moves, ms, P, n, None)
    assert fork(forks=0) == ok and fork(forks=1025, ms=1025) == far
    assert fork(w=2341, n=7 * 12 - 1) == small                        # 7 * 2341 columns: past the one-launch size
    for kw in (dict(p=None), dict(c=None), dict(moves=None), dict(ms=6), dict(forks=-1), dict(page=3)):
        assert fork(**kw) == bad, kw
    assert lib.xt_pages_free(P, 100, P, 9, 9, P, 3, None, 0, None) == ok
    assert lib.xt_pages_free(P, 100, P, 9, 9, P, 3, None, 1, None) == bad
    assert lib.xt_pages_free(P, 100, P, 9, 9, None, 3, P, 1, None) == bad
    assert lib.xt_pages_compact(P, 100, P, 9, 9, 3, None, P, P, 400, None) == bad
    assert lib.xt_pages_compact(P, 100, P, 9, 9, 3, P, P, P, 399, None) == small
    buffers = (_lib.PageBuffer * 2)(_lib.PageBuffer(P, 10, 64, 64), _lib.PageBuffer(P, 10, 63, 64))
    copy = lambda b=buffers, nb=2, m=P, ms=4, n=4: lib.xt_pages_copy(b, nb, m, ms, n, None, None)
    assert copy(nb=0) == ok and copy(n=0) == ok
    assert copy() == bad and b'closer than' in lib.xt_last_error()
    assert copy(nb=1, m=None) == bad and copy(nb=1, ms=3) == bad and copy(nb=-1) == bad and copy(b=None) == bad
    assert copy(nb=65) == far


def test_valid_calls_reach_the_launch(lib):
    """Every host check passes; without a device the launch is what fails."""
    if torch.cuda.is_available():
        pytest.skip('needs no GPU to be visible')
    assert _append(lib, rows=5) == _lib.XT_ELAUNCH
    assert _attend(lib, rows=2, batch=2) == _lib.XT_ELAUNCH
    assert _attend(lib, rows=2000, batch=2, cu=P) == _lib.XT_ELAUNCH
    buffers = (_lib.PageBuffer * 1)(_lib.PageBuffer(P, 10, 64, 64))
    assert lib.xt_pages_copy(buffers, 1, P, 4, 4, None, None) == _lib.XT_ELAUNCH
    assert ctypes.sizeof(_lib.PageBuffer) == 32


def test_python_checks():
    pool = Page8Pool(8, 32, 2, 64, device='cpu')
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='GPU tensors'):
        pool.append(x, x, table, lens)
    with pytest.raises(ValueError, match='GPU tensors'):
        pool.attend(q, table, lens, 0.1)
    for k, v in ((x.float(), x), (x, x[:2]), (x[:, :1], x[:, :1]), (x.transpose(1, 2), x.transpose(1, 2)), (x[0], x[0])):
        with pytest.raises(ValueError, match='BF16 rows'):
            pool.append(k, v, table, lens)
    for bad in (q.float(), q[..., :32], q[0], q.half()):
        with pytest.raises(ValueError, match='BF16 queries'):
            pool.attend(bad, table, lens, 0.1)
    with pytest.raises(ValueError, match='page table'):
        pool.attend(q, table.long(), lens, 0.1)
    with pytest.raises(ValueError, match='page table'):
        pool.attend(q, table[0], lens, 0.1)
    for t, s, cu in ((table, lens[:2], None), (table[:2], lens[:2], None), (table, lens, lens)):
        with pytest.raises(ValueError, match='for a table of'):
            pool.attend(q, t, s, 0.1, cu)
    k, vt, ke, ve = pool.raw
    for raw in ((k.float(), vt, ke, ve), (k, k, ke, ve), (k, vt, ke[:4], ve), (k, vt, ke, ve.int()),
                (k[:, :, ::2], vt, ke, ve), (k.contiguous(), vt, ke, ve), (k[0], vt, ke, ve),
                (k[:1].expand(8, -1, -1, -1), vt[:1].expand(8, -1, -1, -1), ke, ve),
                (k, vt, ke[:1].expand(8, -1), ve[:1].expand(8, -1))):
        with pytest.raises(ValueError, match='expected'):
            ops.page8_append(x, x, raw, table, lens)
    for page, dim in ((8, 64), (64, 96), (256, 128)):
        with pytest.raises(NotImplementedError):
            Page8Pool(4, page, 2, dim, device='cpu')
    with pytest.raises(ValueError, match='power of 2'):
        PageTable(2, 2, 2, 24, device='cpu')
    t = PageTable(3, 2, 8, 16, device='cpu')
    with pytest.raises(ValueError, match='sizes for'):
        t.extend(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match='as many parents'):
        t.fork(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match='int32 refs'):
        ops.pages_free(t.refs.long(), t.table, t.lens, t.lens)
    with pytest.raises(ValueError, match='int32 lens'):
        ops.pages_free(t.refs, t.table, t.lens[:2], t.lens)
    with pytest.raises(ValueError, match='GPU tensors'):
        t.compact()
    with pytest.raises(ValueError, match='contiguous pages'):
        ops.PageBuffers([torch.zeros(4, 6, 6)[:, :, :3]])
    with pytest.raises(ValueError, match='int32 moves'):
        ops.pages_copy([torch.zeros(4, 6)], torch.zeros(2, 3))
    with pytest.raises(ValueError, match='int32 count'):
        ops.pages_copy([torch.zeros(4, 6)], torch.zeros(2, 3, dtype=torch.int32), torch.zeros(0, dtype=torch.int32))
    with pytest.raises(ValueError, match='whole pages'):
        KVPool(40, 1, 64, device='cpu').page_buffers(16)
    assert [b.shape for b in LatentPool(32, device='cpu').page_buffers(16)] == [(2, 16 * 416)]
