"""The 8-bit paged cache on the GPU: the append bit for bit against the CPU restatement, and the attention against it in
float64, at the sizes, masks and layouts where they can go wrong."""
import numpy as np
import pytest
import torch

from tests._page8 import attention_on_gpu, attention_tolerance, bf16, gpu_raw, page8, pool_bytes, table_for
from xtier_amd import ops
from xtier_amd.pool import Page8Pool

pytestmark = pytest.mark.gpu


def _same_pool(pool, raw):
    torch.cuda.synchronize()
    for name, got, want in zip(('k', 'vt', 'k_exp', 'v_exp'), pool.raw, raw):
        got = got.cpu().numpy()
        bad = np.argwhere(got != want)
        assert not len(bad), (name, len(bad), bad[:4].tolist(), got[got != want][:4], want[got != want][:4])


# --- append ---------------------------------------------------------------------------------------------------------

def _append_case(rng, old, new, page, heads, dim, magnitudes=None):
    lens = [o + n for o, n in zip(old, new)]
    pages = sum(-(-x // page) for x in lens) + 3
    raw = pool_bytes(rng, pages, heads, page, dim, spread=6)
    table = table_for(rng, lens, page, pages, max(1, max(-(-x // page) for x in lens)) + 1)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows = int(cu[-1])
    x = rng.standard_normal((2, rows, heads, dim)) * 2.0 ** rng.integers(-12, 6, (2, rows, heads, 1))
    if magnitudes is not None:
        x *= magnitudes
    k, v = bf16(x[0]), bf16(x[1])
    return raw, table, np.array(lens, np.int32), cu, k, v


def _check_append(raw, table, lens, cu, k, v, page, pass_cu=True):
    pool = gpu_raw(raw)
    page8.append(k.double().numpy(), v.double().numpy(), raw, table, page, lens, cu)
    pool.append(k.cuda(), v.cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(),
                torch.from_numpy(cu).cuda() if pass_cu else None)
    _same_pool(pool, raw)


@pytest.mark.parametrize('page,heads,dim', [(16, 2, 64), (32, 1, 256), (64, 4, 128), (128, 3, 64), (128, 2, 128),
                                            (128, 1, 256)])
def test_append_ragged_requests(page, heads, dim):
    rng = np.random.default_rng(page + dim)
    old = [0, 5, page - 1, page, 2 * page + 3, 0, 7]
    new = [1, page + 2, 1, 3 * page + 5, 0, 2 * page, page - 7]
    _check_append(*_append_case(rng, old, new, page, heads, dim), page)


def test_append_many_requests():
    """More requests than lanes of a wave, and than 64 times 64, some without rows, the first one's rows not at 0."""
    rng = np.random.default_rng(37)
    for n, page in ((65, 16), (700, 32), (4200, 16)):
        old, new = rng.integers(0, 40, n).tolist(), rng.integers(0, 4, n).tolist()
        new[n // 2], new[0] = 90, 0
        raw, table, lens, cu, k, v = _append_case(rng, old, new, page, 1, 64)
        _check_append(raw, table, lens, cu, k, v, page)
        _check_append(raw, table[n // 2 + 1:], lens[n // 2 + 1:], cu[n // 2 + 1:], k, v, page)


@pytest.mark.parametrize('page,heads,dim', [(16, 4, 64), (64, 4, 128), (128, 2, 256)])
def test_append_one_row_each(page, heads, dim):
    rng = np.random.default_rng(page * 3 + dim)
    old = [0, 1, page - 1, page, 3 * page + 5, 40]
    _check_append(*_append_case(rng, old, [1] * 6, page, heads, dim), page, pass_cu=False)
    _check_append(*_append_case(rng, old, [1] * 6, page, heads, dim), page)


def test_append_row_by_row_grows_the_scale():
    """One row a call, each larger than the one before: every earlier row is rounded again, down to subnormals."""
    rng = np.random.default_rng(5)
    page, heads, dim = 32, 2, 64
    raw = pool_bytes(rng, 4, heads, page, dim)
    pool = gpu_raw(raw)
    table = np.array([[2, 1]], np.int32)
    for i in range(40):
        x = bf16(rng.standard_normal((2, 1, heads, dim)) * 2.0 ** (i * 0.7 - 10))
        lens = np.array([i + 1], np.int32)
        page8.append(x[0].double().numpy(), x[1].double().numpy(), raw, table, page, lens)
        pool.append(x[0].cuda(), x[1].cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda())
    _same_pool(pool, raw)


def test_append_special_values():
    rng = np.random.default_rng(6)
    raw, table, lens, cu, k, v = _append_case(rng, [3, 0, 0, 0], [9, 4, 4, 40], 16, 2, 64)
    k[0, 0, :3] = torch.tensor([float('nan'), float('inf'), -float('inf')])
    v[10, 1, :] = float('nan')                       # a row with nothing finite
    k[9:13] = 0                                      # a page of zeros
    v[13:17] = 3.38e38                               # beyond the largest scale
    k[13:17] = 1e-38
    k[20, 0, 0], v[20, 1, 1] = -0.0, 448.0
    _check_append(raw, table, lens, cu, k, v, 16)


def test_append_skips_what_has_no_place():
    """Negative positions, columns past the table, ids outside the pool and rows of no request leave the pool alone."""
    rng = np.random.default_rng(7)
    page, heads, dim = 16, 2, 64
    raw = pool_bytes(rng, 6, heads, page, dim)
    table = np.array([[0, 1], [2, 9], [3, -1], [4, 5], [-1, -1]], np.int32)
    lens = np.array([5, 25, 30, 50, -4], np.int32)
    cu = np.array([0, 9, 34, 64, 84, 86], np.int32)     # request 0 has 4 rows before position 0
    k, v = bf16(rng.standard_normal((90, heads, dim))), bf16(rng.standard_normal((90, heads, dim)))
    _check_append(raw, table, lens, cu, k, v, page)


def test_append_strided_rows_and_pools():
    rng = np.random.default_rng(8)
    raw, table, lens, cu, k, v = _append_case(rng, [3, 20], [30, 7], 32, 3, 64)
    fused = torch.empty(37, 9, 64, dtype=torch.bfloat16, device='cuda')     # q, k and v of a fused projection
    fused[:, 3:6], fused[:, 6:] = k.cuda(), v.cuda()
    pool = [torch.from_numpy(x).cuda() for x in raw]                        # packed, K and V apart
    wide = torch.full((2, 8), -1, dtype=torch.int32, device='cuda')
    wide[:, :table.shape[1]] = torch.from_numpy(table).cuda()
    ops.page8_append(fused[:, 3:6], fused[:, 6:], pool, wide[:, :table.shape[1]], torch.from_numpy(lens).cuda().long(),
                     torch.from_numpy(cu).cuda())
    page8.append(k.double().numpy(), v.double().numpy(), raw, table, 32, lens, cu)
    torch.cuda.synchronize()
    for got, want in zip(pool, raw):
        assert np.array_equal(got.cpu().numpy(), want)


# --- attention ------------------------------------------------------------------------------------------------------

def _attention_case(rng, lens, rows, page, heads, group, dim, q_std=1.0, spread=2):
    pages = sum(-(-max(x, 0) // page) for x in lens) + 2
    raw = pool_bytes(rng, pages, heads, page, dim, spread)
    table = table_for(rng, [max(x, 0) for x in lens], page, pages)
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    q = bf16(rng.standard_normal((int(cu[-1]), heads * group, dim)) * q_std)
    return raw, table, np.array(lens, np.int32), cu, q


def _check_attention(raw, table, lens, cu, q, page, window=0, sinks=0, scale=0.01, pass_cu=True, out_dtype=None,
                     pool=None, large=False):
    pool = pool or gpu_raw(raw)
    if large:
        ref, ref_lse, spread, score = attention_on_gpu(q, raw, table, page, lens, scale, cu, window, sinks)
    else:
        ref, ref_lse, spread, score = page8.attention(q.double().numpy(), raw, table, page, lens, scale, cu, window,
                                                      sinks)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device='cuda')
    out = None if out_dtype is None else torch.empty(q.shape, dtype=out_dtype, device='cuda')
    out = pool.attend(q.cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(), scale,
                      torch.from_numpy(cu).cuda() if pass_cu else None, window, sinks, out, lse)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    tol, lse_tol = attention_tolerance(ref, ref_lse, spread, score, raw, int(max(lens.max(), 1)), q.shape[2],
                                       torch.finfo(out.dtype).eps)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    bad = ~(np.abs(got - ref) <= tol) & ~np.isnan(ref)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], ref[bad][:5], tol[bad][:5])
    empty = np.isneginf(ref_lse)
    assert np.isneginf(got_lse[empty]).all() and not np.isneginf(got_lse[~empty]).any()
    real = ~empty & ~np.isnan(ref_lse)
    off = np.abs(got_lse[real] - ref_lse[real])
    assert (off <= lse_tol[real]).all(), (off.max(), lse_tol.min())
    return out, lse


@pytest.mark.parametrize('dim', [64, 128, 256])
@pytest.mark.parametrize('page', [16, 32, 64, 128])
def test_decode_lengths(dim, page):
    rng = np.random.default_rng(dim + page)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300]
    case = _attention_case(rng, lens, [1] * len(lens), page, 2, 4, dim)
    _check_attention(*case, page, pass_cu=False)
    _check_attention(*case, page)


@pytest.mark.parametrize('heads,group', [(1, 1), (8, 1), (1, 8), (2, 5), (1, 16), (1, 20), (2, 33), (1, 128)])
def test_decode_head_groups(heads, group):
    rng = np.random.default_rng(heads * 100 + group)
    _check_attention(*_attention_case(rng, [70, 9, 200], [1, 1, 1], 32, heads, group, 64), 32, pass_cu=False)


@pytest.mark.parametrize('dim,group', [(64, 4), (128, 8), (256, 2), (128, 16)])
def test_several_rows_each(dim, group):
    """Verification and prompt chunks: causal rows, requests without rows, rows that fill whole and part tiles."""
    rng = np.random.default_rng(dim * group)
    lens, rows = [70, 5, 130, 33, 64, 90], [5, 5, 0, 1, 33, 17]
    _check_attention(*_attention_case(rng, lens, rows, 32, 2, group, dim), 32)


def test_long_prompt_chunk():
    rng = np.random.default_rng(11)
    _check_attention(*_attention_case(rng, [403, 150], [300, 131], 64, 1, 4, 64), 64)


@pytest.mark.parametrize('window,sinks', [(1, 0), (1, 1), (17, 0), (64, 4), (100, 70), (129, 1), (1000, 3), (5, 500)])
def test_windows(window, sinks):
    rng = np.random.default_rng(window + sinks)
    lens = [1, 40, 64, 100, 190, 330]
    _check_attention(*_attention_case(rng, lens, [1] * 6, 16, 2, 4, 64), 16, window, sinks, pass_cu=False)
    _check_attention(*_attention_case(rng, lens, [1, 7, 64, 3, 20, 200], 32, 1, 4, 64), 32, window, sinks)


def test_split_over_workgroups():
    """Long contexts that many workgroups share, beside short ones, with scores that move the maximum."""
    rng = np.random.default_rng(12)
    lens = [6000, 3, 2500, 700]
    _check_attention(*_attention_case(rng, lens, [1] * 4, 64, 2, 4, 64, q_std=4.0), 64, pass_cu=False, scale=0.05)


def test_rows_that_see_nothing():
    """Lengths of zero and below, more rows than tokens, pages that are gone: zeros and -inf."""
    rng = np.random.default_rng(13)
    raw, table, _, _, _ = _attention_case(rng, [40, 40, 40, 40, 40], [1] * 5, 16, 2, 4, 64)
    lens, cu = np.array([0, -3, 2, 40, 40], np.int32), np.array([0, 1, 2, 7, 9, 10], np.int32)
    table[3] = -1
    table[4] = raw[0].shape[0]
    q = bf16(rng.standard_normal((10, 8, 64)))
    out, lse = _check_attention(raw, table, lens, cu, q, 16)
    assert (out[[0, 1, 2, 3, 4, 7, 8, 9]] == 0).all() and torch.isneginf(lse[[0, 1, 7, 8, 9]]).all()


def test_a_page_that_is_gone_among_others():
    rng = np.random.default_rng(14)
    raw, table, lens, cu, q = _attention_case(rng, [300, 300], [1, 4], 32, 1, 8, 128)
    table[0, 3], table[1, 0], table[1, 8] = -1, 1 << 20, -(1 << 31)
    _check_attention(raw, table, lens, cu, q, 32)


def test_longer_than_the_table():
    rng = np.random.default_rng(15)
    raw, table, lens, cu, q = _attention_case(rng, [100, 90], [1, 3], 32, 1, 4, 64)
    _check_attention(raw, table, np.array([2000000000, 120], np.int32), cu, q, 32, window=0)


@pytest.mark.parametrize('rows', [[1, 1, 1], [9, 30, 70]])
def test_nan_in_hidden_places_changes_nothing(rows):
    """NaN bytes behind the last token, before the window, in freed pages and, for rows before them, in later tokens."""
    rng = np.random.default_rng(16)
    raw, table, lens, cu, q = _attention_case(rng, [70, 100, 190], rows, 32, 2, 4, 64)
    for b, n in enumerate(lens):                       # the unwritten rest of the last page
        page, t = table[b, (n - 1) // 32], (n - 1) % 32 + 1
        raw[0][page, :, t:], raw[1][page, :, :, t:] = 0x7F, 0xFF
    spare = sorted(set(range(raw[0].shape[0])) - set(table[table >= 0].tolist()))
    raw[0][spare], raw[1][spare] = 0x7F, 0x7F
    raw[2][spare], raw[3][spare] = 254, 254
    _check_attention(raw, table, lens, cu, q, 32)
    raw[0][table[2, 1]], raw[1][table[2, 1]] = 0x7F, 0x7F       # position 32..63 of request 2, behind its window
    if rows[2] == 1:
        _check_attention(raw, table, lens, cu, q, 32, window=100, sinks=7)


@pytest.mark.parametrize('rows', [[1], [4], [40], [150]])
def test_nan_reaches_the_rows_that_see_it(rows):
    rng = np.random.default_rng(17)
    for where in (150, 170, 199):
        raw, table, lens, cu, q = _attention_case(rng, [200], rows, 32, 2, 4, 64)
        raw[1][table[0, where // 32], 1, 3, where % 32] = 0x7F
        raw[1][table[0, where // 32], 0, 60, where % 32] = 0xFF
        _check_attention(raw, table, lens, cu, q, 32)
        _check_attention(raw, table, lens, cu, q, 32, window=20, sinks=2)
    raw[0][table[0, 5], 0, 3, 9] = 0x7F                 # a key: the whole row of its heads
    _check_attention(raw, table, lens, cu, q, 32)


def test_scales_far_apart():
    """Pages whose exponents differ by up to 24: small pages keep their value beside large ones."""
    rng = np.random.default_rng(18)
    raw, table, lens, cu, q = _attention_case(rng, [500, 300], [1, 5], 16, 2, 4, 64, spread=12)
    _check_attention(raw, table, lens, cu, q, 16, scale=1e-4)


def test_large_and_small_queries():
    rng = np.random.default_rng(19)
    for std, scale in ((1e20, 1e-23), (1e-20, 1e18)):
        _check_attention(*_attention_case(rng, [100, 33], [1, 3], 32, 1, 4, 64, q_std=std), 32, scale=scale)


def test_layouts_and_outputs():
    """Strided queries, outputs and pools, FP16 outputs, rows behind the last request, int64 lengths."""
    rng = np.random.default_rng(20)
    raw, table, lens, cu, q = _attention_case(rng, [90, 41], [3, 2], 32, 2, 3, 128)
    _check_attention(raw, table, lens, cu, q, 32, out_dtype=torch.float16)
    ref, _, spread, score = page8.attention(q.double().numpy(), raw, table, 32, lens, 0.01, cu)
    packed = [torch.from_numpy(x).cuda() for x in raw]
    fused = torch.zeros(7, 10, 128, dtype=torch.bfloat16, device='cuda')
    fused[:5, 2:8] = q.cuda()
    out = torch.full((7, 12, 128), 5.0, dtype=torch.bfloat16, device='cuda')
    lse = torch.full((7, 6), 5.0, dtype=torch.float32, device='cuda')
    got = ops.page8_attention(fused[:, 2:8], packed, torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda().long(),
                              0.01, torch.from_numpy(cu).cuda().long(), out=out[:, 6:], lse=lse)
    tol, _ = attention_tolerance(ref, np.zeros((5, 6)), spread, score, raw, 90, 128, 2.0 ** -7)
    assert (np.abs(got[:5].double().cpu().numpy() - ref) <= tol).all()
    assert (out[5:] == 5).all() and (out[:, :6] == 5).all() and (lse[5:] == 5).all() and (lse[:5] != 5).all()


@pytest.mark.parametrize('dim,page', [(64, 16), (64, 128), (128, 32), (128, 64), (256, 16), (256, 64)])
def test_prompt_chunks(dim, page):
    """Many rows a request at every head size, small and large pages, beside requests with few rows and none; windows."""
    rng = np.random.default_rng(dim + page)
    lens, rows = [333, 64, 90, 500, 201], [300, 64, 0, 77, 201]
    case = _attention_case(rng, lens, rows, page, 2, 3, dim)
    _check_attention(*case, page, large=True)
    _check_attention(*case, page, window=70, sinks=3, large=True)
    _check_attention(*case, page, window=200, sinks=130, large=True)


@pytest.mark.parametrize('dim', [64, 128, 256])
def test_nan_in_prompt_chunks(dim):
    """A NaN value that some rows of a tile see and others do not; stale NaN bytes behind the last token."""
    rng = np.random.default_rng(dim)
    for page in (16, 64):
        raw, table, lens, cu, q = _attention_case(rng, [230], [100], page, 1, 4, dim)
        raw[1][table[0, 190 // page], 0, 7, 190 % page] = 0x7F
        raw[1][table[0, 140 // page], 0, dim - 1, 140 % page] = 0xFF
        raw[0][table[0, 229 // page], 0, 229 % page + 1:] = 0x7F
        raw[1][table[0, 229 // page], 0, :, 229 % page + 1:] = 0x7F
        _check_attention(raw, table, lens, cu, q, page)
        _check_attention(raw, table, lens, cu, q, page, window=60, sinks=2)


def test_many_prompts():
    """More entries than workgroups: whole entries in rounds, and runs across entries."""
    rng = np.random.default_rng(31)
    for lens, rows, heads in (([900] * 9, [700] * 9, 4), ([2100] * 5, [2000] * 5, 4)):
        _check_attention(*_attention_case(rng, lens, rows, 64, heads, 4, 64), 64, large=True)
    _check_attention(*_attention_case(rng, [1500] * 7, [1000] * 7, 64, 4, 2, 128), 64, window=300, sinks=4, large=True)


def test_a_long_prompt_cut_into_pieces():
    rng = np.random.default_rng(32)
    for dim, group in ((64, 4), (128, 8), (256, 2)):
        _check_attention(*_attention_case(rng, [9000], [100], 64, 1, group, dim), 64, large=True)
        _check_attention(*_attention_case(rng, [6000, 40], [9, 9], 32, 2, 5, dim), 32, large=True)


def test_many_requests():
    """More entries than lanes of a wave and threads of a workgroup, with and without row offsets, one of them long."""
    rng = np.random.default_rng(33)
    for n in (65, 300):
        lens = (rng.integers(1, 90, n)).tolist()
        lens[n // 2] = 4000
        _check_attention(*_attention_case(rng, lens, [1] * n, 16, 1, 4, 64), 16, pass_cu=False, large=True)
        _check_attention(*_attention_case(rng, lens, rng.integers(0, 2, n).tolist(), 16, 1, 4, 64), 16, large=True)
    lens = rng.integers(40, 90, 130).tolist()
    _check_attention(*_attention_case(rng, lens, [40] * 130, 16, 1, 4, 64), 16, large=True)


@pytest.mark.parametrize('dim,heads,group,n,most,window', [
    (128, 1, 2, 2500, 1, 0),        # decode: several entries to a thread of the plan
    (64, 2, 4, 70, 8, 0), (128, 2, 8, 90, 4, 100), (256, 1, 8, 70, 4, 0),        # 32 rows each
    (64, 1, 16, 70, 4, 50),         # 64 rows each
    (128, 2, 2, 540, 60, 0), (256, 1, 3, 300, 60, 90), (64, 3, 3, 300, 60, 0)])   # prompts
def test_large_batches(dim, heads, group, n, most, window):
    """More row tiles than a workgroup divides by itself: requests of 0 to `most` rows, one of them far longer than the
    others, one without tokens."""
    rng = np.random.default_rng(dim + n)
    rows = rng.integers(most // 2, most + 1, n) if most > 1 else rng.integers(0, 2, n)
    lens = np.maximum(rows, 1) + rng.integers(0, 40, n)
    lens[n // 3], rows[n // 2], lens[n // 5] = 5000, most, rows[n // 5]
    raw, table, lens, cu, q = _attention_case(rng, lens.tolist(), rows.tolist(), 16, heads, group, dim)
    _check_attention(raw, table, lens, cu, q, 16, window, 3 if window else 0, large=True)


@pytest.mark.parametrize('n,most', [(12, 3), (90, 3), (8, 60), (560, 30)])
def test_rows_before_the_first_request(n, most):
    """Offsets that do not begin at 0: the rows before them are left as they are, whichever way the work is divided."""
    rng = np.random.default_rng(38 + n)
    rows = rng.integers(1, most + 1, n)
    lens = rows + rng.integers(0, 60, n)
    raw, table, lens, cu, q = _attention_case(rng, lens.tolist(), rows.tolist(), 16, 1, 8, 128)
    s = n // 4
    at = int(cu[s])
    out = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device='cuda')
    pool = gpu_raw(raw)
    pool.attend(q.cuda(), torch.from_numpy(table[s:]).cuda(), torch.from_numpy(lens[s:]).cuda(), 0.01,
                torch.from_numpy(cu[s:]).cuda(), out=out)
    ref, lse, spread, score = attention_on_gpu(q[at:], raw, table[s:], 16, lens[s:], 0.01, cu[s:] - cu[s])
    tol, _ = attention_tolerance(ref, lse, spread, score, raw, int(lens.max()), 128, 2.0 ** -7)
    assert at > 0 and (out[:at] == 5).all()
    assert (np.abs(out[at:].double().cpu().numpy() - ref) <= tol).all()


def test_a_large_batch_in_a_graph():
    """A replay follows lengths that changed, where a plan is made on the device too."""
    rng = np.random.default_rng(36)
    n = 200
    raw, table, lens, cu, q = _attention_case(rng, rng.integers(200, 900, n).tolist(), [1] * n, 32, 2, 4, 64)
    pool, q, table, lens = gpu_raw(raw), q.cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda()
    out = torch.empty_like(q)
    pool.attend(q, table, lens, 0.02)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.attend(q, table, lens, 0.02, out=out)
    for step in range(4):
        lens.sub_(step * 60).clamp_(min=1)
        lens[17 * step] = table.shape[1] * 32 if step == 2 else 5
        want = pool.attend(q, table, lens, 0.02)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_calls_of_differing_shapes_share_a_workspace():
    """Calls whose partials lie at different places, one after the other in one workspace: each finds its counters zero."""
    rng = np.random.default_rng(34)
    cases = [_attention_case(rng, [5000], [100], 64, 1, 8, 128), _attention_case(rng, [4000, 100], [1, 1], 64, 1, 8, 64),
             _attention_case(rng, [3000], [200], 64, 2, 4, 64), _attention_case(rng, [6000], [1], 64, 4, 2, 256),
             _attention_case(rng, [5000, 3000], [4, 4], 64, 2, 8, 128)]
    pools = [gpu_raw(c[0]) for c in cases]
    ws = torch.zeros(128 << 20, dtype=torch.uint8, device='cuda')

    def run(i, w):
        raw, table, lens, cu, q = cases[i]
        return pools[i].attend(q.cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(), 0.02,
                               torch.from_numpy(cu).cuda(), ws=w)

    alone = [run(i, torch.zeros(128 << 20, dtype=torch.uint8, device='cuda')) for i in range(len(cases))]
    for i in (0, 1, 2, 3, 4, 2, 1, 0, 3, 4, 1):
        assert torch.equal(run(i, ws), alone[i])
        assert (ws[:65536] == 0).all()


def test_wide_windows_are_no_windows():
    rng = np.random.default_rng(35)
    raw, table, lens, cu, q = _attention_case(rng, [300, 70], [20, 1], 32, 1, 4, 64)
    pool = gpu_raw(raw)
    args = (q.cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(), 0.02, torch.from_numpy(cu).cuda())
    want = pool.attend(*args)
    for window, sinks in ((300, 0), (1 << 30, 5), ((1 << 31) - 1, 1 << 40), (1 << 50, 0)):
        assert torch.equal(pool.attend(*args, window=window, sinks=sinks), want)


def test_same_result_every_time():
    rng = np.random.default_rng(21)
    raw, table, lens, cu, q = _attention_case(rng, [5000, 900, 2000], [1, 1, 1], 64, 2, 8, 128)
    pool = gpu_raw(raw)
    args = (q.cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(), 0.02)
    first = pool.attend(*args)
    for _ in range(5):
        assert torch.equal(pool.attend(*args).view(torch.int16), first.view(torch.int16))


def test_two_streams_and_two_graphs():
    """Calls on two streams and replays of two captured graphs, interleaved with eager calls, agree with the eager
    results; the second replay follows lengths that changed."""
    rng = np.random.default_rng(22)
    cases = []
    for lens in ([3000, 40, 1200], [2500, 2500]):
        raw, table, lens, cu, q = _attention_case(rng, lens, [1] * len(lens), 64, 2, 4, 128)
        pool = gpu_raw(raw)
        cases.append((pool, q.cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda()))
    run = lambda c, out=None: c[0].attend(c[1], c[2], c[3], 0.02, out=out)
    want = [run(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(4):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                outs[i].append(run(c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    graphs, got = [], []
    for c in cases:
        got.append(torch.empty_like(c[1]))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(c, got[-1])
        graphs.append(g)
    for step in range(4):
        if step == 2:
            for c in cases:
                c[3].sub_(77).clamp_(min=1)
            want = [run(c) for c in cases]
        for o in got:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(got, want))
        assert torch.equal(run(cases[0]), want[0])


def test_append_then_attend():
    """A serving run: prompts in chunks, then decode steps, the pool's own bytes read back by the oracle."""
    rng = np.random.default_rng(23)
    page, heads, group, dim = 32, 2, 4, 64
    pool = Page8Pool(24, page, heads, dim)
    lens = np.zeros(3, np.int32)
    table = rng.permutation(24)[:18].reshape(3, 6).astype(np.int32)
    t_table = torch.from_numpy(table).cuda()
    for rows in ([40, 3, 0], [33, 64, 90], [1, 1, 1], [1, 1, 1], [4, 4, 4]):
        cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        lens = (lens + np.array(rows)).astype(np.int32)
        k, v = (bf16(rng.standard_normal((cu[-1], heads, dim)) * 3) for _ in range(2))
        q = bf16(rng.standard_normal((cu[-1], heads * group, dim)))
        one = rows == [1, 1, 1]
        pool.append(k.cuda(), v.cuda(), t_table, torch.from_numpy(lens).cuda(),
                    None if one else torch.from_numpy(cu).cuda())
        raw = tuple(x.cpu().numpy() for x in pool.raw)
        _check_attention(raw, table, lens, cu, q, page, 50, 3, scale=0.125, pass_cu=not one, pool=pool)
