"""The CPU restatement of the 8-bit pages against hand-made values and torch's own E4M3 conversion."""
import math

import numpy as np
import torch

from oracle import page8


def test_e4m3_bytes_equal_the_torch_cast():
    gen = torch.Generator().manual_seed(3)
    x = torch.cat([torch.randn(4000, generator=gen) * 2.0 ** torch.randint(-14, 9, (4000,), generator=gen),
                   torch.tensor([0.0, -0.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 448.0, -448.0, 447.0, 0.0146484375])])
    x = x.clamp(-448, 448)
    assert np.array_equal(page8.e4m3_bytes(x.numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    got = page8.e4m3_bytes(np.array([500.0, -1e30, np.inf, -np.inf, np.nan]))
    assert got.tolist() == [0x7E, 0xFE, 0x7E, 0xFE, 0x7F]
    vals = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(page8.e4m3_values(), vals, equal_nan=True)


def test_exponents():
    assert page8.exponent_for(448.0) == 127 and page8.exponent_for(448.5) == 128
    assert page8.exponent_for(0.0) == 63 and page8.exponent_for(3.4e38) == 246


def test_append_grows_a_scale_and_starts_a_page_anew():
    raw = (np.zeros((2, 1, 16, 2), np.uint8), np.zeros((2, 1, 2, 16), np.uint8), np.full((2, 1), 200, np.uint8),
           np.full((2, 1), 200, np.uint8))
    table = np.array([[1]], dtype=np.int32)
    x = np.array([[[448.0, 1.0]]])
    page8.append(x, x, raw, table, 16, np.array([1]))
    assert raw[2][1, 0] == 127 and raw[0][1, 0, 0].tolist() == [0x7E, 0x38]     # the old exponent 200 is gone
    page8.append(8 * x, 8 * x, raw, table, 16, np.array([2]))
    assert raw[2][1, 0] == 130 and raw[0][1, 0, 0].tolist() == [0x66, 0x20]     # 56 and 0.125: exact
    assert raw[1][1, 0, :, :2].tolist() == [[0x66, 0x7E], [0x20, 0x38]]
    page8.append(x, x, raw, table, 16, np.array([3]))
    assert raw[2][1, 0] == 130 and raw[0][1, 0, 2].tolist() == [0x66, 0x20]


def test_attention_by_hand():
    raw = (np.zeros((1, 1, 16, 2), np.uint8), np.zeros((1, 1, 2, 16), np.uint8), np.full((1, 1), 127, np.uint8),
           np.full((1, 1), 128, np.uint8))
    raw[0][0, 0, :3] = [[0x38, 0], [0, 0x38], [0x40, 0]]            # keys (1, 0), (0, 1), (2, 0)
    raw[1][0, 0, 0, :3] = [0x38, 0x40, 0x44]                        # values 1, 2, 3 (times 2)
    table = np.zeros((1, 1), np.int32)
    q = np.tile(np.array([[[1.0, 0.0]]]), (3, 1, 1))
    cu = np.array([0, 3])
    out, lse, _, _ = page8.attention(q, raw, table, 16, np.array([3]), 1.0, cu)
    e = math.e
    assert np.allclose(out[:, 0, 0], [2, (2 * e + 4) / (e + 1), (2 * e + 4 + 6 * e * e) / (e + 1 + e * e)])
    assert np.allclose(lse[:, 0], [1, math.log(e + 1), math.log(e + 1 + e * e)])
    out, _, _, _ = page8.attention(q, raw, table, 16, np.array([3]), 1.0, cu, window=1, sinks=1)
    assert np.allclose(out[:, 0, 0], [2, (2 * e + 4) / (e + 1), (2 * e + 6 * e * e) / (e + e * e)])


def test_pages_by_hand():
    refs, table, lens = np.zeros(6, np.int32), np.full((4, 3), -1, np.int32), np.zeros(4, np.int32)
    assert page8.extend(refs, table, lens, np.array([20, 0, 16, 0]), 16).tolist() == [True] * 4
    assert table.tolist() == [[0, 1, -1], [-1] * 3, [2, -1, -1], [-1] * 3] and refs.tolist() == [1, 1, 1, 0, 0, 0]
    moves = page8.fork(refs, table, lens, np.array([0, 0, 2]), np.array([1, 1, 3]), 16)
    assert moves.tolist() == [[1, -1, -1], [3, -1, -1]]
    assert table.tolist() == [[0, 1, -1], [0, 3, -1], [2, -1, -1], [2, -1, -1]] and refs.tolist() == [2, 1, 2, 1, 0, 0]
    page8.free(refs, table, lens, np.array([0, 2, 2]))
    assert refs.tolist() == [1, 0, 1, 1, 0, 0] and lens.tolist() == [0, 20, 0, 16]
    moves, count = page8.compact(refs, table)
    assert count == 1 and moves.tolist() == [[3, -1, -1], [1, -1, -1]]
    assert table.tolist() == [[-1] * 3, [0, 1, -1], [-1] * 3, [2, -1, -1]] and refs.tolist() == [1, 1, 1, 0, 0, 0]
    assert page8.extend(refs, table, lens, np.array([33, 0, 48, 16]), 16).tolist() == [True, True, False, False]
