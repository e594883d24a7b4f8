"""Known answers for the paged cache's oracle."""

import numpy as np
import torch

from oracle import paged


def test_codes_are_those_of_the_format():
    assert paged.E4M3[0x7E] == 448 and paged.E4M3[1] == 2.0 ** -9 and paged.E4M3[0x38] == 1 and paged.E4M3[0xC0] == -2
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(paged.E4M3, table)


def test_exponents_are_the_least_that_fit():
    x = np.array([[448.0], [448.0 + 2.0 ** -15], [0.0], [1e-44], [1.0], [3.5], [3.5625], [65504.0], [3.38e38], [np.inf]])
    assert paged.row_exponents(x).tolist() == [127, 128, 1, 1, 119, 120, 121, 135, 247, 1]


def test_rounding_is_to_nearest_even():
    x = np.array([[448, 17, 19, 18, 1.0625, 1.1875, -0.0, 2.0 ** -10, 3 * 2.0 ** -10, np.nan, -np.inf, 2.0 ** -30]])
    codes, e = paged.encode(x, "f32")
    assert e.tolist() == [127]
    want = torch.tensor(np.where(np.isfinite(x), x, np.nan), dtype=torch.float32).to(torch.float8_e4m3fn)
    np.testing.assert_array_equal(paged.E4M3[codes], want.double().numpy())
    assert codes[0, 6] == 0x80


def test_random_rows_match_torch_conversion():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((300, 64)) * np.exp2(rng.integers(-140, 127, (300, 1)))).astype(np.float32)
    codes, e = paged.encode(x, "f32")
    y = torch.from_numpy((x.astype(np.float64) * np.exp2(127.0 - e)[:, None]).astype(np.float32)).to(torch.float8_e4m3fn)
    np.testing.assert_array_equal(codes, y.view(torch.uint8).numpy())
    back = paged.decode(codes, e)
    # (the largest is above 224 steps of 2^e, and e4m3's even steps begin below 2^-6: 2^-13.8 of it)
    big = (np.abs(x) >= 2.0 ** -13 * np.abs(x).max(-1, keepdims=True)) & (e > 1)[:, None]
    assert (np.abs(back - x)[big] <= 2.0 ** -4 * np.abs(x)[big]).all()


def test_values_read_back_inside_their_type():
    codes, e = paged.encode(np.array([[65504.0, -65504.0]]), "f16")
    assert paged.decode(codes, e).tolist() == [[61440.0, -61440.0]]
    most = float(torch.finfo(torch.bfloat16).max)
    codes, e = paged.encode(np.array([[most]]), "bf16")
    assert np.isfinite(paged.decode(codes, e).astype(np.float32)).all()


def test_append_gather_and_attention():
    pool = np.full((5, 4, 1, 2), -1.0)
    table = np.array([[3, -1], [0, 4]])
    new = np.arange(2 * 3 * 1 * 2, dtype=np.float64).reshape(2, 3, 1, 2)
    got, lengths = paged.append(pool, new, table, [2, 3], [3, 2])
    assert lengths.tolist() == [5, 5]
    assert got[3, 2, 0].tolist() == [0, 1] and got[3, 3, 0].tolist() == [2, 3]  # the third has no page
    assert got[0, 3, 0].tolist() == [6, 7] and got[4, 0, 0].tolist() == [8, 9]
    assert (got != pool).any(-1).sum() == 4
    rows, there = paged.gather(got, table, [5, 5], 6)
    assert there.tolist() == [[True] * 4 + [False] * 2, [True] * 5 + [False]]
    q = np.ones((2, 2, 1, 2))
    res = paged.paged_decode(q, rows, rows, there, [5, 1], 1.0)
    assert np.isposinf(res["lse"][1, 0, 0]) and not res["out"][1, 0].any()  # the first of two tokens, one key
    np.testing.assert_allclose(res["out"][1, 1, 0], rows[1, 0, 0])
    s = rows[0, :4, 0].sum(-1)
    np.testing.assert_allclose(res["lse"][0, 0, 1], np.log(np.exp(s).sum()))
