"""Cuts of products with nearly 2^31 tokens, the most that are taken."""
import pytest
import torch  # noqa: F401  (loads what the extension links)

B200 = [0, 148, 74, 45, 33, 26, 22, 15, 15]
MOST = 2 ** 31 - 512       # a tile that ends behind the last token still has 32-bit coordinates


@pytest.mark.parametrize("m", [2 ** 30, 2 ** 31 - 9_000_000, 2 ** 31 - 8_000_000, 2 ** 31 - 1025, MOST])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 16), (3, 300)])
def test_every_token_is_in_a_tile(m, n, k):
    native = pytest.importorskip("kunserve_b200._C")
    for el in (2, 4):
        p = native.int8_plan(m, n, k, el, B200)
        assert 16 <= p["width"] <= 256 and p["splits"] == 1
        assert (p["token_tiles"] - 1) * p["width"] < m <= p["token_tiles"] * p["width"] < 2 ** 31
        assert 0 < p["grid"] <= 2 * 148 and 1 <= p["group"] <= p["token_tiles"]
