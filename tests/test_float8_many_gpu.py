"""Attention of single tokens over pages of codes for more requests than one launch takes (256): portions, requests without tokens, long ones in parts."""
import pytest

from tests.test_float8_gpu import check_attention, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def requests_of(n, long):
    """Ragged single tokens; every 50th request is long (its tiles fall to several CTAs), some have no token, some a portion."""
    lens = [(1, 1 + (37 * i) % 300) for i in range(n)]
    for i in range(0, n, 50):
        lens[i] = (1, long - i)
    for i in range(7, n, 31):
        lens[i] = (0, 5)
    for i in range(11, n, 90):
        lens[i] = (40, 100)
    for i in range(12, n, 120):
        lens[i] = (3, 70)
    lens[-1] = (1, long)
    return lens


@pytest.mark.parametrize("n", [256, 257, 300, 513])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(4, 1, 64, 32), (2, 2, 128, 32), (16, 1, 64, 16)])
def test_more_requests_than_a_launch_takes(ops, n, heads, kv_heads, hd, page):  # noqa: F811
    check_attention(ops, heads, kv_heads, hd, page, requests_of(n, 6000), seed=n)


def test_more_requests_than_a_launch_takes_in_a_window(ops):  # noqa: F811
    check_attention(ops, 4, 1, 64, 32, requests_of(300, 3000), window=500, seed=1)


def test_several_hundred_requests_of_few_heads_and_short_ones(ops):  # noqa: F811
    check_attention(ops, 4, 2, 64, 32, [(1, 1 + i % 40) for i in range(600)], seed=2)
