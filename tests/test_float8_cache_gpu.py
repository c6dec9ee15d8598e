"""Cache writes in 8 bits where the block table has no page for a position."""
import pytest
import torch

from tests.plain import float8_plain as plain
from tests.test_float8_gpu import batch, cuda, gen, ops, pools_of  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 128, 32), (4, 2, 64, 16), (3, 1, 48, 8)])
@pytest.mark.parametrize("lens", [[(70, 100), (1, 5)], [(1, 100), (1, 70), (1, 3)]])
@pytest.mark.parametrize("missing", ["behind the table", "given back"])
def test_queries_of_positions_without_a_page(ops, heads, kv_heads, hd, page, lens, missing):  # noqa: F811
    """The queries of all tokens are rotated and written; keys and values of positions without a page go nowhere."""
    cu, kv, table, pages = batch(lens, page, seed=hd)
    g = gen(hd)
    T = int(cu[-1])
    qkv = torch.randn(T, (heads + 2 * kv_heads) * hd, generator=g)
    angle = torch.rand(T, hd // 2, generator=g) * 1000
    cs = torch.stack([angle.cos(), angle.sin()], -1).contiguous()
    k8, v8, ks, vs = pools_of(pages, kv_heads, page, hd, 1)
    cut = 100 // page                                          # the first request's last page
    given, seen = table.clone(), table.clone()
    given[0, cut:] = -1
    seen = given[:, :cut].contiguous() if missing == "behind the table" else given
    dev = cuda(k8, v8, ks, vs)
    q_out = torch.full((T, heads, hd), 7.0, device="cuda")
    ops.kv_append_float8(qkv.cuda(), q_out, *dev, *cuda(cu, kv, seen), heads, kv_heads, hd, cs.cuda(), False, page)
    q, pools, scales = plain.append(qkv, (k8, v8), (ks, vs), cu, kv, given, heads, kv_heads, hd, cs, False, page)
    assert torch.equal(q_out.cpu(), q)
    for got, want in ((dev[0], pools[0]), (dev[1], pools[1]), (dev[2], scales[0]), (dev[3], scales[1])):
        assert torch.equal(got.cpu().double(), want)
