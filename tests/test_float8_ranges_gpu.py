"""Attention over pages of codes where values lie far apart: pages whose scales differ by up to 2^127, hidden from a row, without weight in it or
ruling it; queries with one channel far above the others, infinite ones and ones that are no numbers; weights to their last bits."""
import math

import pytest
import torch

from tests.plain import float8_plain as plain
from tests.test_float8_gpu import E4M3, batch, cuda, gen, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def attend(ops, q, k8, v8, ks, vs, table, cu, kv, scale, window, page, lens):
    T, heads, hd = q.shape
    out = torch.full((T, heads * hd), math.nan, dtype=q.dtype, device="cuda")
    new = [n for n, _ in lens]
    ops.paged_attention_float8(*cuda(q, k8, v8, ks, vs, table, cu, kv), out, scale, window, page, len(lens), max(new), max(n for _, n in lens),
                               min_q_len=min(new))
    ops.check_float8_errors()
    return out.cpu()


def check(out, q, k8, v8, ks, vs, table, cu, kv, scale, window, page):
    """A result in bfloat16 is off by 2^-9 of itself, and by the weights' roundings: 2^-8 of the magnitudes' sum at most (two codes; three and
    halves less). What is 2^-22 of the row's largest weight times its scale or less may be gone, times a code of 448 a key."""
    want, mag = plain.attention(q, k8, v8, ks, vs, table, cu, kv, scale, window, page)
    ones = torch.ones(v8.shape, dtype=torch.float32).to(E4M3)
    ruling, _ = plain.attention(q, k8, ones, ks, vs, table, cu, kv, scale, window, page)       # the sum of weights times scales
    err = (out.double() - want).abs()
    bound = 2.0 ** -8 * (want.abs() + 1.5 * mag) + int(kv.max()) * 448 * 2.0 ** -22 * ruling + 1e-30
    assert torch.isfinite(out).all(), "a result is not a number"
    assert (err <= bound).all(), f"worst {(err / bound).max().item():.3g} of the bound"


def case(heads, kv_heads, hd, page, lens, seed):
    """Queries, codes and scales; channel 0 of keys and queries is free to raise or lower a key's score."""
    cu, kv, table, pages = batch(lens, page, seed=seed)
    g = gen(seed)
    q = torch.randn(int(cu[-1]), heads, hd, generator=g)
    k = (torch.randn(pages, kv_heads, page, hd, generator=g) * 100).clamp(-448, 448)
    v = (torch.randn(pages, kv_heads, page, hd, generator=g) * 100).clamp(-448, 448)
    k[..., 0], q[..., 0] = 0.0, 8.0
    ks, vs = torch.full((pages, kv_heads), 2.0 ** -7), torch.full((pages, kv_heads), 2.0 ** -7)
    return cu, kv, table, q, k, v, ks, vs, 1.0 / math.sqrt(hd)


SHAPES = [(4, 1, 64, 32), (32, 8, 128, 32), (16, 1, 128, 32), (12, 1, 64, 16), (6, 2, 48, 32)]
FAR = [10, 20, 30, 40, 127]            # powers of two (of pages whose other scales are 2^-7; 2^120 is the largest there is)


@pytest.mark.parametrize("heads,kv_heads,hd", [(40, 2, 64), (34, 2, 128), (128, 1, 64), (16, 1, 64)])
def test_groups_of_many_heads_beside_requests_without_tokens(ops, heads, kv_heads, hd):  # noqa: F811
    lens = [(0, 7), (1, 90), (0, 0), (3, 33)]
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, 32, lens, hd)
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, scale, 0, 32)
    check(attend(ops, *args, lens), *args)
