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
    """A result in bfloat16 is off by 2^-8 of itself, and by the weights' roundings: 2^-8 of the magnitudes' sum at most (two codes; three and
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


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("lens", [[(1, 200), (1, 70)], [(1, 2600), (1, 900)], [(130, 200), (1, 70), (40, 100)]])
def test_a_page_of_large_values_without_weight(ops, heads, kv_heads, hd, page, far, lens):  # noqa: F811
    """Scores of the page lie more than 280 powers of two below the others: whatever its values, they count for nothing."""
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, page, lens, far + hd)
    for r in range(len(lens)):
        at = table[r, 1].long()
        k[at, :, :, 0] = -448.0
        vs[at] = 2.0 ** (far - 7)
    q[..., 0] = 300 * math.log(2) / (scale * 448 * 2.0 ** -7)
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, scale, 0, page)
    check(attend(ops, *args, lens), *args)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(4, 1, 64, 32), (2, 1, 128, 32), (2, 2, 64, 16), (6, 2, 48, 32), (40, 2, 64, 32)])
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("lens", [[(2, 33)], [(4, 130), (1, 33)], [(140, 161)], [(300, 321), (40, 65)]])
def test_a_page_of_large_values_behind_a_row(ops, heads, kv_heads, hd, page, far, lens):  # noqa: F811
    """The last page belongs to the last tokens: earlier rows of the same tile may not read it and know nothing of its scale."""
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, page, lens, far + hd)
    for r, (_, n) in enumerate(lens):
        vs[table[r, (n - 1) // page].long()] = 2.0 ** (far - 7)
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, scale, 0, page)
    if far == 127:                      # rows that read the page overflow: they are left out
        out, (want, mag) = attend(ops, *args, lens), plain.attention(*args)
        rows = (want.abs().amax(1) < 2.0 ** 60)
        assert rows.sum() >= len(lens)
        assert ((out.double() - want).abs() <= 2.0 ** -8 * (want.abs() + 1.5 * mag) + 2.0 ** -20)[rows].all()
    else:
        check(attend(ops, *args, lens), *args)


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("lens", [[(1, 150), (1, 40)], [(1, 5000)], [(1, 300 + 170 * i) for i in range(24)], [(5, 640), (200, 700)]])
@pytest.mark.parametrize("window", [0, 100])
def test_pages_of_every_size(ops, heads, kv_heads, hd, page, lens, window):  # noqa: F811
    """Scales of values from 2^-40 to 2^40, of keys from 2^-10 to 2^-6, in any order: parts of a request have references of their own."""
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, page, lens, hd + len(lens))
    g = gen(hd)
    vs = torch.pow(2.0, torch.randint(-40, 41, vs.shape, generator=g).float())
    ks = torch.pow(2.0, torch.randint(-10, -5, ks.shape, generator=g).float())
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, scale, window, page)
    check(attend(ops, *args, lens), *args)


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("lens", [[(1, 96), (1, 70)], [(1, 3000)], [(130, 200), (40, 100)]])
@pytest.mark.parametrize("size", [-100, 8, 40])
def test_pages_of_zeros_count_in_the_denominator(ops, heads, kv_heads, hd, page, lens, size):  # noqa: F811
    """Pages of zeros have the smallest scale there is, 2^-100: their weight is in the sum of weights, next to values of any size."""
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, page, lens, hd)
    vs.fill_(2.0 ** size)
    for r, (_, n) in enumerate(lens):
        for j in range(0, -(-n // page), 2):
            at = table[r, j].long()
            v[at], vs[at] = 0.0, 2.0 ** -100
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, scale, 0, page)
    check(attend(ops, *args, lens), *args)


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES + [(40, 2, 64, 32)])
@pytest.mark.parametrize("lens", [[(1, 90), (1, 300)], [(1, 5000)], [(150, 200), (3, 40)]])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(ops, heads, kv_heads, hd, page, lens, bad):  # noqa: F811
    """An infinite channel makes scores that are infinite or no numbers, and a softmax of these is no number."""
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, page, lens, hd)
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (k8, v8, ks, vs, table, cu, kv, scale, 0, page)
    spoilt = q.clone()
    spoilt[0, 1, 5] = bad
    out = attend(ops, spoilt, *args, lens).view(q.shape)
    assert torch.isnan(out[0, 1]).all()
    want, mag = (t.view(q.shape) for t in plain.attention(q, *args))
    keep = torch.ones(q.shape[:2], dtype=torch.bool)
    keep[0, 1] = False
    err = (out.double() - want).abs()
    assert (err <= 2.0 ** -8 * (want.abs() + 1.5 * mag) + 1e-30)[keep].all()


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES[:4])
@pytest.mark.parametrize("lens", [[(1, 90), (1, 30)], [(1, 2500)]])
def test_single_tokens_with_a_channel_far_above_the_others(ops, heads, kv_heads, hd, page, lens):  # noqa: F811
    """The keys have nothing in the large channel: the others, down to 2^-14 of it, make the scores, and are exact (bfloat16's eight bits are
    the four of a code and the four of what it leaves, in units of 1/16)."""
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, page, lens, hd)
    g = gen(3)
    q = torch.pow(2.0, -14 * torch.rand(q.shape, generator=g)) * torch.where(torch.rand(q.shape, generator=g) < 0.5, -1.0, 1.0) * 2.0 ** 14
    low = torch.rand(q.shape[:2] + (hd // 2,), generator=g) + 1           # half of them between 1 and 2: the smallest
    q[..., hd // 2:] = low
    q[..., 0] = 2.0 ** 14 * 1.75
    k[..., :hd // 2] = 0.0
    ks = torch.full_like(ks, 2.0 ** -8)
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, 4.0, 0, page)
    check(attend(ops, *args, lens), *args)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(4, 1, 64, 32), (4, 4, 128, 32)])
@pytest.mark.parametrize("above", [8, 12])
def test_portions_with_a_channel_far_above_the_others(ops, heads, kv_heads, hd, page, above):  # noqa: F811
    """Both of a query's codes are in the unit of the first, 2^-9 of the scale at least: a channel is off by 2^-10 of it, and a score by as much for
    every channel of the key."""
    lens = [(130, 200), (40, 100)]
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, page, lens, hd)
    q[..., 0] = 1.75 * 2.0 ** above                                       # 448 times 2^(above - 8)
    q[..., 1:] = q[..., 1:].clamp(-3, 3)
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, scale, 0, page)
    out, (want, mag) = attend(ops, *args, lens), plain.attention(*args)
    score_off = 2.0 ** (above - 18) * float(k8.float().abs().sum(-1).max()) * 2.0 ** -7 * scale
    assert ((out.double() - want).abs() <= 2.0 ** -8 * (want.abs() + 1.5 * mag) + math.expm1(2 * score_off) * mag).all()


@pytest.mark.parametrize("heads,kv_heads,hd,page,new", [(32, 4, 64, 32, 1), (64, 8, 128, 32, 1), (64, 4, 128, 32, 1), (8, 8, 64, 32, 40), (8, 8, 128, 32, 40),
                                                        (6, 2, 48, 32, 40)])
def test_the_weights_last_bits(ops, heads, kv_heads, hd, page, new):  # noqa: F811
    """Few keys whose values cancel but for the weights' differences, so that the result's own rounding hides little; and that rounding is allowed for
    exactly: the result lies between the exact one, less and more what weights may be off by, each rounded to bfloat16. A weight is off
    by 2^-12 of itself (three codes of four bits; halves 2^-11; two codes, for groups of more than eight heads, 2^-8), its exponential by
    2^-21 and, through the score's roundings, by 2^-20 of the score; the queries are exact."""
    group = heads // kv_heads
    lens = [(new, max(new, 2 + i % 5)) for i in range(24)]
    cu, kv, table, q, k, v, ks, vs, _ = case(heads, kv_heads, hd, page, lens, hd)
    q = (torch.randint(-64, 65, q.shape, generator=gen(1)) / 32.0)                      # seven bits, every channel above 2^-11 of the largest or zero
    v = torch.where(torch.rand(v.shape, generator=gen(2)) < 0.5, -256.0, 256.0)
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, 0.1, 0, page)
    out = attend(ops, *args, lens)
    want, mag = plain.attention(*args)
    unit = 2.0 ** -11 if new > 1 else 2.0 ** -12 if group <= 8 else 2.0 ** -8
    off = (unit + 2.0 ** -15) * mag
    low, high = ((want + sign * off).to(torch.float32).to(torch.bfloat16) for sign in (-1, 1))
    assert ((low <= out) & (out <= high)).all()


@pytest.mark.parametrize("heads,kv_heads,hd", [(40, 2, 64), (34, 2, 128), (128, 1, 64), (16, 1, 64)])
def test_groups_of_many_heads_beside_requests_without_tokens(ops, heads, kv_heads, hd):  # noqa: F811
    lens = [(0, 7), (1, 90), (0, 0), (3, 33)]
    cu, kv, table, q, k, v, ks, vs, scale = case(heads, kv_heads, hd, 32, lens, hd)
    q, k8, v8 = q.to(torch.bfloat16), k.to(E4M3), v.to(E4M3)
    args = (q, k8, v8, ks, vs, table, cu, kv, scale, 0, 32)
    check(attend(ops, *args, lens), *args)
