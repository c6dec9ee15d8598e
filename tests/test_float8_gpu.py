"""The 8-bit kernels against plain 64-bit forms: products, cache writes and attention, at the sizes, layouts, lengths and
values where they can go wrong; what they refuse; and that results do not depend on what scratch memory or pages held before."""
import math

import pytest
import torch

from tests.plain import float8_plain as plain

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from garuda_b200.kernels.ops import CudaOps
    return CudaOps("cuda:0")


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ products

def operands(M, N, K, dtype, seed=0):
    g = gen(seed + 7 * M + 11 * N + 13 * K)
    a = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(K, generator=g))).to(dtype)
    w = torch.randn(N, K, generator=g) * 0.05
    return a, w


def check_product(got, a, w8, exact=None, before=None, alpha=1.0):
    """Rounding of the result: 2^-9 of it in bfloat16, 2^-24 in 32 bits. Sums: a block's 128 products and the blocks are added in 32
    bits, at most 128 + K / 128 roundings of 2^-24 of the magnitudes' sum, and the tensor cores' own sums may be cut off, not
    rounded: 2^-13 of that sum is far above all of these and far below a lost product."""
    want, mag = plain.linear(a, w8.values.cpu().double(), w8.scales.cpu())
    if before is not None:
        want = before.double() + alpha * want
    unit = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -22
    err = (got.cpu().double() - want).abs()
    bound = unit * want.abs() + 2.0 ** -13 * mag * abs(alpha) + 1e-30
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"worst {(err / bound).max().item():.2f} of the bound"


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 128), (1, 2048, 2048), (2, 127, 100), (5, 129, 129), (7, 1000, 2056), (8, 384, 4096),
                                   (16, 256, 16), (17, 130, 1000), (33, 640, 520), (64, 1, 256), (65, 512, 640), (100, 2048, 384),
                                   (129, 300, 272), (150, 1111, 1030), (256, 128, 512), (257, 264, 648), (301, 512, 1376), (512, 257, 256),
                                   (513, 300, 384), (700, 513, 200), (1025, 1024, 144), (40, 18000, 130)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_products(ops, M, N, K, out_dtype):
    a, w = operands(M, N, K, torch.bfloat16)
    w8 = ops.float8_weight(w.cuda())
    codes, scales = plain.weight(w) if N * K <= 300_000 else (None, None)
    if codes is not None:
        assert torch.equal(w8.values.cpu().double(), codes) and torch.equal(w8.scales.cpu().double(), scales)
    out = torch.full((M, N), math.nan, dtype=out_dtype, device="cuda")
    ops.linear_float8(a.cuda(), w8, out)
    check_product(out, a, w8)
    again = torch.full_like(out, math.nan)
    ops.linear_float8(a.cuda(), w8, again)
    assert torch.equal(out, again)              # whoever finishes last adds in the same order
    ops.check_float8_errors()


@pytest.mark.parametrize("M,N,K", [(1, 200, 300), (9, 128, 2048), (130, 257, 520), (600, 512, 384)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_accumulate(ops, M, N, K, dtype):
    a, w = operands(M, N, K, dtype, seed=1)
    w8 = ops.float8_weight(w.to(dtype).cuda())
    before = torch.randn(M, N, generator=gen(3))
    for alpha in (1.0, -0.37):
        out = before.clone().cuda()
        ops.linear_float8(a.cuda(), w8, out, accumulate=True, alpha=alpha)
        check_product(out, a, w8, before=before, alpha=alpha)


def test_products_of_strided_rows_and_scales_of_any_size(ops):
    """Tokens as a slice of wider rows that start on two bytes; scales far apart; one that is no power of two spoils its rows, loudly."""
    M, N, K = 37, 200, 333
    a, w = operands(M, N, K, torch.bfloat16, seed=2)
    wide = torch.zeros(M, K + 10, dtype=torch.bfloat16)
    wide[:, 3:3 + K] = a
    w8 = ops.float8_weight(w.cuda())
    w8 = type(w8)(w8.values, w8.scales * torch.pow(2.0, torch.randint(-30, 30, w8.scales.shape, generator=gen(4)).float()).cuda())
    out = torch.empty(M, N, dtype=torch.float32, device="cuda")
    ops.linear_float8(wide.cuda()[:, 3:3 + K], w8, out)
    check_product(out, a, w8)
    for wrong in (w8.scales[1, 2].item() * 1.5, -1.0, 0.0, math.nan):
        spoilt = w8.scales.clone()
        spoilt[1, 2] = wrong
        ops.linear_float8(wide.cuda()[:, 3:3 + K], (w8.values, spoilt), out)
        assert torch.isnan(out[:, 128:]).all()
        check_product(out[:, :128], a, type(w8)(w8.values[:128], w8.scales[:1]))


def test_codes_at_the_ends_of_their_range(ops):
    """Zeros, subnormal and huge numbers, infinities and NaN, numbers half way between two codes, and blocks whose largest is 448 times a power of
    two or just above."""
    K = 256
    w = torch.zeros(9 * 128, K)
    g = gen(5)
    w[:128] = 0.0
    w[128:256] = torch.randn(128, K, generator=g) * 1e-38
    w[256:384] = torch.randn(128, K, generator=g) * 1e36
    w[384:512] = torch.randn(128, K, generator=g)
    w[384, 0], w[385, 1], w[386, 200] = math.inf, -math.inf, math.nan
    w[512:640] = torch.arange(-64, 64)[:, None] / 16 + 2.0 ** -4 / 2          # ties
    w[640:768, :] = torch.rand(128, K, generator=g)
    w[640, 5] = 448.0
    w[641, 130] = 448.0 * (1 + 2.0 ** -20)
    w[768:896] = -0.0
    w[896:1024] = torch.randn(128, K, generator=g) * 2.0 ** -120
    w[1024:] = torch.randn(128, K, generator=g) * torch.exp(8 * torch.randn(128, K, generator=g))
    w8 = ops.float8_weight(w.cuda())
    codes, scales = plain.weight(w)
    assert torch.equal(w8.scales.cpu().double(), scales)
    got = w8.values.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(codes)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(codes))
    # the same numbers as tokens: a product with the identity gives the rounded tokens back, block by block
    one = ops.float8_weight(torch.eye(K).cuda())
    out = torch.empty(w.shape[0], K, device="cuda")
    safe = torch.nan_to_num(w, nan=1.0, posinf=3.0, neginf=-3.0)
    ops.linear_float8(safe.cuda(), one, out)
    want = plain.rows(safe)
    assert torch.allclose(out.cpu().double(), want, rtol=2.0 ** -20, atol=0.0)


def test_a_token_that_is_not_a_number_spoils_its_own_row_only(ops):
    a, w = operands(20, 300, 400, torch.bfloat16, seed=6)
    a[7, 33] = math.nan
    w8 = ops.float8_weight(w.cuda())
    out = torch.empty(20, 300, device="cuda")
    ops.linear_float8(a.cuda(), w8, out)
    assert torch.isnan(out[7]).all()
    keep = [i for i in range(20) if i != 7]
    check_product(out[keep], a[keep], w8)


@pytest.mark.parametrize("M,N,K", [(1, 64, 16), (1, 256, 5632), (3, 130, 100), (17, 200, 392), (150, 300, 272), (260, 128, 1376)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_of_a_gated_pair(ops, M, N, K, dtype):
    """silu(gate) * up is 32-bit: the exponential (2 units), a sum, a quotient and a product, 2^-20 of it at most in all. Where the exact
    value lies nearer than 2^-19 of itself to the middle of two codes, the code may be the other one: a step, 2^-3 of the value
    (2^-9 of the scale below the normal numbers)."""
    g = gen(M + N + K)
    pair = (torch.randn(M, 2 * K, generator=g) * 3).to(dtype)
    w = torch.randn(N, K, generator=g) * 0.05
    w8 = ops.float8_weight(w.cuda())
    gate, up = pair.double().split(K, 1)
    a = gate / (1 + torch.exp(-gate)) * up
    want, mag = plain.linear(a, w8.values.cpu().double(), w8.scales.cpu())
    blocks = -(-K // 128)
    padded = torch.nn.functional.pad(a, (0, blocks * 128 - K))
    scale = plain.scales_of(padded.view(M, blocks, 128).abs().amax(-1)).repeat_interleave(128, 1)[:, :K]
    low, high = plain.encode(a * (1 - 2.0 ** -19) / scale), plain.encode(a * (1 + 2.0 ** -19) / scale)
    dense = w8.values.cpu().double() * w8.scales.cpu().double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    flips = torch.where(low != high, a.abs() * 2.0 ** -3 + scale * 2.0 ** -9, 0.0) @ dense.abs().t()
    out = torch.full((M, N), math.nan, device="cuda")
    ops.linear_float8(pair.cuda(), w8, out, gated=True)
    err = (out.cpu().double() - want).abs()
    assert (err <= 2.0 ** -22 * want.abs() + 2.0 ** -13 * mag + flips + 1e-30).all()
    summed = torch.ones(M, N, device="cuda")
    ops.linear_float8(pair.cuda(), w8, summed, accumulate=True, gated=True)
    assert (summed.cpu().double() - 1 - want).abs().le(2.0 ** -22 * (1 + want.abs()) + 2.0 ** -13 * mag + flips).all()
    from garuda_b200.kernels.ops import KernelError
    for bad in (pair[:, :K], pair[:, 1:]):
        with pytest.raises(KernelError):
            ops.linear_float8(bad.cuda(), w8, out, gated=True)


def test_products_refuse(ops):
    from garuda_b200.kernels.ops import KernelError
    a, w = operands(4, 256, 256, torch.bfloat16)
    a, w8, out = a.cuda(), ops.float8_weight(w.cuda()), torch.empty(4, 256, dtype=torch.bfloat16, device="cuda")
    ops.linear_float8(a[:0], w8, out[:0])                     # no tokens: nothing
    bad = [lambda: ops.linear_float8(a[:, :128], w8, out), lambda: ops.linear_float8(a.half(), w8, out),
           lambda: ops.linear_float8(a, (w8.values, w8.scales[:1]), out), lambda: ops.linear_float8(a, (w8.values.float(), w8.scales), out),
           lambda: ops.linear_float8(a, w8, out, accumulate=True), lambda: ops.linear_float8(a, w8, out, alpha=2.0),
           lambda: ops.linear_float8(a, w8, out[:, :128]), lambda: ops.linear_float8(a.t(), w8, out),
           lambda: ops.linear_float8(a, (w8.values[:, 3:131], w8.scales[:, :1]), out),
           lambda: ops.linear_float8(a.cpu(), w8, out), lambda: ops.float8_weight(w.cuda().half()), lambda: ops.float8_weight(w.cuda().t())]
    for call in bad:
        with pytest.raises(KernelError):
            call()


# ------------------------------------------------------------------ the cache

def pools_of(pages, kv_heads, page, hd, seed, stale=True):
    """Random pages (codes as they may be, scales powers of two); ``stale``: with codes that are no numbers strewn in."""
    g = gen(seed)
    out = []
    for i in range(2):
        x = torch.randn(pages, kv_heads, page, hd, generator=g) * 100
        x = x.clamp(-448, 448).to(E4M3)
        s = torch.pow(2.0, torch.randint(-9, -4, (pages, kv_heads), generator=g).float())
        out.append((x, s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def batch(lens, page, seed=0, spare=3):
    """(cu_q, kv_lens, table, pages) of requests ``[(new tokens, positions)]`` with pages drawn at random."""
    counts = [max(1, -(-n // page)) for _, n in lens]
    width, total = max(counts) + 1, sum(counts) + spare
    order = torch.randperm(total, generator=gen(seed)).to(torch.int32)
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for r, (q, n) in enumerate(lens):
        c = -(-n // page)
        table[r, :c] = order[at:at + c]
        at += c
    cu = torch.tensor([0] + torch.tensor([q for q, _ in lens]).cumsum(0).tolist(), dtype=torch.int32)
    return cu, torch.tensor([n for _, n in lens], dtype=torch.int32), table, total


def cuda(*ts):
    return [t.cuda() for t in ts]


APPENDS = [
    # heads, kv heads, head size, page, requests
    (4, 2, 64, 32, [(1, 1)]), (4, 2, 64, 32, [(1, 40), (1, 33), (1, 32), (1, 64)]), (8, 2, 128, 32, [(70, 70), (1, 5), (33, 100), (31, 32)]),
    (4, 4, 128, 16, [(17, 20), (50, 77)]), (6, 2, 64, 64, [(3, 200), (130, 140)]), (3, 1, 48, 8, [(9, 20), (1, 9)]),
    (2, 2, 16, 5, [(11, 23)]), (4, 1, 256, 32, [(40, 50)]), (4, 2, 128, 128, [(200, 300), (1, 129)]), (2, 1, 64, 32, [(0, 7), (5, 12), (0, 3)]),
]


@pytest.mark.parametrize("heads,kv_heads,hd,page,lens", APPENDS)
@pytest.mark.parametrize("mode", ["half", "interleaved", "none"])
@pytest.mark.parametrize("dtype,q_dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
def test_append(ops, heads, kv_heads, hd, page, lens, mode, dtype, q_dtype):
    cu, kv, table, pages = batch(lens, page, seed=hd + page)
    T = int(cu[-1])
    g = gen(T + hd)
    qkv = (torch.randn(T, (heads + 2 * kv_heads) * hd, generator=g) * torch.exp(torch.randn(T, 1, generator=g))).to(dtype)
    cs = None
    if mode != "none":
        angle = torch.rand(T, hd // 2, generator=g) * 1000
        cs = torch.stack([angle.cos(), angle.sin()], -1).contiguous()
    k8, v8, ks, vs = pools_of(pages, kv_heads, page, hd, 1)
    dev = cuda(k8, v8, ks, vs)
    q_out = torch.empty(T, heads, hd, dtype=q_dtype, device="cuda")
    args = (*cuda(cu, kv, table), heads, kv_heads, hd, None if cs is None else cs.cuda(), mode == "interleaved", page)
    ops.kv_append_float8(qkv.cuda(), q_out, *dev, *args)
    q, pools, scales = plain.append(qkv, (k8, v8), (ks, vs), cu, kv, table, heads, kv_heads, hd, cs, mode == "interleaved", page)
    assert torch.equal(q_out.cpu(), q.to(q_dtype))
    for got, want in ((dev[0], pools[0]), (dev[1], pools[1]), (dev[2], scales[0]), (dev[3], scales[1])):
        assert torch.equal(got.cpu().double(), want)           # every row, the untouched ones among them
    ops.kv_append_float8(qkv.cuda(), q_out, *dev, *args)       # the same positions again: nothing changes
    for got, want in ((dev[0], pools[0]), (dev[1], pools[1]), (dev[2], scales[0]), (dev[3], scales[1])):
        assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 128, 32), (12, 3, 64, 16), (40, 8, 64, 32), (2, 1, 256, 32), (3, 3, 16, 5), (4, 1, 128, 128)])
@pytest.mark.parametrize("lens", [[(1, 1 + 13 * i) for i in range(33)], [(40, 100)] + [(0, 5)] * 60 + [(1, 33), (0, 0), (3, 65)],
                                  [(0, 9)] * 70 + [(66, 70)]])
def test_append_of_fewer_tokens_than_requests(ops, heads, kv_heads, hd, page, lens):
    test_append(ops, heads, kv_heads, hd, page, lens, "half", torch.float32, torch.bfloat16)
    test_append(ops, heads, kv_heads, hd, page, lens, "interleaved", torch.bfloat16, torch.bfloat16)


def test_append_token_by_token_is_append_at_once_but_for_the_smallest(ops):
    """A page filled token by token has the scale that it gets when filled at once; its codes differ by the second rounding of
    subnormals at most (half a step of 2^-9 of the scale more)."""
    heads, kv_heads, hd, page, n = 2, 1, 64, 32, 64
    cu, kv, table, pages = batch([(n, n)], page, seed=3)
    g = gen(8)
    qkv = torch.randn(n, 4 * hd, generator=g) * torch.exp(2 * torch.randn(n, 1, generator=g))
    q_out = torch.empty(n, heads, hd, device="cuda")

    def pools():
        return cuda(*pools_of(pages, kv_heads, page, hd, 1))

    once, steps = pools(), pools()
    ops.kv_append_float8(qkv.cuda(), q_out, *once, *cuda(cu, kv, table), heads, kv_heads, hd, None, False, page)
    for i in range(n):
        ops.kv_append_float8(qkv[i:i + 1].cuda(), q_out[:1], *steps, torch.tensor([0, 1], dtype=torch.int32).cuda(),
                             torch.tensor([i + 1], dtype=torch.int32).cuda(), table.cuda(), heads, kv_heads, hd, None, False, page)
    used = table[0, :2].long()
    for pool, scale in ((0, 2), (1, 3)):
        assert torch.equal(once[scale][used], steps[scale][used])
        d = (once[pool][used].cpu().double() - steps[pool][used].cpu().double()).abs()
        assert d.max() <= 2.0 ** -9


def test_append_of_infinities_and_nan(ops):
    """An infinity becomes the largest code of the largest scale, a NaN stays one and counts for no scale."""
    heads, kv_heads, hd, page = 1, 1, 16, 32
    cu, kv, table, pages = batch([(3, 3), (3, 3)], page)
    qkv = torch.randn(6, 3 * hd, generator=gen(9))
    qkv[1, hd + 4] = math.inf
    qkv[4, hd + 5] = math.nan
    k8, v8, ks, vs = pools_of(pages, kv_heads, page, hd, 2)
    dev = cuda(k8, v8, ks, vs)
    q_out = torch.empty(6, heads, hd, device="cuda")
    ops.kv_append_float8(qkv.cuda(), q_out, *dev, *cuda(cu, kv, table), heads, kv_heads, hd, None, False, page)
    _, pools, scales = plain.append(qkv, (k8, v8), (ks, vs), cu, kv, table, heads, kv_heads, hd, None, False, page)
    got, want = dev[0].cpu().double(), pools[0]
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert torch.equal(dev[2].cpu().double(), scales[0])
    assert dev[2][table[0, 0].item(), 0] == 2.0 ** 120


def check_attention(ops, heads, kv_heads, hd, page, lens, window=0, dtype=torch.bfloat16, seed=0, table_edit=None, q_edit=None):
    cu, kv, table, pages = batch(lens, page, seed=seed)
    T = int(cu[-1])
    g = gen(seed + T)
    q = torch.randn(T, heads, hd, generator=g)
    k8, v8, ks, vs = pools_of(pages, kv_heads, page, hd, seed + 1)
    # what no query may read is not a number: rows behind a request's end, and pages that are nobody's
    mine = torch.zeros(pages, page, dtype=torch.bool)
    for r, (_, n) in enumerate(lens):
        for j in range(-(-n // page)):
            mine[table[r, j], :min(page, n - j * page)] = True
    bad = ~mine[:, None, :, None]
    for pool in (k8, v8):
        pool.view(torch.uint8).masked_fill_(bad, 0x7F)
    for s in (ks, vs):
        s[~mine.any(1)] = math.nan
    if table_edit is not None:
        table_edit(table)
    if q_edit is not None:
        q = q_edit(q)
    q = q.to(dtype)
    scale = 1.0 / math.sqrt(hd) / 2
    out = torch.full((T, heads * hd), math.nan, dtype=dtype, device="cuda")
    dev = cuda(q, k8, v8, ks, vs, table, cu, kv)
    meta = (scale, window, page, len(lens), max(q for q, _ in lens), max(n for _, n in lens))
    ops.paged_attention_float8(*dev, out, *meta, min_q_len=min(q for q, _ in lens))
    want, mag = plain.attention(q, k8, v8, ks, vs, table, cu, kv, scale, window, page)
    # bfloat16: the result is rounded (2^-9 of it) and so may the weights be, each (2^-9 of the magnitudes' sum), and the queries
    # and weights are split into two codes that leave 2^-9 of the magnitudes' sum at most; 32 bits: sums of rounded numbers
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -17
    err, bound = (out.cpu().double() - want).abs(), unit * (want.abs() + 1.5 * mag) + 1e-30
    assert torch.isfinite(out).all(), "a result is not a number"
    assert (err <= bound).all(), f"worst {(err / bound).max().item():.2f} of the bound"
    again = torch.full_like(out, math.nan)
    ops.paged_attention_float8(*dev, again, *meta, min_q_len=min(q for q, _ in lens))
    assert torch.equal(out, again)
    ops.check_float8_errors()


SHAPES = [(4, 1, 64, 32), (8, 8, 64, 32), (32, 8, 128, 32), (4, 4, 128, 16), (8, 1, 128, 64), (16, 2, 64, 128), (14, 2, 64, 32),
          (6, 1, 128, 32), (16, 1, 128, 32), (3, 1, 48, 8), (2, 2, 256, 32), (4, 2, 80, 5), (40, 2, 64, 32)]
SINGLES = [[(1, 1)], [(1, 2), (1, 1), (1, 31), (1, 32), (1, 33)], [(1, 700), (1, 64), (1, 1), (1, 129)], [(1, 2500)], [(1, 5 + 37 * i) for i in range(40)]]


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("case", range(len(SINGLES)))
def test_attention_of_single_tokens(ops, heads, kv_heads, hd, page, case):
    check_attention(ops, heads, kv_heads, hd, page, SINGLES[case], seed=case)


@pytest.mark.parametrize("requests", [1, 2, 3, 4, 5, 9, 10, 18, 19])       # 8 heads each: on either side of every number of CTAs that share a head
@pytest.mark.parametrize("heads,hd,page", [(32, 128, 32), (8, 64, 16), (128, 64, 32)])
def test_attention_of_single_tokens_of_few_and_many_heads(ops, requests, heads, hd, page):
    lens = [(1, max(1, 1100 - 61 * i * i % 1093)) for i in range(requests)]
    check_attention(ops, heads, 8, hd, page, lens, seed=requests)
    check_attention(ops, heads, 8, hd, page, lens[:-1] + [(0, 40)] if requests > 1 else [(1, 40)], window=300, seed=requests)


@pytest.mark.parametrize("length", [8191, 8193, 16384, 16385, 20000])         # on either side of the longest that a cluster takes
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 1, 128), (16, 8, 64)])
def test_attention_of_a_long_context(ops, length, heads, kv_heads, hd):
    check_attention(ops, heads, kv_heads, hd, 32, [(1, length)], seed=length)


@pytest.mark.parametrize("window", [1, 20, 33, 100])
@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES[:6])
def test_attention_of_single_tokens_in_a_window(ops, heads, kv_heads, hd, page, window):
    check_attention(ops, heads, kv_heads, hd, page, [(1, 300), (1, 1), (1, 101), (1, 32)], window=window)


PROMPTS = [[(2, 2)], [(3, 70), (1, 40)], [(130, 130)], [(129, 400), (1, 300), (17, 17), (40, 200)], [(300, 301)], [(5, 640), (64, 64)]]


@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
@pytest.mark.parametrize("case", range(len(PROMPTS)))
@pytest.mark.parametrize("window", [0, 50])
def test_attention_of_portions(ops, heads, kv_heads, hd, page, case, window):
    check_attention(ops, heads, kv_heads, hd, page, PROMPTS[case], window=window, seed=case)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(32, 32, 64, 32), (40, 40, 128, 16), (96, 32, 64, 128), (64, 32, 128, 64)])
@pytest.mark.parametrize("window", [0, 200])
def test_attention_of_more_portions_than_multiprocessors(ops, heads, kv_heads, hd, page, window):
    """Several pieces of 256 rows to a CTA, some of them with rows in their first half only, long and short in turn."""
    check_attention(ops, heads, kv_heads, hd, page, [(300, 520), (1, 77), (129, 129), (0, 3), (200, 200), (128, 640)], window=window)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(4, 2, 64, 32), (8, 2, 128, 32), (3, 1, 48, 8)])
def test_attention_in_32_bits(ops, heads, kv_heads, hd, page):
    check_attention(ops, heads, kv_heads, hd, page, [(1, 90), (40, 75), (1, 1)], dtype=torch.float32)
    check_attention(ops, heads, kv_heads, hd, page, [(1, 90), (40, 75), (1, 1)], window=30, dtype=torch.float32)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(4, 1, 64, 32), (8, 2, 128, 32), (4, 2, 80, 5)])
def test_attention_without_tokens_or_pages(ops, heads, kv_heads, hd, page):
    """Requests without tokens; requests whose pages are all given back (zeros); pages given back in front of a window."""
    check_attention(ops, heads, kv_heads, hd, page, [(0, 7), (1, 90), (0, 0), (1, 33)])
    check_attention(ops, heads, kv_heads, hd, page, [(0, 7), (20, 90), (0, 0), (1, 33)])

    def all_of_one(table):
        table[1] = -1
    check_attention(ops, heads, kv_heads, hd, page, [(1, 50), (1, 90), (1, 33)], table_edit=all_of_one)
    check_attention(ops, heads, kv_heads, hd, page, [(40, 50), (60, 90), (1, 33)], table_edit=all_of_one)

    def front(table):
        table[0, :200 // page] = -1
    check_attention(ops, heads, kv_heads, hd, page, [(1, 300), (1, 20)], window=60, table_edit=front)
    check_attention(ops, heads, kv_heads, hd, page, [(30, 300), (50, 60)], window=60, table_edit=front)


@pytest.mark.parametrize("factor", [1e-30, 1e-3, 40.0, 1e4])
@pytest.mark.parametrize("lens", [[(1, 400), (1, 65)], [(70, 200)]])
def test_attention_with_scores_small_and_large(ops, factor, lens):
    """Queries of any size (scores from nothing to thousands: a softmax that is flat, or one key's alone) and rows of zeros."""
    def edit(q):
        q = q * factor
        q[0, 0] = 0.0
        return q
    check_attention(ops, 8, 2, 128, 32, lens, q_edit=edit)
    check_attention(ops, 8, 2, 64, 32, lens, q_edit=edit)


def test_attention_of_a_sink_over_a_long_context(ops):
    """One key takes half of the weight and thousands share the other half: weights of 2^-13 of the largest have to count."""
    hd, page, n = 64, 32, 8000
    cu, kv, table, pages = batch([(1, n)], page, seed=5)
    k = torch.zeros(pages, 1, page, hd)
    k[table[0, 0].item(), 0, 0, 0] = 1.0
    v = torch.randn(pages, 1, page, hd, generator=gen(1)).abs()
    q = torch.zeros(1, 4, hd)
    q[:, :, 0] = math.log(n)                   # the sink's weight is n times another's
    k8, v8 = (k * 256).to(E4M3), (v * 64).to(E4M3)
    ks, vs = torch.full((pages, 1), 2.0 ** -8), torch.full((pages, 1), 2.0 ** -6)
    out = torch.empty(1, 4 * hd, dtype=torch.bfloat16, device="cuda")
    qb = q.to(torch.bfloat16)
    ops.paged_attention_float8(*cuda(qb, k8, v8, ks, vs, table, cu, kv), out, 1.0, 0, page, 1, 1, n)
    want, mag = plain.attention(qb, k8, v8, ks, vs, table, cu, kv, 1.0, 0, page)
    err = (out.cpu().double() - want).abs()
    assert (err <= 2.0 ** -8 * (want.abs() + mag)).all()


def test_append_then_attention_on_streams_of_their_own(ops):
    """The two operators behind one another, on two streams at once: what one writes the other reads, and scratch is a stream's own."""
    heads, kv_heads, hd, page, n = 8, 2, 128, 32, 150
    made = []
    for i in range(2):
        g = gen(20 + i)
        cu, kv, table, pages = batch([(n, n)], page, seed=i)
        one, qkv = torch.tensor([0, 1], dtype=torch.int32), torch.randn(n, 12 * hd, generator=g)
        made.append((qkv, cu, kv, table, one, pools_of(pages, kv_heads, page, hd, i)))
    streams = [torch.cuda.Stream() for _ in made]
    results = []
    inputs = [[t.cuda() for t in m[:5]] + [cuda(*m[5])] for m in made]
    torch.cuda.synchronize()
    for rep in range(3):
        results = []
        for st, (qkv, cu, kv, table, one, pools) in zip(streams, inputs):
            with torch.cuda.stream(st):
                q = torch.empty(n, heads, hd, dtype=torch.bfloat16, device="cuda")
                ops.kv_append_float8(qkv, q, *pools, cu, kv, table, heads, kv_heads, hd, None, False, page)
                last = torch.empty(1, heads * hd, dtype=torch.bfloat16, device="cuda")
                ops.paged_attention_float8(q[-1:].contiguous(), *pools, table, one, kv, last, 0.05, 0, page, 1, 1, n)
                full = torch.empty(n, heads * hd, dtype=torch.bfloat16, device="cuda")
                ops.paged_attention_float8(q, *pools, table, cu, kv, full, 0.05, 0, page, 1, n, n, min_q_len=n)
                results.append((q, pools, last, full))
        torch.cuda.synchronize()
    for (qkv, cu, kv, table, one, _), (q, pools, last, full) in zip(made, results):
        want, mag = plain.attention(q.cpu(), *[t.cpu() for t in pools], table, cu, kv, 0.05, 0, page)
        for got, w, m in ((full, want, mag), (last, want[-1:], mag[-1:])):
            assert ((got.cpu().double() - w).abs() <= 2.0 ** -8 * (w.abs() + 1.5 * m)).all()


def test_cache_refusals(ops):
    from garuda_b200.kernels.ops import KernelError
    heads, kv_heads, hd, page = 4, 2, 64, 32
    cu, kv, table, pages = cuda(*batch([(5, 40)], page)[:3]) + [5]
    k8, v8, ks, vs = cuda(*pools_of(5, kv_heads, page, hd, 1))
    qkv, q = torch.randn(5, 8 * hd, device="cuda"), torch.empty(5, heads, hd, dtype=torch.bfloat16, device="cuda")

    def append(qkv=qkv, q=q, k8=k8, v8=v8, ks=ks, vs=vs, cu=cu, kv=kv, table=table, hd=hd, cs=None, page=page):
        ops.kv_append_float8(qkv, q, k8, v8, ks, vs, cu, kv, table, heads, kv_heads, hd, cs, False, page)

    out = torch.empty(5, heads * hd, dtype=torch.bfloat16, device="cuda")

    def attend(q=q, k8=k8, v8=v8, ks=ks, vs=vs, cu=cu, kv=kv, table=table, out=out, scale=0.1, page=page):
        ops.paged_attention_float8(q, k8, v8, ks, vs, table, cu, kv, out, scale, 0, page, 1, 5, 40)

    append(), attend()
    bad = [lambda: append(qkv=qkv[:, 1:]), lambda: append(q=q[:4]), lambda: append(k8=k8.float()), lambda: append(ks=ks[:, :1]),
           lambda: append(cu=cu.long()), lambda: append(page=16), lambda: append(cs=torch.zeros(5, hd // 2, 2, dtype=torch.float64, device="cuda")),
           lambda: append(qkv=qkv.half()), lambda: append(table=table.long()), lambda: append(v8=v8[:3]), lambda: append(kv=kv.cpu()),
           lambda: attend(q=q.float()), lambda: attend(out=out[:4]), lambda: attend(v8=v8.view(torch.uint8)), lambda: attend(vs=vs.double()),
           lambda: attend(page=64), lambda: attend(scale=0.0), lambda: attend(table=table[:, :1].contiguous()), lambda: attend(cu=cu[:1]), lambda: attend(q=q.half(), out=out.half())]
    for call in bad:
        with pytest.raises(KernelError):
            call()
