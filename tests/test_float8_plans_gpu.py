"""Products in 8 bits in every way that they are cut: single CTAs and pairs, one or two blocks to a stage, rounds of whole tiles, what is left as whole
tiles or in parts, against 64 bits on the device; two streams at once; infinite tokens."""
import math

import pytest
import torch

from tests.test_float8_gpu import E4M3, gen, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu

BLOCK = 128


def blocks_of(a):
    """``a [M, K]`` in 64 bits, padded to whole blocks, and the scales of these, spread over them."""
    M, K = a.shape
    padded = torch.nn.functional.pad(a, (0, -K % BLOCK)).view(M, -1, BLOCK)
    m, e = torch.frexp(padded.abs().amax(-1, keepdim=True))
    e = torch.where(m > 0, e - 9 + (m > 0.875).int(), -100).clamp(-100, 120)         # 448 = 0.875 * 2^9
    return padded, torch.ldexp(torch.ones_like(m), e).expand_as(padded)


def rounded(a):
    """The numbers that the codes of ``a``'s rows stand for (an infinity is 448 of the largest scale), 64-bit."""
    infinite = torch.isinf(a)
    x, s = blocks_of(torch.where(infinite, torch.sign(a) * 448 * 2.0 ** 120, a))
    return ((x / s).clamp(-448, 448).to(E4M3).double() * s).view(a.shape[0], -1)[:, :a.shape[1]]


def dense(w8):
    N, K = w8.values.shape
    return w8.values.double() * w8.scales.double().repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]


def bound(want, mag, K, bfloat16, extra=0.0):
    """32-bit sums: the tensor cores add 32 products to the sum so far and may cut off a last place of it each time, and of the products as much (2^-22 of
    the magnitudes' sum together); parts are added up in 32 bits, at most 16 of them. The result is rounded to nearest."""
    return (2.0 ** -8 if bfloat16 else 2.0 ** -22) * want.abs() + (K / 32 + 8) * 2.0 ** -22 * mag + extra + 1e-30


def kind(ops, M, N, K):  # noqa: F811
    p = ops.linear_float8_plan(M, N, K)
    rest = p["tiles"] - p["rounds"] * p["workers"]
    left = "none" if rest == 0 else "whole" if p["share"] == rest else "even" if p["share"] % rest == 0 else "uneven"
    return p["ctas"], p["blocks"], min(p["rounds"], 2), left, "wide" if p["tokens"] > 128 else "narrow"


# Shapes whose plan is of each kind that the cost model chooses on 148 multiprocessors: CTAs that work together, blocks to a stage, rounds (2: or more),
# what is left behind them (whole tiles; parts, as many for every tile; stretches of all of them), tiles of more than 128 tokens
KINDS = {
    (1, 1, 0, "whole", "wide"): (2048, 130, 130), (1, 1, 1, "none", "wide"): (2048, 130, 128), (1, 1, 1, "whole", "wide"): (1200, 6400, 400),
    (1, 1, 2, "none", "wide"): (480, 18944, 128), (1, 1, 2, "whole", "wide"): (512, 14336, 128),
    (1, 2, 0, "even", "narrow"): (1, 130, 8192), (1, 2, 0, "whole", "narrow"): (64, 3001, 1000), (1, 2, 0, "whole", "wide"): (900, 130, 130),
    (1, 2, 1, "even", "narrow"): (7, 20000, 8192), (1, 2, 1, "none", "narrow"): (1, 130, 128), (1, 2, 1, "none", "wide"): (900, 130, 128),
    (1, 2, 1, "whole", "narrow"): (8, 28672, 4096), (1, 2, 1, "whole", "wide"): (150, 20000, 128), (1, 2, 2, "even", "narrow"): (1, 38000, 8192),
    (1, 2, 2, "none", "narrow"): (241, 18944, 128), (1, 2, 2, "none", "wide"): (300, 18944, 128), (1, 2, 2, "whole", "narrow"): (1, 38000, 128),
    (1, 2, 2, "whole", "wide"): (300, 20000, 128),
    (2, 2, 0, "even", "narrow"): (480, 130, 11008), (2, 2, 0, "even", "wide"): (900, 130, 8192), (2, 2, 0, "whole", "narrow"): (301, 4096, 11008),
    (2, 2, 0, "whole", "wide"): (512, 4096, 4096), (2, 2, 0, "uneven", "wide"): (272, 4753, 28740), (2, 2, 1, "even", "narrow"): (512, 6400, 11008),
    (2, 2, 1, "even", "wide"): (3000, 1500, 11008), (2, 2, 1, "none", "narrow"): (100, 18944, 5632), (2, 2, 1, "none", "wide"): (150, 18944, 2056),
    (2, 2, 1, "whole", "narrow"): (512, 6400, 1376), (2, 2, 1, "whole", "wide"): (1500, 3000, 1000), (2, 2, 1, "uneven", "narrow"): (250, 14234, 31537),
    (2, 2, 2, "even", "narrow"): (241, 20000, 8192), (2, 2, 2, "none", "narrow"): (241, 18944, 1000), (2, 2, 2, "none", "wide"): (480, 18944, 400),
    (2, 2, 2, "whole", "narrow"): (241, 28672, 400), (2, 2, 2, "whole", "wide"): (2048, 6144, 4096),
}


@pytest.mark.parametrize("expected", KINDS, ids=lambda k: "-".join(map(str, k)))
def test_products_cut_in_every_way(ops, expected):  # noqa: F811
    M, N, K = KINDS[expected]
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert kind(ops, M, N, K) == expected, "the cost model chooses otherwise: give this kind another shape"
    g = torch.Generator(device="cuda").manual_seed(M + N + K)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    a = (normal(M, K) * torch.exp(normal(K))).to(torch.bfloat16)
    w8 = ops.float8_weight((normal(N, K) * 0.05).to(torch.bfloat16))
    w = dense(w8)
    x = rounded(a.double())
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    for dtype in (torch.bfloat16, torch.float32):
        out, again = (torch.full((M, N), math.nan, dtype=dtype, device="cuda") for _ in range(2))
        ops.linear_float8(a, w8, out)
        ops.linear_float8(a, w8, again)
        assert ((out.double() - want).abs() <= bound(want, mag, K, dtype == torch.bfloat16)).all()
        assert torch.equal(out, again)
    before = normal(M, N)
    sums = [before.clone() for _ in range(2)]
    for s in sums:
        ops.linear_float8(a, w8, s, accumulate=True, alpha=-0.37)
    total = before.double() - 0.37 * want
    assert ((sums[0].double() - total).abs() <= bound(total, mag, K, False)).all()
    assert torch.equal(*sums)
    del out, again, sums, total, before
    # silu(gate) * up is 32-bit, off by 2^-20 of itself at most: where it lies nearer than 2^-19 to the middle of two codes, the code may be the
    # other one, a step of 2^-3 of the value (2^-9 of the scale below the normal numbers)
    pair = (normal(M, 2 * K) * 2).to(torch.bfloat16)
    gate, up = pair.double().split(K, 1)
    act = gate / (1 + torch.exp(-gate)) * up
    x = rounded(act)
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    part, scale = blocks_of(act)
    flip = (part * (1 - 2.0 ** -19) / scale).clamp(-448, 448).to(E4M3).double() != (part * (1 + 2.0 ** -19) / scale).clamp(-448, 448).to(E4M3).double()
    off = torch.where(flip, part.abs() * 2.0 ** -3 + scale * 2.0 ** -9, 0.0).view(M, -1)[:, :K] @ w.abs().t()
    out = torch.ones(M, N, device="cuda")
    ops.linear_float8(pair, w8, out, accumulate=True, gated=True)
    assert ((out.double() - 1 - want).abs() <= bound(1 + want.abs(), mag, K, False, off)).all()
    ops.check_float8_errors()


def test_products_on_streams_of_their_own(ops):  # noqa: F811
    """Two products at a time on two streams, their tiles in parts: codes, parts and counters belong to the stream."""
    shapes = [(480, 130, 11008), (1, 130, 8192), (33, 640, 5632), (900, 130, 8192)]
    g = torch.Generator(device="cuda").manual_seed(1)
    made = []
    for M, N, K in shapes:
        a = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
        w8 = ops.float8_weight(torch.randn(N, K, generator=g, device="cuda"))
        alone = torch.empty(M, N, device="cuda")
        ops.linear_float8(a, w8, alone)
        made.append((a, w8, alone, [torch.empty(M, N, device="cuda") for _ in range(8)]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(8):
        for i, (a, w8, _, outs) in enumerate(made):
            with torch.cuda.stream(streams[(i + rep) % 2]):
                ops.linear_float8(a, w8, outs[rep])
    torch.cuda.synchronize()
    for _, _, alone, outs in made:
        assert all(torch.equal(alone, out) for out in outs)
    ops.check_float8_errors()


def test_gated_pairs_of_one_channel_need_unit_stride(ops):  # noqa: F811
    """Rows of two numbers, whatever lies between them, and the same rows closed up."""
    from garuda_b200.kernels.ops import KernelError
    g = gen(4)
    apart = torch.randn(5, 2, 3, generator=g).cuda()[:, :, 0]
    w8, out = ops.float8_weight(torch.randn(7, 1, generator=g).cuda()), torch.zeros(5, 7, device="cuda")
    with pytest.raises(KernelError):
        ops.linear_float8(apart, w8, out, gated=True)
    ops.linear_float8(apart.contiguous(), w8, out, gated=True)
    gate, up = apart.double().unbind(1)
    act = gate / (1 + torch.exp(-gate)) * up
    assert torch.allclose(out.double(), act[:, None] * dense(w8)[None, :, 0], rtol=2.0 ** -4, atol=0.0)


@pytest.mark.parametrize("size", [0.05, 40.0])
@pytest.mark.parametrize("M,N,K", [(5, 200, 400), (300, 257, 1000)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_an_infinite_token_is_the_largest_number_of_the_largest_scale(ops, M, N, K, bad, size):  # noqa: F811
    """448 * 2^120, next to which the rest of its 128 channels is nothing; results beyond 32 bits are infinite. Other rows know nothing of it."""
    g = gen(M)
    a = torch.randn(M, K, generator=g).cuda()
    a[3, 130] = bad
    w8 = ops.float8_weight((torch.randn(N, K, generator=g) * size).cuda())
    out = torch.full((M, N), math.nan, device="cuda")
    ops.linear_float8(a, w8, out)
    w, x = dense(w8), rounded(a.double())
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    small = want.abs() < 2.0 ** 127
    assert ((out.double() - want).abs() <= bound(want, mag, K, False))[small].all()
    assert (out[~small].abs() > 2.0 ** 126).all() and torch.equal(out[~small] > 0, want[~small] > 0)
    assert small[torch.arange(M, device="cuda") != 3].all() and (size < 1 or not small.all())
