"""Decoding along branches on the device, against plain implementations in 64 bits at the sizes, masks and values where it can go wrong."""
import math
import random

import numpy as np
import pytest
import torch

from tests.plain import branches_plain as plain

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24        # half a step of float32
U16 = 2.0 ** -8         # of bfloat16


@pytest.fixture(scope="module")
def ops():
    from garuda_b200.kernels.ops import CudaOps
    return CudaOps()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def tree(rng, n, wide=3):
    return [-1 if i == 0 else max(-1, i - 1 - rng.randrange(min(i, wide) + 1)) for i in range(n)]


class Step:
    """Requests with contexts and drafted tokens, their pages in a random order among pages that hold NaN."""

    def __init__(self, seed, lens, heads, kv_heads, hd, page, dtype, window=0, reads=None, spare=3):
        self.rng, self.gen = random.Random(seed), torch.Generator().manual_seed(seed)
        self.q_lens, self.ctx = [q for _, q in lens], [c for c, _ in lens]
        self.heads, self.kv_heads, self.hd, self.page, self.dtype, self.window = heads, kv_heads, hd, page, dtype, window
        self.kv = [c + q for c, q in lens]
        self.cu = [0] + list(np.cumsum(self.q_lens))
        self.T, self.R, self.max_q, self.max_kv = self.cu[-1], len(lens), max(self.q_lens + [1]), max(self.kv + [1])
        need = [-(-n // page) for n in self.kv]
        pages = sum(need) + spare
        order = list(range(pages))
        self.rng.shuffle(order)
        self.table = np.full((self.R, max(max(need), 1)), -1, dtype=np.int32)
        for r, n in enumerate(need):
            self.table[r, :n] = [order.pop() for _ in range(n)]
        nan = float("nan")
        self.k, self.v = (torch.full((pages, kv_heads, page, hd), nan, dtype=dtype) for _ in range(2))
        for r, n in enumerate(self.kv):
            for i, at in enumerate(self.table[r]):
                m = min(page, n - i * page)
                if m > 0:
                    self.k[at, :, :m], self.v[at, :, :m] = (self.normal(kv_heads, m, hd) for _ in range(2))
        self.q = self.normal(self.T, heads, hd)
        self.parents = [p for n in self.q_lens for p in tree(self.rng, n)] if not reads else None
        if reads:
            # any mask: some rows empty, some full, the others at random
            self.reads = []
            for n in self.q_lens:
                for i in range(n):
                    pick = self.rng.randrange(6)
                    self.reads.append(set() if pick == 0 else set(range(n)) if pick == 1 else {j for j in range(n) if self.rng.random() < 0.4})
            self.positions = [self.ctx[r] + self.rng.randrange(n) for r, n in enumerate(self.q_lens) for _ in range(n)]
        else:
            self.positions, self.reads = plain.layout(self.parents, self.cu, self.kv, window)
        self.words = -(-self.max_q // 32) + 1
        self.scale = 1.0 / math.sqrt(hd)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen).to(self.dtype)

    def run(self, ops, ws=None, out=None):
        self.device = [x.cuda() for x in (self.q, self.k, self.v)]
        self.words_of = torch.from_numpy(plain.mask_words(self.reads, self.words)).cuda()
        out = torch.full((self.T, self.heads * self.hd), 7.0, dtype=self.dtype, device="cuda") if out is None else out
        ops.tree_attention(*self.device, torch.from_numpy(self.table).cuda(), ints(self.cu), ints(self.kv), ints(self.positions), self.words_of, out,
                           self.scale, self.window, self.page, self.max_q, self.max_kv, ws=ws)
        return out

    def check(self, out, tensor_cores):
        want, weight, size = plain.attention(self.q.double().numpy(), self.k.double().numpy(), self.v.double().numpy(), self.table, self.cu, self.kv,
                                             self.positions, self.reads, self.scale, self.window)
        got = out.double().cpu().numpy().reshape(want.shape)
        # a score is off by hd + 2 roundings of sums of |q k| (the tensor cores may cut where others round: whole steps), a weight by as much,
        # relatively, and by its exponential (2^-22), the factors that join partial sums (again 2^-22 each, at most 2 of them for each of 40 pieces) and
        # the sum of up to n terms; with the quotient that is twice it
        n = self.max_kv
        off = 2 * ((self.hd + 2) * 2 * U32 * size[:, :, None] + 2.0 ** -22 * 81 + n * U32)
        if tensor_cores:
            off = off + U16               # weights are rounded to bfloat16
        bound = off * weight + (U16 if self.dtype is torch.bfloat16 else U32) * np.abs(want) + 1e-30
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert (np.abs(got - want)[~np.isnan(want)] <= (1.01 * bound)[~np.isnan(want)]).all(), np.nanmax(np.abs(got - want) / bound)


LENS = [(0, 1), (127, 5), (1, 64), (500, 0), (128, 33), (1000, 12), (63, 100), (0, 17)]


@pytest.mark.parametrize("reads", [False, True])
@pytest.mark.parametrize("heads, kv_heads, hd, page, window", [
    (8, 8, 128, 32, 0), (8, 2, 128, 32, 0), (8, 1, 64, 16, 0), (6, 2, 64, 64, 0), (14, 2, 128, 128, 0), (4, 4, 64, 8, 40), (8, 2, 128, 32, 129)])
def test_attention_on_the_tensor_cores(ops, heads, kv_heads, hd, page, window, reads):
    step = Step(heads + hd + page, LENS, heads, kv_heads, hd, page, torch.bfloat16, window, reads)
    step.check(step.run(ops), True)
    ops.check_branch_errors()


@pytest.mark.parametrize("dtype, heads, kv_heads, hd, page, window", [
    (torch.float32, 8, 2, 64, 32, 0), (torch.float32, 8, 1, 128, 16, 70), (torch.float32, 3, 3, 16, 24, 0), (torch.float32, 4, 2, 256, 7, 0),
    (torch.float32, 2, 2, 20, 33, 9), (torch.bfloat16, 8, 2, 96, 32, 0), (torch.bfloat16, 4, 4, 128, 24, 50), (torch.bfloat16, 4, 1, 4, 32, 0)])
def test_attention_in_32_bits(ops, dtype, heads, kv_heads, hd, page, window):
    step = Step(heads + hd + page, LENS, heads, kv_heads, hd, page, dtype, window, hd % 64 == 0)
    step.check(step.run(ops), False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens, heads, kv_heads", [
    ([(9000, 3)], 4, 2), ([(20000, 1)], 2, 1), ([(7000, 40), (0, 2), (6001, 7)], 8, 1), ([(3, 1 + i % 4) for i in range(300)], 2, 2)])
def test_attention_cut_along_the_keys(ops, dtype, lens, heads, kv_heads):
    """Stretches that begin and end anywhere, joined the same way every time; and what an earlier call left in the scratch memory does not matter."""
    step = Step(len(lens), lens, heads, kv_heads, 64, 32, dtype)
    first = step.run(ops)
    step.check(first, dtype is torch.bfloat16)
    Step(5, [(3000, 60), (2000, 9)], 8, 1, 64, 16, dtype).run(ops)
    for _ in range(3):
        assert torch.equal(step.run(ops), first)


@pytest.mark.parametrize("dtype, hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
def test_what_is_masked_has_no_influence(ops, dtype, hd):
    """Infinities and NaN in keys and values of tokens that a row does not read, and of context in front of its window."""
    lens, window = [(300, 40), (0, 30), (90, 3)], 100
    clean = Step(3, lens, 4, 2, hd, 32, dtype, window)
    spoilt = Step(3, lens, 4, 2, hd, 32, dtype, window)
    outs = []
    for step, bad in ((clean, False), (spoilt, True)):
        # nobody reads tokens 5 and 7 of request 0 nor 29 of request 1, which read nothing themselves
        for r, j in ((0, 5), (0, 7), (1, 29)):
            for t in range(step.cu[r], step.cu[r + 1]):
                step.reads[t].discard(j)
            at = step.ctx[r] + j
            page = step.table[r, at // 32]
            if bad:
                step.k[page, :, at % 32], step.v[page, :, at % 32, 3] = float("nan"), float("inf") if j == 5 else float("nan")
        if bad:
            for at in range(0, 201):         # in front of every window of request 0
                page = step.table[0, at // 32]
                step.k[page, :, at % 32], step.v[page, :, at % 32] = float("-inf"), float("nan")
        outs.append(step.run(ops))
    assert torch.equal(*outs)
    clean.check(outs[0], dtype is torch.bfloat16)
    # a value of the tree that is read spoils those that read it, and nobody else
    t0, at = spoilt.cu[2], spoilt.ctx[2] + 1
    spoilt.v[spoilt.table[2, at // 32], 0, at % 32, 9] = float("nan")
    out = spoilt.run(ops).view(spoilt.T, 4, hd)
    for t in range(spoilt.T):
        readers = t >= t0 and 1 in spoilt.reads[t]
        for h in range(4):
            assert bool(out[t, h].isnan().any()) == (readers and h < 2), (t, h)


def test_a_query_that_is_no_number_gives_none(ops):
    for dtype in (torch.bfloat16, torch.float32):
        step = Step(4, [(3000, 6), (10, 3)], 4, 2, 64, 32, dtype)
        step.q[2, 1, 5] = float("nan")
        out = step.run(ops).view(step.T, 4, 64)
        assert out[2, 1].isnan().all() and int(out.isnan().sum()) == 64


def test_rows_behind_the_last_request_and_absent_pages(ops):
    for dtype, hd in ((torch.bfloat16, 128), (torch.float32, 64)):
        step = Step(6, [(200, 5), (70, 9)], 4, 2, hd, 32, dtype)
        step.table[0, 2], step.table[1, 0] = -1, 10 ** 6          # zeros, wherever they may point
        full = torch.full((step.T + 3, 4 * hd), 7.0, dtype=dtype, device="cuda")
        q = torch.cat([step.q, step.normal(3, 4, hd)])
        mask = np.concatenate([plain.mask_words(step.reads, step.words), np.ones((3, step.words), dtype=np.int32)])
        ops.tree_attention(q.cuda(), step.k.cuda(), step.v.cuda(), torch.from_numpy(step.table).cuda(), ints(step.cu), ints(step.kv),
                           ints(step.positions + [0, 0, 0]), torch.from_numpy(mask).cuda(), full, step.scale, 0, 32, step.max_q, step.max_kv)
        assert (full[step.T:] == 7.0).all()
        step.check(full[:step.T], dtype is torch.bfloat16)


# ------------------------------------------------------------------ trees
@pytest.mark.parametrize("dtype, page", [(torch.bfloat16, 32), (torch.bfloat16, 24), (torch.float32, 32)])
def test_pages_behind_two_thousand_million_numbers(ops, dtype, page):
    """The far end of a large pool: attention, moved rows and copied pages are those of a small one, bit for bit."""
    step = Step(3, [(700, 12), (90, 3)], 8, 4, 128, page, dtype)
    want, small = step.run(ops), step.k.cuda()
    pages = 2 ** 31 // (4 * page * 128) + 50
    shift = pages - small.shape[0]
    k, v = (torch.zeros(pages, 4, page, 128, dtype=dtype, device="cuda") for _ in range(2))
    k[shift:], v[shift:] = small, step.v.cuda()
    table = torch.from_numpy(np.where(step.table >= 0, step.table + shift, -1).astype(np.int32)).cuda()
    out = torch.full_like(want, 7.0)
    ops.tree_attention(step.q.cuda(), k, v, table, ints(step.cu), ints(step.kv), ints(step.positions), step.words_of, out, step.scale, 0, page, step.max_q, step.max_kv)
    assert torch.equal(out, want)
    drafted = ints([5, 6, 7, 6]), ints([7, 8, 1, 2]), ints([-1, 0, 0, 1]), ints([0, 4]), ints([10])
    for pool, last in ((k, pages - 1), (small, small.shape[0] - 1)):
        path, kept, after = ints([[9] * 4]), ints([9]), ints([9])
        ops.tree_accept(*drafted, path, kept, after, 4, [pool], ints([[last]]), page)
        assert path.tolist() == [[0, 2, -1, -1]]
    ops.copy_entries([k], ints([pages - 1, 0]), ints([pages - 2, pages - 3]))
    ops.copy_entries([small], ints([small.shape[0] - 1]), ints([small.shape[0] - 2]))
    small[-3] = 0
    assert torch.equal(k[shift:].view(torch.uint8), small.view(torch.uint8))          # (there are NaN in them)
    ops.check_branch_errors()
    del k, v
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests", [3, 90])
def test_a_length_of_zero_reads_nothing(ops, dtype, requests):
    """(Of a padded batch, say: tokens, but no key at all.) Their rows are zeros, the others' what they were."""
    step = Step(requests, [(40 + 9 * (r % 5), 1 + r % 4) for r in range(requests)], 4, 2, 64, 32, dtype, 30 * (requests > 3))
    want = step.run(ops)
    step.kv = [0 if r % 3 == 1 else n for r, n in enumerate(step.kv)]
    for r in range(1, requests, 3):
        want[step.cu[r]:step.cu[r + 1]] = 0
    assert torch.equal(step.run(ops), want)
    ops.check_branch_errors()


@pytest.mark.parametrize("window", [0, 1, 5, 40])
def test_layout(ops, window):
    rng = random.Random(window)
    parents, q_lens = [], [1, 0, 64, 33, 200, 7, 1000]
    for n in q_lens:
        parents += tree(rng, n) if n != 200 else list(range(-1, 199))       # one of them a chain
    parents[len(parents) - 1000 + 50], parents[10] = 60, -7                  # a parent behind its child, and one that is none
    cu = [0] + list(np.cumsum(q_lens))
    kv = [n + 10 * i for i, n in enumerate(q_lens)]
    words = 33
    positions, mask = ints([9] * cu[-1]), ints([[9] * words] * cu[-1])
    ops.tree_layout(ints(parents), ints(cu), ints(kv), positions, mask, 1000, window)
    want, reads = plain.layout(parents, cu, kv, window)
    assert positions.tolist() == want
    assert np.array_equal(mask.cpu().numpy(), plain.mask_words(reads, words))


@pytest.mark.parametrize("dtype, heads, width, page", [(torch.bfloat16, 2, 64, 32), (torch.float32, 1, 6, 16), (torch.bfloat16, 3, 5, 7), (torch.bfloat16, 8, 128, 64)])
def test_accept(ops, dtype, heads, width, page):
    rng = random.Random(page)
    q_lens, ctx = [1, 0, 64, 33, 8, 40, 300], [0, 5, 31, 7, 100, 1, 2]
    cu, kv = [0] + list(np.cumsum(q_lens)), [a + b for a, b in zip(q_lens, ctx)]
    T, R = cu[-1], len(kv)
    parents, tokens, targets = [], [], []
    for n in q_lens:
        # a path through about half of the tokens, the others anywhere; a token that continues the path comes a second time, further behind
        path = [i for i in range(n) if i == 0 or rng.random() < 0.5]
        up, word, model = [-1 if i == 0 else rng.randrange(i) for i in range(n)], [rng.randrange(3) for _ in range(n)], [rng.randrange(3, 5) for _ in range(n)]
        for a, b in zip(path, path[1:]):
            up[b], word[b], model[a] = a, 10 + b, 10 + b
            if b + 1 < n and b + 1 not in path:
                up[b + 1], word[b + 1] = a, 10 + b
        parents, tokens, targets = parents + up, tokens + word, targets + model
    need = [-(-n // page) for n in kv]
    pages = sum(need) + 2
    order = list(range(pages))
    rng.shuffle(order)
    table = np.full((R, max(need) + 1), -1, dtype=np.int32)
    for r, n in enumerate(need):
        table[r, :n] = [order.pop() for _ in range(n)]
    table[5, 1] = -1                                              # a page that was given back
    shapes = [(3, pages, heads, page, width), (3, pages, heads, page, width), (pages, 1, page, 2 * width)]
    pools = [torch.randn(s, generator=torch.Generator().manual_seed(1)).to(dtype) for s in shapes]
    want = [p.float().numpy().reshape((-1,) + tuple(p.shape[-4:])).copy() for p in pools]
    device = [p.cuda() for p in pools]
    path, kept, after = ints([[9] * 300] * R), ints([9] * R), ints([9] * R)
    ops.tree_accept(ints(tokens), ints(targets), ints(parents), ints(cu), ints(kv), path, kept, after, 300, device, torch.from_numpy(table).cuda(), page)
    paths, nexts = plain.accept(tokens, targets, parents, cu)
    assert max(map(len, paths)) > 99
    assert kept.tolist() == [len(p) for p in paths] and after.tolist() == nexts
    assert path.tolist() == [p + [-1] * (300 - len(p)) for p in paths]
    for r in range(R):
        for pool in want:
            plain.move_rows(pool, table[r], page, ctx[r], paths[r])
    for got, pool in zip(device, want):
        assert np.array_equal(got.float().cpu().numpy().reshape(pool.shape), pool)


def test_accept_without_pools(ops):
    path, kept, after = ints([[9] * 4] * 2), ints([9, 9]), ints([9, 9])
    ops.tree_accept(ints([5, 6, 7, 6]), ints([6, 8, 1, 2]), ints([-1, 0, 0, -1]), ints([0, 3, 4]), ints([3, 1]), path, kept, after, 4)
    assert path.tolist() == [[0, 1, -1, -1], [0, -1, -1, -1]] and kept.tolist() == [2, 1] and after.tolist() == [8, 2]


# ------------------------------------------------------------------ beams
def check_beam(ops, logits, scores, n, device=None):
    items, beams = scores.shape
    device = logits.reshape(items * beams, -1).cuda() if device is None else device
    best, parents, tokens = torch.full((items, n), 9.0, device="cuda"), ints([[9] * n] * items), ints([[9] * n] * items)
    ops.beam_select(device, scores.cuda(), best, parents, tokens)
    want = plain.beam(logits.numpy().reshape(items, beams, -1), scores.numpy(), n)
    got = best.cpu().numpy().astype(np.float64)
    dead = np.isinf(want[0])
    assert np.array_equal(np.isinf(got), dead)
    got, exact = got[~dead], want[0][~dead]
    assert (np.abs(got - exact) <= 1.01 * U32 * np.abs(exact) + 1e-7).all()      # (rounded once; the sums are good for 1e-7)
    assert np.array_equal(parents.cpu().numpy(), want[1]) and np.array_equal(tokens.cpu().numpy(), want[2])


@pytest.mark.parametrize("items, beams, n, V", [(1, 1, 1, 1), (1, 4, 8, 32000), (3, 5, 10, 1237), (2, 8, 16, 128256), (40, 3, 6, 5001), (1, 64, 64, 2050), (2, 2, 3, 2),
                                                (7, 1, 17, 20), (5, 16, 33, 16387)])
def test_beam(ops, items, beams, n, V):
    g = torch.Generator().manual_seed(V)
    logits, scores = 3 * torch.randn(items * beams, V, generator=g), -5 * torch.rand(items, beams, generator=g)
    check_beam(ops, logits, scores, n)


def test_beam_with_equal_scores(ops):
    """Alike logits, alike beams, and all that there is alike: the lowest number first."""
    g = torch.Generator().manual_seed(1)
    rough = torch.randint(-3, 3, (6, 3, 9000), generator=g).float()
    check_beam(ops, rough, torch.zeros(6, 3), 64)
    rough[:, 1] = rough[:, 0]
    rough[:, 2] = rough[:, 0]
    check_beam(ops, rough, torch.full((6, 3), -1.5), 48)
    check_beam(ops, torch.zeros(2, 64, 700), torch.zeros(2, 64), 64)
    check_beam(ops, torch.zeros(1, 2, 40000), torch.zeros(1, 2), 7)
    # and zeros of both signs are alike
    signs = torch.where(torch.rand(2, 2, 600, generator=g) < 0.5, 0.0, -0.0)
    check_beam(ops, signs, torch.zeros(2, 2), 9)


def test_beam_without_a_distribution(ops):
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(2)
    logits, scores = torch.randn(8, 4, 5000, generator=g), -torch.rand(8, 4, generator=g)
    scores[0, 1:], scores[1], scores[2, 0], scores[3, 2] = -inf, -inf, nan, inf         # a first step, an item that is over, beams that are
    logits[3, 0, 77], logits[4, 1, 4999], logits[5, 2] = nan, inf, -inf
    logits[1, 0, 0] = nan                                     # (nobody looks at it)
    logits[6, :, 3:], logits[7, :, 20:] = -inf, -inf             # fewer candidates than are asked for
    check_beam(ops, logits, scores, 16)
    check_beam(ops, logits, scores, 64)


def test_beam_of_rows_that_lie_apart(ops):
    """Rows of a wider matrix, which start on any four bytes."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(8, 6007, generator=g)
    for first, V in ((1, 6000), (2, 4099), (3, 17), (0, 6007)):
        check_beam(ops, wide[:, first:first + V].contiguous(), torch.zeros(2, 4), 5, device=wide.cuda()[:, first:first + V])


def test_beam_of_rows_that_lie_far_apart(ops):
    g = torch.Generator().manual_seed(6)
    wide, row = torch.zeros(8, 2 ** 29 + 4, device="cuda")[:, :9001], 2 * torch.randn(9001, generator=g)
    wide[7] = row.cuda()
    logits = torch.zeros(1, 8, 9001)
    logits[0, 7] = row
    check_beam(ops, logits, torch.full((1, 8), -1.0), 12, device=wide)
    del wide
    torch.cuda.empty_cache()


def test_beams_as_near_as_64_bits_tell(ops):
    """Two beams whose scores differ by less than 32-bit sums are good for."""
    g = torch.Generator().manual_seed(4)
    row = torch.randn(1, 1, 30000, generator=g) * 2
    logits = row.expand(1, 6, -1).contiguous()
    scores = torch.tensor([[-1.0, -1.0 - 2 ** -23, -1.0 + 2 ** -24, -1.0, -1.0 - 2 ** -22, -1.0 + 2 ** -23]])
    check_beam(ops, logits, scores, 24)


@pytest.mark.parametrize("n", [1, 2, 16])
def test_beam_of_rows_in_order(ops, n):
    """Every tile's logits are larger than those in front, or smaller: sums are as good as those of rows in no order."""
    g = torch.Generator().manual_seed(n)
    rows = (5 * torch.randn(40, 3, 32000, generator=g)).sort(-1)[0]
    check_beam(ops, rows, -3 * torch.rand(40, 3, generator=g), n)
    check_beam(ops, rows.flip(-1).contiguous(), -3 * torch.rand(40, 3, generator=g), n)


def test_beam_of_rows_that_are_mostly_equal(ops):
    """One logit, and all others d below: the exponentials' errors are one and the same, and do not average out."""
    for V in (1000, 128256):
        d = torch.linspace(0.01, 14, 60)
        rows = (-d[:, None]).repeat(1, V)
        rows[:, 7] = 0
        best, parents, tokens = torch.empty(60, 1, device="cuda"), ints([[9]] * 60), ints([[9]] * 60)
        ops.beam_select(rows.cuda(), torch.zeros(60, 1, device="cuda"), best, parents, tokens)
        exact = -rows.double().logsumexp(-1)
        outside = 1 - exact.exp()
        # 2^-22 of an exponential; half a step each of the difference and of its product (d and d log2(e) ln 2), log2(e)'s 1.3e-8; the result's half step
        bound = outside * (2.0 ** -22 + d * (2 * U32 + 1.4e-8)) + U32 * exact.abs()
        assert tokens.flatten().tolist() == [7] * 60
        assert ((best.flatten().cpu().double() - exact).abs() <= 1.01 * bound).all()


# ------------------------------------------------------------------ copies
@pytest.mark.parametrize("shapes, dim, dtype", [
    ([(3, 40, 2, 16, 64)] * 2, 1, torch.bfloat16), ([(40, 4, 32, 32), (40, 7), (40, 1)], 0, torch.float32), ([(5, 40, 3)], 1, torch.bfloat16),
    ([(2, 40, 13)], 1, torch.uint8), ([(40, 100000)], 0, torch.float32), ([(2, 3, 40, 8)], 2, torch.float32), ([(6, 41, 64), (3, 7, 64)], 1, torch.float32),
    ([(1, 40, 16)] * 200, 1, torch.float32)])
def test_copies(ops, shapes, dim, dtype):
    rng = random.Random(len(shapes))
    for n in (0, 1, 5, 37, 1024):
        arrays = [torch.randint(0, 200, s, generator=torch.Generator().manual_seed(i)).to(dtype) for i, s in enumerate(shapes)]
        # targets that are sources of others, the same twice, themselves, and outside
        source, target = [rng.randrange(-2, 43) for _ in range(n)], [rng.randrange(-2, 43) for _ in range(n)]
        device = [a.cuda() for a in arrays]
        ops.copy_entries(device, ints(source), ints(target), dim)
        for a, got in zip(arrays, device):
            want = a.float().numpy()
            plain.copy(want, source, target, dim)
            assert np.array_equal(got.float().cpu().numpy(), want), n
    ops.check_branch_errors()


# ------------------------------------------------------------------ together
def rotated(x, positions):
    """Rows ``[T, H, hd]`` turned by their positions."""
    half = x.shape[-1] // 2
    angle = positions.double()[:, None, None] * 10000.0 ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], dim=-1).to(x.dtype)


def test_a_tree_that_is_kept_is_the_context_of_the_next_step(ops):
    """Layout, attention and acceptance of one step: the kept tokens' results are those of the same tokens one behind the other, and the next
    step reads them where they have gone to."""
    g = torch.Generator(device="cuda").manual_seed(1)
    heads, kv_heads, hd, page, ctx = 4, 2, 64, 16, [37, 5]
    parents, tokens = [-1, 0, 0, 1, 2, 4, 4, -1, 0, 1], [1, 2, 3, 4, 5, 6, 7, 1, 2, 3]
    targets = [3, 0, 5, 0, 7, 0, 9, 2, 3, 8]
    cu, R = [0, 7, 10], 2
    kv = [c + b - a for c, a, b in zip(ctx, cu, cu[1:])]
    table = ints([[3, 1, 4, 0], [2, 6, -1, -1]])
    pools = [torch.randn(1, 8, kv_heads, page, hd, generator=g, device="cuda").bfloat16() for _ in range(2)]
    straight = [p.clone() for p in pools]
    q, k, v = (torch.randn(10, n, hd, generator=g, device="cuda").bfloat16() for n in (heads, kv_heads, kv_heads))
    positions, mask = ints([0] * 10), ints([[0]] * 10)
    ops.tree_layout(ints(parents), ints(cu), ints(kv), positions, mask, 7)
    q, k = rotated(q, positions), rotated(k, positions)
    for t in range(10):
        r = int(t >= 7)
        at = ctx[r] + t - cu[r]
        for pool, x in zip(pools, (k, v)):
            pool[0, table[r, at // page], :, at % page] = x[t]
    out = torch.empty(10, heads * hd, dtype=torch.bfloat16, device="cuda")
    ops.tree_attention(q, pools[0][0], pools[1][0], table, ints(cu), ints(kv), positions, mask, out, 0.125, 0, page, 7, max(kv))
    path, kept, after = ints([[0] * 7] * R), ints([0] * R), ints([0] * R)
    ops.tree_accept(ints(tokens), ints(targets), ints(parents), ints(cu), ints(kv), path, kept, after, 7, pools, table, page)
    assert [p[:n] for p, n in zip(path.tolist(), kept.tolist())] == [[0, 2, 4, 6], [0, 1, 2]] and after.tolist() == [9, 8]
    # the same tokens as a stretch
    rows = [0, 2, 4, 6, 7, 8, 9]
    new_cu, new_kv = [0, 4, 7], [ctx[0] + 4, ctx[1] + 3]
    for i, t in enumerate(rows):
        r = int(i >= 4)
        at = ctx[r] + i - new_cu[r]
        for pool, x in zip(straight, (k, v)):
            pool[0, table[r, at // page], :, at % page] = x[t]
    again = torch.empty(7, heads * hd, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention(q[rows].contiguous(), straight[0][0], straight[1][0], table, ints(new_cu), ints(new_kv), ints([0] * 4 + [1] * 3), again, 0.125, 0, page, R,
                        4, max(new_kv))
    torch.testing.assert_close(again.float(), out[rows].float(), rtol=4 * U16, atol=4 * U16)
    for r in range(R):                         # (what lies behind the kept tokens is nobody's)
        for at in range(new_kv[r]):
            for a, b in zip(pools, straight):
                assert torch.equal(a[0, table[r, at // page], :, at % page], b[0, table[r, at // page], :, at % page])


@pytest.mark.parametrize("dtype, hd, window", [(torch.bfloat16, 64, 0), (torch.float32, 16, 0), (torch.bfloat16, 128, 6)])
def test_a_layer_of_a_tree_step(ops, dtype, hd, window):
    """A step's projections, rotated by the tree's positions and written to their places, are read as the same tokens one behind the other are."""
    from garuda_b200.parts.rotary import RotaryParams
    rotary = RotaryParams(10000.0, hd, False)
    g = torch.Generator(device="cuda").manual_seed(hd)
    heads, kv_heads, page, ctx, parents = 4, 2, 8, 13, [-1, 0, 0, 2, 1, 3]
    before, now = (torch.randn(n, (heads + 2 * kv_heads) * hd, generator=g, device="cuda") for n in (ctx, 6))
    pools = [torch.zeros(4, kv_heads, page, hd, dtype=dtype, device="cuda") for _ in range(2)]
    table, zero, scale = ints([[2, 0, 3]]), ints([0] * 13), hd ** -0.5
    ops.rope_kv_append(before, torch.empty(ctx, heads, hd, dtype=dtype, device="cuda"), *pools, ints(list(range(ctx))), zero, table, heads, kv_heads, hd, rotary, page)
    kept = [p.clone() for p in pools]
    positions, mask = ints([0] * 6), ints([[0]] * 6)
    ops.tree_layout(ints(parents), ints([0, 6]), ints([ctx + 6]), positions, mask, 6, window)
    assert positions.tolist() == [13, 14, 14, 15, 15, 16]
    turned, q = now.clone(), torch.empty(6, heads, hd, dtype=dtype, device="cuda")
    ops.rope_inplace(turned[:, :(heads + kv_heads) * hd].view(6, heads + kv_heads, hd), positions, rotary)
    ops.rope_kv_append(turned, q, *pools, ints([ctx + i for i in range(6)]), zero[:6], table, heads, kv_heads, hd, None, page)
    out = torch.empty(6, heads * hd, dtype=dtype, device="cuda")
    ops.tree_attention(q, *pools, table, ints([0, 6]), ints([ctx + 6]), positions, mask, out, scale, window, page, 6, ctx + 6)
    for branch in ([0, 1, 4], [0, 2, 3, 5]):
        n = len(branch)
        straight, at = [p.clone() for p in kept], ints(list(range(ctx, ctx + n)))
        q2, again = torch.empty(n, heads, hd, dtype=dtype, device="cuda"), torch.empty(n, heads * hd, dtype=dtype, device="cuda")
        ops.rope_kv_append(now[branch].contiguous(), q2, *straight, at, zero[:n], table, heads, kv_heads, hd, rotary, page)
        ops.paged_attention(q2, *straight, table, ints([0, n]), ints([ctx + n]), zero[:n], again, scale, window, page, 1, n, ctx + n)
        # (weights are rounded to bfloat16 on both sides)
        tol = 4 * U16 if dtype is torch.bfloat16 else 64 * U32
        torch.testing.assert_close(out[branch].float(), again.float(), rtol=tol, atol=tol)


@pytest.mark.parametrize("name, dtype, graphs", [("A", "float32", True), ("B", "float32", False), ("D", "bfloat16", True)])
def test_beam_search(name, dtype, graphs):
    """The engine's search against the plain one, which runs every beam's whole sequence anew; in bfloat16 by the scores that the plain model gives
    the tokens."""
    from garuda_b200 import Engine
    from tests.helpers import TINY, TOL, folder_weights, model_dir, random_tokens
    from tests.plain import llama_plain
    from tests.test_beams import plain_search
    cfg, folder = TINY[name][0], model_dir(name, torch.bfloat16 if dtype == "bfloat16" else torch.float32)
    w = folder_weights(folder)
    prompts = [random_tokens(name, n, n) for n in (30, 1, 17)]
    e = Engine(folder, dtype=dtype, page_size=8, kv_tokens=1024, max_concurrent=8, cuda_graphs=graphs, eos_token_id=())
    got = e.beam_search(prompts, beams=4, max_tokens=6)
    for p, hypotheses in zip(prompts, got):
        if dtype == "float32":
            want = plain_search(cfg, w, p, 4, 6, 1.0, set(), e.max_context)
            assert [h.tokens for h in hypotheses] == [t for t, *_ in want]
        assert [h.score for h in hypotheses] == sorted((h.score for h in hypotheses), reverse=True) and len({tuple(h.tokens) for h in hypotheses}) == 4
        for h in hypotheses:
            x = llama_plain.forward(cfg, w, p + h.tokens)[len(p) - 1:-1].astype(np.float64)
            lse = x.max(axis=1) + np.log(np.exp(x - x.max(axis=1, keepdims=True)).sum(axis=1))
            score = sum(row[t] - n for row, t, n in zip(x, h.tokens, lse))
            # a logit is off by the tolerance times the largest one, a sum of logarithms by as much: twice that a token
            assert abs(h.score - score) <= 2 * 6 * TOL[dtype] * np.abs(x).max()
    assert e.cache.manager.live_requests == 0
    e.cache.manager.check_invariants()


def test_forked_states_on_the_device():
    from garuda_b200 import Engine
    from tests.test_beams import fork_a_model_with_states
    from tests.test_extensibility import toy_dir
    fork_a_model_with_states(Engine(toy_dir(), dtype="float32", page_size=8, max_concurrent=4))


def test_forked_pages_in_8_bits(ops):
    """Codes and their scales go together."""
    from garuda_b200 import Engine
    from tests.helpers import model_dir, random_tokens
    e = Engine(model_dir("D", torch.bfloat16), dtype="bfloat16", cache_dtype="float8_e4m3", page_size=16, kv_tokens=512, max_concurrent=4)
    from garuda_b200 import StepEntry
    toks = random_tokens("D", 37, 1)
    e.step([StepEntry(1, toks, ())])
    e.cache.fork([(1, 2), (1, 3)], e.ops)
    rows = e.step([StepEntry(r, [11], [0]) for r in (1, 2, 3)])
    assert torch.equal(rows[0], rows[1]) and torch.equal(rows[0], rows[2])


def test_captured_and_replayed(ops):
    """All of it in one graph, with new inputs in the same places; without a workspace and with one; beside eager calls."""
    from garuda_b200.engine.batch import Workspace
    shape = ([(900, 20), (4000, 7), (0, 3)], 8, 2, 128, 32, torch.bfloat16)
    one, two = Step(1, *shape), Step(2, *shape)
    logits, scores = torch.randn(6, 9001, device="cuda"), -torch.rand(2, 3, device="cuda")
    for ws in (None, Workspace(torch.device("cuda"))):
        device = [x.cuda() for x in (one.q, one.k, one.v)] + [torch.from_numpy(one.table).cuda(), ints(one.positions),
                                                              torch.from_numpy(plain.mask_words(one.reads, one.words)).cuda()]
        out = torch.zeros(one.T, 8 * 128, dtype=torch.bfloat16, device="cuda")
        best, parents, tokens = torch.zeros(2, 6, device="cuda"), ints([[0] * 6] * 2), ints([[0] * 6] * 2)
        cu, kv = ints(one.cu), ints(one.kv)

        def call():
            q, k, v, table, positions, mask = device
            ops.tree_attention(q, k, v, table, cu, kv, positions, mask, out, one.scale, 0, 32, one.max_q, one.max_kv, ws=ws)
            ops.beam_select(logits, scores, best, parents, tokens, ws=ws)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
            call()
        for step in (two, one):
            for to, x in zip(device, (step.q, step.k, step.v, torch.from_numpy(step.table), torch.tensor(step.positions, dtype=torch.int32),
                                      torch.from_numpy(plain.mask_words(step.reads, step.words)))):
                to.copy_(x)
            logits.normal_()
            graph.replay()
            Step(9, *shape).run(ops)          # (scratch memory of its own)
            graph.replay()
            step.check(out, True)
            want = plain.beam(logits.cpu().numpy().reshape(2, 3, -1), scores.cpu().numpy(), 6)
            assert np.array_equal(parents.cpu().numpy(), want[1]) and np.array_equal(tokens.cpu().numpy(), want[2])


def test_two_streams_at_once(ops):
    steps = [Step(i, [(3000 + 500 * i, 9), (2500, 30)], 8, 2, 64, 32, torch.bfloat16) for i in range(2)]
    first = [s.run(ops) for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(3):
        outs = []
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                outs.append(s.run(ops))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, outs))
