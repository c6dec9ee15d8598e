"""Decoding along branches on the device where calls are large, long or odd: many tiles that some rows must not read, many requests, wide groups, long trees."""
import numpy as np
import pytest
import torch

from tests.plain import branches_plain as plain
from tests.test_branches_gpu import Step, check_beam, ints, ops  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads, kv_heads, hd, copies", [(1, 1, 64, 1), (1, 1, 128, 1), (4, 2, 128, 1), (4, 4, 64, 4), (8, 4, 128, 4)])
def test_values_that_are_not_finite_in_many_tiles_in_a_row(ops, heads, kv_heads, hd, copies):
    """Eight tiles of drafted tokens behind one another, each with values that a few rows read and the others must not notice: one request, whose blocks of rows
    have a cluster each, and many. (Marks of a tile that came too late, or from another tile, would change which rows are no numbers.)"""
    clean = Step(hd, [(50, 1000)] * copies, heads, kv_heads, hd, 32, torch.bfloat16, reads=True)
    spoilt = Step(hd, [(50, 1000)] * copies, heads, kv_heads, hd, 32, torch.bfloat16, reads=True)
    bad = [j for j in range(1000) if j % 41 in (3, 7)]
    for step in (clean, spoilt):
        for t, reads in enumerate(step.reads):
            for j in bad:
                reads.discard(j)
                if (7 * t + j) % 60 == 0:
                    reads.add(j)
    for r in range(copies):
        for j in bad:
            page, line = spoilt.table[r, (50 + j) // 32], (50 + j) % 32
            spoilt.v[page, :, line, j % hd] = (float("nan"), float("inf"), float("-inf"))[j % 3]
    want, got = (s.run(ops).view(s.T, heads, hd) for s in (clean, spoilt))
    reads_bad = torch.tensor([not reads.isdisjoint(bad) for reads in spoilt.reads], device="cuda")
    assert 0 < int(reads_bad.sum()) < len(reads_bad)
    assert got[reads_bad].isnan().all()
    assert torch.equal(got[~reads_bad], want[~reads_bad]) and not want.isnan().any()
    for _ in range(3):
        assert torch.equal(spoilt.run(ops).view(torch.int16), got.reshape(spoilt.T, -1).view(torch.int16))
    ops.check_branch_errors()


@pytest.mark.parametrize("heads, kv_heads, hd", [(2, 2, 64), (4, 2, 128)])
def test_many_pieces_of_one_and_two_tiles(ops, heads, kv_heads, hd):
    """Requests of one to three tiles each, several to a stretch: the warps that bring queries, keys and values go from piece to piece side by side."""
    step = Step(hd, [(64 * (i % 6) + i % 5, 1 + i % 4) for i in range(500)], heads, kv_heads, hd, 32, torch.bfloat16)
    first = step.run(ops)
    step.check(first, True)
    for _ in range(20):
        assert torch.equal(step.run(ops), first)
    ops.check_branch_errors()


# ------------------------------------------------------------------ beams
@pytest.mark.parametrize("V", [3, 1237, 5001, 16387, 50257])
@pytest.mark.parametrize("first", [0, 1])
def test_alike_beams_wherever_their_rows_begin(ops, V, first):
    """Rows of the same logits that begin on different four bytes: their candidates' scores are equal, and come in the order of the beams."""
    items = 12
    g = torch.Generator().manual_seed(V)
    logits = 4 * torch.randn(items, 1, V, generator=g).expand(items, 3, V)
    wide = torch.empty(items * 3, V + (V % 2 == 0) + 2 * first)
    wide[:, first:first + V] = logits.reshape(-1, V)
    device = wide.cuda()[:, first:first + V]
    assert len({device[i].data_ptr() % 16 for i in range(36)}) == 4
    check_beam(ops, logits.contiguous(), torch.full((items, 3), -1.25), min(3 * V, 13), device=device)


def test_beam_repeats_itself(ops):
    """Results do not depend on which of a block's threads come first: sums in 64 bits of rising rows, whose lists are cut often."""
    g = torch.Generator().manual_seed(8)
    logits = torch.cat([3 * torch.randn(30, 50257, generator=g), (3 * torch.randn(30, 50257, generator=g)).sort(-1)[0]]).cuda()
    scores, outs = -torch.rand(12, 5, generator=g).cuda(), []
    for _ in range(20):
        outs.append((torch.empty(12, 40, device="cuda"), ints([[9] * 40] * 12), ints([[9] * 40] * 12)))
        ops.beam_select(logits, scores, *outs[-1])
    for out in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out, outs[0]))


@pytest.mark.parametrize("V", [1 << 17, 1 << 20, 1 << 22])
def test_beam_of_equal_logits_far_below_the_largest(ops, V):
    """What the wrapper states for rows of one logit and others d below, in vocabularies where these are most of the sum although they lie far below."""
    d = torch.linspace(float(np.log(V)) - 4, float(np.log(V)) + 4, 30)
    rows = (-d[:, None]).repeat(1, V)
    rows[:, V // 3] = 0
    best, parents, tokens = torch.empty(30, 1, device="cuda"), ints([[9]] * 30), ints([[9]] * 30)
    ops.beam_select(rows.cuda(), torch.zeros(30, 1, device="cuda"), best, parents, tokens)
    exact = -torch.log1p((V - 1) * torch.exp(-d.double()))
    assert tokens.flatten().tolist() == [V // 3] * 30
    # an exponential's 2^-22, 2^-24 each of the difference, its product with log2(e) and, of four equal terms, the third's and the fourth's sum, log2(e)'s 1.3e-8; and half
    # a step of the result
    assert ((best.flatten().cpu().double() - exact).abs() <= 1.01 * (2.0 ** -21 + 1.35e-7 * d + 2.0 ** -24 * exact.abs())).all()


# ------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("dtype, hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float32, 128), (torch.bfloat16, 96)])
@pytest.mark.parametrize("ctx, window, at, large", [(700, 0, 100, None), (700, 650, 100, None), (700, 0, 100, 600), (700, 0, 600, 100), (700, 650, 70, 130), (700, 650, 200, 600),
                                                    (700, 0, 70, 10), (700, 0, 705, 100), (700, 0, 702, 704), (9000, 0, 100, 8900), (9000, 8990, 8000, 200), (100, 0, 60, 99)])
def test_a_value_that_is_read_and_not_finite_shows(ops, dtype, hd, ctx, window, at, large):
    """Wherever its key lies, in a tile that all rows read or at an edge, and if its weight is nothing beside a much larger one's."""
    clean, spoilt = (Step(ctx + hd, [(ctx, 9), (40, 3)], 4, 2, hd, 32, dtype, window) for _ in range(2))
    for step in (clean, spoilt):
        step.q = step.q.abs() + 0.5
        for reads in step.reads[:9]:
            reads.update({2, 4, 5})
        if large is not None:
            step.k[step.table[0, large // 32], :, large % 32] = 40.0
    for i, bad in enumerate((float("inf"), float("nan"), float("-inf"))):
        spoilt.v[spoilt.table[0, at // 32], 0, at % 32, 3 + i] = bad
    want, got = (s.run(ops).view(s.T, 4, hd).float() for s in (clean, spoilt))
    assert want.isfinite().all()
    assert not got[:9, :2, 3:6].isfinite().any()
    assert torch.equal(got[:, 2:], want[:, 2:]) and torch.equal(got[9:], want[9:])
    rest = [c for c in range(hd) if c not in (3, 4, 5)]
    if dtype is torch.float32 or hd == 96:
        assert torch.equal(got[..., rest], want[..., rest])
    else:
        assert (got[:9, :2].isnan() | (got == want)[:9, :2])[..., rest].all()
    ops.check_branch_errors()


# ------------------------------------------------------------------ threads
def test_threads_that_call_at_once(ops):
    """Several threads, each with a stream of its own, in calls of many shapes: what each gets is what it gets alone."""
    import threading
    shapes = [([(c, q)] * r, 8, 2, hd, 32, dtype) for dtype in (torch.bfloat16, torch.float32) for hd in (64, 128) for c, q, r in ((20, 3, 1), (900, 17, 2), (2500, 5, 40))]
    steps = [Step(i, *shape) for i, shape in enumerate(shapes)]
    got, failed = [[None] * len(steps) for _ in range(4)], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(len(steps)):
                    j = (i + 3 * k) % len(steps)
                    s = steps[j]
                    device = [x.cuda() for x in (s.q, s.k, s.v)]
                    out = torch.empty(s.T, s.heads * s.hd, dtype=s.dtype, device="cuda")
                    ops.tree_attention(*device, torch.from_numpy(s.table).cuda(), ints(s.cu), ints(s.kv), ints(s.positions),
                                       torch.from_numpy(plain.mask_words(s.reads, s.words)).cuda(), out, s.scale, 0, 32, s.max_q, s.max_kv)
                    got[k][j] = out
                torch.cuda.current_stream().synchronize()
        except Exception as e:          # (told by the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for j, s in enumerate(steps):
        want = s.run(ops)
        assert all(torch.equal(got[k][j], want) for k in range(4))
    ops.check_branch_errors()


# ------------------------------------------------------------------ ranges
@pytest.mark.parametrize("dtype, requests", [(torch.bfloat16, 2100), (torch.bfloat16, 4097), (torch.float32, 2100)])
def test_attention_of_thousands_of_requests(ops, dtype, requests):
    """More than one launch has places for: the second one has the same scratch memory."""
    step = Step(requests, [(i * 37 % 150, i % 3) for i in range(requests)], 2, 1, 64, 16, dtype, 60 * (requests == 2100))
    first = step.run(ops)
    step.check(first, dtype is torch.bfloat16)
    assert torch.equal(step.run(ops), first)
    ops.check_branch_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, hd", [(16, 1, 64), (32, 2, 128), (12, 1, 128), (40, 1, 64), (65, 1, 64), (128, 1, 128), (130, 1, 64), (66, 2, 64)])
def test_attention_of_wide_groups(ops, dtype, heads, kv_heads, hd):
    """Blocks of 128 rows that have few tokens, or not a whole number of them; more query heads to a key/value head than a block has rows."""
    step = Step(heads, [(300, 5), (0, 1), (127, 9), (40, 0), (1000, 2)], heads, kv_heads, hd, 32, dtype, reads=heads % 3 == 0)
    step.check(step.run(ops), dtype is torch.bfloat16 and heads // kv_heads <= 128)
    ops.check_branch_errors()


@pytest.mark.parametrize("window", [0, 100, 5000])
def test_layout_of_the_longest_trees(ops, window):
    """A chain of 8,192 tokens, and a tree of as many."""
    n, ctx = 8192, [7, 1000]
    rng = np.random.default_rng(window)
    bushy = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
    positions, mask = ints([9] * (2 * n)), torch.full((2 * n, 256), 9, dtype=torch.int32, device="cuda")
    ops.tree_layout(ints(list(range(-1, n - 1)) + bushy), ints([0, n, 2 * n]), ints([c + n for c in ctx]), positions, mask, n, window)
    want, reads = plain.layout(bushy, [0, n], [ctx[1] + n], window)
    assert positions[n:].tolist() == want
    assert np.array_equal(mask[n:].cpu().numpy(), plain.mask_words(reads, 256))
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = (j <= i) & ((j > i - window) if window else True)
    bits = (mask[:n, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    assert torch.equal(bits.reshape(n, n).bool(), seen) and torch.equal(positions[:n], (i[:, 0] + ctx[0]).int())


@pytest.mark.parametrize("n, page, steps", [(1000, 16, 400), (8192, 64, 500), (8191, 1, 150)])
def test_accept_of_the_longest_trees(ops, n, page, steps):
    """Paths that end near a tree's last token, beside a request of one: every row goes where it belongs."""
    rng = np.random.default_rng(n)
    path = [0] + sorted(rng.choice(np.arange(1, n), steps - 1, replace=False).tolist())
    parents, tokens, targets = [-1] + [0] * (n - 1), [1] * n, [2] * n
    for a, b in zip(path, path[1:]):
        parents[b], tokens[b], targets[a] = a, 10 + b, 10 + b
    ctx, cu = [70, 3], [0, n, n + 1]
    parents, tokens, targets = parents + [-1], tokens + [5], targets + [6]
    need = [-(-(c + q) // page) for c, q in zip(ctx, (n, 1))]
    pages = sum(need)
    order = rng.permutation(pages)
    table = np.full((2, max(need)), -1, dtype=np.int32)
    table[0, :need[0]], table[1, :need[1]] = order[:need[0]], order[need[0]:]
    pool = torch.randn(2, pages, 2, page, 8, generator=torch.Generator().manual_seed(n))
    want = pool.numpy().copy()
    got, out, kept, after = pool.cuda(), torch.full((2, n), 9, dtype=torch.int32, device="cuda"), ints([9, 9]), ints([9, 9])
    ops.tree_accept(ints(tokens), ints(targets), ints(parents), ints(cu), ints([ctx[0] + n, ctx[1] + 1]), out, kept, after, n, [got],
                    torch.from_numpy(table).cuda(), page)
    assert plain.accept(tokens, targets, parents, cu)[0] == [path, [0]]
    assert kept.tolist() == [steps, 1] and after.tolist() == [2, 6]
    assert out.tolist() == [path + [-1] * (n - steps), [0] + [-1] * (n - 1)]
    plain.move_rows(want, table[0], page, ctx[0], path)
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("items, beams, V, n", [(65535, 1, 5, 3), (1023, 64, 33, 64), (3000, 2, 4101, 5)])
def test_beam_of_many_rows(ops, items, beams, V, n):
    g = torch.Generator().manual_seed(items)
    logits, scores = 3 * torch.randn(items, beams, V, generator=g), -torch.rand(items, beams, generator=g)
    best, parents, tokens = torch.empty(items, n, device="cuda"), torch.empty(items, n, dtype=torch.int32, device="cuda"), torch.empty(items, n, dtype=torch.int32, device="cuda")
    ops.beam_select(logits.reshape(-1, V).cuda(), scores.cuda(), best, parents, tokens)
    value = scores.cuda().double()[:, :, None] + logits.cuda().double().log_softmax(-1)
    exact, at = value.reshape(items, -1).sort(dim=1, descending=True, stable=True)
    assert ((best.double() - exact[:, :n]).abs() <= 1.01 * 2.0 ** -24 * exact[:, :n].abs() + 1e-7).all()
    # (scores as near as the sums' errors may change places)
    here = (parents.long() * V + tokens.long())
    assert (value.reshape(items, -1).gather(1, here) - exact[:, :n]).abs().max() <= 4e-7
    assert float((here == at[:, :n]).double().mean()) > 0.999 and int(here.sort(1)[0].diff(dim=1).min()) > 0
    ops.check_branch_errors()
