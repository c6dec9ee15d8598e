"""Decoding along several branches: what is measured of it, and its plain forms.

Four operators over the paged cache and the logits of a step, for drafted tokens that form a tree and for beams:

* ``attention``: grouped-query attention of a request's tree of drafted tokens: each reads the request's context and those of the tree's
  tokens that a mask of bits names (its ancestors and itself);
* ``accept``: the walk from a tree's first token along the drafted tokens that the model would have chosen itself, and the rows of those
  tokens in every layer's pages moved together behind the context;
* ``beam``: the best continuations of an item over all its beams and the whole vocabulary, from logits and the beams' scores;
* ``copy``: pages of a cache, or states of fixed size, copied to other places in every layer at once, as forked beams need them.

``own`` chooses between the plain forms (elementary torch operations) and the framework's kernels.
"""
import math
import random

import numpy as np
import torch

own = False

#: (query heads, key/value heads, head size, layers) of the shapes that the benchmark runs
SHAPES = {"tinyllama": (32, 4, 64, 22), "llama2-7b": (32, 32, 128, 32), "llama3-8b": (32, 8, 128, 32)}
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------ cases

def _attention(name, shape, requests, tokens, longest, ragged, page, window=0, dtype="bfloat16", branches=3):
    return {"name": name, "kind": "attention", "shape": shape, "requests": requests, "tokens": tokens, "longest": longest, "ragged": ragged,
            "page": page, "window": window, "dtype": dtype, "branches": branches}


def _accept(name, shape, layers, requests, tokens, longest, kept, page, dtype="bfloat16"):
    return {"name": name, "kind": "accept", "shape": shape, "layers": layers, "requests": requests, "tokens": tokens, "longest": longest,
            "kept": kept, "page": page, "dtype": dtype}


def _beam(name, items, beams, chosen, vocab, first=False):
    return {"name": name, "kind": "beam", "items": items, "beams": beams, "chosen": chosen, "vocab": vocab, "first": first}


def _pages(name, shape, layers, copies, page, dtype="bfloat16"):
    return {"name": name, "kind": "pages", "shape": shape, "layers": layers, "copies": copies, "page": page, "dtype": dtype}


def _states(name, layers, heads, dim, copies, slots):
    return {"name": name, "kind": "states", "layers": layers, "heads": heads, "dim": dim, "copies": copies, "slots": slots}


def listed():
    return [
        # one user's tree of 8 tokens after a short conversation: all latency
        _attention("tree_1x8_500", "llama3-8b", 1, 8, 500, False, 32),
        # a server's 32 conversations of every length to 8,191 positions, trees of up to 24 tokens
        _attention("tree_32x24_ragged", "llama3-8b", 32, 24, 8191, True, 32),
        # two long contexts, trees of 64 tokens, every query head with keys of its own: the largest
        _attention("tree_2x64_16384", "llama2-7b", 2, 64, 16384, False, 32, branches=4),
        # the 32-bit path: four trees of 12
        _attention("tree_4x12_float32", "tinyllama", 4, 12, 1024, True, 32, dtype="float32"),
        # one user's tree of 8: three of its tokens are kept, in 22 layers
        _accept("accept_1x8", "tinyllama", 22, 1, 8, 500, 3, 32),
        # 64 trees of 64 tokens in 32 layers
        _accept("accept_64x64", "llama3-8b", 32, 64, 64, 110, 6, 32),
        # one item, four beams
        _beam("beam_1x4", 1, 4, 8, 32000),
        # eight items in their first step: of five beams, one has a score yet
        _beam("beam_8x5_first", 8, 5, 10, 128256, first=True),
        # 64 items of eight beams: the most logits
        _beam("beam_64x8", 64, 8, 16, 128256),
        # one item's prompt has just become four beams: the last page three times over, in 22 layers
        _pages("fork_3", "tinyllama", 22, 3, 32),
        # sixteen items of four beams, all of which begin a page
        _pages("fork_48", "llama3-8b", 32, 48, 32),
        # forked beams of a recurrent model: matrix states of eight layers
        _states("states_16", 8, 16, 128, 16, 40),
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "accept", "beam", "beam", "pages", "states"])
    shape = rng.choice(sorted(SHAPES))
    kv_heads, dim = SHAPES[shape][1:3]
    page = rng.choice([16, 32, 32, 64])
    if kind == "attention":
        exact32 = rng.random() < 0.2
        requests = _log_between(rng, 1, 8 if exact32 else 64)
        tokens = _log_between(rng, 1, min(16 if exact32 else 100, 2048 // requests))
        # no more keys than the largest listed case holds, nor more products with them; a sixteenth in 32 bits
        keys = min(2 * 16384 * 32 * 128 // (kv_heads * dim * requests), 2 * 16384 * 64 * 32 * 128 // (requests * tokens * 32 * dim))
        longest = tokens + _log_between(rng, 1, max(2, min(8192, keys // 16) if exact32 else min(32768, keys)))
        return {"kind": kind, "shape": shape, "requests": requests, "tokens": tokens, "longest": longest, "ragged": rng.random() < 0.5,
                "page": page, "window": rng.choice([0, 0, 0, _log_between(rng, 40, 4096)]), "dtype": "float32" if exact32 else "bfloat16",
                "branches": rng.choice([1, 2, 3, 5])}
    if kind == "accept":
        requests, kept = _log_between(rng, 1, 64), rng.randint(1, 8)
        tokens, dtype = kept * 8 + rng.randint(0, 30), rng.choice(["bfloat16", "bfloat16", "float32"])
        longest = tokens + rng.randint(1, 300)
        # the pools hold no more than half a GB
        layers = max(1, min(32, (1 << 29) // (4 * requests * (longest + page) * kv_heads * dim)))
        return {"kind": kind, "shape": shape, "layers": rng.randint(1, layers), "requests": requests, "tokens": tokens, "longest": longest,
                "kept": kept, "page": page, "dtype": dtype}
    if kind == "beam":
        items, beams = _log_between(rng, 1, 64), rng.randint(1, 10)
        vocab = _log_between(rng, 1000, min(131072, 64 * 8 * 128256 // (items * beams)))
        return {"kind": kind, "items": items, "beams": beams, "chosen": rng.randint(1, 2 * beams), "vocab": vocab,
                "first": rng.random() < 0.25}
    if kind == "pages":
        layers = rng.randint(1, 32)
        most = 48 * 32 * 8 * 32 * 128 // (layers * kv_heads * page * dim * 2)
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        return {"kind": kind, "shape": shape, "layers": layers, "copies": _log_between(rng, 1, max(1, min(64, most))), "page": page,
                "dtype": dtype}
    copies = _log_between(rng, 1, 24)
    return {"kind": kind, "layers": rng.randint(1, 8), "heads": rng.choice([4, 8, 16]), "dim": rng.choice([32, 64, 128]), "copies": copies,
            "slots": 2 * copies + rng.randint(0, 9)}


def lengths(case):
    """(drafted tokens, positions behind the step) of every request: from the case alone. Where it is ragged, lengths go from little more
    than the drafted tokens to the longest, and every third request brings about half as many tokens."""
    out = []
    n = case["requests"]
    for i in range(n):
        tokens, total = case["tokens"], case["longest"]
        if case.get("ragged"):
            tokens = tokens - tokens // 2 if i % 3 == 1 else tokens
            total = max(tokens, (total * (i + 1) // n) - (5 * i) % 3 if i + 1 < n else total)
        out.append((tokens, max(tokens, total)))
    return out


def kept_of(case):
    """How many of its tokens each request of an ``accept`` keeps: the first always, at most ``kept``."""
    return [1 + (case["kept"] - 1 + 5 * r) % case["kept"] for r in range(case["requests"])]


def work(case):
    kind = case["kind"]
    if kind == "beam":
        rows = case["items"] * case["beams"]
        return {"bytes": 4 * rows * case["vocab"] + 4 * rows + 12 * case["items"] * case["chosen"], "flops": 4 * rows * case["vocab"]}
    if kind == "states":
        return {"bytes": 2 * 4 * case["layers"] * case["copies"] * case["heads"] * case["dim"] ** 2, "flops": 0}
    heads, kv_heads, dim, _ = SHAPES[case["shape"]]
    item = DTYPES[case["dtype"]].itemsize
    if kind == "pages":
        return {"bytes": 2 * 2 * item * case["layers"] * case["copies"] * kv_heads * case["page"] * dim, "flops": 0}
    if kind == "accept":
        moved = sum(kept - 1 for kept in kept_of(case))
        return {"bytes": 2 * 2 * item * case["layers"] * moved * kv_heads * dim + 12 * case["requests"] * case["tokens"]
                + 4 * sum(kept_of(case)) + 8 * case["requests"], "flops": 0}
    read = seen = tokens = pages = 0
    for q, n in lengths(case):
        window = case["window"] or n
        first = max(0, n - q + 1 - window)
        read += n - first
        pages += (n - 1) // case["page"] - first // case["page"] + 1
        seen += q * (n - q - first + 1)           # the context that the window leaves, and at least the token itself
        tokens += q
    words = (case["tokens"] + 31) // 32
    return {"bytes": 2 * item * read * kv_heads * dim + 2 * item * tokens * heads * dim + 4 * (pages + tokens * (1 + words)),
            "flops": 4 * seen * heads * dim}


# ------------------------------------------------------------------ inputs

def _tree(rng, tokens, branches):
    """A tree's parents, each in front of its children: token 0 is the request's last one, up to ``branches`` candidates continue a token."""
    parents, room = [-1], [0]
    for i in range(1, tokens):
        at = room[0] if rng.random() < 0.6 else rng.choice(room)
        parents.append(at)
        if sum(p == at for p in parents) >= branches:
            room.remove(at)
        room.append(i)
    return parents


def _levels(rng, tokens, kept):
    """Parents of a tree in levels, and a path of ``kept`` tokens through it whose rows do not lie where the kept ones go."""
    wide = max(1, (tokens - 1) // max(1, kept - 1)) if kept > 1 else tokens
    level, parents = [0], [-1]
    path = [0]
    while len(parents) < tokens:
        here = list(range(len(parents), min(tokens, len(parents) + wide)))
        for i, node in enumerate(here):
            parents.append(path[-1] if i == len(here) - 1 else rng.choice(level))
        if len(path) < kept:
            path.append(here[-1])
        level = here
    return parents, path


def _paged(s, asked, page, generator):
    """Block tables over pages in a random order, and the arrays that describe a step's tokens."""
    counts = [(n + page - 1) // page for _, n in asked]
    total, width = sum(counts), max(counts)
    order = torch.randperm(total, generator=generator, device="cuda").to(torch.int32)
    table = torch.full((len(asked), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
    cu = np.cumsum([0] + [q for q, _ in asked])
    s["table"], s["tokens"] = table, int(cu[-1])
    s["cu_q"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    s["kv_lens"] = torch.tensor([n for _, n in asked], dtype=torch.int32, device="cuda")
    s["max_q"], s["max_kv"] = max(q for q, _ in asked), max(n for _, n in asked)
    s["req"] = torch.tensor(np.repeat(np.arange(len(asked)), [q for q, _ in asked]), device="cuda")
    s["first"] = torch.tensor([n - q for q, n in asked], device="cuda")
    return total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rng = random.Random(int(seed))
    kind = case["kind"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    s = {"case": case}
    if kind == "beam":
        rows = case["items"] * case["beams"]
        logits = normal(rows, case["vocab"]) * 2.0
        # a few likely tokens a row, and some that a sampling rule forbids
        likely = torch.randint(0, case["vocab"], (rows, 24), generator=g, device="cuda")
        logits.scatter_add_(1, likely, 4.0 + 6.0 * torch.rand((rows, 24), generator=g, device="cuda"))
        logits[:, :3] = -math.inf
        scores = -8.0 * torch.rand((case["items"], case["beams"]), generator=g, device="cuda") - 1.0
        if case["first"]:
            scores[:, 0], scores[:, 1:] = 0.0, -math.inf
        n = case["chosen"]
        s.update(logits=logits, scores=scores, best=torch.empty(case["items"], n, device="cuda"),
                 parents=torch.empty(case["items"], n, dtype=torch.int32, device="cuda"),
                 chosen=torch.empty(case["items"], n, dtype=torch.int32, device="cuda"))
        return s
    if kind == "states":
        order = torch.randperm(case["slots"], generator=g, device="cuda").to(torch.int32)
        n = case["copies"]
        # a beam may go on in several others: sources come twice
        s["source"], s["target"] = order[:n][torch.randint(0, n, (n,), generator=g, device="cuda")].contiguous(), order[n:2 * n].contiguous()
        s["arrays"] = [normal(case["slots"], case["heads"], case["dim"], case["dim"]) for _ in range(case["layers"])]
        s["dim"] = 0
        return s
    heads, kv_heads, dim, _ = SHAPES[case["shape"]]
    dtype, page = DTYPES[case["dtype"]], case["page"]
    if kind == "pages":
        n = case["copies"]
        order = torch.randperm(2 * n + 5, generator=g, device="cuda").to(torch.int32)
        s["source"], s["target"] = order[:n][torch.randint(0, n, (n,), generator=g, device="cuda")].contiguous(), order[n:2 * n].contiguous()
        s["arrays"] = [normal(case["layers"], 2 * n + 5, kv_heads, page, dim, dtype=dtype) for _ in range(2)]
        s["dim"] = 1
        return s
    asked = lengths(case)
    total = _paged(s, asked, page, g)
    if kind == "accept":
        parents, drafted, wanted = [], [], []
        for (q, _), kept in zip(asked, kept_of(case)):
            up, path = _levels(rng, q, kept)
            tokens = [rng.randrange(32000) for _ in range(q)]
            model = [-1 - i for i in range(q)]                # (what no drafted token is)
            for a, b in zip(path, path[1:]):
                # of several candidates alike the first counts
                tokens[b] = 32000 + b
                model[a] = tokens[b]
            model[path[-1]] = rng.randrange(32000, 33000) + 1000
            parents += up
            drafted += tokens
            wanted += model
        s["parents"], s["drafted"], s["wanted"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (parents, drafted, wanted))
        s["pools"] = [normal(case["layers"], total, kv_heads, page, dim, dtype=dtype) for _ in range(2)]
        n = len(asked)
        s["path"] = torch.empty(n, s["max_q"], dtype=torch.int32, device="cuda")
        s["kept"], s["next"] = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
        return s
    s["parents"] = torch.tensor([p for q, _ in asked for p in _tree(rng, q, case["branches"])], dtype=torch.int32, device="cuda")
    # keys: channels of unequal size; the first position draws attention whatever the token (a sink)
    size = torch.exp(0.5 * normal(kv_heads, 1, dim))
    size = size / size.square().mean(dim=-1, keepdim=True).sqrt()
    pull = normal(kv_heads, dim)
    pull = pull / pull.norm(dim=-1, keepdim=True) * math.sqrt(dim)
    keys = normal(total, kv_heads, page, dim, dtype=dtype).mul_(size.to(dtype))
    keys[s["table"][:, 0].long(), :, 0] = (2.0 * pull).to(dtype)
    s["k_pool"], s["v_pool"] = keys, normal(total, kv_heads, page, dim, dtype=dtype)
    q = normal(s["tokens"], kv_heads, heads // kv_heads, dim) + 0.3 * pull[:, None, :]
    s["q"] = q.reshape(s["tokens"], heads, dim).to(dtype)
    s["out"] = torch.empty(s["tokens"], heads * dim, dtype=dtype, device="cuda")
    # a step's plan, which all its layers share: positions and masks of bits from the trees
    if own:
        s["positions"] = torch.empty(s["tokens"], dtype=torch.int32, device="cuda")
        s["mask"] = torch.empty(s["tokens"], (s["max_q"] + 31) // 32, dtype=torch.int32, device="cuda")
        _ops().tree_layout(s["parents"], s["cu_q"], s["kv_lens"], s["positions"], s["mask"], s["max_q"], case["window"])
    else:
        s["positions"], s["mask"] = _plain_layout(s, case["window"])
    # the plain form's padded rows: the token of (request, place), and where its result lies
    place = torch.arange(s["max_q"], device="cuda")[None, :]
    count = (s["cu_q"][1:] - s["cu_q"][:-1])[:, None]
    s["row"] = torch.where(place < count, s["cu_q"][:-1, None] + place, torch.zeros_like(place)).long()
    s["place"] = (torch.arange(s["tokens"], device="cuda") - s["cu_q"][s["req"]]).long()
    return s


# ------------------------------------------------------------------ the plain forms

def _ancestors(s):
    """(depth, [T, longest] truth) of every drafted token: how far down it is, and whom of its request's tokens it descends from, itself
    among them."""
    parents, cu = s["parents"].tolist(), s["cu_q"].tolist()
    depth, reads = np.zeros(len(parents), dtype=np.int64), np.zeros((len(parents), s["max_q"]), dtype=bool)
    for a, b in zip(cu, cu[1:]):
        for t in range(a, b):
            if parents[t] >= 0:
                depth[t] = depth[a + parents[t]] + 1
                reads[t] = reads[a + parents[t]]
            reads[t, t - a] = True
    return depth, reads


def _plain_layout(s, window):
    depth, reads = _ancestors(s)
    position = s["first"][s["req"]] + torch.from_numpy(depth).cuda()
    if window:
        cu = s["cu_q"].tolist()
        for a, b in zip(cu, cu[1:]):
            reads[a:b, :b - a] &= depth[a:b][:, None] - depth[a:b][None, :] < window
    words = (s["max_q"] + 31) // 32
    bits = np.zeros((reads.shape[0], words * 32), dtype=np.uint8)
    bits[:, :s["max_q"]] = reads
    mask = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    return position.to(torch.int32), torch.from_numpy(mask.copy()).cuda()


def _plain_attention(s):
    case = s["case"]
    heads, kv_heads, dim, _ = SHAPES[case["shape"]]
    group = heads // kv_heads
    requests, most = s["row"].shape
    page = s["table"].clamp(min=0).long()
    length = page.shape[1] * case["page"]

    def cached(pool):
        return pool[page].float().permute(0, 2, 1, 3, 4).reshape(requests, kv_heads, length, dim)       # from [R, W, Hkv, page, dim]

    # what each query reads: the context, as far as its window goes back, and the tokens that its bits name
    key = torch.arange(length, device="cuda")[None, None, :]
    position, first = s["positions"][s["row"]][:, :, None], s["first"][:, None, None]
    sees = key < first
    if case["window"]:
        sees = sees & (key > position - case["window"])
    place = key - first
    words = s["mask"][s["row"]]                                                                         # [R, most, words]
    bit = words.gather(2, (place >> 5).clamp(0, words.shape[2] - 1).expand(-1, most, -1)) >> (place & 31) & 1
    sees = sees | ((place >= 0) & (key < s["kv_lens"][:, None, None]) & (bit == 1))
    q = s["q"].float()[s["row"]].view(requests, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(requests, kv_heads, group * most, dim), cached(s["k_pool"]).transpose(-1, -2))
    score = score.view(requests, kv_heads, group, most, length).mul_(1.0 / math.sqrt(dim)).masked_fill_(~sees[:, None, None], -math.inf)
    weight = score.sub_(score.amax(dim=-1, keepdim=True)).exp_()
    weight = weight.div_(weight.sum(dim=-1, keepdim=True))
    out = torch.matmul(weight.view(requests, kv_heads, group * most, length), cached(s["v_pool"]))
    out = out.view(requests, kv_heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(requests, most, -1)
    return out[s["req"], s["place"]].to(s["q"].dtype)


def _plain_accept(s):
    """All requests' walks at once, a step for every token that may be kept; then the rows, read before any is written."""
    cu, first = s["cu_q"].long(), s["first"]
    requests, most = s["path"].shape
    here = torch.zeros(requests, dtype=torch.long, device="cuda")
    alive = cu[1:] > cu[:-1]
    path = torch.full((requests, most), -1, dtype=torch.int32, device="cuda")
    after = torch.full((requests,), -1, dtype=torch.int32, device="cuda")
    place = torch.arange(s["tokens"], device="cuda") - cu[s["req"]]
    for step in range(min(most, s["case"]["kept"] + 1)):
        path[:, step] = torch.where(alive, here, torch.full_like(here, -1)).to(torch.int32)
        model = s["wanted"][(cu[:-1] + here).clamp(max=s["tokens"] - 1)]
        after = torch.where(alive, model, after)
        fits = (s["parents"] == here[s["req"]]) & (s["drafted"] == model[s["req"]]) & alive[s["req"]]
        child = torch.full((requests,), most, dtype=torch.long, device="cuda")
        child.scatter_reduce_(0, s["req"], torch.where(fits, place, torch.full_like(place, most)), "amin")
        alive = alive & (child < most)
        here = torch.where(alive, child, here)
    kept = (path >= 0).sum(dim=1).to(torch.int32)
    page = s["case"]["page"]
    r, to = (path >= 0).nonzero(as_tuple=True)
    slots = [first[r] + path[r, to].long(), first[r] + to]
    where = [(s["table"][r, x // page].long(), x % page) for x in slots]
    for pool in s["pools"]:
        pool[:, where[1][0], :, where[1][1]] = pool[:, where[0][0], :, where[0][1]]
    return (path, kept, after, *s["pools"])


def _plain_beam(s):
    """In 64 bits: two continuations may be as near as 32 bits can tell apart."""
    items, beams = s["scores"].shape
    n = s["best"].shape[1]
    x = s["logits"].double()
    top = x.amax(dim=1, keepdim=True)
    total = (x - top).exp().sum(dim=1, keepdim=True).log() + top
    score = (s["scores"].double().view(-1, 1) + (x - total)).view(items, -1)
    score = torch.where(score.isnan(), torch.full_like(score, -math.inf), score)
    best, at = torch.sort(score, dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    vocab = s["logits"].shape[1]
    return best.float(), (at // vocab).to(torch.int32), (at % vocab).to(torch.int32)


def _plain_copy(s):
    source, target = s["source"].long(), s["target"].long()
    for array in s["arrays"]:
        array.index_copy_(s["dim"], target, array.index_select(s["dim"], source))
    return tuple(s["arrays"])


# ------------------------------------------------------------------ one pass

_kernels = None


def _ops():
    """The framework's kernel set, as an engine keeps it."""
    global _kernels
    if _kernels is None:
        from garuda_b200.kernels.ops import CudaOps
        _kernels = CudaOps()
    return _kernels


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if not own:
        return {"attention": _plain_attention, "accept": _plain_accept, "beam": _plain_beam, "pages": _plain_copy,
                "states": _plain_copy}[kind](s)
    ops = _ops()
    if kind == "attention":
        ops.tree_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["cu_q"], s["kv_lens"], s["positions"], s["mask"], s["out"],
                           1.0 / math.sqrt(s["q"].shape[2]), case["window"], case["page"], s["max_q"], s["max_kv"])
        return s["out"]
    if kind == "accept":
        ops.tree_accept(s["drafted"], s["wanted"], s["parents"], s["cu_q"], s["kv_lens"], s["path"], s["kept"], s["next"], s["max_q"],
                        s["pools"], s["table"], case["page"])
        return (s["path"], s["kept"], s["next"], *s["pools"])
    if kind == "beam":
        ops.beam_select(s["logits"], s["scores"], s["best"], s["parents"], s["chosen"])
        return s["best"], s["parents"], s["chosen"]
    ops.copy_entries(s["arrays"], s["source"], s["target"], s["dim"])
    return tuple(s["arrays"])


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "beam":
        items, beams = s["scores"].shape
        best, parents, chosen = [], [], []
        for i in range(items):
            rows = s["logits"][i * beams:(i + 1) * beams].double()
            value = s["scores"][i].double()[:, None] + torch.log_softmax(rows, dim=-1)
            value = torch.where(value.isnan(), torch.full_like(value, -math.inf), value).flatten()
            # all that are no worse than the last of the chosen, in the order of their numbers; then by value
            least = torch.topk(value, s["best"].shape[1]).values[-1]
            at = (value >= least).nonzero()[:, 0]
            at = at[torch.argsort(value[at], descending=True, stable=True)][:s["best"].shape[1]]
            best.append(value[at])
            parents.append((at // rows.shape[1]).to(torch.int32))
            chosen.append((at % rows.shape[1]).to(torch.int32))
        return torch.stack(best), torch.stack(parents), torch.stack(chosen)
    if kind in ("pages", "states"):
        arrays = [a.double() for a in s["arrays"]]
        for a, b in zip(s["source"].tolist(), s["target"].tolist()):
            for x in arrays:
                x.select(s["dim"], b).copy_(x.select(s["dim"], a))
        return tuple(arrays)
    asked = lengths(case)
    cu = s["cu_q"].tolist()
    if kind == "accept":
        pools = [x.double() for x in s["pools"]]
        path = torch.full(s["path"].shape, -1, dtype=torch.int32)
        kept, after = [], []
        parents, drafted, wanted, table = (s[k].tolist() for k in ("parents", "drafted", "wanted", "table"))
        for r, (q, n) in enumerate(asked):
            a = cu[r]
            walk = [0]
            while True:
                fits = [i for i in range(q) if parents[a + i] == walk[-1] and drafted[a + i] == wanted[a + walk[-1]]]
                if not fits:
                    break
                walk.append(fits[0])
            path[r, :len(walk)] = torch.tensor(walk, dtype=torch.int32)
            kept.append(len(walk))
            after.append(wanted[a + walk[-1]])
            for to, node in enumerate(walk):                 # (a row only ever moves towards the front)
                x, y = n - q + node, n - q + to
                for pool in pools:
                    pool[:, table[r][y // case["page"]], :, y % case["page"]] = pool[:, table[r][x // case["page"]], :, x % case["page"]]
        return (path.cuda(), torch.tensor(kept, dtype=torch.int32, device="cuda"), torch.tensor(after, dtype=torch.int32, device="cuda"), *pools)
    heads, kv_heads, dim, _ = SHAPES[case["shape"]]
    depth, reads = _ancestors(s)
    out = torch.empty(s["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    for r, (q, n) in enumerate(asked):
        a = cu[r]
        pages = s["table"][r, :(n + case["page"] - 1) // case["page"]].long()
        down = torch.from_numpy(depth[a:a + q]).cuda()
        hidden = torch.zeros(q, n, dtype=torch.bool, device="cuda")
        hidden[:, n - q:] = ~torch.from_numpy(reads[a:a + q, :q]).cuda()
        if case["window"]:
            at = torch.cat([torch.arange(n - q, device="cuda"), n - q + down])
            hidden |= (n - q + down)[:, None] - at[None, :] >= case["window"]
        for h in range(kv_heads):
            k, v = (x[pages, h].double().reshape(-1, dim)[:n] for x in (s["k_pool"], s["v_pool"]))
            mine = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            score = torch.einsum("thd,kd->htk", s["q"][a:a + q, mine].double(), k) / math.sqrt(dim)
            out[a:a + q, mine] = (torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1) @ v).transpose(0, 1)
    return out.flatten(1)
