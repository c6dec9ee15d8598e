"""Serving in 8 bits: what is measured of it, and its plain forms.

Three operators that run one behind the other in a layer whose weights and whose paged cache are held in E4M3:

* ``linear``: ``out = a W^T``, the weights in 8 bits with one scale for each block of 128 x 128, the tokens rounded to 8 bits
  within the call with one scale for each token and 128 channels;
* ``append``: split a projection's rows into heads, rotate queries and keys at their positions, and write keys and values into
  their pages in 8 bits, with one scale for each page and head; a page that held tokens already is re-encoded where its
  scale has to grow;
* ``attention``: causal grouped-query attention over such a cache, for single tokens and for prompt portions.

A scale is a power of two: the smallest that brings the block's largest magnitude to 448 or below, and no smaller than 2^-100. Dividing
by it is exact, so that a value is rounded once, to the nearest E4M3 number.

``own`` chooses between the plain forms (elementary torch operations in 32 bits) and the framework's kernels.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128             # channels (and weight rows) that share a scale in ``linear``
LARGEST = 448.0         # of E4M3
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------ cases

#: (query heads, key/value heads, head size) of the shapes that the benchmark runs
HEADS = {"tinyllama": (32, 4, 64), "llama2-7b": (32, 32, 128), "llama3-8b": (32, 8, 128)}


def _attention(name, shape, requests, tokens, longest, ragged, page, window=0):
    heads, kv_heads, dim = HEADS[shape]
    return {"name": name, "kind": "attention", "heads": heads, "kv_heads": kv_heads, "dim": dim, "requests": requests,
            "tokens": tokens, "longest": longest, "ragged": ragged, "page": page, "window": window}


def _append(name, shape, requests, tokens, longest, ragged, page, interleaved=False):
    heads, kv_heads, dim = HEADS[shape]
    return {"name": name, "kind": "append", "heads": heads, "kv_heads": kv_heads, "dim": dim, "requests": requests,
            "tokens": tokens, "longest": longest, "ragged": ragged, "page": page, "interleaved": interleaved}


def _linear(name, rows, width, inner):
    return {"name": name, "kind": "linear", "rows": rows, "width": width, "inner": inner}


def listed():
    return [
        # one user's next token after a short conversation: the smallest call, all latency
        _attention("decode_1x500", "llama3-8b", 1, 1, 500, False, 32),
        # the benchmark's default: a batch of 8 at 2,048 positions, heads of 64
        _attention("decode_8x2048", "tinyllama", 8, 1, 2048, False, 32),
        # a full server: 64 conversations of every length from a first token to 8,191 positions
        _attention("decode_64_ragged", "llama3-8b", 64, 1, 8191, True, 32),
        # a few very long contexts, where the cache is what is read
        _attention("decode_4x65536", "llama3-8b", 4, 1, 65536, False, 64),
        # a first prompt, no shared heads: every query head has keys of its own
        _attention("prompt_2048", "llama2-7b", 1, 2048, 2048, False, 32),
        # two portions of 509 tokens of long prompts that look back over a window of 4,096
        _attention("portion_2x509_window", "llama3-8b", 2, 509, 8190, True, 32, window=4096),
        # a decode step's tokens of 64 requests go into their pages
        _append("append_64", "llama3-8b", 64, 1, 8191, True, 32),
        # a prompt of 2,047 tokens goes in behind 13 that are there
        _append("append_2047", "llama3-8b", 1, 2047, 2060, False, 32),
        # one token through a square projection: the smallest product
        _linear("linear_1", 1, 2048, 2048),
        # a decode step of 8 through the gate and up projections: bound by the weights
        _linear("linear_8", 8, 28672, 4096),
        # a step of prompt portions and single tokens, an odd number of them
        _linear("linear_301", 301, 4096, 11008),
        # a long prompt through the gate and up projections: bound by the tensor cores
        _linear("linear_4096", 4096, 28672, 4096),
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        case = _drawn(rng)
        if 3 * 1024 not in case.values():       # a size that none of this repository's models has
            return case


def _drawn(rng):
    kind = rng.choice(["decode", "prompt", "append", "linear", "linear"])
    if kind == "linear":
        rows = _log_between(rng, 1, 4096)
        width, inner = _log_between(rng, 512, 28672), 16 * _log_between(rng, 32, 896)
        if rng.random() < 0.5:
            width = -(-width // 64) * 64
        # no more work than the largest listed product
        rows = min(rows, 4096 * 28672 * 4096 // (width * inner))
        return {"kind": "linear", "rows": rows, "width": width, "inner": inner}
    heads, kv_heads, dim = HEADS[rng.choice(sorted(HEADS))]
    page = rng.choice([16, 32, 32, 64])
    base = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": rng.random() < 0.5}
    if kind == "append":
        requests = _log_between(rng, 1, 64)
        tokens = 1 if rng.random() < 0.4 else _log_between(rng, 1, 2048 // requests)
        longest = tokens + _log_between(rng, 1, 4096)
        return dict(base, kind="append", requests=requests, tokens=tokens, longest=longest, interleaved=rng.random() < 0.3)
    window = rng.choice([0, 0, 0, _log_between(rng, 64, 4096)])
    if kind == "decode":
        requests = _log_between(rng, 1, 64)
        longest = _log_between(rng, 1, min(65536, 262144 // requests * 8 // kv_heads))
        return dict(base, kind="attention", requests=requests, tokens=1, longest=longest, window=window)
    requests = rng.choice([1, 1, 2, 3])
    tokens = _log_between(rng, 5, 2048 // requests)
    longest = tokens + rng.choice([0, _log_between(rng, 1, 6144)])
    return dict(base, kind="attention", requests=requests, tokens=tokens, longest=longest, window=window)


def lengths(case):
    """(new tokens, positions behind the step) of every request: from the case alone. Where it is ragged, lengths go from
    little more than the new tokens to the longest, and every third request brings about half as many tokens."""
    out = []
    n = case["requests"]
    for i in range(n):
        tokens, total = case["tokens"], case["longest"]
        if case["ragged"]:
            tokens = tokens - tokens // 2 if i % 3 == 1 else tokens
            total = max(tokens, (total * (i + 1) // n) - (5 * i) % 3 if i + 1 < n else total)
        out.append((tokens, total))
    return out


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["width"], case["inner"]
        blocks = -(-n // BLOCK) * -(-k // BLOCK)
        return {"bytes": m * k * 2 + n * k + 4 * blocks + m * n * 2, "flops": 2 * m * n * k}
    heads, kv_heads, dim, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    asked = lengths(case)
    tokens = sum(q for q, _ in asked)
    if case["kind"] == "append":
        moved = tokens * (heads + 2 * kv_heads) * dim * 4 + tokens * dim * 4          # the projection's rows, cosines and sines
        pages = sum((n - 1) // page - (n - q) // page + 1 for q, n in asked)
        moved += tokens * heads * dim * 2 + 2 * tokens * kv_heads * dim + 8 * pages * kv_heads
        return {"bytes": moved, "flops": 6 * tokens * (heads + kv_heads) * dim // 2 + 2 * tokens * kv_heads * dim}
    read = seen = pages = 0
    for q, n in asked:
        window = case["window"] or n
        first = max(0, n - q + 1 - window)
        read += n - first
        pages += (n - 1) // page - first // page + 1
        # the sum over the new tokens of the keys that each reads
        full = max(0, min(q, n - window)) if case["window"] else 0             # tokens that see a whole window
        part = q - full
        low = n - q + 1                                                        # what the first token sees, without a window
        seen += full * window + part * low + part * (part - 1) // 2
    return {"bytes": 2 * read * kv_heads * dim + 8 * pages * kv_heads + 4 * tokens * heads * dim,
            "flops": 4 * seen * heads * dim}


# ------------------------------------------------------------------ inputs

def _scale_of(largest):
    """The smallest power of two that brings ``largest`` to 448 = 0.875 * 2^9 or below, at least 2^-100 (32-bit)."""
    m, e = torch.frexp(largest)
    e = torch.where(largest > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -100)).clamp(-100, 120)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(x):
    return x.clamp(-LARGEST, LARGEST).to(E4M3)


def _pages_of(x):
    """``x [pages, heads, page, dim]`` in 8 bits and the scale of every page and head."""
    s = _scale_of(x.abs().amax(dim=(2, 3)))
    return _encode(x / s[:, :, None, None]), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["kind"] == "linear":
        m, n, k = case["rows"], case["width"], case["inner"]
        # activations behind a norm: most channels alike, a few tens of times larger
        loud = torch.exp(normal(k).abs().clamp(max=3.0) - 0.8)
        a = (normal(m, k) * loud).to(torch.bfloat16)
        w = normal(n, k) * (0.02 * torch.exp(0.3 * normal(n, 1)))
        nb, kb = -(-n // BLOCK), -(-k // BLOCK)
        whole = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
        whole[:n, :k] = w
        scales = _scale_of(whole.view(nb, BLOCK, kb, BLOCK).abs().amax(dim=(1, 3)))
        spread = scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        values = _encode(w / spread)
        return {"case": case, "a": a, "values": values, "scales": scales,
                "out": torch.empty(m, n, dtype=torch.bfloat16, device="cuda")}

    heads, kv_heads, dim, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    asked = lengths(case)
    requests = len(asked)
    counts = [(n + page - 1) // page for _, n in asked]
    total, width = sum(counts), max(counts)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
    cu = np.cumsum([0] + [q for q, _ in asked])
    tokens = int(cu[-1])
    s = {"case": case, "table": table, "requests": requests, "tokens": tokens,
         "cu_q": torch.tensor(cu, dtype=torch.int32, device="cuda"),
         "kv_lens": torch.tensor([n for _, n in asked], dtype=torch.int32, device="cuda"),
         "max_q": max(q for q, _ in asked), "min_q": min(q for q, _ in asked), "max_kv": max(n for _, n in asked),
         "positions": torch.tensor(np.concatenate([np.arange(n - q, n) for q, n in asked]), dtype=torch.int32, device="cuda"),
         "token_req": torch.tensor(np.repeat(np.arange(requests), [q for q, _ in asked]), dtype=torch.int32, device="cuda")}
    # keys: channels of unequal size, as a rotation's slow pairs have; values: alike. Sizes differ from page to page.
    size = torch.exp(0.5 * normal(kv_heads, 1, dim))
    size = size / size.square().mean(dim=-1, keepdim=True).sqrt()
    keys = normal(total, kv_heads, page, dim) * size
    # the first position draws attention whatever the token (a sink)
    pull = normal(kv_heads, dim)
    pull = pull / pull.norm(dim=-1, keepdim=True) * math.sqrt(dim)
    first = table[:, 0].long()
    keys[first, :, 0] = 2.0 * pull
    s["k_pool"], s["k_scale"] = _pages_of(keys)
    del keys
    values = normal(total, kv_heads, page, dim) * torch.exp(0.3 * normal(total, kv_heads, 1, 1))
    s["v_pool"], s["v_scale"] = _pages_of(values)
    del values
    if case["kind"] == "attention":
        q = normal(tokens, kv_heads, heads // kv_heads, dim) + 0.3 * pull[:, None, :]
        s["q"] = q.reshape(tokens, heads, dim).to(torch.bfloat16)
        s["out"] = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device="cuda")
        # the plain form's padded rows: the token of (request, place), and where its result lies
        place = torch.arange(s["max_q"], device="cuda")[None, :]
        count = (s["cu_q"][1:] - s["cu_q"][:-1])[:, None]
        s["row"] = torch.where(place < count, s["cu_q"][:-1, None] + place, torch.zeros_like(place)).long()
        s["place"] = (torch.arange(tokens, device="cuda") - s["cu_q"][s["token_req"].long()]).long()
        return s
    s["qkv"] = normal(tokens, (heads + 2 * kv_heads) * dim)
    k_part = s["qkv"][:, heads * dim:(heads + kv_heads) * dim]
    k_part *= size.reshape(1, -1)
    angle = s["positions"].double()[:, None] * (10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim))
    s["cos_sin"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()
    s["q_out"] = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device="cuda")
    # the pages that the step writes, how many tokens each held before, and every token's place among them
    page_of = torch.gather(table[s["token_req"].long()], 1, (s["positions"].long() // page)[:, None])[:, 0].long()
    s["touched"], s["slot"] = torch.unique(page_of, return_inverse=True)
    s["line"] = (s["positions"] % page).long()
    held = torch.full((s["touched"].numel(),), page, device="cuda")
    s["held"] = held.scatter_reduce_(0, s["slot"], s["line"], "amin")
    return s


# ------------------------------------------------------------------ the plain forms

def _plain_linear(s):
    m, k = s["a"].shape
    n, kb = s["values"].shape[0], -(-k // BLOCK)
    a = torch.nn.functional.pad(s["a"].float(), (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    scale = _scale_of(a.abs().amax(dim=-1, keepdim=True))
    a = (_encode(a / scale).float() * scale).view(m, kb * BLOCK)[:, :k]
    spread = s["scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return (a @ (s["values"].float() * spread).t()).to(torch.bfloat16)


def _rotated(x, cos_sin, interleaved):
    """``x [T, H, dim]`` by the angles of ``cos_sin [T, dim / 2, 2]``: pairs (2i, 2i + 1), or (i, i + dim / 2)."""
    c, d = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    u, v = a * c - b * d, a * d + b * c
    return torch.stack([u, v], dim=-1).flatten(-2) if interleaved else torch.cat([u, v], dim=-1)


def _plain_append(s):
    case = s["case"]
    heads, kv_heads, dim, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    x = s["qkv"].view(s["tokens"], heads + 2 * kv_heads, dim)
    q = _rotated(x[:, :heads], s["cos_sin"], case["interleaved"]).to(torch.bfloat16)
    k = _rotated(x[:, heads:heads + kv_heads], s["cos_sin"], case["interleaved"])
    _plain_write(s, k, s["k_pool"], s["k_scale"])
    _plain_write(s, x[:, heads + kv_heads:], s["v_pool"], s["v_scale"])
    return q, s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"]


def _plain_write(s, rows, pool, scales):
    touched, slot, line, held = s["touched"], s["slot"], s["line"], s["held"]
    largest = torch.zeros(touched.numel(), rows.shape[1], device="cuda")
    largest.scatter_reduce_(0, slot[:, None].expand(-1, rows.shape[1]), rows.abs().amax(dim=-1), "amax")
    before, need = scales[touched], _scale_of(largest)
    after = torch.where(held[:, None] > 0, torch.maximum(before, need), need)
    old = pool[touched]
    again = _encode(old.float() * (before / after)[:, :, None, None])
    keep = torch.arange(pool.shape[2], device="cuda")[None, None, :, None] < held[:, None, None, None]
    codes = pool.view(torch.uint8)
    codes[touched] = torch.where(keep, again.view(torch.uint8), old.view(torch.uint8))
    codes[touched[slot], :, line] = _encode(rows / after[slot][:, :, None]).view(torch.uint8)
    scales[touched] = after


def _mask(case, position, count, length):
    """True where the query at ``position [R, Q]`` reads key ``[L]`` of a request with ``count [R]`` positions."""
    key = torch.arange(length, device="cuda")
    seen = (key <= position[..., None]) & (key < count[:, None, None])
    return seen & (key > position[..., None] - case["window"]) if case["window"] else seen


def _plain_attention(s):
    case = s["case"]
    kv_heads, dim = case["kv_heads"], case["dim"]
    group = case["heads"] // kv_heads
    requests, most = s["row"].shape
    page = s["table"].clamp(min=0).long()
    length = page.shape[1] * case["page"]

    def cached(pool, scales):
        x = pool[page].float() * scales[page][..., None, None]                     # [R, W, Hkv, page, dim]
        return x.permute(0, 2, 1, 3, 4).reshape(requests, kv_heads, 1, length, dim)

    q = s["q"].float()[s["row"]].view(requests, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    position = (s["kv_lens"] - (s["cu_q"][1:] - s["cu_q"][:-1]))[:, None] + torch.arange(most, device="cuda")
    unseen = ~_mask(case, position, s["kv_lens"], length)[:, None, None]
    score = torch.matmul(q.reshape(requests, kv_heads, 1, group * most, dim), cached(s["k_pool"], s["k_scale"]).transpose(-1, -2))
    score = score.view(requests, kv_heads, group, most, length).mul_(1.0 / math.sqrt(dim)).masked_fill_(unseen, -math.inf)
    weight = score.sub_(score.amax(dim=-1, keepdim=True)).exp_()
    weight = weight.div_(weight.sum(dim=-1, keepdim=True))
    out = torch.matmul(weight.view(requests, kv_heads, 1, group * most, length), cached(s["v_pool"], s["v_scale"]))
    out = out.view(requests, kv_heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(requests, most, -1)
    return out[s["token_req"].long(), s["place"]].to(torch.bfloat16)


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
    if not own:
        return {"linear": _plain_linear, "append": _plain_append, "attention": _plain_attention}[case["kind"]](s)
    ops = _ops()
    if case["kind"] == "linear":
        ops.linear_float8(s["a"], (s["values"], s["scales"]), s["out"])
        return s["out"]
    if case["kind"] == "append":
        ops.kv_append_float8(s["qkv"], s["q_out"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["cu_q"], s["kv_lens"],
                             s["table"], case["heads"], case["kv_heads"], case["dim"], s["cos_sin"], case["interleaved"], case["page"])
        return s["q_out"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"]
    ops.paged_attention_float8(s["q"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["table"], s["cu_q"], s["kv_lens"],
                               s["out"], 1.0 / math.sqrt(case["dim"]), case["window"], case["page"], s["requests"], s["max_q"],
                               s["max_kv"], min_q_len=s["min_q"])
    return s["out"]


# ------------------------------------------------------------------ in 64 bits

def _two_to(e):
    """2^e in 64 bits, to the bit (a library's power may be a last place off)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _power_of_two(largest):
    """The scale of a block in 64 bits, by comparison: 2^e with e the least whole number from -100 on with 448 * 2^e >= largest."""
    e = torch.ceil(torch.log2((largest / LARGEST).clamp(min=2.0 ** -120)))
    e = torch.where(_two_to(e) * LARGEST < largest, e + 1, e)
    e = torch.where(_two_to(e - 1) * LARGEST >= largest, e - 1, e)
    return _two_to(e.clamp(-100, 120))


def _nearest_e4m3(x):
    """The E4M3 number nearest to each of ``x`` (64 bits), ties to the even one: steps of 2^(e - 3) from 2^e on, 2^-9 below 2^-6."""
    x = x.clamp(-LARGEST, LARGEST)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = _two_to(e - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        k, n = case["inner"], case["width"]
        a = s["a"].double()
        out = torch.zeros(case["rows"], n, dtype=torch.float64, device="cuda")
        for b in range(0, k, BLOCK):
            part = a[:, b:b + BLOCK]
            scale = _power_of_two(part.abs().amax(dim=1, keepdim=True))
            row_scale = s["scales"][:, b // BLOCK].double().repeat_interleave(BLOCK)[:n]
            out += (_nearest_e4m3(part / scale) * scale) @ (s["values"][:, b:b + BLOCK].double() * row_scale[:, None]).t()
        return out
    heads, kv_heads, dim, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    asked = lengths(case)
    if case["kind"] == "append":
        x = s["qkv"].double().view(-1, heads + 2 * kv_heads, dim)
        z = torch.view_as_complex(s["cos_sin"].double().contiguous())[:, None, :]
        turn = x[:, :heads + kv_heads]
        if case["interleaved"]:
            turned = torch.view_as_real(torch.view_as_complex(turn.reshape(*turn.shape[:2], dim // 2, 2).contiguous()) * z).flatten(-2)
        else:
            w = torch.complex(turn[..., :dim // 2].contiguous(), turn[..., dim // 2:].contiguous()) * z
            turned = torch.cat([w.real, w.imag], dim=-1)
        out = [turned[:, :heads]]
        pools, scales = [], []
        for rows, pool, scale in ((turned[:, heads:], s["k_pool"], s["k_scale"]), (x[:, heads + kv_heads:], s["v_pool"], s["v_scale"])):
            pool, scale, first = pool.double(), scale.double(), 0
            table = s["table"].cpu().tolist()
            for r, (q, n) in enumerate(asked):
                new, p = rows[first:first + q], n - q
                first += q
                while p < n:                       # page by page
                    at, line = table[r][p // page], p % page
                    end = min(n, p - line + page)
                    part = new[p - (n - q):end - (n - q)]                          # [tokens, heads, dim]
                    need = _power_of_two(part.abs().amax(dim=(0, 2)))
                    now = torch.maximum(scale[at], need) if line else need
                    if line:
                        pool[at, :, :line] = _nearest_e4m3(pool[at, :, :line] * (scale[at] / now)[:, None, None])
                    pool[at, :, line:line + end - p] = _nearest_e4m3(part / now[:, None]).transpose(0, 1)
                    scale[at] = now
                    p = end
            pools.append(pool)
            scales.append(scale)
        return tuple(out + pools + scales)
    out = torch.empty(s["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    first = 0
    for r, (q, n) in enumerate(asked):
        pages = s["table"][r, :(n + page - 1) // page].long()
        position = torch.arange(n - q, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None, :]
        hidden = key > position
        if case["window"]:
            hidden = hidden | (position - key >= case["window"])
        for h in range(kv_heads):
            k = (s["k_pool"][pages, h].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)[:n]
            v = (s["v_pool"][pages, h].double() * s["v_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)[:n]
            for j in range(h * (heads // kv_heads), (h + 1) * (heads // kv_heads)):
                score = (s["q"][first:first + q, j].double() @ k.t() / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                out[first:first + q, j] = torch.softmax(score, dim=-1) @ v
        first += q
    return out.flatten(1)
