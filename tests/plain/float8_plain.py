"""Plain forms of the 8-bit path on the CPU: codes by their definition, products, cache writes and attention in 64 bits."""
import math

import torch

BLOCK, LARGEST = 128, 448.0
E4M3 = torch.float8_e4m3fn


def scale_of(largest: float) -> float:
    """2^e, e the smallest whole number from -100 (to 120) with 448 * 2^e >= largest."""
    if not largest > 0:
        return 2.0 ** -100
    if math.isinf(largest):
        return 2.0 ** 120
    m, e = math.frexp(largest)              # largest = m * 2^e, 448 = 0.875 * 2^9
    return 2.0 ** min(max(e - 9 + (m > 0.875), -100), 120)


def scales_of(x: torch.Tensor) -> torch.Tensor:
    """Scales of the largest magnitudes ``x`` (a NaN counts as nothing), 64-bit."""
    flat = [scale_of(v) for v in torch.nan_to_num(x.double(), nan=0.0, posinf=math.inf).flatten().tolist()]
    return torch.tensor(flat, dtype=torch.float64).view(x.shape)


def encode(x: torch.Tensor) -> torch.Tensor:
    """The nearest E4M3 numbers (ties to the even one), 448 beyond that, NaN for NaN; as numbers in 64 bits, by search over all codes."""
    table = torch.arange(127, dtype=torch.uint8).view(E4M3).double()          # the 127 numbers from 0 to 448
    y = x.double()
    mag = torch.nan_to_num(y.abs(), nan=0.0, posinf=LARGEST).clamp(max=LARGEST)
    hi = torch.searchsorted(table, mag.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = mag - table[lo], table[hi] - mag
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    out = torch.copysign(table[pick], y)
    return torch.where(torch.isnan(y), torch.full_like(y, math.nan), out)


def magnitude(x, dims):
    return torch.nan_to_num(x.double().abs(), nan=0.0, posinf=math.inf).amax(dim=dims)


def rows(a):
    """``a [M, K]`` as its rounded values, 64-bit."""
    M, K = a.shape
    out = torch.empty(M, K, dtype=torch.float64)
    for b in range(0, K, BLOCK):
        part = a[:, b:b + BLOCK].double()
        s = scales_of(magnitude(part, (1,)))[:, None]
        out[:, b:b + BLOCK] = encode(part / s) * s
    return out


def weight(w):
    """(codes as numbers [N, K], scales [ceil(N / 128), ceil(K / 128)]) of ``w``, 64-bit."""
    N, K = w.shape
    codes = torch.empty(N, K, dtype=torch.float64)
    scales = torch.empty((N + 127) // 128, (K + 127) // 128, dtype=torch.float64)
    for i in range(0, N, BLOCK):
        for j in range(0, K, BLOCK):
            part = w[i:i + BLOCK, j:j + BLOCK].double()
            s = scale_of(float(magnitude(part, (0, 1))))
            scales[i // BLOCK, j // BLOCK] = s
            codes[i:i + BLOCK, j:j + BLOCK] = encode(part / s)
    return codes, scales


def linear(a, codes, scales):
    """(product, sum of magnitudes) of ``rows(a)`` and the weight ``codes * scales``, 64-bit."""
    N, K = codes.shape
    w = codes.double() * scales.double().repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    x = rows(a)
    return x @ w.T, x.abs() @ w.abs().T


def rotate(x, cos_sin, interleaved):
    """``x [T, H, hd]`` in ``x``'s own precision, every product and sum rounded by itself."""
    c, d = cos_sin[:, None, :, 0].to(x.dtype), cos_sin[:, None, :, 1].to(x.dtype)
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    u, v = a * c - b * d, a * d + b * c
    return torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)


def append(qkv, pools, scales, cu_q, kv_lens, table, heads, kv_heads, hd, cos_sin, interleaved, page):
    """(queries 32-bit, [keys', values'], [key scales', value scales']): the pools as numbers ``[pages, kv_heads, page, hd]``, 64-bit.
    The rotation is in 32 bits, as the operator's is."""
    x = qkv.float().view(-1, heads + 2 * kv_heads, hd)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    if cos_sin is not None:
        q, k = rotate(q, cos_sin, interleaved), rotate(k, cos_sin, interleaved)
    pools, scales = [p.double().clone() for p in pools], [s.double().clone() for s in scales]
    for new, pool, scale in ((k, pools[0], scales[0]), (v, pools[1], scales[1])):
        for r in range(len(kv_lens)):
            t, n = int(cu_q[r]), int(kv_lens[r])
            p = n - (int(cu_q[r + 1]) - t)
            while p < n:
                at, line = int(table[r, p // page]), p % page
                end = min(n, p - line + page)
                part = new[t:t + end - p].double()
                if at >= 0:
                    need = scales_of(magnitude(part, (0, 2)))
                    now = torch.maximum(scale[at], need) if line else need
                    if line:
                        pool[at, :, :line] = encode(pool[at, :, :line] * (scale[at] / now)[:, None, None])
                    pool[at, :, line:line + end - p] = encode(part / now[:, None]).transpose(0, 1)
                    scale[at] = now
                t, p = t + end - p, end
    return q, pools, scales


def attention(q, k_pool, v_pool, k_scale, v_scale, table, cu_q, kv_lens, scale, window, page):
    """(result, sum of weighted magnitudes) ``[T, Hq * hd]`` in 64 bits; a row with no key it may read is zeros."""
    T, Hq, hd = q.shape
    Hkv = k_pool.shape[1]
    out, mag = torch.zeros(T, Hq, hd, dtype=torch.float64), torch.zeros(T, Hq, hd, dtype=torch.float64)
    k_pool, v_pool = k_pool.double() * k_scale.double()[..., None, None], v_pool.double() * v_scale.double()[..., None, None]
    for r in range(len(kv_lens)):
        n, begin, end = int(kv_lens[r]), int(cu_q[r]), int(cu_q[r + 1])
        if end <= begin:
            continue
        pages = table[r, :(n + page - 1) // page].long()
        have = (pages >= 0).repeat_interleave(page)[:n]
        pos, key = torch.arange(n - (end - begin), n)[:, None], torch.arange(n)[None, :]
        seen = (key <= pos) & have[None, :]
        if window:
            seen = seen & (key > pos - window)
        for h in range(Hq):
            k = k_pool[pages.clamp(min=0), h // (Hq // Hkv)].reshape(-1, hd)[:n]
            v = v_pool[pages.clamp(min=0), h // (Hq // Hkv)].reshape(-1, hd)[:n]
            k, v = torch.where(have[:, None], k, 0), torch.where(have[:, None], v, 0)
            s = (q[begin:end, h].double() @ k.T * scale).masked_fill(~seen, -math.inf)
            w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if not torch.isnan(s).any() else torch.softmax(s, -1)
            out[begin:end, h], mag[begin:end, h] = w @ v, w @ v.abs()
    return out.flatten(1), mag.flatten(1)
