"""Latent attention in 64 bits: what tests/test_gpu_mla*.py compare the kernels with.

A cache here is a dict of the pool, the table and, for every sequence, its rows as
the values that they stand for, so that a check needs none of the operators."""
from __future__ import annotations

import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E4M3 = tuple((k % 8) / 8 * 2.0 ** -6 if k < 8 else (1 + (k % 8) / 8) * 2.0 ** (k // 8 - 7)
             for k in range(127))
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gen(seed, device="cpu"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def quantise(x, fmt):
    """(codes, scale bytes, values) of rows [n][L] in blocks of 32: the least power of two, 2^-110
    at least, by which no code saturates; nearest codes, ties to even."""
    grid = torch.tensor(E4M3 if fmt == "mxfp8" else E2M1, dtype=torch.float64)
    n, L = x.shape
    b = x.double().cpu().reshape(n, L // 32, 32)
    byte = torch.full((n, L // 32, 1), 17)
    for _ in range(240):
        byte = byte + (b.abs().amax(-1, keepdim=True) > grid[-1] * 2.0 ** (byte - 127.0)).int()
    y = b * 2.0 ** (127.0 - byte)
    a = y.abs()
    hi = torch.searchsorted(grid, a).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    k = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    v = grid[k] * torch.where(torch.signbit(y), -1.0, 1.0)
    sign = torch.signbit(y).long() * (128 if fmt == "mxfp8" else 8)
    return ((k + sign).reshape(n, L), byte.reshape(n, L // 32),
            (v * 2.0 ** (byte - 127.0)).reshape(n, L))


def row_bytes(L, R, fmt):
    return {"16bit": 2 * L, "mxfp8": L + 16, "mxfp4": L // 2 + 16}[fmt] + 2 * R


def as_bytes(t):
    return t.contiguous().view(torch.uint8).reshape(t.shape[0], t.shape[1] * t.element_size())


def encode(latent, rotary, fmt):
    """Cached rows [n][bytes] and the latents that they stand for, from 16-bit rows."""
    n, L = latent.shape
    latent, rotary = latent.cpu(), rotary.cpu()
    turned = as_bytes(rotary) if rotary.shape[1] else torch.zeros((n, 0), dtype=torch.uint8)
    if fmt == "16bit":
        return torch.cat([as_bytes(latent), turned], 1), latent.double()
    codes, scales, values = quantise(latent, fmt)
    if fmt == "mxfp4":
        codes = codes[:, 0::2] + 16 * codes[:, 1::2]
    tail = torch.zeros((n, 16), dtype=torch.uint8)
    tail[:, :L // 32] = scales.to(torch.uint8)
    return torch.cat([codes.to(torch.uint8), turned, tail], 1), values


def make_cache(lens, L, R, page, fmt="16bit", dtype=torch.bfloat16, seed=0, spare=2, width=None,
               junk=True, scale=1.0):
    """Random rows of every sequence in pages of random order.  junk: bytes of all ones (NaN in
    16 bits and E4M3) in every slot that no sequence uses, and page numbers past the pool in the
    table's unused entries."""
    g = gen(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    width = max(1, max(counts)) if width is None else width
    perm = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), width), -1 if junk else 0, dtype=torch.int32)
    pool = torch.full((pages, page, row_bytes(L, R, fmt)), 255 if junk else 0, dtype=torch.uint8)
    rows, at = [], 0
    for n, m in enumerate(lens):
        ids = perm[at:at + counts[n]]
        at += counts[n]
        table[n, :counts[n]] = ids.int()
        latent = (torch.randn((m, L), generator=g) * scale).to(dtype)
        rotary = (torch.randn((m, R), generator=g) * scale).to(dtype)
        data, values = encode(latent, rotary, fmt)
        pos = torch.arange(m)
        if m:
            pool[ids[pos // page], pos % page] = data
        rows.append((values, rotary.double()))
    return dict(pool=pool, table=table, rows=rows, lens=lens, L=L, R=R, fmt=fmt, dtype=dtype)


def softmax_rows(q, k, v, sees, scale, dtype, d_extra=4):
    """Attention of rows q [m][D] over k [n][D], v [n][V], of which row i sees sees[i]: outputs,
    logarithms of sums, and the tolerances of both.

    A score is a sum of D products, each step of it off by at most 2^-23 of the sum of their
    sizes (the matrix cores may cut where they do not round), and the scale, its product and the
    exponential's argument a few more: ds.  A weight is then off by a factor of exp(2 ds) (its own
    score and the largest), by 2^-21 for the exponential itself and by half a step of its type;
    the sum over n weights by n 2^-23 of itself, and so is the product with v.  The output is
    rounded once more.

    Below 2^-126 numbers may become zeros: the output, each weight (taken from a maximum that is
    not above the row's, so that the largest weight and the sum that divides are 1 or more), which
    then misses 2^-126 of its value at most, and each product of a weight and a value."""
    n, half = k.shape[0], HALF[dtype]
    sees = sees.clamp(0, n)
    hidden = torch.arange(n) >= sees[:, None]
    x = (q @ k.t() * scale).masked_fill(hidden, -torch.inf)
    lse = torch.logsumexp(x, 1) if n else torch.full((len(q),), -torch.inf, dtype=torch.float64)
    empty = (sees == 0)[:, None]
    w = (x - lse[:, None]).exp().masked_fill(hidden | empty, 0.0)
    out = w @ v
    if not n:
        return out, lse, torch.zeros_like(out), torch.zeros_like(lse)
    size = ((q.abs() @ k.abs().t()) * scale).masked_fill(hidden, 0.0).amax(1)
    far = x.abs().masked_fill(hidden, 0.0).amax(1)
    ds = size * (q.shape[1] + d_extra) * 2.0 ** -23 + far * 2.0 ** -22
    off = half + 2 * ds + 2 * (sees + 8) * 2.0 ** -23 + 2.0 ** -20
    tol = half * out.abs() + (1 + half) * off[:, None] * (w @ v.abs())
    tol += 2.0 ** -126 * (1 + (~hidden).double() @ (v.abs() + 1))
    if dtype == torch.float16:
        tol += 2.0 ** -25  # half a step of its subnormal numbers
    ltol = ds + (sees + 8) * 2.0 ** -23 + 2.0 ** -20 + lse.abs() * 2.0 ** -23
    return out, lse, tol.masked_fill(empty, 0.0), ltol.masked_fill(empty[:, 0], 0.0)


def attention(cache, q, counts, scale):
    """What mla_attention returns for q [T][H][L + R], sequence by sequence, with tolerances."""
    H = q.shape[1]
    outs = []
    first = 0
    for n, m in enumerate(counts):
        latent, rotary = cache["rows"][n]
        rows = q[first:first + m].double().cpu().reshape(m * H, q.shape[2])
        at = torch.arange(m).repeat_interleave(H)
        sees = cache["lens"][n] - m + at + 1
        outs.append(softmax_rows(rows, torch.cat([latent, rotary], 1), latent, sees, scale,
                                 cache["dtype"]))
        first += m
    out, lse, tol, ltol = (torch.cat([o[i] for o in outs]) for i in range(4))
    T = first
    return (out.view(T, H, -1), lse.view(T, H), tol.view(T, H, -1), ltol.view(T, H))


def prompt(q, k, v, rotary, counts, keys, causal, scale):
    """What mla_prompt returns, with tolerances."""
    T, H, _ = q.shape
    res = [torch.zeros((T, H, v.shape[2]), dtype=torch.float64),
           torch.zeros((T, H), dtype=torch.float64)]
    res += [torch.zeros_like(res[0]), torch.zeros_like(res[1])]
    a = b = 0
    for m, n in zip(counts, keys):
        for h in range(H):
            kk = k[b:b + n, h].double().cpu()
            if rotary is not None:
                kk = torch.cat([kk, rotary[b:b + n].double().cpu()], 1)
            sees = torch.arange(m) + n - m + 1 if causal else torch.full((m,), n)
            one = softmax_rows(q[a:a + m, h].double().cpu(), kk, v[b:b + n, h].double().cpu(),
                               sees, scale, q.dtype)
            for r, o in zip(res, one):
                r[a:a + m, h] = o
        a, b = a + m, b + n
    return res


def close(got, want, tol):
    """Largest error over its tolerance; infinities and zeros have to be equal."""
    got = got.double().cpu()
    same = (got == want)
    e = torch.where(same, 0.0, (got - want).abs() / tol.clamp(min=1e-300))
    assert not torch.isnan(e).any()
    return float(e.max()) if e.numel() else 0.0
