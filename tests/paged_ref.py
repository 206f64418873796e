"""Plain 64-bit forms of the paged KV-cache operators and the bounds their
results are held to, shared by the paged tests."""
import math

import torch

# ggml type ids by name, and the torch types that hold them
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def round_away(x):
    t = torch.trunc(x)
    return torch.where((x - t).abs() >= 0.5, t + torch.sign(x), t)


def q8_0(x):
    """Q8_0 blocks of f32 rows [.., dh] in f32 arithmetic (as ggml's quantiser): quants and fp16 scales."""
    b = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    # (a tensor divisor: torch multiplies by the reciprocal of a Python one, which is not the quotient)
    d = b.abs().amax(-1, keepdim=True) / torch.full((1,), 127.0, device=x.device)
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    return round_away(b * inv).to(torch.int8).reshape(x.shape), d[..., 0].to(torch.float16)


def rotate(x, cs):
    """NEOX pairs of x [n, heads, dh] turned by cs [n, dh / 2, 2], every product and sum rounded to x's type."""
    h = x.shape[-1] // 2
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def make_pools(n_pages, n_kv, page, dh, cache, layout, gen, device, mag=1.0):
    """(k, v, k_scale, v_scale) of shape [n_pages, n_kv, page, dh] in the asked memory layout, random rows."""
    out, scales = [], []
    for _ in range(2):
        x = torch.randn((n_pages, n_kv, page, dh), generator=gen, device=device) * mag
        q, s = (x.to(TORCH[cache]), None) if cache != "q8_0" else q8_0(x)
        if layout == "tokens":       # [pages][tokens][heads][dh]
            q = q.transpose(1, 2).contiguous().transpose(1, 2)
            s = None if s is None else s.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "layers":     # a layer of a pool that holds three per page
            w = torch.zeros((n_pages, 3) + tuple(q.shape[1:]), dtype=q.dtype, device=device)
            w[:, 1] = q
            q = w[:, 1]
            if s is not None:
                w = torch.zeros((n_pages, 3) + tuple(s.shape[1:]), dtype=s.dtype, device=device)
                w[:, 1] = s
                s = w[:, 1]
        out.append(q)
        scales.append(s)
    return out[0], out[1], scales[0], scales[1]


def values(pool, scale):
    """What a pool's rows stand for, in 64 bits."""
    x = pool.double()
    return x if scale is None else x * scale.double().repeat_interleave(32, -1)


def attend(k, v, q, table, lens, scale):
    """out, lse and the sums the error bound needs, in 64 bits. k, v: 64-bit pools [pages, kv, page, dh]."""
    n, H, dh = q.shape
    n_kv, page = k.shape[1], k.shape[2]
    G = H // n_kv
    out = torch.zeros((n, H, dh), dtype=torch.float64, device=q.device)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device=q.device)
    absv = torch.zeros_like(out)      # sum p |v| / sum p
    ds = torch.zeros_like(lse)        # largest scale sum |q| |k| over the keys
    vmax = torch.zeros_like(lse)      # largest |v|
    for b in range(n):
        L = int(lens[b])
        if L <= 0:
            continue
        ids = table[b, :(L + page - 1) // page].long()
        kb = k[ids].transpose(0, 1).reshape(n_kv, -1, dh)[:, :L]
        vb = v[ids].transpose(0, 1).reshape(n_kv, -1, dh)[:, :L]
        qb = q[b].double().view(n_kv, G, dh)
        s = torch.einsum("jgd,jtd->jgt", qb, kb) * scale
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        out[b] = (torch.einsum("jgt,jtd->jgd", p, vb) / z).reshape(H, dh)
        absv[b] = (torch.einsum("jgt,jtd->jgd", p, vb.abs()) / z).reshape(H, dh)
        lse[b] = (m + torch.log(z)).reshape(H)
        vmax[b] = vb.abs().amax((1, 2)).repeat_interleave(G)
        ds[b] = (torch.einsum("jgd,jtd->jgt", qb.abs(), kb.abs()).amax(-1) * abs(scale)).reshape(H)
    return out, lse, (absv, vmax), ds


U = 2.0 ** -24


def attend_bounds(out, lse, sums, ds, lens, dh, dtype):
    """Largest |error| of out and lse that the kernel's arithmetic allows.

    A score: operands taken to 2^-21 or better, a product rounded and a sum of
    dh terms in f32, then scaled and moved to base 2 (3 roundings of the score
    itself): |ds| <= (dh + 16) u * scale sum |q||k|. exp turns |ds| into a
    relative error of a weight, twice (numerator and sum); the exponential
    itself is good to 4 u plus the rounding of its argument s - m, which is
    below 2 ds. A weight is used to 2^-21 (8 u). The weighted sums add 16 keys
    at a time, one tile after another and then warps and splits:
    (len / 16 + 256) u of sum p |v|. Then one rounding to the result's type.

    A weight has a floor too: taken as f16 planes it is 2^14 p at most 2^14
    (for Q8_0 times a block scale over a power of two D at or below the largest
    one, so at most 2^15), and the second plane ends at the f16 grid's 2^-24:
    each is off by 2^-25, which is 2^-39 of the largest weight (Q8_0: 2^-39 D,
    times a quant of at most 127, where 127 D is at most the largest |v|). A
    weight below 2^-126 of the largest is 0 for every type. Over len keys, with
    sum p >= 1: len 2^-39 max |v|, seen where the keys of large weight have a
    value of 0.
    """
    absv, vmax = sums
    steps = (lens.double().clamp(min=0) / 16 + 256)[:, None]
    rel = 2 * ((dh + 16) * U * ds + 8 * U + 4 * U * ds) + 2 * steps * U
    step = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    floor = (lens.double().clamp(min=0)[:, None] * 2.0 ** -39 * vmax)[..., None]
    b_out = (rel[..., None] * absv + floor) * (1 + step) + step * out.abs() + tiny
    b_lse = (dh + 20) * U * ds + (steps + 8) * U + 2 * U * torch.nan_to_num(lse, neginf=0.0).abs()
    return b_out, b_lse
