"""The paged key-value cache operators, measured.

Four paths of a serving step over a paged cache, each as a user's program
calls it:

  plan    pages for the tokens a step appends, block tables, slot map
  append  RoPE on q and k, k and v into their pages
  attend  one new token per request over its pages
  step    append, then attend, on a Q8_0 cache

`run` computes them from elementary torch operations, or (own = True) with
toy_b200.paged. `exact` computes them from their definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4.0, "bf16": 2.0, "f16": 2.0, "q8_0": 1.0 + 2.0 / 32}


# ------------------------------------------------------------------ the cases
def _plan(name, n, page, max_len, mix):
    return {"name": name, "op": "plan", "n": n, "page": page, "max_len": max_len, "mix": mix}


def _append(name, tokens, heads, kv, dh, page, dtype, cache, bias=False, padded=0):
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "kv": kv, "dh": dh, "page": page,
            "dtype": dtype, "cache": cache, "bias": bias, "padded": padded}


def _attend(name, n, heads, kv, dh, page, dtype, cache, lo, hi, lse=False, op="attend"):
    return {"name": name, "op": op, "n": n, "heads": heads, "kv": kv, "dh": dh, "page": page, "dtype": dtype,
            "cache": cache, "lo": lo, "hi": hi, "lse": lse}


def listed():
    return [
        # one decode step of a small batch: each request appends one token
        _plan("plan 16 decode", 16, 16, 1024, "decode"),
        # continuous batching: most requests decode, some append a chunk of their prompt, some wait
        _plan("plan 509 mixed", 509, 16, 4096, "mixed"),
        # a burst of new requests whose whole prompts are appended
        _plan("plan 1024 prompts", 1024, 64, 512, "prompt"),
        # a decode step of eight sequences of a 9 / 3-head, width-64 model, f32 throughout
        _append("append 8 f32", 8, 9, 3, 64, 16, "f32", "f32"),
        # a padded decode batch with a q|k|v bias, 28 / 4 heads of width 128
        _append("append 250 bf16", 250, 28, 4, 128, 16, "bf16", "bf16", bias=True, padded=6),
        # a prompt chunk: f32 projections into a bf16 cache
        _append("append 16384 f32 to bf16", 16384, 32, 8, 64, 32, "f32", "bf16"),
        # a short conversation of one user, f32 cache: latency
        _attend("attend 1x77 f32", 1, 9, 3, 64, 16, "f32", "f32", 77, 77),
        # one long document
        _attend("attend 1x131072 bf16", 1, 32, 8, 128, 16, "bf16", "bf16", 131072, 131072),
        # a serving batch of unlike histories, one of them empty; f32 queries over a bf16 cache
        _attend("attend 64 ragged bf16", 64, 28, 4, 128, 16, "f32", "bf16", 0, 8191, lse=True),
        # as many key heads as query heads, f32 cache
        _attend("attend 16 f32", 16, 16, 16, 128, 32, "f32", "f32", 700, 2048),
        # a large batch of middling histories in the smallest cache
        _attend("attend 128 q8_0", 128, 9, 3, 64, 32, "f32", "q8_0", 1, 4096),
        # a layer's share of a decode step: the new rows into a Q8_0 cache and attention over it
        _attend("step 32 q8_0", 32, 28, 4, 128, 16, "f32", "q8_0", 1, 8000, op="step"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "step"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if op == "plan":
        mix = rng.choice(["decode", "mixed", "prompt"])
        c = _plan("", _log(rng, 1, 1024), page, _log(rng, 16, 512 if mix == "prompt" else 4096), mix)
    else:
        heads, kv = rng.choice([(9, 3), (28, 4), (32, 8), (16, 16), (8, 1), (12, 12), (24, 2)])
        dh = rng.choice([32, 64, 64, 96, 128, 128])
        if op == "append":
            tokens = _log(rng, 1, 16384)
            c = _append("", tokens, heads, kv, dh, page, rng.choice(["f32", "bf16", "f16"]),
                        rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.3, rng.randrange(0, 1 + tokens // 2))
            while _append_bytes(c) > 150e6:
                c["tokens"] = c["tokens"] // 2
                c["padded"] = min(c["padded"], c["tokens"] // 2)
        else:
            cache = "q8_0" if op == "step" else rng.choice(["f32", "bf16", "f16", "q8_0"])
            dtype = rng.choice(["f32", "f32", "bf16", "f16"])
            n = _log(rng, 1, 128)
            most = 500e6 / (n * kv * dh * 2 * SIZE[cache])
            hi = _log(rng, 1, max(1, int(min(131072, most))))
            lo = 1 if op == "step" else rng.choice([0, 1, hi // 2, hi])
            c = _attend("", n, heads, kv, dh, page, dtype, cache, min(lo, hi), hi, rng.random() < 0.3, op)
    del c["name"]
    return c


# ------------------------------------------------------------------ their inputs
def _ceil(a, b):
    return (a + b - 1) // b


def _rope_table(rows, dh):
    """cos and sin of pos * 10000^(-2i/dh) (64-bit angles), [rows, dh / 2, 2] f32."""
    inv = 10000.0 ** (-torch.arange(0, dh, 2, device=DEV, dtype=torch.float64) / dh)
    a = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _pools(case, n_pages, g):
    """Page pools [n_pages, kv, page, dh] (and Q8_0 scales [.., dh / 32]) full of what earlier requests left."""
    shape = (n_pages, case["kv"], case["page"], case["dh"])
    s = {}
    for w in "kv":
        if case["cache"] == "q8_0":
            s[w + "_pool"] = torch.randint(-127, 128, shape, device=DEV, generator=g, dtype=torch.int8)
            s[w + "_scale"] = (0.005 + 0.02 * torch.rand(shape[:3] + (shape[3] // 32,), device=DEV,
                                                         generator=g)).half()
        else:
            s[w + "_pool"] = torch.randn(shape, device=DEV, generator=g,
                                         dtype=torch.float32).to(DTYPES[case["cache"]])
            s[w + "_scale"] = None
    return s


def _new_rows(case, n, g):
    """The projections' output q | k | v, one row per token, and views of its parts."""
    H, KV, dh = case["heads"], case["kv"], case["dh"]
    qkv = torch.randn((n, (H + 2 * KV) * dh), device=DEV, generator=g).to(DTYPES[case["dtype"]])
    return {"q": qkv[:, :H * dh].view(n, H, dh), "k": qkv[:, H * dh:(H + KV) * dh].view(n, KV, dh),
            "v": qkv[:, (H + KV) * dh:].view(n, KV, dh),
            "q_out": torch.zeros((n, H, dh), device=DEV, dtype=qkv.dtype)}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ints = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), device=DEV, generator=g, dtype=torch.int32)  # noqa: E731
    s, page = {"case": case}, case["page"]
    if case["op"] == "plan":
        n = case["n"]
        if case["mix"] == "prompt":
            lens, add, most = ints(0, 0, n), ints(1, case["max_len"], n), case["max_len"]
        elif case["mix"] == "decode":
            lens, add, most = ints(0, case["max_len"], n), ints(1, 1, n), 1
        else:
            kind = ints(0, 9, n)
            most = max(1, case["max_len"] // 8)
            lens = ints(0, case["max_len"], n)
            add = torch.where(kind < 7, torch.ones_like(kind), torch.where(kind < 9, ints(1, most, n), 0 * kind))
        width = _ceil(case["max_len"] + most, page)
        n_pages = n * width
        perm = torch.randperm(n_pages, device=DEV, generator=g).int()
        held = _ceil(lens, page)
        first = held.cumsum(0) - held
        col = torch.arange(width, device=DEV)[None, :]
        table = torch.where(col < held[:, None], perm[(first[:, None] + col).clamp(max=n_pages - 1)], -1).int()
        used = held.sum()
        free = perm[(torch.arange(n_pages, device=DEV) + used) % n_pages]
        state = torch.zeros(4, device=DEV, dtype=torch.int32)
        state[0] = n_pages - used
        return s | {"lens": lens, "add": add.int(), "table": table.contiguous(), "free": free.contiguous(),
                    "state": state, "n_pages": n_pages, "n_tokens": n * most}
    if case["op"] == "append":
        n, live = case["tokens"], case["tokens"] - case["padded"]
        n_pages = _ceil(live, page) + 2          # the last page is a spare that no token is put into
        s |= _pools(case, n_pages, g) | _new_rows(case, n, g)
        slots = torch.full((n,), -1, device=DEV, dtype=torch.int64)
        slots[:live] = torch.randperm((n_pages - 1) * page, device=DEV, generator=g)[:live]
        s["slots"], s["positions"] = slots, ints(0, 4095, n)
        s["rope"] = _rope_table(4096, case["dh"])
        W = (case["heads"] + 2 * case["kv"]) * case["dh"]
        s["bias"] = torch.randn(W, device=DEV, generator=g) if case["bias"] else None
        return s
    n, hi = case["n"], case["hi"]
    width = _ceil(hi, page)
    lens = ints(case["lo"], hi, n)
    lens[-1] = hi                                # the longest history is there for certain,
    if case["lo"] == 0 and n > 1:
        lens[0] = 0                              # and an empty one where there may be some
    n_pages = n * width + 1                      # and a spare page
    s |= _pools(case, n_pages, g) | _new_rows(case, n, g)
    s["table"] = torch.randperm(n_pages - 1, device=DEV, generator=g).int().view(n, width).contiguous()
    s["lens"] = lens
    s["out"] = torch.zeros((n, case["heads"], case["dh"]), device=DEV, dtype=DTYPES[case["dtype"]])
    s["lse"] = torch.zeros((n, case["heads"]), device=DEV) if case["lse"] else None
    if case["op"] == "step":
        pos = lens - 1
        s["positions"] = pos
        s["slots"] = s["table"].gather(1, (pos // page)[:, None].long())[:, 0].long() * page + pos % page
        s["rope"], s["bias"] = _rope_table(hi, case["dh"]), None
    return s


# ------------------------------------------------------------------ the framework's calls
def _own_cache(s):
    from toy_b200 import paged
    if "cache" not in s:         # what a user's program makes once beside its pools
        s["cache"] = paged.PagedCache(s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"])
        s["workspace"] = paged.attend_workspace(s["k_pool"].device)
    return paged, s["cache"]


def _own_plan(s):
    from toy_b200 import paged
    p = paged.plan(s["lens"], s["add"], s["table"], s["free"], s["state"], page_size=s["case"]["page"],
                   n_pages=s["n_pages"], n_tokens=s["n_tokens"])
    return {"table": s["table"], "lens": p.lens, "state": p.state, "cu_tokens": p.cu_tokens, "slots": p.slots,
            "positions": p.positions, "requests": p.requests}


def _own_append(s):
    paged, cache = _own_cache(s)
    paged.append(cache, s["slots"], s["k"], s["v"], q=s["q"], q_out=s["q_out"], positions=s["positions"],
                 rope=s["rope"], bias=s["bias"])
    return {"q": s["q_out"], "k_pool": s["k_pool"][:-1], "v_pool": s["v_pool"][:-1]}


def _own_attend(s, q):
    paged, cache = _own_cache(s)
    paged.attend(cache, q, s["table"], s["lens"], out=s["out"], lse=s["lse"], workspace=s["workspace"])
    return [s["out"]] + ([s["lse"]] if s["lse"] is not None else [])


# ------------------------------------------------------------------ the plain forms
def _plain_plan(s):
    case, lens, add, free, state = s["case"], s["lens"], s["add"], s["free"], s["state"]
    page, cap = case["page"], s["n_tokens"]
    held, need = _ceil(lens, page), _ceil(lens + add, page)
    take = need - held
    cu_page = take.cumsum(0) - take
    total = add.sum()
    cu = torch.cat([torch.zeros_like(total)[None], add.cumsum(0)]).int()
    col = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    at = state[0] - 1 - (cu_page[:, None] + col - held[:, None])
    table = torch.where(fresh, free[at.clamp(0, free.numel() - 1).long()], s["table"])
    t = torch.arange(cap, device=DEV, dtype=torch.int32)
    req = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=lens.numel() - 1)
    live = t < total
    pos = lens[req] + (t - cu[req])
    slots = table[req, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    taken = take.sum()
    new_state = torch.stack([state[0] - taken, torch.zeros_like(total), total, taken]).int()
    return {"table": table, "lens": lens + add, "state": new_state, "cu_tokens": cu,
            "slots": torch.where(live, slots, -1), "positions": torch.where(live, pos, 0).int(),
            "requests": torch.where(live, req, -1).int()}


def _rotate(x, cs):
    """x [n, heads, dh] f32, cs [n, dh / 2, 2]: pairs (i, i + dh / 2) turned by their angle."""
    h = x.shape[-1] // 2
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * sn, a * sn + b * c], -1)


def _q8_0(x):
    """Blocks of 32: scale d = amax / 127 held in fp16, quants round-half-away(x / d)."""
    b = x.view(x.shape[:-1] + (x.shape[-1] // 32, 32))
    d = b.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=DEV)
    t = b * torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    w = t.trunc()
    w = torch.where((t - w).abs() >= 0.5, w + t.sign(), w)
    return w.to(torch.int8).view(x.shape), d[..., 0].half()


def _plain_append(s):
    case = s["case"]
    H, KV, dh, page = case["heads"], case["kv"], case["dh"], case["page"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["bias"] is not None:
        b = s["bias"]
        q, k, v = (q + b[:H * dh].view(H, dh), k + b[H * dh:(H + KV) * dh].view(KV, dh),
                   v + b[(H + KV) * dh:].view(KV, dh))
    cs = s["rope"][s["positions"].long()]
    q, k = _rotate(q, cs), _rotate(k, cs)
    spare = (s["k_pool"].shape[0] - 1) * page
    slot = torch.where(s["slots"] >= 0, s["slots"], spare)
    pg, off = slot // page, slot % page
    for w, x in (("k", k), ("v", v)):
        if case["cache"] == "q8_0":
            qx, dx = _q8_0(x)
            s[w + "_pool"][pg, :, off] = qx
            s[w + "_scale"][pg, :, off] = dx
        else:
            s[w + "_pool"][pg, :, off] = x.to(s[w + "_pool"].dtype)
    return {"q": q.to(s["q"].dtype), "k_pool": s["k_pool"][:-1], "v_pool": s["v_pool"][:-1]}


def _gather(s, w):
    """The requests' pages as f32 [n, kv, width * page, dh]."""
    t = s["table"].long()
    x = s[w + "_pool"][t].float()                                  # [n, width, kv, page, dh]
    if s[w + "_scale"] is not None:
        n, width, kv, page, dh = x.shape
        x = (x.view(n, width, kv, page, dh // 32, 32) * s[w + "_scale"][t].float()[..., None]).view(x.shape)
    return x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _plain_attend(s, q):
    case = s["case"]
    n, H, KV, dh = case["n"], case["heads"], case["kv"], case["dh"]
    k, v = _gather(s, "k"), _gather(s, "v")
    sc = torch.matmul(q.float().view(n, KV, H // KV, dh), k.transpose(2, 3)) * (1.0 / math.sqrt(dh))
    dead = (torch.arange(k.shape[2], device=DEV)[None, :] >= s["lens"][:, None])[:, None, None, :]
    sc = sc.masked_fill(dead, float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)     # an empty history: every weight is 0
    p = torch.exp(sc - m)
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(z > 0, z, torch.ones_like(z))
    out = [o.view(n, H, dh).to(q.dtype)]
    return out + ([(m + z.log()).view(n, H)] if case["lse"] else [])


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "plan":
            return _own_plan(state)
        if op == "append":
            return _own_append(state)
        if op == "attend":
            return _own_attend(state, state["q"])
        a = _own_append(state)
        return {"q": a["q"], "out": _own_attend(state, a["q"])}
    if op == "plan":
        return _plain_plan(state)
    if op == "append":
        return _plain_append(state)
    if op == "attend":
        return _plain_attend(state, state["q"])
    a = _plain_append(state)
    return {"q": a["q"], "out": _plain_attend(state, a["q"])}


# ------------------------------------------------------------------ what a pass cannot do without
def _append_bytes(c):
    """Live rows in, rotated q and the cache rows out; a padded row still has its q rotated."""
    live = c["tokens"] - c["padded"]
    H, KV, dh, e = c["heads"], c["kv"], c["dh"], SIZE[c["dtype"]]
    return (c["tokens"] * (2 * H * dh * e + 12 + 4 * dh) + live * 2 * KV * dh * (e + SIZE[c["cache"]])
            + (4 * (H + 2 * KV) * dh if c["bias"] else 0))


def work(case):
    if case["op"] == "plan":
        n = case["n"]
        if case["mix"] == "prompt":
            most, mean = case["max_len"], (1 + case["max_len"]) / 2
        elif case["mix"] == "decode":
            most, mean = 1, 1
        else:
            most = max(1, case["max_len"] // 8)
            mean = 0.7 + 0.2 * (1 + most) / 2
        # lens, add and the open page in; per new page one free entry in, one table entry out; per token slot,
        # position and request out; cu_tokens and lens out; the state in and out
        return {"bytes": n * (8 + 4) + n * mean / case["page"] * 8 + n * most * 16 + n * 8 + 36, "flops": 0}
    if case["op"] == "append":
        rows = case["tokens"] * (case["heads"] + case["kv"])
        return {"bytes": _append_bytes(case), "flops": 3.0 * rows * case["dh"]}
    H, KV, dh, n = case["heads"], case["kv"], case["dh"], case["n"]
    keys = case["hi"] + (n - 1) * (case["lo"] + case["hi"]) / 2     # expected: one longest, the rest uniform
    b = keys * KV * dh * 2 * SIZE[case["cache"]] + 2 * n * H * dh * SIZE[case["dtype"]]
    b += keys / case["page"] * 4 + 4 * n + (4 * n * H if case["lse"] else 0)
    f = 4.0 * keys * H * dh
    if case["op"] == "step":
        e = SIZE[case["dtype"]]
        b += n * ((H + 2 * KV) * dh * e + H * dh * e + 2 * KV * dh * SIZE["q8_0"] + 12 + 4 * dh)
        f += 3.0 * n * (H + KV) * dh
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------ from the definition, in 64 bits
def _exact_rotate(s, w, first, heads):
    dh = s["case"]["dh"]
    x = s[w].double()
    if s["bias"] is not None:
        x = x + s["bias"].double()[first * dh:(first + heads) * dh].view(heads, dh)
    if w == "v":
        return x
    ang = s["rope"].double()[s["positions"].long()]                 # the table is an input
    z = torch.complex(x[..., :dh // 2], x[..., dh // 2:]) * torch.complex(ang[..., 0], ang[..., 1])[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_attend(s, q, k_rows, v_rows):
    """q [n, H, dh]; k_rows(b), v_rows(b): request b's keys and values, [kv, len, dh], all 64-bit."""
    case = s["case"]
    H, KV, dh = case["heads"], case["kv"], case["dh"]
    out = torch.zeros((case["n"], H, dh), device=DEV, dtype=torch.float64)
    lse = torch.full((case["n"], H), float("-inf"), device=DEV, dtype=torch.float64)
    for b, length in enumerate(s["lens"].tolist()):
        if length == 0:
            continue
        k, v = k_rows(b, length), v_rows(b, length)
        for j in range(KV):
            rows = slice(j * (H // KV), (j + 1) * (H // KV))
            sc = (q[b, rows] @ k[j].T) / math.sqrt(dh)
            lse[b, rows] = torch.logsumexp(sc, -1)
            out[b, rows] = torch.softmax(sc, -1) @ v[j]
    return [out] + ([lse] if case["lse"] else [])


def _rows_of(s, w):
    case = s["case"]

    def rows(b, length):
        ids = s["table"][b, :_ceil(length, case["page"])].long()
        x = s[w + "_pool"][ids].double()
        if s[w + "_scale"] is not None:
            x = x * s[w + "_scale"][ids].double().repeat_interleave(32, -1)
        return x.permute(1, 0, 2, 3).reshape(case["kv"], -1, case["dh"])[:, :length]
    return rows


def _exact_q8(x):
    """The values that Q8_0 blocks of x stand for, of 32-bit x as the cache is given it: [.., dh] 64-bit."""
    b = x.float().unflatten(-1, (-1, 32))
    d = b.abs().max(-1, keepdim=True).values.div(torch.tensor(127.0, device=DEV))
    t = b * torch.nan_to_num(1.0 / d, posinf=0.0)
    qn = torch.sign(t) * torch.floor(t.double().abs() + 0.5)
    return (qn * d.half().double()).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None                              # whole numbers: the plain form's are the definition's
    H, KV = case["heads"], case["kv"]
    if case["op"] == "append":
        put = {"q": _exact_rotate(s, "q", 0, H)}
        live = s["slots"] >= 0
        pg, off = s["slots"][live] // case["page"], s["slots"][live] % case["page"]
        for w, first in (("k", H), ("v", H + KV)):
            pool = s[w + "_pool"].double()
            pool[pg, :, off] = _exact_rotate(s, w, first, KV)[live]
            put[w + "_pool"] = pool[:-1]
        return put
    if case["op"] == "attend":
        return _exact_attend(s, s["q"].double(), _rows_of(s, "k"), _rows_of(s, "v"))
    # step: the rotated new rows (rounded to 32 bits, the quantiser's input) as Q8_0 stands at each request's end
    q = _exact_rotate(s, "q", 0, H)
    cs = s["rope"][s["positions"].long()][:, None]
    h = case["dh"] // 2
    x = s["k"].float()
    turned = torch.cat([x[..., :h] * cs[..., 0] - x[..., h:] * cs[..., 1],
                        x[..., :h] * cs[..., 1] + x[..., h:] * cs[..., 0]], -1)
    new = {"k": _exact_q8(turned), "v": _exact_q8(s["v"])}

    def with_new(w):
        rows = _rows_of(s, w)

        def f(b, length):
            x = rows(b, length)
            x[:, length - 1] = new[w][b]
            return x
        return f
    qr = q.to(DTYPES[case["dtype"]]).double()    # attention reads the rotated q as append wrote it
    return {"q": q, "out": _exact_attend(s, qr, with_new("k"), with_new("v"))}
