"""Operators of a fine-tune step outside its matrix products, measured.

  score    log probabilities of given tokens, entropy and top alternatives, from logits
  policy   the same, and the gradient back to the logits
  route    tokens sorted by expert, their rows to the experts and back with weights
  moe      the same with the gradients of both ways
  adamw    one AdamW step over many tensors, moments in 32 or in 8 bits

`run` computes them from elementary torch operations, or (own = True) with
toy_b200.logprobs, toy_b200.experts and toy_b200.multi_adamw. `exact` computes
them from their definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256             # values that share a scale in 8-bit moments
INF = float("inf")


# ------------------------------------------------------------------ the cases
def _score(name, rows, vocab, dtype, scale=1.0, entropy=False, top=0, masked=False, pad=0, op="score"):
    return {"name": name, "op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "scale": scale, "entropy": entropy,
            "top": top, "masked": masked, "pad": pad}


def _route(name, tokens, experts, used, d, dtype, skew=0.0, dropped=0, op="route"):
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "used": used, "d": d, "dtype": dtype,
            "skew": skew, "dropped": dropped}


def _adamw(name, layers, d, ff, kv, vocab, rank, bits, ptype, gtype, ctype):
    """rank > 0: adapters of that rank on q, k, v, o alone. ctype: a 16-bit copy of the weights, or ""."""
    return {"name": name, "op": "adamw", "layers": layers, "d": d, "ff": ff, "kv": kv, "vocab": vocab, "rank": rank,
            "bits": bits, "ptype": ptype, "gtype": gtype, "ctype": ctype}


def listed():
    return [
        # the chosen token and five alternatives of one sequence's decode step
        _score("score 1 f32 top 5", 1, 49152, "f32", top=5),
        # a decode batch, at a sampling temperature
        _score("score 16 f32 top 20", 16, 128256, "f32", scale=1.25, entropy=True, top=20),
        # a batch of answers scored under a frozen reference model
        _score("score 4096 bf16", 4096, 152064, "bf16"),
        # constrained decoding: most of the vocabulary masked, rows of an odd length in a wider buffer
        _score("score 509 f16 masked", 509, 50303, "f16", entropy=True, top=32, masked=True, pad=6),
        # a policy-gradient step with an entropy bonus over padded sequences
        _score("policy 4096 bf16", 4096, 128256, "bf16", entropy=True, op="policy"),
        # a decode batch of a 64-expert model
        _route("route 16 f32", 16, 64, 8, 2048, "f32"),
        # a training batch's forward through it
        _route("route 4096 bf16", 4096, 64, 8, 2048, "bf16"),
        # few large experts, most tokens choosing the same ones, padding tokens that go nowhere, an odd width
        _route("moe 2039 f16 skewed", 2039, 8, 2, 1000, "f16", skew=2.0, dropped=300, op="moe"),
        # forward and backward of a training batch
        _route("moe 8192 f32", 8192, 128, 4, 2048, "f32", op="moe"),
        # adapters of rank 8: many small tensors
        _adamw("adamw adapters 8-bit", 30, 576, 0, 192, 0, 8, 8, "f32", "f32", ""),
        # a whole 135M-parameter model, f32 moments
        _adamw("adamw 135M f32", 30, 576, 1536, 192, 49152, 0, 32, "f32", "f32", ""),
        # the same with 8-bit moments, 16-bit gradients and a 16-bit copy of the weights
        _adamw("adamw 135M 8-bit", 30, 576, 1536, 192, 49152, 0, 8, "f32", "bf16", "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["score", "policy", "route", "moe", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("score", "policy"):
        vocab = rng.choice([_log(rng, 256, 152064), 49152, 50304, 128256, 152064])
        cost = vocab * SIZE[dtype] * (3 if op == "policy" else 1)
        c = _score("", _log(rng, 1, max(1, min(8192, int(2.5e9 / cost)))), vocab, dtype,
                   rng.choice([1.0, 1.0, 0.7, 1.4]), rng.random() < 0.6, rng.choice([0, 0, 1, 5, 20, 32]),
                   rng.random() < 0.3, rng.choice([0, 0, 1, 8]), op)
    elif op in ("route", "moe"):
        experts = rng.choice([4, 8, 16, 64, 128, 160])
        used = rng.randrange(1, min(8, experts) + 1)
        d = rng.choice([_log(rng, 64, 4096), 576, 1024, 2048, 3584])
        tokens = _log(rng, 1, max(1, min(32768, int(5e8 / (used * d * SIZE[dtype])))))
        c = _route("", tokens, experts, used, d, dtype, rng.choice([0.0, 0.0, 1.0, 3.0]),
                   rng.choice([0, 0, rng.randrange(tokens)]), op)
    else:
        bits = rng.choice([8, 8, 32])
        ptype = rng.choice(["f32", "f32", "bf16"])
        d, kv = rng.choice([(576, 192), (256, 64), (1000, 200), (2048, 512)])
        rank = rng.choice([0, 0, 8, 16])
        layers = _log(rng, 1, 30 if d < 2000 else 3)
        c = _adamw("", layers, d, 0 if rank else rng.choice([2, 4]) * d, kv, 0 if rank else _log(rng, 128, 16384),
                   rank, bits, ptype, rng.choice(["f32", "bf16"]), rng.choice(["", "bf16"]) if ptype == "f32" else "")
        while work(c)["bytes"] > 3e9:
            c["layers"] //= 2
    del c["name"]
    return c


def _shapes(c):
    """The tensors of an AdamW step: rank-r pairs on q, k, v, o of every layer, or every weight of the model."""
    d, ff, kv, r = c["d"], c["ff"], c["kv"], c["rank"]
    if r:
        return [s for _ in range(c["layers"]) for w in (d, kv, kv, d) for s in ((r, d), (w, r))]
    layer = [(d,), (d, d), (kv, d), (kv, d), (d, d), (d,), (ff, d), (ff, d), (d, ff)]
    return [(c["vocab"], d)] + layer * c["layers"] + [(d,)]


# ------------------------------------------------------------------ their inputs
def _room(shapes, dtype):
    """Zeroed tensors of these shapes that start at multiples of BLOCK values of one buffer, and the buffer."""
    sizes = [math.prod(sh) for sh in shapes]
    whole = torch.zeros(sum(n + -n % BLOCK for n in sizes), device=DEV, dtype=dtype)
    out, at = [], 0
    for sh, n in zip(shapes, sizes):
        out.append(whole[at:at + n].view(sh))
        at += n + -n % BLOCK
    return out, whole


def _logits(c, g):
    """Logits of a trained model: a bulk, and on each row a few words that stand out; -inf where masked."""
    n, V = c["rows"], c["vocab"]
    buf = torch.empty((n, V + c["pad"]), device=DEV, dtype=DTYPES[c["dtype"]])
    x = buf[:, :V]
    step = max(1, (1 << 28) // V)
    for a in range(0, n, step):
        b = min(n, a + step)
        z = torch.randn((b - a, V), device=DEV, generator=g) * 2.0
        at = torch.randint(0, V, (b - a, 8), device=DEV, generator=g)
        z.scatter_add_(1, at, 4.0 + 6.0 * torch.rand((b - a, 8), device=DEV, generator=g))
        if c["masked"]:
            z.masked_fill_(torch.rand((b - a, V), device=DEV, generator=g) < 0.7, -INF)
            z[:, : min(V, 40)] = torch.randn((b - a, min(V, 40)), device=DEV, generator=g)    # some words stay open
        x[a:b] = z.to(x.dtype)
    return x


def _choices(c, g):
    """ids [tokens, used] of distinct experts, the first ones favoured where skewed; -1 rows for padding tokens."""
    T, E = c["tokens"], c["experts"]
    bias = -c["skew"] * torch.arange(E, device=DEV, dtype=torch.float32).log1p()
    s = torch.randn((T, E), device=DEV, generator=g) + bias
    w, ids = torch.softmax(s, -1).sort(-1, descending=True)
    ids, w = ids[:, :c["used"]].int().contiguous(), w[:, :c["used"]].contiguous()
    if c["dropped"]:
        gone = torch.randperm(T, device=DEV, generator=g)[:c["dropped"]]
        ids[gone] = -1
    return ids, w


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s, op = {"case": case}, case["op"]
    rnd = lambda *shape: torch.randn(shape, device=DEV, generator=g)  # noqa: E731
    if op in ("score", "policy"):
        n, V = case["rows"], case["vocab"]
        s["logits"] = _logits(case, g)
        tokens = torch.randint(0, V, (n,), device=DEV, generator=g)
        if case["masked"]:
            tokens = tokens % min(V, 40)               # a word that is open
        if op == "policy":
            tokens = torch.where(torch.rand(n, device=DEV, generator=g) < 0.1, -1, tokens)      # padding
            s["g_logprob"] = torch.where(tokens >= 0, rnd(n), 0.0)
            s["g_entropy"] = torch.where(tokens >= 0, -0.01 * torch.ones(n, device=DEV), 0.0)
            s["g_top"] = 0.1 * rnd(n, case["top"])
        s["tokens"] = tokens
        return s
    if op in ("route", "moe"):
        T, K, d = case["tokens"], case["used"], case["d"]
        t = DTYPES[case["dtype"]]
        s["ids"], s["w"] = _choices(case, g)
        s["x"], s["z"], s["res"] = rnd(T, d).to(t), rnd(T * K, d).to(t), rnd(T, d).to(t)
        s["xs"] = torch.zeros((T * K, d), device=DEV, dtype=t)      # rows past the last expert's stay as they are
        if op == "moe":
            s["dy"], s["dxs"] = rnd(T, d).to(t), rnd(T * K, d).to(t)
            s["dz"] = torch.zeros((T * K, d), device=DEV, dtype=t)
        return s
    shapes, t = _shapes(case), DTYPES[case["ptype"]]
    flat = [(math.prod(sh),) for sh in shapes]
    s["p"], s["p_all"] = _room(shapes, t)
    s["ms"], s["ms_all"] = _room(shapes, torch.float32)        # the moments as values
    s["vs"], s["vs_all"] = _room(shapes, torch.float32)
    s["copy"], s["copy_all"] = _room(shapes, DTYPES[case["ctype"]]) if case["ctype"] else (None, None)
    s["g"] = [(1e-3 * torch.rand((), device=DEV, generator=g) * rnd(*sh)).to(DTYPES[case["gtype"]]) for sh in shapes]
    s["m_scale"] = s["v_scale"] = None
    if case["bits"] == 8:
        s["m"], s["v"] = (_room(flat, torch.float8_e4m3fn)[0] for _ in "mv")
        s["m_scale"], s["v_scale"] = (_room([(-(-n // BLOCK),) for n, in flat], torch.float32)[0] for _ in "mv")
    else:
        s["m"], s["v"] = s["ms"], s["vs"]
    for i, sh in enumerate(shapes):
        s["p"][i].copy_(0.02 * rnd(*sh))
        if s["copy"]:
            s["copy"][i].copy_(s["p"][i])
        m, v = 3e-4 * rnd(*sh), (6e-4 * rnd(*sh)) ** 2         # step 100 of a run: moments of the gradients' size
        if case["bits"] == 8:
            _put(s, "m", i, _hold(m.double().flatten()))
            _put(s, "v", i, _hold(v.double().flatten().sqrt(), floor=True))
        else:
            s["m"][i].copy_(m)
            s["v"][i].copy_(v)
    s["hp"] = torch.tensor([3e-4, 0.9, 0.999, 1e-8, 0.01, 1 / (1 - 0.9 ** 100), 1 / (1 - 0.999 ** 100)], device=DEV)
    s["clip"] = torch.tensor(0.8, device=DEV)          # the gradients' factor, as a clipping of their norm gives it
    return s


def _weights(s):
    return {"weights": s["p_all"], "m": s["ms_all"], "v": s["vs_all"]} | \
        ({"copies": s["copy_all"]} if s["copy"] else {})


# ------------------------------------------------------------------ the framework's calls
def _own_score(s):
    from toy_b200 import logprobs
    c = s["case"]
    return logprobs.token_logprobs(s["logits"], s["tokens"], scale=c["scale"], entropy=c["entropy"], top=c["top"])


def _own_policy(s):
    from toy_b200 import logprobs
    c, r = s["case"], _own_score(s)
    d = logprobs.token_logprobs_grad(s["logits"], s["tokens"], r, s["g_logprob"],
                                     grad_entropy=s["g_entropy"] if c["entropy"] else None,
                                     grad_top=s["g_top"] if c["top"] else None, scale=c["scale"])
    return r, d


def _own_experts(s):
    from toy_b200 import experts
    c = s["case"]
    r = experts.sort(s["ids"], c["experts"])
    o = {"offsets": r.offsets, "order": r.order, "pos": r.pos, "xs": experts.dispatch(s["x"], r, out=s["xs"]),
         "y": experts.combine(s["z"], r, s["w"], residual=s["res"])}
    if c["op"] == "moe":
        o["dz"], o["dw"] = experts.combine_grad(s["dy"], s["z"], r, s["w"], out=s["dz"])
        o["dx"] = experts.dispatch_grad(s["dxs"], r)
    return o


def _own_adamw(s):
    from toy_b200.multi_adamw import MultiAdamW
    c = s["case"]
    if "opt" not in s:           # what a user's program makes once beside its weights
        s["opt"] = MultiAdamW(s["p"], bits=c["bits"], copies=s["copy"],
                              state=(s["m"], s["v"], s["m_scale"], s["v_scale"]))
    s["opt"].step(s["g"], s["hp"], grad_scale=s["clip"])
    if c["bits"] == 8:           # (moments held in 32 bits are the values themselves)
        s["opt"].moments(out=(s["ms"], s["vs"]))
    return _weights(s)


# ------------------------------------------------------------------ the plain forms
def _keys(x):
    """Whole numbers in the order of (value, lower index first) of x [rows, vocab] f32."""
    b = (x + 0.0).view(torch.int32)
    b = (b ^ ((b >> 31) & 0x7fffffff)).long()
    return (b << 32) | (0x7fffffff - torch.arange(x.shape[1], device=DEV))


def _plain_score(s):
    c, x = s["case"], s["logits"].float()
    z = x * c["scale"]
    m = z.amax(-1, keepdim=True)
    t = z - m
    e = t.exp()
    z_sum = e.sum(-1, keepdim=True)
    ln = z_sum.log()
    live = s["tokens"] >= 0
    lp = torch.where(live, t.gather(1, s["tokens"].clamp(min=0)[:, None])[:, 0] - ln[:, 0], 0.0)
    o = {"logprob": lp, "entropy": None, "top_ids": None, "top_logprobs": None}
    if c["entropy"]:
        o["entropy"] = ln[:, 0] - (e * t.clamp(min=-1e4)).sum(-1) / z_sum[:, 0]
    if c["top"]:
        ids = _keys(x).topk(c["top"], dim=-1).indices          # (keys are all unlike)
        o["top_ids"], o["top_logprobs"] = ids, t.gather(1, ids) - ln
    return o, t - ln


def _plain_policy(s):
    c = s["case"]
    o, lp = _plain_score(s)
    p = lp.exp()
    a = s["g_logprob"]
    if c["top"]:
        a = a + s["g_top"].sum(-1)
    d = -a[:, None] * p
    live = s["tokens"] >= 0
    d.scatter_add_(1, s["tokens"].clamp(min=0)[:, None], torch.where(live, s["g_logprob"], 0.0)[:, None])
    if c["top"]:
        d.scatter_add_(1, o["top_ids"], s["g_top"])
    if c["entropy"]:
        d -= s["g_entropy"][:, None] * p * (lp.clamp(min=-1e4) + o["entropy"][:, None])
    return o, (d * c["scale"]).to(s["logits"].dtype)


def _plain_experts(s):
    c = s["case"]
    T, K, E = c["tokens"], c["used"], c["experts"]
    ids = s["ids"].flatten().long()
    live = ids >= 0
    counts = (ids[:, None] == torch.arange(E, device=DEV)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    order = torch.where(live, ids, E).sort(stable=True).indices
    rank = torch.arange(T * K, device=DEV)
    pos = torch.empty_like(rank).scatter_(0, order, rank)
    n = offsets[-1]
    pos = torch.where(live, pos, -1).view(T, K)
    kept = (rank < n)[:, None]
    xs = torch.where(kept, s["x"][order // K], s["xs"])
    at, on = pos.clamp(min=0), (pos >= 0)
    w = torch.where(on, s["w"], 0.0)
    z = s["z"].float()
    y = s["res"].float()
    for k in range(K):
        y = y + w[:, k, None] * z[at[:, k]]
    o = {"offsets": offsets, "order": torch.where(rank < n, order, -1).int(), "pos": pos.int(), "xs": xs,
         "y": y.to(s["x"].dtype)}
    if c["op"] == "moe":
        dy = s["dy"].float()
        dys = dy[order // K]
        o["dz"] = torch.where(kept, dys * w.flatten()[order][:, None], s["dz"].float()).to(s["x"].dtype)
        dw = torch.where(kept[:, 0], (dys * z).sum(-1), 0.0)
        o["dw"] = torch.zeros(T * K, device=DEV).scatter_(0, order, dw).view(T, K)
        dx = torch.zeros_like(dy)
        for k in range(K):
            dx = dx + torch.where(on[:, k, None], s["dxs"][at[:, k]].float(), 0.0)
        o["dx"] = dx.to(s["x"].dtype)
    return o


def _blocks(x):
    """x [n] in rows of BLOCK, the last one filled up with zeros."""
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _hold(x, floor=False):
    """x [n] f64 as e4m3 codes (nearest, ties to even) and a power-of-two scale per block, the smallest one of at least
    2^-100 that brings the block within 448. floor: a positive value keeps at least the smallest code. (In 64 bits: 32
    would put values next to a border between two codes on either side.)"""
    b = _blocks(x)
    f, e = torch.frexp(b.abs().amax(-1, keepdim=True) / 448.0)
    scale = torch.ldexp(torch.ones_like(f), torch.where(f == 0.5, e - 1, e).clamp(min=-100))
    t = b / scale
    magic = torch.ldexp(torch.full_like(t, 1.5), torch.frexp(t.abs().clamp(min=2.0 ** -6)).exponent + 48)
    t = (t + magic) - magic                                     # three bits behind the leading one stay
    if floor:
        t = torch.where((b > 0) & (t == 0), 2.0 ** -9, t)
    return t.flatten()[:x.numel()].float().to(torch.float8_e4m3fn), scale[:, 0].float()


def _put(s, name, i, held):
    s[name][i].copy_(held[0])
    s[name + "_scale"][i].copy_(held[1])


def _held(q, scale):
    return (_blocks(q.float()) * scale[:, None]).flatten()[:q.numel()]


def _plain_adamw(s):
    c = s["case"]
    lr, b1, b2, eps, wd, b1h, b2h = s["hp"]
    keep, root = 1.0 - lr * wd, b2h.sqrt()
    eight = c["bits"] == 8
    for i, p in enumerate(s["p"]):
        g = s["g"][i].float().flatten() * s["clip"]
        if eight:
            wide = s["g"][i].double().flatten() * s["clip"].double()
            m = _held(s["m"][i], s["m_scale"][i]).double()
            r = _held(s["v"][i], s["v_scale"][i]).double()
            m64 = m * b1.double() + wide * (1.0 - b1.double())
            r64 = (r * r * b2.double() + wide * wide * (1.0 - b2.double())).sqrt()
            m, r = m64.float(), r64.float()
        else:
            m = s["m"][i].flatten() * b1 + g * (1.0 - b1)
            v = s["v"][i].flatten() * b2 + g * g * (1.0 - b2)
            r = v.sqrt()
        w = p.float().flatten() * keep - lr * (m * b1h) / (r * root + eps)
        p.copy_(w.view(p.shape))
        if s["copy"]:
            s["copy"][i].copy_(p)
        if eight:
            _put(s, "m", i, _hold(m64))
            _put(s, "v", i, _hold(r64, floor=True))
            m = _held(s["m"][i], s["m_scale"][i])
            r = _held(s["v"][i], s["v_scale"][i])
            v = r * r
        s["ms"][i].copy_(m.view(p.shape))
        s["vs"][i].copy_(v.view(p.shape))
    return _weights(s)


def _score_outputs(c, o):
    return [o["logprob"]] + ([o["entropy"]] if c["entropy"] else []) + \
        ([o["top_ids"].long(), o["top_logprobs"]] if c["top"] else [])


def run(state):
    c = state["case"]
    if c["op"] == "score":
        return _score_outputs(c, _own_score(state)._asdict() if own else _plain_score(state)[0])
    if c["op"] == "policy":
        o, d = _own_policy(state) if own else _plain_policy(state)
        return _score_outputs(c, o._asdict() if own else o) + [d]
    if c["op"] == "adamw":
        return _own_adamw(state) if own else _plain_adamw(state)
    return _own_experts(state) if own else _plain_experts(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] in ("score", "policy"):
        n, V, e = c["rows"], c["vocab"], SIZE[c["dtype"]]
        b = n * (V * e + 8 + 4 + (4 if c["entropy"] else 0) + 12 * c["top"])
        f = n * V * (7.0 if c["entropy"] else 4.0)
        if c["op"] == "policy":      # the logits cannot be kept on the chip: read again
            b += n * (2 * V * e + 8 + 4 * c["top"])
            f += n * V * (9.0 if c["entropy"] else 5.0)
        return {"bytes": b, "flops": f}
    if c["op"] in ("route", "moe"):
        n, K, e = c["tokens"], c["used"], SIZE[c["dtype"]]
        row, S = c["d"] * e, (c["tokens"] - c["dropped"]) * c["used"]
        b = n * K * 4 * 4 + 4 * c["experts"] + (n + S) * row + (S + 2 * n) * row
        f = 2.0 * S * c["d"]
        if c["op"] == "moe":
            b += (n + 2 * S) * row + n * K * 4 + (S + n) * row
            f += 4.0 * S * c["d"]
        return {"bytes": b, "flops": f}
    n = sum(math.prod(s) for s in _shapes(c))
    held = 2 * (1 + 4 / BLOCK) if c["bits"] == 8 else 8
    b = n * (2 * SIZE[c["ptype"]] + SIZE[c["gtype"]] + 2 * held + (2 if c["ctype"] else 0))
    if c["bits"] == 8:
        b += n * 8                   # the values that the new moments stand for
    return {"bytes": b, "flops": 16.0 * n}


# ------------------------------------------------------------------ from the definition, in 64 bits
def _exact_score(s):
    c, n = s["case"], s["case"]["rows"]
    lp, ent, top, dx = [], [], [], []
    step = max(1, (1 << 27) // c["vocab"])
    for a in range(0, n, step):
        rows = slice(a, min(n, a + step))
        z = s["logits"][rows].double() * c["scale"]
        logp = torch.log_softmax(z, -1)
        p = logp.exp()
        tok = s["tokens"][rows]
        lp.append(torch.where(tok < 0, 0.0, logp.gather(1, tok.clamp(min=0)[:, None])[:, 0]))
        h = -torch.special.xlogy(p, p).sum(-1)
        ent.append(h)
        if c["top"]:
            top.append(logp.sort(dim=-1, descending=True, stable=True))
            top[-1] = (top[-1].values[:, :c["top"]].clone(), top[-1].indices[:, :c["top"]].clone())
        if c["op"] == "policy":
            d = torch.zeros_like(p)
            for i in range(c["top"]):
                gi = s["g_top"][rows, i].double()[:, None]
                d.sub_(gi * p).scatter_add_(1, top[-1][1][:, i:i + 1], gi)
            gl = s["g_logprob"][rows].double()[:, None]
            d.sub_(gl * p).scatter_add_(1, tok.clamp(min=0)[:, None], torch.where(tok[:, None] < 0, 0.0, gl))
            if c["entropy"]:
                d -= s["g_entropy"][rows].double()[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
            dx.append(d * c["scale"])
    o = [torch.cat(lp)] + ([torch.cat(ent)] if c["entropy"] else [])
    if c["top"]:
        o += [None, torch.cat([t[0] for t in top])]
    return o + ([torch.cat(dx)] if dx else [])


def _exact_experts(s):
    c = s["case"]
    T, K, d = c["tokens"], c["used"], c["d"]
    ids = s["ids"].flatten()
    slots = torch.cat([(ids == e).nonzero()[:, 0] for e in range(c["experts"])])      # slots in their experts' order
    tok, wt = slots // K, s["w"].double().flatten()[slots]
    n = slots.numel()
    y = s["res"].double()
    y.index_add_(0, tok, s["z"][:n].double() * wt[:, None])
    o = {"offsets": None, "order": None, "pos": None, "xs": s["xs"].double(), "y": y}
    o["xs"][:n] = s["x"].double()[tok]
    if c["op"] == "moe":
        dy = s["dy"].double()[tok]
        o["dz"] = s["dz"].double()
        o["dz"][:n] = dy * wt[:, None]
        o["dw"] = torch.zeros(T * K, device=DEV, dtype=torch.float64)
        o["dw"][slots] = torch.einsum("nd,nd->n", dy, s["z"][:n].double())
        o["dw"] = o["dw"].view(T, K)
        o["dx"] = torch.zeros((T, d), device=DEV, dtype=torch.float64).index_add_(0, tok, s["dxs"][:n].double())
    return o


def _exact_e4m3(x, floor):
    """The value that each of x [n] f64 is held as: 4 significant bits of it, no finer than 2^-9 of its block's scale
    and, where floor is set and it is positive, no less than that."""
    pad = -x.numel() % BLOCK
    b = torch.cat([x, x.new_zeros(pad)]).unflatten(0, (-1, BLOCK))
    exponent = torch.ceil(torch.log2(b.abs().max(-1, keepdim=True).values / 448.0)).clamp(min=-100.0)
    exponent = torch.where(b.abs().max(-1, keepdim=True).values > 448.0 * torch.exp2(exponent), exponent + 1, exponent)
    fine = torch.exp2(exponent - 9)
    step = torch.maximum(torch.exp2(torch.floor(torch.log2(b.abs().clamp(min=1e-300))) - 3), fine)
    q = torch.round(b / step) * step
    if floor:
        q = torch.where((b > 0) & (q == 0), fine, q)
    return q.flatten()[:x.numel()]


def _exact_adamw(s):
    lr, b1, b2, eps, wd, b1h, b2h = s["hp"].double().tolist()
    o = {k: torch.zeros_like(x, dtype=torch.float64) for k, x in _weights(s).items()}
    at = 0
    for i, p in enumerate(s["p"]):
        n = p.numel()
        g = s["g"][i].double().flatten() * s["clip"].double()
        m, v = s["m"][i].double().flatten(), s["v"][i].double().flatten()
        if s["m_scale"] is not None:
            block = torch.arange(n, device=DEV) // BLOCK
            m, v = m * s["m_scale"][i].double()[block], (v * s["v_scale"][i].double()[block]) ** 2
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        o["weights"][at:at + n] = (1 - lr * wd) * p.double().flatten() - lr * b1h * m / (torch.sqrt(b2h * v) + eps)
        if s["m_scale"] is not None:
            m, v = _exact_e4m3(m, False), _exact_e4m3(torch.sqrt(v), True) ** 2
        o["m"][at:at + n], o["v"][at:at + n] = m, v
        at += n + -n % BLOCK
    if s["copy"]:
        o["copies"] = o["weights"]
    return o


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("score", "policy"):
        return _exact_score(s)
    return _exact_adamw(s) if case["op"] == "adamw" else _exact_experts(s)
