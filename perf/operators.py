"""Cases of the device operators over the INT8 cache: rotary append, tree attention, eviction, token picking.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, 64 where angles and quantization
borders need them), or with `own` set calls this package's operators the way a user's decode loop does.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    pkg = os.path.join(os.getcwd(), "qx-mini-c_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import qxops
    return qxops


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence, the drafting model's own step: latency
        {"name": "rope one token", "op": "rope", "seqs": 1, "nodes": 1, "ragged": False, "q_heads": 32, "kv_heads": 4,
         "head_dim": 128, "rotary": 128, "interleaved": False, "far": 4096, "type": "bf16"},
        # 64 sequences verify trees of up to 16 nodes, positions scaled for long contexts
        {"name": "rope trees", "op": "rope", "seqs": 64, "nodes": 16, "ragged": True, "q_heads": 32, "kv_heads": 4,
         "head_dim": 128, "rotary": 128, "interleaved": False, "far": 65536, "type": "f32"},
        # a prompt chunk, half of each head rotated in interleaved pairs
        {"name": "rope prompt partial", "op": "rope", "seqs": 1, "nodes": 4096, "ragged": False, "q_heads": 32,
         "kv_heads": 4, "head_dim": 128, "rotary": 64, "interleaved": True, "far": 1000000, "type": "f16"},
        # one drafted token of one sequence on a short context: latency
        {"name": "tree one node", "op": "tree", "seqs": 1, "nodes": 1, "ragged": False, "ctx": 513, "q_heads": 32,
         "kv_heads": 4, "head_dim": 128, "chain": True, "mass": False, "type": "bf16"},
        # one sequence, a tree of 13 nodes on a long context, in the engine's activation type
        {"name": "tree long context", "op": "tree", "seqs": 1, "nodes": 13, "ragged": False, "ctx": 32768, "q_heads": 32,
         "kv_heads": 4, "head_dim": 128, "chain": False, "mass": False, "type": "f32"},
        # single-token decode of 64 ragged sequences that collects the weights eviction goes by
        {"name": "tree decode mass", "op": "tree", "seqs": 64, "nodes": 1, "ragged": True, "ctx": 4096, "q_heads": 32,
         "kv_heads": 4, "head_dim": 128, "chain": True, "mass": True, "type": "bf16"},
        # 64 sequences verify trees of 16 nodes at 4096 positions: the largest
        {"name": "tree batch", "op": "tree", "seqs": 64, "nodes": 16, "ragged": False, "ctx": 4096, "q_heads": 32,
         "kv_heads": 4, "head_dim": 128, "chain": False, "mass": False, "type": "bf16"},
        # one layer of one short sequence
        {"name": "evict one layer", "op": "evict", "layers": 1, "seqs": 1, "len": 1025, "budget": 512, "sink": 4,
         "recent": 64, "kv": 512},
        # all layers of eight ragged sequences at the engine's full context
        {"name": "evict all layers", "op": "evict", "layers": 48, "seqs": 8, "len": 4096, "budget": 2048, "sink": 4,
         "recent": 256, "kv": 512},
        # the pick of one sequence's next token over the engine's vocabulary
        {"name": "pick one row", "op": "pick", "rows": 1, "vocab": 151936, "history": 700, "biases": 8, "grammar": True,
         "type": "f32"},
        # 16 trees of 16 nodes verified at once
        {"name": "pick trees", "op": "pick", "rows": 256, "vocab": 151936, "history": 4096, "biases": 64,
         "grammar": True, "type": "f32"},
        # 64 sequences, a vocabulary of odd size, half precision logits, no grammar
        {"name": "pick odd vocabulary", "op": "pick", "rows": 64, "vocab": 50257, "history": 1000, "biases": 0,
         "grammar": False, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "tree", "tree", "evict", "pick"])
    kind = rng.choice(["f32", "f16", "bf16"])
    heads = rng.choice([(32, 4), (8, 2), (16, 16), (12, 4), (5, 1), (64, 8)])
    dim = rng.choice([64, 128, 128])
    if op == "rope":
        seqs = _log(rng, 1, 64)
        nodes = _log(rng, 1, 4096 // seqs)
        return {"op": "rope", "seqs": seqs, "nodes": nodes, "ragged": rng.random() < 0.5, "q_heads": heads[0],
                "kv_heads": heads[1], "head_dim": dim, "rotary": rng.choice([dim, dim // 2, 48, 2]),
                "interleaved": rng.random() < 0.5, "far": _log(rng, 1000, 1000000), "type": kind}
    if op == "tree":
        seqs = _log(rng, 1, 64)
        ctx = _log(rng, 1, 32768)
        nodes = _log(rng, 1, 64)
        while seqs * nodes * heads[0] * (ctx + nodes) > 1 << 27 or seqs * ctx > 1 << 18:
            if seqs > 1:
                seqs = (seqs + 1) // 2
            elif nodes > 1:
                nodes = (nodes + 1) // 2
            else:
                ctx //= 2
        return {"op": "tree", "seqs": seqs, "nodes": nodes, "ragged": rng.random() < 0.6, "ctx": ctx,
                "q_heads": heads[0], "kv_heads": heads[1], "head_dim": dim, "chain": rng.random() < 0.4,
                "mass": rng.random() < 0.3, "type": kind}
    if op == "evict":
        layers = _log(rng, 1, 48)
        seqs = _log(rng, 1, 16)
        length = _log(rng, 16, 8192)
        while layers * seqs * length > 48 * 8 * 4096:
            seqs = max(1, seqs // 2)
            length = length // 2 if seqs == 1 else length
        budget = rng.randint(8, length)
        sink = rng.randint(0, min(8, budget // 2))
        return {"op": "evict", "layers": layers, "seqs": seqs, "len": length, "budget": budget, "sink": sink,
                "recent": rng.randint(0, (budget - sink) // 2), "kv": rng.choice([64, 128, 512, 1024])}
    vocab = _log(rng, 1000, 151936)
    rows = _log(rng, 1, 256)
    return {"op": "pick", "rows": rows, "vocab": vocab, "history": _log(rng, 1, 8192), "biases": rng.choice([0, 1, 40, 300]),
            "grammar": rng.random() < 0.5, "type": kind}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _counts(case, g):
    """Nodes of each sequence: all of them, or a ragged batch whose shortest may be empty."""
    s, n = case["seqs"], case["nodes"]
    if not case["ragged"]:
        return torch.full((s,), n, dtype=torch.int32, device=DEV)
    return torch.randint(0 if s > 1 else 1, n + 1, (s,), generator=g, device=DEV, dtype=torch.int32).clamp_(max=n)


def _prepare_rope(case, seed):
    g = _gen(seed)
    s, n, qh, kh, d = case["seqs"], case["nodes"], case["q_heads"], case["kv_heads"], case["head_dim"]
    t = TYPES[case["type"]]
    r = lambda h: torch.randn(s, n, h, d, generator=g, device=DEV).to(t)  # noqa: E731
    lens = torch.randint(0, 9, (s,), generator=g, device=DEV, dtype=torch.int32)
    rd = case["rotary"]
    # the frequencies of base 1e6, those of long wavelengths slowed by 4 (scaling by parts)
    inv = 1e6 ** (-torch.arange(0, rd, 2, dtype=torch.float64, device=DEV) / rd)
    slow = ((2 * math.pi / inv / 4096 - 1 / 32) / (1 - 1 / 32)).clamp(0, 1)
    inv = inv * (1 - slow) + inv / 4 * slow
    base = torch.randint(0, case["far"], (s, 1), generator=g, device=DEV, dtype=torch.int32)
    depth = torch.randint(0, max(1, n), (s, n), generator=g, device=DEV, dtype=torch.int32)
    ctx = n + 8
    return {"op": "rope", "case": case, "q": r(qh), "k": r(kh), "v": r(kh), "lens": lens, "nodes": _counts(case, g),
            "slots": torch.randperm(s, generator=g, device=DEV).to(torch.int32), "inv_freq": inv, "factor": 1.138,
            "positions": (base + depth).contiguous(), "q_out": torch.zeros(s, n, qh, d, dtype=t, device=DEV),
            "ck": torch.zeros(s, 1, ctx, kh, d, dtype=torch.int8, device=DEV),
            "cv": torch.zeros(s, 1, ctx, kh, d, dtype=torch.int8, device=DEV),
            "ks": torch.ones(s, 1, ctx, device=DEV), "vs": torch.ones(s, 1, ctx, device=DEV)}


def _prepare_tree(case, seed):
    g = _gen(seed)
    s, n, c, qh, kh, d = (case[k] for k in ("seqs", "nodes", "ctx", "q_heads", "kv_heads", "head_dim"))
    t = TYPES[case["type"]]
    nodes = _counts(case, g)
    lens = torch.full((s,), c, dtype=torch.int32, device=DEV)
    if case["ragged"]:
        lens = torch.randint(0, c + 1, (s,), generator=g, device=DEV, dtype=torch.int32)
    rows = c + n
    code = lambda: torch.randint(-127, 128, (s, 1, rows, kh, d), generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
    sc = lambda: 0.01 + 0.02 * torch.rand(s, 1, rows, generator=g, device=DEV)  # noqa: E731
    mask = None
    if not case["chain"]:
        # each node's parent is an earlier node or the last committed token; a node sees its ancestors and itself
        sees = torch.zeros(s, n, n, dtype=torch.bool, device=DEV)
        at = torch.arange(s, device=DEV)
        for i in range(n):
            p = (torch.rand(s, generator=g, device=DEV) * (i + 1)).long() - 1
            sees[:, i] = sees[at, p.clamp(min=0)] & (p >= 0)[:, None]
            sees[:, i, i] = True
        words = -(-n // 64)
        bits = torch.zeros(s, n, words * 64, dtype=torch.int64, device=DEV)
        bits[:, :, :n] = sees.long()
        mask = (bits.view(s, n, words, 64) << torch.arange(64, device=DEV)).sum(-1)
    return {"op": "tree", "case": case, "q": (1.5 * torch.randn(s, n, qh, d, generator=g, device=DEV)).to(t),
            "lens": lens, "nodes": nodes, "slots": torch.randperm(s, generator=g, device=DEV).to(torch.int32),
            "ck": code(), "cv": code(), "ks": sc(), "vs": sc(), "mask": mask, "scale": d ** -0.5,
            "out": torch.zeros(s, n, qh, d, dtype=t, device=DEV),
            "mass": torch.zeros(s, 1, rows, device=DEV) if case["mass"] else None}


def _prepare_evict(case, seed):
    g = _gen(seed)
    ll, s, n, kv = case["layers"], case["seqs"], case["len"], case["kv"]
    perm = torch.randperm(2 * s, generator=g, device=DEV).to(torch.int32)
    lens = n - torch.randint(0, max(1, n // 8), (s,), generator=g, device=DEV, dtype=torch.int32)
    code = lambda: torch.randint(-127, 128, (2 * s, ll, n, 1, kv), generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
    # weights fall off by orders of magnitude, and many rows never got any: ties at zero
    mass = torch.rand(2 * s, ll, n, generator=g, device=DEV).pow(8) * 50
    mass = mass * (torch.rand(2 * s, ll, n, generator=g, device=DEV) < 0.8)
    b = case["budget"]
    return {"op": "evict", "case": case, "ck": code(), "cv": code(),
            "ks": torch.rand(2 * s, ll, n, generator=g, device=DEV), "vs": torch.rand(2 * s, ll, n, generator=g, device=DEV),
            "mass": mass, "slots": perm[:s].contiguous(), "dst": perm[s:].contiguous(), "lens": lens,
            "kept": torch.full((ll, s, b), -1, dtype=torch.int32, device=DEV), "new_lens": torch.zeros_like(lens)}


def _prepare_pick(case, seed):
    g = _gen(seed)
    r, v, h, b = case["rows"], case["vocab"], case["history"], case["biases"]
    # tokens repeat: a Zipf-like spread over the vocabulary
    hist = (v ** torch.rand(r, h, generator=g, device=DEV)).long().clamp(max=v - 1).to(torch.int32)
    u = lambda lo, hi: lo + (hi - lo) * torch.rand(r, generator=g, device=DEV)  # noqa: E731
    state = {"op": "pick", "case": case,
             "logits": (3 * torch.randn(r, v, generator=g, device=DEV)).to(TYPES[case["type"]]), "history": hist,
             "history_lens": torch.randint(h // 2, h + 1, (r,), generator=g, device=DEV, dtype=torch.int32),
             "repetition": u(1.0, 1.3), "frequency": u(0.0, 0.5), "presence": u(0.0, 0.5), "bias_ids": None,
             "bias_values": None, "allowed": None,
             "out": torch.empty(r, v, dtype=TYPES[case["type"]], device=DEV),
             "picked": torch.zeros(r, dtype=torch.int32, device=DEV)}
    if b:
        state["bias_ids"] = torch.randint(0, v, (r, b), generator=g, device=DEV, dtype=torch.int32)
        state["bias_values"] = 4 * torch.randn(r, b, generator=g, device=DEV)
    if case["grammar"]:
        w = -(-v // 32)
        state["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (r, w), generator=g, device=DEV).to(torch.int32)
    return state


def prepare(case, seed):
    state = {"rope": _prepare_rope, "tree": _prepare_tree, "evict": _prepare_evict, "pick": _prepare_pick}[case["op"]](case, seed)
    if state["op"] != "pick":
        state["cache"] = (state["ck"], state["cv"], state["ks"], state["vs"])
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------

def _rotate(x, cos, sin, rd, interleaved):
    rot, rest = x[..., :rd], x[..., rd:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = rot[..., :rd // 2], rot[..., rd // 2:]
        rot = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((rot, rest), -1)


def _quantize(x):
    """x [..., values] F32: the cache's row rule."""
    big = x.abs().amax(-1)
    scale = big / torch.full_like(big, 127.0)               # a quotient: by a Python number torch multiplies by 1/127
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.round(x / scale[..., None]).clamp(-127, 127).to(torch.int8), scale


def _plain_rope(st):
    c = st["case"]
    s, n, kh, d = c["seqs"], c["nodes"], c["kv_heads"], c["head_dim"]
    ang = st["positions"].double()[..., None, None] * st["inv_freq"]
    cos, sin = torch.cos(ang) * st["factor"], torch.sin(ang) * st["factor"]
    valid = torch.arange(n, device=DEV)[None] < st["nodes"][:, None]
    q = _rotate(st["q"].float(), cos.float(), sin.float(), c["rotary"], c["interleaved"]).to(st["q"].dtype)
    q_out = torch.where(valid[..., None, None], q, st["q_out"])
    k = _rotate(st["k"].double(), cos, sin, c["rotary"], c["interleaved"]).float().reshape(s, n, kh * d)
    kc, ks = _quantize(k)
    vc, vs = _quantize(st["v"].float().reshape(s, n, kh * d))
    row = (st["lens"][:, None] + torch.arange(n, device=DEV)[None]).long()
    slot = st["slots"].long()[:, None].expand(s, n)
    ck, cv, cks, cvs = st["cache"]
    at = (slot[valid], torch.zeros_like(slot)[valid], row[valid])
    ck.index_put_(at, kc.view(s, n, kh, d)[valid])
    cv.index_put_(at, vc.view(s, n, kh, d)[valid])
    cks.index_put_(at, ks[valid])
    cvs.index_put_(at, vs[valid])
    return q_out


def _plain_tree(st):
    c = st["case"]
    s, n, qh, kh, d = c["seqs"], c["nodes"], c["q_heads"], c["kv_heads"], c["head_dim"]
    grp = qh // kh
    ck, cv, ks, vs = (x[st["slots"].long(), 0] for x in st["cache"])
    t = ck.shape[1]
    pos = torch.arange(t, device=DEV)
    node = torch.arange(n, device=DEV)
    rel = pos[None] - st["lens"][:, None]                                   # [s, t]: the row's tree node, if >= 0
    inside = rel.clamp(0, n - 1)
    if st["mask"] is None:
        sees = inside[:, None] <= node[None, :, None]
    else:
        word = torch.gather(st["mask"], 2, (inside >> 6)[:, None].expand(s, n, t))
        sees = (word >> (inside & 63)[:, None]) & 1 == 1
    sees = (rel < 0)[:, None] | ((rel < st["nodes"][:, None])[:, None] & sees)      # [s, n, t]
    valid = node[None] < st["nodes"][:, None]
    sees = sees & valid[..., None]
    q = st["q"].float().view(s, n, kh, grp, d).permute(0, 2, 1, 3, 4).reshape(s, kh, n * grp, d)
    k = ck.float().mul_(ks[..., None, None]).permute(0, 2, 1, 3)
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(st["scale"]).view(s, kh, n, grp, t)
    scores.masked_fill_(~sees[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    v = cv.float().mul_(vs[..., None, None]).permute(0, 2, 1, 3)
    o = torch.matmul(p.view(s, kh, n * grp, t), v).view(s, kh, n, grp, d).permute(0, 2, 1, 3, 4).reshape(s, n, qh, d)
    out = torch.where(valid[..., None, None], o.to(st["q"].dtype), st["out"])
    if st["mass"] is not None:
        st["mass"][st["slots"].long(), 0] += p.sum((1, 2, 3))
    return out


def _plain_evict(st):
    c = st["case"]
    ll, s, b = c["layers"], c["seqs"], c["budget"]
    src, dst = st["slots"].long(), st["dst"].long()
    ck, cv, ks, vs = st["cache"]
    t = ks.shape[2]
    pos = torch.arange(t, device=DEV)
    lens = st["lens"].long()[:, None, None]
    key = st["mass"][src].double()
    fixed = (pos < c["sink"]) | (pos >= lens - c["recent"])
    key = torch.where(fixed, torch.full_like(key, math.inf), key)
    key = torch.where(pos < lens, key, torch.full_like(key, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :b]
    new = torch.minimum(lens, torch.full_like(lens, b))
    have = torch.arange(b, device=DEV) < new                                # [s, 1, b]
    idx = torch.sort(torch.where(have, order, torch.full_like(order, t)), dim=-1).values
    kept = torch.where(have, idx, torch.full_like(idx, -1))
    idx = torch.where(have, idx, torch.zeros_like(idx))
    lay = torch.arange(ll, device=DEV)[None, :, None]
    full = have.expand(s, ll, b)
    at = tuple(x.expand(s, ll, b)[full] for x in (dst[:, None, None], lay, torch.arange(b, device=DEV)[None, None]))
    frm = tuple(x.expand(s, ll, b)[full] for x in (src[:, None, None], lay, idx))
    for x in (ck, cv, ks, vs):
        x.index_put_(at, x[frm])
    moved = torch.zeros(s, ll, t, device=DEV)
    moved[..., :b] = torch.where(full, st["mass"][src[:, None, None], lay, idx], torch.zeros((), device=DEV))
    old = st["mass"][dst]
    st["mass"][dst] = torch.where(pos < lens, moved, old)
    return kept.permute(1, 0, 2).to(torch.int32), new[:, 0, 0].to(torch.int32)


def _plain_pick(st):
    x = st["logits"].float()
    r, v = x.shape
    live = torch.arange(st["history"].shape[1], device=DEV)[None] < st["history_lens"][:, None]
    count = torch.zeros(r, v, dtype=torch.int32, device=DEV)
    count.scatter_add_(1, st["history"].long(), live.to(torch.int32))
    rep, freq, pres = (st[k][:, None] for k in ("repetition", "frequency", "presence"))
    seen = count > 0
    y = torch.where(x > 0, x / rep, x * rep)
    y = y - freq * count.float()
    y = y - pres
    x = torch.where(seen, y, x)
    if st["bias_ids"] is not None:
        n = st["bias_ids"].shape[1]
        last = torch.full((r, v), -1, dtype=torch.int32, device=DEV)
        entry = torch.arange(n, device=DEV, dtype=torch.int32)[None].expand(r, n)
        last.scatter_reduce_(1, st["bias_ids"].long(), entry, "amax")          # an id listed twice: the last entry
        bias = torch.gather(st["bias_values"], 1, last.clamp(min=0).long())
        x = torch.where(last >= 0, x + bias, x)
    if st["allowed"] is not None:
        tok = torch.arange(v, device=DEV)
        ok = (st["allowed"][:, tok >> 5] >> (tok & 31).to(torch.int32)) & 1
        x = torch.where(ok == 1, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(v, device=DEV)[None], torch.full((1, 1), v, device=DEV)).amin(-1)
    first = torch.where(torch.isfinite(top[:, 0]), first, torch.full_like(first, -1))
    return x.to(st["logits"].dtype), first.to(torch.int32)


# ---- one pass ----------------------------------------------------------------------------------------------------

def _own_cache(st):
    """The handle on its cache that a user's program keeps."""
    if "handle" not in st:
        st["handle"] = _ops().KvCache(*st["cache"])
    return st["handle"]


def run(st):
    c, op = st["case"], st["op"]
    if op == "rope":
        if own:
            q_out = _ops().rope_append(_own_cache(st), 0, st["slots"], st["lens"], st["q"], st["k"], st["v"], st["inv_freq"],
                                       positions=st["positions"], nodes=st["nodes"], interleaved=c["interleaved"],
                                       factor=st["factor"], q_out=st["q_out"])
        else:
            q_out = _plain_rope(st)
        ck, cv, ks, vs = st["cache"]
        return {"q": q_out, "k": ck * ks[..., None, None], "v": cv * vs[..., None, None]}
    if op == "tree":
        if own:
            out = _ops().tree_attention(_own_cache(st), 0, st["slots"], st["lens"], st["q"], nodes=st["nodes"],
                                        mask=st["mask"], scale=st["scale"], out=st["out"], mass=st["mass"])
        else:
            out = _plain_tree(st)
        return {"out": out, "mass": st["mass"]}
    if op == "evict":
        if own:
            kept, new = _ops().evict(_own_cache(st), st["slots"], st["lens"], st["mass"], c["budget"], c["sink"], c["recent"],
                                     dst_slots=st["dst"], kept=st["kept"], new_lens=st["new_lens"])
        else:
            kept, new = _plain_evict(st)
        ck, cv, ks, vs = st["cache"]
        return {"kept": kept, "lens": new, "k": ck, "v": cv, "ks": ks, "vs": vs, "mass": st["mass"]}
    if own:
        out, picked = _ops().pick_tokens(st["logits"], history=st["history"], history_lens=st["history_lens"],
                                         repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"],
                                         bias_ids=st["bias_ids"], bias_values=st["bias_values"], allowed=st["allowed"],
                                         out=st["out"], picked=st["picked"])
    else:
        out, picked = _plain_pick(st)
    return {"logits": out, "picked": picked}


def work(case):
    op = case["op"]
    if op == "rope":
        e = torch.finfo(TYPES[case["type"]]).bits // 8
        t, d = case["seqs"] * case["nodes"] * (0.5 if case["ragged"] else 1), case["head_dim"]
        kv = case["kv_heads"] * d
        return {"bytes": t * (e * (2 * case["q_heads"] * d + 2 * kv) + 2 * kv + 12), "flops": t * 3 * (case["q_heads"] + case["kv_heads"]) * case["rotary"]}
    if op == "tree":
        e = torch.finfo(TYPES[case["type"]]).bits // 8
        f = 0.5 if case["ragged"] else 1
        keys = case["ctx"] * f + case["nodes"]
        nodes = case["nodes"] * (1 if not case["ragged"] or case["nodes"] == 1 else f)
        kv, q = case["kv_heads"] * case["head_dim"], case["q_heads"] * case["head_dim"]
        return {"bytes": case["seqs"] * (keys * (2 * kv + 8 + (8 if case["mass"] else 0)) + 2 * nodes * q * e),
                "flops": 4 * case["seqs"] * nodes * keys * q}
    if op == "evict":
        units, n, b = case["layers"] * case["seqs"], case["len"] * 15 / 16, min(case["budget"], case["len"])
        return {"bytes": units * (4 * n + b * (2 * (2 * case["kv"] + 8) + 8) + 4 * n), "flops": 0}
    e = torch.finfo(TYPES[case["type"]]).bits // 8
    return {"bytes": case["rows"] * (2 * e * case["vocab"] + 3 * case["history"] + 8 * case["biases"] + (case["vocab"] / 8 if case["grammar"] else 0)),
            "flops": 0}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------

def _exact_rope(case, st):
    d, rd, kh = case["head_dim"], case["rotary"], case["kv_heads"]
    z = torch.polar(torch.full_like(st["inv_freq"], st["factor"]), torch.zeros_like(st["inv_freq"]))
    turn = z * torch.exp(1j * (st["positions"].double().unsqueeze(-1) * st["inv_freq"]))       # [s, n, rd/2]

    def spin(x):
        x = x.double()
        head = x[..., :rd]
        pair = head.unflatten(-1, (rd // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, rd // 2)).transpose(-1, -2)
        w = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn[:, :, None])
        w = w.flatten(-2) if case["interleaved"] else w.transpose(-1, -2).flatten(-2)
        return torch.cat((w, x[..., rd:]), -1)

    q = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    ck, cv, _, _ = st["cache"]
    keys, vals = torch.zeros(ck.shape, dtype=torch.float64, device=DEV), torch.zeros(cv.shape, dtype=torch.float64, device=DEV)
    rq, rk = spin(st["q"]), spin(st["k"]).float().double()
    rv = st["v"].double()
    lens, nodes, slots = st["lens"].tolist(), st["nodes"].tolist(), st["slots"].tolist()
    for i in range(case["seqs"]):
        m = nodes[i]
        q[i, :m] = rq[i, :m]
        for into, x in ((keys, rk[i, :m]), (vals, rv[i, :m])):
            step = x.abs().flatten(1).amax(1) / 127
            step = torch.where(step > 0, step, torch.ones_like(step)).view(-1, 1, 1)
            # the codes come from the scale as it is held, in 32 bits
            held = step.float()
            into[slots[i], 0, lens[i]:lens[i] + m] = torch.round(x.float() / held).double() * step
    return {"q": q, "k": keys, "v": vals}


def _exact_tree(case, st):
    qh, kh, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    mass = torch.zeros(st["ks"].shape, dtype=torch.float64, device=DEV)
    lens, nodes, slots = st["lens"].tolist(), st["nodes"].tolist(), st["slots"].tolist()
    for i in range(case["seqs"]):
        a, m = lens[i], nodes[i]
        if m == 0:
            continue
        k = st["ck"][slots[i], 0, :a + m].double() * st["ks"][slots[i], 0, :a + m, None, None].double()
        v = st["cv"][slots[i], 0, :a + m].double() * st["vs"][slots[i], 0, :a + m, None, None].double()
        hidden = torch.zeros(m, a + m, dtype=torch.bool, device=DEV)
        if st["mask"] is None:
            hidden[:, a:] = torch.ones(m, m, dtype=torch.bool, device=DEV).triu(1)
        else:
            for j in range(m):
                hidden[:, a + j] = (st["mask"][i, :m, j // 64] >> (j % 64)) & 1 == 0
        for h in range(kh):
            qs = st["q"][i, :m, h * (qh // kh):(h + 1) * (qh // kh)].double()
            w = torch.einsum("mgd,td->gmt", qs, k[:, h]) * case["head_dim"] ** -0.5
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[i, :m, h * (qh // kh):(h + 1) * (qh // kh)] = torch.einsum("gmt,td->mgd", w, v[:, h])
            mass[slots[i], 0, :a + m] += w.sum((0, 1))
    return {"out": out, "mass": mass if case["mass"] else None}


def _exact_pick(case, st):
    x = st["logits"].double()
    for i in range(case["rows"]):
        count = torch.bincount(st["history"][i, :int(st["history_lens"][i])].long(), minlength=case["vocab"])
        ids = count.nonzero()[:, 0]
        rep, row = st["repetition"][i].double(), x[i, ids]
        row = torch.maximum(row, torch.zeros_like(row)) / rep + torch.minimum(row, torch.zeros_like(row)) * rep
        x[i, ids] = row - count[ids] * st["frequency"][i].double() - st["presence"][i].double()
        if st["bias_ids"] is not None:
            chosen = dict(zip(st["bias_ids"][i].tolist(), st["bias_values"][i].double().tolist()))
            x[i, torch.tensor(list(chosen), device=DEV)] += torch.tensor(list(chosen.values()), dtype=torch.float64, device=DEV)
    if st["allowed"] is not None:
        bits = (st["allowed"].unsqueeze(-1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        x.masked_fill_(bits.flatten(1)[:, :case["vocab"]] == 0, -math.inf)
    return {"logits": x, "picked": None}


def exact(case, seed):
    if case["op"] == "evict":
        return None                                     # rows are chosen and moved: no computed numbers
    st = prepare(case, seed)
    return {"rope": _exact_rope, "tree": _exact_tree, "pick": _exact_pick}[case["op"]](case, st)
