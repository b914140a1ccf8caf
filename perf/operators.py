"""Operators of a speculative step that verifies a tree of drafted tokens over a paged
KV cache: what they compute, in elementary torch operations, and the framework's calls.

  append   RMSNorm and rotation of a step's queries and keys, its keys and values into
           the pages of a cache
  attn     attention of every sequence's drafted tokens over its pages
  sample   one token per row of logits: temperature, top-k, top-p and min-p, from given
           random numbers
  accept   the accepted path of every sequence's tree, its keys and values moved to the
           positions that follow the context

Cache: k and v [layers][pages][kv heads][page size][head dim], a sequence's position p in
page table[p // page size] at p % page size.  The tokens of a step ("rows") stand
sequence after sequence; row j of a sequence has its K / V at position context + j, sees
the context and, with a mask, the rows whose bits are set, without one the rows up to
itself.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False  # True: the framework's kernels, False: the plain forms

DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
CACHE = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}
# query heads, kv heads, head dim, rotated dims, theta
HEADS = [(24, 4, 256, 64, 1e7), (10, 2, 256, 64, 1e7), (5, 1, 256, 256, 1e6), (32, 8, 128, 128, 5e5),
         (16, 16, 128, 64, 1e4), (8, 8, 64, 64, 1e4)]


def listed():
    q27 = {"nq": 24, "nkv": 4, "hd": 256, "rot": 64, "theta": 1e7}  # the hybrid model's attention layers
    gqa = {"nq": 32, "nkv": 8, "hd": 128, "rot": 128, "theta": 5e5}
    return [
        # One sequence decoding one token: the smallest call there is, once per layer.
        {"name": "append_1", "op": "append", "type": "f32", "rows": 1, "pad": 0, "page": 16, "pos": 32000, **q27},
        # A verify of many ragged trees in a half-precision model, padded to a fixed batch.
        {"name": "append_1013", "op": "append", "type": "bf16", "rows": 1013, "pad": 11, "page": 64, "pos": 9000,
         **gqa},
        # A whole prompt chunk.
        {"name": "append_4096", "op": "append", "type": "f32", "rows": 4096, "pad": 0, "page": 256, "pos": 131072,
         **q27},
        # One sequence, one token, a short conversation.
        {"name": "attn_1x1_700", "op": "attn", "type": "f32", "B": 1, "R": 1, "ctx": 700, "ragged": False,
         "mask": "chain", "gate": True, "page": 16, **q27},
        # One sequence, one token, the longest context.
        {"name": "attn_1x1_131k", "op": "attn", "type": "f16", "B": 1, "R": 1, "ctx": 131071, "ragged": False,
         "mask": "chain", "gate": False, "page": 64, **q27},
        # An odd batch of small trees at contexts of every length.
        {"name": "attn_13x8_8k", "op": "attn", "type": "bf16", "B": 13, "R": 8, "ctx": 8191, "ragged": True,
         "mask": "tree", "gate": False, "page": 32, **gqa},
        # Wide trees over long contexts: the matrix cores' case.
        {"name": "attn_8x64_32k", "op": "attn", "type": "f32", "B": 8, "R": 64, "ctx": 32000, "ragged": False,
         "mask": "tree", "gate": True, "page": 256, **q27},
        # One user's next token.
        {"name": "sample_1", "op": "sample", "type": "f32", "rows": 1, "V": 248320, "mode": "both"},
        # A batch of small-vocabulary requests with logits in half precision (many ties).
        {"name": "sample_13", "op": "sample", "type": "bf16", "rows": 13, "V": 32000, "mode": "mixed"},
        # Every node of a batch's trees, each request with its own settings.
        {"name": "sample_128", "op": "sample", "type": "f32", "rows": 128, "V": 248320, "mode": "mixed"},
        # One sequence's chain of drafts, one layer.
        {"name": "accept_1x4", "op": "accept", "type": "f16", "B": 1, "R": 4, "layers": 1, "ctx": 255, "page": 16,
         **q27},
        # A full batch of wide trees through all attention layers.
        {"name": "accept_48x64", "op": "accept", "type": "f16", "B": 48, "R": 64, "layers": 16, "ctx": 120,
         "page": 32, **q27},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attn", "sample", "accept"])
    nq, nkv, hd, rot, theta = rng.choice(HEADS)
    heads = {"nq": nq, "nkv": nkv, "hd": hd, "rot": rot, "theta": theta}
    typ = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        rows = _log(rng, 1, 4096)
        return {"op": op, "type": typ, "rows": rows, "pad": rng.randint(0, 9) if rows > 20 else 0, "page": page,
                "pos": _log(rng, 1, 131072), **heads}
    if op == "attn":
        ctx = _log(rng, 1, 65536)
        B = _log(rng, 1, max(1, min(64, (8 * 32000 * 4 * 256) // (ctx * nkv * hd))))
        R = _log(rng, 1, max(1, min(64, (8 * 64 * 32000 * 24 * 256) // (B * ctx * nq * hd))))
        return {"op": op, "type": typ, "B": B, "R": R, "ctx": ctx, "ragged": rng.random() < 0.6,
                "mask": rng.choice(["chain", "tree", "tree"]), "gate": rng.random() < 0.5, "page": page, **heads}
    if op == "sample":
        V = rng.choice([248320, 151936, 32000, 1000, 50257])
        return {"op": op, "type": typ, "rows": _log(rng, 1, 128), "V": V,
                "mode": rng.choice(["mixed", "mixed", "both", "topp", "topk", "full"])}
    layers = rng.choice([1, 2, 16])
    return {"op": op, "type": rng.choice(["f16", "bf16"]), "B": _log(rng, 1, 48), "R": _log(rng, 1, 64),
            "layers": layers, "ctx": rng.randint(0, 200), "page": page, **heads}


# ---------------------------------------------------------------- inputs from the seed


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * std


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def _lens(c):
    """Context and rows of every sequence (of the case alone, so that work() knows them)."""
    B, ctx, R = c["B"], c["ctx"], c["R"]
    if not c.get("ragged", c["op"] == "accept"):
        return [ctx] * B, [R] * B
    return ([ctx if b == B - 1 else ctx * (2 * b + 1) // (2 * B) for b in range(B)],
            [R if b == 0 else 1 + (7 * b) % R for b in range(B)])


def _trees(r, rows):
    """Drafted trees, a sequence's nodes in an order that has parents first: parent of
    every row (within its sequence, -1 for the root) and the ancestors' bits, its own too."""
    parents, bits = [], []
    for n in rows:
        own_bits = []
        for i in range(n):
            p = -1 if i == 0 else int(r.integers(max(0, (i - 1) // 2 - 1), i))
            parents.append(p)
            own_bits.append((own_bits[p] if i else 0) | (1 << i))
        bits += own_bits
    bits = np.array(bits, np.uint64).view(np.int64)
    return np.array(parents, np.int32), bits


def _tables(r, lens, page, spare):
    """Pages of every sequence in random order; unused entries hold -1."""
    need = [-(-n // page) for n in lens]
    order = r.permutation(sum(need) + spare)
    table = np.full((len(lens), max(need) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def prepare(case, seed):
    c = dict(case)
    r = np.random.default_rng(seed)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt, ct = TYPES[c["type"]][0], CACHE[c["type"]]
    if c["op"] == "sample":
        n, V = c["rows"], c["V"]
        z = _randn(g, n, V, std=2.0)
        # a head of a few dozen likely tokens over the bulk
        top = torch.randint(0, V, (n, 40), generator=g, device=DEV)
        z.scatter_(1, top, 4.0 + 2.5 * _randn(g, n, 40).abs() + 3.0 * _randn(g, n, 1).abs())
        pick = lambda *v: r.choice(v, n)  # noqa: E731
        m = c["mode"]
        f32 = lambda a: torch.tensor(np.asarray(a, np.float32), device=DEV)  # noqa: E731
        ones = np.ones(n)
        temp = pick(0.0, 0.6, 0.8, 1.0, 1.3) if m == "mixed" else pick(0.7, 0.9, 1.0)
        k = pick(0, 1, 20, 50, 1000) if m == "mixed" else pick(20, 40, 64) if m in ("both", "topk") else 0 * ones
        p = pick(1.0, 0.5, 0.9, 0.95) if m == "mixed" else pick(0.9, 0.95) if m in ("both", "topp") else ones
        mp = pick(0.0, 0.0, 0.02, 0.1) if m == "mixed" else 0 * ones
        return {"c": c, "z": z.to(dt), "temp": f32(temp), "k": _i32(k), "p": f32(p), "mp": f32(mp),
                "u": torch.rand(n, generator=g, device=DEV), "idx": torch.empty(n, dtype=torch.int32, device=DEV),
                "prob": torch.empty(n, device=DEV)}
    nq, nkv, hd, page = c["nq"], c["nkv"], c["hd"], c["page"]
    if c["op"] == "append":
        n, pad = c["rows"], c["pad"]
        # the fused projection's rows: per head q then its gate, then the keys, the values
        y = _randn(g, n, (2 * nq + 2 * nkv) * hd, std=1.5).to(dt)
        pages = -(-n // page) + 2
        start = int(r.integers(0, page))  # the first token's place in its page
        order = r.permutation(pages)
        at = start + np.arange(n)
        slots = order[at // page].astype(np.int64) * page + at % page
        slots[n - pad:] = -1
        pos = c["pos"] + np.arange(n)
        kc = _randn(g, 1, pages, nkv, page, hd).to(ct)
        return {"c": c, "y": y, "qn": _randn(g, hd, std=0.1), "kn": _randn(g, hd, std=0.1), "pos": _i32(pos),
                "slots": torch.tensor(slots, device=DEV), "k": kc, "v": kc.flip(1).contiguous(),
                "q": torch.empty(n, nq, hd, dtype=dt, device=DEV)}
    ctx, rows = _lens(c)
    total = sum(rows)
    start = _i32(np.concatenate([[0], np.cumsum(rows)]))
    table, pages = _tables(r, [a + b for a, b in zip(ctx, rows)], page, 3)
    parents, bits = _trees(r, rows)
    s = {"c": c, "table": _i32(table), "ctx": _i32(ctx), "start": start, "pages": pages}
    L = c.get("layers", 1)
    s["k"] = torch.empty(L, pages, nkv, page, hd, dtype=ct, device=DEV)
    s["v"] = torch.empty_like(s["k"])
    for t in (s["k"], s["v"]):
        flat = t.view(L, -1)
        for layer in range(L):
            flat[layer] = torch.randn(flat.shape[1], generator=g, device=DEV).to(ct)
    if c["op"] == "attn":
        s["q"] = _randn(g, total, nq, hd, std=1.7).to(dt)
        s["y"] = _randn(g, total, nq, 2, hd).to(dt) if c["gate"] else None  # gates at [:, :, 1]
        s["mask"] = torch.tensor(bits, device=DEV).view(total, 1) if c["mask"] == "tree" else None
        s["out"] = torch.empty(total, nq, hd, dtype=dt, device=DEV)
        return s
    # verified trees: most nodes' sampled token is one of their children's
    V = 1000
    toks, samples = r.integers(0, V, total), r.integers(0, V, total)
    base = np.repeat(np.concatenate([[0], np.cumsum(rows)[:-1]]), rows)
    has = np.flatnonzero((parents >= 0) & (r.random(total) < 0.8))
    samples[base[has] + parents[has]] = toks[has]
    s.update(parents=_i32(parents), toks=_i32(toks), samples=_i32(samples), total=total,
             bits=torch.tensor(bits, device=DEV),
             path=torch.empty(c["B"], c["R"], dtype=torch.int32, device=DEV),
             n=torch.empty(c["B"], dtype=torch.int32, device=DEV),
             nxt=torch.empty(c["B"], dtype=torch.int32, device=DEV),
             ctx_out=torch.empty(c["B"], dtype=torch.int32, device=DEV))
    return s


# ---------------------------------------------------------------- the plain forms


def _norm_rope(x, gamma, pos, c):
    """x [rows][heads][hd] in 32 bits: RMSNorm with weight 1 + gamma, then the first rot
    dims rotated in pairs (i, i + rot / 2); angles in 64 bits (far positions)."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + gamma)
    half = c["rot"] // 2
    freq = c["theta"] ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    ang = (pos.double()[:, None] * freq)[:, None, :]
    cos, sin = ang.cos().float(), ang.sin().float()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], -1)


def _plain_append(s, c):
    n, nq, nkv, hd = c["rows"], c["nq"], c["nkv"], c["hd"]
    y = s["y"].float().view(n, -1, hd)
    q, k, v = y[:, 0:2 * nq:2], y[:, 2 * nq:2 * nq + nkv], y[:, 2 * nq + nkv:]
    s["q"].copy_(_norm_rope(q, s["qn"], s["pos"], c))
    k = _norm_rope(k, s["kn"], s["pos"], c)
    # rows without a slot write row 0's values once more
    here = (s["slots"] >= 0)[:, None, None]
    slot = torch.where(s["slots"] >= 0, s["slots"], s["slots"][0])
    ct = s["k"].dtype
    s["k"][0][slot // c["page"], :, slot % c["page"]] = torch.where(here, k, k[:1]).to(ct)
    s["v"][0][slot // c["page"], :, slot % c["page"]] = torch.where(here, v, v[:1]).to(ct)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _gathered(pool, table, c):
    """[B][kv heads][positions][hd] in 32 bits through the table."""
    B = table.shape[0]
    x = pool[table.clamp(min=0).long()]  # [B][entries][kv][page][hd]
    return x.permute(0, 2, 1, 3, 4).reshape(B, c["nkv"], -1, c["hd"]).float()


def _plain_attn(s, c):
    B, nq, nkv, hd = c["B"], c["nq"], c["nkv"], c["hd"]
    G, total = nq // nkv, s["q"].shape[0]
    R = c["R"]
    K, V = _gathered(s["k"][0], s["table"], c), _gathered(s["v"][0], s["table"], c)
    L = K.shape[2]
    dev_rows = torch.arange(R, device=DEV)
    start, count = s["start"][:-1].long(), (s["start"][1:] - s["start"][:-1]).long()
    at = (start[:, None] + dev_rows).clamp(max=total - 1)  # [B][R], padded rows any
    q = s["q"].float()[at].view(B, R, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B * nkv, R * G, hd).contiguous()
    sc = torch.bmm(q, K.view(B * nkv, L, hd).transpose(1, 2).contiguous()) / math.sqrt(hd)
    j = torch.arange(L, device=DEV)[None, None, :] - s["ctx"].long()[:, None, None]  # tree slot of a position
    if s["mask"] is None:
        sees = j <= dev_rows[None, :, None]
    else:
        bits = s["mask"][:, 0][at][:, :, None]
        sees = (j < 0) | ((j < 64) & (((bits >> j.clamp(0, 63)) & 1) == 1))
    sc = sc.view(B, nkv, R, G, L).masked_fill(~sees[:, None, :, None, :], -math.inf)
    sc = sc - sc.amax(-1, keepdim=True)
    p = torch.exp(sc)
    p = p / p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(B * nkv, R * G, L), V.view(B * nkv, L, hd))
    o = o.view(B, nkv, R, G, hd).permute(0, 2, 1, 3, 4).reshape(B * R, nq, hd)
    row = torch.arange(total, device=DEV)
    b = torch.searchsorted(s["start"][1:].long(), row, right=True)
    o = o[b * R + row - start[b]]
    if s["y"] is not None:
        o = o * torch.sigmoid(s["y"].float()[:, :, 1])
    s["out"].copy_(o)
    return s["out"]


def _plain_sample(s, c):
    """Order: temperature, top-k (ties to the lowest index), top-p over what top-k left
    (every token before which less than p of the mass stands), min-p against the likeliest
    token; then the first token, by index, up to which more than u of the mass stands."""
    z = s["z"].float()
    z = torch.where(torch.isnan(z), -math.inf, z)
    n, V = z.shape
    zs, order = torch.sort(z, dim=-1, descending=True, stable=True)
    T = s["temp"].double()[:, None]
    w = torch.exp((zs.double() - zs[:, :1].double()) / torch.where(T > 0, T, 1.0))
    rank = torch.arange(V, device=DEV)[None, :]
    k = s["k"].long()[:, None]
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    cum = torch.cumsum(w, -1)
    p = s["p"].double()[:, None]
    w = torch.where((cum - w < p * cum[:, -1:]) | (p >= 1) | (rank == 0), w, 0.0)
    w = torch.where((w >= s["mp"].double()[:, None]) & ((T > 0) | (rank == 0)), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    cum = torch.cumsum(w, -1)
    total = cum[:, -1:]
    idx = (cum <= s["u"].double()[:, None] * total).sum(-1, keepdim=True).clamp(max=V - 1)
    s["idx"].copy_(idx[:, 0])
    s["prob"].copy_((torch.gather(w, 1, idx) / total)[:, 0])
    return {"idx": s["idx"], "prob": s["prob"]}


def _plain_accept(s, c):
    B, R, total, page = c["B"], c["R"], s["total"], c["page"]
    i = torch.arange(R, device=DEV)
    start, count = s["start"][:-1].long(), (s["start"][1:] - s["start"][:-1]).long()
    at = (start[:, None] + i).clamp(max=total - 1)
    here = i < count[:, None]
    par = s["parents"].long()[at]
    tok, smp = s["toks"][at], s["samples"][at]
    fits = here & (par >= 0) & (torch.gather(smp, 1, par.clamp(min=0)) == tok)
    # of siblings that fit, the first
    same = (par[:, :, None] == par[:, None, :]) & (i[None, :] < i[:, None])
    fits &= ~(same & fits[:, None, :]).any(-1)
    fits |= here & (par < 0)
    anc = ((s["bits"][at][:, :, None] >> i) & 1) == 1
    on = here & (~anc | fits[:, None, :]).all(-1)
    n = on.sum(-1)
    path = torch.sort(torch.where(on, i, R), dim=-1).values  # nodes of the path in order
    last = torch.gather(path, 1, (n - 1).clamp(min=0)[:, None])
    s["path"].copy_(torch.where(path < R, path, -1))
    s["n"].copy_(n)
    s["nxt"].copy_(torch.gather(smp, 1, last)[:, 0])
    s["ctx_out"].copy_(s["ctx"] + n)
    # position context + d takes node path[d]; the others keep what they have
    src = s["ctx"].long()[:, None] + torch.where(path < R, path, i)
    dst = s["ctx"].long()[:, None] + i
    src, dst = torch.where(here, src, s["ctx"].long()[:, None]), torch.where(here, dst, s["ctx"].long()[:, None])
    where = lambda x: (torch.gather(s["table"].long(), 1, x // page), x % page)  # noqa: E731
    (sp, so), (dp, do) = where(src), where(dst)
    for t in (s["k"], s["v"]):
        t[:, dp, :, do] = t[:, sp, :, so]
    return {"path": s["path"], "n": s["n"], "next": s["nxt"], "ctx": s["ctx_out"], "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------- the framework's calls


def _cache(s, c):
    """The cache's descriptor and, once, the workspace: both are kept between calls."""
    from rapidllm_amd import hip

    if "cache" not in s:
        L, pages, nkv, page, hd = s["k"].shape
        s["cache"] = hip.RlPagedCache(s["k"].data_ptr(), s["v"].data_ptr(), pages * nkv * page * hd, L, pages, page,
                                      nkv, hd, 2 if s["k"].dtype == torch.bfloat16 else 1)
        if c["op"] == "attn":
            s["ws"] = torch.empty(hip.lib().rl_hip_tree_attn_workspace_bytes(c["nq"], nkv, hd, c["B"], c["R"]),
                                  dtype=torch.uint8, device=DEV)
    return hip.call, s["cache"]


def _own_append(s, c):
    call, cache = _cache(s, c)
    nq, nkv, hd, e = c["nq"], c["nkv"], c["hd"], s["y"].element_size()
    y, ld = s["y"].data_ptr(), s["y"].shape[1]
    call("rl_hip_paged_append", cache, 0, TYPES[c["type"]][1], y, ld, 2 * hd, y + 2 * nq * hd * e, ld, hd,
         y + (2 * nq + nkv) * hd * e, ld, hd, s["qn"].data_ptr(), s["kn"].data_ptr(), 1, EPS, c["rot"], c["theta"],
         s["pos"].data_ptr(), s["slots"].data_ptr(), c["rows"], nq, s["q"].data_ptr(),
         torch.cuda.current_stream().cuda_stream)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_attn(s, c):
    call, cache = _cache(s, c)
    nq, hd, q, y = c["nq"], c["hd"], s["q"], s["y"]
    gate = y.data_ptr() + hd * y.element_size() if y is not None else None
    call("rl_hip_tree_attn", cache, 0, TYPES[c["type"]][1], q.data_ptr(), nq * hd, hd, gate, 2 * nq * hd, 2 * hd,
         s["table"].data_ptr(), s["table"].shape[1], s["ctx"].data_ptr(), s["start"].data_ptr(), c["B"], q.shape[0],
         c["R"], s["mask"].data_ptr() if s["mask"] is not None else None, 1, nq, 1.0 / math.sqrt(hd),
         s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_sample(s, c):
    from rapidllm_amd import hip

    n, V = s["z"].shape
    if "ws" not in s:
        s["ws"] = torch.empty(hip.lib().rl_hip_sample_workspace_bytes(n, V), dtype=torch.uint8, device=DEV)
    hip.call("rl_hip_sample_rows", TYPES[c["type"]][1], s["z"].data_ptr(), V, n, V, s["temp"].data_ptr(),
             s["k"].data_ptr(), s["p"].data_ptr(), s["mp"].data_ptr(), s["u"].data_ptr(), s["idx"].data_ptr(),
             s["prob"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), torch.cuda.current_stream().cuda_stream)
    return {"idx": s["idx"], "prob": s["prob"]}


def _own_accept(s, c):
    call, cache = _cache(s, c)
    call("rl_hip_tree_accept", cache, s["table"].data_ptr(), s["table"].shape[1], s["ctx"].data_ptr(),
         s["start"].data_ptr(), c["B"], s["total"], s["parents"].data_ptr(), s["toks"].data_ptr(),
         s["samples"].data_ptr(), s["path"].data_ptr(), c["R"], s["n"].data_ptr(), s["nxt"].data_ptr(),
         s["ctx_out"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return {"path": s["path"], "n": s["n"], "next": s["nxt"], "ctx": s["ctx_out"], "k": s["k"], "v": s["v"]}


_PLAIN = {"append": _plain_append, "attn": _plain_attn, "sample": _plain_sample, "accept": _plain_accept}
_OWN = {"append": _own_append, "attn": _own_attn, "sample": _own_sample, "accept": _own_accept}


def run(s):
    return (_OWN if own else _PLAIN)[s["c"]["op"]](s, s["c"])


# ---------------------------------------------------------------- work


def work(case):
    c = case
    e = 4 if c["type"] == "f32" else 2
    if c["op"] == "sample":
        return {"bytes": c["rows"] * (c["V"] * e + 28), "flops": 4 * c["rows"] * c["V"]}
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    if c["op"] == "append":
        n = c["rows"]
        return {"bytes": n * ((2 * nq + 2 * nkv) * hd * e + 2 * nkv * hd * 2 + 12) + 8 * hd,
                "flops": n * (nq + nkv) * (4 * hd + 3 * c["rot"])}
    ctx, rows = _lens(c)
    if c["op"] == "attn":
        seen = sum(a * b + (b * (b + 1) // 2 if c["mask"] == "chain" else b) for a, b in zip(ctx, rows))
        rw = sum(rows) * nq * hd * e * (3 if c["gate"] else 2)
        return {"bytes": rw + sum(a + b for a, b in zip(ctx, rows)) * nkv * hd * 4, "flops": 4 * seen * nq * hd}
    # a path of about a fifth of the nodes at most 8 long, read and written in K and V
    moved = sum(min(8, -(-b // 5)) for b in rows)
    return {"bytes": sum(rows) * 12 + c["B"] * (4 * c["R"] + 20) + moved * c["layers"] * nkv * hd * 8,
            "flops": sum(rows)}


# ---------------------------------------------------------------- 64-bit references


def _exact_append(s, c):
    n, nq, nkv, hd, page = c["rows"], c["nq"], c["nkv"], c["hd"], c["page"]
    y = s["y"].double().view(n, 2 * nq + 2 * nkv, hd)
    half = c["rot"] // 2
    inv = torch.exp(-math.log(c["theta"]) * torch.arange(half, dtype=torch.float64, device=DEV) / half)
    turn = torch.polar(torch.ones(n, half, dtype=torch.float64, device=DEV), torch.outer(s["pos"].double(), inv))

    def head(x, gamma):
        x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * (gamma.double() + 1)
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

    kc, vc = s["k"].double(), s["v"].double()
    k = head(y[:, 2 * nq:2 * nq + nkv], s["kn"])
    m = n - c["pad"]
    slot = s["slots"][:m]
    kc[0].index_put_((slot // page, torch.arange(nkv, device=DEV)[:, None], slot % page), k[:m].transpose(0, 1))
    vc[0].index_put_((slot // page, torch.arange(nkv, device=DEV)[:, None], slot % page),
                     y[:m, 2 * nq + nkv:].transpose(0, 1))
    return {"q": head(y[:, :2 * nq:2], s["qn"]), "k": kc, "v": vc}


def _exact_attn(s, c):
    nq, nkv, hd, page = c["nq"], c["nkv"], c["hd"], c["page"]
    G = nq // nkv
    ctx, rows = _lens(c)
    out = torch.zeros(sum(rows), nq, hd, dtype=torch.float64, device=DEV)
    at = 0
    for b, (a, n) in enumerate(zip(ctx, rows)):
        pos = torch.arange(a + n, device=DEV)
        pg, off = s["table"][b].long()[pos // page], pos % page
        sees = torch.ones(n, a + n, dtype=torch.bool, device=DEV)
        if s["mask"] is None:
            sees[:, a:] = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        else:
            word = s["mask"][at:at + n].cpu().numpy().view(np.uint64)
            sees[:, a:] = torch.tensor((word >> np.arange(n, dtype=np.uint64)) & np.uint64(1) == 1, device=DEV)
        for h in range(nkv):
            kh, vh = s["k"][0][pg, h, off].double(), s["v"][0][pg, h, off].double()
            q = s["q"][at:at + n, h * G:(h + 1) * G].double().reshape(n * G, hd)
            w = (q @ kh.T.contiguous() * hd ** -0.5).masked_fill(~sees.repeat_interleave(G, 0), -math.inf)
            out[at:at + n, h * G:(h + 1) * G] = (torch.softmax(w, -1) @ vh).view(n, G, hd)
        at += n
    if s["y"] is not None:
        out /= 1 + torch.exp(-s["y"][:, :, 1].double())
    return out


def _exact_sample(s, c):
    z = s["z"].float().cpu().numpy().astype(np.float64)
    col = {k: s[k].cpu().numpy() for k in ("temp", "k", "p", "mp", "u")}
    idx, prob = [], []
    for i, row in enumerate(z):
        T = float(col["temp"][i])
        top = int(np.argmax(row))
        if T <= 0:
            idx.append(top)
            prob.append(1.0)
            continue
        w = np.exp((row - row[top]) / T)
        order = np.lexsort((np.arange(row.size), -row))
        if 0 < col["k"][i] < row.size:
            order = order[:int(col["k"][i])]
        if col["p"][i] < 1:
            before = np.concatenate([[0.0], np.cumsum(w[order])])
            order = order[:max(1, int((before[:-1] < float(col["p"][i]) * before[-1]).sum()))]
        keep = np.sort(order[w[order] >= float(col["mp"][i])])
        mass = np.cumsum(w[keep])
        j = min(int(np.searchsorted(mass, float(col["u"][i]) * mass[-1], side="right")), keep.size - 1)
        idx.append(int(keep[j]))
        prob.append(w[keep[j]] / mass[-1])
    return {"idx": torch.tensor(idx, dtype=torch.int32), "prob": torch.tensor(prob, dtype=torch.float64)}


def _exact_accept(s, c):
    par, tok, smp, table = (s[k].cpu().numpy() for k in ("parents", "toks", "samples", "table"))
    ctx, rows = _lens(c)
    page, at = c["page"], 0
    path = np.full((c["B"], c["R"]), -1, np.int32)
    n, nxt, moves = [], [], []
    for b, (a, m) in enumerate(zip(ctx, rows)):
        p, t, q = par[at:at + m], tok[at:at + m], smp[at:at + m]
        walk = [0]
        while True:
            fit = np.flatnonzero((p == walk[-1]) & (t == q[walk[-1]]))
            if not fit.size:
                break
            walk.append(int(fit[0]))
        path[b, :len(walk)] = walk
        n.append(len(walk))
        nxt.append(int(q[walk[-1]]))
        for d, j in enumerate(walk):
            moves.append((table[b][(a + j) // page], (a + j) % page, table[b][(a + d) // page], (a + d) % page))
        at += m
    mv = torch.tensor(np.array(moves, np.int64), device=DEV)
    k, v = s["k"].clone(), s["v"].clone()
    for new, old in ((k, s["k"]), (v, s["v"])):
        new[:, mv[:, 2], :, mv[:, 3]] = old[:, mv[:, 0], :, mv[:, 1]]
    i32 = lambda x: torch.tensor(np.asarray(x, np.int32))  # noqa: E731
    return {"path": i32(path), "n": i32(n), "next": i32(nxt), "ctx": i32(np.array(ctx) + n), "k": k, "v": v}


def exact(case, seed):
    return {"append": _exact_append, "attn": _exact_attn, "sample": _exact_sample,
            "accept": _exact_accept}[case["op"]](prepare(case, seed), case)
