"""The calls of a serving step between its matrix products, with inputs, work and plain forms.

A step of several requests lays its new rows and cache pages out
(launch_page_plan), turns Q and K by their positions and writes K and V into
the cache (launch_rope_cache), lets the new rows attend to the cache
(launch_paged_attention) and draws the next tokens from the logits
(launch_sample). Sizes are those of the 27B shapes that the benchmark uses
(QKV 7168: 5120 query values and two times 1024, in heads of 256 or 128;
vocabulary 248320) and what lies around them.
"""
import math
import os
import random
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "bonsai-ternary-fast_amd")

own = False  # the plain forms; true: the library's calls

EPS = 1e-6
TREE = 64  # nodes of a drafted tree at most; more new tokens are a prompt
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One decoded token each of 8 requests: the smallest step's plan, latency alone.
        {"name": "plan_decode", "op": "plan", "S": 8, "page": 64, "ctx": 4096, "new": 1, "tree": False, "spare": 1.0},
        # 256 requests with drafted trees; the pool runs out for the last of them.
        {"name": "plan_trees", "op": "plan", "S": 256, "page": 16, "ctx": 32768, "new": 48, "tree": True, "spare": 0.8},
        # One token's Q, K and V: norms, a quarter of the head turned in halves.
        {"name": "rope_token", "op": "rope", "T": 1, "H": 20, "HK": 4, "D": 256, "rot": 64, "layout": "half",
         "norm": True, "far": 32768, "page": 64, "type": "f16"},
        # A prompt's rows, neighbouring pairs over the whole head, far positions.
        {"name": "rope_prompt", "op": "rope", "T": 2048, "H": 40, "HK": 8, "D": 128, "rot": 128, "layout": "pairs",
         "norm": False, "far": 1000000, "page": 16, "type": "bf16"},
        # One token of one request over a short cache: latency.
        {"name": "attn_token", "op": "attn", "S": 1, "H": 20, "HK": 4, "D": 256, "page": 64, "ctx": 4096, "new": 1,
         "tree": False, "type": "f16"},
        # One token each of 32 requests of very different lengths: the cache's bytes.
        {"name": "attn_batch", "op": "attn", "S": 32, "H": 20, "HK": 4, "D": 256, "page": 64, "ctx": 32768, "new": 1,
         "tree": False, "type": "f16"},
        # Trees of up to 64 drafted tokens of 8 requests.
        {"name": "attn_trees", "op": "attn", "S": 8, "H": 40, "HK": 8, "D": 128, "page": 16, "ctx": 16384, "new": 64,
         "tree": True, "type": "bf16"},
        # A piece of a prompt over what is there already: products.
        {"name": "attn_prompt", "op": "attn", "S": 1, "H": 20, "HK": 4, "D": 256, "page": 64, "ctx": 6143, "new": 2048,
         "tree": False, "type": "f16"},
        # One token from the whole vocabulary.
        {"name": "sample_token", "op": "sample", "M": 1, "V": 248320, "pad": 0},
        # The tokens of 48 requests, each with its own settings.
        {"name": "sample_batch", "op": "sample", "M": 48, "V": 248320, "pad": 0},
        # Many rows of a smaller vocabulary of an odd size, rows padded.
        {"name": "sample_odd", "op": "sample", "M": 130, "V": 50257, "pad": 7},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "rope", "attn", "attn", "attn", "sample", "sample"])
    if op == "plan":
        tree = rng.random() < 0.5
        return {"op": op, "S": _spread(rng, 1, 256), "page": rng.choice([16, 32, 64, 128, 256]),
                "ctx": _spread(rng, 64, 32768), "new": _spread(rng, 1, TREE if tree else 200), "tree": tree,
                "spare": rng.choice([0.6, 1.0, 1.5])}
    heads = rng.choice([(20, 4, 256), (40, 8, 128), (16, 16, 64), (8, 1, 128), (14, 2, 64), (24, 4, 256), (32, 8, 128)])
    H, HK, D = heads
    page, kind = rng.choice([16, 32, 64, 128, 256]), rng.choice(["f16", "bf16"])
    if op == "rope":
        return {"op": op, "T": _spread(rng, 1, 2048), "H": H, "HK": HK, "D": D,
                "rot": rng.choice([D, D // 2, D // 4, D - 10]), "layout": rng.choice(["half", "pairs"]),
                "norm": rng.random() < 0.5, "far": _spread(rng, 4096, 1000000), "page": page, "type": kind}
    if op == "attn":
        how = rng.choice(["token", "token", "tree", "prompt"])
        c = {"op": op, "S": 1, "H": H, "HK": HK, "D": D, "page": page, "ctx": 0, "new": 1, "tree": how == "tree",
             "type": kind}
        if how == "token":
            c.update(S=_spread(rng, 1, 32), ctx=_spread(rng, 64, 32768))
        elif how == "tree":
            c.update(S=_spread(rng, 1, 8), ctx=_spread(rng, 64, 16384), new=_spread(rng, 2, TREE))
        else:
            c.update(ctx=rng.choice([0, _spread(rng, 64, 6000)]), new=_spread(rng, 65, 2048 if H * D <= 5120 else 1600))
        return c
    V = rng.choice([248320, _spread(rng, 300, 248320)])
    return {"op": op, "M": _spread(rng, 1, 48 if V > 60000 else 130), "V": V, "pad": rng.choice([0, 1, 4])}


# ---- the sizes that a case leaves open: from the case alone, so that work() knows them ----
def _lengths(c):
    """(tokens in the cache, new tokens) of each request: of very different lengths, the first the longest."""
    rng = random.Random("%s" % sorted((k, v) for k, v in c.items() if k != "name"))
    ctx, new = [c["ctx"]], [c["new"]]
    for _ in range(c["S"] - 1):
        ctx.append(rng.randint(c["ctx"] // 16, c["ctx"]))
        new.append(rng.randint(max(1, c["new"] // 4), c["new"]))
    return ctx, new


def _pages_of(tokens, page):
    return -(-tokens // page)


def _plan_sizes(c):
    ctx, new = _lengths(c)
    held = [_pages_of(n, c["page"]) for n in ctx]
    need = [max(0, _pages_of(a + b, c["page"]) - h) for a, b, h in zip(ctx, new, held)]
    return ctx, new, held, need, int(sum(need) * c["spare"])


# ---- inputs (plain torch, from the seed alone) ----
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _zero(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _parents(seed, new, T):
    """Drafted trees: each node hangs on one of the few before it (-1: on the last token of the cache)."""
    rng = np.random.default_rng(seed)
    i = np.concatenate([np.arange(n) for n in new])
    back = rng.integers(1, 6, size=i.size)
    return _ints(np.maximum(i - back, -1).tolist() + [-1] * (T - i.size))


def _table(g, held, ldt, pages):
    """Pages handed out at random: (table, free list)."""
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    h = torch.tensor(held, device="cuda")
    j = torch.arange(ldt, device="cuda")
    at = (torch.cumsum(h, 0) - h)[:, None] + j
    table = torch.where(j < h[:, None], perm[at.clamp(max=pages - 1)], -1).contiguous()
    return table, perm[sum(held):].contiguous()


def _turns(c):
    """Turns per position of each pair, in 64 bits (base 1e7)."""
    i = np.arange(c["rot"] // 2)
    return 1e7 ** (-2.0 * i / c["rot"]) / (2 * math.pi)


def _prepare_plan(c, seed):
    g = _gen(seed)
    ctx, new, held, need, spare = _plan_sizes(c)
    T = sum(new) + 5  # a captured step's buffers hold more rows than this step has
    ldt = max(h + n for h, n in zip(held, need)) + 1
    pages = sum(held) + max(spare, 1)
    table, free = _table(g, held, ldt, pages)
    return {"ctx": _ints(ctx), "new": _ints(new), "held": _ints(held), "table": table, "free": free, "T": T,
            "ldt": ldt, "pages": pages, "n_free": _ints([spare]),
            "parent": _parents(seed, new, T) if c["tree"] else None,
            "row0": _ints([0] * (c["S"] + 1)), "kv_len": _ints([0] * c["S"]), "held_out": _ints([0] * c["S"]),
            "n_free_out": _ints([0]), "pos": _ints([-7] * T), "slot": _ints([-7] * T),
            "bits": torch.full((T,), -7, dtype=torch.int64, device="cuda") if c["tree"] else None}


def _prepare_rope(c, seed):
    g = _gen(seed)
    T, H, HK, D, P = c["T"], c["H"], c["HK"], c["D"], c["page"]
    pages = _pages_of(T, P) + 2
    qkv = torch.randn((T, (H + 2 * HK) * D), generator=g, device="cuda")
    norm = lambda: 1.0 + 0.1 * torch.randn(D, generator=g, device="cuda") if c["norm"] else None  # noqa: E731
    cache = lambda: torch.randn((pages, HK, P, D), generator=g, device="cuda").to(TYPES[c["type"]])  # noqa: E731
    return {"qkv": qkv, "qn": norm(), "kn": norm(), "turns": torch.from_numpy(_turns(c)).cuda(), "mscale": 1.1,
            "pos": torch.randint(0, c["far"], (T,), generator=g, device="cuda", dtype=torch.int32),
            "slot": torch.randperm(pages * P, generator=g, device="cuda")[:T].to(torch.int32),
            "k": cache(), "v": cache(), "pages": pages, "q": _zero(T, H * D, dtype=TYPES[c["type"]])}


def _prepare_attn(c, seed):
    g = _gen(seed)
    H, HK, D, P, S = c["H"], c["HK"], c["D"], c["page"], c["S"]
    ctx, new = _lengths(c)
    kv = [a + b for a, b in zip(ctx, new)]
    T, held = sum(new), [_pages_of(n, P) for n in kv]
    pages, ldt = sum(held) + 3, max(held)
    table, _ = _table(g, held, ldt, pages)
    cache = lambda: torch.randn((pages, HK, P, D), generator=g, device="cuda", dtype=torch.float32).to(TYPES[c["type"]])  # noqa: E731
    # queries of rows of their own sizes: flat and sharp softmax rows
    q = torch.randn((T, H * D), generator=g, device="cuda") * torch.exp(0.5 * torch.randn((T, 1), generator=g, device="cuda"))
    st = {"q": q.to(TYPES[c["type"]]), "k": cache(), "v": cache(), "pages": pages, "table": table, "ldt": ldt, "T": T,
          "row0": _ints([0] + np.cumsum(new).tolist()), "kv_len": _ints(kv), "N": max(new), "L": max(kv),
          "scale": D ** -0.5, "out": _zero(T, H * D), "bits": None}
    if c["tree"]:
        p = _parents(seed, new, T)
        st["bits"] = _row_bits(p, st["row0"].long(), S, torch.ones(S, dtype=torch.bool, device="cuda"))[1]
    return st


def _prepare_sample(c, seed):
    g = _gen(seed)
    M, V = c["M"], c["V"]
    x = 2.5 * torch.randn((M, V + c["pad"]), generator=g, device="cuda")
    # a few tokens that stand out, as a trained model's rows have them
    at = torch.randint(0, V, (M, 12), generator=g, device="cuda")
    x.scatter_(1, at, 9.0 + 3.0 * torch.rand((M, 12), generator=g, device="cuda"))
    pick = lambda v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (M,), generator=g, device="cuda")]  # noqa: E731
    return {"x": x, "temp": pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3]), "top_k": pick([0, 0, 20, 50, 1000]).to(torch.int32),
            "top_p": pick([1.0, 1.0, 0.95, 0.9, 0.5]), "min_p": pick([0.0, 0.0, 0.05, 0.01]),
            "u": torch.rand((M,), generator=g, device="cuda"), "token": _ints([0] * M), "logp": _zero(M)}


def prepare(case, seed):
    st = {"plan": _prepare_plan, "rope": _prepare_rope, "attn": _prepare_attn, "sample": _prepare_sample}[case["op"]](case, seed)
    st["c"] = case
    return st


# ---- the plain forms ----
def _row_bits(parent, row0, S, served):
    """(depth, bits of ancestors and self) of every row, from the closure of the parents' relation."""
    T = parent.numel()
    t = torch.arange(T, device="cuda")
    s = torch.searchsorted(row0[1:].contiguous(), t, right=True).clamp(max=S - 1)
    i, n = t - row0[s], (row0[1:] - row0[:-1])[s]
    node = (t < row0[S]) & (n <= TREE) & served[s] & (i < TREE)
    p = parent.long()
    p = torch.where((p >= 0) & (p < i), p, -1)
    up = torch.zeros((S, TREE, TREE), device="cuda")
    r = node & (p >= 0)
    up[s[r], i[r], p[r]] = 1.0
    up = up + torch.eye(TREE, device="cuda")
    up = (up @ up > 0).float()  # paths of up to 2, 4, ... 64 steps
    up = (up @ up > 0).float()
    up = (up @ up > 0).float()
    up = (up @ up > 0).float()
    up = (up @ up > 0).float()
    up = (up @ up > 0)
    bits = (up.long() << torch.arange(TREE, device="cuda")).sum(-1)
    depth = up.sum(-1) - 1
    k = i.clamp(0, TREE - 1)
    return torch.where(node, depth[s, k], i), torch.where(node, bits[s, k], 0)


def _plain_plan(st):
    c, P, T = st["c"], st["c"]["page"], st["T"]
    S, ldt = c["S"], st["ldt"]
    ctx, new, h = st["ctx"].long(), st["new"].long(), st["held"].long()
    n_free = st["n_free"].long()
    n = new.clamp(min=0)
    end = torch.cumsum(n, 0)
    total = (ctx + new + P - 1) // P
    sound = (ctx >= 0) & (new >= 0) & (h >= 0) & (h <= ldt) & (ctx <= h * P) & (end <= T) & (total <= ldt)
    need = torch.where(sound, (total - h).clamp(min=0), 0)
    got = torch.cumsum(need, 0)
    served = sound & ((need == 0) | (got <= n_free))
    need = torch.where(served, need, 0)
    off = got - need
    j = torch.arange(ldt, device="cuda") - h[:, None]
    at = (n_free - 1 - off[:, None] - j).clamp(0, st["free"].numel() - 1)
    st["table"].copy_(torch.where((j >= 0) & (j < need[:, None]), st["free"][at], st["table"]))
    st["held_out"].copy_(h + need)
    st["kv_len"].copy_(torch.where(served, ctx + new, 0))
    st["n_free_out"].copy_(n_free - need.sum())
    row0 = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), end]).clamp(max=T)
    st["row0"].copy_(row0)
    t = torch.arange(T, device="cuda")
    s = torch.searchsorted(row0[1:].contiguous(), t, right=True).clamp(max=S - 1)
    live, i = t < row0[S], t - row0[s]
    at = ctx[s] + i
    page = st["table"].long()[s, (at // P).clamp(0, ldt - 1)]
    good = served[s] & (page >= 0) & (page < st["pages"])
    depth = i
    if st["parent"] is not None:
        depth, bits = _row_bits(st["parent"], row0, S, served)
        st["bits"].copy_(torch.where(live, bits, st["bits"]))
    st["pos"].copy_(torch.where(live, torch.where(served[s], ctx[s] + depth, 0).int(), st["pos"]))
    st["slot"].copy_(torch.where(live, torch.where(good, page * P + at % P, -1).int(), st["slot"]))


def _turned(x, st, norm):
    """Heads [T][n][D] of x in 32 bits: normed, then turned by their positions."""
    c = st["c"]
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    ang = torch.remainder(st["pos"].double()[:, None] * st["turns"], 1.0) * (2 * math.pi)
    cos, sin = ((f(ang) * st["mscale"]).float()[:, None] for f in (torch.cos, torch.sin))
    r = c["rot"]
    if c["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., r:]], -1)


def _plain_rope(st):
    c, t = st["c"], TYPES[st["c"]["type"]]
    T, H, HK, D, P = c["T"], c["H"], c["HK"], c["D"], c["page"]
    x = st["qkv"].view(T, H + 2 * HK, D)
    page, at = st["slot"].long() // P, st["slot"].long() % P
    st["q"].copy_(_turned(x[:, :H], st, st["qn"]).to(t).view(T, H * D))
    st["k"][page, :, at] = _turned(x[:, H: H + HK], st, st["kn"]).to(t)
    st["v"][page, :, at] = x[:, H + HK:].to(t)


def _plain_attn(st):
    c = st["c"]
    S, H, HK, D, P, N, L = c["S"], c["H"], c["HK"], c["D"], c["page"], st["N"], st["L"]
    row0, kv = st["row0"].long(), st["kv_len"].long()
    new = row0[1:] - row0[:-1]
    i, j = torch.arange(N, device="cuda"), torch.arange(L, device="cuda")
    row = (row0[:-1, None] + i).clamp(max=st["T"] - 1)  # [S][N]
    page = st["table"].long()[:, j // P].clamp(min=0)  # [S][L]
    k = st["k"][page, :, j % P].float().permute(0, 2, 3, 1).contiguous()  # [S][HK][D][L]
    q = st["q"].float().view(-1, HK, H // HK, D)[row].permute(0, 2, 1, 3, 4).reshape(S, HK, N * (H // HK), D)
    x = (q @ k).view(S, HK, N, H // HK, L) * st["scale"]
    del k
    ctx = (kv - new)[:, None, None]
    seen = j - ctx <= i[:, None]
    if st["bits"] is not None:
        bit = (st["bits"][row][..., None] >> (j - ctx).clamp(0, TREE - 1)) & 1
        seen = (j < ctx) | ((bit == 1) & (j - ctx < TREE))
    seen = (seen & (j < kv[:, None, None]))[:, None, :, None]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    w = x.sum(-1, keepdim=True)
    v = st["v"][page, :, j % P].float()
    v = torch.where((j < kv[:, None])[..., None, None], v, 0.0).permute(0, 2, 1, 3).contiguous()  # [S][HK][L][D]
    o = (x.view(S, HK, -1, L) @ v).view(S, HK, N, H // HK, D)
    o = torch.where(w > 0, o / torch.where(w > 0, w, 1.0), 0.0).permute(0, 2, 1, 3, 4).reshape(S, N, H * D)
    live = i < new[:, None]
    st["out"][row[live]] = o[live]


def _plain_sample(st):
    V = st["c"]["V"]
    x = st["x"][:, :V].double()
    x = torch.where(x.isnan(), -math.inf, x)
    hot = st["temp"] > 0
    xs, idx = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((xs - xs[:, :1]) / torch.where(hot, st["temp"].double(), 1.0)[:, None])
    rank = torch.arange(V, device="cuda")
    k = torch.where(st["top_k"] > 0, st["top_k"], V).clamp(max=V)[:, None]
    w = torch.where(rank < k, w, 0.0)
    full = torch.cumsum(w, 1)
    p = st["top_p"].double()[:, None]
    keep = (p >= 1) | (rank == 0) | (full - w < p * full[:, -1:])
    keep = keep & (w >= st["min_p"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, idx, torch.where(keep, w, 0.0))
    full = torch.cumsum(w, 1)
    total = full[:, -1:]
    tok = (full <= st["u"].double()[:, None] * total).sum(1, keepdim=True)
    last = torch.where(w > 0, rank, 0).amax(1, keepdim=True)
    tok = torch.minimum(tok, last)
    logp = torch.log(w.gather(1, tok) / total)
    st["token"].copy_(torch.where(hot, tok[:, 0], idx[:, 0]))
    st["logp"].copy_(torch.where(hot, logp[:, 0], 0.0))


# ---- the library's calls ----
def _hip():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import btf_hip
    btf_hip.kernels_init(0)
    return btf_hip


def _bytes(n):
    return torch.zeros(max(1, -(-n // 8)), dtype=torch.int64, device="cuda")


def _cache(hip, c, st):
    HK, P, D = c["HK"], c["page"], c["D"]
    return hip.KvCache(st["k"], st["v"], hip.CacheType[c["type"]], P, HK, D, st["pages"], HK * P * D, P * D, D)


def _bind(st):
    """What a program keeps from step to step: the argument structs and the workspace."""
    hip, c = _hip(), st["c"]
    if c["op"] == "plan":
        a = hip.PagePlan(S=c["S"], T=st["T"], page=c["page"], pages=st["pages"], ldt=st["ldt"], ctx=st["ctx"],
                         n_new=st["new"], parent=st["parent"], free=st["free"], n_free=st["n_free"], held=st["held"],
                         table=st["table"], n_free_out=st["n_free_out"], held_out=st["held_out"], row0=st["row0"],
                         kv_len=st["kv_len"], pos=st["pos"], slot=st["slot"], tree=st["bits"])
        return lambda s: hip.launch_page_plan(a, s)
    if c["op"] == "rope":
        H, HK, D = c["H"], c["HK"], c["D"]
        q, k, v = (st["qkv"][:, n * D:] for n in (0, H, H + HK))
        ld = (H + 2 * HK) * D
        a = hip.RopeCache(T=c["T"], heads=H, q=q, ldq=ld, k=k, ldk=ld, v=v, ldv=ld, q_norm=st["qn"], k_norm=st["kn"],
                          eps=EPS, n_rot=c["rot"], layout=hip.RopeLayout[c["layout"]], turns=st["turns"],
                          mscale=st["mscale"], pos=st["pos"], slot=st["slot"], rows=None, q_out=st["q"], ldqo=H * D)
        kv = _cache(hip, c, st)
        return lambda s: hip.launch_rope_cache(a, kv, s)
    if c["op"] == "attn":
        H, D = c["H"], c["D"]
        kv = _cache(hip, c, st)
        ws = _bytes(hip.paged_attention_ws_bytes(c["S"], st["T"], H, kv))
        a = hip.PagedAttention(S=c["S"], T=st["T"], heads=H, q=st["q"], ldq=H * D, table=st["table"], ldt=st["ldt"],
                               row0=st["row0"], kv_len=st["kv_len"], tree=st["bits"], scale=st["scale"],
                               out=st["out"], ldo=H * D, ws=ws)
        return lambda s: hip.launch_paged_attention(a, kv, s)
    M, V = c["M"], c["V"]
    a = hip.Sampling(M=M, V=V, logits=st["x"], ldl=V + c["pad"], temperature=st["temp"], top_k=st["top_k"],
                     top_p=st["top_p"], min_p=st["min_p"], u=st["u"], token=st["token"], logprob=st["logp"],
                     ws=_bytes(hip.sample_ws_bytes(M, V)))
    return lambda s: hip.launch_sample(a, s)


def _outputs(st):
    names = {"plan": ("table", "held_out", "n_free_out", "row0", "kv_len", "pos", "slot", "bits"),
             "rope": ("q", "k", "v"), "attn": ("out",), "sample": ("token", "logp")}[st["c"]["op"]]
    return {n: st[n] for n in names if st[n] is not None}


def run(st):
    if own:
        if "call" not in st:
            st["call"] = _bind(st)
        st["call"](torch.cuda.current_stream().cuda_stream)
    else:
        {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn, "sample": _plain_sample}[st["c"]["op"]](st)
    return _outputs(st)


# ---- what a pass cannot do without ----
def work(case):
    c = case
    if c["op"] == "plan":
        ctx, new, held, need, spare = _plan_sizes(c)
        S, T = c["S"], sum(new)
        return {"bytes": 4 * (3 * S + min(spare, sum(need))) + 4 * (3 * S + 2 + min(spare, sum(need))) + 8 * T + (12 * T if c["tree"] else 0),
                "flops": 4 * T}
    if c["op"] == "rope":
        n = c["T"] * (c["H"] + 2 * c["HK"]) * c["D"]
        turned = c["T"] * (c["H"] + c["HK"])
        return {"bytes": 6 * n + 8 * c["T"] + 4 * c["rot"] + (8 * c["D"] if c["norm"] else 0),
                "flops": 3 * turned * c["rot"] + (4 * turned * c["D"] if c["norm"] else 0)}
    if c["op"] == "attn":
        ctx, new = _lengths(c)
        kv = sum(ctx) + sum(new)
        # a tree's rows see the cache and, of their own request's rows, at most their ancestors; a prompt's those before them
        pairs = sum(n * a + (n if c["tree"] else n * (n + 1) // 2) for a, n in zip(ctx, new))
        return {"bytes": 4 * c["HK"] * c["D"] * kv + 6 * c["H"] * c["D"] * sum(new) + 4 * kv // c["page"],
                "flops": 4 * c["H"] * c["D"] * pairs}
    return {"bytes": 4 * c["M"] * c["V"] + 28 * c["M"], "flops": 4 * c["M"] * c["V"]}


# ---- the definitions in 64 bits, on the host or row by row ----
def _exact_plan(c, st):
    P, T, S = c["page"], st["T"], c["S"]
    get = lambda n: st[n].cpu().numpy().astype(np.int64)  # noqa: E731
    ctx, new, held, table, free = get("ctx"), get("new"), get("held").copy(), get("table").copy(), get("free")
    out = {n: get(n).copy() for n in ("row0", "kv_len", "pos", "slot")}
    bits = get("bits").astype(np.uint64) if st["bits"] is not None else None
    parent = get("parent") if st["parent"] is not None else None
    stack = free[: int(st["n_free"][0])].tolist()
    blocked, row = False, 0
    for s in range(S):
        n = int(new[s])
        out["row0"][s] = min(row, T)
        total = -(-(int(ctx[s]) + n) // P)
        need = max(0, total - int(held[s]))
        ok = total <= st["ldt"] and row + n <= T
        if ok and need and (blocked or need > len(stack)):
            ok, blocked = False, True
        if ok:
            for k in range(need):
                table[s, held[s] + k] = stack.pop()
            held[s] += need
        out["kv_len"][s] = ctx[s] + n if ok else 0
        depth, mask = [], []
        for i in range(n):
            p = int(parent[row + i]) if parent is not None and n <= TREE else i - 1
            depth.append(depth[p] + 1 if p >= 0 else 0)
            mask.append((mask[p] if p >= 0 else 0) | 1 << i)
            at = int(ctx[s]) + i
            out["pos"][row + i] = ctx[s] + depth[i] if ok else 0
            out["slot"][row + i] = table[s, at // P] * P + at % P if ok else -1
            if bits is not None:
                bits[row + i] = mask[i] if ok and n <= TREE else 0
        row += n
    out["row0"][S] = min(row, T)
    out.update(table=table, held_out=held, n_free_out=np.array([len(stack)]))
    out = {n: torch.from_numpy(v).to(torch.int32) for n, v in out.items()}
    if bits is not None:
        out["bits"] = torch.from_numpy(bits.view(np.int64))
    return out


def _exact_rope(c, st):
    T, H, HK, D, P, r = c["T"], c["H"], c["HK"], c["D"], c["page"], c["rot"]
    x = st["qkv"].double().cpu().numpy().reshape(T, H + 2 * HK, D).copy()
    for norm, lo, hi in ((st["qn"], 0, H), (st["kn"], H, H + HK)):
        if norm is not None:
            h = x[:, lo:hi]
            x[:, lo:hi] = h / np.sqrt(np.mean(h * h, -1, keepdims=True) + EPS) * norm.double().cpu().numpy()
    t = st["pos"].cpu().numpy().astype(np.float64)[:, None] * st["turns"].cpu().numpy()
    turn = np.exp(2j * np.pi * (t - np.floor(t)))[:, None] * st["mscale"]
    first = slice(0, r // 2) if c["layout"] == "half" else slice(0, r, 2)
    second = slice(r // 2, r) if c["layout"] == "half" else slice(1, r, 2)
    h = x[:, : H + HK]
    z = (h[..., first] + 1j * h[..., second]) * turn
    h[..., first], h[..., second] = z.real, z.imag
    k, v = (st[n].double().cpu().numpy() for n in ("k", "v"))
    slot = st["slot"].cpu().numpy()
    k[slot // P, :, slot % P] = x[:, H: H + HK]
    v[slot // P, :, slot % P] = x[:, H + HK:]
    return {"q": torch.from_numpy(x[:, :H].reshape(T, H * D).copy()), "k": torch.from_numpy(k), "v": torch.from_numpy(v)}


def _exact_attn(c, st):
    H, HK, D, P = c["H"], c["HK"], c["D"], c["page"]
    G = H // HK
    row0, kv = st["row0"].tolist(), st["kv_len"].tolist()
    out = torch.zeros((st["T"], H * D), dtype=torch.float64, device="cuda")
    for s in range(c["S"]):
        a, b, L = row0[s], row0[s + 1], kv[s]
        ctx = L - (b - a)
        pages = st["table"][s, : _pages_of(L, P)].long()
        k = st["k"][pages].double().transpose(0, 1).reshape(HK, -1, D)[:, :L]
        v = st["v"][pages].double().transpose(0, 1).reshape(HK, -1, D)[:, :L]
        seen = torch.ones((b - a, L), dtype=torch.bool, device="cuda")
        if st["bits"] is not None:
            seen[:, ctx:] = (st["bits"][a:b, None] >> torch.arange(b - a, device="cuda")) & 1 == 1
        else:
            seen[:, ctx:] = torch.ones((b - a, b - a), device="cuda").tril() > 0
        for h in range(H):
            x = st["q"][a:b, h * D: (h + 1) * D].double() @ k[h // G].T * st["scale"]
            x = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
            out[a:b, h * D: (h + 1) * D] = x @ v[h // G]
    return {"out": out}


def _exact_sample(c, st):
    x = st["x"][:, : c["V"]].double().cpu().numpy()
    par = {n: st[n].double().cpu().numpy() for n in ("temp", "top_k", "top_p", "min_p", "u")}
    token, logp = np.zeros(c["M"], np.int64), np.zeros(c["M"])
    for m in range(c["M"]):
        best = int(np.argmax(x[m]))
        if par["temp"][m] <= 0:
            token[m] = best
            continue
        w = np.exp((x[m] - x[m, best]) / par["temp"][m])
        order = np.argsort(-x[m], kind="stable")
        if par["top_k"][m] > 0:
            order = order[: int(par["top_k"][m])]
        if par["top_p"][m] < 1:
            run_ = np.cumsum(w[order])
            order = order[: int(np.searchsorted(run_, par["top_p"][m] * run_[-1])) + 1]
        order = np.sort(order[w[order] >= par["min_p"][m]])
        run_ = np.cumsum(w[order])
        at = min(int(np.searchsorted(run_, par["u"][m] * run_[-1], side="right")), order.size - 1)
        token[m], logp[m] = order[at], math.log(w[order[at]] / run_[-1])
    return {"token": torch.from_numpy(token).to(torch.int32), "logp": torch.from_numpy(logp)}


def exact(case, seed):
    st = prepare(case, seed)
    return {"plan": _exact_plan, "rope": _exact_rope, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](case, st)
