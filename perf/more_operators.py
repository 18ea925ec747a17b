"""Operators of a server whose requests share what they can, with inputs, work and plain forms.

Requests that go on from the same tokens share the cache's pages
(launch_page_fork, launch_page_copy and launch_page_free, as a set of samples
or a beam needs them), tokens that stay are moved together (launch_cache_move:
the accepted path of a drafted tree, a cache that drops tokens), a shared prefix
is attended to once for all rows that see it (launch_shared_attention), and the
requests' own low-rank adapters come on top of the projection that they share
(launch_lora). Sizes are those of the 27B shapes that the benchmark uses (width
5120, FFN 17408, QKV 7168 as 5120 + 1024 + 1024) and what lies around them.
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

TREE = 64  # nodes of a drafted tree at most
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # Four samples from one prompt, begun and given back: the smallest call, latency.
        {"name": "fork_samples", "op": "fork", "S": 1, "F": 4, "HK": 4, "D": 256, "page": 64, "ctx": 1000, "layers": 1,
         "type": "f16"},
        # 64 samples of 8 prompts with the pages that end inside, over 16 layers: copies.
        {"name": "fork_batch", "op": "fork", "S": 8, "F": 64, "HK": 4, "D": 256, "page": 64, "ctx": 4096, "layers": 16,
         "type": "f16"},
        # The accepted path of 8 drafted trees, moved together in 16 layers.
        {"name": "move_trees", "op": "move", "S": 8, "HK": 4, "D": 256, "page": 64, "ctx": 4096, "new": 48, "list": False,
         "other": False, "layers": 16, "type": "f16"},
        # Half of the tokens of long caches stay, in their own pages.
        {"name": "move_long", "op": "move", "S": 8, "HK": 8, "D": 128, "page": 16, "ctx": 16384, "new": 0, "list": True,
         "other": False, "layers": 2, "type": "bf16"},
        # Four samples soon after the end of a prompt of an odd length: latency.
        {"name": "shared_samples", "op": "shared", "S": 4, "groups": 1, "H": 20, "HK": 4, "D": 256, "page": 64,
         "shared": 1000, "own": 40, "new": 1, "tree": False, "type": "f16"},
        # 64 requests behind one long instruction, each with a conversation of its own.
        {"name": "shared_batch", "op": "shared", "S": 64, "groups": 1, "H": 20, "HK": 4, "D": 256, "page": 64,
         "shared": 16384, "own": 1000, "new": 1, "tree": False, "type": "f16"},
        # Drafted trees of 24 requests behind three prefixes.
        {"name": "shared_trees", "op": "shared", "S": 24, "groups": 3, "H": 40, "HK": 8, "D": 128, "page": 16,
         "shared": 6000, "own": 2000, "new": 16, "tree": True, "type": "bf16"},
        # Many samples of two long prompts: the largest.
        {"name": "shared_large", "op": "shared", "S": 128, "groups": 2, "H": 32, "HK": 8, "D": 128, "page": 64,
         "shared": 16384, "own": 500, "new": 1, "tree": False, "type": "bf16"},
        # One token's output projection: latency.
        {"name": "lora_token", "op": "lora", "S": 1, "new": 1, "K": 5120, "N": 5120, "N2": 0, "segs": 1, "mode": "add",
         "adapters": 4, "rank": 16, "pad": 0, "type": "f16"},
        # Q, K and V of 64 requests with adapters of many ranks, some with none.
        {"name": "lora_batch", "op": "lora", "S": 64, "new": 1, "K": 5120, "N": 5120, "N2": 1024, "segs": 3, "mode": "add",
         "adapters": 100, "rank": 64, "pad": 0, "type": "bf16"},
        # Gate and up of 32 requests, with the activation behind them.
        {"name": "lora_gateup", "op": "lora", "S": 32, "new": 1, "K": 5120, "N": 17408, "N2": 17408, "segs": 2,
         "mode": "swiglu", "adapters": 32, "rank": 32, "pad": 0, "type": "f16"},
        # Three prompts of odd lengths through down: the longest sums, most rows.
        {"name": "lora_prompt", "op": "lora", "S": 3, "new": 2048, "K": 17408, "N": 5120, "N2": 0, "segs": 1, "mode": "add",
         "adapters": 8, "rank": 64, "pad": 4, "type": "bf16"},
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], even over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["fork", "move", "shared", "shared", "shared", "lora", "lora", "lora"])
    H, HK, D = rng.choice([(20, 4, 256), (40, 8, 128), (16, 16, 64), (8, 1, 128), (14, 2, 64), (24, 4, 256), (32, 8, 128)])
    page, kind = rng.choice([16, 32, 64, 128, 256]), rng.choice(["f16", "bf16"])
    if op == "fork":
        S = _spread(rng, 1, 8)
        return {"op": op, "S": S, "F": _spread(rng, 1, 64), "HK": HK, "D": D, "page": min(page, 64),
                "ctx": _spread(rng, 20, 4096), "layers": rng.choice([1, 2, 16]) if HK * D <= 1024 else 1, "type": kind}
    if op == "move":
        c = {"op": op, "S": _spread(rng, 1, 8), "HK": HK, "D": D, "page": page, "ctx": _spread(rng, 64, 16384), "new": 0,
             "list": rng.random() < 0.5, "other": rng.random() < 0.3, "layers": 1, "type": kind}
        if not c["list"]:
            c.update(S=_spread(rng, 1, 32), ctx=_spread(rng, 64, 2048), new=_spread(rng, 2, TREE), other=False,
                     layers=rng.choice([1, 4, 16]) if HK * D <= 1024 else 4)
        return c
    if op == "shared":
        tree = rng.random() < 0.4
        S = _spread(rng, 2, 24 if tree else 96)
        return {"op": op, "S": S, "groups": min(S, rng.choice([1, 1, 2, 3, 5])), "H": H, "HK": HK, "D": D, "page": page,
                "shared": _spread(rng, 100, 16384 if not tree else 6000), "own": _spread(rng, 1, 1000),
                "new": _spread(rng, 2, 16) if tree else 1, "tree": tree, "type": kind}
    mode, segs = rng.choice([("add", 1), ("add", 3), ("swiglu", 2)])
    K, N = _spread(rng, 512, 17408, 32), _spread(rng, 64, 17408)
    c = {"op": op, "S": _spread(rng, 1, 64), "new": 1, "K": K, "N": N,
         "N2": 0 if segs == 1 else N if segs == 2 else max(1, N // 5), "segs": segs, "mode": mode, "adapters": _spread(rng, 1, 64),
         "rank": rng.choice([8, 16, 32, 64] if K + N * segs > 20000 else [8, 16, 32, 64, 128]), "pad": rng.choice([0, 4, 20]),
         "type": kind}
    how = rng.choice(["token", "token", "few", "prompt"])
    if how == "few":
        c.update(new=_spread(rng, 2, 40), S=_spread(rng, 1, 16))
    elif how == "prompt":
        c.update(S=rng.randint(1, 4))
        c.update(new=_spread(rng, 64, max(65, min(2048, int(2e8 / c["S"] / (2 * K + 2 * N * segs))))))
    return c


# ---- the sizes that a case leaves open: from the case alone, so that work() knows them ----
def _case_rng(c):
    return random.Random("%s" % sorted((k, v) for k, v in c.items() if k != "name"))


def _pages_of(tokens, page):
    return -(-tokens // page)


def _parts(rng, most, n):
    """n numbers, the first `most`, the others in its upper three quarters."""
    return [most] + [rng.randint(max(1, most // 4), most) for _ in range(n - 1)]


def _fork_sizes(c):
    """(tokens of each prompt, prompt and tokens of each fork): some forks go on from inside, some at a page's end."""
    rng = _case_rng(c)
    ctx = _parts(rng, c["ctx"], c["S"])
    src = [rng.randrange(c["S"]) for _ in range(c["F"])]
    n = [rng.choice([ctx[s], ctx[s], rng.randint(0, ctx[s]), ctx[s] // c["page"] * c["page"]]) for s in src]
    return ctx, src, n


def _move_sizes(c):
    """(tokens before the moved ones, tokens among which some stay) of each request, and how many of these stay."""
    rng = _case_rng(c)
    if c["list"]:
        ctx = _parts(rng, c["ctx"], c["S"])
        base = [rng.randint(0, n // 8) for n in ctx]
        new = [n - b for n, b in zip(ctx, base)]
        return base, new, [n // 2 for n in new]
    base, new = _parts(rng, c["ctx"], c["S"]), _parts(rng, c["new"], c["S"])
    return base, new, [min(n, rng.randint(1, 9)) for n in new]


def _shared_sizes(c):
    """(first request of each group, its prefix; own tokens and new tokens of each request)."""
    rng = _case_rng(c)
    S, n = c["S"], c["groups"]
    cut = sorted(rng.sample(range(1, S), n - 1)) if n > 1 else []
    prefix = _parts(rng, c["shared"], n)
    return [0] + cut + [S], prefix, _parts(rng, c["own"], S), _parts(rng, c["new"], S)


def _lora_sizes(c):
    """(rows of each request, its adapter or -1, rank of each adapter)."""
    rng = _case_rng(c)
    new = _parts(rng, c["new"], c["S"])
    who = [rng.randrange(c["adapters"]) if i == 0 or rng.random() < 0.9 else -1 for i in range(c["S"])]
    ranks = [rng.choice([c["rank"], c["rank"], c["rank"] // 2, rng.randint(1, c["rank"])]) for _ in range(c["adapters"])]
    return new, who, ranks


def _widths(c):
    return [c["N"]] + [c["N2"]] * (c["segs"] - 1)


# ---- inputs (plain torch, from the seed alone) ----
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randn(g, shape, kind):
    return torch.randn(shape, generator=g, device="cuda", dtype=TYPES[kind])


def _starts(n):
    return [0] + np.cumsum(n).tolist()


def _prepare_fork(c, seed):
    g = _gen(seed)
    ctx, src, n = _fork_sizes(c)
    P, S, F, L = c["page"], c["S"], c["F"], c["layers"]
    held = [_pages_of(t, P) for t in ctx] + [0] * F
    pages, ldt = sum(held) + F + 5, max(held) + 1
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    j, h = torch.arange(ldt, device="cuda"), torch.tensor(held, device="cuda")
    at = (torch.cumsum(h, 0) - h)[:, None] + j
    free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    free[: pages - sum(held)] = perm[sum(held):]
    cache = lambda: _randn(g, (L, pages, c["HK"], P, c["D"]), c["type"])  # noqa: E731
    out = lambda: _ints([-7] * F)  # noqa: E731
    return {"table": torch.where(j < h[:, None], perm[at.clamp(max=pages - 1)], -1).contiguous(), "ldt": ldt,
            "pages": pages, "held": h.to(torch.int32), "free": free, "n_free": _ints([pages - sum(held)]),
            "shared": torch.zeros(pages, dtype=torch.int32, device="cuda"), "src": _ints(src),
            "dst": _ints(random.Random(seed).sample(range(S, S + F), F)), "tokens": _ints(n),
            "keep": _ints([2 ** 31 - 1] * S + [0] * F), "got": out(), "from": out(), "to": out(), "count": out(),
            "k": cache(), "v": cache()}


def _prepare_move(c, seed):
    g = _gen(seed)
    base, new, stay = _move_sizes(c)
    P, L, rng = c["page"], c["layers"], random.Random(seed)
    kept = [sorted(rng.sample(range(n), m)) for n, m in zip(new, stay)]
    held = [_pages_of(b + n, P) for b, n in zip(base, new)]
    rows = 2 if c["other"] else 1  # the pages that tokens move to are the request's own, or others
    pages, ldt = rows * sum(held) + 3, max(held)
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    j, h = torch.arange(ldt, device="cuda"), torch.tensor(held, device="cuda")
    at = (torch.cumsum(h, 0) - h)[:, None] + j
    table = lambda k: torch.where(j < h[:, None], perm[(at + k * sum(held)).clamp(max=pages - 1)], -1).contiguous()  # noqa: E731
    cache = lambda: _randn(g, (L, pages, c["HK"], P, c["D"]), c["type"])  # noqa: E731
    st = {"table": table(0), "other": table(1) if c["other"] else None, "ldt": ldt, "pages": pages, "first": _ints(base),
          "kv_len": _ints([-7] * c["S"]), "k": cache(), "v": cache(), "most": max(stay)}
    if c["list"]:
        st.update({"from": _ints([b + t for b, ts in zip(base, kept) for t in ts]), "from0": _ints(_starts(stay))})
    else:  # the path of the accepted node: its bits among its tree's; other rows' trees are others
        row0 = _starts(new)
        bits = np.random.default_rng(seed).integers(0, 2 ** 62, sum(new))
        leaf = [a + rng.randrange(n) for a, n in zip(row0, new)]
        bits[leaf] = [sum(1 << t for t in ts) if ts[-1] < 63 else sum(1 << t for t in ts) - 2 ** 64 for ts in kept]
        st.update({"tree": torch.from_numpy(bits).cuda(), "leaf": _ints(leaf), "T": sum(new)})
    return st


def _prepare_shared(c, seed):
    g = _gen(seed)
    H, HK, D, P, S = c["H"], c["HK"], c["D"], c["page"], c["S"]
    group0, prefix, lone, new = _shared_sizes(c)
    which = np.repeat(np.arange(len(prefix)), np.diff(group0))
    kv = [prefix[w] + a + b for w, a, b in zip(which, lone, new)]
    T, held = sum(new), [_pages_of(n, P) for n in kv]
    whole = [n // P for n in prefix]  # pages that all of the group hold
    ldt, pages = max(held), sum(held) + 3
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    j, h = torch.arange(ldt, device="cuda"), torch.tensor(held, device="cuda")
    at = (torch.cumsum(h, 0) - h)[:, None] + j
    table = torch.where(j < h[:, None], perm[at.clamp(max=pages - 1)], -1)
    lead = torch.tensor(group0[:-1], device="cuda")[torch.from_numpy(which).cuda()]
    all_of = torch.tensor(whole, device="cuda")[torch.from_numpy(which).cuda()]
    table = torch.where(j < all_of[:, None], table[lead], table).contiguous()
    k, v = (_randn(g, (pages, HK, P, D), c["type"]) for _ in range(2))
    for s, w in enumerate(which):  # a page that the prefix ends in is copied, as a fork leaves it
        a, b, n = int(table[group0[w], whole[w]]), int(table[s, whole[w]]), prefix[w] % P
        if n and a != b:
            k[b, :, :n], v[b, :, :n] = k[a, :, :n], v[a, :, :n]
    q = torch.randn((T, H * D), generator=g, device="cuda") * torch.exp(0.5 * torch.randn((T, 1), generator=g, device="cuda"))
    st = {"q": q.to(TYPES[c["type"]]), "k": k, "v": v, "pages": pages, "table": table, "ldt": ldt, "T": T,
          "row0": _ints(_starts(new)), "kv_len": _ints(kv), "N": max(new), "scale": D ** -0.5,
          "LO": max(a + b for a, b in zip(lone, new)), "NG": max(sum(new[a:b]) for a, b in zip(group0, group0[1:])),
          "out": torch.zeros((T, H * D), device="cuda"), "bits": None, "group0": _ints(group0),
          "lead": _ints(group0[:-1]), "shared": _ints(prefix)}
    if c["tree"]:
        rng, rows = np.random.default_rng(seed), []
        for n in new:
            own_rows = []
            for i in range(n):
                p = i - int(rng.integers(1, 4))
                own_rows.append((own_rows[p] if p >= 0 else 0) | 1 << i)
            rows += own_rows
        st["bits"] = torch.tensor(rows, dtype=torch.int64, device="cuda")
    return st


def _prepare_lora(c, seed):
    g = _gen(seed)
    new, who, ranks = _lora_sizes(c)
    T, K, R, ids = sum(new), c["K"], c["rank"], c["adapters"]
    t = TYPES[c["type"]]
    f = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    perm = torch.randperm(ids, generator=g, device="cuda").tolist()  # other adapters for another seed
    st = {"T": T, "row0": _ints(_starts(new)), "adapter": _ints([perm[w] if w >= 0 else -1 for w in who]), "N": max(new),
          "x": f(T, K + c["pad"]), "scale": 0.5 + torch.rand(ids, generator=g, device="cuda"), "ranks": None,
          "a": [(f(ids, R, K) * K ** -0.5).to(t) for _ in _widths(c)], "b": [(0.3 * f(ids, n, R)).to(t) for n in _widths(c)],
          "y": [f(T, n + c["pad"]) for n in _widths(c)], "out": None}
    order = [0] * ids
    for i, p in enumerate(perm):
        order[p] = ranks[i]
    st["ranks"] = _ints(order)
    if c["mode"] == "swiglu":
        st["out"] = torch.zeros((T, c["N"]), device="cuda")
    return st


def prepare(case, seed):
    st = {"fork": _prepare_fork, "move": _prepare_move, "shared": _prepare_shared, "lora": _prepare_lora}[case["op"]](case, seed)
    st["c"] = case
    return st


# ---- the plain forms ----
def _plain_fork(st):
    """Children begun, the page that each prefix ends in copied, and all given back."""
    c, P, ldt, pages = st["c"], st["c"]["page"], st["ldt"], st["pages"]
    src, dst, n = (st[k].long() for k in ("src", "dst", "tokens"))
    held, table, free, count = st["held"].long(), st["table"].long(), st["free"].long(), st["n_free"].long()
    rows = held.numel()
    sound = (src >= 0) & (src < rows) & (dst >= 0) & (dst < rows) & (src != dst) & (n >= 0)
    a, b = src.clamp(0, rows - 1), dst.clamp(0, rows - 1)
    sound = sound & (n <= held[a] * P) & (held[b] == 0)
    sound = sound & ~((b[:, None] == b) & sound).tril(-1).any(1)  # the first fork of a row has it
    need = sound & (n % P != 0)
    upto = torch.cumsum(need, 0)
    ok = sound & (~need | (upto <= count))
    need = need & ok
    whole = n // P
    page = free[(count - upto).clamp(0, pages - 1)]
    j = torch.arange(ldt, device="cuda")
    old = table[a]
    ids = torch.where(j < whole[:, None], old, torch.where((j == whole[:, None]) & need[:, None], page[:, None], table[b]))
    table[b[ok]] = ids[ok]
    st["table"].copy_(table)
    both = ok[:, None] & (j < whole[:, None]) & (old >= 0) & (old < pages)
    st["shared"].index_add_(0, old[both], torch.ones_like(old[both], dtype=torch.int32))
    held[b[ok]] = (whole + need)[ok]
    count = count - need.sum()
    st["got"].copy_(torch.where(ok, n, -1))
    st["from"].copy_(torch.where(need, old.gather(1, whole.clamp(0, ldt - 1)[:, None])[:, 0], -1))
    st["to"].copy_(torch.where(need, page, -1))
    st["count"].copy_(torch.where(need, n % P, 0))
    # the copies
    go = (st["from"] >= 0) & (st["to"] >= 0)
    at, to = st["from"].long()[go], st["to"].long()[go]
    here = (torch.arange(P, device="cuda") < st["count"][go][:, None])[None, :, None, :, None]
    st["k"][:, to] = torch.where(here, st["k"][:, at], st["k"][:, to])
    st["v"][:, to] = torch.where(here, st["v"][:, at], st["v"][:, to])
    # what is kept of no request goes back
    first = (st["keep"].long().clamp(min=0) + P - 1) // P
    out = (j >= first[:, None]) & (j < held.clamp(0, ldt)[:, None])
    ids = torch.where(out, table, -1)
    real = (ids >= 0) & (ids < pages)
    share = st["shared"].long()
    share.index_add_(0, ids[real], torch.full_like(ids[real], -1))
    e = torch.arange(ids.numel(), device="cuda").view(ids.shape)
    least = torch.full((pages,), ids.numel(), device="cuda").scatter_reduce(0, ids[real], e[real], "amin")
    mine = real & (share[ids.clamp(0, pages - 1)] < 0) & (least[ids.clamp(0, pages - 1)] == e)
    behind = mine.sum() - torch.cumsum(mine.flatten(), 0).view(mine.shape)
    st["free"][(count + behind)[mine]] = ids[mine].to(torch.int32)
    st["n_free"].copy_(count + mine.sum())
    st["shared"].copy_(share.clamp(min=0))
    st["held"].copy_(torch.minimum(held, torch.maximum(first, torch.zeros_like(first))))
    st["table"].copy_(torch.where(out, -1, table))


def _plain_move(st):
    c, P, ldt, S, N = st["c"], st["c"]["page"], st["ldt"], st["c"]["S"], st["most"]
    first = st["first"].long()
    i = torch.arange(N, device="cuda")
    if c["list"]:
        lo, n = st["from0"][:-1].long(), (st["from0"][1:] - st["from0"][:-1]).long()
        at = st["from"].long()[(lo[:, None] + i).clamp(max=st["from"].numel() - 1)]
    else:
        bit = (st["tree"][st["leaf"].long()][:, None] >> torch.arange(TREE, device="cuda")) & 1
        n = bit.sum(1)
        at = first[:, None] + torch.argsort(1 - bit, dim=1, stable=True)[:, :N]
    live = i < n[:, None]
    to = first[:, None] + i
    page = lambda t, p: t.long().gather(1, (p // P).clamp(0, ldt - 1))[live]  # noqa: E731
    a, b = page(st["table"], at), page(st["other"] if st["other"] is not None else st["table"], to)
    at, to = (at % P)[live], (to % P)[live]
    st["k"][:, b, :, to] = st["k"][:, a, :, at]
    st["v"][:, b, :, to] = st["v"][:, a, :, at]
    st["kv_len"].copy_(first + n)


def _rows_of(start, most, T):
    """Rows of each run of rows start[i] .. start[i + 1] - 1, padded to `most`: (their numbers, which there are)."""
    i = torch.arange(most, device="cuda")
    return (start[:-1, None] + i).clamp(max=T - 1), i < (start[1:] - start[:-1])[:, None]


def _scores(st, row, page, at):
    """Scores of the padded rows [B][N] over the keys at (page, at) [B][L]: [B][HK][N][heads of a KV head][L]; and the keys' V."""
    H, HK, D = (st["c"][n] for n in ("H", "HK", "D"))
    B, N = row.shape
    k = st["k"][page, :, at].permute(0, 2, 3, 1).float().contiguous()  # [B][HK][D][L]
    q = st["q"].float().view(-1, HK, H // HK, D)[row].permute(0, 2, 1, 3, 4).reshape(B, HK, N * (H // HK), D)
    v = st["v"][page, :, at].float().permute(0, 2, 1, 3).contiguous()  # [B][HK][L][D]
    return (q @ k).view(B, HK, N, H // HK, -1) * st["scale"], v


def _plain_shared(st):
    """The rows of a group over its prefix as one product, each request's rows over its own keys, one softmax over both."""
    c = st["c"]
    H, HK, D, P, T, ldt = c["H"], c["HK"], c["D"], c["page"], st["T"], st["ldt"]
    row0, kv, group0, prefix = (st[n].long() for n in ("row0", "kv_len", "group0", "shared"))
    table = st["table"].long()
    j = torch.arange(c["shared"], device="cuda")
    rows_g, live_g = _rows_of(row0[group0], st["NG"], T)
    xg, vg = _scores(st, rows_g, table[st["lead"].long()][:, j // P].clamp(min=0), j % P)
    in_g = (j < prefix[:, None])[:, None, None, None]
    begin = torch.repeat_interleave(prefix, group0[1:] - group0[:-1], output_size=c["S"])[:, None]
    o = begin + torch.arange(st["LO"], device="cuda")  # own keys
    rows, live = _rows_of(row0, st["N"], T)
    page = table.gather(1, (o // P).clamp(max=ldt - 1)).clamp(min=0)
    xo, vo = _scores(st, rows, page, o % P)
    new = o - (kv - row0[1:] + row0[:-1])[:, None]  # a key's number among the new rows
    seen = new[:, None] <= torch.arange(st["N"], device="cuda")[:, None]
    if st["bits"] is not None:
        bit = (st["bits"][rows][..., None] >> new[:, None].clamp(0, TREE - 1)) & 1
        seen = (new < 0)[:, None] | ((bit == 1) & (new < TREE)[:, None])
    seen = (seen & (o < kv[:, None])[:, None])[:, None, :, None]
    xg, xo = torch.where(in_g, xg, -math.inf), torch.where(seen, xo, -math.inf)
    vg = torch.where((j < prefix[:, None])[:, None, :, None], vg, 0.0)
    vo = torch.where((o < kv[:, None])[:, None, :, None], vo, 0.0)

    def flat(of_g, of_o):
        """What the rows have of their groups and of their own, [T][HK][heads of a KV head]..."""
        a, b = (torch.zeros((T, HK) + x.shape[3:], device="cuda") for x in (of_g, of_o))
        a[rows_g[live_g]], b[rows[live]] = of_g.transpose(1, 2)[live_g], of_o.transpose(1, 2)[live]
        return a, b

    top = torch.maximum(*flat(xg.amax(-1), xo.amax(-1)))
    top = torch.where(top == -math.inf, 0.0, top)[..., None]
    xg, xo = (torch.exp(x - top[r].transpose(1, 2)) for x, r in ((xg, rows_g), (xo, rows)))
    w = torch.add(*flat(xg.sum(-1), xo.sum(-1)))[..., None]
    values = lambda x, v: (x.flatten(2, 3) @ v).view(x.shape[:-1] + (D,))  # noqa: E731
    y = torch.add(*flat(values(xg, vg), values(xo, vo)))
    st["out"].copy_(torch.where(w > 0, y / torch.where(w > 0, w, 1.0), 0.0).view(T, H * D))


def _delta(st, k, row):
    """scale B (A x) of segment k for the padded rows [S][N], zero where there is no adapter."""
    c = st["c"]
    who = st["adapter"].long()
    real = (who >= 0) & (who < c["adapters"])
    at = who.clamp(0, c["adapters"] - 1)
    x = st["x"][:, : c["K"]][row]
    h = x @ st["a"][k][at].float().transpose(1, 2).contiguous()  # [S][N][rank]
    in_rank = torch.arange(c["rank"], device="cuda") < st["ranks"][at][:, None]
    h = torch.where((in_rank & real[:, None])[:, None], h, 0.0)
    return (h @ st["b"][k][at].float().transpose(1, 2).contiguous()) * st["scale"][at][:, None, None]


def _plain_lora(st):
    c = st["c"]
    row0 = st["row0"].long()
    row, live = _rows_of(row0, st["N"], st["T"])
    at = row[live]
    if c["mode"] == "swiglu":
        gate = st["y"][0][at, : c["N"]] + _delta(st, 0, row)[live]
        up = st["y"][1][at, : c["N"]] + _delta(st, 1, row)[live]
        st["out"][at] = gate / (1 + torch.exp(-gate)) * up
        return
    add = lambda k: st["y"][k][:, : _widths(c)[k]].index_add_(0, at, _delta(st, k, row)[live])  # noqa: E731
    list(map(add, range(c["segs"])))


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
    if c["op"] == "fork":
        S, P, ldt, pages = st["held"].numel(), c["page"], st["ldt"], st["pages"]
        kv = _cache(hip, c, st)
        fork = hip.PageFork(F=c["F"], S=S, page=P, ldt=ldt, pages=pages, src=st["src"], dst=st["dst"], tokens=st["tokens"],
                            free=st["free"], n_free=st["n_free"], table=st["table"], held=st["held"], shared=st["shared"],
                            got=st["got"], copy_from=st["from"], copy_to=st["to"], copy_tokens=st["count"])
        copy = hip.PageCopy(n=c["F"], source=st["from"], to=st["to"], tokens=st["count"], layers=c["layers"],
                            layer_stride=pages * c["HK"] * P * c["D"])
        back = hip.PageFree(S=S, page=P, ldt=ldt, pages=pages, keep=st["keep"], table=st["table"], held=st["held"],
                            shared=st["shared"], free=st["free"], n_free=st["n_free"],
                            ws=_bytes(hip.page_free_ws_bytes(S, ldt)))

        def cycle(s):
            hip.launch_page_fork(fork, s)
            hip.launch_page_copy(copy, kv, s)
            hip.launch_page_free(back, s)
        return cycle
    if c["op"] == "move":
        kv = _cache(hip, c, st)
        a = hip.CacheMove(S=c["S"], table=st["table"], ldt=st["ldt"], to_table=st["other"], ldt_to=st["ldt"],
                          first=st["first"], kv_len=st["kv_len"], layers=c["layers"],
                          layer_stride=st["pages"] * c["HK"] * c["page"] * c["D"])
        if c["list"]:
            a.source, a.source0, a.T = st["from"], st["from0"], st["from"].numel()
        else:
            a.tree, a.leaf, a.T = st["tree"], st["leaf"], st["T"]
        return lambda s: hip.launch_cache_move(a, kv, s)
    if c["op"] == "shared":
        H, D = c["H"], c["D"]
        kv = _cache(hip, c, st)
        ws = _bytes(hip.shared_attention_ws_bytes(c["S"], st["T"], H, kv))
        a = hip.SharedAttention(S=c["S"], T=st["T"], heads=H, q=st["q"], ldq=H * D, table=st["table"], ldt=st["ldt"],
                                row0=st["row0"], kv_len=st["kv_len"], tree=st["bits"], scale=st["scale"], out=st["out"],
                                ldo=H * D, ws=ws, groups=c["groups"], group0=st["group0"], lead=st["lead"],
                                shared=st["shared"])
        return lambda s: hip.launch_shared_attention(a, kv, s)
    K, R = c["K"], c["rank"]
    segs = [hip.LoraSeg(a=a, b=b, a_stride=R * K, b_stride=n * R, N=n, y=y, ldy=n + c["pad"])
            for a, b, n, y in zip(st["a"], st["b"], _widths(c), st["y"])]
    a = hip.Lora(S=c["S"], T=st["T"], K=K, rank=R, adapters=c["adapters"], type=hip.CacheType[c["type"]],
                 mode=hip.GemvMode.kSwiglu if c["mode"] == "swiglu" else hip.GemvMode.kAdd, row0=st["row0"],
                 adapter=st["adapter"], ranks=st["ranks"], scale=st["scale"], x=st["x"], ldx=K + c["pad"], out=st["out"],
                 ldo=c["N"] if st["out"] is not None else 0, ws=_bytes(hip.lora_ws_bytes(c["S"], st["T"], K, R, c["segs"])))
    return lambda s: hip.launch_lora(a, segs, s)


def _outputs(st):
    names = {"fork": ("table", "held", "free", "n_free", "shared", "got", "from", "to", "count", "k", "v"),
             "move": ("k", "v", "kv_len"), "shared": ("out",), "lora": ("out",) if st["c"].get("mode") == "swiglu" else ("y",)}
    return {n: st[n] for n in names[st["c"]["op"]]}


def run(st):
    if own:
        if "call" not in st:
            st["call"] = _bind(st)
        st["call"](torch.cuda.current_stream().cuda_stream)
    else:
        {"fork": _plain_fork, "move": _plain_move, "shared": _plain_shared, "lora": _plain_lora}[st["c"]["op"]](st)
    return _outputs(st)


# ---- what a pass cannot do without ----
def work(case):
    c = case
    if c["op"] == "fork":
        ctx, src, n = _fork_sizes(c)
        P = c["page"]
        ids = sum(_pages_of(t, P) for t in n)
        return {"bytes": 2 * 4 * c["HK"] * c["D"] * c["layers"] * sum(t % P for t in n) + 4 * (5 * ids + 9 * c["F"]),
                "flops": 2 * ids}
    if c["op"] == "move":
        base, new, stay = _move_sizes(c)
        return {"bytes": (2 * 4 * c["HK"] * c["D"] * c["layers"] + 4) * sum(stay) + 16 * c["S"], "flops": 2 * sum(stay)}
    if c["op"] == "shared":
        group0, prefix, lone, new = _shared_sizes(c)
        which = np.repeat(np.arange(len(prefix)), np.diff(group0)).tolist()
        kv = sum(prefix) + sum(lone) + sum(new)  # the prefix is read once
        pairs = sum(n * (prefix[w] + a) + n * (n + 1) // 2 for w, a, n in zip(which, lone, new))
        return {"bytes": 4 * c["HK"] * c["D"] * kv + 6 * c["H"] * c["D"] * sum(new) + 4 * kv // c["page"],
                "flops": 4 * c["H"] * c["D"] * pairs}
    new, who, ranks = _lora_sizes(c)
    T, n = sum(new), sum(_widths(c))
    used = sum(ranks[w] for w in set(who) if w >= 0)
    ends = 4 * T * (2 * n if c["mode"] == "add" else n + c["N"])
    return {"bytes": 2 * used * (c["K"] * c["segs"] + n) + 4 * T * c["K"] + ends,
            "flops": sum(2 * m * ranks[w] * (c["K"] * c["segs"] + n) for m, w in zip(new, who) if w >= 0)}


# ---- the definitions in 64 bits, on the host or row by row ----
def _exact_fork(c, st):
    P, pages, ldt = c["page"], st["pages"], st["ldt"]
    get = lambda n: st[n].tolist()  # noqa: E731
    table, held, share, free = get("table"), get("held"), get("shared"), get("free")
    stack, blocked = free[: get("n_free")[0]], False
    start, had, taken = list(held), len(free), set()
    got, frm, to, cnt = [], [], [], []
    k, v = st["k"].clone(), st["v"].clone()
    for s, d, n in zip(get("src"), get("dst"), get("tokens")):
        ok = 0 <= s < len(held) and 0 <= d < len(held) and s != d and 0 <= n <= start[s] * P and start[d] == 0 and d not in taken
        if ok:
            taken.add(d)
        if ok and n % P and (blocked or not stack):
            ok, blocked = False, True
        entry = (-1, -1, 0)
        if ok:
            for i in range(n // P):
                table[d][i] = table[s][i]
                share[table[s][i]] += 1
            held[d] = n // P
            if n % P:
                entry = (table[s][n // P], stack.pop(), n % P)
                table[d][n // P] = entry[1]
                held[d] += 1
                k[:, entry[1], :, : n % P] = st["k"][:, entry[0], :, : n % P]
                v[:, entry[1], :, : n % P] = st["v"][:, entry[0], :, : n % P]
        got.append(n if ok else -1)
        frm.append(entry[0]), to.append(entry[1]), cnt.append(entry[2])
    back, holders = [], {}
    for s, n in enumerate(get("keep")):
        for j in range(_pages_of(max(0, n), P), held[s]):
            holders[table[s][j]] = holders.get(table[s][j], 0) + 1
            if holders[table[s][j]] == 1:
                back.append(table[s][j])
            table[s][j] = -1
        held[s] = min(held[s], _pages_of(max(0, n), P))
    back = [p for p in back if holders[p] > share[p]]
    for p, n in holders.items():
        share[p] = max(0, share[p] - n)
    stack += back[::-1]
    free[: len(stack)] = stack
    out = {"table": table, "held": held, "free": free[:had], "n_free": [len(stack)], "shared": share, "got": got, "from": frm,
           "to": to, "count": cnt}
    return {**{n: torch.tensor(x, dtype=torch.int32) for n, x in out.items()}, "k": k, "v": v}


def _exact_move(c, st):
    P = c["page"]
    table, first = st["table"].tolist(), st["first"].tolist()
    there = st["other"].tolist() if st["other"] is not None else table
    a, b, ends = [], [], []
    for s in range(c["S"]):
        if c["list"]:
            lo, hi = st["from0"][s: s + 2].tolist()
            at = st["from"][lo:hi].tolist()
        else:
            bits = int(st["tree"][int(st["leaf"][s])]) % 2 ** 64
            at = [first[s] + t for t in range(TREE) if bits >> t & 1]
        a += [table[s][t // P] * P + t % P for t in at]
        b += [there[s][t // P] * P + t % P for t in range(first[s], first[s] + len(at))]
        ends.append(first[s] + len(at))
    a, b = (torch.tensor(x, device="cuda") for x in (a, b))
    out = {"kv_len": torch.tensor(ends, dtype=torch.int32)}
    for n in ("k", "v"):
        x = st[n].transpose(2, 3).reshape(c["layers"], -1, c["HK"], c["D"]).clone()
        x[:, b] = x[:, a]
        out[n] = x.view(c["layers"], -1, P, c["HK"], c["D"]).transpose(2, 3).contiguous()
    return out


def _exact_shared(c, st):
    H, HK, D, P = c["H"], c["HK"], c["D"], c["page"]
    G = H // HK
    row0, kv = st["row0"].tolist(), st["kv_len"].tolist()
    out = torch.zeros((st["T"], H * D), dtype=torch.float64, device="cuda")
    for s in range(c["S"]):
        a, b, L = row0[s], row0[s + 1], kv[s]
        ctx = L - (b - a)
        pages = st["table"][s, : _pages_of(L, P)].long()
        seen = torch.ones((b - a, L), dtype=torch.bool, device="cuda")
        if st["bits"] is not None:
            seen[:, ctx:] = (st["bits"][a:b, None] >> torch.arange(b - a, device="cuda")) & 1 == 1
        else:
            seen[:, ctx:] = torch.ones((b - a, b - a), device="cuda").tril() > 0
        for h in range(HK):
            k, v = (st[n][pages, h].reshape(-1, D)[:L].double() for n in ("k", "v"))
            q = st["q"][a:b, h * G * D: (h + 1) * G * D].double().view(-1, D)  # rows of a token's heads
            x = (q @ k.T * st["scale"]).masked_fill(~seen.repeat_interleave(G, 0), -math.inf)
            out[a:b, h * G * D: (h + 1) * G * D] = (torch.softmax(x, -1) @ v).view(b - a, G * D)
    return {"out": out}


def _exact_lora(c, st):
    row0, who, ranks, scale = (st[n].tolist() for n in ("row0", "adapter", "ranks", "scale"))
    y = [t.double() for t in st["y"]]
    x = st["x"][:, : c["K"]]
    for s, w in enumerate(who):
        rows = slice(row0[s], row0[s + 1])
        if w >= 0:
            for k, n in enumerate(_widths(c)):
                r = ranks[w]
                h = x[rows].double() @ st["a"][k][w, :r].double().T
                y[k][rows, :n] += scale[w] * (h @ st["b"][k][w, :, :r].double().T)
    if c["mode"] == "swiglu":
        g, u = (t[:, : c["N"]] for t in y)
        return {"out": g * torch.sigmoid(g) * u}
    return {"y": y}


def exact(case, seed):
    st = prepare(case, seed)
    return {"fork": _exact_fork, "move": _exact_move, "shared": _exact_shared, "lora": _exact_lora}[case["op"]](case, st)
