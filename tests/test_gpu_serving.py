"""GPU tests of a serving step's operators against plain references in 64 bits
(serving_ref.py): the page plan, rotary positions with the cache write, paged
attention and sampling, each alone at the sizes and masks where it can go
wrong, then together as a serving loop runs them, eager and as a captured graph.
"""
import dataclasses
import math

import numpy as np
import pytest

import serving_ref as ref

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def dev(a):
    return _torch().from_numpy(np.ascontiguousarray(a).copy()).cuda()


def ints(a):
    return dev(np.asarray(a, np.int32))


def host(t):
    _torch().cuda.synchronize()
    return t.cpu().numpy()


def stream():
    return _torch().cuda.current_stream().cuda_stream


def kind_of(kind):
    torch = _torch()
    return torch.float16 if kind == "f16" else torch.bfloat16


def words(n):
    """n bytes of scratch, filled with what an earlier user may have left."""
    torch = _torch()
    return torch.full((max(1, -(-n // 8)),), -1, dtype=torch.int64, device="cuda")


# ---- page plan ----
def run_plan(hip, ctx, n_new, held, parent, free, n_free, table, T, page, pages, in_place=False):
    torch = _torch()
    S, ldt = table.shape
    full = lambda n, v, t=torch.int32: torch.full((n,), v, dtype=t, device="cuda")  # noqa: E731
    d = {"table": ints(table), "held_out": full(S, -9), "n_free_out": full(1, -9), "row0": full(S + 1, -9),
         "kv_len": full(S, -9), "pos": full(T, -9), "slot": full(T, -9), "tree": full(T, -9, torch.int64)}
    held_d, n_free_d = ints(held), ints([n_free])
    if in_place:
        d["held_out"], d["n_free_out"] = held_d, n_free_d
    hip.launch_page_plan(hip.PagePlan(
        S=S, T=T, page=page, ldt=ldt, pages=pages, ctx=ints(ctx), n_new=ints(n_new), held=held_d,
        parent=ints(parent) if parent is not None else None, free=ints(free), n_free=n_free_d, table=d["table"],
        held_out=d["held_out"], n_free_out=d["n_free_out"], row0=d["row0"], kv_len=d["kv_len"], pos=d["pos"],
        slot=d["slot"], tree=d["tree"] if parent is not None else None), stream())
    return {n: host(t) for n, t in d.items()}


def check_plan(got, want, T, tree):
    for n in ("table", "held_out", "row0", "kv_len"):
        np.testing.assert_array_equal(got[n], want[n], err_msg=n)
    assert got["n_free_out"][0] == want["n_free_out"]
    for n in ("pos", "slot") + (("tree",) if tree else ()):
        w = np.full(T, -9, np.int64)  # rows behind the last request stay as they were
        for r, v in want[n].items():
            w[r] = v if v < 2 ** 63 else v - 2 ** 64
        np.testing.assert_array_equal(got[n], w, err_msg=n)


def plan_case(rng, S, page, ctx_hi, new_hi, tree, spare, bad=0.0, T=None):
    ctx = rng.integers(0, ctx_hi + 1, S)
    n_new = rng.integers(0, new_hi + 1, S)
    held = -(-ctx // page) + (rng.random(S) < 0.3)  # some hold a page more than they need
    ldt = int(max(1, (-(-(ctx + n_new) // page)).max(), held.max()))
    need = int(np.maximum(0, -(-(ctx + n_new) // page) - held).sum())
    pages = int(held.sum()) + need + 4
    perm = rng.permutation(pages)
    table = np.full((S, ldt), -5, np.int64)
    at = 0
    for s in range(S):
        table[s, :held[s]] = perm[at:at + held[s]]
        at += int(held[s])
    rows = int(n_new.sum())
    parent = None
    if tree:
        parent = np.concatenate([np.maximum(-1, np.arange(n) - rng.integers(1, 4, n)) for n in n_new] + [np.zeros(0)])
        parent = np.concatenate([parent, np.zeros(3 + max(0, (T or 0) - rows))]).astype(np.int64)
    for s in np.flatnonzero(rng.random(S) < bad):
        what = rng.integers(4)
        if what == 0:
            ctx[s] = -1
        elif what == 1:
            n_new[s] = -3
        elif what == 2:
            held[s] = -1
        else:
            ctx[s] = held[s] * page + 1
    free = np.concatenate([perm[at:], [0]])
    T = T if T is not None else rows + 3
    return ctx, n_new, held, parent[:T] if parent is not None else None, free, int(need * spare), table, T, page, pages


@pytest.mark.parametrize("S,page,ctx_hi,new_hi,tree,spare,bad", [
    (1, 16, 0, 1, False, 1, 0), (1, 64, 100, 1, True, 1, 0), (5, 16, 40, 64, True, 1, 0), (7, 32, 200, 130, True, 1, 0),
    (9, 256, 3000, 300, False, 1, 0), (33, 16, 50, 20, True, 0.5, 0), (64, 64, 500, 1, False, 0.3, 0),
    (40, 16, 60, 10, True, 1, 0.4), (1024, 16, 30, 5, False, 1, 0), (1025, 16, 30, 5, True, 0.9, 0.05),
    (2500, 32, 64, 3, False, 0.6, 0.1), (3, 16, 10, 2500, False, 1, 0), (4, 16, 0, 0, True, 1, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_plan(hip, S, page, ctx_hi, new_hi, tree, spare, bad, in_place):
    c = plan_case(np.random.default_rng(S * 1000 + page + new_hi), S, page, ctx_hi, new_hi, tree, spare, bad)
    check_plan(run_plan(hip, *c, in_place=in_place), ref.plan(*c), c[7], tree)


def test_page_plan_rows_that_do_not_fit(hip):
    """Requests whose rows pass T are refused; a piece of one keeps its place in the rows."""
    rng = np.random.default_rng(5)
    for T in (0, 1, 7, 20, 33):
        c = plan_case(rng, 6, 16, 40, 12, T > 0, 1, T=T)
        check_plan(run_plan(hip, *c), ref.plan(*c), T, T > 0)


def test_page_plan_trees(hip):
    """Chains, stars, parents that are none (themselves, later ones, below -1), 64 and 65 nodes."""
    rng = np.random.default_rng(6)
    n_new = [64, 64, 65, 64, 1, 30]
    parent = np.concatenate([np.arange(64) - 1, np.zeros(64) - (np.arange(64) == 0), np.arange(65) - 1,
                             rng.integers(-3, 70, 64), [5], rng.integers(-1, 30, 30)]).astype(np.int64)
    ctx, held = np.array([0, 100, 5, 17, 64, 9]), np.array([0, 7, 1, 2, 4, 1])
    pages = 60
    perm = rng.permutation(pages)
    table = np.full((6, 20), -1)
    for s in range(6):
        table[s, :held[s]] = perm[s * 7:s * 7 + held[s]]
    c = (ctx, np.array(n_new), held, parent, perm[42:], 18, table, 288, 16, pages)
    check_plan(run_plan(hip, *c), ref.plan(*c), 288, True)


def test_page_plan_bad_page_ids(hip):
    """Ids outside the cache, in the table and in the free list, give slot -1."""
    table = np.array([[3, -1, 9, 0], [10 ** 9, 2, 0, 0]])
    c = (np.array([33, 20]), np.array([40, 5]), np.array([3, 2]), None, np.array([1, 7, -4, 50]), 4, table, 50, 16, 8)
    check_plan(run_plan(hip, *c), ref.plan(*c), 50, False)
    c = (np.array([33, 20]), np.array([40, 5]), np.array([3, 2]), None, np.array([1, 7, -4, 50]), -2, table, 50, 16, 8)
    check_plan(run_plan(hip, *c), ref.plan(*c), 50, False)


# ---- rotary positions and the cache write ----
def rope_inputs(rng, T, H, HK, D, page, kind, gap=0, lead=0):
    torch = _torch()
    ld = lead + (H + 2 * HK) * D + gap
    qkv = rng.standard_normal((T, ld)).astype(np.float32) * 3
    pages = -(-T // page) + 2
    slot = rng.permutation(pages * page)[:T]
    old = [torch.from_numpy(rng.standard_normal((pages, HK, page, D))).to(kind_of(kind)).cuda() for _ in range(2)]
    return qkv, slot, old, pages


def run_rope(hip, qkv, slot, cache, pages, pos, turns, H, HK, D, page, kind, n_rot, layout, mscale=1.0, norms=None,
             eps=1e-6, lead=0, rows=None, do=("q", "kv"), strides=None):
    torch = _torch()
    T, ld = qkv.shape
    x = dev(qkv)
    q_out = torch.full((T, H * D), 7.0, dtype=kind_of(kind), device="cuda")
    part = lambda n: x.view(-1)[lead + n * D:]  # noqa: E731
    kv = hip.KvCache(cache[0], cache[1], hip.CacheType[kind], page, HK, D, pages, *(strides or (HK * page * D, page * D, D)))
    a = hip.RopeCache(T=T, heads=H, eps=eps, n_rot=n_rot, layout=hip.RopeLayout[layout], turns=dev(np.asarray(turns, np.float64)),
                      mscale=mscale, pos=ints(pos), slot=ints(slot), rows=rows, q_norm=dev(norms[0]) if norms else None,
                      k_norm=dev(norms[1]) if norms else None)
    if "q" in do:
        a = dataclasses.replace(a, q=part(0), ldq=ld, q_out=q_out, ldqo=H * D)
    if "kv" in do:
        a = dataclasses.replace(a, k=part(H), ldk=ld, v=part(H + HK), ldv=ld)
    hip.launch_rope_cache(a, kv, stream())
    torch.cuda.synchronize()
    return q_out


def rope_tol(y, size, kind, D):
    """Half a step of the 16-bit type, and the 32-bit roundings before it: the norm's sum of D squares in a tree of
    fours and pairs (at most 4 + 6 roundings, halved by the root), its product, sine, cosine and scale (3 ulp), the
    two products and their sum: under 32 half-steps of 2^-24 of the pair's size. fp16's smallest step below its
    normal range is 2^-24."""
    return ref.HALF_STEP[kind] * (np.abs(y) + 32 * 2.0 ** -24 * size) + 32 * 2.0 ** -24 * size + \
        (2.0 ** -25 if kind == "f16" else 0)


def check_rope(q_out, cache, old, qkv, slot, pos, turns, H, HK, D, page, kind, n_rot, layout, mscale=1.0, norms=None,
               eps=1e-6, lead=0, rows=None, do=("q", "kv")):
    T = qkv.shape[0]
    n = T if rows is None else rows
    x = qkv[:n, lead:lead + (H + 2 * HK) * D].reshape(n, H + 2 * HK, D)
    qn, kn = norms or (None, None)
    got = q_out.double().cpu().numpy().reshape(T, H, D)
    if "q" in do:
        y, size = ref.turned(x[:, :H], pos, turns, mscale, n_rot, layout, qn, eps)
        assert np.all(np.abs(got[:n] - y) <= rope_tol(y, size, kind, D))
    else:
        n = 0
    assert np.all(got[n:] == 7.0)
    k, v = (c.double().cpu().numpy() for c in cache)
    wk, wv = (c.double().cpu().numpy().copy() for c in old)
    if "kv" in do:
        yk, size = ref.turned(x[:, H:H + HK], pos, turns, mscale, n_rot, layout, kn, eps)
        yv = ref.to16(x[:, H + HK:].astype(np.float32), kind)
        for t in range(x.shape[0]):
            if 0 <= slot[t] < k.shape[0] * page:
                at = (slot[t] // page, slice(None), slot[t] % page)
                assert np.all(np.abs(k[at] - yk[t]) <= rope_tol(yk[t], size[t], kind, D))
                np.testing.assert_array_equal(v[at], yv[t])
                wk[at], wv[at] = k[at], v[at]
    np.testing.assert_array_equal(k, wk)  # nothing else of the cache was touched
    np.testing.assert_array_equal(v, wv)


ROPE_CASES = [(T, heads, n_rot, layout, kind, norm) for T, heads, n_rot, layout, kind, norm in [
    (1, (20, 4, 256), 64, "half", "f16", True), (1, (1, 1, 64), 64, "pairs", "bf16", False),
    (3, (40, 8, 128), 128, "half", "bf16", True), (17, (5, 1, 128), 64, "pairs", "f16", True),
    (2, (20, 4, 256), 246, "half", "f16", True), (2, (20, 4, 256), 246, "pairs", "bf16", True),
    (5, (7, 7, 64), 2, "half", "f16", False), (5, (7, 7, 64), 54, "half", "bf16", True),
    (33, (3, 3, 128), 0, "half", "f16", True), (4, (2, 1, 256), 256, "pairs", "f16", False),
    (70, (4, 2, 64), 32, "half", "bf16", False), (700, (20, 4, 256), 64, "half", "f16", True),
    (1200, (17, 1, 128), 32, "pairs", "bf16", True), (9, (9, 3, 128), 126, "half", "f16", False)]]


@pytest.mark.parametrize("T,heads,n_rot,layout,kind,norm", ROPE_CASES, ids=str)
@pytest.mark.parametrize("gap,lead", [(0, 0), (1, 0), (4, 4), (3, 1)])
def test_rope_cache(hip, T, heads, n_rot, layout, kind, norm, gap, lead):
    """Heads, parts of the head, layouts, types; row strides and starts that allow vector accesses or not."""
    H, HK, D = heads
    rng = np.random.default_rng(T * 7 + n_rot)
    page = int(rng.choice([16, 64, 256]))
    qkv, slot, old, pages = rope_inputs(rng, T, H, HK, D, page, kind, gap, lead)
    if T > 4:
        slot[1], slot[2], slot[3] = -1, pages * page, 2 ** 31 - 1  # rows without a place in the cache
    pos = rng.integers(0, 200000, T)
    pos[0] = 0
    turns, _ = hip.rope_table(n_rot, 1e7) if n_rot else ([], 1.0)
    norms = tuple(1 + 0.2 * rng.standard_normal((2, D)).astype(np.float32)) if norm else None
    cache = [c.clone() for c in old]
    args = (H, HK, D, page, kind, n_rot, layout)
    q = run_rope(hip, qkv, slot, cache, pages, pos, turns or [0.0], *args, mscale=1.25, norms=norms, lead=lead)
    check_rope(q, cache, old, qkv, slot, pos, turns, *args, mscale=1.25, norms=norms, lead=lead)


@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_rope_far_positions(hip, layout):
    """Positions up to 2^31 - 1: in 32 bits the angle of the fastest pair would be off by whole turns."""
    rng = np.random.default_rng(3)
    H, HK, D, page, kind = 2, 1, 64, 16, "f16"
    qkv, slot, old, pages = rope_inputs(rng, 8, H, HK, D, page, kind)
    pos = np.array([0, 1, 10 ** 5, 10 ** 6 + 7, 2 ** 24 + 1, 10 ** 9 + 3, 2 ** 31 - 2, 2 ** 31 - 1])
    # (exact in 64 bits: the reference's product rounds as the kernel's does)
    turns = np.array([0.25 + 2.0 ** -20, 2.0 ** -3, 0.15915494309189535] + [1e-4] * 29)
    cache = [c.clone() for c in old]
    q = run_rope(hip, qkv, slot, cache, pages, pos, turns, H, HK, D, page, kind, 64, layout)
    check_rope(q, cache, old, qkv, slot, pos, turns, H, HK, D, page, kind, 64, layout)


@pytest.mark.parametrize("rows", [0, 1, 5, 9, 40])
def test_rope_row_count_on_the_device(hip, rows):
    rng = np.random.default_rng(4)
    H, HK, D, page, kind = 3, 1, 128, 16, "bf16"
    qkv, slot, old, pages = rope_inputs(rng, 9, H, HK, D, page, kind)
    pos, (turns, _) = rng.integers(0, 99, 9), hip.rope_table(64, 1e4)
    cache = [c.clone() for c in old]
    q = run_rope(hip, qkv, slot, cache, pages, pos, turns, H, HK, D, page, kind, 64, "half", rows=ints([rows]))
    check_rope(q, cache, old, qkv, slot, pos, turns, H, HK, D, page, kind, 64, "half", rows=min(rows, 9))


@pytest.mark.parametrize("do", [("q",), ("kv",)])
def test_rope_one_part(hip, do):
    rng = np.random.default_rng(5)
    H, HK, D, page, kind = 4, 2, 64, 16, "f16"
    qkv, slot, old, pages = rope_inputs(rng, 6, H, HK, D, page, kind)
    pos, (turns, _) = rng.integers(0, 99, 6), hip.rope_table(64, 1e4)
    cache = [c.clone() for c in old]
    q = run_rope(hip, qkv, slot, cache, pages, pos, turns, H, HK, D, page, kind, 64, "pairs", do=do)
    check_rope(q, cache, old, qkv, slot, pos, turns, H, HK, D, page, kind, 64, "pairs", do=do)


def test_rope_cache_strides(hip):
    """A cache of tokens before heads, in a wider array."""
    torch = _torch()
    rng = np.random.default_rng(6)
    H, HK, D, page, kind, pages = 2, 3, 64, 16, "f16", 4
    wide = [torch.zeros((pages, page, HK, D + 8), dtype=torch.float16, device="cuda") for _ in range(2)]
    qkv, slot, _, _ = rope_inputs(rng, 9, H, HK, D, page, kind)
    pos, (turns, _) = rng.integers(0, 99, 9), hip.rope_table(64, 1e4)
    q = run_rope(hip, qkv, slot, wide, pages, pos, turns, H, HK, D, page, kind, 64, "half",
                 strides=(page * HK * (D + 8), D + 8, HK * (D + 8)))
    view = [w[..., :D].permute(0, 2, 1, 3).contiguous() for w in wide]
    old = [torch.zeros_like(c) for c in view]
    check_rope(q, view, old, qkv, slot, pos, turns, H, HK, D, page, kind, 64, "half")
    assert all(bool((w[..., D:] == 0).all()) for w in wide)


# ---- attention ----
def attn_inputs(rng, kv_len, new, heads, kind, page, sharp=1.0, ldt_more=0, fill=0.0):
    """Cache pages shuffled; what no request holds is `fill`."""
    torch = _torch()
    H, HK, D = heads
    S, t = len(kv_len), kind_of(kind)
    held = [-(-max(0, n) // page) for n in kv_len]
    pages, ldt = sum(held) + 3, max(held + [1]) + ldt_more
    perm = rng.permutation(pages)
    table = np.full((S, ldt), -1)
    k = np.full((pages, HK, page, D), fill)
    v = np.full((pages, HK, page, D), fill)
    at = 0
    for s in range(S):
        table[s, :held[s]] = perm[at:at + held[s]]
        at += held[s]
        for j in range(max(0, kv_len[s])):
            k[table[s, j // page], :, j % page] = rng.standard_normal((HK, D))
            v[table[s, j // page], :, j % page] = rng.standard_normal((HK, D))
    T = sum(new)
    q = rng.standard_normal((T, H * D)) * sharp * np.exp(0.7 * rng.standard_normal((T, 1)))
    cast = lambda a: torch.from_numpy(a).to(t).cuda()  # noqa: E731
    return cast(q), cast(k), cast(v), table, np.cumsum([0] + list(new))


def run_attn(hip, q, k, v, table, row0, kv_len, tree, heads, kind, page, pages=None, scale=None, T=None, ld=0,
             strides=None, st=None, ws=None):
    torch = _torch()
    H, HK, D = heads
    pages = pages or k.shape[0]
    kv = hip.KvCache(k, v, hip.CacheType[kind], page, HK, D, pages, *(strides or (HK * page * D, page * D, D)))
    T = T if T is not None else q.shape[0]
    out = torch.full((max(T, q.shape[0]), H * D + ld), -77.0, dtype=torch.float32, device="cuda")
    S = len(kv_len)
    ws = ws if ws is not None else words(hip.paged_attention_ws_bytes(S, T, H, kv))
    tree_d = dev(np.asarray(tree, np.uint64).view(np.int64)) if tree is not None else None
    a = hip.PagedAttention(S=S, T=T, heads=H, q=q, ldq=q.shape[1], table=ints(table), ldt=table.shape[1],
                           row0=ints(row0), kv_len=ints(kv_len), tree=tree_d, scale=D ** -0.5 if scale is None else scale,
                           out=out, ldo=H * D + ld, ws=ws)
    torch.cuda.synchronize()
    hip.launch_paged_attention(a, kv, st or stream())
    torch.cuda.synchronize()
    return out


def check_attn(out, q, k, v, table, row0, kv_len, tree, heads, kind, page, pages=None, scale=None):
    H, HK, D = heads
    n = int(row0[-1])
    got = out.double().cpu().numpy()
    f = lambda a: a.double().cpu().numpy()  # noqa: E731
    want, tol = ref.attention(f(q)[:n, :H * D], f(k), f(v), table, row0, kv_len, tree, D ** -0.5 if scale is None else scale,
                              page, pages or k.shape[0], H, HK)
    # the probabilities' own rounding for the products: carried in two 16-bit parts, each off by half a step of its own
    want_p = ref.HALF_STEP[kind] ** 2
    vmax = np.abs(np.nan_to_num(f(v), nan=0, posinf=0, neginf=0)).max()
    bad = ~np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got[:n, :H * D]), np.isnan(want))
    d = np.abs(np.where(bad, 0, got[:n, :H * D]) - np.where(bad, 0, want))
    worst = np.max(d - np.where(bad, 1e30, tol + want_p * vmax)) if d.size else -1
    assert worst <= 0, f"off by {d.max():.3g}, over its tolerance by {worst:.3g}"
    assert np.all(got[:, H * D:] == -77.0)
    assert np.all(got[n:] == -77.0)  # rows behind the last request stay as they were


def trees(rng, new, T):
    bits = np.zeros(T, np.uint64)
    at = 0
    for n in new:
        for i in range(min(n, 64)):
            p = i - int(rng.integers(1, 5))
            bits[at + i] = (int(bits[at + p]) if p >= 0 else 0) | 1 << i
        at += n
    return bits


HEADS = [(5, 1, 256), (20, 4, 256), (10, 2, 128), (6, 6, 64), (14, 2, 64), (3, 1, 128), (16, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("kv_len", [[1], [2, 16, 17], [31, 32, 33, 1], [63, 64, 65], [257, 1, 500], [1100]], ids=str)
def test_attention_single_tokens(hip, heads, kind, kv_len):
    rng = np.random.default_rng(sum(kv_len))
    page = [16, 32, 64, 128, 256][sum(kv_len) % 5]
    new = [1] * len(kv_len)
    x = attn_inputs(rng, kv_len, new, heads, kind, page)
    check_attn(run_attn(hip, *x, kv_len, None, heads, kind, page), *x, kv_len, None, heads, kind, page)


@pytest.mark.parametrize("heads", HEADS[:6], ids=str)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("page,ctx,new", [(16, 0, [1, 2, 3]), (64, 50, [17, 0, 64, 5]), (32, 130, [64]), (16, 15, [65]),
                                          (256, 300, [8, 100])], ids=str)
@pytest.mark.parametrize("tree", [False, True])
def test_attention_prompts_and_trees(hip, heads, kind, page, ctx, new, tree):
    rng = np.random.default_rng(ctx + sum(new))
    kv_len = [ctx + 3 * s + n for s, n in enumerate(new)]
    x = attn_inputs(rng, kv_len, new, heads, kind, page)
    bits = trees(rng, new, sum(new)) if tree else None
    check_attn(run_attn(hip, *x, kv_len, bits, heads, kind, page), *x, kv_len, bits, heads, kind, page)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,new", [((5, 1, 256), [200, 129]), ((10, 2, 128), [256, 63, 1]), ((2, 2, 64), [385]),
                                       ((4, 1, 64), [128, 127])], ids=str)
def test_attention_longer_prompts(hip, kind, heads, new):
    """Several row tiles, their ends inside tiles and pages."""
    rng = np.random.default_rng(sum(new))
    kv_len = [n + 37 * s for s, n in enumerate(new)]
    x = attn_inputs(rng, kv_len, new, heads, kind, 16)
    check_attn(run_attn(hip, *x, kv_len, None, heads, kind, 16), *x, kv_len, None, heads, kind, 16)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_rows_that_see_nothing(hip, kind):
    """Requests without rows, without length, refused ones (length 0 with rows), trees with empty masks, a length
    below the rows (some rows see nothing)."""
    rng = np.random.default_rng(8)
    heads, page = (10, 2, 128), 16
    kv_len, new = [0, 40, 0, 5, 30, 3], [0, 2, 4, 5, 0, 6]
    x = attn_inputs(rng, kv_len, new, heads, kind, page, fill=math.nan)
    check_attn(run_attn(hip, *x, kv_len, None, heads, kind, page), *x, kv_len, None, heads, kind, page)
    bits = trees(rng, new, sum(new))
    bits[6:11] = [0, 0, 4, 0, 1]  # request 3: no cache before its rows
    check_attn(run_attn(hip, *x, kv_len, bits, heads, kind, page), *x, kv_len, bits, heads, kind, page)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [[20], [70]], ids=["tree", "prompt"])
def test_attention_masked_infinities_and_nan(hip, kind, what, new):
    """K and V that a row does not see (other branches, later rows, what lies behind the end, pages' rests) may hold
    anything; what it sees counts as the formula says."""
    torch = _torch()
    rng = np.random.default_rng(9)
    heads, page, kv_len = (5, 1, 256), 32, [new[0] + 45]
    q, k, v, table, row0 = attn_inputs(rng, kv_len, new, heads, kind, page, fill=what)
    bits = trees(rng, new, sum(new)) if new[0] <= 64 else None
    for j, (a, b) in enumerate([(k, None), (None, v), (k, v)]):
        kk, vv = k.clone(), v.clone()
        for n in (3, 11, new[0] - 1):  # new rows
            pg, off = table[0][(45 + n) // page], (45 + n) % page
            if a is not None:
                kk[pg, :, off] = what
            if b is not None:
                vv[pg, :, off, 5 * j:5 * j + 9] = what
        x = (q, kk, vv, table, row0)
        with np.errstate(invalid="ignore"):
            check_attn(run_attn(hip, *x, kv_len, bits, heads, kind, page), *x, kv_len, bits, heads, kind, page)
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_sharp_and_flat_rows(hip, kind):
    """Scores far apart (up to hundreds) and all equal; a negative scale; a scale of zero."""
    rng = np.random.default_rng(10)
    heads, page, kv_len, new = (10, 2, 128), 16, [333, 70], [1, 3]
    for sharp, scale in ((12.0, None), (0.0, None), (1.0, -0.1), (1.0, 0.0), (1.0, 1e-30), (3.0, 2.0)):
        x = attn_inputs(rng, kv_len, new, heads, kind, page, sharp=sharp)
        check_attn(run_attn(hip, *x, kv_len, None, heads, kind, page, scale=scale), *x, kv_len, None, heads, kind, page,
                   scale=scale)


def test_attention_large_values(hip):
    """Values near the type's ends: scores beyond 32 bits become infinities as the formula's would."""
    torch = _torch()
    rng = np.random.default_rng(11)
    heads, page, kv_len, new = (2, 1, 64), 16, [40], [1]
    q, k, v, table, row0 = attn_inputs(rng, kv_len, new, heads, "f16", page)
    v = torch.full_like(v, 65504.0)
    x = (q, k, v, table, row0)
    check_attn(run_attn(hip, *x, kv_len, None, heads, "f16", page), *x, kv_len, None, heads, "f16", page)


def test_attention_bad_pages(hip):
    """Page ids outside the cache are not seen; a length beyond the table is cut there."""
    rng = np.random.default_rng(12)
    heads, page, kind = (5, 1, 128), 16, "f16"
    kv_len, new = [70, 40, 33], [2, 1, 1]
    q, k, v, table, row0 = attn_inputs(rng, kv_len, new, heads, kind, page)
    table[0][1], table[1][0], table[1][1], table[1][2] = -1, 10 ** 9, k.shape[0], -2 ** 31
    x = (q, k, v, table, row0)
    check_attn(run_attn(hip, *x, kv_len, None, heads, kind, page), *x, kv_len, None, heads, kind, page)
    long = [70, 40, 10 ** 6]
    check_attn(run_attn(hip, *x, long, None, heads, kind, page), *x, long, None, heads, kind, page)


def test_attention_strides(hip):
    """Tokens before heads in wider arrays; rows of q and out with gaps; more rows than the requests have."""
    torch = _torch()
    rng = np.random.default_rng(13)
    heads, page, kind, kv_len, new = (6, 2, 64), 16, "bf16", [50, 20], [4, 1]
    H, HK, D = heads
    q, k, v, table, row0 = attn_inputs(rng, kv_len, new, heads, kind, page)
    wide = []
    for c in (k, v):
        w = torch.full((c.shape[0], page, HK, D + 16), math.nan, dtype=c.dtype, device="cuda")
        w[..., :D] = c.permute(0, 2, 1, 3)
        wide.append(w)
    qw = torch.full((9, H * D + 8), math.nan, dtype=q.dtype, device="cuda")
    qw[:5, :H * D] = q
    out = run_attn(hip, qw, *wide, table, row0, kv_len, None, heads, kind, page, ld=12,
                   strides=(page * HK * (D + 16), D + 16, HK * (D + 16)))
    check_attn(out, qw, k, v, table, row0, kv_len, None, heads, kind, page)


def against_gpu64(out, q, k, v, table, row0, kv_len, heads, page):
    """Causal attention of f16 values in 64 bits on the GPU; the tolerance is the worst case of the 32-bit sums."""
    torch = _torch()
    H, HK, D = heads
    out = out[:, :H * D].double()
    for s in range(len(kv_len)):
        L, a, b = kv_len[s], int(row0[s]), int(row0[s + 1])
        if b == a:
            continue
        ids = torch.from_numpy(table[s, :-(-L // page)]).cuda().long()
        kk, vv = (c[ids].double().transpose(0, 1).reshape(HK, -1, D)[:, :L] for c in (k, v))
        seen = torch.ones((b - a, L), dtype=torch.bool, device="cuda").tril(L - (b - a))
        for h in range(H):
            qq = q[a:b, h * D:(h + 1) * D].double()
            p = torch.softmax((qq @ kk[h // (H // HK)].T * D ** -0.5).masked_fill(~seen, -math.inf), -1)
            want, size = p @ vv[h // (H // HK)], p @ vv[h // (H // HK)].abs()
            d = (out[a:b, h * D:(h + 1) * D] - want).abs()
            assert bool((d <= ((L + 2 * D + 200) * 2.0 ** -24 + 2.0 ** -20) * size).all()), (s, h, float(d.max()))


def gpu_cache(g, kv_len, heads, page):
    torch = _torch()
    H, HK, D = heads
    held = [-(-n // page) for n in kv_len]
    pages = sum(held) + 1
    perm = torch.randperm(pages, generator=g, device="cuda").cpu().numpy()
    table, at = np.full((len(kv_len), max(held)), -1), 0
    for s, n in enumerate(held):
        table[s, :n] = perm[at:at + n]
        at += n
    k, v = (torch.randn((pages, HK, page, D), generator=g, device="cuda").to(torch.float16) for _ in range(2))
    return k, v, table


@pytest.mark.parametrize("heads,page", [((20, 4, 256), 32), ((16, 2, 128), 16), ((8, 8, 64), 64)], ids=str)
@pytest.mark.parametrize("new_hi", [1, 6, 40])
def test_attention_many_requests(hip, heads, page, new_hi):
    """More requests than a wave has lanes, lengths from 1 to 9000 in one batch, some without rows: cut and whole
    requests side by side, found over several chunks."""
    torch = _torch()
    rng = np.random.default_rng(new_hi)
    g = torch.Generator(device="cuda").manual_seed(new_hi)
    S = 150
    new = [int(n) for n in rng.integers(0 if new_hi > 1 else 1, new_hi + 1, S)]
    kv_len = [n + int(c) for n, c in zip(new, np.exp(rng.uniform(0, 6, S)).astype(int))]
    kv_len[7], kv_len[77], kv_len[149] = 9001, 5003, 3001
    kv_len = [max(1, n) for n in kv_len]
    k, v, table = gpu_cache(g, kv_len, heads, page)
    q = torch.randn((sum(new), heads[0] * heads[2]), generator=g, device="cuda").to(torch.float16)
    row0 = np.cumsum([0] + new)
    out = run_attn(hip, q, k, v, table, row0, kv_len, None, heads, "f16", page)
    against_gpu64(out, q, k, v, table, row0, kv_len, heads, page)


@pytest.mark.parametrize("heads", [(128, 1, 64), (64, 1, 128), (48, 1, 256)], ids=str)
def test_attention_many_heads_of_one_kv_head(hip, heads):
    rng = np.random.default_rng(30)
    kv_len, new = [200, 31], [1, 3]
    x = attn_inputs(rng, kv_len, new, heads, "bf16", 16)
    check_attn(run_attn(hip, *x, kv_len, None, heads, "bf16", 16), *x, kv_len, None, heads, "bf16", 16)


def test_attention_shared_pages(hip):
    """Requests with a common beginning hold the same pages."""
    rng = np.random.default_rng(31)
    heads, page, kv_len, new = (10, 2, 128), 16, [60, 60, 40], [1, 2, 1]
    q, k, v, table, row0 = attn_inputs(rng, kv_len, new, heads, "f16", page)
    table[1, :3], table[2, :2] = table[0, :3], table[0, :2]
    x = (q, k, v, table, row0)
    check_attn(run_attn(hip, *x, kv_len, None, heads, "f16", page), *x, kv_len, None, heads, "f16", page)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_infinities_in_a_long_cache(hip, new):
    """An infinity in V that the rows of one request see: infinities there (the formula's), nothing in the other's."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(5)
    heads, page, kv_len = (10, 2, 128), 64, [2500, 2400]
    k, v, table = gpu_cache(g, kv_len, heads, page)
    q = torch.randn((2 * new, 1280), generator=g, device="cuda").to(torch.float16)
    row0 = np.array([0, new, 2 * new])
    v[int(table[0][1500 // page]), 1, 1500 % page, 77] = math.inf
    out = run_attn(hip, q, k, v, table, row0, kv_len, None, heads, "f16", page)
    for h in range(5, 10):
        assert bool((out[:new, h * 128 + 77] == math.inf).all())
    out[:new, 640:][:, 77::128] = 0
    clean = v.clone()
    clean[int(table[0][1500 // page]), 1, 1500 % page, 77] = 0
    want = run_attn(hip, q, k, clean, table, row0, kv_len, None, heads, "f16", page)
    want[:new, 640:][:, 77::128] = 0
    # request 0's KV head 1 goes through the plain loop: other orders of the same sums of 2500 terms
    assert bool(((out - want).abs() <= 2 * 2900 * 2.0 ** -24 * 5).all())
    assert torch.equal(out[new:], want[new:]) and torch.equal(out[:new, :640], want[:new, :640])


@pytest.mark.parametrize("heads,S,new", [((20, 4, 256), 3, 1), ((10, 2, 128), 2, 33), ((4, 4, 64), 40, 1), ((10, 2, 128), 2, 11),
                                         ((8, 8, 64), 3, 70), ((10, 2, 128), 3, 5), ((14, 2, 64), 2, 4), ((20, 4, 256), 2, 30)],
                         ids=str)
def test_attention_long_caches(hip, heads, S, new):
    """Lengths that are split over many workgroups, one request much longer than the others; against 64 bits on the
    GPU. The tolerance is the worst case of the 32-bit sums over the keys."""
    torch = _torch()
    H, HK, D = heads
    g = torch.Generator(device="cuda").manual_seed(S)
    kv_len = [20011] + [97 + 301 * s for s in range(1, S)]
    k, v, table = gpu_cache(g, kv_len, heads, 64)
    q = torch.randn((S * new, H * D), generator=g, device="cuda").to(torch.float16)
    row0 = np.arange(S + 1) * new
    out = run_attn(hip, q, k, v, table, row0, kv_len, None, heads, "f16", 64)
    against_gpu64(out, q, k, v, table, row0, kv_len, heads, 64)


# ---- sampling ----
def run_sample(hip, x, T=None, k=None, p=None, mp=None, u=None, ld=0, logprob=True, ws=None):
    torch = _torch()
    M, V = x.shape
    wide = np.full((M, V + ld), np.inf, np.float32)  # (columns past V are not logits)
    wide[:, :V] = x
    tok = torch.full((M,), -5, dtype=torch.int32, device="cuda")
    lp = torch.full((M,), -5.0, dtype=torch.float32, device="cuda")
    opt = lambda v, t: dev(np.broadcast_to(np.asarray(v, t), (M,))) if v is not None else None  # noqa: E731
    a = hip.Sampling(M=M, V=V, logits=dev(wide), ldl=V + ld, temperature=opt(T, np.float32), top_k=opt(k, np.int32),
                     top_p=opt(p, np.float32), min_p=opt(mp, np.float32), u=opt(u, np.float32), token=tok,
                     logprob=lp if logprob else None, ws=ws if ws is not None else words(hip.sample_ws_bytes(M, V)))
    hip.launch_sample(a, stream())
    return host(tok), host(lp)


def check_sample(hip, x, T=None, k=None, p=None, mp=None, u=None, ld=0):
    x = np.asarray(x, np.float32)
    M = x.shape[0]
    tok, lp = run_sample(hip, x, T, k, p, mp, u, ld)
    row = lambda v, m, none, t: t(none if v is None else np.broadcast_to(np.asarray(v, t), (M,))[m])  # noqa: E731
    f = np.float32
    for m in range(M):
        want = ref.sample(x[m], row(T, m, 1, f), row(k, m, 0, np.int32), row(p, m, 1, f), row(mp, m, 0, f), row(u, m, 0, f))
        assert tok[m] == want[0], (m, tok[m], want)
        # one rounding to 32 bits (half a step), and weights in units of 2^-43: half a unit each of up to V of them
        assert abs(lp[m] - want[1]) <= 2.0 ** -23 * abs(want[1]) + x.shape[1] * 2.0 ** -42 + 1e-7, (m, lp[m], want)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1023, 4097, 50257])
@pytest.mark.parametrize("ld", [0, 1, 4])
def test_sample_settings(hip, V, ld):
    rng = np.random.default_rng(V)
    M = 24
    x = 3 * rng.standard_normal((M, V))
    check_sample(hip, x, T=rng.choice([0.0, 0.3, 1.0, 2.0], M), k=rng.choice([0, 1, 2, 40, V, V + 5], M),
                 p=rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0], M), mp=rng.choice([0.0, 0.02, 0.3, 1.0], M),
                 u=rng.random(M).astype(np.float32), ld=ld)


@pytest.mark.parametrize("M", [1, 3, 130, 600])
def test_sample_rows(hip, M):
    rng = np.random.default_rng(M)
    x = 2 * rng.standard_normal((M, 700))
    check_sample(hip, x, T=0.8, k=50, p=0.95, mp=0.05, u=rng.random(M).astype(np.float32))


def test_sample_whole_vocabulary(hip):
    rng = np.random.default_rng(2)
    V = 248320
    x = 2.5 * rng.standard_normal((4, V))
    x[0, [5, 77, V - 1]] = 12.0
    for args in (dict(), dict(k=50), dict(p=0.9), dict(mp=0.05), dict(k=1000, p=0.5, mp=0.01), dict(T=1.5, p=0.99)):
        check_sample(hip, x, u=np.array([0.0, 0.3, 0.77, 0.9999999], np.float32), **args)


def test_sample_absent_settings_and_uniforms_at_the_ends(hip):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 300))
    u = np.array([0.0, -1.0, 1.0, 5.0, np.nan, 1 - 2.0 ** -24], np.float32)
    check_sample(hip, x, u=u)
    check_sample(hip, x, u=u, k=7, p=0.8)
    nan = np.nan
    check_sample(hip, x, u=u, T=[nan, -1.0, 1.0, np.inf, 1e-30, 1e30], p=[nan, 0.5, -3.0, 2.0, 0.5, 0.5],
                 mp=[0.5, nan, -1.0, 7.0, 0.0, 0.5], k=[-1, -(2 ** 31), 2 ** 31 - 1, 0, 3, 3])


def test_sample_ties(hip):
    """Equal logits: the smaller index first, at the top-k's and the top-p's border too."""
    rng = np.random.default_rng(4)
    M, V = 40, 5000
    x = np.round(rng.standard_normal((M, V)) * 2) / 2  # a dozen values
    check_sample(hip, x, k=rng.integers(1, V, M), p=rng.choice([0.05, 0.3, 0.8, 1.0], M), u=rng.random(M).astype(np.float32))
    flat = np.full((8, 3001), -2.5)
    check_sample(hip, flat, k=[0, 1, 7, 3000, 0, 0, 100, 100], p=[1, 1, 1, 1, 0.5, 1e-5, 0.5, 0.999],
                 u=np.array([0.3, 0.9, 0.99, 0.9999, 0.9999, 0.5, 0.99, 0.99], np.float32))
    zeros = np.where(rng.random((2, 100)) < 0.5, 0.0, -0.0)  # one value, by its meaning
    check_sample(hip, zeros, k=3, u=np.array([0.5, 0.99], np.float32))


def test_sample_infinities_and_nan(hip):
    rng = np.random.default_rng(5)
    V = 2000
    x = rng.standard_normal((9, V))
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, 10:] = -np.inf
    x[3, [7, 1900]] = np.inf
    x[4, ::2] = np.nan
    x[5, :] = -np.inf
    x[5, 1234] = -1e30
    x[6, :] = np.finfo(np.float32).min
    x[7, 3], x[7, 5] = np.finfo(np.float32).max, np.finfo(np.float32).min
    x[8, :] = 1e-42
    u = np.linspace(0, 0.99, 9).astype(np.float32)
    for args in (dict(), dict(k=5), dict(p=0.6), dict(mp=0.3), dict(T=0.0), dict(T=1e-3, k=30, p=0.9)):
        check_sample(hip, x, u=u, **args)


def test_sample_far_apart_and_wide(hip):
    """Logits spread over hundreds, clusters within one part in 10^6, and many equal far ones."""
    rng = np.random.default_rng(6)
    x = np.concatenate([300 * rng.standard_normal((3, 3000)), 1000 + 1e-3 * rng.standard_normal((3, 3000)),
                        np.concatenate([np.full((3, 2990), -40.0), rng.standard_normal((3, 10))], 1)])
    for args in (dict(), dict(k=20, p=0.9), dict(p=0.999), dict(T=100.0, p=0.7), dict(T=0.01, mp=0.1)):
        check_sample(hip, x, u=rng.random(9).astype(np.float32), **args)


def test_sample_many_equal_logits_of_a_large_row(hip):
    """More logits in a border's bin than candidates are held: the row is done by its own workgroup alone."""
    rng = np.random.default_rng(14)
    x = np.round(rng.standard_normal((5, 100003)))
    check_sample(hip, x, k=[30000, 0, 30000, 1, 0], p=[1, 0.4, 0.4, 0.9, 1], mp=[0, 0, 0, 0, 0.01],
                 u=rng.random(5).astype(np.float32))


def test_sample_the_largest_vocabulary(hip):
    rng = np.random.default_rng(15)
    x = 2 * rng.standard_normal((3, 1 << 20))
    check_sample(hip, x, k=[0, 900, 0], p=[0.7, 0.9, 1.0], u=[0.2, 0.5, 0.8])


def test_sample_the_largest_sum(hip):
    """2^20 weights of one: sums up to 2^63."""
    check_sample(hip, np.zeros((4, 1 << 20)), p=[1, 1, 0.999, 0.999], u=[0.99, 1 - 2.0 ** -24, 0.99, 1 - 2.0 ** -24])


def test_sample_more_rows_than_a_grid_has(hip):
    """66001 rows, in two launches of each kernel; settings by the row."""
    rng = np.random.default_rng(18)
    M, V = 66001, 7
    x = (2 * rng.standard_normal((M, V))).astype(np.float32)
    T, k = rng.choice([0.0, 0.7, 1.5], M).astype(np.float32), rng.choice([0, 1, 3], M).astype(np.int32)
    p, mp = rng.choice([0.4, 0.9, 1.0], M).astype(np.float32), rng.choice([0.0, 0.2], M).astype(np.float32)
    u = rng.random(M).astype(np.float32)
    tok, lp = run_sample(hip, x, T, k, p, mp, u)
    for m in list(range(0, M, 97)) + list(range(65500, 65580)) + [M - 1]:
        want = ref.sample(x[m], T[m], k[m], p[m], mp[m], u[m])
        assert tok[m] == want[0] and abs(lp[m] - want[1]) <= 2.0 ** -23 * abs(want[1]) + V * 2.0 ** -42 + 1e-7, (m, want)


def test_sample_a_flat_row_beside_one_far_logit(hip):
    """A finite logit far below the others makes the bins wide: more logits lie in the border's than candidates are held."""
    rng = np.random.default_rng(19)
    x = rng.standard_normal((3, 248320)).astype(np.float32)
    x[:, 77] = -1e4
    check_sample(hip, x, T=2.0, p=[0.7, 0.5, 0.7], k=[0, 0, 200000], u=[0.1, 0.5, 0.9])


@pytest.mark.parametrize("k", [1, 2, 7, 8, 9, 500, 2000])
def test_sample_sorted_and_clustered_logits(hip, k):
    """The largest logits all next to each other: the maxima of 128 say little, top-k has to be exact all the same."""
    rng = np.random.default_rng(16)
    V = 30000
    up = np.sort(2 * rng.standard_normal(V))
    one = rng.standard_normal(V)
    one[5000:5128] += 40
    check_sample(hip, np.stack([up, up[::-1], one, one]), k=k, p=[1, 0.9, 1, 0.99], u=[0.1, 0.6, 0.9, 0.999])


def test_sample_without_logprob_and_same_result_twice(hip):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((50, 9000)).astype(np.float32)
    u = rng.random(50).astype(np.float32)
    a, _ = run_sample(hip, x, 0.9, 100, 0.95, 0.01, u)
    b, lp = run_sample(hip, x, 0.9, 100, 0.95, 0.01, u, logprob=False)
    np.testing.assert_array_equal(a, b)
    assert np.all(lp == -5.0)
    c, l1 = run_sample(hip, x, 0.9, 100, 0.95, 0.01, u)
    d, l2 = run_sample(hip, x, 0.9, 100, 0.95, 0.01, u)
    np.testing.assert_array_equal(c, d)
    np.testing.assert_array_equal(l1.view(np.uint32), l2.view(np.uint32))


def test_sample_agrees_with_the_greedy_pick(hip):
    torch = _torch()
    rng = np.random.default_rng(8)
    V = 70001
    x = rng.standard_normal((3, V)).astype(np.float32)
    x[1, [9, 400]] = 50.0
    x[2, :] = np.nan
    tok, lp = run_sample(hip, x, T=0.0, u=0.5)
    part = torch.zeros(hip.argmax_part_bytes(V) // 4, dtype=torch.int32, device="cuda")
    for m in range(3):
        out = ints([-1])
        hip.launch_argmax(dev(x[m]), V, part, out, stream())
        assert host(out)[0] == tok[m]
    assert np.all(lp == 0.0)
    k1, _ = run_sample(hip, x[:2], k=1, u=0.7)
    np.testing.assert_array_equal(k1, tok[:2])


# ---- together, as a serving loop runs them ----
class Loop:
    """Steps of a small model's one layer over a paged cache: plan, QKV rows, rope and cache write, attention, a fixed
    head product, sampling; the state (pages, lengths) stays on the device."""
    H, HK, D, page, pages, V = 10, 2, 64, 16, 64, 999

    def __init__(self, hip, S, T, kind="f16"):
        torch = _torch()
        self.hip, self.S, self.T, self.kind = hip, S, T, kind
        H, HK, D = self.H, self.HK, self.D
        z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        i32 = torch.int32
        self.k, self.v = (torch.full((self.pages, HK, self.page, D), math.nan, dtype=kind_of(kind), device="cuda")
                          for _ in range(2))
        self.kv = hip.KvCache(self.k, self.v, hip.CacheType[kind], self.page, HK, D, self.pages, HK * self.page * D,
                              self.page * D, D)
        self.ldt = 8
        self.free = ints(np.random.default_rng(1).permutation(self.pages))
        self.n_free, self.held = ints([self.pages]), z(S, t=i32)
        self.table = torch.full((S, self.ldt), -1, dtype=i32, device="cuda")
        self.ctx, self.n_new, self.parent = z(S, t=i32), z(S, t=i32), z(T, t=i32)
        self.row0, self.kv_len, self.pos, self.slot = z(S + 1, t=i32), z(S, t=i32), z(T, t=i32), z(T, t=i32)
        self.tree = z(T, t=torch.int64)
        self.qkv = z(T, (H + 2 * HK) * D)
        self.q = z(T, H * D, t=kind_of(kind))
        self.out = z(T, H * D)
        g = torch.Generator(device="cuda").manual_seed(3)
        self.head = torch.randn((H * D, self.V), generator=g, device="cuda") * 0.05
        self.logits, self.u = z(T, self.V), torch.rand((T,), generator=g, device="cuda")
        self.token, self.lp = z(T, t=i32), z(T)
        self.turns = dev(np.array(hip.rope_table(D, 1e6, hip.RopeScale(hip.RopeScaling.yarn, 4.0, 64.0))[0]))
        self.ws = words(hip.paged_attention_ws_bytes(S, T, H, self.kv))
        self.ws2 = words(hip.sample_ws_bytes(T, self.V))

    def launch(self, st):
        hip, S, T, H, HK, D = self.hip, self.S, self.T, self.H, self.HK, self.D
        hip.launch_page_plan(hip.PagePlan(
            S=S, T=T, page=self.page, ldt=self.ldt, pages=self.pages, ctx=self.ctx, n_new=self.n_new, held=self.held,
            parent=self.parent, free=self.free, n_free=self.n_free, table=self.table, held_out=self.held,
            n_free_out=self.n_free, row0=self.row0, kv_len=self.kv_len, pos=self.pos, slot=self.slot, tree=self.tree), st)
        ld = (H + 2 * HK) * D
        hip.launch_rope_cache(hip.RopeCache(
            T=T, heads=H, q=self.qkv, ldq=ld, k=self.qkv[:, H * D:], ldk=ld, v=self.qkv[:, (H + HK) * D:], ldv=ld,
            n_rot=D, layout=hip.RopeLayout.half, turns=self.turns, mscale=1.0, pos=self.pos, slot=self.slot,
            rows=self.row0[S:], q_out=self.q, ldqo=H * D), self.kv, st)
        hip.launch_paged_attention(hip.PagedAttention(
            S=S, T=T, heads=H, q=self.q, ldq=H * D, table=self.table, ldt=self.ldt, row0=self.row0, kv_len=self.kv_len,
            tree=self.tree, scale=D ** -0.5, out=self.out, ldo=H * D, ws=self.ws), self.kv, st)

    def sample(self, st):
        self.hip.launch_sample(self.hip.Sampling(
            M=self.T, V=self.V, logits=self.logits, ldl=self.V, top_k=None, top_p=None, u=self.u, token=self.token,
            logprob=self.lp, ws=self.ws2), st)

    def set(self, ctx, n_new, parent, seed):
        torch = _torch()
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx.copy_(ints(ctx))
        self.n_new.copy_(ints(n_new))
        self.parent.copy_(ints(list(parent) + [-1] * (self.T - len(parent))))
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g, device="cuda"))


STEPS = [([0, 0, 0], [20, 3, 0], [-1] * 23), ([20, 3, 0], [1, 4, 7], [-1] + [-1, 0, 0, 1] + list(range(-1, 6))),
         ([21, 5, 7], [1, 0, 1], [-1, -1]), ([22, 5, 8], [3, 2, 1], [-1, 0, 1, -1, -1, -1]), ([25, 6, 9], [6, 6, 6], [-1] * 18)]


def check_step(L, dense):
    """The step's attention from the requests' own histories: dense[s] = list of (k, v) by cache place."""
    S, H, HK, D, G = L.S, L.H, L.HK, L.D, L.H // L.HK
    row0, kv_len = host(L.row0), host(L.kv_len)
    table, tree, out = host(L.table), host(L.tree), L.out.double().cpu().numpy()
    k, v, q = (t.double().cpu().numpy() for t in (L.k, L.v, L.q))
    want, tol = ref.attention(q[:row0[S]], k, v, table, row0, kv_len, tree.view(np.uint64), D ** -0.5, L.page, L.pages, H, HK)
    d = np.abs(out[:row0[S]] - want)
    assert np.all(d <= tol + ref.HALF_STEP[L.kind] ** 2 * 8), d.max()
    for s in range(S):  # what earlier steps wrote is still where they wrote it
        ctx = int(kv_len[s]) - int(row0[s + 1] - row0[s])
        for j in range(max(0, ctx)):
            if j in dense[s]:
                np.testing.assert_array_equal(k[table[s, j // L.page], :, j % L.page], dense[s][j])
        for j in range(int(kv_len[s])):
            dense[s][j] = k[table[s, j // L.page], :, j % L.page].copy()


# strides with which the last page, token or head starts beyond 2^32 bytes
FAR = [(16, lambda HK, D, page: (2 ** 30 + 64, page * D, D)), (256, lambda HK, D, page: (HK * D, D, 2 ** 24)),
       (32, lambda HK, D, page: (page * D, 2 ** 31, D))]


def far_cache(shape, strides, kind, fill=None):
    """Two caches of (pages, heads, tokens, dim) at these strides, as flat arrays and as views of what the strides reach."""
    torch = _torch()
    flat = [torch.empty(sum((n - 1) * st for n, st in zip(shape, (*strides, 1))) + 1, dtype=kind_of(kind), device="cuda")
            for _ in range(2)]
    view = [torch.as_strided(f, shape, (*strides, 1)) for f in flat]
    for i, w in enumerate(view):
        w.copy_(fill[i]) if fill else w.zero_()
    return flat, view


@pytest.mark.parametrize("page,strides", FAR, ids=["pages", "tokens", "heads"])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_attention_offsets_beyond_32_bits(hip, page, strides, new):
    rng = np.random.default_rng(page + new)
    heads, kind = (8, 2, 128), "f16"
    kv_len = [3 * page + 7] if page < 256 else [page + 9]
    new = min(new, kv_len[0])
    q, k, v, table, row0 = attn_inputs(rng, kv_len, [new], heads, kind, page)
    flat, view = far_cache(k.shape, strides(2, 128, page), kind, (k, v))
    out = run_attn(hip, q, *flat, table, row0, kv_len, None, heads, kind, page, pages=k.shape[0], strides=strides(2, 128, page))
    check_attn(out, q, k, v, table, row0, kv_len, None, heads, kind, page)


def test_attention_rows_beyond_32_bits(hip):
    """Rows of q and out that lie gigabytes apart."""
    torch = _torch()
    rng = np.random.default_rng(16)
    heads, kind, page, kv_len, ld = (4, 2, 64), "bf16", 16, [40], 2 ** 29 + 8
    q, k, v, table, row0 = attn_inputs(rng, kv_len, [6], heads, kind, page)
    far_q = torch.as_strided(torch.empty(5 * ld + 256, dtype=q.dtype, device="cuda"), (6, 256), (ld, 1)).copy_(q)
    far_o = torch.as_strided(torch.empty(5 * ld + 256, dtype=torch.float32, device="cuda"), (6, 256), (ld, 1))
    kv = hip.KvCache(k, v, hip.CacheType[kind], page, 2, 64, k.shape[0], 2 * page * 64, page * 64, 64)
    hip.launch_paged_attention(hip.PagedAttention(
        S=1, T=6, heads=4, q=far_q, ldq=ld, table=ints(table), ldt=table.shape[1], row0=ints(row0), kv_len=ints(kv_len),
        scale=0.125, out=far_o, ldo=ld, ws=words(hip.paged_attention_ws_bytes(1, 6, 4, kv))), kv, stream())
    torch.cuda.synchronize()
    check_attn(far_o.contiguous(), q, k, v, table, row0, kv_len, None, heads, kind, page, scale=0.125)


@pytest.mark.parametrize("page,strides", FAR, ids=["pages", "tokens", "heads"])
def test_rope_offsets_beyond_32_bits(hip, page, strides):
    rng = np.random.default_rng(page)
    H, HK, D, kind, pages = 2, 2, 128, "bf16", 5 if page < 256 else 2
    flat, view = far_cache((pages, HK, page, D), strides(HK, D, page), kind)
    T = 24
    qkv, slot = rope_inputs(rng, T, H, HK, D, page, kind)[:2]
    slot = rng.permutation(pages * page)[:T]
    if pages * page - 1 not in slot:  # (no slot twice)
        slot[0] = pages * page - 1
    pos, (turns, _) = rng.integers(0, 999, T), hip.rope_table(64, 1e4)
    q = run_rope(hip, qkv, slot, flat, pages, pos, turns, H, HK, D, page, kind, 64, "half", strides=strides(HK, D, page))
    got = [w.contiguous() for w in view]
    check_rope(q, got, [w.new_zeros(w.shape) for w in got], qkv, slot, pos, turns, H, HK, D, page, kind, 64, "half")


def test_sample_rows_beyond_32_bits(hip):
    torch = _torch()
    rng = np.random.default_rng(17)
    x, ld = (2 * rng.standard_normal((3, 5000))).astype(np.float32), 2 ** 30 + 1
    far = torch.as_strided(torch.empty(2 * ld + 5000, dtype=torch.float32, device="cuda"), (3, 5000), (ld, 1)).copy_(dev(x))
    tok, u = torch.full((3,), -5, dtype=torch.int32, device="cuda"), np.array([0.1, 0.5, 0.9], np.float32)
    hip.launch_sample(hip.Sampling(M=3, V=5000, logits=far, ldl=ld, top_k=ints([0, 40, 0]), top_p=dev(np.array([1, 1, 0.8], np.float32)),
                                   u=dev(u), token=tok, ws=words(hip.sample_ws_bytes(3, 5000))), stream())
    want = [ref.sample(x[m], 1.0, [0, 40, 0][m], np.float32([1, 1, 0.8][m]), 0.0, u[m])[0] for m in range(3)]
    assert host(tok).tolist() == want


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "captured"])
def test_serving_steps(hip, graph):
    """Prompt, drafted trees, single tokens and idle requests in turn; one graph captured once serves every step."""
    torch = _torch()
    L = Loop(hip, 3, 32)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    if graph:
        g = hip.Graph(st)
        with g:
            L.launch(st)
        g2 = hip.Graph(st)
        with g2:
            L.sample(st)
    dense = [{}, {}, {}]
    for n, (ctx, new, parent) in enumerate(STEPS):
        L.set(ctx, new, parent, 100 + n)
        torch.cuda.synchronize()
        if graph:
            g.launch()
        else:
            L.launch(st)
        torch.cuda.synchronize()
        check_step(L, dense)
        L.logits.copy_(L.out @ L.head)  # rows behind the last one hold what earlier steps left: finite
        torch.cuda.synchronize()
        if graph:
            g2.launch()
        else:
            L.sample(st)
        torch.cuda.synchronize()
        tok, x, u = host(L.token), host(L.logits), host(L.u)
        for r in range(int(host(L.row0)[-1])):
            assert tok[r] == ref.sample(x[r], 1.0, 0, 1.0, 0.0, u[r])[0]


def test_two_streams_with_their_own_workspaces(hip):
    """The same launches on two streams at once, each with its own outputs and workspace, give the eager results."""
    torch = _torch()
    rng = np.random.default_rng(20)
    heads, page, kind = (20, 4, 128), 64, "bf16"
    kv_len, new = [900, 40, 2000], [1, 1, 1]
    x = attn_inputs(rng, kv_len, new, heads, kind, page)
    y = attn_inputs(rng, kv_len[::-1], new, heads, kind, page)
    want = [run_attn(hip, *a, n, None, heads, kind, page) for a, n in ((x, kv_len), (y, kv_len[::-1]))]
    H, HK, D = heads
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    calls, outs = [], []
    for a, n in ((x, kv_len), (y, kv_len[::-1])):
        q, k, v, table, row0 = a
        kv = hip.KvCache(k, v, hip.CacheType[kind], page, HK, D, k.shape[0], HK * page * D, page * D, D)
        out = torch.zeros((3, H * D), device="cuda")
        outs.append(out)
        calls.append((hip.PagedAttention(S=3, T=3, heads=H, q=q, ldq=H * D, table=ints(table), ldt=table.shape[1],
                                         row0=ints(row0), kv_len=ints(n), scale=D ** -0.5, out=out, ldo=H * D,
                                         ws=words(hip.paged_attention_ws_bytes(3, 3, H, kv))), kv))
    torch.cuda.synchronize()
    for _ in range(20):
        for (a, kv), s in zip(calls, streams):
            hip.launch_paged_attention(a, kv, s)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_graph_replays_equal_eager(hip):
    """Attention and sampling captured, replayed with other work between, inputs changed in place."""
    torch = _torch()
    rng = np.random.default_rng(21)
    heads, page, kind, kv_len, new = (10, 2, 256), 32, "f16", [3000, 77], [1, 2]
    H, HK, D = heads
    q, k, v, table, row0 = attn_inputs(rng, kv_len, new, heads, kind, page)
    kv = hip.KvCache(k, v, hip.CacheType[kind], page, HK, D, k.shape[0], HK * page * D, page * D, D)
    out, lens = torch.zeros((3, H * D), device="cuda"), ints(kv_len)
    a = hip.PagedAttention(S=2, T=3, heads=H, q=q, ldq=H * D, table=ints(table), ldt=table.shape[1], row0=ints(row0),
                           kv_len=lens, scale=D ** -0.5, out=out, ldo=H * D, ws=words(hip.paged_attention_ws_bytes(2, 3, H, kv)))
    V = 30001
    logits, u = torch.randn((3, V), device="cuda"), torch.rand(3, device="cuda")
    tok = ints([0, 0, 0])
    b = hip.Sampling(M=3, V=V, logits=logits, ldl=V, top_k=ints([0, 40, 7]), top_p=dev(np.float32([0.9, 0.5, 1.0])), u=u,
                     token=tok, ws=words(hip.sample_ws_bytes(3, V)))
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = hip.Graph(st)
    with g:
        hip.launch_paged_attention(a, kv, st)
        hip.launch_sample(b, st)
    for n in range(4):
        lens.copy_(ints([3000 - 700 * n, 77 + n]))
        logits.copy_(torch.randn((3, V), device="cuda") * (1 + n))
        torch.cuda.synchronize()
        g.launch()
        torch.cuda.synchronize()
        o1, t1 = out.clone(), tok.clone()
        out.zero_()
        tok.zero_()
        torch.cuda.synchronize()
        hip.launch_paged_attention(a, kv, st)
        hip.launch_sample(b, st)
        torch.cuda.synchronize()
        assert torch.equal(o1, out) and torch.equal(t1, tok)
