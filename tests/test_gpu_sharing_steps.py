"""GPU tests of what a serving loop over shared pages must not lose (include/btf/hip_abi.h, requests that share): a request
cut back inside a page that others hold, the pages of a request that the free list did not reach for."""
import numpy as np
import pytest

import serving_ref
import sharing_ref as ref
from test_gpu_pages import State, pool
from test_gpu_serving import check_plan, dev, host, ints, kind_of, plan_case, stream

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def run_plan(hip, ctx, n_new, held, parent, free, n_free, table, T, page, pages, shared):
    torch = _torch()
    S, ldt = table.shape
    full = lambda n, t=torch.int32: torch.full((max(1, n),), -9, dtype=t, device="cuda")  # noqa: E731
    d = {"table": ints(table), "held_out": full(S), "n_free_out": full(1), "row0": full(S + 1), "kv_len": full(S), "pos": full(T),
         "slot": full(T), "tree": full(T, torch.int64)}
    hip.launch_page_plan(hip.PagePlan(
        S=S, T=T, page=page, ldt=ldt, pages=pages, ctx=ints(ctx), n_new=ints(n_new), held=ints(held),
        parent=ints(parent) if parent is not None else None, free=ints(free), n_free=ints([n_free]), table=d["table"],
        held_out=d["held_out"], n_free_out=d["n_free_out"], row0=d["row0"], kv_len=d["kv_len"], pos=d["pos"], slot=d["slot"],
        tree=d["tree"] if parent is not None else None, shared=ints(shared) if shared is not None else None), stream())
    return {n: host(t) for n, t in d.items()}


@pytest.mark.parametrize("S,page,ctx_hi,new_hi,tree,spare", [
    (1, 16, 30, 1, False, 1), (5, 16, 60, 40, True, 1), (64, 64, 500, 3, False, 1), (60, 16, 90, 200, True, 0.7),
    (200, 32, 200, 20, True, 1), (1024, 16, 60, 4, False, 0.8), (2500, 16, 50, 3, True, 1), (6, 16, 40, 3000, False, 1)])
def test_plan_gives_out_no_shared_page(hip, S, page, ctx_hi, new_hi, tree, spare):
    """Requests that go on inside a page with other holders, or that hold such pages behind their last token, are refused;
    full shared pages before it, and any counts without `shared`, change nothing."""
    rng = np.random.default_rng(S * 100 + page)
    ctx, n_new, held, parent, free, n_free, table, T, page, pages = plan_case(rng, S, page, ctx_hi, new_hi, tree, spare)
    cut = rng.random(S) < 0.4
    ctx = np.where(cut, rng.integers(0, ctx + 1), ctx)
    shared = rng.integers(-1, 3, pages) * (rng.random(pages) < 0.5)
    table[rng.random(table.shape) < 0.02] = pages + 3  # (no page of the cache: nobody else's either)
    c = (ctx, n_new, held, parent, free, n_free, table, T, page, pages)
    check_plan(run_plan(hip, *c, None), serving_ref.plan(*c), T, tree)
    theirs = np.zeros(S, bool)
    for s in range(S):
        for j in range(ctx[s] // page, min(held[s], -(-(ctx[s] + n_new[s]) // page)) if n_new[s] else 0):
            theirs[s] |= table[s, j] < pages and shared[table[s, j]] > 0
    assert S == 1 or 0 < theirs.sum() < S
    check_plan(run_plan(hip, *c, shared), serving_ref.plan(np.where(theirs, -1, ctx), *c[1:]), T, tree)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_request_cut_back_inside_a_shared_page(hip, kind):
    """Two requests of 128 tokens in the same two pages, the second cut back to 100: it does not write over the first one's
    token 100, and goes on from a fork into an empty row."""
    torch = _torch()
    rng = np.random.default_rng(7)
    HK, D, page, keep = 2, 64, 64, 100
    table, held, free, n_free, shared, pages = pool(rng, [128], 3, page, 4, 1)
    st = State(hip, table, held, free, n_free, shared, pages, page)
    k, v = (torch.from_numpy(rng.standard_normal((pages, HK, page, D))).to(kind_of(kind)).cuda() for _ in range(2))
    kv = hip.KvCache(k, v, hip.CacheType[kind], page, HK, D, pages, HK * page * D, page * D, D)
    st.fork([0], [1], [128])
    first = k.clone(), v.clone()

    def step(ctx, n_new):
        """A step's plan and cache write, its values; slots and lengths."""
        T = sum(n_new)
        d = {n: ints(np.full(m, -9)) for n, m in (("row0", 4), ("kv_len", 3), ("pos", T), ("slot", T))}
        hip.launch_page_plan(hip.PagePlan(
            S=3, T=T, page=page, ldt=st.ldt, pages=pages, ctx=ints(ctx), n_new=ints(n_new), held=st.held, free=st.free, n_free=st.n_free,
            table=st.table, held_out=st.held, n_free_out=st.n_free, shared=st.shared, **d), stream())
        x = torch.from_numpy(rng.standard_normal((2, T, HK * D)).astype(np.float32)).cuda()
        hip.launch_rope_cache(hip.RopeCache(T=T, heads=1, k=x[0], ldk=HK * D, v=x[1], ldv=HK * D, n_rot=D, layout=hip.RopeLayout.half,
                                            turns=dev(np.zeros(D // 2)), pos=d["pos"], slot=d["slot"]), kv, stream())
        return x.to(k.dtype).double().cpu().numpy().reshape(2, T, HK, D), host(d["slot"]), host(d["kv_len"])

    st.give_back([2 ** 31 - 1, keep, 0])
    _, slot, kv_len = step([128, keep, 0], [0, 3, 0])
    assert kv_len.tolist() == [128, 0, 0] and slot.tolist() == [-1] * 3
    assert torch.equal(k, first[0]) and torch.equal(v, first[1])
    out = st.fork([1], [2], [keep])
    hip.launch_page_copy(hip.PageCopy(n=1, source=out["copy_from"], to=out["copy_to"], tokens=out["copy_tokens"]), kv, stream())
    st.give_back([2 ** 31 - 1, 0, 2 ** 31 - 1])
    new, slot, kv_len = step([128, 0, keep], [1, 0, 3])
    assert host(out["got"]).tolist() == [keep] and kv_len.tolist() == [129, 0, keep + 3] and np.all(slot >= 0)
    t, counts = host(st.table), host(st.shared)
    for x, old, add in zip((k, v), first, new):
        x, old = x.double().cpu().numpy(), old.double().cpu().numpy()
        for s, n, rows in ((0, 128, add[:1]), (2, keep, add[1:])):  # what each has, then its new tokens
            for j in range(n + len(rows)):
                want = rows[j - n] if j >= n else old[table[0, j // page], :, j % page]
                np.testing.assert_array_equal(x[t[s, j // page], :, j % page], want)
    assert counts[t[0, 0]] == 1 and counts.sum() == 1 and ref.pages_of(keep + 3, page) == host(st.held)[2]


class Steps:
    """Plans, cache writes, moves and returns of three requests over a small pool, nothing of it on the host."""
    S, T, HK, D, page, pages, ldt = 3, 128, 1, 64, 16, 8, 7

    def __init__(self, hip):
        torch = _torch()
        self.hip, z = hip, lambda n, t=torch.int32: torch.zeros(n, dtype=t, device="cuda")  # noqa: E731
        self.k, self.v = (torch.zeros((self.pages, self.HK, self.page, self.D), device="cuda").half() for _ in range(2))
        self.kv = hip.KvCache(self.k, self.v, hip.CacheType.f16, self.page, self.HK, self.D, self.pages, self.HK * self.page * self.D,
                              self.page * self.D, self.D)
        self.table = torch.full((self.S, self.ldt), -1, dtype=torch.int32, device="cuda")
        self.free, self.n_free, self.held, self.shared = ints(np.arange(self.pages)), ints([self.pages]), z(self.S), z(self.pages)
        self.ctx, self.row0, self.kv_len, self.stay = z(self.S), z(self.S + 1), z(self.S), z(self.S)
        self.pos, self.slot, self.tree = z(self.T), z(self.T), z(self.T, torch.int64)
        self.ws = z(max(1, hip.page_free_ws_bytes(self.S, self.ldt) // 4))
        self.wrote = 0

    def step(self, n_new, parent=None):
        """New tokens of values 1, 2, ... (what each request's should be is up to the test)."""
        hip, HD = self.hip, self.HK * self.D
        common = dict(S=self.S, page=self.page, ldt=self.ldt, pages=self.pages, table=self.table)
        hip.launch_page_plan(hip.PagePlan(
            T=self.T, ctx=self.ctx, n_new=ints(n_new), held=self.held, parent=ints(parent) if parent is not None else None, free=self.free,
            n_free=self.n_free, held_out=self.held, n_free_out=self.n_free, row0=self.row0, kv_len=self.kv_len, pos=self.pos,
            slot=self.slot, tree=self.tree if parent is not None else None, shared=self.shared, **common), stream())
        x = (_torch().arange(self.T, device="cuda") + self.wrote + 1).float()[:, None].repeat(1, HD)
        self.wrote += sum(n_new)
        hip.launch_rope_cache(hip.RopeCache(T=self.T, heads=1, k=x, ldk=HD, v=x, ldv=HD, n_rot=2, turns=dev(np.zeros(1)), pos=self.pos,
                                            slot=self.slot, rows=self.row0[self.S:]), self.kv, stream())

    def give_back(self):
        hip = self.hip
        hip.launch_page_free(hip.PageFree(
            S=self.S, page=self.page, ldt=self.ldt, pages=self.pages, keep=self.stay, table=self.table, held=self.held, shared=self.shared,
            free=self.free, n_free=self.n_free, ws=self.ws), stream())

    def tokens(self, s, n):
        t, v = host(self.table), self.v.float().cpu().numpy()
        return [int(v[t[s, j // self.page], 0, j % self.page, 0]) for j in range(n)]


def test_a_refused_request_keeps_its_cache(hip):
    """Steps without trees, what stays worked out from the plan's lengths and the tokens before: the request that the free
    pages do not reach for has its tokens when there are pages again."""
    L = Steps(hip)

    def behind(ended=()):
        L.stay.copy_(_torch().where(L.kv_len > 0, L.kv_len, L.ctx))
        L.stay[list(ended)] = 0
        L.give_back()
        L.ctx.copy_(L.stay)

    L.step([48, 32, 40])  # 3 + 2 + 3 pages: all there are
    behind()
    assert host(L.held).tolist() == [3, 2, 3] and host(L.n_free)[0] == 0
    L.step([0, 1, 1])  # request 1 needs a third page
    assert host(L.kv_len).tolist() == [48, 0, 41]
    behind(ended=[0])
    assert host(L.held).tolist() == [0, 2, 3] and host(L.n_free)[0] == 3 and host(L.ctx).tolist() == [0, 32, 41]
    assert L.tokens(1, 32) == list(range(49, 81))
    L.step([0, 1, 0])
    assert host(L.kv_len).tolist() == [0, 33, 41] and L.tokens(1, 33) == list(range(49, 81)) + [123]
    assert L.tokens(2, 41) == list(range(81, 121)) + [122]


def test_a_refused_request_and_a_prompt_beside_a_tree(hip):
    """A step with trees: the move leaves the plan's lengths as they are, says ctx for the refused request, and for the
    prompt of more than 64 rows, whose stay is the program's to set."""
    L = Steps(hip)
    L.step([0, 16, 2], np.full(L.T, -1))
    L.stay.copy_(L.kv_len)
    L.give_back()
    L.ctx.copy_(L.stay)
    L.free[6:], L.n_free[0] = -1, 5  # (one page is somebody else's)
    L.step([70, 1, 3], np.array([-1] * 72 + [0, 0] + [-1] * 54))  # 5 pages for the prompt, none left for request 1
    hip.launch_cache_move(hip.CacheMove(S=3, T=L.T, table=L.table, ldt=L.ldt, first=L.ctx, tree=L.tree, leaf=ints([69, 70, 73]),
                                        kv_len=L.stay), L.kv, stream())
    assert host(L.kv_len).tolist() == [70, 0, 5] and host(L.stay).tolist() == [0, 16, 4]
    L.stay[0] = L.kv_len[0]
    L.give_back()
    assert host(L.held).tolist() == [5, 1, 1] and host(L.n_free)[0] == 0
    assert L.tokens(0, 70) == list(range(19, 89)) and L.tokens(1, 16) == list(range(1, 17)) and L.tokens(2, 4) == [17, 18, 90, 92]
