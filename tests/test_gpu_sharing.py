"""GPU test of the operators for requests that share, together as a serving loop runs them: forks and their copies, the page
plan, adapters beside QKV, rope and cache write, attention behind shared prefixes, the accepted path's move, pages given back."""
import math

import numpy as np
import pytest

import serving_ref
import sharing_ref as ref
from test_gpu_lora import tol as lora_tol
from test_gpu_serving import dev, host, ints, kind_of, words

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


class Loop:
    """Steps of a small model's attention layers; pages, counts and lengths stay on the device."""
    S, T, H, HK, D, K, rank, adapters, layers, page, pages, ldt, F = 6, 48, 10, 2, 64, 96, 16, 3, 2, 16, 40, 8, 4

    def __init__(self, hip, kind):
        torch = _torch()
        self.hip, self.kind = hip, kind
        S, T, H, HK, D, F = self.S, self.T, self.H, self.HK, self.D, self.F
        i32, t16 = torch.int32, kind_of(kind)
        z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        rng = np.random.default_rng(2)
        self.k, self.v = (torch.full((self.layers, self.pages, HK, self.page, D), math.nan, dtype=t16, device="cuda") for _ in range(2))
        self.stride = self.pages * HK * self.page * D
        self.kv = [hip.KvCache(self.k[l], self.v[l], hip.CacheType[kind], self.page, HK, D, self.pages, HK * self.page * D,
                               self.page * D, D) for l in range(self.layers)]
        self.free, self.n_free = ints(rng.permutation(self.pages)), ints([self.pages])
        self.table = torch.full((S, self.ldt), -1, dtype=i32, device="cuda")
        self.held, self.shared = z(S, t=i32), z(self.pages, t=i32)
        self.src, self.dst, self.tokens, self.got = (z(F, t=i32) for _ in range(4))
        self.copy = [z(F, t=i32) for _ in range(3)]
        self.ctx, self.n_new, self.parent = z(S, t=i32), z(S, t=i32), z(T, t=i32)
        self.row0, self.kv_len, self.pos, self.slot = z(S + 1, t=i32), z(S, t=i32), z(T, t=i32), z(T, t=i32)
        self.tree, self.leaf, self.after = z(T, t=torch.int64), z(S, t=i32), z(S, t=i32)
        self.group0, self.lead, self.prefix = z(4, t=i32), z(3, t=i32), z(3, t=i32)
        self.x, self.who = z(T, self.K), ints([0, 1, -1, 2, 1, 0])
        self.ranks, self.scale = ints([16, 5, 9]), dev(np.array([1.5, -0.5, 2.0], np.float32))
        self.Ns = [H * D, HK * D, HK * D]
        self.a = [[torch.from_numpy(rng.standard_normal((self.adapters, self.rank, self.K)) * 0.1).to(t16).cuda() for _ in self.Ns]
                  for _ in range(self.layers)]
        self.b = [[torch.from_numpy(rng.standard_normal((self.adapters, n, self.rank)) * 0.3).to(t16).cuda() for n in self.Ns]
                  for _ in range(self.layers)]
        self.qkv, self.q, self.out = z(self.layers, T, sum(self.Ns)), z(self.layers, T, H * D, t=t16), z(self.layers, T, H * D)
        self.turns = dev(np.array(hip.rope_table(D, 1e6)[0]))
        self.ws = words(hip.shared_attention_ws_bytes(S, T, H, self.kv[0]))
        self.ws_lora = words(hip.lora_ws_bytes(S, T, self.K, self.rank, 3))
        self.ws_free = words(hip.page_free_ws_bytes(S, self.ldt))

    def forks(self, st):
        hip = self.hip
        hip.launch_page_fork(hip.PageFork(
            F=self.F, S=self.S, page=self.page, ldt=self.ldt, pages=self.pages, src=self.src, dst=self.dst, tokens=self.tokens,
            free=self.free, n_free=self.n_free, table=self.table, held=self.held, shared=self.shared, got=self.got,
            copy_from=self.copy[0], copy_to=self.copy[1], copy_tokens=self.copy[2]), st)
        hip.launch_page_copy(hip.PageCopy(n=self.F, source=self.copy[0], to=self.copy[1], tokens=self.copy[2],
                                          layers=self.layers, layer_stride=self.stride), self.kv[0], st)

    def step(self, st):
        hip, S, T, H, HK, D = self.hip, self.S, self.T, self.H, self.HK, self.D
        hip.launch_page_plan(hip.PagePlan(
            S=S, T=T, page=self.page, ldt=self.ldt, pages=self.pages, ctx=self.ctx, n_new=self.n_new, held=self.held,
            parent=self.parent, free=self.free, n_free=self.n_free, table=self.table, held_out=self.held,
            n_free_out=self.n_free, row0=self.row0, kv_len=self.kv_len, pos=self.pos, slot=self.slot, tree=self.tree), st)
        ld, at = sum(self.Ns), np.cumsum([0] + self.Ns)
        for l, kv in enumerate(self.kv):
            part = [self.qkv[l][:, c:] for c in at[:3]]
            hip.launch_lora(hip.Lora(
                S=S, T=T, K=self.K, rank=self.rank, adapters=self.adapters, type=hip.CacheType[self.kind], row0=self.row0,
                adapter=self.who, ranks=self.ranks, scale=self.scale, x=self.x, ldx=self.K, ws=self.ws_lora), [
                    hip.LoraSeg(a=a, b=b, a_stride=a[0].numel(), b_stride=b[0].numel(), N=n, y=y, ldy=ld)
                    for a, b, n, y in zip(self.a[l], self.b[l], self.Ns, part)], st)
            hip.launch_rope_cache(hip.RopeCache(
                T=T, heads=H, q=part[0], ldq=ld, k=part[1], ldk=ld, v=part[2], ldv=ld, n_rot=D, layout=hip.RopeLayout.half,
                turns=self.turns, pos=self.pos, slot=self.slot, rows=self.row0[S:], q_out=self.q[l], ldqo=H * D), kv, st)
            hip.launch_shared_attention(hip.SharedAttention(
                S=S, T=T, heads=H, q=self.q[l], ldq=H * D, table=self.table, ldt=self.ldt, row0=self.row0, kv_len=self.kv_len,
                tree=self.tree, scale=D ** -0.5, out=self.out[l], ldo=H * D, ws=self.ws, groups=3, group0=self.group0,
                lead=self.lead, shared=self.prefix), kv, st)

    def accept(self, st):
        hip = self.hip
        hip.launch_cache_move(hip.CacheMove(
            S=self.S, T=self.T, table=self.table, ldt=self.ldt, first=self.ctx, tree=self.tree, leaf=self.leaf, kv_len=self.after,
            layers=self.layers, layer_stride=self.stride), self.kv[0], st)

    def give_back(self, st):  # (self.after: what the caller keeps, 0 for a request that has ended)
        hip = self.hip
        hip.launch_page_free(hip.PageFree(
            S=self.S, page=self.page, ldt=self.ldt, pages=self.pages, keep=self.after, table=self.table, held=self.held,
            shared=self.shared, free=self.free, n_free=self.n_free, ws=self.ws_free), st)

    def state(self):
        return [t.clone() for t in (self.k, self.v, self.table, self.held, self.shared, self.n_free, self.row0, self.kv_len, self.after,
                                    self.got, self.qkv, self.out, self.slot)]


# Each step: forks (source, new row, tokens), new tokens a request, parents of its rows, its leaf among them (-1: none taken),
# groups (starts, lead, prefix), requests that end behind it.
CHAIN = lambda n: list(range(-1, n - 1))  # noqa: E731
STEPS = [
    ([], [30, 0, 0, 0, 18, 0], [CHAIN(30), [], [], [], CHAIN(18), []], [29, -1, -1, -1, 17, -1], ([0, 0, 0, 0], [0, 0, 0], [0, 0, 0]), []),
    ([(0, 1, 30), (0, 2, 30), (0, 3, 33), (4, 5, 16)], [1, 2, 1, 0, 1, 1], [[-1], CHAIN(2), [-1], [], [-1], [-1]],
     [0, 1, 0, -1, 0, 0], ([0, 4, 6, 6], [0, 4, 0], [30, 16, 0]), []),
    ([(0, 3, 31)], [4, 7, 1, 5, 0, 9], [[-1, 0, 0, 1], [-1, 0, 0, 1, 2, 4, 4], [-1], [-1, -1, 1, 0, 3], [], [-1, 0, 1, 1, 2, 3, 3, 6, 6]],
     [3, 6, 0, 4, -1, 8], ([0, 4, 6, 6], [1, 4, 0], [30, 16, 0]), [2]),
    ([(1, 2, 17)], [1, 1, 3, 12, 1, 1], [[-1], [-1], CHAIN(3), [-1] + [0] * 11, [-1], [-1]], [0, 0, 1, 5, 0, -1],
     ([0, 2, 4, 6], [0, 1, 5], [30, 17, 16]), [0]),
    ([(2, 0, 18), (2, 2, 4), (9, 1, 1)], [2, 1, 1, 1, 20, 0], [CHAIN(2), [-1], [-1], [-1], CHAIN(20), []], [1, 0, 0, 0, 19, -1],
     ([0, 3, 6, 6], [2, 4, 0], [17, 16, 0]), [0, 1, 2, 3, 4, 5])]


def fill(L, n, ctx):
    torch = _torch()
    forks, new, parents, leaf, (group0, lead, prefix), _ = STEPS[n]
    pad = lambda a, m, v: list(a) + [v] * (m - len(a))  # noqa: E731
    for t, i in ((L.src, 0), (L.dst, 1), (L.tokens, 2)):
        t.copy_(ints(pad([f[i] for f in forks], L.F, -1)))
    L.n_new.copy_(ints(new))
    L.parent.copy_(ints(pad(sum(parents, []), L.T, -1)))
    at = np.cumsum([0] + new)
    L.leaf.copy_(ints([at[s] + m if m >= 0 else -1 for s, m in enumerate(leaf)]))
    L.group0.copy_(ints(group0)), L.lead.copy_(ints(lead)), L.prefix.copy_(ints(prefix))
    L.ctx.copy_(ints(ctx))
    g = torch.Generator(device="cuda").manual_seed(40 + n)
    L.qkv.copy_(torch.randn(L.qkv.shape, generator=g, device="cuda"))
    L.x.copy_(torch.randn(L.x.shape, generator=g, device="cuda"))
    torch.cuda.synchronize()


def pages_add_up(L):
    """Each page is free or held by one request more than shared says."""
    table, held, shared = host(L.table), host(L.held), host(L.shared)
    count = np.zeros(L.pages, int)
    for s in range(L.S):
        np.add.at(count, table[s, :held[s]], 1)
    free = host(L.free)[:int(host(L.n_free)[0])]
    assert len(set(free.tolist())) == len(free) and np.all(count[free] == 0) and np.all(shared[free] == 0)
    used = np.setdiff1d(np.arange(L.pages), free)
    np.testing.assert_array_equal(count[used], shared[used] + 1)


def tokens_of(L, s, n):
    """K and V of request s's first n tokens, all layers."""
    table = host(L.table)
    return [np.stack([t[:, table[s, j // L.page], :, j % L.page].double().cpu().numpy() for j in range(n)]) if n else np.zeros((0,))
            for t in (L.k, L.v)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_requests_that_share(hip, kind):
    """Five steps, eager and as four graphs captured once: the same bits; each part against its plain form."""
    torch = _torch()
    both = [Loop(hip, kind), Loop(hip, kind)]
    L, st = both[0], torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    for f in (both[1].forks, both[1].step, both[1].accept, both[1].give_back):
        g = hip.Graph(st)
        with g:
            f(st)
        graphs.append(g)

    def run(i, name):
        torch.cuda.synchronize()
        getattr(L, name)(st)
        graphs[i].launch()
        torch.cuda.synchronize()
        for x, y in zip(both[0].state(), both[1].state()):
            assert torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0))

    ctx, have = np.zeros(L.S, int), [None] * L.S  # tokens of each request's cache, and what they hold
    for n, (forks, new, parents, leaf, _, ends) in enumerate(STEPS):
        for l in both:
            fill(l, n, ctx)
        run(0, "forks")
        want = [m if s != d and 0 <= s < L.S and m <= -(-ctx[s] // L.page) * L.page and ctx[d] == 0 else -1 for s, d, m in forks]
        assert host(L.got).tolist() == want + [-1] * (L.F - len(forks))
        for (s, d, _), m in zip(forks, want):
            if m >= 0:
                ctx[d] = min(m, ctx[s])
                have[d] = [t[:ctx[d]] for t in have[s]]
        pages_add_up(L)
        for l in both:
            l.ctx.copy_(ints(ctx))
        before = L.qkv.double().cpu().numpy()
        run(1, "step")
        row0, kv_len, table = host(L.row0), host(L.kv_len), host(L.table)
        assert row0.tolist() == np.cumsum([0] + new).tolist() and kv_len.tolist() == (ctx + new).tolist()
        pages_add_up(L)
        at, x, who = np.cumsum([0] + L.Ns), host(L.x), host(L.who)
        for l in range(L.layers):
            qkv = L.qkv[l].double().cpu().numpy()
            for i in range(3):
                a, b = (t[l][i].double().cpu().numpy() for t in (L.a, L.b))
                delta, deep, flat = ref.lora(x, row0, who, host(L.ranks), host(L.scale), a, b, L.T)
                y = before[l][:, at[i]:at[i + 1]]
                assert np.all(np.abs(qkv[:, at[i]:at[i + 1]] - (y + delta)) <= lora_tol(L.K, L.rank, kind, deep, flat, y, delta))
            q, k, v, out = (t[l].double().cpu().numpy() for t in (L.q, L.k, L.v, L.out))
            m = row0[-1]
            want, t = serving_ref.attention(q[:m], k, v, table, row0, kv_len, host(L.tree).view(np.uint64), L.D ** -0.5, L.page, L.pages,
                                            L.H, L.HK)
            assert np.all(np.abs(out[:m] - want) <= t + serving_ref.HALF_STEP[kind] ** 2 * 8)
        for s in range(L.S):  # nothing that was there has changed
            if ctx[s]:
                for x, y in zip(tokens_of(L, s, ctx[s]), have[s]):
                    np.testing.assert_array_equal(x, y)
        paths = []
        for s in range(L.S):
            path, r = [], leaf[s]
            while r >= 0:
                path.append(r)
                r = parents[s][r]
            every = tokens_of(L, s, kv_len[s])
            paths.append([t[list(range(ctx[s])) + [ctx[s] + r for r in path[::-1]]] for t in every] if kv_len[s] else None)
            ctx[s] += len(path)
        run(2, "accept")
        assert host(L.after).tolist() == ctx.tolist()
        for s in range(L.S):
            if ctx[s]:
                for x, y in zip(tokens_of(L, s, ctx[s]), paths[s]):
                    np.testing.assert_array_equal(x, y)
        ctx[ends] = 0
        for l in both:
            l.after[torch.tensor(ends, dtype=torch.long, device="cuda")] = 0
        run(3, "give_back")
        pages_add_up(L)
        assert host(L.held).tolist() == [ref.pages_of(c, L.page) for c in ctx]
        have = paths
    assert host(L.n_free)[0] == L.pages and not host(L.shared).any()


def test_two_streams(hip):
    """Two loops, each with a workspace of its own, at once on two streams: what each gives alone."""
    torch = _torch()
    alone, loops = [Loop(hip, k) for k in ("f16", "bf16")], [Loop(hip, k) for k in ("f16", "bf16")]
    streams = [torch.cuda.Stream() for _ in loops]
    ctx = np.zeros(Loop.S, int)
    for n in (0, 1):
        for L in alone + loops:
            fill(L, n, ctx)
        if n:  # as the first step left them
            ctx[1], ctx[2], ctx[5] = 30, 30, 16
        at = ints(ctx)
        for L in alone:
            for part in (L.forks, lambda st, L=L: L.ctx.copy_(at), L.step, L.accept, L.give_back):
                part(torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
        for L, st in zip(loops, streams):
            with torch.cuda.stream(st):
                L.forks(st)
                L.ctx.copy_(at)
                for part in (L.step, L.accept, L.give_back):
                    part(st)
        torch.cuda.synchronize()
        for x, y in zip(alone, loops):
            for a, b in zip(x.state(), y.state()):
                assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))
        ctx = host(alone[0].after).astype(int)
