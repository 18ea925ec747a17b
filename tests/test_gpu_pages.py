"""GPU tests of pages that several requests hold (launch_page_fork, launch_page_copy, launch_page_free) and of tokens
that change their places (launch_cache_move), against plain references on the host (sharing_ref.py): whole numbers
and bytes, equal to the last bit."""
import dataclasses

import numpy as np
import pytest

import sharing_ref as ref

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def ints(a):
    return _torch().from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def host(t):
    _torch().cuda.synchronize()
    return t.cpu().numpy()


def stream():
    return _torch().cuda.current_stream().cuda_stream


def pool(rng, tokens, rows, page, more, ldt_more=0):
    """Rows of table that hold pages for `tokens` (then empty ones, `rows` in all), and the free list."""
    held = np.zeros(rows, np.int64)
    held[:len(tokens)] = [ref.pages_of(t, page) for t in tokens]
    pages, ldt = int(held.sum()) + more, int(max(1, held.max())) + ldt_more
    perm, table, at = rng.permutation(pages), np.full((rows, ldt), -1), 0
    for s in range(rows):
        table[s, :held[s]] = perm[at:at + held[s]]
        at += int(held[s])
    free = np.full(pages, -3)
    free[:pages - at] = perm[at:]
    return table, held, free, pages - at, np.zeros(pages, np.int64), pages


class State:
    """A pool on the device."""

    def __init__(self, hip, table, held, free, n_free, shared, pages, page):
        self.hip, self.page, self.pages = hip, page, pages
        self.S, self.ldt = table.shape
        self.table, self.held, self.free, self.n_free, self.shared = (ints(x) for x in (table, held, free, [n_free], shared))

    def fork(self, src, dst, tokens):
        F = len(src)
        out = {n: ints(np.full(F, -9)) for n in ("got", "copy_from", "copy_to", "copy_tokens")}
        self.hip.launch_page_fork(self.hip.PageFork(
            F=F, S=self.S, page=self.page, ldt=self.ldt, pages=self.pages, src=ints(src), dst=ints(dst), tokens=ints(tokens),
            free=self.free, n_free=self.n_free, table=self.table, held=self.held, shared=self.shared, **out), stream())
        return out

    def give_back(self, keep, shared=True):
        n = self.hip.page_free_ws_bytes(self.S, self.ldt)
        ws = ints(np.full(max(1, n // 4), -1))
        self.hip.launch_page_free(self.hip.PageFree(
            S=self.S, page=self.page, ldt=self.ldt, pages=self.pages, keep=ints(keep), table=self.table, held=self.held,
            shared=self.shared if shared else None, free=self.free, n_free=self.n_free, ws=ws), stream())

    def values(self):
        return {n: host(getattr(self, n)) for n in ("table", "held", "free", "n_free", "shared")}


def same(got, want):
    for n, w in want.items():
        if w is not None:
            np.testing.assert_array_equal(host(got[n]) if not isinstance(got[n], np.ndarray) else got[n], w, err_msg=n)


@pytest.mark.parametrize("S,F,page,hi,spare", [(1, 1, 16, 40, 9), (1, 4, 64, 1000, 9), (3, 7, 16, 300, 2), (8, 64, 64, 4000, 80),
                                               (5, 64, 16, 200, 10), (4, 65, 256, 3000, 70), (9, 300, 16, 900, 320),
                                               (2, 1024, 32, 100, 1100), (2, 1024, 32, 6000, 500), (6, 40, 1, 30, 0)])
def test_fork_and_free(hip, S, F, page, hi, spare):
    """Forks of random lengths, too few pages for some; then some rows give up some of what they hold, then all do."""
    rng = np.random.default_rng(S * 1000 + F)
    tokens = rng.integers(0, hi + 1, S)
    tokens[0] = hi
    table, held, free, n_free, shared, pages = pool(rng, tokens, S + F, page, spare, int(rng.integers(0, 3)))
    src = rng.integers(0, S, F)
    n = np.where(rng.random(F) < 0.3, tokens[src] // page * page, rng.integers(0, tokens[src] + 1))
    dst = S + rng.permutation(F)
    st = State(hip, table, held, free, n_free, shared, pages, page)
    want = ref.fork(src, dst, n, free, n_free, table, held, shared, page, pages)
    out = st.fork(src, dst, n)
    same({**out, **st.values()}, want)
    now = st.values()
    for part in (0.5, 1.0):
        keep = np.where(rng.random(S + F) < part, rng.integers(-5, hi + 1, S + F) if part < 1 else 0, 2 ** 31 - 1)
        want = ref.free(keep, now["table"], now["held"], now["shared"], now["free"], int(now["n_free"][0]), page, pages)
        st.give_back(keep)
        now = st.values()
        same(now, want)
    assert now["n_free"][0] == pages and sorted(now["free"]) == list(range(pages)) and not now["shared"].any()


@pytest.mark.parametrize("S,F,page,ctx", [(2, 9, 16, 77), (8, 64, 64, 4000)])
def test_giving_back_what_was_handed_out_restores_the_list(hip, S, F, page, ctx):
    rng = np.random.default_rng(F)
    tokens = rng.integers(1, ctx + 1, S)
    start = pool(rng, tokens, S + F, page, F + 3)
    st = State(hip, *start[:6], page)
    st.fork(rng.integers(0, S, F), S + np.arange(F), np.full(F, tokens.min()))
    st.give_back([2 ** 31 - 1] * S + [0] * F)
    now = st.values()
    np.testing.assert_array_equal(now["free"], start[2])
    np.testing.assert_array_equal(now["table"], start[0])
    assert now["n_free"][0] == start[3] and not now["shared"].any()


def test_forks_refused(hip):
    """Rows and lengths out of range, the same row twice, a row that holds pages, a source that a fork of the call begins."""
    rng = np.random.default_rng(3)
    start = pool(rng, [50, 20, 16], 10, 16, 4, 1)
    held = start[1].copy()
    held[9] = start[0].shape[1] + 1  # (more than a row has)
    big = 2 ** 31 - 1
    forks = [(-1, 4, 5), (10, 4, 5), (0, -1, 5), (0, 10, 5), (0, 0, 5), (0, 1, 5), (0, 4, -1), (0, 4, 65), (0, 4, big), (9, 4, 5),
             (0, 4, 17), (1, 4, 3), (4, 5, 3), (1, 5, 32), (4, 6, 0), (0, 6, 1), (0, 7, 1), (0, 8, 16), (-big - 1, big, big),
             (2, 3, 5), (0, 3, 48), (1, 9, 1)]
    src, dst, n = np.array(forks).T
    for n_free in (4, 2, 0, -3):
        st = State(hip, start[0], held, start[2], n_free, start[4], start[5], 16)
        same({**st.fork(src, dst, n), **st.values()}, ref.fork(src, dst, n, start[2], n_free, start[0], held, start[4], 16, start[5]))


@pytest.mark.parametrize("S,ldt", [(6, 20), (80, 40), (150, 40), (600, 50)])  # one workgroup with one, four and eight places a thread, several
@pytest.mark.parametrize("counted", [True, False])
def test_free_of_what_is_wrong(hip, S, ldt, counted):
    """Ids outside the cache, rows that hold more than they have or less than nothing, a page in a row twice, pages given up
    more often than they are held, a list that is full."""
    rng = np.random.default_rng(S)
    pages, page = 500, 16
    table = rng.integers(-3, pages + 3, (S, ldt))
    if not counted:  # (each page once: without counts nothing tells a second holder)
        table = np.where(rng.random((S, ldt)) < 0.02, np.arange(S * ldt).reshape(S, ldt) % pages, -1)
        _, at = np.unique(table, return_index=True)
        table = np.where(np.isin(np.arange(S * ldt), at).reshape(S, ldt), table, -1)
    held = rng.integers(-2, ldt + 4, S)
    held[0], held[-1] = ldt + 100, 2 ** 31 - 1
    keep = rng.choice([-2 ** 31, -1, 0, 1, 16, 17, page * ldt // 2, 2 ** 31 - 1], S)
    shared = rng.integers(0, 3, pages)
    for n_free in (0, 37, pages - 2, pages, pages + 5, -4):
        st = State(hip, table, held, np.arange(pages) * 7, n_free, shared, pages, page)
        want = ref.free(keep, table, held, shared if counted else None, np.arange(pages) * 7, n_free, page, pages)
        st.give_back(keep, counted)
        same(st.values(), want)


def caches(rng, kind, L, pages, HK, page, D):
    torch = _torch()
    t = torch.float16 if kind == "f16" else torch.bfloat16
    x = [torch.from_numpy(rng.integers(-2 ** 15, 2 ** 15, (L, pages, HK, page, D)).astype(np.int16)).cuda().view(t) for _ in range(2)]
    return x, [host(c.view(torch.int16)) for c in x]


def cache_of(hip, kv, kind, HK, page, D, pages):
    return hip.KvCache(kv[0], kv[1], hip.CacheType[kind], page, HK, D, pages, HK * page * D, page * D, D)


@pytest.mark.parametrize("HK,D,page,L,kind", [(4, 256, 64, 3, "f16"), (1, 128, 16, 1, "bf16"), (3, 64, 256, 2, "f16"), (2, 256, 128, 1, "bf16")])
@pytest.mark.parametrize("lengths", [True, False])
def test_page_copy(hip, HK, D, page, L, kind, lengths):
    """Any bits (NaN among them) of the first tokens; entries that name no page, the page itself or no tokens."""
    torch = _torch()
    rng = np.random.default_rng(D + page)
    pages = 24
    kv, old = caches(rng, kind, L, pages, HK, page, D)
    frm = np.array([0, 5, -1, 3, 7, 8, 24, 2, 9, 1])
    to = np.array([20, 21, 22, -1, 7, 23, 19, 24, 18, 17])
    n = np.array([page, 1, 3, 3, 3, 0, 5, 5, page + 9, page // 2 + 1])
    hip.launch_page_copy(hip.PageCopy(n=10, source=ints(frm), to=ints(to), tokens=ints(n) if lengths else None, layers=L,
                                      layer_stride=pages * HK * page * D), cache_of(hip, kv, kind, HK, page, D, pages), stream())
    for x, o in zip(kv, old):
        want = o.copy()
        for a, b, m in zip(frm, to, n if lengths else [page] * 10):
            if 0 <= a < pages and 0 <= b < pages and a != b:
                want[:, b, :, :min(m, page)] = o[:, a, :, :min(m, page)]
        np.testing.assert_array_equal(host(x.view(torch.int16)), want)


def test_page_copy_of_a_strided_cache(hip):
    """Tokens before heads in a wider array; layers inside a page."""
    torch = _torch()
    rng = np.random.default_rng(5)
    pages, L, page, HK, D = 6, 3, 16, 2, 64
    x = [torch.from_numpy(rng.standard_normal((pages, L, page, HK, D + 8))).half().cuda() for _ in range(2)]
    old = [t.clone() for t in x]
    kv = hip.KvCache(x[0], x[1], hip.CacheType.f16, page, HK, D, pages, L * page * HK * (D + 8), D + 8, HK * (D + 8))
    hip.launch_page_copy(hip.PageCopy(n=2, source=ints([4, 1]), to=ints([0, 5]), tokens=ints([16, 7]), layers=L,
                                      layer_stride=page * HK * (D + 8)), kv, stream())
    for t, o in zip(x, old):
        o[0, :, :, :, :D] = o[4, :, :, :, :D]
        o[5, :, :7, :, :D] = o[1, :, :7, :, :D]
        assert torch.equal(t, o)


def run_move(hip, kv, kind, table, HK, page, D, L, pages, first, to_table=None, lists=None, tree=None, leaf=None, want_len=True):
    S = len(first)
    n = ints(np.full(S, -9))
    a = hip.CacheMove(S=S, table=ints(table), ldt=table.shape[1], to_table=ints(to_table) if to_table is not None else None,
                      ldt_to=to_table.shape[1] if to_table is not None else 0, first=ints(first),
                      kv_len=n if want_len else None, layers=L, layer_stride=pages * HK * page * D)
    if tree is not None:
        bits = _torch().from_numpy(np.asarray(tree, np.uint64).view(np.int64)).cuda()
        a = dataclasses.replace(a, T=len(tree), tree=bits, leaf=ints(leaf))
    else:
        flat = np.concatenate([np.asarray(x, np.int64) for x in lists] + [np.zeros(0, np.int64)])
        a = dataclasses.replace(a, T=len(flat), source=ints(np.append(flat, 0)), source0=ints(np.cumsum([0] + [len(x) for x in lists])))
    hip.launch_cache_move(a, cache_of(hip, kv, kind, HK, page, D, pages), stream())
    return host(n)


@pytest.mark.parametrize("HK,D,page,L,kind", [(8, 256, 64, 2, "bf16"), (4, 256, 64, 2, "f16"), (2, 128, 16, 1, "bf16"), (1, 64, 32, 3, "f16")])
@pytest.mark.parametrize("hi,part", [(1, 1.0), (40, 0.5), (700, 0.9), (2500, 0.5), (2500, 1.0), (5000, 0.02)])
@pytest.mark.parametrize("other", [False, True])
def test_move_listed_tokens(hip, HK, D, page, L, kind, hi, part, other):
    """Lists of none to thousands of tokens, in place and to other pages; ones that all move one place down."""
    torch = _torch()
    rng = np.random.default_rng(hi + D)
    L = 1 if hi > 1000 else L
    tokens = [hi, 0, max(1, hi // 3), min(hi, 17)]
    table, held, free, n_free, _, pages = pool(rng, tokens * 2, 8, page, 2, 1)
    kv, old = caches(rng, kind, L, pages, HK, page, D)
    first = [int(rng.integers(0, n // 4 + 1)) for n in tokens]
    lists = [sorted(rng.choice(np.arange(f, n), int((n - f) * part), replace=False)) for f, n in zip(first, tokens)]
    if part == 1.0:  # all but the first: every place is the next one's new place
        lists = [x[1:] for x in lists]
    to = table[4:] if other else None
    n = run_move(hip, kv, kind, table[:4], HK, page, D, L, pages, first, to, lists)
    np.testing.assert_array_equal(n, [f + len(x) for f, x in zip(first, lists)])
    for x, w in zip(kv, ref.move(*old, table[:4], to, first, lists, page)):
        np.testing.assert_array_equal(host(x.view(torch.int16)), w)


@pytest.mark.parametrize("HK,D,page,L,kind", [(4, 256, 64, 3, "f16"), (2, 128, 16, 1, "bf16"), (1, 64, 16, 2, "bf16")])
def test_move_accepted_paths(hip, HK, D, page, L, kind):
    """One node to 64, places that cross pages, the whole tree, leaves that there are not."""
    torch = _torch()
    rng = np.random.default_rng(D)
    full = 2 ** 64 - 1
    bits = [1, 0b10110, full, 1 << 63, full ^ 1, int(rng.integers(0, 2 ** 63)), 0x8000000080000001, 0, 5]
    first = [0, 14, 33, 7, 100, 15, 16, 9, 3]
    leaf = [2, 0, 8, 1, 5, 3, 4, 6, 99]
    tree = [0] * 9
    for b, r in zip(bits, leaf):
        if r < 9:
            tree[r] = b
    table, *_, pages = pool(rng, [f + 64 for f in first], 9, page, 1)
    kv, old = caches(rng, kind, L, pages, HK, page, D)
    n = run_move(hip, kv, kind, table, HK, page, D, L, pages, first, tree=tree, leaf=leaf)
    lists = [[f + j for j in range(64) if b >> j & 1] for f, b in zip(first, bits[:8] + [0])]
    np.testing.assert_array_equal(n, [f + len(x) for f, x in zip(first, lists)])
    for x, w in zip(kv, ref.move(*old, table, None, first, lists, page)):
        np.testing.assert_array_equal(host(x.view(torch.int16)), w)


@pytest.mark.parametrize("how", ["tree", "few", "some", "many"])  # lists: in runs of 32, 64, 128 bytes
def test_move_with_lengths_in_place(hip, how):
    """kv_len is `first` itself: every workgroup finds the lengths as they were, also in a graph's replays."""
    torch = _torch()
    rng = np.random.default_rng(len(how))
    HK, D, page, L, S = {"tree": (8, 128, 16, 4, 40), "few": (1, 64, 16, 3, 5), "some": (1, 128, 16, 3, 8), "many": (4, 256, 16, 2, 30)}[how]
    tokens = rng.integers(60, 120, S) + 64
    table, *_, pages = pool(rng, tokens, S, page, 2)
    first = [int(n) - 64 for n in tokens]
    kv, old = caches(rng, "f16", L, pages, HK, page, D)
    want_first = [int(rng.integers(0, f + 1)) for f in first]
    if how == "tree":
        want_first = first
        tree = np.array([int(x) for x in rng.integers(0, 2 ** 63, S)], np.uint64)
        lists = [[f + j for j in range(64) if int(b) >> j & 1] for f, b in zip(first, tree)]
        what = dict(T=S, tree=torch.from_numpy(tree.view(np.int64)).cuda(), leaf=ints(np.arange(S)))
    else:
        lists = [sorted(rng.choice(np.arange(f, n), int((n - f) * 0.7), replace=False)) for f, n in zip(want_first, tokens)]
        flat = np.concatenate(lists)
        what = dict(T=len(flat), source=ints(flat), source0=ints(np.cumsum([0] + [len(x) for x in lists])))
    lens, start = ints(want_first), ints(want_first)
    a = hip.CacheMove(S=S, table=ints(table), ldt=table.shape[1], first=lens, kv_len=lens, layers=L, layer_stride=pages * HK * page * D, **what)
    cache = cache_of(hip, kv, "f16", HK, page, D, pages)
    want, fresh = ref.move(*old, table, None, want_first, lists, page), [x.clone() for x in kv]

    def check():
        np.testing.assert_array_equal(host(lens), [f + len(x) for f, x in zip(want_first, lists)])
        for x, w in zip(kv, want):
            np.testing.assert_array_equal(host(x.view(torch.int16)), w)
    hip.launch_cache_move(a, cache, stream())
    check()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        hip.launch_cache_move(a, cache, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        lens.copy_(start)
        for x, f in zip(kv, fresh):
            x.copy_(f)
        g.replay()
        check()


def test_move_of_places_that_are_none(hip):
    """Places before or behind the table, pages that there are not, row starts out of range: those tokens stay out."""
    torch = _torch()
    rng = np.random.default_rng(8)
    HK, D, page, pages = 2, 64, 16, 12
    table = np.array([[3, -1, 5, 99], [1, 2, 7, 8]])
    kv, old = caches(rng, "f16", 1, pages, HK, page, D)
    lists = [[0, 5, 17, 33, 40, 47, 49, 64, 10 ** 6], [-5, 3, 20, 63, 64, 2 ** 31 - 1]]
    first = [0, 0]
    run_move(hip, kv, "f16", table, HK, page, D, 1, pages, first, np.array([[0, 4], [6, 9]]), lists, want_len=False)
    for x, w in zip(kv, ref.move(*old, table, np.array([[0, 4], [6, 9]]), first, lists, page)):
        np.testing.assert_array_equal(host(x.view(torch.int16)), w)
    kv, old = caches(rng, "f16", 1, pages, HK, page, D)
    n = run_move(hip, kv, "f16", table, HK, page, D, 1, pages, [-2, 60], lists=[[0, 1, 2, 3], [61, 62, 63]])
    np.testing.assert_array_equal(n, [2, 63])
    for x, w in zip(kv, ref.move(*old, table, None, [-2, 60], [[0, 1, 2, 3], [61, 62, 63]], page)):
        np.testing.assert_array_equal(host(x.view(torch.int16)), w)
    # starts of the lists at the ends of their type: none of request 0, the first two of request 1
    kv, old = caches(rng, "f16", 1, pages, HK, page, D)
    n = ints([-9, -9])
    hip.launch_cache_move(hip.CacheMove(S=2, T=4, table=ints(table), ldt=4, first=ints([0, 0]), source=ints([18, 40, 41, 42]),
                                        source0=ints([2 ** 31 - 1, -2 ** 31, 2]), kv_len=n), cache_of(hip, kv, "f16", HK, page, D, pages), stream())
    assert host(n).tolist() == [0, 2]
    for x, w in zip(kv, ref.move(*old, table, None, [0, 0], [[], [18, 40]], page)):
        np.testing.assert_array_equal(host(x.view(torch.int16)), w)


def test_far_pages(hip):
    """Pages, layers and heads beyond 2^32 bytes of the cache's start."""
    torch = _torch()
    HK, D, page, pages, L = 2, 64, 16, 3, 2
    # 5 GiB between pages, 2.5 GiB between layers; both caches are views of one array
    big = torch.zeros(3 * (5 << 29) + (1 << 24), dtype=torch.float16, device="cuda")
    ps, ls, hs, ts = 5 << 29, (5 << 28), 1 << 20, 1 << 8
    vals = torch.randn((pages, L, HK, page, D), device="cuda").half()
    at = [(p, l, h, t, p * ps + l * ls + h * hs + t * ts) for p in range(pages) for l in range(L) for h in range(HK) for t in range(page)]
    def put(x, off):
        for p, l, h, t, o in at:
            big[off + o: off + o + D] = x[p, l, h, t]
    def get(off):
        return torch.stack([big[off + o: off + o + D] for *_, o in at]).view(pages, L, HK, page, D)
    put(vals, 0), put(-vals, 128)
    kv = hip.KvCache(big.data_ptr(), big.data_ptr() + 256, hip.CacheType.f16, page, HK, D, pages, ps, hs, ts)
    hip.launch_page_copy(hip.PageCopy(n=1, source=ints([0]), to=ints([2]), tokens=ints([5]), layers=L, layer_stride=ls), kv, stream())
    vals[2, :, :, :5] = vals[0, :, :, :5]
    assert torch.equal(get(0), vals) and torch.equal(get(128), -vals)
    table = ints([[1, 2]])
    hip.launch_cache_move(hip.CacheMove(S=1, T=3, table=table, ldt=2, first=ints([2]), source=ints([3, 20, 31]),
                                        source0=ints([0, 3]), layers=L, layer_stride=ls), kv, stream())
    vals[1, :, :, 2], vals[1, :, :, 3], vals[1, :, :, 4] = vals[1, :, :, 3].clone(), vals[2, :, :, 4].clone(), vals[2, :, :, 15].clone()
    assert torch.equal(get(0), vals) and torch.equal(get(128), -vals)


def test_captured(hip):
    """Forks, copies and the return of the pages as one graph, replayed with other lengths and with eager work between."""
    torch = _torch()
    rng = np.random.default_rng(11)
    S, F, HK, D, page, L = 3, 6, 2, 128, 16, 2
    tokens = np.array([70, 33, 16])
    start = pool(rng, tokens, S + F, page, F + 2)
    table, held, free, n_free, shared, pages = start
    kv, old = caches(rng, "f16", L, pages, HK, page, D)
    st = State(hip, *start, page)
    src, n = ints(np.zeros(F)), ints(np.zeros(F))
    out = {k: ints(np.zeros(F)) for k in ("got", "copy_from", "copy_to", "copy_tokens")}
    common = dict(page=page, ldt=st.ldt, pages=pages, table=st.table, held=st.held, shared=st.shared, free=st.free, n_free=st.n_free)
    fork = hip.PageFork(F=F, S=S + F, src=src, dst=ints(S + np.arange(F)), tokens=n, **common, **out)
    copy = hip.PageCopy(n=F, source=out["copy_from"], to=out["copy_to"], tokens=out["copy_tokens"], layers=L,
                        layer_stride=pages * HK * page * D)
    back = hip.PageFree(S=S + F, keep=ints([2 ** 31 - 1] * S + [0] * F), **common)
    cache = cache_of(hip, kv, "f16", HK, page, D, pages)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        q = torch.cuda.current_stream().cuda_stream
        hip.launch_page_fork(fork, q)
        hip.launch_page_copy(copy, cache, q)
        hip.launch_page_free(back, q)
    for _ in range(4):
        who = rng.integers(0, S, F)
        m = rng.integers(0, tokens[who] + 1)
        src.copy_(ints(who)), n.copy_(ints(m))
        g.replay()
        torch.cuda.synchronize()
        want = ref.fork(who, S + np.arange(F), m, free, n_free, table, held, shared, page, pages)
        same(out, {k: want[k] for k in out})
        same(st.values(), {"table": table, "held": held, "free": free, "n_free": np.array([n_free]), "shared": shared})
        for a, b, c in zip(want["copy_from"], want["copy_to"], want["copy_tokens"]):
            for o in old:
                if a >= 0:
                    o[:, b, :, :c] = o[:, a, :, :c]
        for x, o in zip(kv, old):
            np.testing.assert_array_equal(host(x.view(torch.int16)), o)
