"""GPU tests of low-rank adapters beside a shared projection (launch_lora) against the formula in 64 bits (sharing_ref.py)."""
import dataclasses
import math

import numpy as np
import pytest

import sharing_ref as ref

pytestmark = pytest.mark.gpu
GUARD = 7.25  # what rows, columns and gaps that are not written hold


def _torch():
    import torch
    return torch


def dev(a):
    return _torch().from_numpy(np.ascontiguousarray(a)).cuda()


def ints(a):
    return dev(np.asarray(a, np.int32))


def kind_of(kind):
    torch = _torch()
    return torch.float16 if kind == "f16" else torch.bfloat16


def words(n):
    """n bytes of scratch, filled with what an earlier user may have left."""
    torch = _torch()
    return torch.full((max(1, -(-n // 8)),), -1, dtype=torch.int64, device="cuda")


def stream():
    return _torch().cuda.current_stream().cuda_stream


def tol(K, rank, kind, deep, flat, y, delta):
    """Every product of parts is exact; a sum of n terms has at most n roundings (2^-24, and twice that as the matrix
    instruction may cut off), each of at most the sum of its terms' sizes. h: K columns times 3 parts of x and 1 or 2 of
    A, the waves' and slices' sums; scale; delta: the rank's steps of 32 likewise; the sum with y."""
    parts = 3 if kind == "bf16" else 6
    n_h, n_d = K * parts + 4 + K // 256 + 2, (rank + 31) // 32 * 32 * parts
    u = 2.0 ** -23
    # (columns go through an instruction by eights that are summed at once, so that only an eighth of the roundings is there)
    return u * (n_h / 8 * deep + n_d / 8 * flat + 4 * (np.abs(y) + np.abs(delta))) + 1e-30


class Case:
    def __init__(self, new, K, Ns, kind, rank, adapters=3, who=None, ranks="mixed", scale=True, seed=0, spare=3, pad=(0, 0), big=1.0):
        rng = np.random.default_rng(seed + K + sum(Ns) + rank)
        torch, t = _torch(), kind_of(kind)
        self.S, self.T, self.K, self.Ns, self.kind, self.rank, self.adapters = len(new), sum(new) + spare, K, Ns, kind, rank, adapters
        self.row0 = np.cumsum([0] + list(new))
        self.who = rng.integers(-1, adapters, self.S) if who is None else np.asarray(who)
        self.ranks = rng.integers(0, rank + 1, adapters) if isinstance(ranks, str) else ranks
        self.scale = rng.uniform(-2, 2, adapters).astype(np.float32) if scale else None
        self.ldx, self.ypad = K + pad[0], pad[1]
        self.x = (rng.standard_normal((self.T, self.ldx)) * big * np.exp(rng.standard_normal((self.T, 1)))).astype(np.float32)
        cast = lambda a: torch.from_numpy(a).to(t)  # noqa: E731
        self.a = [cast(rng.standard_normal((adapters, rank, K)) * K ** -0.5) for _ in Ns]
        self.b = [cast(rng.standard_normal((adapters, n, rank))) for n in Ns]
        self.y = [rng.standard_normal((self.T, n + self.ypad)).astype(np.float32) for n in Ns]

    def run(self, hip, mode="add", shift=0, device_x=None, into_gate=False, stream_=None):
        """(y of each segment, out) on the host. shift: y starts so many floats into its array."""
        torch = _torch()
        self.dy = []
        for y in self.y:
            t = torch.full((y.size + shift,), GUARD, device="cuda")
            t[shift:] = dev(y.reshape(-1))
            self.dy.append(t)
        segs = [hip.LoraSeg(a.cuda(), b.cuda(), self.rank * self.K, n * self.rank, n, y[shift:], n + self.ypad)
                for a, b, n, y in zip(self.a, self.b, self.Ns, self.dy)]
        out = None
        if mode == "swiglu":
            out = self.dy[0][shift:] if into_gate else torch.full((self.T * (self.Ns[0] + self.ypad),), GUARD, device="cuda")
        ws = words(hip.lora_ws_bytes(self.S, self.T, self.K, self.rank, len(segs)))
        x = dev(self.x) if device_x is None else device_x
        a = hip.Lora(S=self.S, T=self.T, K=self.K, rank=self.rank, adapters=self.adapters, type=hip.CacheType[self.kind],
                     mode=hip.GemvMode.kSwiglu if mode == "swiglu" else hip.GemvMode.kAdd, row0=ints(self.row0), adapter=ints(self.who),
                     ranks=ints(self.ranks) if self.ranks is not None else None, scale=dev(self.scale) if self.scale is not None else None,
                     x=x, ldx=self.ldx, out=out, ldo=(self.Ns[0] + self.ypad) if out is not None else 0, ws=ws)
        hip.launch_lora(a, segs, stream_ if stream_ is not None else stream())
        torch.cuda.synchronize()
        ys = [t[shift:].cpu().numpy().reshape(y.shape) for t, y in zip(self.dy, self.y)]
        return ys, out.cpu().numpy().reshape(self.T, -1) if out is not None else None

    def want(self):
        """(delta, tolerance) of each segment's columns."""
        got = []
        for a, b, n, y in zip(self.a, self.b, self.Ns, self.y):
            d, deep, flat = ref.lora(self.x[:, :self.K], self.row0, self.who, self.ranks, self.scale, a.double().numpy(), b.double().numpy(), self.T)
            got.append((d, tol(self.K, self.rank, self.kind, deep, flat, y[:, :n], d)))
        return got

    def check_add(self, ys):
        live = np.zeros(self.T, bool)
        for s in range(self.S):
            live[max(0, self.row0[s]):min(self.T, self.row0[s + 1])] = 0 <= self.who[s] < self.adapters
        for y, old, n, (d, t) in zip(ys, self.y, self.Ns, self.want()):
            err = np.abs(y[:, :n].astype(np.float64) - (old[:, :n] + d))
            assert np.all(err <= t), (err / t).max()
            # as a whole the roundings are far smaller than their bound
            assert np.linalg.norm(err) <= 2e-6 * np.linalg.norm(old[:, :n] + d)
            np.testing.assert_array_equal(y[~live], old[~live])
            np.testing.assert_array_equal(y[:, n:], old[:, n:])

    def check_swiglu(self, out, rows=None):
        (dg, tg), (du, tu) = self.want()
        n = self.Ns[0]
        g, u = self.y[0][:, :n] + dg, self.y[1][:, :n] + du
        sig = 1 / (1 + np.exp(-g))
        w = g * sig * u
        # d(silu) is at most 1.1; the exponential, the sum, the division and the product: under 16 half-steps
        t = 1.1 * tg * (np.abs(u) + tu) + np.abs(g * sig) * tu + 16 * 2.0 ** -24 * np.abs(w) + 1e-30
        rows = self.row0[-1] if rows is None else rows
        assert np.all(np.abs(out[:rows, :n] - w[:rows]) <= t[:rows])
        assert np.linalg.norm(out[:rows, :n] - w[:rows]) <= 2e-6 * max(1e-30, np.linalg.norm(w[:rows]))


SIZES = [  # rows of each request, K, outputs, rank
    ([1], 512, [64], 16), ([1], 32, [1], 8), ([1, 1, 1, 1, 1], 5120, [512], 16), ([2, 0, 5, 16, 17], 1056, [100], 24),
    ([1] * 70, 544, [33], 8), ([100], 2048, [300], 64), ([65, 130, 1], 512, [257], 40), ([40, 3, 0, 0, 90], 96, [16], 128),
    ([33], 17408, [64], 32), ([20, 20], 640, [700], 256), ([300], 256, [1100], 16), ([2, 1, 3], 2880, [547], 128), ([4, 0, 3], 1056, [65], 256),
    ([12], 5120, [225], 128), ([700, 500], 96, [130], 200), ([1100], 544, [65, 8], 72)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new,K,Ns,rank", SIZES, ids=str)
def test_add(hip, new, K, Ns, rank, kind):
    c = Case(new, K, Ns, kind, rank, seed=1)
    c.check_add(c.run(hip)[0])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new,K,N,rank", [([1], 512, 64, 16), ([1, 2, 1], 1024, 1000, 32), ([64, 7], 512, 333, 64), ([70], 256, 128, 128),
                                          ([1] * 9, 5120, 200, 200), ([1100], 96, 70, 128), ([600, 500], 64, 33, 256), ([1100], 288, 130, 40)], ids=str)
@pytest.mark.parametrize("into_gate", [False, True])
def test_swiglu(hip, new, K, N, rank, kind, into_gate):
    c = Case(new, K, [N, N], kind, rank, seed=2)
    ys, out = c.run(hip, "swiglu", into_gate=into_gate)
    c.check_swiglu(out)
    np.testing.assert_array_equal(ys[1], c.y[1])
    if not into_gate:
        np.testing.assert_array_equal(ys[0], c.y[0])
        assert np.all(out[c.row0[-1]:] == GUARD)
    else:
        np.testing.assert_array_equal(out[c.row0[-1]:], c.y[0][c.row0[-1]:])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new,K,N,rank", [([1], 32, 1, 8), ([1], 5120, 300, 16), ([1], 5120, 700, 32), ([1, 1, 1], 1056, 513, 40), ([1] * 8, 96, 8, 256),
                                          ([1, 0, 1, 1], 17408, 40, 8), ([2, 1, 0], 544, 1000, 24), ([1] * 60, 640, 1025, 128),
                                          ([1] * 70, 1024, 1100, 64)], ids=str)
def test_one_row_each(hip, new, K, N, rank, kind):
    """As many rows as requests: one launch while A is small, two beyond; every number of waves that share ranks."""
    for ranks in (None, "mixed"):
        c = Case(new, K, [N, N, 8], kind, rank, spare=0, seed=3, ranks=ranks, pad=(8, 1))
        c.check_add(c.run(hip)[0])
        c = Case(new, K, [N, N], kind, rank, spare=0, seed=4, ranks=ranks, scale=ranks is None)
        for into_gate in (False, True):
            ys, out = c.run(hip, "swiglu", into_gate=into_gate)
            c.check_swiglu(out)
            np.testing.assert_array_equal(ys[1], c.y[1])


# A workgroup's outputs in several passes: rows of 16, 32 and 64 a tile, chunks of 512 and 1024 outputs, the last of each in
# part; the forms of a row and of four; the one launch of a row and a small A.
PASSES = [([600, 500], 64, 8213, 16), ([1100], 96, 7700, 200), ([1300, 900], 64, 7701, 40), ([700, 401], 64, 7703, 72), ([1, 1030], 32, 15001, 136),
          ([1] * 70, 96, 8001, 128), ([2] * 40, 64, 9301, 24), ([1], 640, 700, 256), ([1, 1, 1], 640, 513, 128), ([1, 1], 320, 1000, 248)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new,K,N,rank", PASSES, ids=lambda x: str(x)[:24])
def test_outputs_in_several_passes(hip, new, K, N, rank, kind):
    spare = 3 if max(new) > 2 else 0  # (none where the form goes by a row, or four, a request)
    for ranks in (None, "mixed"):
        c = Case(new, K, [N, 9], kind, rank, adapters=2, ranks=ranks, seed=14, spare=spare, pad=(0, 1))
        c.check_add(c.run(hip)[0])
    c = Case(new, K, [N, N], kind, rank, adapters=2, ranks=None, seed=15, spare=spare)
    for into_gate in (False, True):
        ys, out = c.run(hip, "swiglu", into_gate=into_gate)
        c.check_swiglu(out)
        np.testing.assert_array_equal(ys[1], c.y[1])
        np.testing.assert_array_equal(out[c.row0[-1]:], c.y[0][c.row0[-1]:] if into_gate else np.full_like(out[c.row0[-1]:], GUARD))


@pytest.mark.parametrize("Ns", [[512, 96, 96], [40, 41]])
@pytest.mark.parametrize("new", [[1, 1, 1], [50, 30]])
@pytest.mark.parametrize("pad,shift", [((0, 0), 0), ((4, 3), 0), ((20, 4), 0), ((0, 0), 1), ((0, 4), 2)])
def test_segments_strides_and_starts(hip, Ns, new, pad, shift):
    c = Case(new, 640, Ns, "bf16", 16, pad=pad, seed=3)
    c.check_add(c.run(hip, shift=shift)[0])
    if len(Ns) == 2:
        c = Case(new, 640, [41, 41], "f16", 16, pad=pad, seed=3)
        c.check_swiglu(c.run(hip, "swiglu", shift=shift)[1])


@pytest.mark.parametrize("ranks,scale", [(None, True), ([0, 7, 16], False), ([-3, 99, 1], True)])
def test_ranks_and_scales(hip, ranks, scale):
    """No ranks or scales; ranks of nothing, odd ones, ones that pass the room."""
    for new in ([1, 2, 1, 1], [30, 40, 1, 0]):
        c = Case(new, 512, [80], "f16", 16, who=[0, 1, 2, 1], ranks=ranks, scale=scale, seed=4)
        c.check_add(c.run(hip)[0])


def test_adapters_that_are_none(hip):
    """Ids below zero, the number of adapters and beyond; no adapter at all. With the activation the rows still get theirs."""
    who = [-1, 3, 2 ** 31 - 1, -2 ** 31, 2]
    for new in ([1, 1, 1, 1, 1], [40, 40, 1, 2, 30]):
        c = Case(new, 256, [48], "bf16", 8, who=who, seed=5)
        c.check_add(c.run(hip)[0])
        c = Case(new, 256, [48, 48], "bf16", 8, who=who, seed=5)
        c.check_swiglu(c.run(hip, "swiglu")[1])
    c = Case([2, 1], 64, [8], "f16", 8, who=[-1, -1], seed=6)
    c.check_add(c.run(hip)[0])


@pytest.mark.parametrize("new", [[1, 1], [40, 30]])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_what_lies_behind_the_rank_has_no_effect(hip, new, kind):
    """NaN and infinities behind the ranks, in other adapters, in rows without one and in columns behind K."""
    c = Case(new, 288, [90], kind, 24, who=[1, -1], ranks=[24, 11, 24], pad=(4, 0), seed=7)
    clean, _ = c.run(hip)
    for a, b in zip(c.a, c.b):
        a[1, 11:], b[1, :, 11:] = math.nan, math.inf
        a[0], a[2], b[0], b[2] = math.nan, math.inf, -math.inf, math.nan
    c.x[c.row0[1]:] = math.nan
    c.x[:, c.K:] = math.inf
    got, _ = c.run(hip)
    np.testing.assert_array_equal(got[0], clean[0])


def test_rows_of_other_requests_do_not_matter(hip):
    """A NaN row stays in its row."""
    c = Case([40, 3], 256, [70], "bf16", 16, who=[0, 1], ranks=[16, 16, 16], seed=8)
    clean, _ = c.run(hip)
    c.x[5, 17], c.x[41, 3] = math.nan, math.inf
    got, _ = c.run(hip)
    bad = np.isnan(got[0]).any(1)
    assert list(np.flatnonzero(bad)) == [5, 41]
    np.testing.assert_array_equal(got[0][~bad], clean[0][~bad])


@pytest.mark.parametrize("big", [1e-30, 1e-6, 1e6, 1e30])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_sizes_of_x(hip, big, kind):
    """Values far from 1: the parts of x have its range."""
    c = Case([3, 30], 512, [64], kind, 16, who=[0, 1], ranks=[16, 16, 16], big=big, seed=9)
    c.y = [np.zeros_like(y) for y in c.y]
    c.check_add(c.run(hip)[0])


def test_rows_that_do_not_fit(hip):
    """Row starts below zero or beyond T, requests of no rows, starts that fall."""
    c = Case([3, 4, 5], 128, [40], "f16", 8, who=[0, 1, 2], ranks=None, seed=10, spare=0)
    c.row0 = np.array([-2, 3, 3, 40])
    c.check_add(c.run(hip)[0])
    c.row0 = np.array([5, 2, 6, 6])
    c.check_add(c.run(hip)[0])
    c.row0 = np.array([-2 ** 31, 4, 2 ** 31 - 1, -2 ** 31])
    c.check_add(c.run(hip)[0])


@pytest.mark.parametrize("new,rank", [([1] * 20, 16), ([80, 41], 64)])
def test_the_same_twice_and_captured(hip, new, rank):
    """Equal bits call for call; one workspace in two graphs, replayed with other adapters and with eager work between."""
    torch = _torch()
    c = Case(new, 1024, [256, 64], "bf16", rank, who=[i % 4 - 1 for i in range(len(new))], seed=11)
    first, _ = c.run(hip)
    again, _ = c.run(hip)
    for a, b in zip(first, again):
        np.testing.assert_array_equal(a, b)
    segs = [hip.LoraSeg(a.cuda(), b.cuda(), rank * c.K, n * rank, n, dev(y), n) for a, b, n, y in zip(c.a, c.b, c.Ns, c.y)]
    adapter = ints(c.who)
    ws = words(hip.lora_ws_bytes(c.S, c.T, c.K, rank, 2))
    a = hip.Lora(S=c.S, T=c.T, K=c.K, rank=rank, adapters=3, type=hip.CacheType.bf16, mode=hip.GemvMode.kAdd, row0=ints(c.row0),
                 adapter=adapter, ranks=ints(c.ranks), scale=dev(c.scale), x=dev(c.x), ldx=c.ldx, ws=ws)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    for seg in segs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            hip.launch_lora(a, [seg], torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(0)
    for k in range(4):
        c.who = rng.integers(-1, 3, c.S)
        adapter.copy_(ints(c.who))
        for seg, y in zip(segs, c.y):
            seg.y.copy_(dev(y))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        ys = [seg.y.cpu().numpy() for seg in segs]
        c.check_add(ys)
        for i, (n, got) in enumerate(zip(c.Ns, ys)):  # (alone, as in the graph)
            one = dataclasses.replace(segs[i], y=dev(c.y[i]))
            hip.launch_lora(a, [one], stream())
            torch.cuda.synchronize()
            np.testing.assert_array_equal(one.y.cpu().numpy(), got)


def test_workspace_of_the_largest_serves_smaller_ones(hip):
    torch = _torch()
    big = hip.lora_ws_bytes(40, 500, 2048, 64, 3)
    ws = torch.full((big // 4 + 64,), GUARD, device="cuda")
    for new, K, Ns, rank in [([1], 2048, [64], 64), ([1] * 40, 512, [64, 8, 8], 8), ([500], 2048, [64, 8, 8], 64), ([12, 13], 1024, [40], 64)]:
        c = Case(new, K, Ns, "bf16", rank, ranks=None, spare=0, seed=12)
        segs = [hip.LoraSeg(a.cuda(), b.cuda(), rank * K, n * rank, n, dev(y), n) for a, b, n, y in zip(c.a, c.b, Ns, c.y)]
        hip.launch_lora(hip.Lora(S=c.S, T=c.T, K=K, rank=rank, adapters=3, type=hip.CacheType.bf16, row0=ints(c.row0), adapter=ints(c.who),
                                 scale=dev(c.scale), x=dev(c.x), ldx=K, ws=ws), segs, stream())
        torch.cuda.synchronize()
        c.check_add([s.y.cpu().numpy() for s in segs])
        assert bool((ws[big // 4:] == GUARD).all())


@pytest.mark.parametrize("new,K,Ns,rank", [([700, 600, 650], 7776, [40, 8, 8], 16), ([300, 1], 17408, [8, 8, 8], 32), ([600], 4096, [16], 128),
                                           ([5, 4, 3], 17408, [8, 9, 10], 256), ([1, 2, 1], 17408, [8, 9, 10], 256)], ids=str)
def test_nothing_is_written_behind_the_workspace(hip, new, K, Ns, rank):
    """Many slices of K, sums of several segments."""
    torch = _torch()
    c = Case(new, K, Ns, "f16", rank, ranks=None, spare=0, seed=13)
    n = hip.lora_ws_bytes(c.S, c.T, K, rank, len(Ns))
    ws = torch.full((3 * n // 4 + 64,), GUARD, device="cuda")
    segs = [hip.LoraSeg(a.cuda(), b.cuda(), rank * K, m * rank, m, dev(y), m) for a, b, m, y in zip(c.a, c.b, Ns, c.y)]
    hip.launch_lora(hip.Lora(S=c.S, T=c.T, K=K, rank=rank, adapters=3, type=hip.CacheType.f16, row0=ints(c.row0), adapter=ints(c.who),
                             scale=dev(c.scale), x=dev(c.x), ldx=K, ws=ws), segs, stream())
    torch.cuda.synchronize()
    assert bool((ws[n // 4:] == GUARD).all())
    c.check_add([s.y.cpu().numpy() for s in segs])


def test_far_adapters_and_rows(hip):
    """Adapters and rows beyond 2^32 bytes of their arrays' start."""
    torch = _torch()
    K, N, rank, T = 32, 40, 8, 3
    stride, ld = 3 << 30, 1 << 29  # values
    a, b = (torch.zeros(stride + 4096, dtype=torch.float16, device="cuda") for _ in range(2))
    x, y = (torch.zeros(2 * ld + 4096, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    A, B, X = r(rank, K).half(), r(N, rank).half(), r(T, K)
    a[stride:stride + rank * K], b[stride:stride + N * rank] = A.flatten(), B.flatten()
    for i in range(T):
        x[i * ld:i * ld + K] = X[i]
    for new, who in (([1, 1, 1], [1, 0, 1]), ([0, 0, 3], [0, 0, 1])):
        y.zero_()
        ws = words(hip.lora_ws_bytes(3, T, K, rank, 1))
        hip.launch_lora(hip.Lora(S=3, T=T, K=K, rank=rank, adapters=2, type=hip.CacheType.f16, row0=ints(np.cumsum([0] + new)),
                                 adapter=ints(who), x=x, ldx=ld, ws=ws), [hip.LoraSeg(a, b, stride, stride, N, y, ld)], stream())
        d = (X.double() @ A.double().T @ B.double().T).cpu()
        t = (X.double().abs() @ A.double().abs().T @ B.double().abs().T).cpu() * 2.0 ** -23 * (6 * K + 6 * 32)
        for i, (w, n) in enumerate(zip([1, 0, 1] if new[0] else [1, 1, 1], [1] * 3)):
            got = y[i * ld:i * ld + N].double().cpu()
            assert bool(((got - (d[i] if w else 0)).abs() <= t[i]).all())
