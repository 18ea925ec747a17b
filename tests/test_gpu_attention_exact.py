"""GPU tests of how exact paged attention's probabilities are: rows in which one key takes nearly all of the weight and
holds nothing (V = 0), as the first token of a trained model's rows does, so that the output is made of small
probabilities alone; in every kernel and both types, against 64 bits.

K has few values that are not zero, so that a score is a sum of few products and the tolerances can be narrow. With
u = 2^-24, half a step of 32 bits, a weight's relative error is at most
  u * (10 * size + 4 * range + 8),
size the sum of its score's products in absolute value (fewer than ten roundings of at most that, the products being
exact), range the largest distance to the row's maximum (the rounding of the scores' scale and of the exponent), 8 for
the exponential and what follows. It counts twice, in the values and in their sum.
"""
import math

import numpy as np
import pytest

from test_gpu_serving import kind_of, run_attn

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
PARTS = {"f16": 2.0 ** -22, "bf16": 2.0 ** -24}  # half a step of a probability's two or three parts


# (heads, new rows): tiles of 16 rows, of 32 (64 for heads of 256), of 64, of 128
FORMS = [((4, 4, 64), 1), ((8, 4, 128), 1), ((20, 4, 256), 1), ((12, 2, 64), 4), ((8, 2, 128), 6), ((20, 4, 256), 5),
         ((8, 2, 64), 40), ((4, 2, 128), 50), ((8, 2, 128), 60), ((10, 2, 256), 30)]
IDS = ["%dx%dx%d-%d" % (*h, n) for h, n in FORMS]


def case(rng, S, n, ctx, heads, kind, sink, gap):
    """S requests of n new rows behind the same ctx tokens (shared pages; the new ones in pages of their own), all of a
    row's keys but `sink` within 2 of each other, that one `gap` above zero."""
    import torch
    H, HK, D = heads
    page, G = 64, H // HK
    shared, own = ctx // page, -(-(ctx % page + n) // page)
    pages = shared + S * own
    k, v = np.zeros((pages, HK, page, D)), 1 + 0.25 * rng.standard_normal((pages, HK, page, D))
    k[..., 1:4] = rng.choice([-0.5, -0.25, 0.0, 0.25, 0.5], (pages, HK, page, 3))
    q = np.zeros((S * n, H, D))
    q[..., 0] = 4.0
    q[..., 1:4] = rng.choice([-1.0, 1.0], (S * n, H, 3)) * D ** 0.5 / 2
    at = (sink // page, slice(None), sink % page)
    k[at], v[at] = 0, 0
    k[at][..., 0] = gap * D ** 0.5 / 4.0
    table = np.array([list(range(shared)) + [shared + s * own + i for i in range(own)] for s in range(S)])
    t = kind_of(kind)
    cast = lambda a: torch.from_numpy(a).to(t).cuda()  # noqa: E731
    return cast(q.reshape(S * n, H * D)), cast(k), cast(v), table, np.arange(S + 1) * n, [ctx + n] * S, page


def check(out, q, k, v, table, row0, kv_len, page, heads, kind, sink, gap, chain):
    H, HK, D = heads
    G, S, L = H // HK, len(kv_len), kv_len[0]
    n = int(row0[1])
    f = lambda a: a.double().cpu().numpy()  # noqa: E731
    q, k, v, out = f(q).reshape(S, n, H, D), f(k), f(v), f(out).reshape(S, n, H, D)
    block = np.arange(L) // 32
    for s in range(0, S, S // 8):
        kk, vv = (np.moveaxis(a[table[s]], 1, 0).reshape(HK, -1, D)[:, :L] for a in (k, v))
        seen = np.tril(np.ones((n, L)), L - n) > 0
        for h in range(H):
            x = q[s, :, h] @ kk[h // G].T * D ** -0.5
            size = np.abs(q[s, :, h]) @ np.abs(kk[h // G]).T * D ** -0.5
            top = np.where(seen, x, -np.inf).max(1, keepdims=True)
            w = np.where(seen, np.exp(x - top), 0.0)
            w /= w.sum(1, keepdims=True)
            a = np.abs(vv[h // G])
            e = U * (10 * size + 4 * np.where(seen, top - x, 0).max(1, keepdims=True) + 8) + PARTS[kind]
            err = (w * (e + e.max(1, keepdims=True))) @ a + chain * U * (w @ a)
            if kind == "f16":
                # A part ends at 2^-25. The largest of a block's 32 keys is at least 2^-5 in its scale; the sink, more
                # than gap - 2 above the keys before it, 2^((gap - 2) log2 e) times that, or 2^11 where the scale is new.
                most = np.zeros((n, block[-1] + 1))
                np.maximum.at(most.T, block, w.T)
                most[:, block[sink]] *= 2.0 ** -min(16.0, (gap - 2) * 1.4427)
                err += 2.0 ** -20 * (most[:, block] * seen) @ a
            d = np.abs(out[s, :, h] - w @ vv[h // G]) - err
            assert d.max() <= 0, f"request {s} head {h}: over its tolerance by {d.max():.3g} of {np.abs(out[s, :, h]).max():.3g}"


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("gap", [6, 8, 11, 14])
def test_a_key_that_takes_the_weight(hip, form, kind, gap):
    """A sink at the beginning, in the middle of the cache. So many requests that a wave has several blocks of keys: the
    pieces have up to 640 (16 or 32 rows; a wave has a quarter) or 512 keys (more rows), so a sum's chain is at most
    512 keys times three parts and the joins."""
    heads, n = form
    S = {1: 320, 4: 100, 5: 100, 6: 100}.get(n, 48)
    rng = np.random.default_rng(gap)
    for sink in (0, 333):
        q, k, v, table, row0, kv_len, page = case(rng, S, n, 650, heads, kind, sink, gap)
        out = run_attn(hip, q, k, v, table, row0, kv_len, None, heads, kind, page)
        check(out, q, k, v, table, row0, kv_len, page, heads, kind, sink, gap, 3 * 512 + 64)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_two_keys(hip, form, kind):
    """The sink and one more key with V = 1, 0 to 11 below it: the output is that key's probability, which has to have
    its bits (a part left out, the last of three too, is seen; the sink is 2^11 or more in the parts' scale, and they end
    at 2^-25). Its score x is one exact product: its exponent is off by the roundings of the scale, of log2 e, of their
    product, of the maximum and of the difference, five of x; the exponential, the sum of two, its inverse and the
    product are eight more."""
    heads, n = form
    H, HK, D = heads
    rng = np.random.default_rng(n)
    for i in range(24):
        gap = 11 * rng.random()
        q, k, v, table, row0, kv_len, page = case(rng, 2, n, 640, heads, kind, 0, gap)
        # only the first two keys of the cache are there: the rest lies in pages that the table does not name
        k[0, :, 1], v[0, :, 1] = 0, 1
        table[:, 1:] = -1
        full = run_attn(hip, q, k, v, table, row0, [2 + n] * 2, tree_of_nothing(n), heads, kind, page)
        x = float(k[0, 0, 0, 0].double()) * 4.0 * D ** -0.5
        want = math.exp(-x) / (1 + math.exp(-x))
        err = want * (U * (5 * x + 8) + max(PARTS[kind], 2.0 ** -36 * math.exp(x) if kind == "f16" else 0))
        d = (full.double() - want).abs().max().item()
        assert d <= err, (gap, d / want, err / want)


def tree_of_nothing(n):
    """Rows that see none of the new ones: the cache alone."""
    return np.zeros(2 * n, np.uint64)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-44, 3e-39, -3e-39, 1.17e-38])
def test_scales_next_to_zero(hip, form, scale):
    """bf16 scores of 2^126 times a scale below the smallest normal number, or of zero: weights that are equal for zero,
    and as the formula has them else."""
    import torch
    heads, n = form
    H, HK, D = heads
    rng = np.random.default_rng(n)
    q, k, v, table, row0, kv_len, page = case(rng, 2, n, 128, heads, "bf16", 0, 0)
    q.zero_()
    k.zero_()
    q[:, ::D] = 2.0 ** 63
    k[..., 0] = torch.from_numpy(rng.choice([-2.0 ** 63, 0.0, 2.0 ** 63], tuple(k.shape[:-1]))).cuda()
    out = run_attn(hip, q, k, v, table, row0, kv_len, None, heads, "bf16", page, scale=scale).double().cpu().numpy()
    s = float(np.float32(scale))
    kk, vv = k.double().cpu().numpy(), v.double().cpu().numpy()
    for r in range(2 * n):
        t, L = table[r // n], 128 + r % n + 1
        a, b = (np.moveaxis(c[t], 1, 0).reshape(HK, -1, D)[:, :L] for c in (kk, vv))
        for h in range(H):
            w = np.exp(2.0 ** 63 * a[h // (H // HK), :, 0] * s)
            w /= w.sum()
            want = w @ b[h // (H // HK)]
            # The scale's product with log2 e is a multiple of 2^-149, as the smallest stand-in for zero is: scores up to
            # 2^126 are off by up to 2^-23 times ln 2 each, the weights by twice that. Sums of 190 positive terms in
            # three parts each, and the exponentials.
            assert np.all(np.abs(out[r, h * D:(h + 1) * D] - want) <= want * (2 * 2.0 ** -23 + (3 * 190 + 40) * U))


@pytest.mark.parametrize("heads,new,tree", [((20, 4, 256), [1, 1, 1], False), ((20, 4, 256), [20, 3, 31], True), ((10, 2, 256), [90, 1, 70], False),
                                            ((8, 8, 128), [1, 1, 1], False), ((8, 2, 128), [6, 2, 8], True), ((8, 2, 128), [64, 9, 40], True),
                                            ((10, 2, 128), [150, 64, 1], False), ((4, 2, 64), [1, 2, 1], True),
                                            ((14, 2, 64), [4, 4, 3], False), ((8, 2, 64), [64, 33, 64], True)], ids=str)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_long_caches_in_which_each_row_looks_for_a_key(hip, heads, new, tree, kind):
    """Caches of thousands of keys, cut into pieces and joined; each row and head's query is twice some key, before its
    request's rows, among them or one that it must not see, so that a few keys carry its output wherever they lie."""
    import torch
    from test_gpu_serving import gpu_cache, trees
    H, HK, D = heads
    G, page = H // HK, 16
    g = torch.Generator(device="cuda").manual_seed(sum(new))
    rng = np.random.default_rng(sum(new))
    ctx = [9011, 700, 2500]
    kv_len = [c + n for c, n in zip(ctx, new)]
    k, v, table = gpu_cache(g, kv_len, heads, page)
    k, v = k.to(kind_of(kind)), v.to(kind_of(kind))
    row0 = np.cumsum([0] + new)
    bits = trees(rng, new, sum(new)) if tree else None
    dense = []
    for s, L in enumerate(kv_len):
        ids = torch.from_numpy(table[s, :-(-L // page)]).cuda().long()
        dense.append([c[ids].transpose(0, 1).reshape(HK, -1, D)[:, :L] for c in (k, v)])
    q = torch.zeros((sum(new), H, D), dtype=kind_of(kind), device="cuda")
    for s, L in enumerate(kv_len):
        for r in range(int(row0[s]), int(row0[s + 1])):
            at = torch.from_numpy(np.where(rng.random(H) < 0.5, rng.integers(0, L, H), rng.integers(ctx[s] - 40, L, H))).cuda()
            q[r] = 2 * dense[s][0][torch.arange(H, device="cuda") // G, at]
    q = q.reshape(-1, H * D)
    out = run_attn(hip, q, k, v, table, row0, kv_len, bits, heads, kind, page).double()
    for s, L in enumerate(kv_len):
        a, b = int(row0[s]), int(row0[s + 1])
        j = torch.arange(L, device="cuda")
        i = torch.arange(b - a, device="cuda")[:, None]
        seen = j - ctx[s] <= i
        if tree:
            own = torch.from_numpy(bits[a:b].view(np.int64)).cuda()[:, None] >> (j - ctx[s]).clamp(0, 63) & 1
            seen = (j < ctx[s]) | (own == 1)
        for h in range(H):
            kk, vv = (c[h // G].double() for c in dense[s])
            qq = q[a:b, h * D:(h + 1) * D].double()
            x, size = qq @ kk.T * D ** -0.5, qq.abs() @ kk.abs().T * D ** -0.5
            p = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
            # Scores: sums of D products, the scale and the exponent; the sums over the keys (pieces of at most 512 keys
            # in three parts, 72 pieces joined); the parts; fp16's small end, 2^-20 of a block's largest for its 32 keys.
            e = 2 * U * ((D + 8) * size.amax(-1, keepdim=True) + 8 * x.abs().amax(-1, keepdim=True)) + (3 * 512 + 200) * U + PARTS[kind]
            tol = e * (p @ vv.abs()) + (32 * 2.0 ** -20 * vv.abs().max() if kind == "f16" else 0)
            d = (out[a:b, h * D:(h + 1) * D] - p @ vv).abs() - tol
            assert float(d.max()) <= 0, (s, h, float(d.max()))
