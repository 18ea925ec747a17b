"""GPU tests of attention behind shared prefixes (launch_shared_attention): what launch_paged_attention's definition gives
over each request's own row of table, which the plain reference in 64 bits (serving_ref.py) reads."""
import dataclasses
import math

import numpy as np
import pytest

from test_gpu_serving import attn_inputs, check_attn, dev, host, ints, kind_of, run_attn, stream, trees, words

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def shared_inputs(rng, group0, prefix, lone, new, heads, kind, page, sharp=1.0, fill=0.0):
    """Requests whose groups hold the prefix's whole pages together; the page that it ends in is each one's own, with the
    same values. lone: tokens between prefix and new rows (all the tokens there of a request without a group)."""
    S = len(new)
    which = np.full(S, -1)
    for g in range(len(prefix)):
        which[group0[g]:group0[g + 1]] = g
    kv_len = [(prefix[w] if w >= 0 else 0) + a + n for w, a, n in zip(which, lone, new)]
    q, k, v, table, row0 = attn_inputs(rng, kv_len, new, heads, kind, page, sharp=sharp, fill=fill)
    for s in range(S):
        g = which[s]
        if g < 0 or s == group0[g]:
            continue
        lead, whole = group0[g], prefix[g] // page
        table[s, :whole] = table[lead, :whole]
        rest = prefix[g] % page
        if rest:
            for c in (k, v):
                c[table[s, whole], :, :rest] = c[table[lead, whole], :, :rest]
    return (q, k, v, table, row0), kv_len


def run_shared(hip, q, k, v, table, row0, kv_len, tree, heads, kind, page, group0, lead, prefix, scale=None, T=None, ld=0,
               strides=None, ws=None, pages=None):
    torch = _torch()
    H, HK, D = heads
    kv = hip.KvCache(k, v, hip.CacheType[kind], page, HK, D, pages or k.shape[0], *(strides or (HK * page * D, page * D, D)))
    T = T if T is not None else q.shape[0]
    S = len(kv_len)
    out = torch.full((max(T, q.shape[0]), H * D + ld), -77.0, dtype=torch.float32, device="cuda")
    ws = ws if ws is not None else words(hip.shared_attention_ws_bytes(S, T, H, kv))
    tree_d = dev(np.asarray(tree, np.uint64).view(np.int64)) if tree is not None else None
    a = hip.SharedAttention(S=S, T=T, heads=H, q=q, ldq=q.shape[1], table=ints(table), ldt=table.shape[1], row0=ints(row0),
                            kv_len=ints(kv_len), tree=tree_d, scale=D ** -0.5 if scale is None else scale, out=out, ldo=H * D + ld,
                            ws=ws, groups=len(prefix), group0=ints(group0) if len(prefix) else None,
                            lead=ints(lead) if len(prefix) else None, shared=ints(prefix) if len(prefix) else None)
    torch.cuda.synchronize()
    hip.launch_shared_attention(a, kv, stream())
    torch.cuda.synchronize()
    return out


def case(hip, rng, group0, prefix, lone, new, heads, kind, page, tree=False, sharp=1.0, fill=0.0, scale=None):
    x, kv_len = shared_inputs(rng, group0, prefix, lone, new, heads, kind, page, sharp, fill)
    bits = trees(rng, new, sum(new)) if tree else None
    out = run_shared(hip, *x, kv_len, bits, heads, kind, page, group0, group0[:-1], prefix, scale=scale)
    check_attn(out, *x, kv_len, bits, heads, kind, page, scale=scale)


HEADS = [(5, 1, 256), (20, 4, 256), (10, 2, 128), (6, 6, 64), (14, 2, 64), (3, 1, 128), (32, 8, 128)]
GROUPS = [  # first requests of the groups, their prefixes, tokens of each request's own, new rows
    ([0, 2], [64], [1, 0], [1, 1]), ([0, 4], [1000], [40, 17, 0, 33], [1] * 4), ([0, 3], [31], [5, 70, 0], [1] * 3),
    ([0, 3, 4, 7], [129, 200, 33], [9] * 7, [1] * 7), ([1, 3], [96], [300, 0, 20, 7, 64], [1] * 5), ([0, 5], [257], [0] * 5, [4, 1, 0, 9, 2]),
    ([0, 1, 3], [130, 65], [100, 3, 8], [1] * 3), ([0, 0, 2, 2], [50, 100, 70], [3, 300, 8], [2, 17, 1])]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("group0,prefix,lone,new", GROUPS, ids=str)
def test_groups(hip, heads, kind, group0, prefix, lone, new):
    """Prefixes that end inside pages and blocks, of less than a block, groups of one and of nobody, requests in no group."""
    rng = np.random.default_rng(sum(prefix))
    case(hip, rng, group0, prefix, lone, new, heads, kind, [16, 32, 64, 128, 256][sum(prefix) % 5], tree=sum(new) % 2 == 0)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,S,new", [((20, 4, 256), 12, 1), ((10, 2, 128), 70, 1), ((8, 1, 128), 40, 3), ((4, 4, 64), 40, 1),
                                         ((6, 2, 64), 30, 16), ((40, 8, 128), 6, 16), ((5, 1, 256), 3, 64), ((4, 1, 128), 2, 200)], ids=str)
def test_tiles(hip, kind, heads, S, new):
    """Rows of a group in one tile of every size and in several; prompts behind a prefix."""
    rng = np.random.default_rng(S)
    case(hip, rng, [0, S], [333], list(rng.integers(0, 40, S)), [new] * S, heads, kind, 16, tree=new == 16)


@pytest.mark.parametrize("heads,kind", [((20, 4, 256), "f16"), ((16, 2, 128), "bf16"), ((14, 2, 64), "f16")], ids=str)
def test_long_prefixes(hip, heads, kind):
    """Prefixes of many pieces and short ones beside them; own tokens of many pieces."""
    rng = np.random.default_rng(5)
    case(hip, rng, [0, 2, 5], [3000, 200], [10, 1500, 0, 33, 64], [1, 1, 2, 1, 1], heads, kind, 64)
    case(hip, rng, [0, 4], [40], [2000, 3, 5, 900], [1] * 4, heads, kind, 64)


def test_no_groups(hip):
    """Without groups, and with requests past the groups: as launch_paged_attention, to the tolerance."""
    rng = np.random.default_rng(6)
    case(hip, rng, [0], [], [30, 200], [1, 3], (10, 2, 128), "f16", 16)
    x, kv_len = shared_inputs(rng, [0], [], [30, 200], [1, 3], (10, 2, 128), "f16", 16)
    a = host(run_shared(hip, *x, kv_len, None, (10, 2, 128), "f16", 16, [0], [], []))
    b = host(run_attn(hip, *x, kv_len, None, (10, 2, 128), "f16", 16))
    assert np.abs(a - b).max() < 1e-5


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_members_that_do_not_take_part(hip, kind):
    """Refused requests (length 0 with rows), ones shorter than the prefix, without rows, with NaN queries; the lead among them."""
    torch = _torch()
    heads, page = (10, 2, 128), 16
    rng = np.random.default_rng(7)
    x, kv_len = shared_inputs(rng, [0, 6], [100], [5, 0, 20, 33, 7, 0], [2, 1, 3, 0, 1, 2], heads, kind, page, fill=math.nan)
    kv_len[0] = 0       # the lead, refused
    kv_len[2] = 60      # has less than the prefix
    kv_len[4] = 100     # its new row is the prefix's last token
    q = x[0].clone()
    q[:2] = math.nan
    x = (q,) + x[1:]
    out = run_shared(hip, *x, kv_len, None, heads, kind, page, [0, 6], [0], [100])
    assert bool((out[:2] == 0).all())
    q = q.clone()
    q[:2] = 0
    check_attn(out, q, *x[1:], kv_len, None, heads, kind, page)
    for none in (0, -1, -2 ** 31):
        assert bool((run_shared(hip, *x, [none] * 6, None, heads, kind, page, [0, 6], [0], [100]) == 0).all())


@pytest.mark.parametrize("S", [6, 70, 130])
def test_lengths_and_row_starts_at_the_ends_of_their_type(hip, S):
    """Lengths below zero give zeros, ones beyond the table what it holds; a row start beyond all others leaves its request
    the rows up to T, one below zero those from 0 on; where starts fall, the request before them is right."""
    heads, kind, page = (10, 2, 128), "f16", 16
    rng = np.random.default_rng(17)
    x, kv_len = shared_inputs(rng, [0, S], [100], [4] * S, [1] * S, heads, kind, page)
    q, k, v, table, row0 = x
    low, high = -2 ** 31, 2 ** 31 - 1
    full = table.shape[1] * page
    kv_len[1], kv_len[3] = low, high
    out = run_shared(hip, *x, kv_len, None, heads, kind, page, [0, S], [0], [100])
    want = list(kv_len)
    want[1], want[3] = 0, full  # (its row sees all that the table holds)
    check_attn(out, *x, want, None, heads, kind, page)
    row0 = row0.copy()
    row0[0], row0[S] = low, high
    check_attn(run_shared(hip, q, k, v, table, row0, kv_len, None, heads, kind, page, [0, S], [0], [100]), *x, want, None, heads, kind, page)
    row0[2:] = low
    out = run_shared(hip, q, k, v, table, row0, kv_len, None, heads, kind, page, [0, S], [0], [100])
    check_attn(out[:1], q[:1], k, v, table, np.array([0] + [1] * S), want, None, heads, kind, page)


@pytest.mark.parametrize("group0,lead,prefix", [
    ([0, 3], [-1], [64]), ([0, 3], [4], [64]), ([0, 3], [2 ** 31 - 1], [64]), ([0, 4], [0], [0]), ([0, 4], [0], [-5]), ([0, 4], [0], [2 ** 31 - 1]),
    ([3, 1], [0], [64]), ([-4, 9], [0], [64]), ([0, 2, 1, 4], [0, 1, 2], [64, 64, 64]), ([4, 4], [0], [64]), ([-2 ** 31, 2 ** 31 - 1], [0], [64]),
    ([0, 2, 4], [2, 0], [64, 64])], ids=str)
def test_groups_that_are_wrong(hip, group0, lead, prefix):
    """Leads and prefixes out of range, starts that fall or leave the batch: requests are done alone. (All hold the same first
    pages, so every group that is taken is right.)"""
    heads, kind, page = (5, 1, 128), "f16", 16
    rng = np.random.default_rng(8)
    x, kv_len = shared_inputs(rng, [0, 4], [64], [3, 40, 7, 0], [1, 2, 1, 1], heads, kind, page)
    out = run_shared(hip, *x, kv_len, None, heads, kind, page, group0, lead, prefix)
    check_attn(out, *x, kv_len, None, heads, kind, page)


@pytest.mark.parametrize("S", [6, 70, 130, 1100])
def test_a_workspace_at_16_bytes(hip, S):
    """Its start is at a multiple of 16 bytes and no more, as the header asks; nothing behind its end is written."""
    heads, kind, page = (10, 2, 64), "f16", 16
    rng = np.random.default_rng(S)
    x, kv_len = shared_inputs(rng, [0, S - 1], [96], list(rng.integers(0, 40, S)), [1] * S, heads, kind, page)
    kv = hip.KvCache(x[1], x[2], hip.CacheType[kind], page, 2, 64, x[1].shape[0], 2 * page * 64, page * 64, 64)
    n = -(-hip.shared_attention_ws_bytes(S, S, 10, kv) // 8)
    all_of = words(8 * (n + 66))
    skip = 2 + all_of.data_ptr() // 8 % 2
    out = run_shared(hip, *x, kv_len, None, heads, kind, page, [0, S - 1], [0], [96], ws=all_of[skip:])
    assert all_of[skip:].data_ptr() % 64 == 16 and bool((all_of[:skip] == -1).all()) and bool((all_of[skip + n:] == -1).all())
    check_attn(out, *x, kv_len, None, heads, kind, page)


def test_the_lead_is_another_row(hip):
    """The prefix is read through the lead's row alone: other pages with the same values, the members' own left unread."""
    torch = _torch()
    heads, kind, page = (6, 2, 64), "bf16", 16
    rng = np.random.default_rng(9)
    x, kv_len = shared_inputs(rng, [0, 3], [96], [10, 5, 0, 200], [1, 1, 1, 1], heads, kind, page)
    q, k, v, table, row0 = x
    for c in (k, v):  # request 3, in no group, holds the same six pages
        c[table[3, :6]] = c[table[0, :6]]
    want = table.copy()
    table = table.copy()
    table[:3, :6] = -1
    out = run_shared(hip, q, k, v, table, row0, kv_len, None, heads, kind, page, [0, 3], [3], [96])
    check_attn(out, q, k, v, want, row0, kv_len, None, heads, kind, page)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_infinities_and_nan(hip, kind, what):
    """In pages' rests, other branches and behind the end they have no effect; in what all see they count."""
    heads, page = (5, 1, 256), 32
    rng = np.random.default_rng(10)
    for new, tree in (([1, 1, 1], False), ([9, 20, 30], True)):
        x, kv_len = shared_inputs(rng, [0, 3], [140], [3, 0, 60], new, heads, kind, page, fill=what)
        bits = trees(rng, new, sum(new)) if tree else None
        check_attn(run_shared(hip, *x, kv_len, bits, heads, kind, page, [0, 3], [0], [140]), *x, kv_len, bits, heads, kind, page)
        q, k, v, table, row0 = x
        k, v = k.clone(), v.clone()
        v[table[0, 2], :, 7, 3:9] = what      # the prefix
        k[table[2, 5], :, 1, 5] = math.nan    # request 2's own
        x = (q, k, v, table, row0)
        with np.errstate(invalid="ignore"):
            check_attn(run_shared(hip, *x, kv_len, bits, heads, kind, page, [0, 3], [0], [140]), *x, kv_len, bits, heads, kind, page)


def test_sharp_rows(hip):
    """Scores far apart, a negative scale and one of zero: pieces of prefix and own keys with maxima far from each other."""
    rng = np.random.default_rng(11)
    for sharp, scale in ((12.0, None), (1.0, -0.3), (1.0, 0.0), (4.0, 1.0)):
        for kind in ("f16", "bf16"):
            case(hip, rng, [0, 3], [300], [50, 0, 170], [1, 2, 1], (10, 2, 128), kind, 16, sharp=sharp, scale=scale)


def test_strides_and_spare_rows(hip):
    """Tokens before heads in wider arrays; rows of q and out with gaps; more rows than the requests have."""
    torch = _torch()
    rng = np.random.default_rng(12)
    heads, page, kind = (6, 2, 64), 16, "bf16"
    H, HK, D = heads
    (q, k, v, table, row0), kv_len = shared_inputs(rng, [0, 2], [80], [5, 9], [4, 1], heads, kind, page)
    wide = []
    for c in (k, v):
        w = torch.full((c.shape[0], page, HK, D + 16), math.nan, dtype=c.dtype, device="cuda")
        w[..., :D] = c.permute(0, 2, 1, 3)
        wide.append(w)
    qw = torch.full((50, H * D + 8), math.nan, dtype=q.dtype, device="cuda")
    qw[:5, :H * D] = q
    out = run_shared(hip, qw, *wide, table, row0, kv_len, None, heads, kind, page, [0, 2], [0], [80], ld=12,
                     strides=(page * HK * (D + 16), D + 16, HK * (D + 16)))
    check_attn(out, qw, k, v, table, row0, kv_len, None, heads, kind, page)


@pytest.mark.parametrize("S,groups", [(64, 64), (65, 3), (100, 64), (127, 65), (128, 5), (129, 1), (300, 7), (1100, 2), (1500, 1100)])
def test_many_requests(hip, S, groups):
    """More requests and groups than the plan takes at once."""
    rng = np.random.default_rng(S)
    heads, kind, page = (2, 1, 64), "f16", 16
    group0 = [0] + sorted(rng.integers(0, S + 1, groups - 1).tolist()) + [S - 3]
    group0 = sorted(group0)
    prefix = rng.choice([32, 50, 64, 100], groups).tolist()
    case(hip, rng, group0, prefix, rng.integers(0, 30, S).tolist(), rng.integers(0, 3, S).tolist(), heads, kind, page)


def test_one_workspace(hip):
    """The bytes of the largest S and T serve smaller launches, without being cleared, and nothing is written behind them."""
    torch = _torch()
    rng = np.random.default_rng(13)
    for heads, kind in (((20, 4, 256), "f16"), ((8, 2, 128), "bf16"), ((4, 4, 64), "f16")):
        H, HK, D = heads
        kv = hip.KvCache(0, 0, hip.CacheType[kind], 16, HK, D, 9, 8, 8, D)
        big = hip.shared_attention_ws_bytes(40, 300, H, kv)
        ws = torch.full((big // 4 + 64,), math.nan, device="cuda")
        for S, new in ((1, 300), (40, 1), (40, 7), (3, 100), (2, 1), (9, 30)):
            x, kv_len = shared_inputs(rng, [0, S], [200], [11] * S, [new] * S, heads, kind, 16)
            out = run_shared(hip, *x, kv_len, None, heads, kind, 16, [0, S], [0], [200], ws=ws)
            check_attn(out, *x, kv_len, None, heads, kind, 16)
            assert bool(ws[big // 4:].isnan().all())


@pytest.mark.parametrize("heads", [(32, 8, 64), (16, 8, 256), (32, 8, 128)], ids=str)
def test_many_requests_behind_one_prefix(hip, heads):
    """One group in tiles of many rows, its members of one row each: nothing is written behind the workspace. Then row starts
    that do not ascend, each of whose requests claims all rows: no answer is defined, but nothing is written behind it either."""
    torch = _torch()
    rng = np.random.default_rng(16)
    S, kind, page = 700, "f16", 16
    x, kv_len = shared_inputs(rng, [0, S], [40], rng.integers(0, 9, S).tolist(), [1] * S, heads, kind, page)
    H, HK, D = heads
    kv = hip.KvCache(0, 0, hip.CacheType[kind], page, HK, D, 9, 8, 8, D)
    size = hip.shared_attention_ws_bytes(S, S, H, kv)
    ws = torch.full((size // 4 + 4096,), math.nan, device="cuda")
    out = run_shared(hip, *x, kv_len, None, heads, kind, page, [0, S], [0], [40], ws=ws)
    check_attn(out, *x, kv_len, None, heads, kind, page)
    assert bool(ws[size // 4:].isnan().all())
    q, k, v, table, row0 = x
    out = run_shared(hip, q, k, v, table, np.resize([0, S], S + 1), [10000] * S, None, heads, kind, page, [0, S], [0], [40], ws=ws)
    assert bool(ws[size // 4:].isnan().all()) and out.shape[0] == S


def test_captured(hip):
    """A graph, replayed with other lengths and groups and with eager work between; equal bits call for call."""
    torch = _torch()
    rng = np.random.default_rng(14)
    heads, kind, page, S = (10, 2, 128), "f16", 16, 5
    H, HK, D = heads
    (q, k, v, table, row0), kv_len = shared_inputs(rng, [0, S], [200], [60] * S, [2] * S, heads, kind, page)
    kv = hip.KvCache(k, v, hip.CacheType.f16, page, HK, D, k.shape[0], HK * page * D, page * D, D)
    T = 2 * S + 3
    qd = torch.zeros((T, H * D), dtype=q.dtype, device="cuda")
    qd[:2 * S] = q
    d = {"row0": ints(row0), "kv_len": ints(kv_len), "group0": ints([0, S, S]), "lead": ints([0, 0]), "shared": ints([200, 0])}
    out = torch.zeros((T, H * D), device="cuda")
    a = hip.SharedAttention(S=S, T=T, heads=H, q=qd, ldq=H * D, table=ints(table), ldt=table.shape[1], scale=D ** -0.5, out=out,
                            ldo=H * D, ws=words(hip.shared_attention_ws_bytes(S, T, H, kv)), groups=2, **d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        hip.launch_shared_attention(a, kv, torch.cuda.current_stream().cuda_stream)
    for group0, prefix in (([0, 5, 5], [200, 0]), ([0, 2, 5], [100, 200]), ([1, 3, 4], [64, 150]), ([0, 5, 5], [0, 0])):
        new = rng.integers(0, 3, S)
        r0 = np.cumsum(np.concatenate([[0], new]))
        n = [200 + int(rng.integers(0, 59)) + int(m) for m in new]
        for name, x in (("row0", r0), ("kv_len", n), ("group0", group0), ("shared", prefix)):
            d[name].copy_(ints(x))
        d["lead"].copy_(ints(group0[:2]))
        out.fill_(-77.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        check_attn(got, qd, k, v, table, r0, n, None, heads, kind, page)
        out.fill_(-77.0)
        hip.launch_shared_attention(a, kv, stream())
        torch.cuda.synchronize()
        assert torch.equal(out, got)


def test_far_pages(hip):
    """Pages beyond 2^32 bytes of the cache's start."""
    torch = _torch()
    rng = np.random.default_rng(15)
    heads, kind, page = (4, 1, 64), "f16", 16
    H, HK, D = heads
    (q, k, v, table, row0), kv_len = shared_inputs(rng, [0, 3], [50], [3, 20, 0], [1, 2, 1], heads, kind, page)
    n = k.shape[0]
    stride = 1 << 28  # values: 8 pages pass 2^32 bytes
    far = torch.zeros((n - 1) * stride + 4096, dtype=torch.float16, device="cuda")
    for p in range(n):
        far[p * stride:p * stride + page * D] = k[p].flatten()
        far[p * stride + 2048:p * stride + 2048 + page * D] = v[p].flatten()
    out = run_shared(hip, q, far, far[2048:], table, row0, kv_len, None, heads, kind, page, [0, 3], [0], [50], pages=n,
                     strides=(stride, 1024, D))
    check_attn(out, q, k, v, table, row0, kv_len, None, heads, kind, page)
