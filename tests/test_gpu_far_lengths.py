"""GPU tests of the attentions over as many keys as lengths can say, by tables that name the same pages again and again."""
import math

import numpy as np
import pytest

from test_gpu_lora import words
from test_gpu_serving import host, ints, kind_of, stream

pytestmark = pytest.mark.gpu
D, PAGE, MOST = 64, 256, 2 ** 31 - 8192  # keys that are read of a request


def _torch():
    import torch
    return torch


def case(hip, kind, HK, H, S, n, ends):
    """Page 0: keys of score 0, the values a whole number for each dim (sums of 32 keys, and so of all, are exact in 32 bits);
    page 1, the pages `ends` of each row: keys of score 20, any whole numbers."""
    torch = _torch()
    rng = np.random.default_rng(n + HK)
    k = torch.zeros((2, HK, PAGE, D), device="cuda")
    k[1] = 20 / 64
    v = torch.from_numpy(rng.integers(0, 4, (2, HK, PAGE, D))).float().cuda()
    v[0] = v[0, :, :1]
    kv = hip.KvCache(k.to(kind_of(kind)), v.to(kind_of(kind)), hip.CacheType[kind], PAGE, HK, D, 2, HK * PAGE * D, PAGE * D, D)
    table = torch.zeros((S, 2 ** 31 // PAGE), dtype=torch.int32, device="cuda")
    table[:, ends] = 1
    T = S * n
    a = dict(S=S, T=T, heads=H, q=torch.ones((T, H * D), device="cuda").to(kind_of(kind)), ldq=H * D, table=table, ldt=table.shape[1],
             row0=ints(np.arange(S + 1) * n), scale=1.0, ldo=H * D)
    return kv, a, v.double().cpu().numpy()


def run(hip, kv, a, kv_len, shared):
    torch = _torch()
    out = torch.full((a["T"], a["ldo"]), math.nan, device="cuda")
    a = dict(a, kv_len=ints(kv_len), out=out)
    if shared is None:
        ws = words(hip.paged_attention_ws_bytes(a["S"], a["T"], a["heads"], kv))
        hip.launch_paged_attention(hip.PagedAttention(ws=ws, **a), kv, stream())
    else:
        ws = words(hip.shared_attention_ws_bytes(a["S"], a["T"], a["heads"], kv))
        hip.launch_shared_attention(hip.SharedAttention(ws=ws, groups=1, group0=ints([0, a["S"]]), lead=ints([0]), shared=ints([shared]), **a),
                                    kv, stream())
    return host(out).reshape(a["T"], a["heads"], D)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", [1, 24, 80])
@pytest.mark.parametrize("shared", [None, 0, 2 ** 30 + 5, 2 ** 31 - 1])
def test_lengths_at_the_end_of_their_type(hip, kind, n, shared):
    """The last page read has the keys of score 20. Sums of the others are exact; what is left are
    a score's rounding (20 / ln 2 in 32 bits: 2^-19), an exponential's and those of the joins, on values up to 3."""
    kv, a, v = case(hip, kind, 1, 1, 1 if shared is None else 2, n, MOST // PAGE - 1)
    for kv_len in (MOST, 2 ** 31 - 1):
        out = run(hip, kv, a, [kv_len] * a["S"], shared)
        for r in range(a["T"]):
            last = PAGE - max(0, n - 1 - r % n - (kv_len - MOST))  # keys of the last page that the row sees
            w = np.concatenate([np.full(PAGE, (MOST - PAGE) / PAGE), np.exp(20.0) * (np.arange(PAGE) < last)])
            want = (w[:, None] * v[:, 0].reshape(2 * PAGE, D)).sum(0) / w.sum()
            assert np.all(np.abs(out[r, 0] - want) <= 3 * 2.0 ** -17), (kv_len, r)


@pytest.mark.parametrize("shared", [None, 1000])
def test_pieces_of_many_keys(hip, shared):
    """32 KV heads over 1.9e9 keys: more than 2^27 in a piece. All scores 0."""
    n = 1900000000
    kv, a, v = case(hip, "f16", 32, 32, 2, 1, 0)
    a["table"].zero_()
    out = run(hip, kv, a, [n, 0], shared)
    assert np.all(np.abs(out[0] - v[0, :, 0]) <= 3 * 2.0 ** -20) and not out[1].any()
