"""Plain references of a serving step's operators, in 64 bits on the host.

They follow the definitions in include/btf/hip_abi.h request by request, row by
row; the tests compare the kernels with them.
"""
import math

import numpy as np

TREE = 64


def to16(x, kind):
    """Rounded to the 16-bit type (to nearest even) and back, as float64."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).to(torch.float16 if kind == "f16" else torch.bfloat16)
    return t.double().numpy()


HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of a rounding, relative to the value


def plan(ctx, n_new, held, parent, free, n_free, table, T, page, pages):
    """Outputs of launch_page_plan as a dict; table is copied. Rows past the last are None."""
    S, ldt = table.shape
    table, held_out = table.copy(), np.array(held).copy()
    row0, kv_len = np.zeros(S + 1, np.int64), np.zeros(S, np.int64)
    pos, slot, tree = {}, {}, {}
    left, refused, row = max(0, n_free), False, 0
    for s in range(S):
        c, n, h = int(ctx[s]), int(n_new[s]), int(held[s])
        rows = max(n, 0)
        row0[s] = min(row, T)
        total = -(-(c + n) // page)
        ok = c >= 0 and n >= 0 and 0 <= h <= ldt and c <= h * page and row + rows <= T and total <= ldt \
            and c + n < 2 ** 31
        if ok and total > h:
            if refused or total - h > left:
                ok, refused = False, True
            else:
                for j in range(h, total):
                    left -= 1
                    table[s, j] = free[left]
                held_out[s] = total
        kv_len[s] = c + n if ok else 0
        depth, bits = {}, {}
        for i in range(min(rows, T - min(row, T))):
            r = row + i
            tr = parent is not None and n <= TREE
            p = int(parent[r]) if tr else i - 1
            if not 0 <= p < i:
                p = -1
            depth[i] = depth[p] + 1 if p >= 0 else 0
            bits[i] = (bits[p] if p >= 0 else 0) | (1 << i)
            pos[r], slot[r], tree[r] = 0, -1, 0
            if ok:
                pg = int(table[s, (c + i) // page])
                pos[r] = c + depth[i]
                slot[r] = pg * page + (c + i) % page if 0 <= pg < pages else -1
                tree[r] = bits[i] if tr else 0
        row += rows
    row0[S] = min(row, T)
    return {"table": table, "held_out": held_out, "n_free_out": left if n_free >= 0 else 0, "row0": row0,
            "kv_len": kv_len, "pos": pos, "slot": slot, "tree": tree}


def turned(x, pos, turns, mscale, n_rot, layout, norm=None, eps=0.0):
    """(heads [T][n][D] normed and turned, a bound of |values| for the tolerance)."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * norm.astype(np.float64)
    y, size = x.copy(), np.abs(x)
    for t in range(x.shape[0]):
        for i in range(n_rot // 2):
            a, b = (i, i + n_rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
            w = float(pos[t]) * float(turns[i])
            w = 2 * math.pi * (w - math.floor(w))
            c, s = math.cos(w) * mscale, math.sin(w) * mscale
            y[t, :, a] = x[t, :, a] * c - x[t, :, b] * s
            y[t, :, b] = x[t, :, a] * s + x[t, :, b] * c
            size[t, :, a] = size[t, :, b] = (np.abs(x[t, :, a]) + np.abs(x[t, :, b])) * abs(mscale)
    return y, size


def visible(row0, kv_len, tree, s, i, L):
    """What new row i of request s sees of its L tokens."""
    n = int(row0[s + 1] - row0[s])
    ctx = int(kv_len[s]) - n
    j = np.arange(L)
    if tree is not None and n <= TREE:
        bits = int(tree[row0[s] + i]) & (2 ** 64 - 1)
        new = np.array([0 <= k - ctx < 64 and bits >> (k - ctx) & 1 == 1 for k in range(L)], bool)
        return (j < ctx) | new
    return j - ctx <= i


def attention(q, k, v, table, row0, kv_len, tree, scale, page, pages, heads, kv_heads):
    """(out [T][heads * D], tolerance [T][heads * D]) of 16-bit values given as float64: q [T][heads * D],
    k and v [pages][kv_heads][page][D]. The tolerance counts 32-bit roundings: each score's sum, the exponential,
    the sums over the keys, at their worst."""
    T, D, G, u = q.shape[0], k.shape[-1], heads // kv_heads, 2.0 ** -24
    out, tol = np.zeros((T, heads * D)), np.zeros((T, heads * D))
    for s in range(len(kv_len)):
        L = min(int(kv_len[s]), table.shape[1] * page)
        ids = np.repeat(table[s], page)[:L].astype(np.int64)
        good = (ids >= 0) & (ids < pages)
        at = np.where(good, ids, 0)
        off = np.arange(L) % page
        for i in range(int(row0[s + 1] - row0[s])):
            see = visible(row0, kv_len, tree, s, i, L) & good
            if not see.any():
                continue
            t = int(row0[s]) + i
            for h in range(heads):
                kk, vv = k[at[see], h // G, off[see]], v[at[see], h // G, off[see]]
                qq = q[t, h * D:(h + 1) * D]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = kk @ qq * scale
                    size = np.abs(kk) @ np.abs(qq) * abs(scale)
                    if np.all(x == -np.inf):
                        continue
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    out[t, h * D:(h + 1) * D] = w @ vv
                    err = 2 * ((D + 8) * u * size.max() + 8 * u * np.abs(x).max()) + (see.sum() + 32) * u
                    tol[t, h * D:(h + 1) * D] = err * (w @ np.abs(vv))
    return out, tol


def sample(x, T, top_k, top_p, min_p, u):
    """(token, logprob) of one row of logits, weights in whole units of 2^-43."""
    V = x.size
    key = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    live = ~np.isnan(x)
    if not live.any():
        return 0, 0.0
    order = sorted(np.flatnonzero(live).tolist(), key=lambda i: (-key[i], i))
    best = order[0]
    if not T > 0:
        return best, 0.0

    def weight(i):
        if key[i] == key[best]:
            return 2 ** 43
        return int(np.rint(np.exp((key[i] - key[best]) / float(T)) * 2.0 ** 43))
    w = {i: weight(i) for i in order}
    if top_k > 0:
        order = order[:int(top_k)]
    if top_p < 1:
        want, s, kept = float(top_p) * sum(w[i] for i in order), 0, []
        for i in order:
            if kept and not s < want:
                break
            kept.append(i)
            s += w[i]
        order = kept
    if min_p > 0:
        order = [i for i in order if w[i] >= min(float(min_p), 1.0) * 2.0 ** 43]
    total = sum(w[i] for i in order)
    at = min(max(int(float(u) * total) if u > 0 else 0, 0), total - 1)
    s = 0
    for i in sorted(order):
        s += w[i]
        if s > at:
            return i, math.log(w[i] / total)
    raise AssertionError
