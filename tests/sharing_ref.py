"""Plain references of the operators for requests that share (include/btf/hip_abi.h), in
whole numbers or 64 bits on the host, one fork, place, token or row after another."""
import numpy as np


def pages_of(tokens, page):
    return -(-int(tokens) // page)


def fork(src, dst, tokens, free, n_free, table, held, shared, page, pages):
    """Outputs of launch_page_fork; the inputs are copied."""
    S, ldt = table.shape
    table, held, shared, before = table.copy(), held.copy(), shared.copy(), held.copy()
    left, refused, taken = max(0, n_free), False, set()
    got, frm, to, count = ([] for _ in range(4))
    for s, d, n in zip(src, dst, tokens):
        ok = 0 <= s < S and 0 <= d < S and s != d and n >= 0
        ok = ok and before[s] <= ldt and n <= int(before[s]) * page and before[d] == 0 and d not in taken
        if ok:
            taken.add(d)
        entry = (-1, -1, 0)
        if ok and n % page:
            if refused or left == 0:
                ok, refused = False, True
            else:
                left -= 1
                entry = (table[s, n // page], free[left], n % page)
        if ok:
            for j in range(n // page):
                p = table[d, j] = table[s, j]
                if 0 <= p < pages:
                    shared[p] += 1
            if n % page:
                table[d, n // page] = entry[1]
            held[d] = pages_of(n, page)
        got.append(n if ok else -1)
        frm.append(entry[0]), to.append(entry[1]), count.append(entry[2])
    return {"table": table, "held": held, "shared": shared, "n_free": np.array([left]), "got": np.array(got),
            "copy_from": np.array(frm), "copy_to": np.array(to), "copy_tokens": np.array(count)}


def free(keep, table, held, shared, free_list, n_free, page, pages):
    """Outputs of launch_page_free; shared may be None."""
    S, ldt = table.shape
    table, held, free_list = table.copy(), held.copy(), free_list.copy()
    holders, order = {}, []
    for s in range(S):
        first = pages_of(max(0, keep[s]), page)
        for j in range(first, min(ldt, int(held[s]))):
            p = int(table[s, j])
            table[s, j] = -1
            if 0 <= p < pages:
                if p not in holders or shared is None:
                    order.append(p)
                holders[p] = holders.get(p, 0) + 1
        held[s] = min(int(held[s]), first)
    if shared is not None:
        shared = shared.copy()
        order = [p for p in order if holders[p] > shared[p]]
        for p, n in holders.items():
            shared[p] = max(0, shared[p] - n)
    n = min(max(0, n_free), pages)
    for p in order[::-1]:
        if n < pages:
            free_list[n] = p
            n += 1
    return {"table": table, "held": held, "shared": shared, "free": free_list, "n_free": np.array([n])}


def move(k, v, table, to_table, first, lists, page):
    """k and v [layers][pages][heads][page][dim] after launch_cache_move; lists: the kept places of each request."""
    out = [k.copy(), v.copy()]
    pages = k.shape[1]
    there = table if to_table is None else to_table

    def at(t, s, place):
        if not 0 <= place < t.shape[1] * page:
            return None
        p = int(t[s, place // page])
        return (p, place % page) if 0 <= p < pages else None
    for s, places in enumerate(lists):
        for i, place in enumerate(places):
            a, b = at(table, s, int(place)), at(there, s, int(first[s]) + i)
            if a and b:
                for x, y in zip((k, v), out):
                    y[:, b[0], :, b[1]] = x[:, a[0], :, a[1]]
    return out


def lora(x, row0, adapter, ranks, scale, a, b, T):
    """Delta [T][N] of one segment, and the sizes of its sums: sum |b| sum |a x| and sum |b h|."""
    N = b.shape[1]
    delta, deep, flat = (np.zeros((T, N)) for _ in range(3))
    for s, w in enumerate(adapter):
        lo, hi = max(0, int(row0[s])), min(T, int(row0[s + 1]))
        if hi <= lo or not 0 <= w < a.shape[0]:
            continue
        r = a.shape[1] if ranks is None else min(max(0, int(ranks[w])), a.shape[1])
        f = 1.0 if scale is None else float(scale[w])
        A, B = a[w, :r].astype(np.float64), b[w, :, :r].astype(np.float64)
        h = x[lo:hi].astype(np.float64) @ A.T
        delta[lo:hi] = f * (h @ B.T)
        deep[lo:hi] = abs(f) * ((np.abs(x[lo:hi]).astype(np.float64) @ np.abs(A).T) @ np.abs(B).T)
        flat[lo:hi] = abs(f) * (np.abs(h) @ np.abs(B).T)
    return delta, deep, flat
