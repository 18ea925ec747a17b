"""CPU tests of a serving step's operators: what the launches refuse before any
HIP call (no device exists in this process, so reaching one gives another
code), the layout of the argument structs, and the table of rotary frequencies.
"""
import dataclasses
import math
import os
import subprocess

import numpy as np
import pytest

import btf_hip as h

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x100000  # an aligned address; nothing reads it
ARGS, NOT_INIT = h.BTF_ERR_ARGS, h.BTF_ERR_NOT_INIT

KV = h.KvCache(A, A, h.CacheType.f16, 64, 4, 256, 100, 4 * 64 * 256, 64 * 256, 256)
PLAN = h.PagePlan(S=2, T=8, page=64, ldt=4, pages=100, ctx=A, n_new=A, held=A, parent=A, free=A, n_free=A, table=A,
                  held_out=A, n_free_out=A, row0=A, kv_len=A, pos=A, slot=A, tree=A)
ROPE = h.RopeCache(T=3, heads=20, q=A, ldq=7168, k=A, ldk=7168, v=A, ldv=7168, q_norm=A, k_norm=A, eps=1e-6, n_rot=64,
                   layout=0, turns=A, mscale=1.0, pos=A, slot=A, rows=A, q_out=A, ldqo=5120)
ATTN = h.PagedAttention(S=2, T=8, heads=20, q=A, ldq=5120, table=A, ldt=4, row0=A, kv_len=A, tree=A, scale=0.0625,
                        out=A, ldo=5120, ws=A)
SAMPLE = h.Sampling(M=2, V=1000, logits=A, ldl=1000, temperature=A, top_k=A, top_p=A, min_p=A, u=A, token=A, logprob=A,
                    ws=A)


def launch(op, a, kv=KV):
    return {"plan": lambda: h.launch_page_plan_raw(a), "rope": lambda: h.launch_rope_cache_raw(a, kv),
            "attn": lambda: h.launch_paged_attention_raw(a, kv), "sample": lambda: h.launch_sample_raw(a)}[op]()


VALID = {"plan": PLAN, "rope": ROPE, "attn": ATTN, "sample": SAMPLE}
REFUSED = [
    ("plan", dict(T=-1)), ("plan", dict(page=48)), ("plan", dict(page=0)), ("plan", dict(ldt=0)),
    ("plan", dict(pages=0)), ("plan", dict(pages=1 << 25, page=64)), ("plan", dict(parent=None)),
    ("plan", dict(tree=None)), ("plan", dict(tree=A + 4)),
    *[("plan", {n: None}) for n in ("ctx", "n_new", "held", "free", "n_free", "table", "held_out", "n_free_out", "row0",
                                    "kv_len", "pos", "slot")],
    ("rope", dict(q=None, k=None, v=None)), ("rope", dict(v=None)), ("rope", dict(k=None)), ("rope", dict(heads=0)),
    ("rope", dict(q_out=None)), ("rope", dict(ldq=5119)), ("rope", dict(ldqo=5119)), ("rope", dict(ldk=1023)),
    ("rope", dict(ldv=1023)), ("rope", dict(slot=None)), ("rope", dict(n_rot=63)), ("rope", dict(n_rot=258)),
    ("rope", dict(n_rot=-2)), ("rope", dict(layout=2)), ("rope", dict(turns=None)), ("rope", dict(pos=None)),
    ("rope", dict(q=A + 2)), ("rope", dict(turns=A + 4)),
    ("attn", dict(heads=0)), ("attn", dict(heads=18)), ("attn", dict(q=A + 8)), ("attn", dict(ldq=5124)),
    ("attn", dict(ldq=5112)), ("attn", dict(out=A + 4)), ("attn", dict(ldo=5122)), ("attn", dict(ldo=5116)),
    ("attn", dict(T=1 << 28, heads=20)), ("attn", dict(ldt=0)), ("attn", dict(tree=A + 4)), ("attn", dict(scale=math.nan)),
    *[("attn", {n: None}) for n in ("q", "table", "row0", "kv_len", "out")],
    ("sample", dict(V=0)), ("sample", dict(V=(1 << 20) + 1, ldl=1 << 21)), ("sample", dict(ldl=999)),
    *[("sample", {n: None}) for n in ("logits", "u", "token")],
]


@pytest.mark.parametrize("op,change", REFUSED, ids=lambda v: str(v))
def test_refused_before_any_hip_call(op, change):
    assert launch(op, dataclasses.replace(VALID[op], **change)) == ARGS
    assert h.last_error()


@pytest.mark.parametrize("op", ["rope", "attn"])
@pytest.mark.parametrize("change", [
    dict(type=2), dict(page=8), dict(page=512), dict(page=24), dict(dim=96), dict(heads=0), dict(k=None), dict(v=None),
    dict(k=A + 8), dict(v=A + 8), dict(pages=0), dict(pages=1 << 25), dict(tok_stride=248), dict(tok_stride=260),
    dict(head_stride=-8), dict(head_stride=4), dict(page_stride=12),
    dict(tok_stride=(1 << 24) + 8)], ids=str)
def test_caches_refused(op, change):
    assert launch(op, VALID[op], dataclasses.replace(KV, **change)) == ARGS


@pytest.mark.parametrize("op", list(VALID))
def test_null_arguments(op):
    assert launch(op, None) == ARGS
    if op in ("rope", "attn"):
        assert launch(op, VALID[op], None) == ARGS


@pytest.mark.parametrize("op,change", [("plan", {}), ("plan", dict(parent=None, tree=None)), ("plan", dict(T=0, pos=None, slot=None)),
                                       ("rope", {}), ("rope", dict(q=None)), ("rope", dict(k=None, v=None, slot=None)),
                                       ("rope", dict(n_rot=0, turns=None, pos=None)), ("rope", dict(n_rot=62)),
                                       ("attn", {}), ("attn", dict(tree=None)), ("sample", {}),
                                       ("sample", dict(temperature=None, top_k=None, top_p=None, min_p=None, logprob=None)),
                                       ("sample", dict(M=1, ldl=0))], ids=lambda v: str(v))
def test_valid_arguments_need_a_device(op, change):
    assert launch(op, dataclasses.replace(VALID[op], **change)) == NOT_INIT


@pytest.mark.parametrize("op,change", [("plan", dict(S=0)), ("plan", dict(S=-1)), ("rope", dict(T=0)), ("attn", dict(T=0)),
                                       ("attn", dict(S=0)), ("sample", dict(M=0)), ("sample", dict(M=-3))], ids=lambda v: str(v))
def test_nothing_to_do(op, change):
    assert launch(op, dataclasses.replace(VALID[op], **change)) == h.BTF_OK


def test_missing_workspace():
    if h.paged_attention_ws_bytes(2, 8, 20, KV) > 0:
        assert launch("attn", dataclasses.replace(ATTN, ws=None)) == ARGS
        assert launch("attn", dataclasses.replace(ATTN, ws=A + 8)) == ARGS
    if h.sample_ws_bytes(2, 1000) > 0:
        assert launch("sample", dataclasses.replace(SAMPLE, ws=None)) == ARGS
        assert launch("sample", dataclasses.replace(SAMPLE, ws=A + 4)) == ARGS


def test_workspace_for_the_largest_launch_serves_smaller_ones():
    for dim in (64, 128, 256):
        kv = dataclasses.replace(KV, dim=dim)
        sizes = [h.paged_attention_ws_bytes(1, T, 20, kv) for T in (1, 3, 4, 5, 6, 7, 50, 512, 4096)]
        assert sizes == sorted(sizes)
        for S in (2, 16, 400):
            assert all(h.paged_attention_ws_bytes(S, T, 20, kv) <= sizes[-1] for T in (1, 16, 400, 4096))
    assert h.sample_ws_bytes(3, 1000) == 3 * h.sample_ws_bytes(1, 1000) < h.sample_ws_bytes(3, 200000)


def test_workspace_of_nothing():
    assert h.paged_attention_ws_bytes(0, 8, 20, KV) == 0
    assert h.paged_attention_ws_bytes(2, 8, 18, KV) == 0
    assert h.paged_attention_ws_bytes(2, 8, 20, dataclasses.replace(KV, dim=96)) == 0
    assert h.sample_ws_bytes(0, 1000) == 0 and h.sample_ws_bytes(2, 0) == 0


def test_struct_layouts(tmp_path):
    """The ctypes structs have the header's sizes and field offsets."""
    structs = {"btf_kv_cache": h._KvCache, "btf_page_plan": h._PagePlan, "btf_rope_scale": h._RopeScale,
               "btf_rope_cache": h._RopeCache, "btf_paged_attention": h._PagedAttention, "btf_sampling": h._Sampling}
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "btf/hip_abi.h"', "int main(void) {"]
    want = []
    for name, c in structs.items():
        src.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(str(__import__("ctypes").sizeof(c)))
        for f, _ in c._fields_:
            src.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(str(getattr(c, f).offset))
    (tmp_path / "s.c").write_text("\n".join(src + ["return 0; }"]))
    subprocess.run(["cc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    assert subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split() == want


# ---- the table of frequencies (host) ----
@pytest.mark.parametrize("n_rot", [2, 6, 64, 128, 246, 256])
@pytest.mark.parametrize("base", [1e4, 1e7])
def test_rope_table_plain_linear_ntk(n_rot, base):
    i = np.arange(n_rot // 2)
    plain = base ** (-2.0 * i / n_rot) / (2 * math.pi)
    turns, m = h.rope_table(n_rot, base)
    np.testing.assert_allclose(turns, plain, rtol=1e-13)
    assert m == 1.0
    turns, m = h.rope_table(n_rot, base, h.RopeScale(h.RopeScaling.linear, 8.0))
    np.testing.assert_allclose(turns, plain / 8, rtol=1e-13)
    assert m == 1.0
    if n_rot > 2:
        turns, m = h.rope_table(n_rot, base, h.RopeScale(h.RopeScaling.ntk, 4.0))
        np.testing.assert_allclose(turns, (base * 4.0 ** (n_rot / (n_rot - 2))) ** (-2.0 * i / n_rot) / (2 * math.pi), rtol=1e-12)
        # the slowest pair is stretched by the whole factor, the fastest not at all
        np.testing.assert_allclose([turns[0], turns[-1]], [plain[0], plain[-1] / 4.0], rtol=1e-12)


@pytest.mark.parametrize("n_rot,trained,factor", [(64, 32768, 4.0), (128, 4096, 16.0), (256, 8192, 2.0)])
def test_rope_table_yarn(n_rot, trained, factor):
    base = 1e6
    plain = np.array(h.rope_table(n_rot, base)[0])
    turns, m = h.rope_table(n_rot, base, h.RopeScale(h.RopeScaling.yarn, factor, trained, 32.0, 1.0))
    assert m == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-7)
    ratio = plain / np.array(turns)
    # pairs that turn often over the trained context keep their frequency, slow ones are stretched, between them a ramp
    assert np.all(np.diff(ratio) >= -1e-9)
    np.testing.assert_allclose(ratio[plain * trained > 32.0 * base ** (2.0 / n_rot)], 1.0, rtol=1e-12)
    np.testing.assert_allclose(ratio[plain * trained < 1.0 / base ** (2.0 / n_rot)], factor, rtol=1e-12)
    assert ratio[0] == pytest.approx(1.0) and ratio[-1] == pytest.approx(factor)


@pytest.mark.parametrize("n_rot,base,scale", [
    (0, 1e4, None), (3, 1e4, None), (64, 1.0, None), (64, math.nan, None), (64, 1e4, h.RopeScale(4, 2.0)),
    (64, 1e4, h.RopeScale(1, 0.5)), (2, 1e4, h.RopeScale(2, 2.0)), (64, 1e4, h.RopeScale(3, 2.0, 0.0)),
    (64, 1e4, h.RopeScale(3, 2.0, 4096.0, 1.0, 32.0)), (64, 1e4, h.RopeScale(1, math.nan))], ids=str)
def test_rope_table_refused(n_rot, base, scale):
    with pytest.raises(RuntimeError, match="rope_table"):
        h.rope_table(n_rot, base, scale)


# ---- the native launch calls ----
@pytest.mark.skipif(not os.path.exists(h.CALL_PATH), reason="native launch calls not built")
@pytest.mark.parametrize("op", list(VALID))
@pytest.mark.parametrize("stream", [None, 0, 1 << 45])
def test_native_calls_hand_over_the_same_structs(op, stream):
    """Recorders in place of the launchers: the struct bytes of the native call are those of the ctypes path."""
    import ctypes as C
    import torch
    t = torch.zeros(64)
    two = op in ("rope", "attn")
    c_types = {"plan": h._PagePlan, "rope": h._RopeCache, "attn": h._PagedAttention, "sample": h._Sampling}
    seen = []
    ptr = [C.POINTER(c_types[op])] + ([C.POINTER(h._KvCache)] if two else []) + [C.c_void_p]

    def record(*v):
        seen.append(([tuple(getattr(x[0], f) for f, _ in x[0]._fields_) for x in v[:-1]], v[-1]))
        return 5
    f = C.CFUNCTYPE(C.c_int, *ptr)(record)
    a = VALID[op]
    for name in a.__dataclass_fields__:  # tensors and None among the addresses
        if getattr(a, name) is A:
            a = dataclasses.replace(a, **{name: t})
            break
    a = dataclasses.replace(a, **{[n for n in a.__dataclass_fields__ if getattr(a, n) is A][-1]: None})
    kv = dataclasses.replace(KV, v=t) if two else None
    layout = {"plan": h._plan_layout, "rope": h._rope_layout, "attn": h._attn_layout, "sample": h._sample_layout}[op]
    rc = h._call.launch(C.cast(f, C.c_void_p).value, layout, a, h._kv_layout if two else -1, kv, stream)
    assert rc == 5
    want = [tuple(getattr(x._c(), n) for n, _ in x._c()._fields_) for x in ([a, kv] if two else [a])]
    assert seen == [(want, stream or None)]


@pytest.mark.skipif(not os.path.exists(h.CALL_PATH), reason="native launch calls not built")
def test_native_calls_leave_other_forms_to_ctypes():
    class Sub(h.Sampling):
        pass
    sample = lambda a: h._call.launch(h._addr_sample, h._sample_layout, a, -1, None, None)  # noqa: E731
    rope = lambda a, kv: h._call.launch(h._addr_rope_cache, h._rope_layout, a, h._kv_layout, kv, None)  # noqa: E731
    assert sample(Sub()) is NotImplemented
    assert sample(None) is NotImplemented
    assert sample(PLAN) is NotImplemented  # (a struct of another launch)
    assert sample(dataclasses.replace(SAMPLE, V=3.5)) is NotImplemented
    assert rope(dataclasses.replace(ROPE, eps=1), KV) is NotImplemented
    assert rope(ROPE, None) is NotImplemented
    assert rope(ROPE, SAMPLE) is NotImplemented
    with pytest.raises(AttributeError):
        sample(dataclasses.replace(SAMPLE, u=object()))
    with pytest.raises(TypeError):
        h._call.launch(h._addr_sample, SAMPLE)
    with pytest.raises(RuntimeError, match="sample"):
        h.launch_sample(dataclasses.replace(SAMPLE, V=0))
    with pytest.raises(RuntimeError, match="null arguments"):
        h.launch_sample(None)
    with pytest.raises(RuntimeError, match="null cache"):
        h.launch_rope_cache(ROPE, None)
    import ctypes
    with pytest.raises(ctypes.ArgumentError):
        h.launch_sample(PLAN)


@pytest.mark.skipif(not os.path.exists(h.CALL_PATH), reason="native launch calls not built")
@pytest.mark.parametrize("how", ["reload", "second name"])
def test_module_executed_again(how):
    """btf_hip executed twice in one process, by importlib.reload or under another name: launches of both go through, the
    newer one's by the native calls, and as often as one likes."""
    code = f"""
import gc, importlib, importlib.util, sys
sys.path.insert(0, {os.path.dirname(h.__file__)!r})
import btf_hip
first = btf_hip
for i in range(9):
    if {how == "reload"}:
        old = first.Sampling(M=1, V=0)
        new = importlib.reload(btf_hip)
    else:
        spec = importlib.util.spec_from_file_location("again%d" % i, btf_hip.__file__)
        new = importlib.util.module_from_spec(spec)
        sys.modules[spec.name] = new
        spec.loader.exec_module(new)
        old = first.Sampling(M=1, V=0)
    gc.collect()
    args = lambda m, a: (m._addr_sample, m._sample_layout, a, -1, None, None)
    assert new._call.launch(*args(new, new.Sampling(M=1, V=0))) == {ARGS}
    assert new._call.launch(*args(new, old)) is NotImplemented
    for m in (first, new):
        for call in (lambda: m.launch_sample(m.Sampling(M=1, V=0)), lambda: m.launch_rope_cache(m.RopeCache(T=1), None),
                     lambda: m.launch_paged_attention(m.PagedAttention(S=1, T=1), m.KvCache()),
                     lambda: m.launch_page_plan(m.PagePlan(S=1, T=-1))):
            try:
                call()
            except RuntimeError:
                continue
            raise SystemExit("not refused")
print("done")
"""
    r = subprocess.run([os.sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


@pytest.mark.skipif(not os.path.exists(h.CALL_PATH), reason="native launch calls not built")
@pytest.mark.parametrize("args", [(), (0, h.Sampling, ()), (-1, h.Sampling, (), 8), (8, h.Sampling, (), 8), (0, h.Sampling, [], 8),
                                  (0, h.Sampling, (), 257), (0, h.Sampling, (), -1), (5, h.Sampling, (("M", "i", 253),), 256),
                                  (5, h.Sampling, (("M", "i", -8),), 8), (5, h.Sampling, (("M", "i"),), 8), (5, h.Sampling, ("M",), 8),
                                  (5, h.Sampling, (("M", "", 0),), 8), (5, h.Sampling, (("M", "i", 0),) * 25, 8),
                                  (2 ** 70, h.Sampling, (), 8)], ids=str)
def test_layouts_refused(args):
    """A refused registration changes nothing: the launches still read their structs, slot 5 is still empty."""
    with pytest.raises((ValueError, TypeError, OverflowError)):
        h._call.layout(*args)
    assert h._call.launch(h._addr_sample, h._sample_layout, dataclasses.replace(SAMPLE, V=0), -1, None, None) == ARGS
    assert h._call.launch(h._addr_sample, 5, SAMPLE, -1, None, None) is NotImplemented


@pytest.mark.parametrize("op,change,kv", [
    ("plan", dict(S=1 << 26), {}), ("plan", dict(S=2 ** 31 - 1), {}), ("plan", dict(T=65535 * 1024 + 1), {}),
    ("plan", dict(T=2 ** 31 - 1), {}), ("rope", dict(T=1 << 24), {}), ("rope", dict(T=2 ** 31 - 1), {}),
    ("rope", dict(heads=65528, ldq=2 ** 31 - 1, ldqo=2 ** 31 - 1), {}),
    ("rope", dict(ldk=2 ** 31 - 1, ldv=2 ** 31 - 1), dict(heads=32768)),
    ("attn", dict(T=1 << 24), {}), ("attn", dict(S=1 << 22), {}), ("attn", dict(S=1 << 26), {}),
    ("attn", dict(S=2 ** 31 - 1, heads=65535, ldq=2 ** 31 - 8, ldo=2 ** 31 - 4), dict(heads=65535, dim=64, tok_stride=64)),
    # 2^32 items and 1536: a grid that would wrap to 1536
    ("attn", dict(S=1 << 26, T=1, heads=64, ldq=64 * 64, ldo=64 * 64), dict(heads=64, dim=64, tok_stride=64))], ids=str)
def test_launches_beyond_the_grid_refused(op, change, kv):
    """Before the first kernel, since a launch of several could otherwise stop after it, and a grid could wrap."""
    assert launch(op, dataclasses.replace(VALID[op], **change), dataclasses.replace(KV, **kv)) == ARGS


@pytest.mark.parametrize("op,change,kv", [
    ("plan", dict(S=(1 << 26) - 1), {}), ("plan", dict(T=65535 * 1024), {}), ("rope", dict(T=(1 << 24) - 1), {}),
    ("rope", dict(heads=65527, ldq=2 ** 31 - 1, ldqo=2 ** 31 - 1), {}), ("attn", dict(T=(1 << 24) - 1, S=1), {}),
    ("attn", dict(S=4000000), {})], ids=str)
def test_the_largest_launches(op, change, kv):
    assert launch(op, dataclasses.replace(VALID[op], **change), dataclasses.replace(KV, **kv)) == NOT_INIT


@pytest.mark.parametrize("n_rot,base,scale", [
    (64, math.inf, None), (64, 1e4, h.RopeScale(h.RopeScaling.linear, math.inf)), (64, 1e4, h.RopeScale(h.RopeScaling.ntk, math.inf)),
    (64, 1e4, h.RopeScale(h.RopeScaling.ntk, 1e305)), (64, 1e4, h.RopeScale(h.RopeScaling.yarn, math.inf, 4096.0)),
    (64, 1e4, h.RopeScale(h.RopeScaling.yarn, 2.0, math.inf)), (64, 1e4, h.RopeScale(h.RopeScaling.yarn, 2.0, 4096.0, math.inf)),
    (64, 1e4, h.RopeScale(h.RopeScaling.yarn, 2.0, 4096.0, math.inf, math.inf)),
    (64, 1e4, h.RopeScale(h.RopeScaling.yarn, 2.0, math.nan)), (64, 1e4, h.RopeScale(h.RopeScaling.yarn, 2.0, 4096.0, math.nan))],
    ids=str)
def test_rope_tables_of_infinite_numbers_refused(n_rot, base, scale):
    """A base, a factor, a context or turns that are not finite (or a base that ntk makes so) would give frequencies of zero."""
    with pytest.raises(RuntimeError, match="rope_table"):
        h.rope_table(n_rot, base, scale)


def test_rope_tables_of_large_numbers():
    for scale in (None, h.RopeScale(h.RopeScaling.linear, 1e6), h.RopeScale(h.RopeScaling.ntk, 1e6),
                  h.RopeScale(h.RopeScaling.yarn, 1e6, 1e9, 1e8, 1e-8), h.RopeScale(h.RopeScaling.none, math.inf)):
        turns, m = h.rope_table(128, 1e30, scale)
        assert all(0 < t < 0.16 for t in turns) and turns == sorted(turns, reverse=True) and 1 <= m < 3


@pytest.mark.parametrize("change", [dict(head_stride=248), dict(head_stride=0), dict(page_stride=0), dict(page_stride=248)], ids=str)
def test_rope_refuses_caches_whose_heads_or_pages_overlap(change):
    """They would be written over one another; the attention may read them."""
    assert launch("rope", ROPE, dataclasses.replace(KV, **change)) == ARGS
    assert launch("attn", ATTN, dataclasses.replace(KV, **change)) == NOT_INIT
    q_only = dataclasses.replace(ROPE, k=None, v=None)
    assert launch("rope", q_only, dataclasses.replace(KV, **change)) == NOT_INIT
    one = dataclasses.replace(KV, heads=1, pages=1, **change)
    assert launch("rope", ROPE, one) == NOT_INIT
