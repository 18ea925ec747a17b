"""CPU tests of the operators for requests that share: what the launches refuse before any HIP call (no device exists in
this process), the layout of their argument structs, their workspaces and the native launch calls."""
import ctypes as C
import dataclasses
import math
import os
import subprocess

import pytest

import btf_hip as h

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x100000  # an aligned address; nothing reads it
ARGS, NOT_INIT = h.BTF_ERR_ARGS, h.BTF_ERR_NOT_INIT

KV = h.KvCache(A, A, h.CacheType.f16, 64, 4, 256, 100, 4 * 64 * 256, 64 * 256, 256)
FORK = h.PageFork(F=3, S=8, page=64, ldt=4, pages=100, src=A, dst=A, tokens=A, free=A, n_free=A, table=A, held=A, shared=A, got=A,
                  copy_from=A, copy_to=A, copy_tokens=A)
COPY = h.PageCopy(n=3, source=A, to=A, tokens=A, layers=2, layer_stride=1 << 20)
FREE = h.PageFree(S=300, page=64, ldt=60, pages=100, keep=A, table=A, held=A, shared=A, free=A, n_free=A, ws=A)
TREE = h.CacheMove(S=2, T=8, table=A, ldt=4, first=A, tree=A, leaf=A, kv_len=A, layers=2, layer_stride=1 << 20)
LIST = h.CacheMove(S=2, T=8, table=A, ldt=4, to_table=A, ldt_to=3, first=A, source=A, source0=A)
SHARED = h.SharedAttention(S=2, T=8, heads=20, q=A, ldq=5120, table=A, ldt=4, row0=A, kv_len=A, tree=A, scale=0.0625, out=A,
                           ldo=5120, ws=A, groups=1, group0=A, lead=A, shared=A)
LORA = h.Lora(S=2, T=8, K=512, rank=16, adapters=3, type=h.CacheType.f16, mode=h.GemvMode.kAdd, row0=A, adapter=A, ranks=A,
              scale=A, x=A, ldx=512, ws=A)
GLU = dataclasses.replace(LORA, mode=h.GemvMode.kSwiglu, out=A, ldo=64)
SEG = h.LoraSeg(a=A, b=A, a_stride=16 * 512, b_stride=64 * 16, N=64, y=A, ldy=64)
VALID = {"fork": FORK, "copy": COPY, "free": FREE, "tree": TREE, "list": LIST, "shared": SHARED, "lora": LORA, "glu": GLU}
WITH_KV = ("copy", "tree", "list", "shared")


def launch(op, a, kv=KV, segs=None):
    return {"fork": lambda: h.launch_page_fork_raw(a), "copy": lambda: h.launch_page_copy_raw(a, kv),
            "free": lambda: h.launch_page_free_raw(a), "tree": lambda: h.launch_cache_move_raw(a, kv),
            "list": lambda: h.launch_cache_move_raw(a, kv), "shared": lambda: h.launch_shared_attention_raw(a, kv),
            "lora": lambda: h.launch_lora_raw(a, segs or [SEG], len(segs or [SEG])),
            "glu": lambda: h.launch_lora_raw(a, segs or [SEG, SEG], len(segs or [SEG, SEG]))}[op]()


POINTERS = {"fork": ("src", "dst", "tokens", "free", "n_free", "table", "held", "shared", "got", "copy_from", "copy_to", "copy_tokens"),
            "copy": ("source", "to"), "free": ("keep", "table", "held", "free", "n_free", "ws"), "tree": ("table", "first", "tree", "leaf"),
            "list": ("table", "first", "source", "source0"),
            "shared": ("q", "table", "row0", "kv_len", "out", "ws", "group0", "lead", "shared"), "lora": ("row0", "adapter", "x", "ws"),
            "glu": ("out",)}
REFUSED = [
    *[(op, {n: None}) for op, names in POINTERS.items() for n in names],
    ("fork", dict(F=1025)), ("fork", dict(S=0)), ("fork", dict(page=48)), ("fork", dict(page=0)), ("fork", dict(ldt=0)),
    ("fork", dict(pages=0)), ("fork", dict(pages=1 << 25)),
    ("copy", dict(layers=0)), ("copy", dict(layers=65536)), ("copy", dict(layer_stride=255)), ("copy", dict(layer_stride=0)),
    ("copy", dict(layer_stride=-(1 << 20))), ("copy", dict(layer_stride=(1 << 20) + 4)), ("copy", dict(n=1 << 21)), ("copy", dict(n=2 ** 31 - 1)),
    ("free", dict(page=3)), ("free", dict(ldt=0)), ("free", dict(pages=0)), ("free", dict(pages=1 << 25)), ("free", dict(ws=A + 2)),
    ("free", dict(S=1 << 20, ldt=1 << 9)), ("free", dict(S=2 ** 31 - 1, ldt=2 ** 31 - 1)),
    ("tree", dict(T=-1)), ("tree", dict(source=A)), ("tree", dict(tree=A + 4)), ("tree", dict(ldt=0)), ("tree", dict(layers=0)),
    ("tree", dict(layer_stride=8)), ("tree", dict(S=1 << 18)), ("list", dict(ldt_to=0)), ("list", dict(tree=A)), ("list", dict(S=2 ** 31 - 1)),
    ("shared", dict(heads=18)), ("shared", dict(q=A + 8)), ("shared", dict(ldq=5124)), ("shared", dict(out=A + 4)), ("shared", dict(ldo=5116)),
    ("shared", dict(ldt=0)), ("shared", dict(tree=A + 4)), ("shared", dict(scale=math.nan)), ("shared", dict(groups=3)),
    ("shared", dict(groups=-1)), ("shared", dict(ws=A + 8)), ("shared", dict(T=1 << 24)), ("shared", dict(S=1 << 22)),
    ("shared", dict(S=2 ** 31 - 1)),
    ("lora", dict(K=0)), ("lora", dict(K=500)), ("lora", dict(rank=0)), ("lora", dict(rank=12)), ("lora", dict(rank=264)),
    ("lora", dict(adapters=-1)), ("lora", dict(type=2)), ("lora", dict(mode=0)), ("lora", dict(mode=3)), ("lora", dict(x=A + 8)),
    ("lora", dict(ldx=511)), ("lora", dict(ldx=514)), ("lora", dict(ws=A + 8)), ("lora", dict(T=1 << 24)), ("lora", dict(S=2 ** 31 - 1)),
    ("glu", dict(ldo=63)), ("glu", dict(out=A + 2))]


@pytest.mark.parametrize("op,change", REFUSED, ids=str)
def test_refused_before_any_hip_call(op, change):
    assert launch(op, dataclasses.replace(VALID[op], **change)) == ARGS
    assert h.last_error()


@pytest.mark.parametrize("op", WITH_KV)
@pytest.mark.parametrize("change", [dict(type=2), dict(page=8), dict(page=24), dict(dim=96), dict(heads=0), dict(k=None), dict(v=None),
                                    dict(k=A + 8), dict(pages=0), dict(tok_stride=248), dict(head_stride=4), dict(page_stride=12)], ids=str)
def test_caches_refused(op, change):
    assert launch(op, VALID[op], dataclasses.replace(KV, **change)) == ARGS


@pytest.mark.parametrize("op", ["copy", "tree", "list"])
@pytest.mark.parametrize("change", [dict(head_stride=248), dict(page_stride=0)], ids=str)
def test_caches_that_overlap_are_not_written(op, change):
    assert launch(op, VALID[op], dataclasses.replace(KV, **change)) == ARGS
    assert launch("shared", SHARED, dataclasses.replace(KV, **change)) == NOT_INIT


@pytest.mark.parametrize("segs", [
    [], [SEG] * 4, [dataclasses.replace(SEG, N=0)], [dataclasses.replace(SEG, y=None)], [dataclasses.replace(SEG, ldy=63)],
    [dataclasses.replace(SEG, a=None)], [dataclasses.replace(SEG, b=None)], [dataclasses.replace(SEG, a=A + 8)], [SEG, dataclasses.replace(SEG, b=A + 2)],
    [dataclasses.replace(SEG, a_stride=-8)], [dataclasses.replace(SEG, b_stride=12)], [dataclasses.replace(SEG, y=A + 2)],
    [dataclasses.replace(SEG, N=1 << 24, ldy=1 << 24)] * 2], ids=str)
def test_segments_refused(segs):
    assert h.launch_lora_raw(LORA, segs, len(segs)) == ARGS


def test_more_workgroups_than_a_launch_takes():
    wide = dataclasses.replace(SEG, N=20480, ldy=20480)
    for S, T, code in ((1 << 21, 1 << 21, ARGS), (1, 1 << 22, ARGS), (1, 1 << 21, NOT_INIT), (1 << 18, 1 << 18, NOT_INIT)):
        assert h.launch_lora_raw(dataclasses.replace(LORA, S=S, T=T), [wide], 1) == code


@pytest.mark.parametrize("op,change,code", [
    ("lora", dict(K=1 << 24, ldx=1 << 24), NOT_INIT), ("lora", dict(K=(1 << 24) + 32, ldx=1 << 25), ARGS),
    ("lora", dict(K=2 ** 31 - 32, ldx=2 ** 31 - 4), ARGS), ("list", dict(T=1 << 30), NOT_INIT), ("list", dict(T=(1 << 30) + 1), ARGS),
    ("list", dict(T=2 ** 31 - 1), ARGS)], ids=str)
def test_counts_that_pass_32_bits_in_a_kernel(op, change, code):
    """A loop's next column or entry is beyond the last one by a step."""
    assert launch(op, dataclasses.replace(VALID[op], **change)) == code


@pytest.mark.parametrize("S,T,Ns,glu,code", [
    ((1 << 22) - 1, (1 << 22) - 1, [64], False, NOT_INIT), (1 << 22, 1, [64], False, ARGS), (1, 1 << 22, [64], False, ARGS),
    (1, 1, [1 << 24], False, NOT_INIT), (1, 1, [1 << 23, 1 << 23], False, NOT_INIT), (1, 1, [1 << 23, 1 << 23], True, NOT_INIT),
    (1, 1, [(1 << 24) - 8, 9], False, ARGS), (1, 1, [(1 << 23) + 1] * 2, True, ARGS),
    # n * T, n * (T / 16 + S)
    (1 << 20, 1 << 20, [15 * 1024 - 1], False, NOT_INIT), (1 << 20, 1 << 20, [15 * 1024], False, ARGS),
    (1 << 20, 1 << 20, [14 * 1024 - 1] * 2, True, NOT_INIT), (1 << 20, 1 << 20, [14 * 1024] * 2, True, ARGS),
    (1, (1 << 22) - 16, [1024 * 61, 1024, 1024], False, ARGS), (1, (1 << 22) - 16, [1024 * 60], False, NOT_INIT)], ids=str)
def test_limits_of_the_adapters_launches(S, T, Ns, glu, code):
    """The header's numbers, and one more."""
    segs = [dataclasses.replace(SEG, N=n, ldy=n) for n in Ns]
    a = dataclasses.replace(GLU if glu else LORA, S=S, T=T, ldo=Ns[0])
    assert h.launch_lora_raw(a, segs, len(segs)) == code
    n = (Ns[0] if glu else sum(Ns)) // 1024 + len(Ns)
    fits = max(S, T) < 1 << 22 and sum(Ns) <= 1 << 24 and n * (T if T <= 4 * S else T // 16 + S) < 1 << 24
    assert code == (NOT_INIT if fits else ARGS)


@pytest.mark.parametrize("S,T,heads,kv_heads", [
    (1, 6710521, 20, 4), (1, 6710525, 20, 4), (8388159, 1, 1, 1), (8388160, 1, 1, 1), (1, (1 << 24) - 1, 8, 8), (1, 1 << 24, 1, 1),
    (1 << 20, 1 << 20, 7, 7), (1 << 20, 1 << 20, 8, 8)])
def test_limits_of_the_shared_attention(S, T, heads, kv_heads):
    a = dataclasses.replace(SHARED, S=S, T=T, heads=heads, ldq=heads * 64, ldo=heads * 64)
    kv = dataclasses.replace(KV, heads=kv_heads, dim=64, tok_stride=64, head_stride=64 * 64, page_stride=kv_heads * 64 * 64)
    fits = T < 1 << 24 and 2 * kv_heads * (T * (heads // kv_heads) // 16 + S) < (1 << 24) - 896
    assert launch("shared", a, kv) == (NOT_INIT if fits else ARGS)


@pytest.mark.parametrize("S,heads,dim", [((1 << 17) - 1, 4, 256), (1 << 17, 4, 256), ((1 << 19) - 1, 4, 64), (1 << 19, 4, 64), (1, (1 << 20) - 1, 128),
                                         (1, 1 << 20, 128)])
@pytest.mark.parametrize("op", ["tree", "list"])
def test_limits_of_a_move(op, S, heads, dim):
    kv = dataclasses.replace(KV, heads=heads, dim=dim, tok_stride=dim, head_stride=64 * dim, page_stride=heads * 64 * dim)
    code = NOT_INIT if S * heads * dim < 1 << 27 else ARGS
    assert launch(op, dataclasses.replace(VALID[op], S=S, layers=1), kv) == code


def test_swiglu_segments_refused():
    for segs in ([SEG], [SEG] * 3, [SEG, dataclasses.replace(SEG, N=32)]):
        assert launch("glu", GLU, segs=segs) == ARGS
    assert h.launch_lora_raw(LORA, None, 1) == ARGS


@pytest.mark.parametrize("op", list(VALID))
def test_null_arguments(op):
    assert launch(op, None) == ARGS
    if op in WITH_KV:
        assert launch(op, VALID[op], None) == ARGS


@pytest.mark.parametrize("op,change", [
    *[(op, {}) for op in VALID], ("fork", dict(F=1024)), ("copy", dict(tokens=None)), ("copy", dict(layers=1, layer_stride=0)),
    ("free", dict(shared=None)), ("free", dict(S=3, ws=None)), ("tree", dict(kv_len=None)), ("tree", dict(T=0)), ("list", dict(to_table=None, ldt_to=0)),
    ("shared", dict(groups=0, group0=None, lead=None, shared=None)), ("shared", dict(tree=None)), ("lora", dict(ranks=None, scale=None)),
    ("lora", dict(ldx=1024)), ("lora", dict(adapters=0))], ids=str)
def test_valid_arguments_need_a_device(op, change):
    assert launch(op, dataclasses.replace(VALID[op], **change)) == NOT_INIT


@pytest.mark.parametrize("op,change", [("fork", dict(F=0)), ("fork", dict(F=-1)), ("copy", dict(n=0)), ("free", dict(S=0)), ("tree", dict(S=-2)),
                                       ("shared", dict(S=0)), ("shared", dict(T=0)), ("lora", dict(T=0)), ("lora", dict(S=0))], ids=str)
def test_nothing_to_do(op, change):
    assert launch(op, dataclasses.replace(VALID[op], **change)) == h.BTF_OK


def test_workspaces():
    """None where nothing is launched; those of the largest launch serve the smaller ones."""
    assert h.page_free_ws_bytes(0, 8) == h.page_free_ws_bytes(8, 0) == h.page_free_ws_bytes(1 << 20, 1 << 9) == 0
    assert h.page_free_ws_bytes(200, 40) == 0 < h.page_free_ws_bytes(300, 60) < h.page_free_ws_bytes(301, 4000)
    assert h.shared_attention_ws_bytes(0, 8, 20, KV) == h.shared_attention_ws_bytes(2, 8, 18, KV) == 0
    assert h.lora_ws_bytes(0, 1, 512, 16, 1) == h.lora_ws_bytes(1, 1, 512, 16, 4) == h.lora_ws_bytes(1, 1, 512, 512, 1) == 0
    for dim in (64, 128, 256):
        kv = dataclasses.replace(KV, dim=dim)
        for S, T in ((1, 1), (3, 500), (64, 64), (128, 2000)):
            most = h.shared_attention_ws_bytes(S, T, 20, kv)
            assert all(0 < h.shared_attention_ws_bytes(s, t, 20, kv) <= most for s in (1, (S + 1) // 2, S) for t in (1, (T + 1) // 2, T))
    for S, T, K, rank, n in ((1, 1, 5120, 16, 1), (64, 64, 5120, 64, 3), (3, 4000, 17408, 256, 2)):
        most = h.lora_ws_bytes(S, T, K, rank, n)
        assert all(0 < h.lora_ws_bytes(s, t, k, r, m) <= most for s in (1, S) for t in (1, (T + 1) // 2, T) for k in (32, K // 2, K)
                   for r in (8, rank) for m in (1, n))


STRUCTS = {"btf_page_fork": h._PageFork, "btf_page_copy": h._PageCopy, "btf_page_free": h._PageFree, "btf_cache_move": h._CacheMove,
           "btf_shared_attention": h._SharedAttention, "btf_lora_seg": h._LoraSeg, "btf_lora": h._Lora}


def test_struct_layouts(tmp_path):
    """The ctypes structs have the header's sizes and field offsets."""
    src, want = ["#include <stdio.h>", "#include <stddef.h>", '#include "btf/hip_abi.h"', "int main(void) {"], []
    for name, c in STRUCTS.items():
        src.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(str(C.sizeof(c)))
        for f, _ in c._fields_:
            src.append(f'printf("%zu\\n", offsetof({name}, {f.rstrip("_")}));')
            want.append(str(getattr(c, f).offset))
    (tmp_path / "s.c").write_text("\n".join(src + ["return 0; }"]))
    subprocess.run(["cc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    assert subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split() == want


def test_cpp_wrappers_compile(tmp_path):
    (tmp_path / "s.cpp").write_text('''
#include "btf/kernels.hpp"
using namespace btf::hip;
int main() {
  KvCache kv{};
  try { launch_page_fork(PageFork{.F = 2000}, nullptr); return 1; } catch (const std::runtime_error&) {}
  try { launch_page_copy(PageCopy{.n = 1}, kv, nullptr); return 1; } catch (const std::runtime_error&) {}
  try { launch_page_free(PageFree{.S = 1}, nullptr); return 1; } catch (const std::runtime_error&) {}
  try { launch_cache_move(CacheMove{.S = 1}, kv, nullptr); return 1; } catch (const std::runtime_error&) {}
  try { launch_shared_attention(SharedAttention{.S = 1, .T = 1}, kv, nullptr); return 1; } catch (const std::runtime_error&) {}
  LoraSeg seg{};
  try { launch_lora(Lora{.S = 1, .T = 1}, &seg, 1, nullptr); return 1; } catch (const std::runtime_error&) {}
  return page_free_ws_bytes(300, 60) && lora_ws_bytes(1, 1, 512, 16, 1) && !shared_attention_ws_bytes(1, 1, 1, kv) ? 0 : 1;
}''')
    exe = tmp_path / "s"
    subprocess.run(["g++", "-std=c++20", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.cpp"), h.LIB_PATH, "-o", str(exe),
                    f"-Wl,-rpath,{h.HERE}", "-Wl,--allow-shlib-undefined"], check=True)
    assert subprocess.run([str(exe)]).returncode == 0


LAYOUTS = {"fork": h._fork_layout, "copy": h._copy_layout, "free": h._free_layout, "tree": h._move_layout, "shared": h._shared_layout}


@pytest.mark.skipif(not os.path.exists(h.CALL_PATH), reason="native launch calls not built")
@pytest.mark.parametrize("op", list(LAYOUTS))
def test_native_calls_hand_over_the_same_structs(op):
    """A recorder in place of the launcher: the struct of the native call is that of the ctypes path."""
    a, seen = VALID[op], []
    two = op in WITH_KV
    ptr = [C.POINTER(type(a._c()))] + ([C.POINTER(h._KvCache)] if two else []) + [C.c_void_p]
    f = C.CFUNCTYPE(C.c_int, *ptr)(lambda *v: seen.append([bytes(x[0]) for x in v[:-1]]) or 5)
    a = dataclasses.replace(a, **{n: 1000 + i for i, n in enumerate(a.__dataclass_fields__) if getattr(a, n) == A})
    assert h._call.launch(C.cast(f, C.c_void_p).value, LAYOUTS[op], a, h._kv_layout if two else -1, KV if two else None, None) == 5
    assert seen == [[bytes(a._c())] + ([bytes(KV._c())] if two else [])]


@pytest.mark.skipif(not os.path.exists(h.CALL_PATH), reason="native launch calls not built")
@pytest.mark.parametrize("n", [1, 2, 3])
@pytest.mark.parametrize("kind", [list, tuple])
def test_native_calls_hand_over_lists(n, kind):
    seen = []

    def record(a, segs, count, stream):
        seen.append((bytes(a[0]), [bytes(segs[i]) for i in range(count)], stream))
        return 7
    f = C.CFUNCTYPE(C.c_int, C.POINTER(h._Lora), C.POINTER(h._LoraSeg), C.c_int, C.c_void_p)(record)
    at = C.cast(f, C.c_void_p).value
    segs = kind(dataclasses.replace(SEG, N=3 + i, a=None if i else A, y=4096 * i + 4096) for i in range(n))
    call = lambda a, s, lay=h._lora_layout: h._call.launch_list(at, lay, a, h._lora_seg_layout, s, 9)  # noqa: E731
    assert call(LORA, segs) == 7
    assert seen == [(bytes(LORA._c()), [bytes(s._c()) for s in segs], 9)]
    for other in ((LORA, []), (LORA, [SEG] * 4), (LORA, None), (LORA, [SEG, None]), (LORA, [LORA]), (SEG, [SEG]), (None, [SEG]),
                  (dataclasses.replace(LORA, K=3.5), [SEG]), (LORA, iter([SEG]))):
        assert call(*other) is NotImplemented
    assert call(LORA, segs, 99) is NotImplemented
    with pytest.raises(TypeError):
        h._call.launch_list(at, h._lora_layout, LORA)
    assert len(seen) == 1


def test_errors_raise_the_library_message():
    for f, args, text in ((h.launch_page_fork, (dataclasses.replace(FORK, F=2000),), "1024 forks"), (h.launch_page_copy, (COPY, None), "null cache"),
                          (h.launch_page_free, (dataclasses.replace(FREE, ldt=0),), "page_free"),
                          (h.launch_cache_move, (dataclasses.replace(TREE, source=A), KV), "either tree or source"),
                          (h.launch_shared_attention, (dataclasses.replace(SHARED, groups=9), KV), "groups must be"),
                          (h.launch_lora, (LORA, []), "1..3 segments"), (h.launch_lora, (dataclasses.replace(LORA, rank=9), [SEG]), "rank must be"),
                          (h.launch_page_fork, (None,), "null arguments"), (h.launch_lora, (None, [SEG]), "null arguments")):
        with pytest.raises(RuntimeError, match=text):
            f(*args)
