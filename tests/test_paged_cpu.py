"""The paged-cache operators' host side: what they refuse (before any device
work), their workspace sizes, the rotary plan against its formulas, and the
layout of their structs."""
import ctypes as C
import math
import os
import subprocess

import pytest

from mlxcat_b200 import _abi as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
L = A.lib()
P = 1 << 20   # a 16-byte aligned address that is never read: every call below is refused


def kv(**change):
    c = dict(k=P, v=2 * P, page_table=3 * P, page_stride=8 * 16 * 128, head_stride=16 * 128, token_stride=128, dtype=A.F16, n_pages=10,
             page_size=16, n_kv_heads=8, head_dim=128, rows=4, max_pages=6)
    c.update(change)
    return A.PagedKVC(*[c[n] for n, _ in A.PagedKVC._fields_])


BAD_KV = [dict(k=None), dict(v=None), dict(page_table=None), dict(dtype=A.F32), dict(dtype=7), dict(head_dim=96), dict(head_dim=0),
          dict(page_size=4), dict(page_size=24), dict(page_size=0), dict(page_size=131072), dict(n_pages=0), dict(n_kv_heads=0),
          dict(rows=0), dict(max_pages=-1), dict(k=P + 2), dict(v=2 * P + 8), dict(token_stride=64), dict(token_stride=132),
          dict(head_stride=15 * 128), dict(page_stride=0), dict(page_stride=7 * 16 * 128), dict(token_stride=-128)]


def append(c, **change):
    a = dict(q=4 * P, k=5 * P, v=6 * P, dt=A.F16, qs=32 * 128, ks=1024, vs=1024, M=3, heads=32, qn=None, kn=None, eps=1e-6, trow=7 * P, tpos=8 * P,
             q_out=9 * P, rope=None)
    a.update(change)
    return L.mlxcat_op_rope_append(c and C.byref(c), a["rope"] and C.byref(a["rope"]), a["q"], a["k"], a["v"], a["dt"], a["qs"], a["ks"], a["vs"],
                                   a["M"], a["heads"], a["qn"], a["kn"], a["eps"], a["trow"], a["tpos"], a["q_out"], None, None)


def paged(c, prefix=None, **change):
    a = dict(q=4 * P, M=4, qg=1, heads=32, scale=0.0, trow=5 * P, tpos=6 * P, out=7 * P, ws=8 * P, size=1 << 30)
    a.update(change)
    rest = (a["q"], a["M"], a["qg"], a["heads"], a["scale"], a["trow"], a["tpos"], a["out"], a["ws"], a["size"], None, None)
    if prefix is None:
        return L.mlxcat_op_paged_attention(c and C.byref(c), *rest)
    return L.mlxcat_op_shared_prefix_attention(c and C.byref(c), prefix, *rest)


def packed(**change):
    a = dict(q=4 * P, k=5 * P, v=6 * P, dt=A.BF16, qs=4096, ks=1024, vs=1024, Tq=10, Tk=12, cu_q=7 * P, cu_k=8 * P, n=2, causal=1, heads=32, kv=8,
             D=128, scale=0.0, out=9 * P)
    a.update(change)
    return L.mlxcat_op_packed_attention(a["q"], a["k"], a["v"], a["dt"], a["qs"], a["ks"], a["vs"], a["Tq"], a["Tk"], a["cu_q"], a["cu_k"], a["n"],
                                        a["causal"], a["heads"], a["kv"], a["D"], a["scale"], a["out"], None, None)


@pytest.mark.parametrize("change", BAD_KV, ids=str)
def test_cache_descriptions_refused(change):
    assert append(kv(**change)) == A.E_INVALID
    assert L.mlxcat_op_last_error()
    assert paged(kv(**change)) == A.E_INVALID
    assert paged(kv(**change), prefix=0) == A.E_INVALID


def test_null_cache_refused():
    assert append(None) == A.E_INVALID and paged(None) == A.E_INVALID and paged(None, 16) == A.E_INVALID


@pytest.mark.parametrize("change", [
    dict(k=None), dict(v=None), dict(trow=None), dict(tpos=None), dict(q=None), dict(q_out=None), dict(dt=5), dict(M=0), dict(M=-1),
    dict(heads=0), dict(eps=-1.0), dict(eps=float("nan")), dict(q=4 * P + 4), dict(qs=4100), dict(qs=4088), dict(ks=1016), dict(vs=0),
    dict(q_out=9 * P + 2), dict(q_out=4 * P), dict(q_out=5 * P + 16), dict(rope=A.RopeC(130, 0, 1.0)), dict(rope=A.RopeC(7, 0, 1.0)),
    dict(rope=A.RopeC(64, 2, 1.0)), dict(rope=A.RopeC(0, 0, 1.0))], ids=str)
def test_append_refusals(change):
    assert append(kv(), **change) == A.E_INVALID


@pytest.mark.parametrize("change", [
    dict(q=None), dict(trow=None), dict(tpos=None), dict(out=None), dict(ws=None), dict(M=0), dict(qg=0), dict(heads=0), dict(heads=12),
    dict(heads=8 * 65), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(q=4 * P + 8), dict(out=7 * P + 2),
    dict(ws=8 * P + 4), dict(size=16), dict(M=1 << 28)], ids=str)
def test_paged_attention_refusals(change):
    assert paged(kv(), **change) == A.E_INVALID
    assert paged(kv(), prefix=16, **change) == A.E_INVALID


@pytest.mark.parametrize("prefix", [-16, 8, 17, 7 * 16])
def test_prefix_refusals(prefix):
    assert paged(kv(), prefix=prefix) == A.E_INVALID   # whole pages of 16, six per row at most


@pytest.mark.parametrize("change", [
    dict(q=None), dict(k=None), dict(v=None), dict(cu_q=None), dict(cu_k=None), dict(out=None), dict(dt=A.F32), dict(Tq=0), dict(Tk=0),
    dict(n=0), dict(heads=12), dict(heads=0), dict(kv=0), dict(D=96), dict(heads=8 * 65), dict(scale=-0.5), dict(qs=4088), dict(ks=1020),
    dict(vs=512), dict(k=5 * P + 8), dict(out=9 * P + 4)], ids=str)
def test_packed_attention_refusals(change):
    assert packed(**change) == A.E_INVALID


def test_workspaces():
    ws, pre = L.mlxcat_op_paged_attention_workspace, L.mlxcat_op_shared_prefix_attention_workspace
    assert ws(0, 1, 8, 2, 64) == 0 and ws(4, 1, 8, 3, 64) == 0 and ws(4, 1, 8, 2, 96) == 0
    assert pre(4, 1, 8, 2, 64, -1) == 0
    assert pre(4, 1, 8, 2, 64, 0) == ws(4, 1, 8, 2, 64) > 0
    # a prefix adds the partials of every query row
    assert pre(64, 1, 32, 8, 128, 8192) >= ws(64, 1, 32, 8, 128) + 64 * 32 * 128 * 4
    assert ws(5, 9, 8, 2, 64) == ws(5, 5, 8, 2, 64)   # a group is never longer than the batch


# ---- rotary plan -----------------------------------------------------------------
def plan(rd, layout=A.ROPE_HALF, theta=10000.0, scaling=None):
    r = A.RopeC()
    A.check(L.mlxcat_rope_init(C.byref(r), rd, layout, theta, scaling and C.byref(scaling)))
    return r


def scaling(kind, orig=8192, factor=8.0, low=1.0, high=4.0, fast=32.0, slow=1.0, mscale=0.0):
    return A.RopeScalingC(kind, orig, factor, low, high, fast, slow, mscale)


@pytest.mark.parametrize("rd,theta", [(2, 10000.0), (20, 500000.0), (64, 1e6), (128, 500000.0), (256, 10000.0)])
def test_rope_plan_frequencies(rd, theta):
    r = plan(rd, A.ROPE_INTERLEAVED, theta)
    assert (r.rotary_dim, r.layout, r.mscale) == (rd, A.ROPE_INTERLEAVED, 1.0)
    for i in range(rd // 2):
        f = theta ** (-2.0 * i / rd)
        assert r.turns[i] * 2 * math.pi == pytest.approx(f, rel=1e-14)
    lin = plan(rd, theta=theta, scaling=scaling(A.ROPE_SCALE_LINEAR, factor=4.0))
    for i in range(rd // 2):
        assert lin.turns[i] == pytest.approx(r.turns[i] / 4.0, rel=1e-14)


def test_rope_plan_banded_scaling():
    r, s = plan(128, theta=500000.0), plan(128, theta=500000.0, scaling=scaling(A.ROPE_SCALE_LLAMA3))
    kinds = set()
    for i in range(64):
        n = 8192 * r.turns[i]            # turns within the original context
        if n >= 4.0:
            want, kind = r.turns[i], "kept"
        elif n <= 1.0:
            want, kind = r.turns[i] / 8.0, "divided"
        else:
            t = (n - 1.0) / 3.0
            want, kind = (1 - t) * r.turns[i] / 8.0 + t * r.turns[i], "between"
        kinds.add(kind)
        assert s.turns[i] == pytest.approx(want, rel=1e-13)
    assert kinds == {"kept", "divided", "between"}


def test_rope_plan_yarn():
    r, s = plan(128, theta=1e6), plan(128, theta=1e6, scaling=scaling(A.ROPE_SCALE_YARN, orig=32768))
    assert s.mscale == pytest.approx(0.1 * math.log(8.0) + 1.0, rel=1e-6)
    assert plan(128, theta=1e6, scaling=scaling(A.ROPE_SCALE_YARN, mscale=1.25)).mscale == 1.25
    ratio = [s.turns[i] / r.turns[i] for i in range(64)]
    assert ratio[0] == pytest.approx(1.0) and ratio[-1] == pytest.approx(1 / 8.0)
    assert all(a >= b - 1e-12 for a, b in zip(ratio, ratio[1:]))
    for i in range(64):   # the ends of the ramp: 32 turns and one turn within 32768 positions
        n = 32768 * r.turns[i]
        if n > 32.0 * 1e6 ** (2 / 128):
            assert ratio[i] == pytest.approx(1.0)
        if n < 1.0 / 1e6 ** (2 / 128):
            assert ratio[i] == pytest.approx(1 / 8.0)


@pytest.mark.parametrize("args", [
    (0, 0, 1e4, None), (3, 0, 1e4, None), (258, 0, 1e4, None), (64, 2, 1e4, None), (64, 0, 1.0, None), (64, 0, float("nan"), None),
    (64, 0, float("inf"), None), (64, 0, 1e4, scaling(9)), (64, 0, 1e4, scaling(1, factor=0.5)), (64, 0, 1e4, scaling(1, factor=float("nan"))),
    (64, 0, 1e4, scaling(2, orig=0)), (64, 0, 1e4, scaling(2, low=4.0)), (64, 0, 1e4, scaling(3, slow=0.0)), (64, 0, 1e4, scaling(3, mscale=-1.0))],
    ids=str)
def test_rope_plan_refusals(args):
    r = A.RopeC()
    assert L.mlxcat_rope_init(C.byref(r), args[0], args[1], args[2], args[3] and C.byref(args[3])) == A.E_INVALID
    assert L.mlxcat_rope_init(None, 64, 0, 1e4, None) == A.E_INVALID


def test_structs_match_the_header(tmp_path):
    structs = {"mlxcat_paged_kv": A.PagedKVC, "mlxcat_rope_scaling": A.RopeScalingC, "mlxcat_rope": A.RopeC}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "mlxcat_cuda.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    for ln in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        cname, key, val = ln.split()
        assert int(val) == (C.sizeof(structs[cname]) if key == "size" else getattr(structs[cname], key).offset), ln


@pytest.mark.parametrize("change", [
    dict(page_stride=1 << 38, n_pages=(1 << 26) + 1), dict(page_stride=1 << 38, n_pages=2 ** 31 - 1),
    dict(page_stride=1 << 37, n_pages=(1 << 25) + 1, head_stride=1 << 33),
    dict(head_stride=1 << 38, n_kv_heads=1 << 26, page_stride=2048, page_size=16)], ids=str)
def test_cache_extent_past_64_bits_refused(change):
    """Strides times counts past 2^63 elements: the sum that finds them too large must not wrap."""
    assert append(kv(**change)) == A.E_INVALID
    assert paged(kv(**change), heads=change.get("n_kv_heads", 8)) == A.E_INVALID
