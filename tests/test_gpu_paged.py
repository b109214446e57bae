"""The paged-cache operators on the GPU against their formulas in 64 bits.

Tolerances, per element, from the arithmetic (u = eps / 2 of the output type):
* append: the result rounded once (u |y|) and a few fp32 operations before it:
  the sum of D squares moves the norm by at most D 2^-25 relatively, the angle's
  fraction and sin / cos by 2^-22, the rotation's products by 3 * 2^-24; all of it
  stays below 2^-16 (|a| + |b|) for D = 128.
* attention: every weight is rounded once to the type (u, in the sum of the
  weights as well), its score carries the fp32 dot product's error e = 2 D 2^-24
  |q| |k| scale (2: the tensor cores truncate) and 2^-21 of the exponential, and
  the result is rounded once.  With A = sum w |v|, the error is at most
  u |y| + 2 A (u + e + 2^-21).  fp16 weights below 2^-14 of the largest have an
  absolute error of 2^-25 each instead: n 2^-25 max|v| / sum 2^(z - max).
"""
import ctypes as C
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from mlxcat_b200 import _abi as A  # noqa: E402

L = A.lib()
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODE = {"f16": A.F16, "bf16": A.BF16, "f32": A.F32}
NAN = float("nan")


def ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def half_step(dt):
    return torch.finfo(DT[dt]).eps / 2


class Paged:
    """A cache of NaN pages, [page][head][token][d] or [page][token][head][d]."""

    def __init__(self, hk, d, ps, n_pages, dt, table, nhd=False, fill=NAN):
        shape = (n_pages, ps, hk, d) if nhd else (n_pages, hk, ps, d)
        self.k = torch.full(shape, fill, dtype=DT[dt], device="cuda")
        self.v = torch.full(shape, fill, dtype=DT[dt], device="cuda")
        self.table = table if torch.is_tensor(table) else ints(table)
        self.ps, self.hk, self.d, self.nhd = ps, hk, d, nhd
        strides = (ps * hk * d, d, hk * d) if nhd else (ps * hk * d, ps * d, d)
        self.c = A.PagedKVC(self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(), *strides, CODE[dt], n_pages, ps, hk, d,
                            *self.table.shape)

    def view(self, x):
        return x.transpose(1, 2) if self.nhd else x          # [page][head][token][d]

    def put(self, row, k, v, start=0):
        """k, v [n, hk, d] at positions start.. of a row."""
        pos = torch.arange(start, start + k.shape[0], device="cuda")
        page = self.table[row, pos // self.ps].long()
        self.view(self.k)[page, :, pos % self.ps] = k
        self.view(self.v)[page, :, pos % self.ps] = v

    def row(self, row, n):
        pos = torch.arange(n, device="cuda")
        page = self.table[row, pos // self.ps].long()
        return self.view(self.k)[page, :, pos % self.ps], self.view(self.v)[page, :, pos % self.ps]


def tables(lens, ps, spare=2, seed=0, lead=()):
    """Shuffled page tables; entries past a row's end are -1.  lead: pages every row starts with."""
    need = [max(0, math.ceil((n - len(lead) * ps) / ps)) for n in lens]
    ids = torch.randperm(sum(need) + spare + len(lead), generator=torch.Generator().manual_seed(seed))
    lead_ids, ids = ids[:len(lead)], ids[len(lead):]
    t = torch.full((len(lens), len(lead) + max(1, max(need))), -1, dtype=torch.int32)
    t[:, :len(lead)] = lead_ids
    at = 0
    for r, n in enumerate(need):
        t[r, len(lead):len(lead) + n] = ids[at:at + n]
        at += n
    return t.cuda(), sum(need) + spare + len(lead)


def attend64(q, k, v, limit, scale=None):
    """q [n, h, d], k, v [keys, hk, d]; query i sees keys 0..limit[i].  Returns the result and the
    tolerance's parts in 64 bits: A = sum w |v|, and the sum of 2^(z - max)."""
    n, h, d = q.shape
    g = h // k.shape[1]
    if k.shape[0] == 0:
        z = torch.zeros((n, h, d), dtype=torch.float64, device="cuda")
        return z, z, torch.ones((n, h, 1), dtype=torch.float64, device="cuda")
    kk, vv = k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    s = torch.einsum("nhd,khd->nhk", q.double(), kk) * (scale or 1 / math.sqrt(d))
    seen = (torch.arange(k.shape[0], device="cuda")[None, :] <= limit[:, None])[:, None, :]
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True).clamp(min=-1e300)
    e = torch.exp(s - top)
    tot = e.sum(-1, keepdim=True)
    w = e / tot.clamp(min=1e-300)
    return torch.einsum("nhk,khd->nhd", w, vv), torch.einsum("nhk,khd->nhd", w, vv.abs()), tot.clamp(min=1.0)


def check(got, ref, dt, q, k, v, scale=None):
    y, a, tot = ref
    d = q.shape[-1]
    assert torch.isfinite(got.double()).all()
    e = 0.0 if k.shape[0] == 0 else (2 * d * 2.0 ** -24 * q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max() *
                                     (scale or 1 / math.sqrt(d))).item()
    u = half_step(dt)
    tol = u * y.abs() + 2 * a * (u + e + 2.0 ** -21) + 1e-7
    if dt == "f16" and k.shape[0]:
        tol = tol + k.shape[0] * 2.0 ** -25 * v.double().abs().max() / tot
    worst = ((got.double() - y).abs() / tol).max().item()
    assert worst <= 1.0, worst


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(shape, g, dt, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(DT[dt])


# ------------------------------------------------------------------------------------------------- append
def rope_plan(rd, layout, theta=500000.0, kind=0):
    r, s = A.RopeC(), A.RopeScalingC(kind, 8192, 8.0, 1.0, 4.0, 32.0, 1.0, 0.0)
    A.check(L.mlxcat_rope_init(C.byref(r), rd, layout, theta, C.byref(s)))
    return r


def append(cache, plan, q, k, v, src, trow, tpos, q_out, qn=None, kn=None, eps=1e-6, err=None, heads=None):
    return L.mlxcat_op_rope_append(C.byref(cache.c), plan and C.byref(plan), ptr(q), ptr(k), ptr(v), CODE[src], q.stride(0) if q is not None else 0,
                                   k.stride(0), v.stride(0), k.shape[0], heads if heads is not None else (q.shape[1] // cache.d if q is not None else 0),
                                   ptr(qn), ptr(kn), eps, ptr(trow), ptr(tpos), ptr(q_out), ptr(err), stream())


def turned64(x, pos, plan, w, eps=1e-6):
    """x [m, heads, d] -> normalised and rotated in 64 bits, and |a| + |b| of each pair."""
    x = x.double()
    if w is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = x.abs()
    if plan is not None:
        rd = plan.rotary_dim
        turns = torch.tensor(plan.turns[:rd // 2], dtype=torch.float64, device="cuda")
        ang = (pos.double()[:, None] * turns)[:, None, :] * (2 * math.pi)
        z = torch.arange(rd // 2, device="cuda")
        ia, ib = (z, z + rd // 2) if plan.layout == A.ROPE_HALF else (2 * z, 2 * z + 1)
        a, b = x[..., ia], x[..., ib]
        x = x.clone()
        x[..., ia] = plan.mscale * (a * ang.cos() - b * ang.sin())
        x[..., ib] = plan.mscale * (b * ang.cos() + a * ang.sin())
        size = size.clone()
        size[..., ia] = size[..., ib] = plan.mscale * (a.abs() + b.abs())
    return x, size


def near(got, y, size, dt):
    tol = half_step(dt) * y.abs() + 2.0 ** -16 * size + 1e-7
    worst = ((got.double() - y).abs() / tol).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("d,h,hk,dt,src,rd,layout,kind,norm,ps,nhd", [
    (64, 8, 2, "f16", "f16", 64, 0, 0, False, 16, False),
    (128, 32, 8, "f16", "f32", 128, 0, 2, False, 64, True),
    (128, 32, 8, "bf16", "bf16", 128, 1, 3, True, 256, False),
    (128, 10, 2, "bf16", "f32", 32, 0, 1, True, 8, False),
    (64, 3, 1, "f16", "bf16", 20, 0, 0, True, 32, True),      # half of the rotary width no multiple of 8
    (64, 5, 5, "bf16", "f16", 6, 1, 0, False, 8, False),
    (128, 1, 1, "f16", "f16", 2, 0, 0, False, 128, False),
    (128, 4, 4, "f16", "f32", 0, 0, 0, True, 16, False),      # no rotation
])
@pytest.mark.parametrize("t", [1, 37])
def test_append(d, h, hk, dt, src, rd, layout, kind, norm, ps, nhd, t):
    g = gen(d + h + t)
    past = [0, 5, 130]
    table, n_pages = tables([p + t for p in past], ps)
    cache = Paged(hk, d, ps, n_pages, dt, table, nhd, fill=7.0)
    m = 3 * t
    x = rnd((m, (h + 2 * hk) * d + 8), g, src, 2.0)           # a fused projection with padding behind it
    q, k, v = x[:, :h * d], x[:, h * d:(h + hk) * d], x[:, (h + hk) * d:(h + 2 * hk) * d]
    trow = ints([r for r in range(3) for _ in range(t)])
    tpos = ints([past[r] + j for r in range(3) for j in range(t)])
    trow[1 if t > 1 else 0] = -1                              # a padding token
    plan = rope_plan(rd, layout, kind=kind) if rd else None
    qn = kn = None
    if norm:
        qn, kn = 1 + 0.3 * torch.randn(d, device="cuda", generator=g), 1 + 0.3 * torch.randn(d, device="cuda", generator=g)
    q_out = torch.full((m, h, d), 9.0, dtype=DT[dt], device="cuda")
    err = ints([0])
    A.check(append(cache, plan, q, k, v, src, trow, tpos, q_out, qn, kn, err=err))
    torch.cuda.synchronize()
    assert err.item() == 0
    on = trow >= 0
    y, size = turned64(q.reshape(m, h, d), tpos, plan, qn)
    near(q_out[on], y[on], size[on], dt)
    assert (q_out[~on] == 9.0).all()
    y, size = turned64(k.reshape(m, hk, d), tpos, plan, kn)
    page, off = table[trow.long().clamp(min=0), (tpos // ps).long()].long()[on], (tpos % ps).long()[on]
    near(cache.view(cache.k)[page, :, off], y[on], size[on], dt)
    assert torch.equal(cache.view(cache.v)[page, :, off], v.reshape(m, hk, d)[on].to(DT[dt]))
    for c in (cache.k, cache.v):                              # nothing else was written
        w = cache.view(c).clone()
        w[page, :, off] = 7.0
        assert (w == 7.0).all()


def test_append_far_positions():
    """Positions up to 2^30: the angle keeps its fraction."""
    ps, d = 65536, 128
    pos = [0, 1, 65535, 65536, 10 ** 6 + 1, 2 ** 24 + 3, 2 ** 30 - 1]
    pages = sorted({p // ps for p in pos})
    table = torch.full((1, 2 ** 30 // ps), -1, dtype=torch.int32)
    for i, p in enumerate(pages):
        table[0, p] = i
    cache = Paged(1, d, ps, len(pages), "f16", table.cuda(), fill=0.0)
    g = gen(3)
    q, k = rnd((len(pos), 2 * d), g, "f32"), rnd((len(pos), d), g, "f32")
    q_out = torch.zeros((len(pos), 2, d), dtype=torch.float16, device="cuda")
    plan = rope_plan(d, A.ROPE_HALF, 10000.0)
    A.check(append(cache, plan, q, k, k, "f32", ints([0] * len(pos)), ints(pos), q_out))
    y, size = turned64(q.view(-1, 2, d), torch.tensor(pos, device="cuda"), plan, None)
    near(q_out, y, size, "f16")


def test_append_out_of_range():
    d, ps = 64, 16
    table = ints([[0, 1], [2, 99]])
    for trow, tpos, bad in [(0, 32, True), (0, -1, True), (2, 0, True), (1, 16, True), (1, 15, False)]:
        cache = Paged(2, d, ps, 3, "f16", table, fill=5.0)
        x = torch.ones((1, 2 * d), dtype=torch.float16, device="cuda")
        q_out = torch.zeros((1, 2, d), dtype=torch.float16, device="cuda")
        err = ints([0])
        A.check(append(cache, None, x, x, x, "f16", ints([trow]), ints([tpos]), q_out, err=err))
        assert (err.item() != 0) == bad
        assert bool((cache.k == 5.0).all()) == bad
        assert (q_out == 1).all()
        A.check(append(cache, None, x, x, x, "f16", ints([trow]), ints([tpos]), q_out))   # err may be NULL


def test_append_keys_only():
    cache = Paged(2, 64, 16, 1, "bf16", ints([[0]]), fill=0.0)
    x = rnd((3, 128), gen(1), "bf16")
    A.check(append(cache, None, None, x, x, "bf16", ints([0, 0, 0]), ints([0, 5, 15]), None))
    k, v = cache.row(0, 16)
    assert torch.equal(k[[0, 5, 15]].reshape(3, 128), x) and torch.equal(v, k)


# ---------------------------------------------------------------------------------------- paged attention
def fill_rows(cache, lens, g, dt, shared=0):
    for r, n in enumerate(lens):
        a = shared if r else 0
        if n > a:
            cache.put(r, rnd((n - a, cache.hk, cache.d), g, dt), rnd((n - a, cache.hk, cache.d), g, dt), a)


def paged(cache, q, qg, trow, tpos, out, prefix=None, scale=0.0, err=None, ws=None, st=None):
    m, h, d = q.shape
    size = (L.mlxcat_op_paged_attention_workspace(m, qg, h, cache.hk, d) if prefix is None else
            L.mlxcat_op_shared_prefix_attention_workspace(m, qg, h, cache.hk, d, prefix))
    ws = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda") if ws is None else ws
    rest = (ptr(q), m, qg, h, scale, ptr(trow), ptr(tpos), ptr(out), ptr(ws), size, ptr(err), st or stream())
    if prefix is None:
        return L.mlxcat_op_paged_attention(C.byref(cache.c), *rest)
    return L.mlxcat_op_shared_prefix_attention(C.byref(cache.c), prefix, *rest)


def check_rows(cache, q, qg, trow, tpos, out, dt, scale=None):
    for i in range(q.shape[0]):
        r, p = trow[i].item(), tpos[i].item()
        if r < 0:
            assert (out[i] == 9.0).all()
            continue
        if p < 0:
            assert (out[i] == 0).all()
            continue
        k, v = cache.row(r, p + 1)
        check(out[i:i + 1], attend64(q[i:i + 1], k, v, tpos[i:i + 1].long(), scale), dt, q[i:i + 1], k, v, scale)


LENS = [1, 2, 63, 64, 65, 127, 300, 1027]


@pytest.mark.parametrize("h,hk,d,dt,qg,ps,nhd", [
    (8, 2, 64, "f16", 1, 16, False), (32, 8, 128, "f16", 5, 64, False), (32, 8, 128, "bf16", 1, 256, True), (64, 8, 128, "bf16", 4, 8, False),
    (10, 2, 128, "f16", 3, 32, True), (4, 4, 64, "bf16", 1, 8, False), (40, 1, 64, "f16", 2, 128, False), (32, 4, 128, "bf16", 8, 16, False),
    (3, 1, 128, "f16", 1, 1024, False), (12, 4, 64, "f16", 7, 32, False)])
def test_paged_attention(h, hk, d, dt, qg, ps, nhd):
    g = gen(h + d + qg)
    lens = [n + qg - 1 for n in LENS]
    table, n_pages = tables(lens, ps)
    cache = Paged(hk, d, ps, n_pages, dt, table, nhd)       # what no row holds is NaN
    fill_rows(cache, lens, g, dt)
    trow = ints([r for r in range(len(lens)) for _ in range(qg)])
    tpos = ints([n - qg + j for n in lens for j in range(qg)])
    q = rnd((len(trow), h, d), g, dt)
    out = torch.full_like(q, 9.0)
    err = ints([0])
    A.check(paged(cache, q, qg, trow, tpos, out, err=err))
    torch.cuda.synchronize()
    assert err.item() == 0
    check_rows(cache, q, qg, trow, tpos, out, dt)
    again = torch.full_like(q, 9.0)
    A.check(paged(cache, q, qg, trow, tpos, again))
    assert torch.equal(out, again)                           # no order of arrival in the result


def test_paged_attention_many_splits_and_many_rows():
    for lens, h, hk in (([20000], 8, 1), ([5] * 300 + [900], 8, 2)):
        g = gen(len(lens))
        table, n_pages = tables(lens, 16)
        cache = Paged(hk, 128, 16, n_pages, "f16", table)
        fill_rows(cache, lens, g, "f16")
        trow, tpos = ints(list(range(len(lens)))), ints([n - 1 for n in lens])
        q = rnd((len(lens), h, 128), g, "f16")
        out = torch.full_like(q, 9.0)
        A.check(paged(cache, q, 1, trow, tpos, out))
        check_rows(cache, q, 1, trow, tpos, out, "f16")


@pytest.mark.parametrize("prefix", [None, 32])
def test_paged_attention_empty_and_padding(prefix):
    """Rows without keys give zeros, padding stays as it was, groups end in padding, a short last group."""
    qg, ps, dt, h, hk, d = 3, 16, "bf16", 8, 2, 64
    lens = [40, 0, 50, 33, 36]
    table, n_pages = tables(lens, ps, lead=(0, 0) if prefix else ())
    cache = Paged(hk, d, ps, n_pages, dt, table)
    g = gen(5)
    fill_rows(cache, lens, g, dt, shared=prefix or 0)
    if prefix:
        table[1] = table[0]
    trow = ints([0, 0, 0, 1, 1, 1, 2, 2, -1, -1, -1, -1, 3, 3, 3, 4])
    tpos = ints([37, 38, 39, -1, -1, -1, 48, 49, 0, 7, 8, 9, -1, 0, 32, 35])
    q = rnd((len(trow), h, d), g, dt)
    out = torch.full_like(q, 9.0)
    A.check(paged(cache, q, qg, trow, tpos, out, prefix))
    check_rows(cache, q, qg, trow, tpos, out, dt)


@pytest.mark.parametrize("prefix", [None, 16])
def test_paged_attention_out_of_range(prefix):
    """Rows, positions and pages outside the cache set the flag; nothing is read there."""
    ps, h, hk, d = 16, 8, 2, 64
    for trow, tpos, table in ([5, 3, ints([[0, 1]])], [0, 32, ints([[0, 1]])], [0, 0x7fffffff, ints([[0, 1]])], [0, 20, ints([[0, 44]])],
                              [0, 20, ints([[-7, 1]])]):
        cache = Paged(hk, d, ps, 2, "f16", table, fill=0.5)
        q, err = rnd((1, h, d), gen(1), "f16"), ints([0])
        out = torch.full_like(q, 9.0)
        A.check(paged(cache, q, 1, ints([trow]), ints([tpos]), out, prefix, err=err))
        torch.cuda.synchronize()
        assert err.item() != 0 and torch.isfinite(out).all()
        A.check(paged(cache, q, 1, ints([trow]), ints([tpos]), out, prefix))


def test_paged_attention_scale_and_large_scores():
    """A scale of its own; scores far apart, so that the running maximum moves often."""
    lens, g = [700, 90], gen(8)
    table, n_pages = tables(lens, 32)
    cache = Paged(2, 64, 32, n_pages, "bf16", table)
    fill_rows(cache, lens, g, "bf16")
    for r, n in enumerate(lens):
        k, v = cache.row(r, n)
        cache.put(r, k * torch.linspace(0.1, 6.0, n, device="cuda").to(k.dtype)[:, None, None], v)
    trow, tpos = ints([0, 1]), ints([699, 89])
    q = rnd((2, 8, 64), g, "bf16", 3.0)
    for prefix, copies in ((None, 1), (64, 1), (64, 5000)):   # per row, and once for all
        if prefix:
            table[1, :2] = table[0, :2]
        qq, rr, pp = q.repeat(copies, 1, 1), trow.repeat(copies), tpos.repeat(copies)
        out = torch.full_like(qq, 9.0)
        A.check(paged(cache, qq, 1, rr, pp, out, prefix, scale=0.3))
        check_rows(cache, q, 1, trow, tpos, out[-2:], "bf16", 0.3)
        check_rows(cache, q, 1, trow, tpos, out[copies // 2 * 2:][:2], "bf16", 0.3)


def test_paged_attention_far_pages():
    """Pages whose elements lie past 2^32."""
    ps, hk, d = 256, 2, 128
    n_pages = 2 ** 32 // (ps * hk * d) + 3
    k, v = (torch.empty((n_pages, hk, ps, d), dtype=torch.float16, device="cuda") for _ in range(2))
    table = ints([[n_pages - 1, 0, n_pages - 2]])
    cache = Paged(hk, d, ps, 1, "f16", table)
    cache.k, cache.v = k, v
    cache.c.k, cache.c.v, cache.c.n_pages = k.data_ptr(), v.data_ptr(), n_pages
    g = gen(2)
    x = rnd((700, 4 * hk * d), g, "f32")
    q_out = torch.zeros((700, 2 * hk, d), dtype=torch.float16, device="cuda")
    A.check(append(cache, None, x[:, :2 * hk * d], x[:, 2 * hk * d:3 * hk * d], x[:, 3 * hk * d:], "f32", ints([0] * 700),
                   ints(list(range(700))), q_out))
    kk, vv = cache.row(0, 700)
    assert torch.equal(kk.reshape(700, -1), x[:, 2 * hk * d:3 * hk * d].half()) and torch.equal(vv.reshape(700, -1), x[:, 3 * hk * d:].half())
    for prefix, copies in ((None, 1), (512, 1), (512, 300)):   # per row, and once for all
        q = q_out[:1].repeat(copies, 1, 1)
        out = torch.full_like(q, 9.0)
        A.check(paged(cache, q, 1, ints([0] * copies), ints([699] * copies), out, prefix))
        check_rows(cache, q[:1], 1, ints([0]), ints([699]), out[-1:], "f16")


# ------------------------------------------------------------------------------------------ shared prefix
def shared_case(h, hk, d, dt, qg, ps, prefix, rows, nhd, sample=None):
    g = gen(h + d + rows)
    own = [(1, 2, 63, 64, 65, 200)[r % 6] + qg - 1 for r in range(rows)]
    lens = [prefix + n for n in own]
    table, n_pages = tables(lens, ps, lead=(0,) * (prefix // ps))
    cache = Paged(hk, d, ps, n_pages, dt, table, nhd)
    fill_rows(cache, lens, g, dt, shared=prefix)
    trow = [r for r in range(rows) for _ in range(qg)]
    tpos = [n - qg + j for n in lens for j in range(qg)]
    if rows > 4:                       # rows that end inside the prefix, padding first
        tpos[-qg:] = [max(0, prefix // 2 - 3) + j for j in range(qg)]
        tpos[-2 * qg:-qg] = list(range(qg))
        trow[:qg] = [-1] * qg
    trow, tpos = ints(trow), ints(tpos)
    q = rnd((len(trow), h, d), g, dt)
    out, err = torch.full_like(q, 9.0), ints([0])
    A.check(paged(cache, q, qg, trow, tpos, out, prefix, err=err))
    torch.cuda.synchronize()
    assert err.item() == 0
    m = len(trow)
    at = torch.arange(m, device="cuda") if sample is None else torch.tensor(sorted({0, qg, m - 1, m - qg - 1} | {i * m // sample for i in range(sample)}),
                                                                          device="cuda")
    check_rows(cache, q[at], qg, trow[at], tpos[at], out[at], dt)
    again = torch.full_like(q, 9.0)
    A.check(paged(cache, q, qg, trow, tpos, again, prefix))
    assert torch.equal(out, again)


@pytest.mark.parametrize("h,hk,d,dt,qg,ps,prefix,rows,nhd", [
    (8, 2, 64, "f16", 1, 16, 48, 3, False), (32, 8, 128, "f16", 5, 64, 320, 9, True), (64, 1, 128, "f16", 1, 128, 1024, 5, False),
    (4, 4, 128, "f16", 1, 16, 16, 1, False), (48, 16, 64, "f16", 3, 8, 136, 70, False)])
def test_shared_prefix_attention_read_per_row(h, hk, d, dt, qg, ps, prefix, rows, nhd):
    assert rows * prefix * hk * d * 4 <= 128 << 20
    shared_case(h, hk, d, dt, qg, ps, prefix, rows, nhd)


@pytest.mark.parametrize("h,hk,d,dt,qg,ps,prefix,rows,nhd", [
    (32, 8, 128, "bf16", 1, 256, 2048, 40, False),      # page of two blocks, whole blocks
    (32, 4, 128, "bf16", 4, 8, 2056, 40, False),        # last block of 8 keys, pages of 8
    (10, 2, 64, "bf16", 2, 32, 4000, 70, True),         # last block of 32 keys, token-major pages
    (64, 1, 128, "f16", 1, 128, 2944, 97, False),       # 2 tokens fill a tile
    (4, 4, 128, "f16", 1, 16, 1040, 70, True),          # one head a group, last block of 16 keys
    (48, 16, 64, "f16", 3, 8, 1000, 37, False),
    (33, 1, 64, "f16", 1, 64, 16384, 33, False),        # rows of a tile that no token owns
    (8, 8, 64, "bf16", 8, 1024, 5120, 20, False)])
def test_shared_prefix_attention_read_once(h, hk, d, dt, qg, ps, prefix, rows, nhd):
    assert rows * prefix * hk * d * 4 > 128 << 20
    shared_case(h, hk, d, dt, qg, ps, prefix, rows, nhd, sample=24)


def test_shared_prefix_attention_bad_page():
    """A page of the prefix outside the cache sets the flag and reads as zeros."""
    rows, hk, d, ps, prefix = 70, 4, 128, 256, 1024
    lens = [prefix + 5] * rows
    table, n_pages = tables(lens, ps, lead=(0,) * (prefix // ps))
    cache = Paged(hk, d, ps, n_pages, "bf16", table)
    g = gen(1)
    fill_rows(cache, lens, g, "bf16", shared=prefix)
    q = rnd((rows, 8, d), g, "bf16")
    trow, tpos = ints(list(range(rows))), ints([n - 1 for n in lens])
    for bad in (-1, n_pages, 2 ** 31 - 1):
        table[:, 1] = bad
        out, err = torch.full_like(q, 9.0), ints([0])
        A.check(paged(cache, q, 1, trow, tpos, out, prefix, err=err))
        torch.cuda.synchronize()
        assert err.item() != 0
        k, v = (torch.cat([x[:256], torch.zeros_like(x[:256]), x[512:]]) for x in (lambda t: (t[0], t[1]))(cache_row_with(cache, 3, lens[3], 1)))
        check(out[3:4], attend64(q[3:4], k, v, tpos[3:4].long()), "bf16", q[3:4], k, v)


def cache_row_with(cache, row, n, hole):
    """A row's keys and values with page `hole` of its table read as page 0 (the caller blanks it)."""
    keep = cache.table[row, hole].item()
    cache.table[row, hole] = 0
    k, v = cache.row(row, n)
    cache.table[row, hole] = keep
    return k, v


# ------------------------------------------------------------------------------------------------- packed
def packed(q, k, v, cu_q, cu_k, causal, out, dt, scale=0.0, err=None):
    return L.mlxcat_op_packed_attention(ptr(q), ptr(k), ptr(v), CODE[dt], q.stride(0), k.stride(0), v.stride(0), q.shape[0], k.shape[0],
                                        ptr(cu_q), ptr(cu_k), len(cu_q) - 1, causal, q.shape[1], k.shape[1], q.shape[2], scale, ptr(out),
                                        ptr(err), stream())


def check_packed(q, k, v, cu_q, cu_k, causal, out, dt, scale=None):
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for i in range(len(cq) - 1):
        nq, nk = cq[i + 1] - cq[i], ck[i + 1] - ck[i]
        if not nq:
            continue
        lim = torch.arange(nq, device="cuda") + nk - nq if causal else torch.full((nq,), nk - 1, device="cuda")
        qq, kk, vv = q[cq[i]:cq[i + 1]], k[ck[i]:ck[i + 1]], v[ck[i]:ck[i + 1]]
        o = out[cq[i]:cq[i + 1]]
        assert (o[lim < 0] == 0).all()
        check(o, attend64(qq, kk, vv, lim, scale), dt, qq, kk, vv, scale)


@pytest.mark.parametrize("h,hk,d,dt", [(8, 2, 64, "f16"), (32, 8, 128, "bf16"), (32, 8, 128, "f16"), (10, 2, 128, "f16"), (4, 4, 64, "bf16"),
                                       (33, 1, 64, "f16"), (64, 1, 128, "bf16"), (6, 2, 128, "bf16")])
@pytest.mark.parametrize("lens,past,causal", [
    ([1], [0], 1), ([1, 1, 1], [0, 5, 200], 1), ([3, 0, 77, 128, 1], [0, 9, 0, 0, 127], 1), ([257, 31, 640], [0, 300, 1], 1),
    ([64, 129], [0, 63], 0), ([5, 130, 40], [-3, -70, -40], 1)])
def test_packed_attention(h, hk, d, dt, lens, past, causal):
    g = gen(h + d + sum(lens))
    klens = [a + b for a, b in zip(lens, past)]
    cu_q, cu_k = ints([0] + torch.tensor(lens).cumsum(0).tolist()), ints([0] + torch.tensor(klens).cumsum(0).tolist())
    x = rnd((sum(lens), (h + 2) * d), g, dt)                   # strided queries
    q = x.view(sum(lens), h + 2, d)[:, 1:h + 1]
    k, v = rnd((max(1, sum(klens)), hk, d), g, dt), rnd((max(1, sum(klens)), hk, d), g, dt)
    out = torch.full((sum(lens), h, d), 9.0, dtype=DT[dt], device="cuda")
    err = ints([0])
    if (q.data_ptr() & 15):
        pytest.skip("unaligned slice")
    A.check(packed(q, k, v, cu_q, cu_k, causal, out, dt, err=err))
    torch.cuda.synchronize()
    assert err.item() == 0
    check_packed(q, k, v, cu_q, cu_k, causal, out, dt)


def test_packed_attention_keeps_sequences_apart():
    """Non-finite keys and values of one sequence, or behind all, reach no other; tokens outside stay."""
    lens, d, h, hk = [70, 33, 90], 128, 8, 2
    for dt in ("f16", "bf16"):
        g = gen(4)
        q, k, v = rnd((230, h, d), g, dt), rnd((230, hk, d), g, dt), rnd((230, hk, d), g, dt)
        cu = ints([10, 80, 113, 203])
        for bad in (NAN, float("inf"), float("-inf")):
            kb, vb = k.clone(), v.clone()
            for x in (kb, vb):
                x[:10] = bad
                x[80:113] = bad
                x[203:] = bad
            out = torch.full((230, h, d), 9.0, dtype=DT[dt], device="cuda")
            A.check(packed(q, kb, vb, cu, cu, 1, out, dt))
            for a, b in ((10, 80), (113, 203)):
                n = b - a
                check(out[a:b], attend64(q[a:b], k[a:b], v[a:b], torch.arange(n, device="cuda")), dt, q[a:b], k[a:b], v[a:b])
            assert (out[:10] == 9.0).all() and (out[203:] == 9.0).all()
            assert not torch.isfinite(out[80:113].float()).any()


def test_packed_attention_large_scores_and_scale():
    g = gen(6)
    q, k, v = rnd((700, 8, 64), g, "bf16", 3.0), rnd((700, 2, 64), g, "bf16"), rnd((700, 2, 64), g, "bf16")
    k = k * torch.linspace(0.1, 6.0, 700, device="cuda").to(k.dtype)[:, None, None]
    cu = ints([0, 700])
    out = torch.full_like(q, 9.0)
    A.check(packed(q, k, v, cu, cu, 1, out, "bf16", scale=0.3))
    check_packed(q, k, v, cu, cu, 1, out, "bf16", 0.3)


@pytest.mark.parametrize("n,h,hk,d,dt", [(31, 8, 2, 64, "f16"), (100, 32, 8, 128, "bf16"), (1500, 4, 2, 64, "f16"), (33, 16, 1, 128, "f16")])
def test_packed_attention_many_sequences(n, h, hk, d, dt):
    """More items than SMs, more sequences than one round of the search; empty ones among them."""
    g = torch.Generator().manual_seed(n)
    top = 300 if n <= 100 else 9
    lens = torch.randint(0, top, (n,), generator=g)
    past = torch.randint(0, 200, (n,), generator=g) * (torch.rand(n, generator=g) < 0.5)
    lens[n // 2] = 0
    cu_q, cu_k = ints([0] + lens.cumsum(0).tolist()), ints([0] + (lens + past).cumsum(0).tolist())
    gc = gen(n)
    tq, tk = int(lens.sum()), int((lens + past).sum())
    q, k, v = rnd((tq, h, d), gc, dt), rnd((tk, hk, d), gc, dt), rnd((tk, hk, d), gc, dt)
    out, err = torch.full_like(q, 9.0), ints([0])
    A.check(packed(q, k, v, cu_q, cu_k, 1, out, dt, err=err))
    torch.cuda.synchronize()
    assert err.item() == 0
    check_packed(q, k, v, cu_q, cu_k, 1, out, dt)
    again = torch.full_like(q, 9.0)
    A.check(packed(q, k, v, cu_q, cu_k, 1, again, dt))
    assert torch.equal(out, again)


def test_packed_attention_bad_offsets_stay_inside():
    """Offsets past the buffers are cut to them: finite results, nothing written outside the queries."""
    g = gen(7)
    q, k, v = rnd((40, 8, 64), g, "f16"), rnd((40, 2, 64), g, "f16"), rnd((40, 2, 64), g, "f16")
    for cq, ck in (([0, 1000], [0, 1000]), ([-50, 20], [-9, 30]), ([30, 10, 60], [50, 2, 3]), ([0, 2 ** 31 - 1], [0, 2 ** 31 - 1])):
        out = torch.full((48, 8, 64), 9.0, dtype=torch.float16, device="cuda")
        A.check(packed(q, k, v, ints(cq), ints(ck), 1, out, "f16"))
        torch.cuda.synchronize()
        assert torch.isfinite(out).all() and (out[40:] == 9.0).all()


# ------------------------------------------------------------------------------------ graphs and streams
def test_graph_replay_and_two_streams():
    """One capture of append + attention replayed on new lengths, and two streams with a workspace each."""
    rows, h, hk, d, ps, dt = 4, 8, 2, 64, 16, "f16"
    g = gen(9)
    lens = [30, 17, 64, 200]
    table, n_pages = tables([n + 8 for n in lens], ps)
    cache = Paged(hk, d, ps, n_pages, dt, table)
    fill_rows(cache, lens, g, dt)
    trow, tpos = ints(list(range(rows))), ints(lens)
    x = rnd((rows, (h + 2 * hk) * d), g, "f32")
    q, k, v = x[:, :h * d], x[:, h * d:(h + hk) * d], x[:, (h + hk) * d:]
    q_out, out = torch.zeros((rows, h, d), dtype=DT[dt], device="cuda"), torch.zeros((rows, h, d), dtype=DT[dt], device="cuda")
    plan = rope_plan(d, A.ROPE_HALF)
    ws = torch.empty(L.mlxcat_op_paged_attention_workspace(rows, 1, h, hk, d), dtype=torch.uint8, device="cuda")

    def step():
        A.check(append(cache, plan, q, k, v, "f32", trow, tpos, q_out))
        A.check(paged(cache, q_out, 1, trow, tpos, out, ws=ws))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(rnd(x.shape, g, "f32"))
        graph.replay()
        torch.cuda.synchronize()
        check_rows(cache, q_out, 1, trow, tpos, out, dt)
        tpos += 1
    outs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    tpos -= 1
    torch.cuda.synchronize()
    qs = [rnd((rows, h, d), g, dt) for _ in range(2)]
    for s, qq in zip(streams, qs):
        with torch.cuda.stream(s):
            outs.append(torch.full_like(qq, 9.0))
            for _ in range(20):
                A.check(paged(cache, qq, 1, trow, tpos, outs[-1]))
    torch.cuda.synchronize()
    for qq, o in zip(qs, outs):
        check_rows(cache, qq, 1, trow, tpos, o, dt)


def test_graph_of_packed_and_shared_attention():
    """Both tensor-core paths captured together and replayed on new values and lengths."""
    g, dt, h, hk, d, ps, rows, prefix = gen(11), "bf16", 16, 4, 128, 64, 40, 2048
    lens = [prefix + 3 + r for r in range(rows)]
    table, n_pages = tables([n + 4 for n in lens], ps, lead=(0,) * (prefix // ps))
    cache = Paged(hk, d, ps, n_pages, dt, table)
    fill_rows(cache, [n + 4 for n in lens], g, dt, shared=prefix)
    trow, tpos = ints(list(range(rows))), ints([n - 1 for n in lens])
    q, out = rnd((rows, h, d), g, dt), torch.zeros((rows, h, d), dtype=DT[dt], device="cuda")
    ws = torch.empty(L.mlxcat_op_shared_prefix_attention_workspace(rows, 1, h, hk, d, prefix), dtype=torch.uint8, device="cuda")
    pq, pk, pv = rnd((700, h, d), g, dt), rnd((700, hk, d), g, dt), rnd((700, hk, d), g, dt)
    cu, po = ints([0, 100, 101, 700]), torch.zeros((700, h, d), dtype=DT[dt], device="cuda")

    def step():
        A.check(packed(pq, pk, pv, cu, cu, 1, po, dt))
        A.check(paged(cache, q, 1, trow, tpos, out, prefix, ws=ws))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        q.copy_(rnd(q.shape, g, dt))
        pq.copy_(rnd(pq.shape, g, dt))
        cu.copy_(ints([[0, 100, 101, 700], [0, 0, 333, 700], [0, 650, 651, 700]][i]))
        graph.replay()
        torch.cuda.synchronize()
        check_rows(cache, q[::7], 1, trow[::7], tpos[::7], out[::7], dt)
        check_packed(pq, pk, pv, cu, cu, 1, po, dt)
        tpos += 1


# -------------------------------------------------------------------------------------- a serving run
@pytest.mark.parametrize("dt,d", [("f16", 128), ("bf16", 64)])
def test_serving_run(dt, d):
    """Admission of three prompts behind one shared instruction block, then verify steps of three tokens:
    append + packed attention, append + paged / shared-prefix attention, against the dense formula on the
    keys and values that the formula itself rotates."""
    h, hk, ps, qg, prefix = 8, 2, 32, 3, 64
    prompts = [70, 128, 33]                     # tokens after the shared block
    rows, steps = 3, 4
    g = gen(d)
    lens = [prefix + p + qg * steps for p in prompts]
    table, n_pages = tables(lens, ps, lead=(0, 0))
    cache = Paged(hk, d, ps, n_pages, dt, table)
    plan = rope_plan(d, A.ROPE_HALF)
    qn, kn = (1 + 0.2 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    width = (h + 2 * hk) * d
    keys, vals = [None] * rows, [None] * rows   # what the formula has, rounded to the cache's type

    def project(x, tpos):
        m = x.shape[0]
        q = turned64(x[:, :h * d].view(m, h, d), tpos, plan, qn)[0]
        k = turned64(x[:, h * d:(h + hk) * d].view(m, hk, d), tpos, plan, kn)[0]
        return q.to(DT[dt]), k.to(DT[dt]), x[:, (h + hk) * d:].view(m, hk, d).to(DT[dt])

    def run_append(x, trow, tpos):
        q_out = torch.zeros((x.shape[0], h, d), dtype=DT[dt], device="cuda")
        A.check(append(cache, plan, x[:, :h * d], x[:, h * d:(h + hk) * d], x[:, (h + hk) * d:], "f32", trow, tpos, q_out, qn, kn))
        return q_out

    def loose(got, q, k, v, lim):
        # the operands themselves are one rounding apart (2 u each way in q and k): scores differ by up to
        # 4 u |q| |k| / sqrt(d), the values by u
        y, a, _ = attend64(q, k, v, lim)
        u = half_step(dt)
        ds = 4 * u * (q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()).item() / math.sqrt(d)
        tol = u * y.abs() + 2 * a * (2 * u + math.expm1(2 * ds)) + 1e-6
        assert ((got.double() - y).abs() <= tol).all()

    x = rnd((prefix, width), g, "f32")          # the shared block, appended once
    pos = torch.arange(prefix, device="cuda", dtype=torch.int32)
    run_append(x, ints([0] * prefix), pos)
    _, k0, v0 = project(x, pos)
    xs = [rnd((p, width), g, "f32") for p in prompts]
    x = torch.cat(xs)
    trow = ints([r for r in range(rows) for _ in range(prompts[r])])
    tpos = ints([prefix + j for r in range(rows) for j in range(prompts[r])])
    q_out = run_append(x, trow, tpos)
    kv = [cache.row(r, prefix + prompts[r]) for r in range(rows)]
    k, v = torch.cat([a for a, _ in kv]), torch.cat([b for _, b in kv])
    cu_q = ints([0] + torch.tensor(prompts).cumsum(0).tolist())
    cu_k = ints([0] + (torch.tensor(prompts) + prefix).cumsum(0).tolist())
    out = torch.zeros_like(q_out)
    A.check(packed(q_out, k, v, cu_q, cu_k, 1, out, dt))
    for r in range(rows):
        a, b = cu_q[r].item(), cu_q[r + 1].item()
        qq, kk, vv = project(xs[r], tpos[a:b])
        keys[r], vals[r] = torch.cat([k0, kk]), torch.cat([v0, vv])
        loose(out[a:b], qq, keys[r], vals[r], tpos[a:b].long())
    at = [prefix + p for p in prompts]
    for _ in range(steps):
        x = rnd((rows * qg, width), g, "f32")
        trow = ints([r for r in range(rows) for _ in range(qg)])
        tpos = ints([at[r] + j for r in range(rows) for j in range(qg)])
        q_out = run_append(x, trow, tpos)
        o1, o2 = torch.zeros_like(q_out), torch.zeros_like(q_out)
        A.check(paged(cache, q_out, qg, trow, tpos, o1))
        A.check(paged(cache, q_out, qg, trow, tpos, o2, prefix))
        for r in range(rows):
            s = slice(r * qg, (r + 1) * qg)
            qq, kk, vv = project(x[s], tpos[s])
            keys[r], vals[r] = torch.cat([keys[r], kk]), torch.cat([vals[r], vv])
            loose(o1[s], qq, keys[r], vals[r], tpos[s].long())
            loose(o2[s], qq, keys[r], vals[r], tpos[s].long())
            at[r] += qg


# ------------------------------------------------- shared prefix read once, every token against the formula
class Once:
    """Rows behind one prefix with at most a page of own keys each, so that the formula takes all tokens in
    one go; keys no token sees are NaN.  Tokens come in groups of qg, the last ones of their row."""

    def __init__(self, h, hk, d, dt, qg, ps, prefix, rows, seed=0):
        self.h, self.hk, self.d, self.dt, self.qg, self.ps, self.prefix, self.rows = h, hk, d, dt, qg, ps, prefix, rows
        g = gen(seed + h + rows)
        own = [qg + r % (ps - qg + 1) for r in range(rows)]
        table, n_pages = tables([prefix + n for n in own], ps, seed=seed, lead=(0,) * (prefix // ps))
        self.cache = Paged(hk, d, ps, n_pages, dt, table)
        self.cache.put(0, rnd((prefix, hk, d), g, dt), rnd((prefix, hk, d), g, dt))
        for r, n in enumerate(own):
            self.cache.put(r, rnd((n, hk, d), g, dt), rnd((n, hk, d), g, dt), prefix)
        self.trow = ints([r for r in range(rows) for _ in range(qg)])
        self.tpos = ints([prefix + n - qg + j for n in own for j in range(qg)])
        self.q = rnd((rows * qg, h, d), g, dt)
        assert rows * prefix * hk * d * 4 > 128 << 20        # read once

    def run(self, ws=None, err=None):
        out = torch.full_like(self.q, 9.0)
        A.check(paged(self.cache, self.q, self.qg, self.trow, self.tpos, out, self.prefix, ws=ws, err=err))
        return out

    def check(self, out, sees=None):
        """sees: tokens that see keys at all (default: those of a row, at a position >= 0)."""
        c, g = self.cache, self.h // self.hk
        live = (self.trow >= 0) & (self.tpos >= 0) if sees is None else sees
        assert (out[self.trow < 0] == 9.0).all()
        assert (out[(self.trow >= 0) & ~live] == 0).all()
        at = live.nonzero()[:, 0]
        if not len(at):
            return
        row, pos = self.trow[at].long(), self.tpos[at].long()
        q = self.q[at].double().view(len(at), self.hk, g, self.d)
        kp, vp = (x.double() for x in c.row(0, self.prefix))
        page = c.table[row, self.prefix // self.ps].long()
        ko, vo = (x[page].double() for x in (c.view(c.k), c.view(c.v)))       # [token][kv head][key][d]
        seen = torch.arange(self.prefix + self.ps, device="cuda")[None, :] <= pos[:, None]
        own_seen = seen[:, None, self.prefix:, None]
        ko, vo = ko.masked_fill(~own_seen, 0.0), vo.masked_fill(~own_seen, 0.0)
        s = torch.cat([torch.einsum("nkgd,pkd->nkgp", q, kp), torch.einsum("nkgd,nkpd->nkgp", q, ko)], -1) / math.sqrt(self.d)
        s = s.masked_fill(~seen[:, None, None, :], float("-inf"))
        e = torch.exp(s - s.amax(-1, keepdim=True))
        tot = e.sum(-1, keepdim=True)
        w = e / tot
        wp, wo = w[..., :self.prefix], w[..., self.prefix:]
        y = torch.einsum("nkgp,pkd->nkgd", wp, vp) + torch.einsum("nkgp,nkpd->nkgd", wo, vo)
        a = torch.einsum("nkgp,pkd->nkgd", wp, vp.abs()) + torch.einsum("nkgp,nkpd->nkgd", wo, vo.abs())
        err = 2 * self.d * 2.0 ** -24 * q.norm(dim=-1).max() * max(kp.norm(dim=-1).max(), ko.norm(dim=-1).max()) / math.sqrt(self.d)
        u = half_step(self.dt)
        tol = u * y.abs() + 2 * a * (u + err + 2.0 ** -21) + 1e-7
        if self.dt == "f16":
            tol = tol + s.shape[-1] * 2.0 ** -25 * max(vp.abs().max(), vo.abs().max()) / tot
        got = out[at].double().view_as(y)
        assert torch.isfinite(got).all()
        worst = ((got - y).abs() / tol).flatten(1).amax(1)
        assert worst.max().item() <= 1.0, (worst.max().item(), at[worst > 1.0][:20].tolist(), int((worst > 1.0).sum()))


def test_shared_prefix_after_append_replayed():
    """Keys, queries, positions and page ids written right before the call, captured and replayed: the pass over
    the prefix and the kernel beside it both see them, whatever the workspace held."""
    qg, ps, prefix, rows, h, hk, d = 2, 64, 2048, 70, 32, 8, 128
    x = Once(h, hk, d, "f16", qg, ps, prefix, rows)
    for c in (x.cache.k, x.cache.v):
        c.nan_to_num_(nan=0.5)                       # a row's page is full
    m, g, cg = rows * qg, gen(31), torch.Generator().manual_seed(31)
    xin = torch.zeros((m, (h + 2 * hk) * d), device="cuda")
    table, tpos = x.cache.table.clone(), x.tpos.clone()
    out = torch.zeros((m, h, d), dtype=torch.float16, device="cuda")
    ws = torch.empty(L.mlxcat_op_shared_prefix_attention_workspace(m, qg, h, hk, d, prefix), dtype=torch.uint8, device="cuda")

    def step():
        x.cache.table.copy_(table)
        x.tpos.copy_(tpos)
        A.check(append(x.cache, None, xin[:, :h * d], xin[:, h * d:(h + hk) * d], xin[:, (h + hk) * d:], "f32", x.trow, x.tpos, x.q))
        A.check(paged(x.cache, x.q, qg, x.trow, x.tpos, out, prefix, ws=ws))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(12):
        xin.copy_(torch.randn(xin.shape, device="cuda", generator=g))
        first = prefix + torch.randint(0, ps - qg + 1, (rows,), generator=cg)
        tpos.copy_((first[:, None] + torch.arange(qg)).flatten())
        table.copy_(table[torch.randperm(rows, generator=cg).cuda()])        # rows change their own pages
        if i % 3 == 0:
            ws.fill_(0xff)
        if i % 3 == 1:
            ws.random_(generator=g)
        graph.replay() if i % 4 else step()
        torch.cuda.synchronize()
        x.check(out)


def once_items(h, hk, m):
    """(pair of tiles, KV head) items of the pass over the prefix: two tiles of 128 (token, head) rows each."""
    return -(-m // (2 * (128 // (h // hk)))) * hk


@pytest.mark.parametrize("h,hk,d,dt,qg,ps,prefix,rows", [
    (64, 8, 128, "f16", 8, 64, 256, 300),       # two key blocks, 600 items
    (32, 8, 128, "bf16", 5, 128, 128, 960),     # one key block, 600 items
    (32, 16, 64, "f16", 4, 8, 1160, 650),       # ten blocks, the last of 8 keys
    (8, 8, 128, "bf16", 1, 16, 272, 11000)])    # one head a group, many rows of one token
def test_shared_prefix_many_items_a_cta(h, hk, d, dt, qg, ps, prefix, rows):
    """A CTA of the pass takes three items and more: descriptors, queries and O change hands, every token is right."""
    x = Once(h, hk, d, dt, qg, ps, prefix, rows)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert once_items(h, hk, rows * qg) > 2 * sms
    err = ints([0])
    out = x.run(err=err)
    torch.cuda.synchronize()
    assert err.item() == 0
    x.check(out)
    for _ in range(5):
        assert torch.equal(out, x.run())


@pytest.mark.parametrize("once", [True, False])
def test_workspace_on_any_16_byte_boundary(once):
    """A workspace cut from an arena: 16-byte aligned is enough, nothing outside it is written."""
    x = Once(32, 8, 128, "bf16", 1, 64, 2048, 70)
    n = 70 if once else 9                                    # 9 rows read the prefix one by one
    q, trow, tpos = x.q[:n], x.trow[:n], x.tpos[:n]
    assert (n * x.prefix * x.hk * x.d * 4 > 128 << 20) == once
    size = L.mlxcat_op_shared_prefix_attention_workspace(n, 1, x.h, x.hk, x.d, x.prefix)
    arena, outs = torch.empty(size + 256, dtype=torch.uint8, device="cuda"), []
    for at in (0, 16, 32, 48, 112):
        arena.fill_(0xab)
        ws = arena[at:at + size]
        assert ws.data_ptr() % 256 == at
        outs.append(torch.full_like(q, 9.0))
        A.check(paged(x.cache, q, 1, trow, tpos, outs[-1], x.prefix, ws=ws))
        torch.cuda.synchronize()
        assert (arena[:at] == 0xab).all() and (arena[at + size:] == 0xab).all()
    assert all(torch.equal(outs[0], o) for o in outs)
    if once:
        x.check(outs[1])
    else:
        check_rows(x.cache, q, 1, trow, tpos, outs[1], "bf16")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_shared_prefix_read_once_empty_padding_and_out_of_range(dt):
    """Read once or row by row, the call says the same: tokens of a row outside the table and tokens before
    position 0 get zeros, padding stays, positions past the table are cut to it, the flag tells."""
    qg, rows = 3, 70
    x = Once(32, 8, 128, dt, qg, 64, 2048, rows)
    for c in (x.cache.k, x.cache.v):
        c.nan_to_num_(nan=0.5)                                # whole own pages, for the cut positions
    cap = x.prefix + x.ps
    x.q, x.trow, x.tpos = x.q[:-2].contiguous(), x.trow[:-2].contiguous(), x.tpos[:-2].contiguous()   # a short last group
    def group(i):
        return slice(i * qg, (i + 1) * qg)
    x.trow[group(0)] = -1                                     # padding first
    x.tpos[group(1)] = -1                                     # no key
    x.tpos[group(2)] = ints([-2, -1, 0])                      # a key for the last of the group
    x.trow[6 * qg + 1:7 * qg] = -1                            # a group that ends in padding
    x.tpos[group(7)] = ints([x.prefix - 2, x.prefix - 1, x.prefix])
    x.tpos[group(8)] = ints([5, 6, 7])
    err = ints([0])
    x.check(x.run(err=err))
    assert err.item() == 0
    outside = [(3, rows), (4, rows + 1), (9, 2 ** 31 - 1)]
    for bad in (outside, outside + [(1, rows)], [(i, rows + i) for i in range(rows)]):
        keep = x.trow.clone()
        for i, r in bad:
            x.trow[group(i)] = r
        err.zero_()
        out = x.run(err=err)
        assert err.item() == 51
        x.check(out, (x.trow >= 0) & (x.trow < rows) & (x.tpos >= 0))
        few = slice(0, 10 * qg)                               # the same tokens row by row
        assert 10 * x.prefix * x.hk * x.d * 4 <= 128 << 20
        apart = torch.full_like(x.q[few], 9.0)
        A.check(paged(x.cache, x.q[few], qg, x.trow[few], x.tpos[few], apart, x.prefix))
        none = (x.trow[few] < 0) | (x.trow[few] >= rows) | (x.tpos[few] < 0)
        assert torch.equal(apart[none], out[few][none])
        x.trow = keep
    x.tpos[group(5)] = ints([cap - 1, cap, 2 ** 31 - 1])
    err.zero_()
    out = x.run(err=err)
    assert err.item() == 52
    x.tpos[group(5)] = cap - 1
    x.check(out)


def test_append_same_place_twice():
    """Tokens that share a place: every 16 bytes there are one of the tokens', the queries are each its own."""
    h, hk, d, n = 8, 8, 128, 64
    cache = Paged(hk, d, 16, 2, "f16", ints([[0, 1]]), fill=9.0)
    x = rnd((n, (h + 2 * hk) * d), gen(5), "f16")
    q, k, v = x[:, :h * d], x[:, h * d:(h + hk) * d], x[:, (h + hk) * d:]
    q_out = torch.zeros((n, h, d), dtype=torch.float16, device="cuda")
    A.check(append(cache, None, q, k, v, "f16", ints([0] * n), ints([5] * (n - 1) + [17]), q_out))
    assert torch.equal(q_out.view(n, -1), q)
    for c, src in ((cache.k, k), (cache.v, v)):
        got = c[0, :, 5].reshape(-1, 8)
        assert (got[None] == src[:-1].reshape(n - 1, -1, 8)).all(-1).any(0).all()
        assert torch.equal(c[1, :, 1].reshape(-1), src[-1])
        c[0, :, 5] = c[1, :, 1] = 9.0
        assert (c == 9.0).all()


# ------------------------------------------------------------------------------------------ more of the range
@pytest.mark.parametrize("d,rd,layout,src,dt", [(128, 96, 0, "f32", "f16"), (128, 72, 0, "bf16", "bf16"), (64, 48, 0, "f16", "bf16"),
                                                (128, 96, 1, "f16", "f16"), (64, 32, 0, "f32", "f16"), (128, 64, 0, "bf16", "f16")])
def test_append_rotary_widths(d, rd, layout, src, dt):
    """Rotary widths between half a head and a head, and those whose partner is another lane's."""
    test_append(d, 6, 2, dt, src, rd, layout, 0, True, 16, False, 21)


@pytest.mark.parametrize("keys", [8, 64, 72, 130, 192, 200, 320, 384, 3904, 3912])
def test_paged_attention_every_cluster_size(keys):
    """One row, one KV head, tables of 1 to 62 units: one cluster of 4 to 8 CTAs, then two kernels."""
    g, ps = gen(keys), 8
    table, n_pages = tables([keys], ps, spare=0)
    cache = Paged(1, 64, ps, n_pages, "bf16", table)
    fill_rows(cache, [keys], g, "bf16")
    for n in {1, keys // 2, keys}:
        q = rnd((1, 5, 64), g, "bf16")
        out = torch.full_like(q, 9.0)
        A.check(paged(cache, q, 1, ints([0]), ints([n - 1]), out))
        check_rows(cache, q, 1, ints([0]), ints([n - 1]), out, "bf16")


@pytest.mark.parametrize("width", [0, 500])
def test_shared_prefix_without_own_keys(width):
    """The prefix is all there is: a table that ends with it, and one with empty pages behind it."""
    rows, h, hk, d, ps, prefix, dt = 70, 32, 8, 128, 64, 2048, "f16"
    table, n_pages = tables([prefix] * rows, ps, lead=(0,) * (prefix // ps))
    table = torch.cat([table[:, :prefix // ps], torch.full((rows, width), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    cache, g = Paged(hk, d, ps, n_pages, dt, table), gen(3)
    cache.put(0, rnd((prefix, hk, d), g, dt), rnd((prefix, hk, d), g, dt))
    q, trow = rnd((rows, h, d), g, dt), ints(list(range(rows)))
    tpos = ints([prefix - 1 if r % 3 else r * 29 for r in range(rows)])
    out, err = torch.full_like(q, 9.0), ints([0])
    assert rows * prefix * hk * d * 4 > 128 << 20
    A.check(paged(cache, q, 1, trow, tpos, out, prefix, err=err))
    check_rows(cache, q, 1, trow, tpos, out, dt)
    assert err.item() == 0


@pytest.mark.parametrize("qg,rows", [(1, 257), (3, 300), (2, 4000)])
def test_paged_attention_many_groups(qg, rows):
    """More groups than a CTA keeps, groups of several tokens, rows without keys and padding among them."""
    h, hk, d, ps, dt = 8, 2, 64, 16, "bf16"
    lens = [(1, 30, 0, 64, 129, 17, 300)[r % 7] for r in range(rows)]
    lens = [n + qg - 1 if n else 0 for n in lens]
    table, n_pages = tables(lens, ps)
    cache, g = Paged(hk, d, ps, n_pages, dt, table), gen(rows)
    fill_rows(cache, lens, g, dt)
    trow = ints([r if r % 11 else -1 for r in range(rows) for _ in range(qg)])
    tpos = ints([max(-1, n - qg + j) if n else -1 for n in lens for j in range(qg)])
    q = rnd((rows * qg, h, d), g, dt)
    out, err = torch.full_like(q, 9.0), ints([0])
    A.check(paged(cache, q, qg, trow, tpos, out, err=err))
    torch.cuda.synchronize()
    assert err.item() == 0
    at = torch.arange(0, rows * qg, max(1, rows * qg // 400), device="cuda")
    check_rows(cache, q[at], qg, trow[at], tpos[at], out[at], dt)
    assert (out[trow < 0] == 9.0).all() and (out[(trow >= 0) & (tpos < 0)] == 0).all() and torch.isfinite(out).all()


def test_shared_prefix_on_two_streams():
    """Calls that read the prefix once, side by side on two streams, a workspace and queries each."""
    x = Once(32, 8, 128, "f16", 2, 64, 2048, 600)
    q0 = x.q
    want = x.run()
    x.check(want)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    wss = [torch.full((L.mlxcat_op_shared_prefix_attention_workspace(1200, 2, 32, 8, 128, 2048),), 0xff, dtype=torch.uint8, device="cuda")
           for _ in streams]
    qs = [q0, q0.flip(0).contiguous()]
    rr, pp = [x.trow, x.trow.flip(0).contiguous()], [x.tpos, x.tpos.flip(0).contiguous()]
    pp[1] = pp[1].view(-1, 2).flip(1).flatten().contiguous()      # within a group the positions rise again
    qs[1] = qs[1].view(-1, 2, 32, 128).flip(1).flatten(0, 1).contiguous()
    torch.cuda.synchronize()
    for _ in range(15):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(torch.full_like(q0, 9.0))
                A.check(paged(x.cache, qs[i], 2, rr[i], pp[i], outs[i][-1], x.prefix, ws=wss[i]))
    torch.cuda.synchronize()
    for o in outs[0]:
        assert torch.equal(o, want)
    for o in outs[1]:
        x.q, x.trow, x.tpos = qs[1], rr[1], pp[1]
        x.check(o)


@pytest.mark.parametrize("h,hk,d,dt,at", [(8, 2, 128, "bf16", 0), (6, 2, 64, "f16", 8), (32, 8, 128, "f16", 24)])
def test_packed_attention_on_slices_of_a_projection(h, hk, d, dt, at):
    """q, k and v side by side in one buffer, the output on a 16-byte boundary."""
    lens, g = [130, 1, 300], gen(at)
    m, width = sum(lens), (h + 2 * hk) * d
    x = rnd((m, width + 8), g, dt)
    q, k, v = (x[:, a * d:(a + n) * d].unflatten(1, (n, d)) for a, n in ((0, h), (h, hk), (h + hk, hk)))
    cu = ints([0, 130, 131, 431])
    arena = torch.full((m * h * d + 64,), 9.0, dtype=DT[dt], device="cuda")
    out = arena[at:at + m * h * d].view(m, h, d)
    A.check(packed(q, k, v, cu, cu, 1, out, dt))
    check_packed(q, k, v, cu, cu, 1, out, dt)
    assert (arena[:at] == 9.0).all() and (arena[at + m * h * d:] == 9.0).all()


@pytest.mark.parametrize("m", [8, 160])
def test_projection_append_attention_launched_early(m):
    """Each kernel of the chain starts before the one in front has ended, on memory that has just been read with
    other contents: what is read is what that one wrote."""
    h, hk, d, ps, qg, dt = 8, 2, 128, 64, 4, "f16"
    rows, n, kk, g = m // qg, (h + 2 * hk) * d, 512, gen(m)
    wq = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, kk // 8), dtype=torch.int32, device="cuda", generator=g)
    sc, bi = ((torch.rand((n, kk // 64), device="cuda", generator=g) * 0.01 + b).half() for b in (0.005, -0.1))
    xs = [rnd((m, kk), g, dt) for _ in range(3)]
    lens = [70 + 3 * r for r in range(rows)]
    table, n_pages = tables([x + qg for x in lens], ps)
    cache = Paged(hk, d, ps, n_pages, dt, table)
    fill_rows(cache, [x + qg for x in lens], g, dt)
    trow = ints([r for r in range(rows) for _ in range(qg)])
    ends = [ints([x + j - s for x in lens for j in range(qg)]) for s in (0, 40, 11)]
    tpos, x = ends[0].clone(), xs[0].clone()
    y = torch.zeros((m, n), device="cuda")
    q_out, out = torch.zeros((m, h, d), dtype=torch.float16, device="cuda"), torch.zeros((m, h, d), dtype=torch.float16, device="cuda")
    size = L.mlxcat_op_q4_linear_workspace(n, kk, m)
    lw, ws = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty(
        L.mlxcat_op_paged_attention_workspace(m, qg, h, hk, d), dtype=torch.uint8, device="cuda")
    seen = set()
    for i in range(30):
        x.copy_(xs[i % 3])
        tpos.copy_(ends[i % 3 if i % 2 else 0])
        A.check(L.mlxcat_op_q4_linear(ptr(wq), ptr(sc), ptr(bi), n, kk, ptr(x), m, ptr(y), ptr(lw), size, stream()))
        A.check(append(cache, None, y[:, :h * d], y[:, h * d:(h + hk) * d], y[:, (h + hk) * d:], "f32", trow, tpos, q_out))
        A.check(paged(cache, q_out, qg, trow, tpos, out, ws=ws))
        torch.cuda.synchronize()
        half = y.half()
        assert torch.isfinite(half).all() and half.float().std() > 0.05
        assert torch.equal(q_out.view(m, -1), half[:, :h * d])
        page, off = table[trow.long(), (tpos // ps).long()].long(), (tpos % ps).long()
        assert torch.equal(cache.k[page, :, off].reshape(m, -1), half[:, h * d:(h + hk) * d])
        assert torch.equal(cache.v[page, :, off].reshape(m, -1), half[:, (h + hk) * d:])
        at = torch.arange(0, m, 7, device="cuda")
        check_rows(cache, q_out[at], qg, trow[at], tpos[at], out[at], dt)
        seen.add(round(y.double().sum().item(), 3))
    assert len(seen) == 3
