"""The paged-serving operators on their cases: plain form, framework's form, exact values.

A paged KV cache (pages of `ps` tokens, [page][kv head][token][d]) is written by `rope_append` (RMSNorm of
each q / k head, rotary position, append) and read by `paged_attention` (single tokens or groups of
consecutive tokens per row) and `shared_prefix_attention` (a batch whose first keys are the same pages);
`packed_attention` is the causal attention of several prompts laid end to end.

Where `own` is false `run` is elementary torch arithmetic in 32 bits (angles in 64), rounded once.
"""
import ctypes
import math

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODE = {"f16": 0, "bf16": 1, "f32": 2}
HALF, INTERLEAVED = 0, 1
SCALING = {"none": 0, "linear": 1, "llama3": 2, "yarn": 3}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    """Head counts are the tiny, Llama-3-8B, Qwen3-4B, Llama-3-70B and Qwen3-30B-A3B configurations'."""
    return [
        # eight rows of the tiny model decode one token each: launch latency
        dict(name="append-decode", op="append", h=8, hk=2, d=64, dt="f16", src="f16", rows=8, t=1, ctx=300, ps=16,
             rd=64, layout=0, scaling="none", theta=500000.0, norm=False),
        # the verify step's 32 rows x 5 tokens from an fp32 projection, wavelength-banded long-context scaling
        dict(name="append-verify", op="append", h=32, hk=8, d=128, dt="f16", src="f32", rows=32, t=5, ctx=4200, ps=64,
             rd=128, layout=0, scaling="llama3", theta=500000.0, norm=False),
        # admission of four prompts of the q/k-normalised model, far positions under interpolated rotation
        dict(name="append-prompts", op="append", h=32, hk=8, d=128, dt="bf16", src="bf16", rows=4, t=4099, ctx=0, ps=256,
             rd=128, layout=1, scaling="yarn", theta=1000000.0, norm=True),
        # one short row of the tiny model, one token
        dict(name="paged-one-row", op="paged", h=8, hk=2, d=64, dt="f16", rows=1, qg=1, lo=300, hi=300, ps=16),
        # the Llama-3-8B verify step: 32 rows x 5 tokens over about 4.2k keys
        dict(name="paged-verify", op="paged", h=32, hk=8, d=128, dt="f16", rows=32, qg=5, lo=4000, hi=4400, ps=64),
        # single tokens, very uneven rows, 70B heads
        dict(name="paged-ragged", op="paged", h=64, hk=8, d=128, dt="bf16", rows=64, qg=1, lo=1, hi=16384, ps=256),
        # four short requests over one instruction block
        dict(name="shared-small", op="shared", h=8, hk=2, d=64, dt="bf16", rows=4, qg=1, prefix=512, lo=1, hi=64, ps=32),
        # 64 requests over one 8k document
        dict(name="shared-document", op="shared", h=32, hk=8, d=128, dt="f16", rows=64, qg=1, prefix=8192, lo=1, hi=512,
             ps=256),
        # 96 requests in verify groups over a 32k document
        dict(name="shared-verify", op="shared", h=32, hk=4, d=128, dt="bf16", rows=96, qg=4, prefix=32704, lo=100, hi=1500,
             ps=64),
        # three tiny prompts, one of a single token
        dict(name="packed-tiny", op="packed", h=8, hk=2, d=64, dt="f16", n=3, lo=1, hi=150, cached=0),
        # sixteen chat prompts, some after a cached part
        dict(name="packed-chat", op="packed", h=32, hk=8, d=128, dt="f16", n=16, lo=33, hi=1500, cached=300),
        # three long documents
        dict(name="packed-long", op="packed", h=32, hk=8, d=128, dt="bf16", n=3, lo=2045, hi=6144, cached=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "paged", "shared", "packed"])
    h, hk, d = rng.choice([(8, 2, 64), (8, 8, 64), (32, 8, 128), (16, 4, 128), (64, 8, 128), (32, 4, 128), (12, 4, 64), (10, 2, 128)])
    dt = rng.choice(["f16", "bf16"])
    ps = rng.choice([8, 16, 32, 64, 128, 256])
    c = dict(op=op, h=h, hk=hk, d=d, dt=dt)
    if op == "append":
        rows = _log(rng, 1, 64)
        t = max(1, min(_log(rng, 1, 4096), 400000 // (rows * (h + 2 * hk))))
        rd = d if rng.random() < 0.6 else rng.choice([d // 2, d // 4, 20])
        c.update(src=rng.choice(["f16", "bf16", "f32"]), rows=rows, t=t, ctx=rng.choice([0, _log(rng, 1, 100000 // rows)]), ps=ps,
                 rd=rd, layout=rng.choice([0, 1]), scaling=rng.choice(["none", "linear", "llama3", "yarn"]),
                 theta=rng.choice([10000.0, 500000.0, 1000000.0]), norm=rng.random() < 0.5)
    elif op == "paged":
        rows = _log(rng, 1, 64)
        hi = min(_log(rng, 1, 16384), 500000 // rows)
        c.update(rows=rows, qg=rng.choice([1, 1, 2, 3, 5, 8]), lo=max(1, int(hi * rng.random())), hi=hi, ps=ps)
    elif op == "shared":
        rows = _log(rng, 1, 96)
        hi = _log(rng, 1, 1024)
        c.update(rows=rows, qg=rng.choice([1, 1, 2, 4]), prefix=ps * max(1, _log(rng, 64, 24576) // ps), lo=max(1, int(hi * rng.random())),
                 hi=hi, ps=ps)
    else:
        n = _log(rng, 1, 24)
        hi = min(_log(rng, 1, 5000), int(math.sqrt(2.0e9 / (n * h))))
        c.update(n=n, lo=max(1, int(hi * rng.random())), hi=hi, cached=rng.choice([0, 0, _log(rng, 1, 700)]))
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """The case's length of each row or sequence (the bounds and values between them) and of what is cached before it."""
    n, g = case.get("rows") or case.get("n"), torch.Generator().manual_seed(17)
    if case["op"] == "append":
        past = torch.randint(0, case["ctx"] + 1, (n,), generator=g)
        past[0] = case["ctx"]
        return torch.full((n,), case["t"]), past
    x = torch.randint(case["lo"], case["hi"] + 1, (n,), generator=g)
    x[-1] = case["lo"]
    x[0] = case["hi"]
    return x, torch.randint(0, case.get("cached", 0) + 1, (n,), generator=g)


def _pages(rows, lens, ps, g):
    """Page tables of rows of `lens` keys on shuffled pages; entries past a row's end are -1."""
    need = (lens + ps - 1) // ps
    width = max(1, int(need.max()))
    total = int(need.sum())
    n_pages = total + 3
    ids = torch.randperm(n_pages, generator=g)[:total].to(torch.int32)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    table[torch.arange(width)[None, :] < need[:, None]] = ids
    return table, n_pages


def _normal(shape, g, dt, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g, dtype=torch.float32) * scale).to(dt)


def _frequencies(rd, theta, scaling):
    """Angular frequency of each pair (64 bits) and the factor on cos and sin, long-context factor 8."""
    f = theta ** (-2.0 * torch.arange(rd // 2, dtype=torch.float64) / rd)
    if scaling == "linear":
        return f / 8.0, 1.0
    if scaling == "llama3":
        turns = 8192.0 * f / (2 * math.pi)               # rotations within the original context
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return (1 - keep) * f / 8.0 + keep * f, 1.0
    if scaling == "yarn":
        def at(rot):
            return rd * math.log(32768.0 / (rot * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(0.0, float(math.floor(at(32.0)))), min(rd - 1.0, float(math.ceil(at(1.0))))
        ramp = ((torch.arange(rd // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return f / 8.0 * ramp + f * (1 - ramp), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    gc = torch.Generator().manual_seed(seed * 1000003 + 17)
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)
    h, hk, d, dt = case["h"], case["hk"], case["d"], DT[case["dt"]]
    s = {"case": dict(case)}
    if case["op"] == "append":
        rows, t, ps = case["rows"], case["t"], case["ps"]
        lens, base = _lengths(case)
        lens = lens + base
        table, n_pages = _pages(rows, lens, ps, gc)
        pos = base[:, None] + torch.arange(t)[None, :]
        row = torch.arange(rows)[:, None].expand(rows, t)
        m = rows * t
        x = _normal((m, (h + 2 * hk) * d), g, DT[case["src"]])
        s.update(x=x, q_norm=None, k_norm=None)
        if case["norm"]:
            s["q_norm"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
            s["k_norm"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
        f, mscale = _frequencies(case["rd"], case["theta"], case["scaling"])
        s.update(freq=f.cuda(), mscale=mscale, q=torch.empty((m, h, d), dtype=dt, device="cuda"),
                 row=row.reshape(-1).to(torch.int32).cuda(), pos=pos.reshape(-1).to(torch.int32).cuda())
    elif case["op"] in ("paged", "shared"):
        rows, qg, ps, pre = case["rows"], case["qg"], case["ps"], case.get("prefix", 0)
        own_len = _lengths(case)[0] + (qg - 1)          # keys of the row itself, the group's own tokens among them
        table, n_pages = _pages(rows, own_len, ps, gc)
        if pre:                                          # the shared pages come first in every row's table
            shared = torch.arange(n_pages, n_pages + pre // ps, dtype=torch.int32)
            table = torch.cat([shared[None, :].expand(rows, -1), table], 1).contiguous()
            n_pages += pre // ps
        lens = own_len + pre
        pos = (lens - qg)[:, None] + torch.arange(qg)[None, :]
        row = torch.arange(rows)[:, None].expand(rows, qg)
        m = rows * qg
        s.update(q=_normal((m, h, d), g, dt), out=torch.empty((m, h, d), dtype=dt, device="cuda"), lens=lens.cuda(),
                 row=row.reshape(-1).to(torch.int32).cuda(), pos=pos.reshape(-1).to(torch.int32).cuda(), longest=int(own_len.max()))
    else:
        lens, past = _lengths(case)
        klens = lens + past
        tq, tk = int(lens.sum()), int(klens.sum())
        zero = torch.zeros(1, dtype=torch.int64)
        s.update(q=_normal((tq, h, d), g, dt), k=_normal((tk, hk, d), g, dt), v=_normal((tk, hk, d), g, dt),
                 cu_q=torch.cat([zero, lens.cumsum(0)]).to(torch.int32).cuda(), cu_k=torch.cat([zero, klens.cumsum(0)]).to(torch.int32).cuda(),
                 out=torch.empty((tq, h, d), dtype=dt, device="cuda"), max_q=int(lens.max()), max_k=int(klens.max()))
        return s
    # pages that hold keys of other tokens as well: [page][kv head][token][d]
    s.update(table=table.cuda(), n_pages=n_pages, kc=_normal((n_pages, hk, ps, d), g, dt), vc=_normal((n_pages, hk, ps, d), g, dt))
    return s


# -------------------------------------------------------------------------------------------- plain form
def _rotate(x, cos, sin, rd, layout):
    """x [m, heads, d] fp32; cos, sin [m, 1, rd/2]."""
    r, rest = x[..., :rd], x[..., rd:]
    a, b = (r[..., :rd // 2], r[..., rd // 2:]) if layout == HALF else (r[..., 0::2], r[..., 1::2])
    p, q = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.cat([p, q], -1) if layout == HALF else torch.stack([p, q], -1).flatten(-2), rest], -1)


def _append_plain(s):
    c = s["case"]
    h, hk, d, ps = c["h"], c["hk"], c["d"], c["ps"]
    m = s["x"].shape[0]
    x = s["x"].float().view(m, h + 2 * hk, d)
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    if s["q_norm"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["k_norm"]
    angle = s["pos"].double()[:, None] * s["freq"][None, :]
    cos, sin = (s["mscale"] * angle.cos()).float()[:, None, :], (s["mscale"] * angle.sin()).float()[:, None, :]
    s["q"].copy_(_rotate(q, cos, sin, c["rd"], c["layout"]))
    page = s["table"][s["row"].long(), (s["pos"] // ps).long()].long()
    off = (s["pos"] % ps).long()
    s["kc"][page, :, off] = _rotate(k, cos, sin, c["rd"], c["layout"]).to(s["kc"].dtype)
    s["vc"][page, :, off] = v.to(s["vc"].dtype)
    return [s["q"], s["kc"], s["vc"]]


def _gather(cache, table):
    """[rows, pages] -> fp32 [rows, kv heads, keys, d]."""
    x = cache[table.clamp(min=0).long()].float()
    r, p, hk, ps, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(r, hk, p * ps, d)


def _paged_plain(s):
    """Scores of the shared keys once for all queries, of each row's own keys by row; one softmax over both."""
    c = s["case"]
    h, hk, d, qg, rows, pre = c["h"], c["hk"], c["d"], c["qg"], c["rows"], c.get("prefix", 0)
    q = s["q"].float().view(rows, qg, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(rows, hk, -1, d) / math.sqrt(d)
    pos = s["pos"].view(rows, qg)
    n_pre = pre // c["ps"]
    k, v = _gather(s["kc"], s["table"][:, n_pre:]), _gather(s["vc"], s["table"][:, n_pre:])
    ok = (torch.arange(k.shape[2], device="cuda")[None, None, :] + pre <= pos[:, :, None]).repeat_interleave(h // hk, 1)[:, None]
    sc = (q @ k.transpose(2, 3)).masked_fill_(~ok, float("-inf"))
    if pre:
        pk, pv = _gather(s["kc"], s["table"][:1, :n_pre])[0], _gather(s["vc"], s["table"][:1, :n_pre])[0]
        n = q.shape[2]
        qa = q.transpose(0, 1).reshape(hk, rows * n, d)
        sp = (qa @ pk.transpose(1, 2)).view(hk, rows, n, pre).transpose(0, 1)
        top = torch.maximum(sc.amax(-1, keepdim=True), sp.amax(-1, keepdim=True))
        sc, sp = torch.exp(sc - top), torch.exp(sp - top)
        o = sc @ v + (sp.transpose(0, 1).reshape(hk, rows * n, pre) @ pv).view(hk, rows, n, d).transpose(0, 1)
        o = o / (sc.sum(-1, keepdim=True) + sp.sum(-1, keepdim=True))
    else:
        sc = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = (sc @ v) / sc.sum(-1, keepdim=True)
    o = o.view(rows, hk, qg, h // hk, d).permute(0, 2, 1, 3, 4).reshape(rows * qg, h, d)
    return [o.to(s["q"].dtype)]


def _packed_plain(s):
    """Sequences padded to the longest: [sequence, kv head, query, group head, key] scores."""
    c = s["case"]
    h, hk, d = c["h"], c["hk"], c["d"]
    cq, ck = s["cu_q"].long(), s["cu_k"].long()
    lq, lk = cq[1:] - cq[:-1], ck[1:] - ck[:-1]
    iq, ik = torch.arange(s["max_q"], device="cuda"), torch.arange(s["max_k"], device="cuda")
    at_q = (cq[:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)
    at_k = (ck[:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    q = s["q"].float()[at_q].view(-1, s["max_q"], hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(-1, hk, (h // hk) * s["max_q"], d)
    k, v = s["k"].float()[at_k].permute(0, 2, 1, 3), s["v"].float()[at_k].permute(0, 2, 1, 3)
    sc = ((q / math.sqrt(d)) @ k.transpose(2, 3)).view(-1, hk, h // hk, s["max_q"], s["max_k"])
    seen = (ik[None, None, :] <= (lk - lq)[:, None, None] + iq[None, :, None])[:, None, None]
    sc.masked_fill_(~seen, float("-inf"))
    sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    total = sc.sum(-1, keepdim=True)
    o = (sc.view(-1, hk, (h // hk) * s["max_q"], s["max_k"]) @ v).view(-1, hk, h // hk, s["max_q"], d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, s["max_q"], h, d)
    return [o[iq[None, :] < lq[:, None]].to(s["q"].dtype)]


# ---------------------------------------------------------------------------------------- framework's form
def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _bind(s):
    """The library call of this state, bound once: descriptor, workspace and arguments, as a program keeps them."""
    from mlxcat_b200 import _abi as A

    lib, c = A.lib(), s["case"]
    h, hk, d = c["h"], c["hk"], c["d"]
    s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    err = _ptr(s["err"])
    if c["op"] == "packed":
        return lib.mlxcat_op_packed_attention, (
            _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), CODE[c["dt"]], h * d, hk * d, hk * d, s["q"].shape[0], s["k"].shape[0],
            _ptr(s["cu_q"]), _ptr(s["cu_k"]), c["n"], 1, h, hk, d, 0.0, _ptr(s["out"]), err, stream), [s["out"]]
    ps = c["ps"]
    kv = A.PagedKVC(s["kc"].data_ptr(), s["vc"].data_ptr(), s["table"].data_ptr(), hk * ps * d, ps * d, d, CODE[c["dt"]], s["n_pages"],
                    ps, hk, d, s["table"].shape[0], s["table"].shape[1])
    s["kv"] = kv
    m = s["row"].shape[0]
    if c["op"] == "append":
        rope = A.RopeC()
        sc = A.RopeScalingC(SCALING[c["scaling"]], 32768 if c["scaling"] == "yarn" else 8192, 8.0, 1.0, 4.0, 32.0, 1.0, 0.0)
        A.check(lib.mlxcat_rope_init(ctypes.byref(rope), c["rd"], c["layout"], c["theta"], ctypes.byref(sc)))
        s["rope"] = rope
        x = s["x"]
        step, n = x.element_size(), x.shape[1]
        part = [ctypes.c_void_p(x.data_ptr() + o * d * step) for o in (0, h, h + hk)]
        return lib.mlxcat_op_rope_append, (
            ctypes.byref(kv), ctypes.byref(rope), part[0], part[1], part[2], CODE[c["src"]], n, n, n, m, h, _ptr(s["q_norm"]),
            _ptr(s["k_norm"]), 1e-6, _ptr(s["row"]), _ptr(s["pos"]), _ptr(s["q"]), err, stream), [s["q"], s["kc"], s["vc"]]
    if c["op"] == "paged":
        size = lib.mlxcat_op_paged_attention_workspace(m, c["qg"], h, hk, d)
        s["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        return lib.mlxcat_op_paged_attention, (
            ctypes.byref(kv), _ptr(s["q"]), m, c["qg"], h, 0.0, _ptr(s["row"]), _ptr(s["pos"]), _ptr(s["out"]), _ptr(s["ws"]), size, err,
            stream), [s["out"]]
    size = lib.mlxcat_op_shared_prefix_attention_workspace(m, c["qg"], h, hk, d, c["prefix"])
    s["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return lib.mlxcat_op_shared_prefix_attention, (
        ctypes.byref(kv), c["prefix"], _ptr(s["q"]), m, c["qg"], h, 0.0, _ptr(s["row"]), _ptr(s["pos"]), _ptr(s["out"]), _ptr(s["ws"]), size,
        err, stream), [s["out"]]


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _bind(state)
        f, args, out = state["call"]
        if f(*args) != 0:
            from mlxcat_b200 import _abi as A

            raise RuntimeError(A.lib().mlxcat_op_last_error().decode())
        return out
    return {"append": _append_plain, "paged": _paged_plain, "shared": _paged_plain, "packed": _packed_plain}[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------------------- work
def work(case):
    h, hk, d = case["h"], case["hk"], case["d"]
    if case["op"] == "append":
        n = case["rows"] * case["t"] * (h + 2 * hk) * d
        return {"bytes": n * ((4 if case["src"] == "f32" else 2) + 2), "flops": 6 * n}
    lens, past = (x.tolist() for x in _lengths(case))
    if case["op"] == "packed":
        pairs = sum(x * p + x * (x + 1) // 2 for x, p in zip(lens, past))
        return {"bytes": sum(lens) * 2 * h * d * 2 + (sum(lens) + sum(past)) * 2 * hk * d * 2, "flops": 4 * h * d * pairs}
    qg, pre = case["qg"], case.get("prefix", 0)
    keys = sum(x + qg - 1 for x in lens)
    pairs = sum(qg * pre + qg * x + qg * (qg - 1) // 2 for x in lens)
    return {"bytes": (keys + pre) * 2 * hk * d * 2 + 2 * len(lens) * qg * h * d * 2, "flops": 4 * h * d * pairs}


# -------------------------------------------------------------------------------------------------- exact
def _exact_append(case, s):
    h, hk, d, ps, rd = case["h"], case["hk"], case["d"], case["ps"], case["rd"]
    m = s["x"].shape[0]
    x = s["x"].double().view(m, h + 2 * hk, d).clone()
    if case["norm"]:
        w = torch.cat([s["q_norm"].double().expand(h, d), s["k_norm"].double().expand(hk, d)])
        y = x[:, :h + hk]
        x[:, :h + hk] = y / ((y ** 2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * w
    z = torch.arange(rd // 2, device="cuda")
    ia, ib = (z, z + rd // 2) if case["layout"] == HALF else (2 * z, 2 * z + 1)
    w = torch.polar(torch.full((m, 1, rd // 2), s["mscale"], dtype=torch.float64, device="cuda"),
                    (s["pos"].double()[:, None] * s["freq"])[:, None, :])
    turned = torch.complex(x[:, :h + hk, ia], x[:, :h + hk, ib]) * w
    x[:, :h + hk, ia], x[:, :h + hk, ib] = turned.real, turned.imag
    kc, vc = s["kc"].double(), s["vc"].double()
    slot = s["table"][s["row"].long(), (s["pos"] // ps).long()].long() * ps + (s["pos"] % ps).long()
    kc = kc.transpose(1, 2).reshape(-1, hk, d).index_copy(0, slot, x[:, h:h + hk]).view(-1, ps, hk, d).transpose(1, 2)
    vc = vc.transpose(1, 2).reshape(-1, hk, d).index_copy(0, slot, x[:, h + hk:]).view(-1, ps, hk, d).transpose(1, 2)
    return [x[:, :h].contiguous(), kc.contiguous(), vc.contiguous()]


def _exact_attend(q, k, v, limit):
    """q [n, h, d], k, v [keys, hk, d], limit [n]: keys 0..limit; 64 bits."""
    n, h, d = q.shape
    hk = k.shape[1]
    hidden = torch.arange(k.shape[0], device="cuda")[None, None, None, :] > limit[:, None, None, None]
    sc = torch.einsum("nigd,kid->nigk", q.double().view(n, hk, h // hk, d), k.double()) / math.sqrt(d)
    return torch.einsum("nigk,kid->nigd", torch.softmax(sc.masked_fill(hidden, float("-inf")), -1), v.double()).reshape(n, h, d)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    out = []
    if case["op"] == "packed":
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        for i in range(case["n"]):
            nq, nk = cq[i + 1] - cq[i], ck[i + 1] - ck[i]
            for a in range(0, nq, 1024):
                b = min(nq, a + 1024)
                seen = nk - nq + b
                out.append(_exact_attend(s["q"][cq[i] + a:cq[i] + b], s["k"][ck[i]:ck[i] + seen], s["v"][ck[i]:ck[i] + seen],
                                         torch.arange(nk - nq + a, seen, device="cuda")))
        return [torch.cat(out)]
    qg, ps = case["qg"], case["ps"]
    for r in range(case["rows"]):
        n = int(s["lens"][r])
        pages = s["table"][r, :(n + ps - 1) // ps].long()
        k, v = (x[pages].transpose(1, 2).reshape(-1, case["hk"], case["d"])[:n] for x in (s["kc"], s["vc"]))
        out.append(_exact_attend(s["q"][r * qg:(r + 1) * qg], k, v, s["pos"][r * qg:(r + 1) * qg].long()))
    return [torch.cat(out)]
