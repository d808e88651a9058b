"""Workloads of the key/value-cache operators: rotary positions with several axes, the quantised cache's write and
read back, attention of new tokens over the cache, and the same attention for a batch that shares a prefix.

`run` computes a case in plain torch operations (32 bits, rounded once to the output type), or, with `own` set, by
the calls a program makes of the package's operators. `exact` restates every definition in 64 bits.

Shapes: 20 query heads on 5 key/value heads of 128 is the BitVLA decoder, 25 heads its stacked query and key heads,
288 tokens one of its prompts (256 image tokens and 32 text tokens), 8 its batch and 64 its request queue; 32 heads on
8 is a generic decoder shape.
"""
import math
import os
import random
import sys

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
CODE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"i8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -100  # the smallest absolute maximum a scale is made from


def _kv():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "robot.cpp_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from b2s import kv
    return kv


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of 8 sequences: the new tokens' query and key heads, time/height/width positions
        {"name": "rope_step", "op": "rope", "type": "f32", "rows": 8, "heads": 25, "hd": 128, "sections": "24,20,20",
         "interleaved": True, "far": 4096},
        # the prompts of many requests at once, in bf16
        {"name": "rope_prompt", "op": "rope", "type": "bf16", "rows": 16384, "heads": 25, "hd": 128,
         "sections": "16,24,24", "interleaved": False, "far": 32768},
        # the new tokens of 8 sequences written into the cache
        {"name": "write_step", "op": "write", "type": "f32", "code": "i8", "rows": 8, "kv_heads": 5, "hd": 128,
         "page": 64, "padded": 0},
        # 64 prompts of 288 tokens written at once
        {"name": "write_prompt", "op": "write", "type": "bf16", "code": "e4m3", "rows": 18432, "kv_heads": 5, "hd": 128,
         "page": 64, "padded": 100},
        # one prompt read back to continue it elsewhere (an odd length)
        {"name": "read_prompt", "op": "read", "type": "f32", "code": "i8", "rows": 289, "kv_heads": 5, "hd": 128,
         "page": 64, "padded": 0},
        # a whole long context read back in bf16
        {"name": "read_long", "op": "read", "type": "bf16", "code": "e4m3", "rows": 65537, "kv_heads": 8, "hd": 128,
         "page": 128, "padded": 0},
        # the smallest call: one token of one sequence, one prompt long
        {"name": "attn_one", "op": "attn", "type": "f32", "code": "i8", "batch": 1, "new": 1, "ragged": False,
         "len": 317, "heads": 20, "kv_heads": 5, "hd": 128, "page": 64, "causal": True},
        # one decoding step of 64 sequences of uneven lengths
        {"name": "attn_step", "op": "attn", "type": "f32", "code": "i8", "batch": 64, "new": 1, "ragged": True,
         "len": 8192, "heads": 20, "kv_heads": 5, "hd": 128, "page": 64, "causal": True},
        # 8 prompts of the BitVLA decoder
        {"name": "attn_prompt", "op": "attn", "type": "f32", "code": "i8", "batch": 8, "new": 288, "ragged": False,
         "len": 288, "heads": 20, "kv_heads": 5, "hd": 128, "page": 32, "causal": True},
        # long prompts taken in chunks onto a long cache
        {"name": "attn_chunk", "op": "attn", "type": "bf16", "code": "e4m3", "batch": 2, "new": 2048, "ragged": True,
         "len": 8192, "heads": 32, "kv_heads": 8, "hd": 128, "page": 128, "causal": True},
        # one step of 16 requests that share one prompt, few own tokens each
        {"name": "prefix_step", "op": "prefix", "type": "f32", "code": "i8", "batch": 16, "new": 1, "ragged": True,
         "len": 60, "prefix": 545, "heads": 20, "kv_heads": 5, "hd": 128, "page": 16, "causal": True},
        # one step of a large batch on a long shared document
        {"name": "prefix_wide", "op": "prefix", "type": "bf16", "code": "i8", "batch": 128, "new": 1, "ragged": True,
         "len": 300, "prefix": 16384, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "causal": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attn", "attn", "attn", "prefix", "prefix"])
    c = {"op": op, "type": rng.choice(["f32", "bf16"])}
    if op == "rope":
        c["hd"] = rng.choice([32, 64, 72, 80, 96, 128])
        c["heads"] = rng.randint(1, 25)
        c["rows"] = _log(rng, 1, 16384 if c["type"] == "bf16" else 8192)
        axes, half = rng.randint(1, 4), c["hd"] // 2
        cut = sorted(rng.sample(range(1, half), axes - 1))
        c["sections"] = ",".join(str(b - a) for a, b in zip([0] + cut, cut + [half]))
        c["interleaved"] = rng.random() < 0.5
        c["far"] = _log(rng, 16, 500000)
        return c
    c["code"] = rng.choice(["i8", "e4m3"])
    c["page"] = rng.choice([16, 32, 64, 128])
    c["hd"] = rng.choice([32, 64, 80, 96, 112, 128, 128, 128])
    c["kv_heads"] = rng.randint(1, 8)
    if op in ("write", "read"):
        c["rows"] = _log(rng, 1, 18000 if op == "write" else 30000)
        c["padded"] = rng.choice([0, 0, min(3, c["rows"] // 3)])
        return c
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    c["ragged"] = rng.random() < 0.7
    c["causal"] = rng.random() < 0.75
    shape = rng.choice(["step", "step", "draft", "prompt"])
    if op == "prefix":
        c["batch"], c["new"] = _log(rng, 1, 64), 1 if shape in ("step", "prompt") else rng.randint(2, 6)
        c["len"], c["prefix"] = _log(rng, 8, 300), _log(rng, 1, 8192)
    elif shape == "step":
        c["batch"], c["new"], c["len"] = _log(rng, 1, 48), 1, _log(rng, 1, 6000)
    elif shape == "draft":
        c["batch"], c["new"], c["len"] = _log(rng, 1, 32), rng.randint(2, 9), _log(rng, 10, 4000)
    else:
        c["new"] = _log(rng, 10, 1024)
        c["batch"] = max(1, min(8, 1500 // c["new"]))
        c["len"] = c["new"] + rng.choice([0, _log(rng, 1, 3000)])
    return c


def _lengths(case):
    """(new tokens, keys) of each sequence: from the case alone."""
    r = random.Random("%(batch)d %(new)d %(len)d" % case)
    n, L = [], []
    for _ in range(case["batch"]):
        L.append(r.randint(max(1, case["len"] // 8), case["len"]) if case["ragged"] else case["len"])
        n.append(r.randint(max(1, case["new"] // 2), case["new"]) if case["ragged"] else case["new"])
    L[0], n[0] = case["len"], case["new"]
    if case["op"] == "prefix":
        L = [max(a, b) for a, b in zip(n, L)]
    return n, L


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _pair_axis(case):
    """The axis of each rotated pair: blocks of the sections' sizes, or dealt in turn."""
    sec, half = _sections(case), case["hd"] // 2
    if not case["interleaved"]:
        return [a for a, n in enumerate(sec) for _ in range(n)]
    left, out = list(sec), []
    while len(out) < half:
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


# ------------------------------------------------------------------------------------------------ inputs
def _codes(g, code, shape):
    x = torch.randn(shape, generator=g, device="cuda")
    x.mul_(TOP[code] / 3.5)
    if code == "i8":
        return x.round_().clamp_(-127, 127).to(torch.int8)
    return x.clamp_(-448, 448).to(torch.float8_e4m3fn)


def _cache(g, case, pages):
    shape = (pages, case["kv_heads"], case["page"])
    st = {}
    for name, size in (("k", 1.0), ("v", 1.0)):
        st[name + "_codes"] = _codes(g, case["code"], shape + (case["hd"],))
        st[name + "_scale"] = (0.6 + 0.8 * torch.rand(shape, generator=g, device="cuda")) * (3.5 * size / TOP[case["code"]])
    return st


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    st = {"case": case}
    if case["op"] == "rope":
        sec = _sections(case)
        st["x"] = torch.randn((case["rows"], case["heads"] * case["hd"]), generator=g, device="cuda").to(DT[case["type"]])
        st["pos"] = torch.randint(0, case["far"], (case["rows"], len(sec)), generator=g, device="cuda", dtype=torch.int32)
        st["axis"] = torch.tensor(_pair_axis(case), device="cuda")
        st["y"] = torch.empty_like(st["x"])
        return st
    hd, ps, hkv = case["hd"], case["page"], case["kv_heads"]
    if case["op"] in ("write", "read"):
        rows = case["rows"]
        pages = -(-rows * 9 // (8 * ps))
        st.update(_cache(g, case, pages))
        slots = torch.randperm(pages * ps, generator=g, device="cuda")[:rows]
        if case["op"] == "write" or case["padded"]:
            slots = slots.sort().values if case["op"] == "write" else slots
        if case["padded"]:
            slots[torch.randperm(rows, generator=g, device="cuda")[:case["padded"]]] = -1
        st["slots"] = slots
        shape = (rows, hkv * hd)
        if case["op"] == "write":
            gain = torch.exp(0.5 * torch.randn((2, 1, shape[1]), generator=g, device="cuda"))  # channels of uneven size
            st["k"] = (torch.randn(shape, generator=g, device="cuda") * gain[0]).to(DT[case["type"]])
            st["v"] = (torch.randn(shape, generator=g, device="cuda") * gain[1]).to(DT[case["type"]])
        else:
            st["k"], st["v"] = (torch.empty(shape, dtype=DT[case["type"]], device="cuda") for _ in range(2))
        return st
    n, L = _lengths(case)
    need = [-(-x // ps) for x in L]
    pre = -(-case.get("prefix", 0) // ps)
    pool = sum(need) + pre
    st.update(_cache(g, case, pool + 3))
    order = torch.randperm(pool + 3, generator=cpu).to(torch.int32)
    table, at = torch.zeros((len(L), max(need)), dtype=torch.int32), pre
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    st["pages"] = table.cuda()
    st["prefix_pages"] = order[:pre].cuda()
    start = [0]
    for m in n:
        start.append(start[-1] + m)
    st["q_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    st["kv_len"] = torch.tensor(L, dtype=torch.int32, device="cuda")
    st["max_q"] = max(n)
    q = torch.randn((start[-1], case["heads"] * hd), generator=g, device="cuda") * 1.5
    st["q"] = q.to(DT[case["type"]])
    st["o"] = torch.zeros_like(st["q"])
    st["scale"] = 1.0 / math.sqrt(hd)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _rope(st):
    c, x = st["case"], st["x"]
    half = c["hd"] // 2
    inv = torch.pow(torch.tensor(500000.0, dtype=torch.float64, device=x.device),
                    torch.arange(half, dtype=torch.float64, device=x.device) * (-2.0 / c["hd"]))
    angle = st["pos"][:, st["axis"]].double() * inv
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    xs = x.float().view(-1, c["heads"], 2, half)
    a, b = xs[:, :, 0], xs[:, :, 1]
    y = torch.stack((a * cos - b * sin, a * sin + b * cos), 2)
    st["y"].copy_(y.view_as(x))
    return st["y"]


def _quantise(x, code, hkv, hd):
    """(codes as values, scale): one scale for each token and head; nothing finite is left of a head that is not."""
    x = x.float().view(-1, hkv, hd)
    big = x.abs().amax(-1)
    bad = ~torch.isfinite(big)
    big = torch.where(bad, torch.ones_like(big), big).clamp_min(TINY)
    top = torch.full_like(big, TOP[code])
    p = torch.where(bad[..., None], torch.zeros_like(x), x * (top / big)[..., None])
    scale = torch.where(bad, torch.full_like(big, math.nan), big / top)
    if code == "i8":  # halves go away from zero
        p = p.double()
        return (torch.sign(p) * torch.floor(p.abs() + 0.5)).clamp_(-127, 127), scale
    return p.clamp(-448, 448), scale


def _rows(st, slots):
    """The row of each (slot, head) in the cache's [pages * heads * page] rows."""
    c = st["case"]
    h = torch.arange(c["kv_heads"], device=slots.device)
    return ((slots // c["page"])[:, None] * c["kv_heads"] + h) * c["page"] + (slots % c["page"])[:, None]


def _write(st):
    c = st["case"]
    keep = (st["slots"] >= 0).nonzero()[:, 0]
    at = _rows(st, st["slots"][keep]).reshape(-1)
    for name in ("k", "v"):
        values, scale = _quantise(st[name][keep], c["code"], c["kv_heads"], c["hd"])
        codes = values.float().to(CODE[c["code"]]).view(torch.uint8)
        st[name + "_codes"].view(torch.uint8).view(-1, c["hd"])[at] = codes.reshape(-1, c["hd"])
        st[name + "_scale"].view(-1)[at] = scale.reshape(-1)
    return [st["k_codes"], st["k_scale"], st["v_codes"], st["v_scale"]]


def _read(st):
    c = st["case"]
    there = st["slots"] >= 0
    at = _rows(st, st["slots"].clamp_min(0))
    for name in ("k", "v"):
        codes = st[name + "_codes"].view(torch.uint8).view(-1, c["hd"])[at].view(CODE[c["code"]]).float()
        x = codes * st[name + "_scale"].view(-1)[at][..., None]
        st[name].copy_(torch.where(there[:, None, None], x, torch.zeros_like(x)).view_as(st[name]))
    return [st["k"], st["v"]]


def _gather(st, name, pages):
    """Keys or values of every page in the table, [batch, kv heads, tokens, hd] in 32 bits."""
    c = st["case"]
    b, p = pages.shape
    codes = st[name + "_codes"].view(torch.uint8)[pages.long()].view(CODE[c["code"]])
    x = codes.float() * st[name + "_scale"][pages.long()][..., None]
    return x.permute(0, 2, 1, 3, 4).reshape(b, c["kv_heads"], p * c["page"], c["hd"])


def _attend(st):
    c, q = st["case"], st["q"]
    hkv, group, hd = c["kv_heads"], c["heads"] // c["kv_heads"], c["hd"]
    start, n = st["q_start"][:-1].long(), (st["q_start"][1:] - st["q_start"][:-1]).long()
    b, i = n.numel(), torch.arange(st["max_q"], device=q.device)
    rows = (start[:, None] + i).clamp_max(q.shape[0] - 1)
    qs = q[rows].float().view(b, -1, hkv, group, hd).permute(0, 2, 3, 1, 4)  # [b, hkv, group, new, hd]
    qs = qs.reshape(b, hkv, group * i.numel(), hd)
    last = st["kv_len"].long()[:, None] - n[:, None] + i if c["causal"] else (st["kv_len"].long()[:, None] - 1 + 0 * i)
    s = qs @ _gather(st, "k", st["pages"]).transpose(-1, -2) * st["scale"]
    keys = torch.arange(s.shape[-1], device=q.device)
    seen = (keys <= last[..., None])[:, None, None]  # [b, 1, 1, new, keys]
    s = s.view(b, hkv, group, i.numel(), -1).masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    if c["op"] == "prefix":
        pk, pv = (_gather(st, x, st["prefix_pages"][None])[0, :, :c["prefix"]] for x in ("k", "v"))
        every = qs.transpose(0, 1).reshape(hkv, -1, hd)
        sp = (every @ pk.transpose(-1, -2) * st["scale"]).view(hkv, b, group, i.numel(), -1).transpose(0, 1)
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = (s - m).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hkv, group * i.numel(), -1) @ _gather(st, "v", st["pages"])).view(b, hkv, group, i.numel(), hd)
    if c["op"] == "prefix":
        p = (sp - m).exp_()
        total = total + p.sum(-1, keepdim=True)
        o = o + (p.transpose(0, 1).reshape(hkv, every.shape[1], -1) @ pv).view(hkv, b, group, i.numel(), hd).transpose(0, 1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(b, i.numel(), -1)
    mine = i < n[:, None]
    st["o"][rows[mine]] = o[mine].to(q.dtype)
    return st["o"]


def _run_own(st):
    c, op = st["case"], st["case"]["op"]
    kv = st.get("kv")
    if kv is None:  # what a program keeps from step to step: the cache's and the batch's handles, a workspace
        kv = st["kv"] = _kv()
        if op == "rope":
            st["sec"] = _sections(c)
        else:
            st["cache"] = kv.Cache(st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
        if op in ("attn", "prefix"):
            st["b"] = kv.Batch(st["q_start"], st["kv_len"], st["pages"], st["max_q"])
            size = kv.attention_workspace_size(st["cache"], st["b"], st["q"].shape[0], c["heads"], c.get("prefix", 0))
            st["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    if op == "rope":
        kv.rope_axes(st["x"], c["heads"], c["hd"], st["pos"], st["sec"], 500000.0, st["y"], c["interleaved"])
        return st["y"]
    if op == "write":
        kv.write(st["cache"], st["k"], st["v"], st["slots"])
        return [st["k_codes"], st["k_scale"], st["v_codes"], st["v_scale"]]
    if op == "read":
        kv.read(st["cache"], st["slots"], st["k"], st["v"])
        return [st["k"], st["v"]]
    if op == "attn":
        kv.attention(st["cache"], st["b"], st["q"], c["heads"], st["scale"], c["causal"], st["o"], st["ws"])
    else:
        kv.attention_prefix(st["cache"], st["b"], st["prefix_pages"], c["prefix"], st["q"], c["heads"], st["scale"],
                            c["causal"], st["o"], st["ws"])
    return st["o"]


def run(st):
    if own:
        return _run_own(st)
    return {"rope": _rope, "write": _write, "read": _read, "attn": _attend, "prefix": _attend}[st["case"]["op"]](st)


# ------------------------------------------------------------------------------------------------ work
def _pairs(n, L, causal):
    """Visible (query, key) pairs of a sequence."""
    return sum(max(0, min(L, L - n + i + 1)) for i in range(n)) if causal else n * L


def work(case):
    e = 4 if case["type"] == "f32" else 2
    if case["op"] == "rope":
        x = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 2 * x * e + 4 * case["rows"] * len(_sections(case)), "flops": 3 * x}
    token = case["kv_heads"] * (2 * case["hd"] + 8)  # codes and scales of one token's keys and values
    if case["op"] in ("write", "read"):
        m = case["rows"] - case["padded"]
        x = 2 * case["kv_heads"] * case["hd"]
        there = m if case["op"] == "write" else case["rows"]
        return {"bytes": m * token + there * x * e + 8 * case["rows"], "flops": 2 * m * x}
    n, L = _lengths(case)
    pre = case.get("prefix", 0)
    pairs = sum(_pairs(a, b, case["causal"]) + a * pre for a, b in zip(n, L))
    io = 2 * sum(n) * case["heads"] * case["hd"] * e + 4 * sum(-(-x // case["page"]) for x in L + [pre]) + 8 * len(L)
    return {"bytes": io + (sum(L) + pre) * token, "flops": 4 * pairs * case["heads"] * case["hd"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "rope":
        hd, half, sec = case["hd"], case["hd"] // 2, _sections(case)
        x = st["x"].to(f64).view(case["rows"], case["heads"], hd)
        y = torch.empty_like(x)
        axis = _pair_axis(case)
        for j in range(half):
            t = st["pos"][:, axis[j]].to(f64) / 500000.0 ** (2 * j / hd)
            z = torch.complex(x[:, :, j], x[:, :, half + j]) * torch.polar(torch.ones_like(t), t)[:, None]
            y[:, :, j], y[:, :, half + j] = z.real, z.imag
        return y.view(case["rows"], -1)
    hkv, hd, ps = case["kv_heads"], case["hd"], case["page"]
    if case["op"] == "write":
        out = []
        for name in ("k", "v"):
            # the codes are defined on the 32-bit product with the 32-bit quotient, so they are exact as they stand
            x = st[name].to(f64).view(-1, hkv, hd)
            big = x.abs().max(-1).values
            by = (TOP[case["code"]] / big).float().to(f64)
            p = (x * by[..., None]).float().to(f64)
            if case["code"] == "i8":
                p = torch.where(p < 0, (p - 0.5).ceil(), (p + 0.5).floor())
            codes, scale = st[name + "_codes"].clone(), st[name + "_scale"].to(f64)
            page, off = st["slots"] // ps, st["slots"] % ps
            on = st["slots"] >= 0
            codes.view(torch.uint8)[page[on], :, off[on]] = p[on].float().to(CODE[case["code"]]).view(torch.uint8)
            scale[page[on], :, off[on]] = (big / TOP[case["code"]])[on]
            out += [codes, scale]
        return out
    kx, vx = (st[n + "_codes"].float().to(f64) * st[n + "_scale"].to(f64)[..., None] for n in ("k", "v"))
    if case["op"] == "read":
        on = (st["slots"] >= 0)[:, None, None]
        return [torch.where(on, x[st["slots"] // ps, :, st["slots"] % ps], 0.0).reshape(case["rows"], -1) for x in (kx, vx)]
    n, L = _lengths(case)
    pre, group = case.get("prefix", 0), case["heads"] // hkv
    if sum(a * (b + pre) for a, b in zip(n, L)) * case["heads"] * hd > 2e11:
        return None
    tok = lambda x, pages, m: x[pages.long()].transpose(1, 2).reshape(-1, hkv, hd)[:m]  # noqa: E731
    out, at = torch.zeros(st["q"].shape, dtype=f64, device="cuda").view(-1, hkv, group, hd), 0
    shared = [tok(x, st["prefix_pages"], pre) for x in (kx, vx)] if pre else None
    for b in range(len(L)):
        pages = st["pages"][b, :-(-L[b] // ps)]
        k, v = (tok(x, pages, L[b]) for x in (kx, vx))
        if pre:
            k, v = torch.cat((shared[0], k)), torch.cat((shared[1], v))
        q = st["q"][at:at + n[b]].to(f64).view(-1, hkv, group, hd)
        for h in range(hkv):
            s = torch.einsum("igd,jd->igj", q[:, h], k[:, h]) * st["scale"]
            if case["causal"]:
                far = pre + L[b] - n[b] + torch.arange(n[b], device="cuda")
                s = s.masked_fill((torch.arange(pre + L[b], device="cuda") > far[:, None])[:, None], -math.inf)
            out[at:at + n[b], h] = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) @ v[:, h]
        at += n[b]
    return out.view(st["q"].shape)
