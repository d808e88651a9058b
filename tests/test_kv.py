"""The key/value cache operators (include/b2s_kv.h): refusals and host-side rules without a GPU; on a B200 every
operator against its definition in 64 bits.

Tolerances are derived, not fitted. u = 2^-24 is half a step of fp32, h the output type's (bf16 2^-8).
  rope:       the cosine, the sine and two products are rounded, then the sum: |err| <= 4 u (|a| + |b|), and h.
  write:      codes are defined on fp32 steps, so they are equal; a scale is one fp32 quotient.
  read:       one product, then h.
  attention:  a score's products carry 2^-22 (two fp16 parts) and the fp32 sum of hd of them, three products with
              scales follow: e_s = (2^-22 + (hd + 8) u) S, S = |scale| sum |q_d k_d|, plus u |s| for the argument of the
              exponential and 2^-21 for the exponential itself. Numerator and denominator each carry that, the
              probabilities' split 2^-22 (or 2^-11 where bf16 calls keep one fp16 part) and the fp32 sum of n keys n u:
              |err| <= (2 (e_s + 2^-21) + 2^-22 + 2 n u + 8 u) max |v|, and h.
"""
import ctypes as C
import math
import os
import re

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from b2s import B2SError  # noqa: E402
from b2s import kv  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
gpu = pytest.mark.gpu
F32, BF16, I8, E4M3 = torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn


# ------------------------------------------------------------------------------------------------ without a GPU
def test_exports_kv_symbols(b2s):
    src = open(os.path.join(ROOT, "include", "b2s_kv.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    decl = sorted(set(re.findall(r"\b(b2s_\w+)\s*\(", src)))
    lib = C.CDLL(b2s.LIB_PATH)
    assert decl and not [s for s in decl if not hasattr(lib, s)]
    assert sorted(kv.EXPORTED) == decl


P = 0x10000  # a 16-byte aligned address that no refused call follows


def cache_struct(**over):
    c = kv.CacheStruct(kv.TYPE_I8, 5, 128, 64, 100, P, P, P, P)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def batch_struct(**over):
    b = kv.BatchStruct(3, 4, P, P, P, 10, 10)
    for k, v in over.items():
        setattr(b, k, v)
    return b


INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3


@pytest.mark.parametrize("over,status", [
    ({"type": 0}, UNSUPPORTED), ({"k": None}, INVALID), ({"v_scale": None}, INVALID), ({"n_kv_heads": 0}, INVALID),
    ({"head_dim": 24}, UNSUPPORTED), ({"head_dim": 144}, UNSUPPORTED), ({"head_dim": -16}, INVALID),
    ({"page_size": 8}, UNSUPPORTED), ({"page_size": 48}, UNSUPPORTED), ({"page_size": 2048}, UNSUPPORTED),
    ({"n_pages": 0}, INVALID), ({"n_pages": 2 ** 31}, UNSUPPORTED), ({"k": P + 8}, UNSUPPORTED),
    ({"k_scale": P + 2}, UNSUPPORTED)])
def test_cache_refusals(b2s, over, status):
    L, c, b = kv._bind(), cache_struct(**over), batch_struct()
    assert L.b2s_kv_write(C.byref(c), 0, P, 640, P, 640, 4, P, None) == status
    assert L.b2s_kv_read(C.byref(c), P, 4, 0, P, 640, P, 640, None) == status
    assert L.b2s_attention_kv(C.byref(c), C.byref(b), 0, P, 2560, 4, 20, 1.0, 1, P, 2560, P, 1 << 40, None) == status
    assert L.b2s_attention_kv_workspace_size(C.byref(c), C.byref(b), 4, 20, 0) == 0
    assert b2s.last_error()


def test_null_structs_are_refused(b2s):
    L, c = kv._bind(), cache_struct()
    assert L.b2s_kv_write(None, 0, P, 640, P, 640, 4, P, None) == INVALID
    assert L.b2s_attention_kv(C.byref(c), None, 0, P, 2560, 4, 20, 1.0, 1, P, 2560, P, 1 << 40, None) == INVALID


@pytest.mark.parametrize("args,status", [
    (dict(type=1), UNSUPPORTED), (dict(k=None), INVALID), (dict(ldk=639), INVALID), (dict(ldv=642), UNSUPPORTED),
    (dict(v=P + 4), UNSUPPORTED), (dict(M=-1), INVALID), (dict(slots=None), INVALID)])
def test_write_refusals(b2s, args, status):
    d = dict(type=0, k=P, ldk=640, v=P, ldv=640, M=4, slots=P)
    d.update(args)
    c = cache_struct()
    assert kv._bind().b2s_kv_write(C.byref(c), d["type"], d["k"], d["ldk"], d["v"], d["ldv"], d["M"], d["slots"], None) == status


def test_read_refusals(b2s):
    L, c = kv._bind(), cache_struct()
    assert L.b2s_kv_read(C.byref(c), P, 4, 0, None, 0, None, 0, None) == INVALID
    assert L.b2s_kv_read(C.byref(c), None, 4, 0, P, 640, None, 0, None) == INVALID
    assert L.b2s_kv_read(C.byref(c), P, 4, 24, P, 640, None, 0, None) == UNSUPPORTED
    assert L.b2s_kv_read(C.byref(c), P, 4, 30, P, 644, None, 0, None) == UNSUPPORTED


@pytest.mark.parametrize("args,status", [
    (dict(type=24), UNSUPPORTED), (dict(heads=18), INVALID), (dict(heads=0), INVALID), (dict(q=None), INVALID),
    (dict(o=None), INVALID), (dict(ldq=2559), INVALID), (dict(ldo=2562), UNSUPPORTED), (dict(q=P + 8), UNSUPPORTED),
    (dict(M=-1), INVALID), (dict(M=2 ** 31), UNSUPPORTED), (dict(scale=math.nan), INVALID), (dict(ws=None), WORKSPACE),
    (dict(bytes=1000), WORKSPACE), (dict(ws=P + 128), WORKSPACE), (dict(prefix_len=-1), INVALID),
    (dict(prefix_len=2 ** 31), UNSUPPORTED), (dict(prefix_pages=None), INVALID),
    (dict(batch=batch_struct(batch=-1)), INVALID), (dict(batch=batch_struct(batch=20000)), UNSUPPORTED),
    (dict(batch=batch_struct(q_start=None)), INVALID), (dict(batch=batch_struct(kv_len=None)), INVALID),
    (dict(batch=batch_struct(pages=None)), INVALID), (dict(batch=batch_struct(ld_pages=9)), INVALID),
    (dict(batch=batch_struct(max_pages=2 ** 26, ld_pages=2 ** 26)), UNSUPPORTED), (dict(batch=batch_struct(max_q=-1)), INVALID)])
def test_attention_refusals(b2s, args, status):
    d = dict(type=0, q=P, ldq=2560, M=4, heads=20, scale=0.1, o=P, ldo=2560, ws=P, bytes=1 << 40, batch=batch_struct(),
             prefix_pages=P, prefix_len=100)
    d.update(args)
    L, c = kv._bind(), cache_struct()
    call = (d["type"], d["q"], d["ldq"], d["M"], d["heads"], d["scale"], 1, d["o"], d["ldo"], d["ws"], d["bytes"], None)
    assert L.b2s_attention_kv_prefix(C.byref(c), C.byref(d["batch"]), d["prefix_pages"], d["prefix_len"], *call) == status
    if not any(k.startswith("prefix") for k in args):
        assert L.b2s_attention_kv(C.byref(c), C.byref(d["batch"]), *call) == status
    assert b2s.last_error()


@pytest.mark.parametrize("args,status", [
    (dict(type=24), UNSUPPORTED), (dict(hd=127), INVALID), (dict(hd=258, sec=[129]), UNSUPPORTED), (dict(heads=0), INVALID),
    (dict(ldx=100), INVALID), (dict(ldy=100), INVALID), (dict(sec=[32, 31]), INVALID), (dict(sec=[65, -1]), INVALID),
    (dict(sec=[]), INVALID), (dict(sec=[16, 16, 16, 8, 8]), INVALID), (dict(theta=0.0), INVALID),
    (dict(theta=math.inf), INVALID), (dict(x=None), INVALID), (dict(pos=None), INVALID), (dict(x=P + 2), UNSUPPORTED),
    (dict(M=-1), INVALID), (dict(ldpos=1, sec=[32, 32]), INVALID), (dict(y=P, ldy=2600), INVALID)])
def test_rope_refusals(b2s, args, status):
    d = dict(type=0, x=P, ldx=2560, M=4, heads=20, hd=128, pos=P, sec=[64], theta=1e4, y=2 * P, ldy=2560, ldpos=8)
    d.update(args)
    n = len(d["sec"])
    assert kv._bind().b2s_rope_axes(d["type"], d["x"], d["ldx"], d["M"], d["heads"], d["hd"], d["pos"], d["ldpos"], n,
                                    (C.c_int32 * max(n, 1))(*d["sec"]), 0, d["theta"], d["y"], d["ldy"], None) == status


def test_workspace_grows_with_the_prefix(b2s):
    c, b = cache_struct(), batch_struct(batch=64, max_q=1)
    size = kv._bind().b2s_attention_kv_workspace_size
    plain, shared = size(C.byref(c), C.byref(b), 64, 20, 0), size(C.byref(c), C.byref(b), 64, 20, 100000)
    assert plain > 0 and shared >= plain + 64 * 20 * 130 * 4 and shared % 256 == 0


@pytest.mark.parametrize("scale", [math.inf, -math.inf, 2.0 ** 127, -3e38])
def test_scales_without_room_are_refused(b2s, scale):
    c, b = cache_struct(), batch_struct()
    assert kv._bind().b2s_attention_kv(C.byref(c), C.byref(b), 0, P, 2560, 4, 20, scale, 1, P, 2560, P, 1 << 40, None) == INVALID
    assert "scale" in b2s.last_error()


@pytest.mark.parametrize("M,batch,max_q,heads,prefix", [
    (0, 3, 1000, 20, 5000), (0, 0, 0, 20, 0), (0, 16384, 2 ** 31 - 1, 2 ** 31 - 8, 2 ** 20), (7, 1, 2 ** 31 - 1, 20, 2 ** 20),
    (7, 16384, 0, 20, 2 ** 20), (2 ** 24, 1, 2 ** 24, 20, 2 ** 20)])
def test_workspace_of_unusual_batches(b2s, M, batch, max_q, heads, prefix):
    c, b = cache_struct(), batch_struct(batch=batch, max_q=max_q)
    heads -= heads % 5
    size = kv._bind().b2s_attention_kv_workspace_size(C.byref(c), C.byref(b), M, heads, prefix)
    assert size > 0 and size <= 2 ** 24 + 33 * (M + 1) * heads * 130 * 4


def test_binding_refuses_host_tensors_and_shapes(b2s):
    x = torch.zeros(4, 640)
    with pytest.raises(ValueError, match="CUDA"):
        kv._rows(x, 640, "x", 0)
    with pytest.raises(ValueError, match="CUDA"):
        kv._ints(torch.zeros(4, dtype=torch.int64), torch.int64, (4,), "slots", 0)
    with pytest.raises(ValueError, match="codes"):
        kv.Cache(x, x, x, x)
    k, s = torch.zeros(2, 5, 16, 64, dtype=torch.int8), torch.zeros(2, 5, 16)
    kv.Cache(k, k, s, s)
    with pytest.raises(ValueError, match="v_scale"):
        kv.Cache(k, k, s, s.double())
    with pytest.raises(ValueError, match="k_scale"):
        kv.Cache(k, k, s[:1], s)


# ------------------------------------------------------------------------------------------------ on a B200
def ok(b2s, bits=0):
    torch.cuda.synchronize()
    assert b2s.device_error() == bits


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def pair_axes(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def rope_ref(x, heads, hd, pos, sections, theta, interleaved):
    half = hd // 2
    axis = torch.tensor(pair_axes(sections, interleaved), device="cuda")
    inv = torch.tensor([theta ** (-2.0 * i / hd) for i in range(half)], dtype=torch.float64, device="cuda")
    t = (pos.double()[:, axis] * inv)[:, None]
    xs = x.double().view(x.shape[0], heads, 2, half)
    a, b = xs[:, :, 0], xs[:, :, 1]
    y = torch.stack((a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()), 2)
    return y.view(x.shape), (a.abs() + b.abs())[:, :, None].expand(-1, -1, 2, -1).reshape(x.shape)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,heads,hd,sections,inter", [
    (1, 1, 2, [1], False), (5, 3, 72, [36], False), (8, 25, 128, [24, 20, 20], True), (7, 25, 128, [16, 24, 24], False),
    (3, 2, 80, [10, 10, 10, 10], True), (300, 4, 64, [32, 0], True), (2, 3, 256, [0, 100, 28], True), (1201, 5, 32, [5, 11], False)])
def test_rope_axes(b2s, dtype, M, heads, hd, sections, inter):
    g = gen(M * heads + hd)
    pos = torch.randint(0, 100000, (M, len(sections)), generator=g, device="cuda", dtype=torch.int32)
    if M > 2:
        pos[0] = 0
        pos[1] = -17
        pos[2] = 2 ** 31 - 1
    x = randn(g, M, heads * hd, dtype=dtype)
    ref, mag = rope_ref(x, heads, hd, pos, sections, 500000.0, inter)
    # the angle pos * base^(-2i/hd) is a double: its own rounding is pos * 2^-52, which matters at 2^31
    slack = 4 * U * mag + HALF[dtype] * ref.abs() + pos.double().abs().amax() * 2.0 ** -51 * mag
    y = torch.full((M + 2, heads * hd), 7.0, dtype=dtype, device="cuda")
    kv.rope_axes(x, heads, hd, pos, sections, 500000.0, y[1:M + 1], inter)
    ok(b2s)
    assert bool(((y[1:M + 1].double() - ref).abs() <= slack).all())
    assert bool((y[0] == 7).all() and (y[M + 1] == 7).all())
    kv.rope_axes(x, heads, hd, pos, sections, 500000.0, x, inter)  # in place
    ok(b2s)
    assert torch.equal(x, y[1:M + 1])


@gpu
def test_rope_axes_strided_and_one_axis_is_rope_neox(b2s):
    g = gen(3)
    big = randn(g, 33, 1000)
    x = big[:, 5:5 + 6 * 128]  # rows that are aligned to one value only
    before = big.clone()
    pos = (torch.arange(33, device="cuda", dtype=torch.int32) + 40)[:, None].contiguous()
    y = torch.empty(33, 6 * 128, device="cuda")
    kv.rope_axes(x, 6, 128, pos, [64], 500000.0, y)
    ok(b2s)
    assert torch.equal(big, before)
    z = x.contiguous()
    b2s.rope_neox(z, 6, 128, 500000.0, 40)
    ok(b2s)
    assert float((y - z).abs().max()) <= 4 * U * float(x.abs().max()) * 2
    kv.rope_axes(torch.empty(0, 768, device="cuda"), 6, 128, torch.empty(0, 1, dtype=torch.int32, device="cuda"), [64], 1e4,
                 torch.empty(0, 768, device="cuda"))
    ok(b2s)


def quantise_ref(x, code, hkv, hd):
    """(codes as float64, scale as float32) by the definition; numpy on the host."""
    x = x.float().cpu().numpy().reshape(-1, hkv, hd)
    with np.errstate(all="ignore"):
        a = np.abs(x).max(-1)
        bad = ~np.isfinite(a)
        a = np.maximum(np.where(bad, np.float32(1), a), np.float32(2.0 ** -100)).astype(np.float32)
        top = np.float32(TOP[code])
        p = np.where(bad[..., None], np.float32(0), x * (top / a)[..., None]).astype(np.float32)
        scale = np.where(bad, np.float32(np.nan), a / top).astype(np.float32)
    if code == I8:
        p = p.astype(np.float64)
        return np.clip(np.sign(p) * np.floor(np.abs(p) + 0.5), -127, 127), scale
    return torch.from_numpy(p).clamp(-448, 448).to(E4M3).double().numpy(), scale


def row_index(cache, slots):
    ps = cache.page_size
    return slots // ps, slots % ps


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("M,hkv,hd,ps", [(1, 1, 16, 16), (9, 5, 128, 64), (130, 3, 80, 16), (77, 2, 48, 32), (513, 8, 64, 128),
                                         (33, 1, 112, 1024)])
def test_write_and_read(b2s, dtype, code, M, hkv, hd, ps):
    g = gen(M + hd)
    cache = kv.Cache.empty(-(-M // ps) + 2, hkv, ps, hd, code)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x2a)
    cache.k_scale.fill_(3.0)
    cache.v_scale.fill_(3.0)
    n = cache.n_pages * ps
    slots = torch.randperm(n, generator=g, device="cuda")[:M]
    wide = randn(g, M, 2 * hkv * hd + 16, dtype=dtype) * torch.exp(2 * randn(g, M, 1)).to(dtype)
    k, v = wide[:, :hkv * hd], wide[:, hkv * hd + 16:]
    k[0, :hd] = 0  # a head of zeros
    if M > 8:
        k[1, 0], v[2, 1], k[3, hd - 1] = math.nan, math.inf, -math.inf
        v[4, :hd] = 1e-30
        slots[5] = -1
        v[6, :hd] = torch.arange(hd, device="cuda").to(dtype) - hd // 2 + 0.5  # halves: ties
        v[6, 0] = 127.0 if hd < 250 else 0
    kv.write(cache, k, v, slots)
    ok(b2s)
    on = slots >= 0
    page, off = row_index(cache, slots[on])
    touched = torch.zeros(cache.n_pages, ps, dtype=torch.bool, device="cuda")
    touched[page, off] = True
    for x, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        rc, rs = quantise_ref(x[on], code, hkv, hd)
        assert np.array_equal(codes.float()[page, :, off].cpu().numpy().astype(np.float64), rc)
        assert np.array_equal(scales[page, :, off].cpu().numpy(), rs, equal_nan=True)
        rest = codes.view(torch.uint8).permute(0, 2, 1, 3)[~touched]
        assert bool((rest == 0x2a).all()) and bool((scales.permute(0, 2, 1)[~touched] == 3.0).all())
    # read back, a slot twice, into strided rows
    again = torch.cat((slots, slots[:1], torch.full((1,), -5, device="cuda")))
    out = torch.full((M + 3, 2 * hkv * hd + 32), 9.0, dtype=dtype, device="cuda")
    ko, vo = out[:M + 2, :hkv * hd], out[:M + 2, hkv * hd + 16:2 * hkv * hd + 16]
    kv.read(cache, again, ko, vo)
    ok(b2s)
    for o, codes, scales in ((ko, cache.k, cache.k_scale), (vo, cache.v, cache.v_scale)):
        p, f = row_index(cache, again.clamp_min(0))
        ref = (codes.double()[p, :, f] if code == I8 else codes.float().double()[p, :, f]) * scales.double()[p, :, f][..., None]
        ref = torch.where((again >= 0)[:, None, None], ref, 0.0).reshape(M + 2, -1)
        bad = ~torch.isfinite(ref)
        assert torch.equal(torch.isnan(o), torch.isnan(ref))
        err = (o.double() - ref).abs()
        assert bool((err <= U * ref.abs() + HALF[dtype] * ref.abs())[~bad].all())
    assert bool((out[M + 2] == 9).all() and (out[:, -16:] == 9).all())
    one = torch.empty(M + 2, hkv * hd, dtype=dtype, device="cuda")
    kv.read(cache, again, None, one)
    ok(b2s)
    assert torch.equal(one.nan_to_num(5.0), vo.nan_to_num(5.0))
    # a quantised value is within half a code of what was written
    fine = torch.isfinite(k.float()).view(M, hkv, hd).all(-1) & on[:, None]
    a = k.double().view(M, hkv, hd).abs().amax(-1)[fine]
    d = (ko[:M].double() - k.double()).view(M, hkv, hd)[fine].abs().amax(-1)
    # int8: half a step of a / 127; e4m3: half a step of the largest binade, 16 / 448 of a
    assert bool((d <= (0.5 / 127 if code == I8 else 16 / 448) * a * (1 + 1e-6) + HALF[dtype] * a + 2.0 ** -100).all())


@gpu
def test_bad_slots_are_left_out_and_reported(b2s):
    cache = kv.Cache.empty(2, 2, 16, 64)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        t.fill_(1)
    x = torch.ones(3, 128, device="cuda") * 5
    kv.write(cache, x, x, torch.tensor([32, 2 ** 40, 7], device="cuda"))
    ok(b2s, 4)
    assert int((cache.k != 1).sum()) == 128 and bool((cache.k[0, :, 7] == 127).all())
    out = torch.ones(2, 128, device="cuda")
    kv.read(cache, torch.tensor([32, 7], device="cuda"), out)
    ok(b2s, 4)
    assert bool((out[0] == 0).all()) and bool((out[1] == 5).all())


# ---- attention
class Case:
    """A random paged cache, batch and queries; reference and tolerance in 64 bits on the device."""

    def __init__(self, seed, new, keys, heads, hkv, hd, ps=16, dtype=F32, code=I8, causal=True, prefix=0, scale=None,
                 extra_rows=0, sharp=1.5, table=None):
        g, cpu = gen(seed), torch.Generator().manual_seed(seed)
        self.new, self.keys, self.heads, self.hkv, self.hd = new, keys, heads, hkv, hd
        self.dtype, self.causal, self.prefix = dtype, causal, prefix
        self.scale = 1 / math.sqrt(hd) if scale is None else scale
        need = [-(-x // ps) for x in keys]
        pre = -(-prefix // ps)
        n_pages = sum(need) + pre + 2
        codes = []
        for _ in range(2):
            x = torch.randn((n_pages, hkv, ps, hd), generator=g, device="cuda") * (TOP[code] / 3.5)
            codes.append(x.round().clamp(-127, 127).to(I8) if code == I8 else x.clamp(-448, 448).to(E4M3))
        scales = [(0.5 + torch.rand((n_pages, hkv, ps), generator=g, device="cuda")) * 3.5 / TOP[code] for _ in range(2)]
        self.cache = kv.Cache(*codes, *scales)
        order = torch.randperm(n_pages, generator=cpu).to(torch.int32)
        width = max(need + [1]) if table is None else table
        # entries behind a sequence's pages are never followed
        self.pages = torch.full((len(new), width), -7, dtype=torch.int32)
        at = pre
        for b, m in enumerate(need):
            self.pages[b, :m] = order[at:at + m]
            at += m
        self.pages = self.pages.cuda()
        self.prefix_pages = order[:pre].cuda()
        start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        self.q_start = torch.from_numpy(start).cuda()
        self.kv_len = torch.tensor(keys, dtype=torch.int32, device="cuda")
        self.rows = int(start[-1])
        self.q = (randn(g, self.rows + extra_rows, heads * hd) * sharp).to(dtype)
        self.batch = kv.Batch(self.q_start, self.kv_len, self.pages, max(list(new) + [0]))

    def workspace(self):
        n = kv.attention_workspace_size(self.cache, self.batch, self.q.shape[0], self.heads, self.prefix)
        assert n > 0
        return torch.empty(n, dtype=torch.uint8, device="cuda").fill_(0xff)

    def run(self, o=None, ws=None, q=None, stream=None):
        q = self.q if q is None else q
        o = torch.full_like(q, 7.0) if o is None else o
        ws = self.workspace() if ws is None else ws
        if self.prefix:
            kv.attention_prefix(self.cache, self.batch, self.prefix_pages, self.prefix, q, self.heads, self.scale,
                                self.causal, o, ws, stream)
        else:
            kv.attention(self.cache, self.batch, q, self.heads, self.scale, self.causal, o, ws, stream)
        return o

    def tokens(self, codes, scale, pages, n):
        x = codes.float().double() * scale.double()[..., None]
        return x[pages.long()].transpose(1, 2).reshape(-1, self.hkv, self.hd)[:n]

    def reference(self):
        """(o, tolerance) of rows [0, self.rows)."""
        c, G = self.cache, self.heads // self.hkv
        o = torch.zeros(self.rows, self.heads, self.hd, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(o)
        at = 0
        for b, (n, L) in enumerate(zip(self.new, self.keys)):
            if n == 0:
                continue
            pages = self.pages[b, :-(-L // c.page_size)]
            k, v = self.tokens(c.k, c.k_scale, pages, L), self.tokens(c.v, c.v_scale, pages, L)
            if self.prefix:
                k = torch.cat((self.tokens(c.k, c.k_scale, self.prefix_pages, self.prefix), k))
                v = torch.cat((self.tokens(c.v, c.v_scale, self.prefix_pages, self.prefix), v))
            k, v = (x.repeat_interleave(G, 1) for x in (k, v))
            q = self.q[at:at + n].double().view(n, self.heads, self.hd)
            s = torch.einsum("ihd,jhd->hij", q, k) * self.scale
            size = torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * abs(self.scale)
            j = torch.arange(k.shape[0], device="cuda")
            last = L - n + torch.arange(n, device="cuda") if self.causal else torch.full((n,), L - 1, device="cuda")
            last = self.prefix + last.clamp_min(-1)  # every row sees the whole prefix, more rows than own tokens or not
            seen = (j <= last[:, None])[None].expand_as(s)
            s = s.masked_fill(~seen, -math.inf)
            any_seen = seen.any(-1, keepdim=True)
            p = torch.where(any_seen, torch.softmax(s.masked_fill(~any_seen, 0.0), -1), 0.0)
            o[at:at + n] = torch.einsum("hij,jhd->ihd", p, v)
            if k.shape[0]:
                es = ((2.0 ** -22 + (self.hd + 8) * U) * size + U * s.abs()).masked_fill(~seen, 0.0).amax(-1)
                part = 2.0 ** -22 if self.dtype == F32 else 2.0 ** -11
                e = 2 * (es + 2.0 ** -21) + part + 2 * k.shape[0] * U + 8 * U
                tol[at:at + n] = e.transpose(0, 1)[..., None] * v.abs().amax(0)
            at += n
        tol += HALF[self.dtype] * (o.abs() + tol)
        return o.view(self.rows, -1), tol.view(self.rows, -1)

    def check(self, o):
        ref, tol = self.reference()
        err = (o[:self.rows].double() - ref).abs()
        worst = (err - tol).max() if err.numel() else -1
        assert bool((err <= tol).all()), f"worst excess {float(worst):.3g}, largest error {float(err.max()):.3g}"
        assert bool((o[self.rows:] == 7).all())


SHAPES = [
    # new, keys, heads, kv heads, hd
    ([1], [1], 1, 1, 16), ([1], [0], 4, 2, 64), ([1], [317], 20, 5, 128), ([1], [31], 8, 1, 128), ([1], [32], 5, 5, 96),
    ([1], [33], 6, 2, 80), ([2, 0, 1, 3], [5, 9, 0, 3], 4, 2, 48), ([4], [2], 8, 4, 32), ([7], [7], 3, 1, 112),
    ([1] * 9, [1, 15, 16, 17, 63, 64, 65, 700, 2], 20, 5, 128), ([3, 5, 1], [300, 40, 1000], 32, 4, 64),
    ([1], [4000], 2, 1, 128), ([9], [600], 20, 5, 128), ([40, 3], [40, 129], 8, 2, 128),
    ([288], [288], 20, 5, 128), ([130, 1, 0, 64], [513, 77, 12, 64], 16, 2, 128), ([65], [1000], 4, 4, 64),
    ([200], [150], 12, 1, 80)]


@gpu
@pytest.mark.parametrize("new,keys,heads,hkv,hd", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,code", [(F32, I8), (F32, E4M3), (BF16, I8), (BF16, E4M3)])
def test_attention(b2s, new, keys, heads, hkv, hd, causal, dtype, code):
    c = Case(len(new) + hd + sum(keys), new, keys, heads, hkv, hd, 16 if sum(keys) % 2 else 64, dtype, code, causal,
             extra_rows=3)
    o = c.run()
    ok(b2s)
    c.check(o)


@gpu
@pytest.mark.parametrize("new,keys,heads,hkv,hd,prefix", [
    ([1], [1], 4, 2, 64, 1), ([1], [0], 20, 5, 128, 317), ([1, 2, 0, 1], [5, 9, 4, 0], 8, 2, 48, 33),
    ([1] * 16, list(range(1, 17)), 20, 5, 128, 545), ([1] * 40, [30] * 40, 32, 8, 128, 1000), ([6], [3], 4, 1, 80, 16),
    ([100, 1, 30], [120, 5, 30], 16, 4, 128, 300)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,code", [(F32, I8), (BF16, E4M3)])
def test_attention_prefix(b2s, new, keys, heads, hkv, hd, prefix, causal, dtype, code):
    c = Case(hd + prefix, new, keys, heads, hkv, hd, 16, dtype, code, causal, prefix, extra_rows=2)
    o = c.run()
    ok(b2s)
    c.check(o)


@gpu
def test_attention_in_place_strided_and_repeatable(b2s):
    c = Case(5, [1, 3, 90, 1], [900, 40, 200, 5], 20, 5, 128)
    first = c.run()
    wide = torch.full((c.rows, 20 * 128 + 24), 3.0, device="cuda")
    wide[:, 8:8 + 2560] = c.q
    view = wide[:, 8:8 + 2560]
    c.run(o=view, q=view)
    ok(b2s)
    assert torch.equal(view, first) and bool((wide[:, :8] == 3).all() and (wide[:, 2568:] == 3).all())
    c.check(first)
    for _ in range(3):
        assert torch.equal(c.run(), first)


@gpu
def test_attention_sharp_scores_and_outlier_scales(b2s):
    """Large scores, a negative scale, value scales over 12 decades, and garbage behind the lengths."""
    for scale, code in ((0.9, I8), (-0.3, E4M3), (0.0, I8)):
        c = Case(11, [1, 70], [400, 130], 8, 2, 128, 32, F32, code, scale=scale)
        c.cache.v_scale.copy_(c.cache.v_scale * torch.pow(10.0, torch.randint(-6, 7, c.cache.v_scale.shape, generator=gen(1), device="cuda")))
        o = c.run()
        ok(b2s)
        c.check(o)
    c = Case(12, [1, 70], [400, 133], 8, 2, 128, 32)
    want = c.run()
    for b, n in enumerate(c.keys):  # what is behind a sequence's last token in its last page
        page, off = int(c.pages[b, (n - 1) // 32]), (n - 1) % 32 + 1
        c.cache.k_scale[page, :, off:] = math.nan
        c.cache.v_scale[page, :, off:] = math.inf
    assert torch.equal(c.run(), want)
    ok(b2s)


@gpu
@pytest.mark.parametrize("rows", [4, 90])
def test_attention_masked_tokens_may_be_nan(b2s, rows):
    """A token that is NaN or infinite reaches the rows that see it and no other."""
    c = Case(21, [rows], [rows + 50], 8, 2, 64, 16)
    bad = 50 + rows // 2
    want = c.run()
    for t, x in ((c.cache.k_scale, math.nan), (c.cache.v_scale, math.inf)):
        t[int(c.pages[0, bad // 16]), :, bad % 16] = x
    got = c.run()
    ok(b2s)
    sees = torch.arange(rows, device="cuda") >= rows // 2
    # a block's tiles, and with them the order of sums, are the same: rows before it are equal
    assert torch.equal(got[~sees], want[~sees])
    assert bool((~torch.isfinite(got[sees])).all())


@gpu
@pytest.mark.parametrize("new", [[1, 1, 1], [80, 1, 70]])
def test_bad_pages_and_lengths_are_left_out_and_reported(b2s, new):
    c = Case(31, new, [100, 64, 90], 8, 2, 64, 16, causal=False)
    for bad in (-1, 2 ** 30, c.cache.n_pages):
        pages = c.pages.clone()
        c.pages[1, 2] = bad
        got = c.run()
        ok(b2s, 4)
        # the reference without that page's 16 keys
        keep = torch.tensor([0, 1, 3], device="cuda")
        d = Case(31, new, [100, 48, 90], 8, 2, 64, 16, causal=False)
        d.cache, d.q = c.cache, c.q
        d.pages = pages.clone()
        d.pages[1, :3] = pages[1, keep]
        ref, tol = d.reference()
        assert bool(((got[:c.rows].double() - ref).abs() <= tol).all())
        c.pages.copy_(pages)
    c.kv_len[0] = 10 ** 6  # past the table: taken as its capacity
    c.pages.clamp_(0)
    got = c.run()
    ok(b2s, 4)
    c.keys = [c.pages.shape[1] * 16, 64, 90]
    c.check(got)
    c.kv_len[0] = -3
    got = c.run()
    ok(b2s, 4)
    c.keys = [0, 64, 90]
    c.check(got)
    c.kv_len[0] = 64
    c.keys = [64, 64, 90]
    c.q_start[3] = c.rows + 5  # rows that q does not have: the sequence is left out
    got = c.run()
    ok(b2s, 4)
    part = new[0] + new[1]
    ref, tol = c.reference()
    assert bool(((got.double() - ref).abs() <= tol)[:part].all()) and bool((got[part:] == 7).all())


@gpu
def test_attention_many_sequences_and_long_tables(b2s):
    """More sequences than a block has threads, most of them empty, behind a table much longer than they are."""
    g = np.random.default_rng(5)
    new = g.integers(0, 3, 700).tolist()
    keys = [int(x) if g.random() < 0.6 else 0 for x in g.integers(0, 90, 700)]
    c = Case(41, new, keys, 4, 2, 64, 16, table=300)
    o = c.run()
    ok(b2s)
    c.check(o)


@gpu
@pytest.mark.parametrize("prefix", [0, 200])
def test_attention_captured_replayed_and_on_two_streams(b2s, prefix):
    """Two captured calls with their own workspaces replayed together with lengths that changed after the capture."""
    a = Case(51, [1, 1, 2], [500, 30, 64], 20, 5, 128, prefix=prefix)
    b = Case(52, [80, 1], [300, 700], 20, 5, 128, prefix=prefix)
    runs, s = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for c, st in zip((a, b), s):
        ws, o = c.workspace(), torch.full_like(c.q, 7.0)
        with torch.cuda.stream(st):
            c.run(o, ws)
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            c.run(o, ws)
        runs.append((graph, o))
    a.kv_len[0] = 123
    a.keys[0] = 123
    torch.cuda.synchronize()
    for _ in range(3):
        for (graph, o), st in zip(runs, s):
            with torch.cuda.stream(st):
                graph.replay()
    ok(b2s)
    a.check(runs[0][1])
    b.check(runs[1][1])


LONG = [  # new, keys, heads, kv heads, hd: several row blocks, pairs of them (bf16), cut keys, odd tails
    ([300], [1500], 2, 2, 64), ([520, 3, 257], [3000, 40, 700], 8, 2, 128), ([1100], [1100], 4, 1, 112), ([65], [4096], 2, 1, 32),
    ([129], [130], 3, 3, 96), ([96, 1, 96], [2049, 2049, 127], 6, 1, 128)]


@gpu
@pytest.mark.parametrize("new,keys,heads,hkv,hd", LONG)
@pytest.mark.parametrize("dtype,code", [(F32, E4M3), (BF16, I8)])
def test_attention_many_rows_on_long_sequences(b2s, new, keys, heads, hkv, hd, dtype, code):
    c = Case(7 + hd + sum(keys), new, keys, heads, hkv, hd, 32, dtype, code, extra_rows=5)
    o = c.run()
    ok(b2s)
    c.check(o)
    assert torch.equal(c.run(), o)


@gpu
@pytest.mark.parametrize("rows", [1, 4, 40, 150])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("down", [False, True])
def test_attention_scores_that_grow_or_shrink_along_the_keys(b2s, rows, dtype, down):
    """Keys whose scales go over four decades along the sequence: the softmax reference is raised in most tiles, and with a
    shared prefix the two parts have far references."""
    for prefix in (0, 400):
        c = Case(91 + rows, [rows], [700], 8, 2, 128, 16, dtype, I8, prefix=prefix, scale=0.4)
        for pages, n in ((c.prefix_pages, prefix), (c.pages[0, :44], 700)):
            if n:
                ramp = torch.logspace(-3, 1, 16 * len(pages), device="cuda").view(-1, 1, 16)
                c.cache.k_scale[pages.long()] *= ramp.flip(0, 2) if down else ramp
                c.cache.v_scale[pages.long()] *= ramp.flip(0, 2)
        o = c.run()
        ok(b2s)
        c.check(o)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [5, 160])
def test_attention_rows_of_far_magnitudes(b2s, dtype, rows):
    """Query rows of one block over 60 decades: each keeps its own precision. Rows far above the rest have sharp scores."""
    for big in (1e4, 1e28):
        c = Case(93, [rows], [300], 8, 2, 64, 16, dtype, E4M3)
        by = torch.ones(rows, 1, device="cuda")
        by[::7] = big
        by[3::7] = 1 / big
        by[4::11] = 0.0
        c.q = (c.q.float() * by).to(dtype)
        o = c.run()
        ok(b2s)
        c.check(o)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("rows", [6, 160])
def test_attention_query_heads_that_are_not_finite(b2s, dtype, code, rows):
    """An infinity or a NaN makes its (row, head) NaN, whatever the signs of the keys, and no other one."""
    for prefix in (0, 70):
        c = Case(94, [rows], [rows + 20], 8, 2, 64, 16, dtype, code, prefix=prefix)
        c.cache.k.view(torch.uint8 if code == E4M3 else I8).bitwise_and_(0x7f)  # no negative keys: one infinity gives equal signs
        bad = [(0, 0, -math.inf), (2, 5, math.inf), (3, 7, math.nan), (rows - 1, 1, -math.inf)]
        clean = c.q.clone()
        for row, head, x in bad:
            c.q[row, head * 64 + 9] = x
        o = c.run()
        ok(b2s)
        o = o.view(rows, 8, 64)
        c.q = clean
        ref, tol = (x.view(rows, 8, 64) for x in c.reference())
        good = torch.ones(rows, 8, dtype=torch.bool, device="cuda")
        for row, head, _ in bad:
            good[row, head] = False
        assert bool(torch.isnan(o[~good]).all())
        assert bool(((o.double() - ref).abs() <= tol)[good].all())


@gpu
def test_attention_huge_and_tiny_queries_under_a_scale(b2s):
    for sharp, scale in ((1e30, 1e-31), (1e-30, 1e29)):
        for code in (I8, E4M3):
            c = Case(95, [2, 80], [200, 150], 4, 2, 128, 16, F32, code, scale=scale, sharp=sharp)
            o = c.run()
            ok(b2s)
            c.check(o)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_with_another_max_q(b2s, dtype):
    """max_q chooses kernels: too small or too large, the results stay within their bounds."""
    for prefix in (0, 90):
        c = Case(97, [1, 100, 0, 17], [30, 260, 5, 400], 12, 3, 128, 16, dtype, E4M3, prefix=prefix)
        for max_q in (0, 1, 17, 100, 5000):
            c.batch = kv.Batch(c.q_start, c.kv_len, c.pages, max_q)
            o = c.run()
            ok(b2s)
            c.check(o)


@gpu
@pytest.mark.parametrize("prefix", [4096, 4097])
def test_attention_prefix_on_both_sides_of_its_rule(b2s, prefix):
    """8 sequences x 8 heads x one block of rows x 128 steps is the last prefix that is read with the own tokens."""
    c = Case(99, [1, 2, 1, 1, 2, 1, 1, 1], [3, 40, 0, 17, 1, 9, 300, 64], 32, 8, 64, 64, F32, I8, prefix=prefix)
    o = c.run()
    ok(b2s)
    c.check(o)
    assert torch.equal(c.run(), o)


@gpu
@pytest.mark.parametrize("dtype,code,hd", [(F32, I8, 128), (BF16, E4M3, 128), (F32, E4M3, 80), (BF16, I8, 48)])
@pytest.mark.parametrize("prefix", [0, 40])
def test_attention_many_short_sequences(b2s, dtype, code, hd, prefix):
    """Units of few tiles that a warp takes alone: more of them than resident warps, several a warp, ragged, some empty."""
    g = np.random.default_rng(17)
    new = [int(x) for x in g.integers(0, 4, 900)]
    keys = [int(x) for x in g.integers(0, 66, 900)]
    c = Case(107, new, keys, 9, 3, hd, 16, dtype, code, prefix=prefix, extra_rows=3)
    o = c.run()
    ok(b2s)
    c.check(o)
    assert torch.equal(c.run(), o)


@gpu
def test_attention_graphs_that_share_a_workspace(b2s):
    """Two captured calls, of few rows and of many with cut keys, on one workspace, replayed in turn on one stream."""
    a = Case(101, [1, 1, 2], [900, 30, 64], 20, 5, 128)
    b = Case(102, [80, 1], [700, 900], 4, 1, 128, prefix=130)
    ws = torch.empty(max(a.workspace().numel(), b.workspace().numel()), dtype=torch.uint8, device="cuda").fill_(0xff)
    want, s, graphs = [c.run() for c in (a, b)], torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for c in (a, b):
        o = torch.empty_like(c.q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            c.run(o, ws)
        graphs.append((graph, o))
    with torch.cuda.stream(s):
        for graph, o in graphs * 3:
            graph.replay()
    ok(b2s)
    for (_, o), w in zip(graphs, want):
        assert torch.equal(o, w)


@gpu
def test_attention_of_a_large_batch_with_one_prompt(b2s):
    """The largest batch: single tokens, most without keys, and one prompt."""
    new, keys = [1] * 16384, [0] * 16384
    new[9000], keys[9000] = 90, 95
    for b in range(0, 16384, 37):
        keys[b] = 1 + b % 50
    c = Case(103, new, keys, 8, 1, 32, 16)
    o = c.run()
    ok(b2s)
    c.check(o)


@gpu
def test_long_cache_offsets_pass_32_bits(b2s):
    """Pages whose code rows lie past 2^32 bytes and whose scales lie past 2^31."""
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of device memory")
    pages, ps = 33_000, 1024  # 33.8e6 tokens of 128 bytes: 4.3e9 bytes each for keys and values
    cache = kv.Cache.empty(pages, 1, ps, 128)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        t.zero_()
    g, n = gen(61), 2000
    slots = torch.arange(n, device="cuda") + (pages - 2) * ps
    k, v = randn(g, n, 128), randn(g, n, 128)
    kv.write(cache, k, v, slots)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    kv.read(cache, slots, ko, vo)
    ok(b2s)
    assert float((ko - k).abs().max()) <= float(k.abs().max()) * 0.51 / 127
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device="cuda")
    for rows in (1, 100):
        q, o = randn(g, rows, 512), torch.empty(rows, 512, device="cuda")
        batch = kv.Batch(torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                         torch.tensor([n], dtype=torch.int32, device="cuda"), table, rows)
        ws = torch.empty(kv.attention_workspace_size(cache, batch, rows, 4), dtype=torch.uint8, device="cuda")
        kv.attention(cache, batch, q, 4, 0.1, False, o, ws)
        ok(b2s)
        p = torch.softmax(torch.einsum("ihd,jd->hij", q.double().view(rows, 4, 128), ko.double()) * 0.1, -1)
        ref = torch.einsum("hij,jd->ihd", p, vo.double()).reshape(rows, 512)
        # 2 n u of the sums leads the bound
        assert float((o.double() - ref).abs().max()) <= (2 * n * U + 2e-5) * float(vo.abs().max())


@gpu
@pytest.mark.parametrize("dtype,code", [(F32, I8), (BF16, E4M3)])
def test_decoding_with_the_cache(b2s, dtype, code):
    """The operators together, as a server uses them: two prompts behind a shared prefix are rotated, written and
    attended, then three tokens are decoded one by one; a 64-bit model of the same steps runs on what was read back."""
    heads, hkv, hd, ps, sections, theta = 8, 2, 64, 16, [16, 8, 8], 10000.0
    g = gen(71)
    prefix, lens, steps = 50, [37, 21], 3
    cache = kv.Cache.empty(20, hkv, ps, hd, code)
    order = torch.randperm(20, generator=torch.Generator().manual_seed(1))
    prefix_pages = order[:4].to(torch.int32).cuda()
    pages = order[4:12].view(2, 4).to(torch.int32).cuda()

    def slots_of(table, first, n):
        j = torch.arange(first, first + n, device="cuda")
        return table[j // ps].long() * ps + j % ps

    def tokens(n, first):
        x = randn(g, n, (heads + 2 * hkv) * hd, dtype=dtype)
        pos = torch.stack([torch.arange(first, first + n, device="cuda", dtype=torch.int32) // d for d in (1, 4, 9)], 1).contiguous()
        qk = x[:, :(heads + hkv) * hd]
        ref, mag = rope_ref(qk, heads + hkv, hd, pos, sections, theta, True)
        kv.rope_axes(qk, heads + hkv, hd, pos, sections, theta, qk, True)
        assert bool(((qk.double() - ref).abs() <= 4 * U * mag + HALF[dtype] * ref.abs()).all())
        return x[:, :heads * hd], x[:, heads * hd:(heads + hkv) * hd], x[:, (heads + hkv) * hd:]

    _, k, v = tokens(prefix, 0)
    kv.write(cache, k, v, slots_of(prefix_pages, 0, prefix))
    have = [0, 0]
    for step in range(1 + steps):
        n = lens if step == 0 else [1, 1]
        qs = []
        for b in range(2):
            q, k, v = tokens(n[b], prefix + have[b])
            kv.write(cache, k, v, slots_of(pages[b], have[b], n[b]))
            have[b] += n[b]
            qs.append(q)
        c = Case.__new__(Case)
        c.new, c.keys, c.heads, c.hkv, c.hd, c.dtype, c.causal, c.prefix = n, list(have), heads, hkv, hd, dtype, True, prefix
        c.scale, c.cache, c.pages, c.prefix_pages, c.rows, c.q = 0.125, cache, pages, prefix_pages, sum(n), torch.cat(qs)
        c.q_start = torch.tensor([0, n[0], sum(n)], dtype=torch.int32, device="cuda")
        c.kv_len = torch.tensor(have, dtype=torch.int32, device="cuda")
        c.batch = kv.Batch(c.q_start, c.kv_len, pages, max(n))
        o = c.run()
        ok(b2s)
        c.check(o)


@gpu
def test_binding_refusals_on_the_device(b2s):
    c = Case(81, [1], [20], 4, 2, 64)
    ws, o = c.workspace(), torch.empty_like(c.q)
    with pytest.raises(B2SError, match="workspace"):
        kv.attention(c.cache, c.batch, c.q, 4, 1.0, True, o, ws[:256])
    with pytest.raises(ValueError, match="o has dtype"):
        kv.attention(c.cache, c.batch, c.q, 4, 1.0, True, o.bfloat16(), ws)
    with pytest.raises(ValueError, match="slots"):
        kv.write(c.cache, torch.zeros(1, 128, device="cuda"), torch.zeros(1, 128, device="cuda"),
                 torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="prefix_pages"):
        kv.attention_prefix(c.cache, c.batch, c.pages[0, :1], 100, c.q, 4, 1.0, True, o, ws)
    with pytest.raises(ValueError, match="q_start"):
        kv.Batch(c.q_start.long(), c.kv_len, c.pages, 1)
    ok(b2s)
