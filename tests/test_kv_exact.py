"""The key/value cache attention against tighter bounds than test_kv.py's, whose `2 n u max |v|` grows with the keys while the
outputs shrink: here every weight has its own error and sums count their real depth, so that a probability held in too few
bits, a key left out or a key taken twice shows at any length.

u = 2^-24. A weight p_j = 2^(s_j - m) of a row carries
  e_j = (2^-22 + (t + 8) u) S_j + 8 u |s_j| + 2^-33 max |q| K_j,   S_j = |scale| sum |q_d k_jd|,   K_j = |scale| sum of |k_jd| where q_d is not 0,
for scores of t products (two fp16 parts of q: 2^-22 of the element or 2^-33 of the row's largest; fp32 sums; the factors'
roundings), 2 u (|s_j - s_max| + 8) / ln 2 for the argument of the exponential, 2^-21 for the exponential, 2^-22 for the
weight's own two parts. Those parts end at 2^-33 of the row's largest weight times its largest value scale (2^-32 next to a
reference that is a whole number above the largest score). Sums of n keys: products are added 16 at a time for each of the
two parts, each addition within 2^-23 (the tensor cores may cut off), 16 + n / 8 of them; the denominator 32 + n / 16 in u.
  |err| <= sum p_j |v_j| (e_j + D_N) + |o| (sum p_j e_j + D_D + 4 u) + 2^-32 sum_j max p * max vs * |code_j|
An output is then one rounding of what lies within that: o is between the rounded ends of the interval.
"""
import ctypes as C
import math
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from b2s import kv  # noqa: E402
from test_kv import BF16, E4M3, F32, HALF, I8, INVALID, U, UNSUPPORTED, Case, P, batch_struct, cache_struct, gen, gpu, ok, randn, rope_ref  # noqa: E402


def interval(c, products):
    """The ends of rows [0, c.rows) of the outputs in c's type, for scores of `products` nonzero products."""
    cache, G = c.cache, c.heads // c.hkv
    lo = torch.zeros(c.rows, c.heads, c.hd, dtype=torch.float64, device="cuda")
    hi = torch.zeros_like(lo)
    at = 0
    for b, (n, L) in enumerate(zip(c.new, c.keys)):
        def tokens(x):
            x = x.float().double()
            own = x[c.pages[b, :-(-L // cache.page_size)].long()].transpose(1, 2).reshape(-1, c.hkv, *x.shape[3:])[:L]
            if c.prefix:
                own = torch.cat((x[c.prefix_pages.long()].transpose(1, 2).reshape(-1, c.hkv, *x.shape[3:])[:c.prefix], own))
            return own
        k = tokens(cache.k) * tokens(cache.k_scale)[..., None]
        vc, vs = tokens(cache.v), tokens(cache.v_scale)
        q = c.q[at:at + n].double().view(n, c.hkv, G, c.hd)
        N = k.shape[0]
        last = L - n + torch.arange(n, device="cuda") if c.causal else torch.full((n,), L - 1, device="cuda")
        seen = (torch.arange(N, device="cuda") <= c.prefix + last.clamp_min(-1)[:, None])[:, None].expand(n, G, N)
        any_seen = seen.any(-1, keepdim=True)
        for h in range(c.hkv if n and N else 0):
            s = torch.einsum("igd,jd->igj", q[:, h], k[:, h]) * c.scale
            S = torch.einsum("igd,jd->igj", q[:, h].abs(), k[:, h].abs()) * abs(c.scale)
            K = abs(c.scale) * q[:, h].abs().amax(-1)[..., None] * ((q[:, h] != 0).double() @ k[:, h].abs().T)
            low = s.masked_fill(~seen, -math.inf)
            top = torch.where(any_seen, low.amax(-1, keepdim=True), 0.0)
            p = torch.where(seen, torch.exp(low - top), 0.0)
            total = torch.where(any_seen, p.sum(-1, keepdim=True), 1.0)
            p = p / total
            # up to 32 rows on int8 codes take a query as integers of 24 bits under its largest element
            low_q = U if cache.k.dtype == I8 and n * G <= 32 else 2.0 ** -33
            e = (2.0 ** -22 + (products + 8) * U) * S + 8 * U * s.abs() + low_q * K
            e = e + 2 * U * ((s - top).abs() + 8) / math.log(2) + 2.0 ** -21 + 2.0 ** -22
            e = torch.where(seen, e, 0.0)
            count = seen.sum(-1, keepdim=True).double()
            v = vc[:, h] * vs[:, h][:, None]
            o = p @ v
            most = torch.where(seen, vs[:, h].abs(), 0.0).amax(-1, keepdim=True) / total
            tol = (p * (e + (16 + count / 8) * 2.0 ** -23)) @ v.abs() + o.abs() * ((p * e).sum(-1, keepdim=True) + (36 + count / 16) * U)
            tol = 1.01 * (tol + 2.0 ** -32 * most * (seen.double() @ vc[:, h].abs())) + 1e-37
            tol = torch.where(any_seen, tol, 0.0)
            lo[at:at + n, h * G:(h + 1) * G], hi[at:at + n, h * G:(h + 1) * G] = o - tol, o + tol
        at += n
    return [x.view(c.rows, -1).float().to(c.dtype) for x in (lo, hi)]


def inside(c, o, products):
    lo, hi = interval(c, products)
    got = o[:c.rows]
    out = ~((got >= lo) & (got <= hi))
    where = out.nonzero()[0].tolist() if bool(out.any()) else None
    assert where is None, (f"{int(out.sum())} of {out.numel()} outputs, the first at {where}: {float(got[tuple(where)])!r} is not in "
                           f"[{float(lo[tuple(where)])!r}, {float(hi[tuple(where)])!r}]")
    assert bool((o[c.rows:] == 7).all())


def one_product(c, gain):
    """Queries with one nonzero element a head, of about `gain`, so that a score is one product and as good as exact."""
    g = gen(c.rows + c.heads)
    at = torch.randint(0, c.hd, (c.rows, c.heads, 1), generator=g, device="cuda")
    q = torch.zeros(c.rows, c.heads, c.hd, device="cuda")
    q.scatter_(2, at, gain * randn(g, c.rows, c.heads, 1))
    c.q = q.view(c.rows, -1).to(c.dtype)
    return c


MANY = [  # new, keys, heads, kv heads, hd, prefix: one row block and several, pairs of them (bf16), cut keys, both prefix forms
    ([90], [300], 2, 2, 64, 0), ([70, 3, 260], [70, 90, 700], 8, 2, 128, 0), ([1100], [1100], 4, 1, 112, 0),
    ([1] * 40, [30] * 40, 32, 8, 128, 1000), ([100, 1, 30], [120, 5, 30], 16, 4, 48, 300), ([1] * 9, [1, 15, 16, 17, 63, 64, 65, 700, 2], 20, 5, 128, 0)]


@gpu
@pytest.mark.parametrize("new,keys,heads,hkv,hd,prefix", MANY)
@pytest.mark.parametrize("dtype,code", [(BF16, E4M3), (BF16, I8), (F32, I8), (F32, E4M3)])
def test_outputs_are_one_rounding_of_the_exact_ones(b2s, new, keys, heads, hkv, hd, prefix, dtype, code):
    """Sharp scores that are single products: weights of a few keys, each held to 2^-22 whatever the type of the rows."""
    c = one_product(Case(3 + hd + sum(keys), new, keys, heads, hkv, hd, 16, dtype, code, True, prefix), 25.0)
    o = c.run()
    ok(b2s)
    inside(c, o, 1)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [8, 96, 300])
@pytest.mark.parametrize("down", [13.0, 18.0, 21.0])
def test_weights_far_below_the_largest_keep_their_bits(b2s, dtype, rows, down):
    """One token of value zero has all but 2^-down .. 2^-(down + 2) of each weight of the others: they alone make the output, and all
    are rounded alike, so that errors add up."""
    c = Case(113, [rows], [120], 1, 1, 64, 16, dtype, I8, False, scale=1.0)
    c.cache.k.zero_()
    c.cache.k_scale.fill_(1.0)
    c.cache.v.fill_(100)
    c.cache.v_scale.fill_(0.013)
    page = int(c.pages[0, 0])
    c.cache.k[page, :, 0, 5] = 16
    c.cache.v[page, :, 0] = 0
    c.q = torch.zeros(rows, 64, device="cuda")
    c.q[:, 5] = (down + torch.arange(rows, device="cuda") * (2.0 / rows)) * math.log(2) / 16
    c.q = c.q.to(dtype)
    o = c.run()
    ok(b2s)
    inside(c, o, 1)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [8, 64, 300])
@pytest.mark.parametrize("what", ["score", "value scale"])
def test_a_jump_along_the_keys_leaves_the_earlier_ones_their_weight(b2s, dtype, rows, what):
    """One token of value zero whose score lies 24 to 29 powers of two above the others', or whose value scale does: wherever it
    stands in a tile, the weights before it are taken under its reference, none is lost."""
    for at in (33, 40, 64, 95, 127, 128, 200, 330):
        for jump in (24, 27, 29):
            c = Case(117, [rows], [340], 1, 1, 64, 16, dtype, I8, False, scale=1.0)
            c.cache.k.zero_()
            c.cache.k_scale.fill_(1.0)
            c.cache.v.fill_(100)
            c.cache.v_scale.fill_(1.0)
            page, off = int(c.pages[0, at // 16]), at % 16
            c.cache.v[page, :, off] = 0
            c.q = torch.zeros(rows, 64, device="cuda")
            if what == "score":
                c.cache.k[page, :, off, 5] = 16
                c.q[:, 5] = jump * math.log(2) / 16
            else:
                c.cache.v_scale[page, :, off] = 2.0 ** jump
            c.q = c.q.to(dtype)
            o = c.run()
            ok(b2s)
            inside(c, o, 1)


@gpu
@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("rows", [6, 64, 200])
def test_a_query_row_keeps_its_bits_beside_a_larger_one(b2s, code, rows):
    """Rows 2^0 to 2^13 below the block's largest whose scores come from elements 2^-20 of their own largest one: even keys look at
    one of them, odd keys at another, so that the elements' own errors part their weights."""
    c = Case(121, [rows], [200], 2, 1, 64, 16, F32, code, False, scale=2.0 ** 21)
    k, v = torch.zeros(200, 64, device="cuda"), torch.full((200, 64), 96.0, device="cuda")
    k[0::2, 7], k[1::2, 8], v[1::2] = 96.0, 96.0, -96.0
    j = torch.arange(200, device="cuda")
    for to, x in ((c.cache.k, k), (c.cache.v, v)):
        to.view(torch.uint8)[c.pages[0, j // 16].long(), 0, j % 16] = x.to(code).view(torch.uint8)
    for t in (c.cache.k_scale, c.cache.v_scale):
        t.fill_(0.01)
    g = gen(122)
    q = torch.zeros(rows, 2, 64, device="cuda")
    q[:, :, 3] = 1.0 + torch.rand((rows, 2), generator=g, device="cuda")
    q[:, :, 7:9] = (1.0 + 0.1 * torch.rand((rows, 2, 2), generator=g, device="cuda")) * 2.0 ** -20
    by = torch.pow(2.0, (torch.arange(rows, device="cuda") % 14).float())
    c.q = (q * by[:, None, None]).view(rows, -1)
    o = c.run()
    ok(b2s)
    inside(c, o, 3)


@gpu
@pytest.mark.parametrize("new,prefix", [([1] * 70, 600), ([80, 1, 70], 300), ([3, 120, 2, 90], 5000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_bad_row_range_behind_a_prefix_touches_no_other_sequence(b2s, new, prefix, dtype):
    """The prefix as a pass of its own over all rows: a sequence whose range is out of order is left out, the others see the
    prefix all the same. A last entry below their rows leaves them out, rather than without a prefix."""
    keys = [5 + 7 * (i % 9) + (x if x > 4 else 0) for i, x in enumerate(new)]
    c = Case(131, new, keys, 32, 8, 64, 16, dtype, I8, True, prefix, extra_rows=4)
    start = c.q_start.clone()
    ref, tol = c.reference()
    first, last = new[0], c.rows - new[-1]
    second = int(start[2])
    for at, value, good in ((0, -1, slice(first, c.rows)), (0, first + 1, slice(first, c.rows)), (0, 2 ** 31 - 1, slice(first, c.rows)),
                            (1, -5, slice(second, c.rows)), (len(new), c.rows + 5, slice(0, last)), (len(new), -2 ** 31, slice(0, last)),
                            (len(new), 0, slice(0, 0))):
        c.q_start.copy_(start)
        c.q_start[at] = value
        o = c.run()
        ok(b2s, 4)
        assert bool(((o[:c.rows].double() - ref).abs() <= tol)[good].all())
        rest = torch.ones(o.shape[0], dtype=torch.bool, device="cuda")
        rest[good] = False
        assert bool((o[rest] == 7).all())


@gpu
@pytest.mark.parametrize("prefix", [0, 300])
def test_a_bad_row_range_in_the_middle_touches_no_sequence_before_it(b2s, prefix):
    """Rows whose pieces are joined find their sequence although an entry of q_start behind theirs is out of order."""
    new = [80, 40, 60, 2]
    c = Case(133, new, [400, 300, 200, 9], 8, 2, 64, 16, F32, I8, True, prefix, extra_rows=4)
    start = c.q_start.clone()
    ref, tol = c.reference()
    for at in (1, 2, 3):
        for value in (-5, 2 ** 31 - 1):
            c.q_start.copy_(start)
            c.q_start[at] = value
            o = c.run()
            ok(b2s, 4)
            good = torch.ones(c.rows, dtype=torch.bool, device="cuda")
            good[int(start[at - 1]):int(start[at + 1])] = False
            assert bool(((o[:c.rows].double() - ref).abs() <= tol)[good].all())
            assert bool((o[:c.rows][~good] == 7).all() and (o[c.rows:] == 7).all())


def workspace(M, batch, max_q, max_pages, prefix, heads, hkv, hd, ps):
    c = cache_struct(n_kv_heads=hkv, head_dim=hd, page_size=ps)
    b = batch_struct(batch=batch, max_q=max_q, max_pages=max_pages, ld_pages=max_pages)
    return kv._bind().b2s_attention_kv_workspace_size(C.byref(c), C.byref(b), M, heads, prefix)


def test_the_workspace_of_the_largest_call_is_enough_for_smaller_ones(b2s):
    """Sized once for the largest shapes it serves every call of no larger ones, also those that cut their keys."""
    big = workspace(8 * 512, 8, 512, 128, 0, 20, 5, 128, 64)
    for M, batch, max_q in ((100, 1, 100), (900, 3, 300), (1152, 4, 288), (1, 1, 1), (512, 1, 512)):
        assert 0 < workspace(M, batch, max_q, 128, 0, 20, 5, 128, 64) <= big
    g = np.random.default_rng(3)

    def log(hi):
        return int(np.exp(g.uniform(0, np.log(hi)))) if hi > 1 else hi

    for _ in range(400):
        hkv = log(16)
        fixed = (hkv * log(12), hkv, 16 * int(g.integers(1, 9)), 1 << int(g.integers(4, 11)))
        M, batch, max_q, pages, prefix = log(20000), log(3000), log(20000), log(4000), int(g.integers(0, 2)) * log(200000)
        size = workspace(M, batch, max_q, pages, prefix, *fixed)
        assert size > 0 and size % 256 == 0
        for _ in range(12):
            less = (log(M), log(batch), log(max_q), log(pages), log(prefix) * int(g.integers(0, 2)))
            assert workspace(*less, *fixed) <= size, (less, (M, batch, max_q, pages, prefix), fixed)


class Elsewhere:
    """A tensor on a device of the given index, as far as the binding looks at one."""

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self.device, self.index = torch.Size(shape), dtype, f"cuda:{device}", device
        self.nbytes = 1 << 40

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        s = [1]
        for n in self.shape[:0:-1]:
            s.insert(0, s[0] * n)
        return tuple(s) if i is None else s[i]

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return P


def test_a_batch_of_another_device_is_refused(b2s, monkeypatch):
    """A batch built under one device and used under another: its pointers are not passed on."""
    monkeypatch.setattr(kv, "_raw_stream", lambda dev: 0)

    def on(device):
        monkeypatch.setattr(kv, "_device", lambda: device)
        i32 = torch.int32
        cache = kv.Cache(*[Elsewhere((4, 2, 16, 64), I8, device) for _ in range(2)], *[Elsewhere((4, 2, 16), F32, device) for _ in range(2)])
        batch = kv.Batch(Elsewhere((3,), i32, device), Elsewhere((2,), i32, device), Elsewhere((2, 2), i32, device), 1)
        return cache, batch, Elsewhere((2, 256), F32, device), Elsewhere((1,), torch.uint8, device), Elsewhere((2,), i32, device)

    _, batch, *_ = on(0)
    cache, _, q, ws, pages = on(1)
    with pytest.raises(ValueError, match="batch"):
        kv.attention(cache, batch, q, 4, 1.0, True, q, ws)
    with pytest.raises(ValueError, match="batch"):
        kv.attention_prefix(cache, batch, pages, 20, q, 4, 1.0, True, q, ws)


@pytest.mark.parametrize("heads,hd", [(2 ** 24, 256), (2 ** 25, 128), (2 ** 30, 4), (2 ** 30 - 64, 4)])
def test_rope_axes_refuses_rows_past_32_bits(b2s, heads, hd):
    """A row of nearly 2^31 pairs or more: its pairs are counted in 32 bits."""
    width = heads * hd
    assert kv._bind().b2s_rope_axes(30, P, width, 1, heads, hd, P, 1, 1, (C.c_int32 * 1)(hd // 2), 0, 1e4, 2 * P, width, None) == UNSUPPORTED
    assert "2^31" in b2s.last_error()


def test_attention_in_place_needs_one_stride(b2s):
    """o may be q; with another row stride rows would be written over queries that are still to be read."""
    L, c, b = kv._bind(), cache_struct(), batch_struct()
    args = (0, P, 2560, 4, 20, 0.1, 1, P, 2564, 2 * P, 1 << 40, None)
    assert L.b2s_attention_kv(C.byref(c), C.byref(b), *args) == INVALID
    assert "in place" in b2s.last_error()
    assert L.b2s_attention_kv_prefix(C.byref(c), C.byref(b), P, 100, *args) == INVALID


def test_no_grid_is_let_in_before_tensor_memory_is_allocated():
    """A kernel that lets the next grid start first may find its tensor memory taken by a block of that grid, which waits for it."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "robot.cpp_b200", "csrc")
    seen = 0
    for name in sorted(os.listdir(csrc)):
        if name.endswith(".cu"):
            for kernel in open(os.path.join(csrc, name)).read().split("__global__")[1:]:
                if "tmem_alloc(" in kernel:
                    seen += 1
                    assert "griddep_launch()" not in kernel[:kernel.index("tmem_alloc(")], name
    assert seen >= 4


@gpu
@pytest.mark.parametrize("new,keys,heads,hkv,hd,prefix", MANY + [
    ([1], [1], 1, 1, 16, 0), ([1], [4000], 2, 1, 128, 0), ([1], [3000], 4, 4, 64, 5000), ([3, 5, 1], [300, 40, 1000], 32, 4, 64, 0),
    ([65], [4096], 2, 1, 32, 0), ([129], [1301], 3, 3, 96, 77), ([96, 1, 96], [2049, 2049, 127], 6, 1, 128, 0), ([9], [600], 20, 5, 128, 0),
    ([1] * 300, [1 + 7 * (i % 40) for i in range(300)], 6, 3, 64, 0), ([2, 1] * 100, [40, 3] * 100, 8, 4, 80, 33)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,code", [(F32, I8), (BF16, E4M3)])
def test_every_key_counts_once(b2s, new, keys, heads, hkv, hd, prefix, causal, dtype, code):
    """Queries of zero give every visible key the same weight. Token j's value is a whole number in column j % head_dim and zero in
    the others: sums and counts are exact, and one key too few or too many changes a column by more than 2^-10 of it and every other
    one by 1 / n, where fp32 outputs are held to 2^-13 at the longest."""
    c = Case(141, new, keys, heads, hkv, hd, 16, dtype, code, causal, prefix, extra_rows=2)
    c.q.zero_()
    c.cache.k_scale.fill_(1.0)
    c.cache.v_scale.fill_(1.0)
    c.cache.v.view(torch.uint8).zero_()
    for pages, n, first in [(c.prefix_pages, prefix, 0)] + [(c.pages[b], n, prefix) for b, n in enumerate(keys)]:
        if n:
            j = torch.arange(n, device="cuda")
            value = (1 + (first + j) // hd % 8).to(F32)  # 1 .. 8: also exact in e4m3
            row = torch.zeros(n, hkv, hd, device="cuda")
            row[j, :, (first + j) % hd] = value[:, None]
            c.cache.v.view(torch.uint8)[pages[j // 16].long(), :, j % 16] = row.to(c.cache.v.dtype).view(torch.uint8)
    o = c.run()
    ok(b2s)
    inside(c, o, 0)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,heads,hd,sections,inter", [
    (40, 5, 128, [24, 20, 20], True), (33, 3, 72, [36], False), (700, 2, 32, [5, 11], False), (9, 2, 256, [0, 100, 28], True)])
def test_rope_axes_within_its_roundings(b2s, dtype, M, heads, hd, sections, inter):
    """Each row against its own positions' bound: the angle is a double, 2^-51 of the position in radians; cosine and sine within 1.5 * 2^-24
    (read off rows that are zero in one half), two products and a sum of 2^-24 each, one rounding to the type."""
    g = gen(M + hd)
    pos = (10.0 ** (9 * torch.rand((M, len(sections)), generator=g, device="cuda"))).to(torch.int32)
    x = randn(g, M, heads * hd, dtype=dtype)
    ref, mag = rope_ref(x, heads, hd, pos, sections, 500000.0, inter)
    y = torch.empty_like(x)
    kv.rope_axes(x, heads, hd, pos, sections, 500000.0, y, inter)
    ok(b2s)
    angle = pos.double().amax(1, keepdim=True) * 2.0 ** -51
    assert bool(((y.double() - ref).abs() <= (4 * U + angle) * mag + HALF[dtype] * ref.abs()).all())
    if dtype == F32:
        x.view(M, heads, 2, hd // 2)[:, :, 1] = 0
        x.view(M, heads, 2, hd // 2)[:, :, 0] = 1
        ref, _ = rope_ref(x, heads, hd, pos, sections, 500000.0, inter)
        kv.rope_axes(x, heads, hd, pos, sections, 500000.0, y, inter)
        ok(b2s)
        assert bool(((y.double() - ref).abs() <= 1.5 * U + angle).all())


@gpu
def test_scale_offsets_pass_32_bits(b2s):
    """Scales whose byte offsets, and codes whose offsets, lie past 2^31 and 2^32."""
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of device memory")
    pages, ps = 2 ** 19 + 2 ** 14, 1024  # 5.5e8 tokens: 8.9e9 code bytes and 2.2e9 scale bytes each for keys and values
    cache = kv.Cache.empty(pages, 1, ps, 16)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        t.zero_()
    g, n = gen(61), 1500
    slots = torch.arange(n, device="cuda") + (pages - 2) * ps
    k, v = randn(g, n, 16), randn(g, n, 16)
    kv.write(cache, k, v, slots)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    kv.read(cache, slots, ko, vo)
    ok(b2s)
    assert float((ko - k).abs().max()) <= float(k.abs().max()) * 0.51 / 127 and float((vo - v).abs().max()) <= float(v.abs().max()) * 0.51 / 127
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device="cuda")
    for rows in (1, 100):
        q, o = torch.zeros(rows, 64, device="cuda"), torch.empty(rows, 64, device="cuda")
        batch = kv.Batch(torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                         torch.tensor([n], dtype=torch.int32, device="cuda"), table, rows)
        ws = torch.empty(kv.attention_workspace_size(cache, batch, rows, 4), dtype=torch.uint8, device="cuda")
        kv.attention(cache, batch, q, 4, 0.1, False, o, ws)
        ok(b2s)
        ref = vo.double().mean(0).repeat(rows, 4)  # equal weights
        assert float((o.double() - ref).abs().max()) <= ((16 + n / 8) * 2.0 ** -23 + 2.0 ** -21) * float(vo.double().abs().mean(0).max())
