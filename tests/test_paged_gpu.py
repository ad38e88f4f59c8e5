"""Paged-cache operators on the GPU against plain implementations in 64 bits.

Tolerances are the roundings that the formulas contain (half a step of the type:
u = eps / 2), counted per value:

* append, 16-bit: one rounding to the type (u relative), and at most 16 f32
  roundings (2^-24 each) of |x| + |y| before it.  int8: the code is the nearest
  to within a half step plus that f32 noise; a scale has two f32 roundings more.
* read: one rounding of code * scale to the type over one f32 rounding.
* attention: rounding of the output (u |o|); of each probability to 16 bits and
  of the sums (u + 2^-12 relative to sum p |v| / sum p; the f32 sums of up to
  2^12 terms and exp2's few steps stay below 2^-12).
* verification: equal tokens; log-probabilities to 2^-18 relative to 1 + |log p|
  (f32 sums of up to 2^18 terms, pairwise over at least 2^9 threads).
"""
import math

import pytest

pytestmark = pytest.mark.gpu

D = 128


@pytest.fixture(scope="module")
def torch(cuda):
    import torch as _t
    return _t


@pytest.fixture(scope="module")
def P(cuda):
    from dial_cuda import paged
    return paged


@pytest.fixture(autouse=True)
def no_device_error(cuda):
    import dial_cuda
    yield
    assert dial_cuda.lib().dial_device_error(1) == 0, "a kernel reported an error"


def device_error():
    import dial_cuda
    return dial_cuda.lib().dial_device_error(1)


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def dtype_of(torch, name):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def quantise64(torch, x):
    """Row codes and scales of x [..., 128] as the header states them."""
    a = x.double().abs().amax(-1, keepdim=True)
    s = torch.where(a > 0, a / 127, torch.ones_like(a))
    y = x.double() / s
    return (torch.floor(y.abs() + 0.5) * y.sign()).clamp(-127, 127).to(torch.int8), s.squeeze(-1).float()


class Setup:
    """Pages in any order with filled rows, a block table with junk behind each last page."""

    def __init__(self, torch, P, q, kv, dtype, quant, page, hkv, seed=0, pad=0, fill=None, junk=-1):
        g = gen(torch, 1000 + seed)
        self.torch, self.q, self.kv, self.page, self.hkv, self.quant = torch, q, kv, page, hkv, quant
        dt = dtype_of(torch, dtype)
        need = [-(-L // page) for L in kv]
        n = sum(need) + 2
        order = torch.randperm(n, generator=g, device="cuda").tolist()
        self.table = torch.full((len(q), max(need + [1]) + 1), junk, dtype=torch.int32)
        used = 0
        for b, m in enumerate(need):
            self.table[b, :m] = torch.tensor(order[used:used + m], dtype=torch.int32)
            used += m
        self.host_table = self.table.tolist()
        self.table = self.table.cuda()
        x = [torch.randn((n, hkv, page, D), generator=g, device="cuda") + m for m in (0.0, 0.3)]
        if quant:
            self.pages, self.scales = map(list, zip(*(quantise64(torch, y) for y in x)))
        else:
            self.pages, self.scales = [y.to(dt) for y in x], [None, None]
        start = [0]
        for m in q:
            start.append(start[-1] + m)
        self.start, self.T = start, start[-1] + pad
        if fill is not None:  # rows of the sequences' pages behind their last row
            for b, L in enumerate(kv):
                if L % page:
                    at = self.host_table[b][L // page]
                    for i in (0, 1):
                        if quant:
                            self.scales[i][at, :, L % page:] = fill
                        else:
                            self.pages[i][at, :, L % page:] = fill
        self.cache = P.PagedKVCache.from_tensors(*self.pages, *self.scales)
        self.kv_len = torch.tensor(kv, dtype=torch.int32, device="cuda")
        self.q_start = torch.tensor(start, dtype=torch.int32, device="cuda")
        self.batch = P.PagedBatch(self.table, self.kv_len, self.q_start, max_q=max(max(q), 1), max_kv=max(max(kv), 1))

    def rows(self, i, b, first, last, pages=None, scales=None):
        """Rows first..last of sequence b's keys (i = 0) or values in 64 bits, [rows, hkv, 128]."""
        torch = self.torch
        pages, scales = pages or self.pages, scales or self.scales
        r = torch.arange(first, last, device="cuda")
        at = self.table[b].long()[r // self.page]
        x = pages[i][at, :, r % self.page].double()
        return x * scales[i][at, :, r % self.page].double()[..., None] if self.quant else x


# ------------------------------------------------------------------ append
SECTIONS = {1: (64,), 2: (40, 24), 3: (24, 20, 20), 4: (16, 16, 16, 16)}


def axis_of(axes, interleaved):
    out = []
    for i in range(64):
        if interleaved:
            a = i % axes
            out.append(a if i < SECTIONS[axes][a] * axes else 0)
        else:
            a, end = 0, SECTIONS[axes][0]
            while i >= end:
                a += 1
                end += SECTIONS[axes][a]
            out.append(a)
    return out


@pytest.mark.parametrize("q,kv,pad", [([1], [1], 0), ([1], [2049], 3), ([7, 0, 33, 1], [7, 5, 49, 16], 2),
                                      ([20, 40], [64, 31], 0), ([1] * 70, list(range(1, 71)), 1),
                                      ([(2, 0, 1)[b % 3] for b in range(1100)], [3 + b % 40 for b in range(1100)], 2)])
@pytest.mark.parametrize("dtype,quant,page,hq,hkv,axes,interleaved,norm", [
    ("f16", False, 16, 32, 8, 1, True, True), ("bf16", False, 64, 8, 8, 3, True, True),
    ("f16", True, 32, 7, 1, 3, False, False), ("bf16", True, 16, 10, 2, 4, True, True),
    ("bf16", True, 128, 4, 4, 2, False, True), ("f16", True, 256, 24, 3, 2, True, False)])
def test_append(torch, P, q, kv, pad, dtype, quant, page, hq, hkv, axes, interleaved, norm):
    s = Setup(torch, P, q, kv, dtype, quant, page, hkv, seed=len(q) + axes, pad=pad)
    g = gen(torch, 5)
    dt = dtype_of(torch, dtype)
    u = torch.finfo(dt).eps / 2
    qkv = (torch.randn((s.T, (hq + 2 * hkv) * D), generator=g, device="cuda") * 2).to(dt)
    qkv[0, (hq + hkv) * D:(hq + hkv + 1) * D] = 0  # a value row of zeros
    w = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt) for _ in range(2)] if norm else [None, None]
    pos = torch.randint(0, 500, (axes, s.T), generator=g, device="cuda", dtype=torch.int32)
    angle = torch.rand((500, 64), generator=g, device="cuda") * 7
    cos, sin = angle.cos(), angle.sin()
    before = [p.clone() for p in s.pages], [p.clone() if quant else None for p in s.scales]
    out = torch.full((s.T, hq, D), 77.0, dtype=dt, device="cuda")
    s.cache.append(qkv, s.batch, cos, sin, pos if axes > 1 else pos[0], q_norm=w[0], k_norm=w[1], eps=1e-5,
                   sections=SECTIONS[axes], interleaved=interleaved, out=out)
    x = qkv.double().view(s.T, -1, D)
    ax = axis_of(axes, interleaved)
    c = torch.stack([cos[pos[a].long(), i] for i, a in enumerate(ax)], -1).double()[:, None]
    n = torch.stack([sin[pos[a].long(), i] for i, a in enumerate(ax)], -1).double()[:, None]

    def turned(y, wt):
        if norm:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * wt.double()
        a, z = y[..., :64], y[..., 64:]
        size = torch.cat([(a * c).abs() + (z * n).abs(), (a * n).abs() + (z * c).abs()], -1)
        return torch.cat([a * c - z * n, a * n + z * c], -1), size

    want, size = turned(x[:, :hq], w[0])
    real = s.start[-1]
    assert torch.all((out[:real].double() - want[:real]).abs() <= u * want[:real].abs() + 16 * 2.0 ** -24 * size[:real] + 1e-7)
    assert torch.all(out[real:] == 77)  # rows behind the last sequence
    k, ksize = turned(x[:, hq:hq + hkv], w[1])
    v = x[:, hq + hkv:]
    changed = torch.zeros(s.pages[0].shape[:3], dtype=torch.bool, device="cuda")
    for b in range(len(q)):
        first = max(0, kv[b] - q[b])  # tokens in front of row 0 have none
        r = torch.arange(first, kv[b], device="cuda")
        t = s.start[b] + q[b] - kv[b] + r
        at = s.table[b].long()[r // page]
        changed[at, :, r % page] = True
        for i, (val, sz) in enumerate(((k, ksize), (v, v.abs()))):
            got, ref, sz = s.pages[i][at, :, r % page], val[t], sz[t]
            if quant:
                _, sc = quantise64(torch, ref)
                gs = s.scales[i][at, :, r % page]
                noise = 20 * 2.0 ** -24 * sz.amax(-1)
                assert torch.all((gs.double() - sc.double()).abs() <= noise / 127 + 4 * 2.0 ** -24 * sc.double())
                off = (got.double() * gs.double()[..., None] - ref).abs()
                assert torch.all(off <= gs.double()[..., None] * 0.5 + 3 * noise[..., None])
                assert torch.all(got.abs().amax(-1)[ref.abs().amax(-1) > 0] == 127)
            else:
                assert torch.all((got.double() - ref).abs() <= u * ref.abs() + 16 * 2.0 ** -24 * sz + 1e-7)
    for i in (0, 1):  # nothing else was touched
        assert torch.equal(s.pages[i][~changed], before[0][i][~changed])
        if quant:
            assert torch.equal(s.scales[i][~changed], before[1][i][~changed])


def test_append_int8_codes_do_not_depend_on_a_sums_order(torch, P):
    """The codes equal those of the same f32 steps in torch, bit for bit."""
    s = Setup(torch, P, [300], [300], "bf16", True, 64, 8)
    g = gen(torch, 9)
    qkv = torch.randn((300, 24 * D), generator=g, device="cuda").to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
    cos, sin = P.rope_tables(512, 1e6)
    pos = torch.arange(300, device="cuda", dtype=torch.int32)
    s.cache.append(qkv, s.batch, cos, sin, pos, q_norm=w, k_norm=w)
    x = qkv.view(300, 24, D)[:, 8:16].float()
    inv = (1.0 / (x.double().square().sum(-1, keepdim=True) / D + float(torch.tensor(1e-6))).sqrt()).float()
    x = x * inv * w.float()
    a, z, c, n = x[..., :64], x[..., 64:], cos[:300, None], sin[:300, None]
    x = torch.cat([a * c - z * n, a * n + z * c], -1)
    top = x.abs().amax(-1, keepdim=True)
    sc = (top.double() / 127).float()
    y = x * (1.0 / sc)
    r = torch.trunc(y)
    r = (r + torch.sign(y) * ((y - r).abs() >= 0.5)).clamp(-127, 127)
    at = s.table[0].long()[pos.long() // 64]
    assert torch.equal(s.pages[0][at, :, pos.long() % 64], r.to(torch.int8))
    assert torch.equal(s.scales[0][at, :, pos.long() % 64], sc[..., 0])


def test_append_keeps_rows_with_nan_or_infinity_as_nan(torch, P):
    s = Setup(torch, P, [4], [4], "f16", True, 16, 2)
    qkv = torch.ones((4, 8 * D), dtype=torch.float16, device="cuda")
    qkv[1, 6 * D + 5] = math.inf
    qkv[2, 7 * D + 9] = math.nan
    cos, sin = P.rope_tables(8, 1e4)
    s.cache.append(qkv, s.batch, cos, sin, torch.arange(4, dtype=torch.int32, device="cuda"))
    _, v = s.cache.read(s.batch, tokens=4)
    bad = torch.isnan(v).all(-1)
    assert bad.tolist() == [[False, False], [True, False], [False, True], [False, False]]
    assert torch.equal(v[~bad], torch.ones_like(v[~bad]))


def test_append_reports_bad_pages_and_positions(torch, P):
    s = Setup(torch, P, [40], [40], "f16", False, 16, 2)
    s.table[0, 1] = s.cache.n_pages  # rows 16..31: no such page
    before = [p.clone() for p in s.pages]
    qkv = torch.randn((40, 8 * D), generator=gen(torch, 1), device="cuda").half()
    cos, sin = P.rope_tables(64, 1e4)
    pos = torch.arange(40, dtype=torch.int32, device="cuda")
    s.cache.append(qkv, s.batch, cos, sin, pos)
    assert device_error() == 1
    ok = [s.host_table[0][0], s.host_table[0][2]]
    other = [i for i in range(s.cache.n_pages) if i not in ok]
    for i in (0, 1):
        assert torch.equal(s.pages[i][other], before[i][other])
    v = qkv.view(40, 8, D)[:, 6:]
    assert torch.equal(s.pages[1][ok[0]].transpose(0, 1), v[:16])
    assert torch.equal(s.pages[1][ok[1], :, :8].transpose(0, 1), v[32:])
    s.table[0, 1] = s.host_table[0][1]
    good = s.cache.append(qkv, s.batch, cos, sin, pos.clamp(min=0, max=63))
    for bad, near in ((-5, 0), (64, 63), (1 << 30, 63)):  # outside the table: its nearest row, and reported
        pos[3] = near
        want = s.cache.append(qkv, s.batch, cos, sin, pos)
        assert device_error() == 0
        pos[3] = bad
        got = s.cache.append(qkv, s.batch, cos, sin, pos)
        assert device_error() == 1
        assert torch.equal(got, want) and torch.equal(got[:3], good[:3])


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("q,kv,pad", [([1], [1], 0), ([33, 0, 100], [33, 3, 130], 5), ([50], [20], 0),
                                      ([0, 0] + [b % 3 for b in range(1500)], [4] * 1502, 1)])
@pytest.mark.parametrize("dtype,quant,page,hkv", [("f16", False, 16, 8), ("bf16", False, 256, 3), ("f16", True, 32, 1),
                                                  ("bf16", True, 64, 8)])
def test_read(torch, P, q, kv, pad, dtype, quant, page, hkv):
    s = Setup(torch, P, q, kv, dtype, quant, page, hkv, pad=pad, fill=math.nan)
    dt = dtype_of(torch, dtype)
    out = tuple(torch.full((s.T, hkv, D), 7.0, dtype=dt, device="cuda") for _ in range(2))
    s.cache.read(s.batch, out=out)
    for i in (0, 1):
        for b in range(len(q)):
            first = max(0, kv[b] - q[b])
            have = kv[b] - first
            got = out[i][s.start[b]:s.start[b + 1]]
            ref = s.rows(i, b, first, kv[b])
            if quant:
                u = torch.finfo(dt).eps / 2
                assert torch.all((got[q[b] - have:].double() - ref).abs() <= u * ref.abs() * (1 + 1e-3) + 1e-7)
            else:
                assert torch.equal(got[q[b] - have:].double(), ref)
            assert torch.all(got[:q[b] - have] == 0)  # rows that the cache does not have
        assert torch.all(out[i][s.start[-1]:] == 7)


# ------------------------------------------------------------------ attention
def attention64(torch, s, q, scale):
    """(out, sum p |v| / sum p) of every token in 64 bits; zeros where nothing is attended."""
    T, hq, _ = q.shape
    out = torch.zeros((T, hq, D), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    rep = hq // s.hkv
    for b, (n, L) in enumerate(zip(s.q, s.kv)):
        if not n or not L:
            continue
        k, v = (s.rows(i, b, 0, L).repeat_interleave(rep, 1) for i in (0, 1))
        last = L - n + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None]
        x = torch.einsum("thd,jhd->htj", q[s.start[b]:s.start[b + 1]].double(), k) * scale
        x = x.masked_fill(j > last, -math.inf)
        x = torch.softmax(x, -1)
        x = torch.where((last < 0)[None], 0.0, x)
        out[s.start[b]:s.start[b + 1]] = torch.einsum("htj,jhd->thd", x, v)
        size[s.start[b]:s.start[b + 1]] = torch.einsum("htj,jhd->thd", x, v.abs())
    return out, size


def check_attention(torch, s, q, got, scale=D ** -0.5, fill=None):
    want, size = attention64(torch, s, q, scale)
    u = torch.finfo(q.dtype).eps / 2
    real = s.start[-1]
    off = (got[:real].double() - want[:real]).abs()
    bad = ~(off <= u * want[:real].abs() + (u + 2.0 ** -12) * size[:real] + 1e-7)
    assert not bad.any(), (int(bad.sum()), float(off.max()), bad.nonzero()[:3].tolist())
    if fill is not None:
        assert torch.all(got[real:] == fill)


LENGTHS = [
    ([1], [1]), ([1], [2]), ([1, 1, 1], [15, 16, 17]), ([1] * 5, [127, 128, 129, 1000, 0]), ([1], [4097]),
    ([2, 5, 3], [2, 300, 1025]), ([9, 0, 1], [9, 7, 600]), ([8, 16], [8, 4000]),
    ([33], [33]), ([64, 17, 0, 1], [200, 17, 3, 900]), ([130], [130]), ([257, 3], [1300, 5]), ([40, 40], [10, 0]),
    ([5] * 20, [1700 + 37 * b for b in range(20)]), ([1] * 20, [1701 + 37 * b for b in range(20)]),
    ([40] * 19, [900 + 41 * b for b in range(19)]),
    ([(0, 1, 3, 2)[b % 4] for b in range(330)], [(7 * b) % 50 for b in range(330)]),
    ([(1, 0, 45, 1, 2)[b % 5] for b in range(330)], [30 + b % 60 for b in range(330)]),
]


@pytest.mark.parametrize("q,kv", LENGTHS)
@pytest.mark.parametrize("dtype,quant,page,hq,hkv", [
    ("f16", False, 64, 32, 8), ("bf16", False, 16, 8, 8), ("f16", True, 16, 7, 1), ("bf16", True, 64, 16, 2),
    ("bf16", False, 256, 10, 2), ("f16", True, 128, 6, 2), ("f16", False, 32, 9, 3), ("bf16", True, 256, 4, 4)])
def test_attention(torch, P, q, kv, dtype, quant, page, hq, hkv):
    s = Setup(torch, P, q, kv, dtype, quant, page, hkv, seed=hq, pad=3, fill=math.nan)
    x = (torch.randn((s.T, hq, D), generator=gen(torch, 3), device="cuda") * 1.5).to(dtype_of(torch, dtype))
    out = torch.full_like(x, 5.0)
    s.cache.attention(x, s.batch, out=out)
    check_attention(torch, s, x, out, fill=5.0)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("scale", [0.02, 1.0])
@pytest.mark.parametrize("q,kv", [([3], [700]), ([150], [700])])
def test_attention_scale_and_peaked_rows(torch, P, quant, scale, q, kv):
    s = Setup(torch, P, q, kv, "f16", quant, 32, 2)
    x = (torch.randn((s.T, 8, D), generator=gen(torch, 4), device="cuda") * 3).half()
    check_attention(torch, s, x, s.cache.attention(x, s.batch, scale=scale), scale=scale)


@pytest.mark.parametrize("q,kv", [(2, 3), (5, 300), (60, 90), (40, 2000)])
def test_a_key_of_minus_infinity_weighs_nothing_beside_unseen_nans(torch, P, q, kv):
    """Scores of minus infinity in the rows that are computed again for an unseen NaN value."""
    s = Setup(torch, P, [q], [kv], "f16", False, 16, 2, seed=4)
    x = torch.randn((q, 8, D), generator=gen(torch, 9), device="cuda").half()
    x[..., 0] = 1
    s.pages[0][s.host_table[0][0], :, 0, 0] = -math.inf
    want = torch.empty_like(x)
    s.cache.attention(x, s.batch, out=want)
    check_attention(torch, s, x, want)
    s.pages[1][s.host_table[0][(kv - 1) // 16], :, (kv - 1) % 16] = math.nan
    got = s.cache.attention(x, s.batch)
    assert torch.isnan(got[-1]).all()
    s.pages[1][s.host_table[0][(kv - 1) // 16], :, (kv - 1) % 16] = 0
    want, size = attention64(torch, s, x, D ** -0.5)
    off = (got[:-1].double() - want[:-1]).abs()
    assert torch.all(off <= 2.0 ** -11 * want[:-1].abs() + (2.0 ** -11 + 2.0 ** -12) * size[:-1] + 1e-7)


@pytest.mark.parametrize("q,kv", [([6], [300]), ([70, 40], [300, 141])])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("quant", [False, True])
def test_rows_that_a_token_does_not_attend_do_not_touch_it(torch, P, q, kv, bad, quant):
    """A non-finite key or value row among the new tokens' own: earlier tokens do not see it."""
    s = Setup(torch, P, q, kv, "bf16", quant, 64, 2)
    at = kv[0] - 3  # the row of the third-last token of sequence 0
    page, row = s.host_table[0][at // 64], at % 64
    x = torch.randn((s.T, 8, D), generator=gen(torch, 4), device="cuda").to(torch.bfloat16)
    for i in (0, 1):
        keep = (s.scales if quant else s.pages)[i][page, 0, row].clone()
        want, size = attention64(torch, s, x, D ** -0.5)
        (s.scales if quant else s.pages)[i][page, 0, row] = bad
        got = s.cache.attention(x, s.batch)
        (s.scales if quant else s.pages)[i][page, 0, row] = keep
        sees = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
        sees[q[0] - 3:q[0], :4] = True
        u = 2.0 ** -8
        off = (got.double() - want).abs()
        assert torch.all(off[~sees] <= u * want[~sees].abs() + (u + 2.0 ** -12) * size[~sees] + 1e-7)
        if i == 1 or quant or bad != -math.inf:
            assert not torch.isfinite(got[sees]).all(-1).any() or i == 0


def test_attention_reports_bad_pages_and_lengths(torch, P):
    for q in ([1, 1], [80, 1]):
        s = Setup(torch, P, q, [200, 90], "f16", False, 16, 2)
        x = torch.randn((s.T, 8, D), generator=gen(torch, 4), device="cuda").half()
        good = s.cache.attention(x, s.batch)
        check_attention(torch, s, x, good)
        for page in (-1, s.cache.n_pages, 1 << 30, -(1 << 31)):
            keep = int(s.table[0, 2])
            s.table[0, 2] = page
            got = s.cache.attention(x, s.batch)
            assert device_error() == 1
            assert torch.equal(got[q[0]:], good[q[0]:])  # the other sequence
            s.table[0, 2] = keep
        for where, i, value in ((s.kv_len, 0, 1 << 20), (s.kv_len, 0, -3), (s.q_start, 1, -7), (s.q_start, 2, 1 << 20)):
            keep = int(where[i])
            where[i] = value
            s.cache.attention(x, s.batch)
            assert device_error() == 1, (i, value)
            where[i] = keep
        assert torch.equal(s.cache.attention(x, s.batch), good)


@pytest.mark.parametrize("q,kv,quant", [([1, 1], [3000, 70], False), ([5], [2000], True), ([300, 20], [900, 333], False),
                                        ([300, 20], [900, 333], True)])
def test_attention_gives_the_same_bits_again_and_in_graphs(torch, P, q, kv, quant):
    s = Setup(torch, P, q, kv, "bf16", quant, 64, 4)
    x = torch.randn((s.T, 16, D), generator=gen(torch, 4), device="cuda").to(torch.bfloat16)
    first = s.cache.attention(x, s.batch)
    side = torch.cuda.Stream()
    outs = [torch.zeros_like(x) for _ in range(2)]
    graphs = []
    for o in outs:  # two graphs over the same cache
        gr = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(gr, stream=side):
            s.cache.attention(x, s.batch, out=o)
        graphs.append(gr)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    x.copy_(torch.randn(x.shape, generator=gen(torch, 5), device="cuda"))  # replays read the new contents
    s.kv_len[0] -= 2
    s.kv[0] -= 2
    graphs[0].replay()
    check_attention(torch, s, x, outs[0])


@pytest.mark.parametrize("q", [1, 40])
def test_attention_and_append_pass_32_bits(torch, P, q):
    """Pages past 2^31 values (and 2^32 bytes) into the pool."""
    page, hkv, L = 256, 8, 600
    n = (1 << 31) // (page * hkv * D) + 8
    pages = [torch.zeros((n, hkv, page, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    table = torch.tensor([[n - 1, n - 3, 2]], dtype=torch.int32, device="cuda")
    cache = P.PagedKVCache.from_tensors(*pages)
    g = gen(torch, 8)
    qkv = torch.randn((L, 3 * hkv * D), generator=g, device="cuda").half()
    cos, sin = P.rope_tables(L, 1e6)
    pos = torch.arange(L, dtype=torch.int32, device="cuda")
    kv = torch.tensor([L], dtype=torch.int32, device="cuda")
    whole = P.PagedBatch(table, kv, torch.tensor([0, L], dtype=torch.int32, device="cuda"))
    x = cache.append(qkv, whole, cos, sin, pos)
    k, v = cache.read(whole, tokens=L)
    assert torch.equal(v, qkv.view(L, 3 * hkv, D)[:, 2 * hkv:])
    assert torch.equal(pages[1][n - 1].transpose(0, 1), v[:256])
    last = P.PagedBatch(table, kv, torch.tensor([0, q], dtype=torch.int32, device="cuda"), max_q=q)
    got = cache.attention(x[L - q:], last)
    p = torch.einsum("thd,jhd->htj", x[L - q:].double(), k.double()) * D ** -0.5
    p = torch.softmax(p.masked_fill(pos[None, None].long() > (L - q + pos[:q, None].long()), -math.inf), -1)
    want, size = (torch.einsum("htj,jhd->thd", p, y) for y in (v.double(), v.double().abs()))
    u = 2.0 ** -11
    assert torch.all((got.double() - want).abs() <= u * want.abs() + (u + 2.0 ** -12) * size + 1e-7)


# ------------------------------------------------------------------ verification
def verify64(torch, logits, ids, start, temperature, accept_u, sample_u, probs):
    """The header's definition, one sequence and row at a time."""
    R, V = logits.shape
    out, told, count = [-1] * R, [0.0] * R, []
    for b in range(len(start) - 1):
        r, n = start[b], 0
        while r < start[b + 1]:
            x = logits[r].double()
            x = torch.where(torch.isnan(x), -math.inf, x)
            top, T = int(x.argmax()), float(temperature[b])
            if x.max() == -math.inf:
                p, logp, top = torch.zeros_like(x), torch.full_like(x, -math.inf), 0
            elif x.max() == math.inf:
                p = (x == math.inf).double()
                p /= p.sum()
                logp = p.log()
            else:
                logp = torch.log_softmax(x / (T or 1.0), -1)
                p = logp.exp()
            judge, take = r + 1 < start[b + 1], top
            d = int(ids[r + 1]) if judge else -1
            inside = 0 <= d < V
            qd = float(probs[r, d]) if judge and inside and probs is not None else 1.0
            ok = judge and inside and (d == top if T == 0 else float(accept_u[r]) * qd < float(p[d]))
            if ok:
                take = d
            elif T > 0 and float(p.sum()) > 0:
                w = p
                if judge:
                    w = p.clone()
                    if probs is not None:
                        w = (p - probs[r].double()).clamp(min=0)
                    elif inside:
                        w[d] = 0
                    if float(w.sum()) == 0:
                        w = p
                cum = w.cumsum(0)
                at = float(sample_u[b]) * float(cum[-1])
                above = (cum > at).nonzero()
                take = int(above[0]) if len(above) else int((w > 0).nonzero()[-1])
            out[r], told[r] = take, float(logp[take])
            n += 1
            r += 1
            if not ok:
                break
        count.append(n)
    return out, count, told


def run_verify(torch, P, logits, ids, start, temperature, accept_u, sample_u, probs=None):
    f = dict(dtype=torch.float32, device="cuda")
    i = dict(dtype=torch.int32, device="cuda")
    return P.verify_drafts(logits, torch.as_tensor(ids).to(**i), torch.tensor(start, **i), torch.as_tensor(temperature).to(**f),
                           torch.as_tensor(accept_u).to(**f), torch.as_tensor(sample_u).to(**f), draft_probs=probs)


def check_verify(torch, P, logits, ids, start, temperature, accept_u, sample_u, probs=None):
    got = run_verify(torch, P, logits, ids, start, temperature, accept_u, sample_u, probs)
    f = dict(dtype=torch.float32, device="cuda")
    out, count, told = verify64(torch, logits, ids, start, torch.as_tensor(temperature).to(**f),
                                torch.as_tensor(accept_u).to(**f), torch.as_tensor(sample_u).to(**f), probs)
    R = start[-1]
    assert got[0][:R].tolist() == out[:R]
    assert got[1].tolist() == count
    for a, b in zip(got[2][:R].tolist(), told):
        assert a == b or abs(a - b) <= 2.0 ** -18 * (1 + abs(b)), (a, b)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [1, 7, 1000, 4099, 32768, 151936])
@pytest.mark.parametrize("with_probs", [False, True])
def test_verify(torch, P, dtype, V, with_probs):
    rows = [1, 4, 0, 9, 2, 6]
    g = gen(torch, V + with_probs)
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    R = start[-1]
    logits = torch.randn((R, V), generator=g, device="cuda") * 3
    draft = (logits + 0.5 * torch.randn((R, V), generator=g, device="cuda")).softmax(-1)
    d = (draft / torch.empty((R, V), device="cuda").exponential_(generator=g)).argmax(-1) if with_probs else draft.argmax(-1)
    ids = torch.cat([d[:1], d[:-1]])
    u = torch.rand((R + 12,), generator=g, device="cuda")
    check_verify(torch, P, logits.to(dtype_of(torch, dtype)), ids, start, [0.7, 1.0, 1.0, 0.3, 0.0, 2.0], u[:R], u[R:R + 6],
                 draft if with_probs else None)


def test_verify_many_sequences(torch, P):
    rows = [(1, 2, 0, 3)[b % 4] for b in range(150)]
    g = gen(torch, 12)
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    R, B, V = start[-1], len(rows), 517
    logits = torch.randn((R, V), generator=g, device="cuda") * 2
    ids = logits.argmax(-1).roll(1).int()
    u = torch.rand((R + B,), generator=g, device="cuda")
    check_verify(torch, P, logits.half(), ids, start, [(0.0, 0.9, 1.3)[b % 3] for b in range(B)], u[:R], u[R:])


@pytest.mark.parametrize("T", [0.2, 0.01, 1e-3, 2e-5, 1e-6, 2e-7, 1e-8, 2e-9, 3e-10, 1e-20, 1e-38, 1.4e-45])
@pytest.mark.parametrize("dtype,offset", [("f32", 0), ("f32", -700), ("f16", 50), ("bf16", 0)])
@pytest.mark.parametrize("with_probs", [False, True])
def test_verify_cold(torch, P, T, dtype, offset, with_probs):
    """Temperatures down to the least positive one: masked logits stay undrawn, near ones keep
    their odds, ties share."""
    rows = [1, 1, 3, 2, 1, 4, 1, 2, 5, 1]
    g = gen(torch, 77)
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    R, V = start[-1], 3001
    logits = (torch.randn((R, V), generator=g, device="cuda") + offset).to(dtype_of(torch, dtype))
    near = logits.amax(-1, keepdim=True).double() - T * 3 * torch.rand((R, 40), generator=g, device="cuda").double()
    at = torch.randperm(V, generator=g, device="cuda")
    logits[:, at[:40]] = near.to(logits.dtype)  # of the largest one's order, some tied with it
    logits[:, at[40:1500]] = -math.inf
    draft = torch.rand((R, V), generator=g, device="cuda")
    draft[:, at[40:]] *= 1e-3
    draft /= draft.sum(-1, keepdim=True)
    ids = at[torch.randint(0, 40, (R,), generator=g, device="cuda")].int()
    u = torch.rand((R + len(rows),), generator=g, device="cuda")
    check_verify(torch, P, logits, ids, start, [T] * len(rows), u[:R], u[R:], draft if with_probs else None)


def test_verify_greedy_ties_take_the_first_index(torch, P):
    logits = torch.zeros((4, 999), device="cuda").half()
    logits[0, [5, 700]] = 3
    logits[1, [17, 998]] = 2
    logits[2, 40] = 1
    got = check_verify(torch, P, logits, [0, 5, 998, 40], [0, 4], [0.0], [0.5] * 4, [0.5])
    assert got[0].tolist() == [5, 17, -1, -1] and got[1].tolist() == [2]


@pytest.mark.parametrize("T", [0.0, 0.8])
def test_verify_infinite_and_nan_logits(torch, P, T):
    g = gen(torch, 3)
    logits = torch.randn((6, 3001), generator=g, device="cuda")
    logits[0] = -math.inf                 # no probability at all
    logits[1, 7:] = math.nan              # NaN counts as minus infinity
    logits[2, [100, 2000]] = math.inf     # all of it to two tokens
    logits[3, 1500:] = -math.inf
    logits[4] = math.nan
    check_verify(torch, P, logits, [0, 0, 5, 2000, 12, 4], [0, 1, 3, 4, 5, 6], [T] * 5, [0.1] * 6, [0.0, 0.9, 0.7, 0.999999, 0.5])


def test_verify_refused_drafts(torch, P):
    """Drafts outside the vocabulary, drafts the draft model could not have made, and a target equal to the draft."""
    g = gen(torch, 6)
    logits = torch.randn((9, 500), generator=g, device="cuda")
    probs = logits.softmax(-1)
    probs[3] = 0
    probs[3, 77] = 1.0
    ids = [0, 500, 0, -1, 12, 5, 1 << 30, 3, 4]
    for p in (None, probs):
        check_verify(torch, P, logits, ids, [0, 2, 4, 6, 9], [1.0] * 4, [0.0, 0.9, 0.5, 0.999, 0.2, 0.7, 0.1, 0.9, 0.3],
                     [0.0, 0.5, 0.25, 0.99], p)
    same = torch.zeros((2, 64), device="cuda")
    flat = torch.full((2, 64), 1 / 64, device="cuda")  # nothing left of max(p - q, 0): drawn from p
    got = check_verify(torch, P, same, [0, 64], [0, 2], [1.0], [0.5, 0.5], [0.5], flat)
    assert got[0].tolist() == [32, -1]


def test_verify_one_row_draws_from_the_distribution(torch, P):
    p = torch.tensor([0.1, 0.0, 0.25, 0.4, 0.25], device="cuda")
    logits = p.log().repeat(5, 1)
    got = run_verify(torch, P, logits, [0] * 5, list(range(6)), [1.0] * 5, [0.0] * 5, [0.0, 0.0999, 0.1001, 0.5, 0.9999])
    assert got[0].tolist() == [0, 0, 2, 3, 4] and got[1].tolist() == [1] * 5
    assert torch.allclose(got[2], p[got[0].long()].log(), atol=1e-6)


def test_verify_leaves_rows_behind_the_last_sequence(torch, P):
    logits = torch.randn((5, 100), generator=gen(torch, 1), device="cuda")
    a = run_verify(torch, P, logits, [0] * 5, [0, 3], [0.0], [0.5] * 5, [0.5])
    b = run_verify(torch, P, logits[:3].contiguous(), [0] * 3, [0, 3], [0.0], [0.5] * 3, [0.5])
    assert torch.equal(a[0][:3], b[0]) and torch.equal(a[1], b[1])


def test_verify_reports_bad_row_ranges(torch, P):
    logits = torch.randn((6, 300), generator=gen(torch, 1), device="cuda")
    for start in ([0, -2, 6], [0, 4, 2], [0, 3, 1 << 20]):
        run_verify(torch, P, logits, [0] * 6, start, [1.0, 0.5], [0.5] * 6, [0.5, 0.5])
        assert device_error() == 1, start


@pytest.mark.parametrize("T", [-1.0, -math.inf, math.nan])
def test_verify_temperatures_that_are_not_positive_are_greedy(torch, P, T):
    g = gen(torch, 31)
    logits = torch.randn((7, 2100), generator=g, device="cuda").bfloat16()
    ids = logits.argmax(-1).roll(1).int()
    ids[6] += 1
    u = torch.rand((10,), generator=g, device="cuda")
    run = lambda t: run_verify(torch, P, logits, ids, [0, 3, 3, 7], [t] * 3, u[:7], u[7:])
    for a, b in zip(run(T), run(0.0)):
        assert torch.equal(a, b)


def test_verify_numbers_outside_their_range_stay_inside_the_vocabulary(torch, P):
    """u of 1, above, below 0 and NaN, draft weights that are NaN or infinite: some token that has
    a probability is drawn."""
    logits = torch.randn((12, 777), generator=gen(torch, 32), device="cuda")
    logits[:, ::3] = -math.inf
    ids = torch.full((12,), 4, dtype=torch.int32, device="cuda")
    draft = torch.zeros((12, 777), device="cuda")
    draft[:, 5], draft[:, 7], draft[:, 8] = math.nan, math.inf, -1.0
    u = torch.tensor([1.0, 7.0, -2.0, math.nan, 1 - 2.0 ** -24, math.inf], device="cuda")
    for probs in (None, draft):
        out, count, logp = run_verify(torch, P, logits, ids, [0, 2, 4, 6, 8, 10, 12], [1.0] * 6, u.repeat(2), u, probs)
        for b in range(6):
            told = out[2 * b:2 * b + int(count[b])]
            assert 1 <= int(count[b]) <= 2 and torch.all((told >= 0) & (told < 777) & (told % 3 != 0))


def test_calls_on_several_streams_at_once(torch, P):
    """Calls on streams of their own, over shared and other caches, give the bits of calls in turn."""
    s = Setup(torch, P, [3, 60, 1], [300, 700, 2000], "bf16", True, 32, 4, seed=8)
    d = Setup(torch, P, [1] * 6, [100 * b + 9 for b in range(6)], "bf16", True, 32, 4, seed=9)
    g = gen(torch, 33)
    x, y = (torch.randn((z.T, 16, D), generator=g, device="cuda").bfloat16() for z in (s, d))
    logits = torch.randn((s.T, 9001), generator=g, device="cuda")
    ids, u = logits.argmax(-1).roll(1).int(), torch.rand((s.T + 3,), generator=g, device="cuda")
    temp = torch.tensor([0.0, 0.8, 1.5], device="cuda")
    calls = [lambda: s.cache.attention(x, s.batch), lambda: d.cache.attention(y, d.batch), lambda: s.cache.read(s.batch, s.T)[0],
             lambda: P.verify_drafts(logits, ids, s.q_start, temp, u[:s.T], u[s.T:])[0][:s.start[-1]]]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for _ in range(10):
        for f, st in zip(calls, streams):
            with torch.cuda.stream(st):
                got.append(f())
    torch.cuda.synchronize()
    for i, z in enumerate(got):
        assert torch.equal(z, want[i % len(calls)])


def test_verify_in_graphs(torch, P):
    g = gen(torch, 1)
    R, V = 8, 151936
    logits = torch.randn((R, V), generator=g, device="cuda").to(torch.bfloat16)
    ids = logits.float().argmax(-1).to(torch.int32).roll(1)
    start = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")
    T = torch.tensor([0.0, 0.9], device="cuda")
    u, v = torch.rand(R, generator=g, device="cuda"), torch.rand(2, generator=g, device="cuda")
    P.verify_drafts(logits, ids, start, T, u, v)
    outs, graphs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(P.verify_drafts(logits, ids, start, T, u, v))
        graphs.append(gr)
    logits.copy_(torch.randn((R, V), generator=g, device="cuda"))
    want = P.verify_drafts(logits, ids, start, T, u, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("quant", [False, True])
def test_chunks_drafts_and_verification_together(torch, P, quant):
    """A prompt in chunks, then drafts: the pages and the attention of the pieces are those
    of one chunk with everything, and the drafts are accepted up to the first wrong one."""
    g = gen(torch, 21)
    hq, hkv, L, page = 8, 2, 211, 32
    qkv = torch.randn((L, (hq + 2 * hkv) * D), generator=g, device="cuda").half()
    w = [(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).half() for _ in range(2)]
    cos, sin = P.rope_tables(L, 1e6)
    at = torch.arange(L, dtype=torch.int32, device="cuda")
    pos = torch.stack([at, at // 5, at % 7]).contiguous()
    i32 = dict(dtype=torch.int32, device="cuda")

    def pieces(cuts):
        cache = P.PagedKVCache(12, hkv, page, torch.float16, quant)
        table = torch.tensor([[3, 0, 11, 7, 5, 8, 2]], **i32)
        out = []
        for a, b in zip(cuts[:-1], cuts[1:]):
            batch = P.PagedBatch(table, torch.tensor([b], **i32), torch.tensor([0, b - a], **i32))
            q = cache.append(qkv[a:b], batch, cos, sin, pos[:, a:b].contiguous(), q_norm=w[0], k_norm=w[1], sections=(24, 20, 20))
            out.append(cache.attention(q, batch))
        whole = P.PagedBatch(table, torch.tensor([L], **i32), torch.tensor([0, L], **i32))
        return torch.cat(out), cache.read(whole, tokens=L), cache

    one, kv1, c1 = pieces([0, L])
    many, kv2, c2 = pieces([0, 1, 64, 100, 200, 206, L])
    for a, b in zip(kv1, kv2):
        assert torch.equal(a, b)
    for a, b in ((c1.k_pages, c2.k_pages), (c1.v_pages, c2.v_pages)):
        assert torch.equal(a, b)
    # the two only round differently: each is within its own bound of the exact result
    u, size = 2.0 ** -11, kv1[1].float().abs().max()
    assert (one.float() - many.float()).abs().max() <= 2 * (2 * u + 2.0 ** -12) * size
    # the last five tokens as drafts: logits whose best token repeats the draft, but for the fourth
    V = 1009
    ids = torch.tensor([11, 22, 33, 44, 55], **i32)
    head = torch.randn((hq * D, V), generator=g, device="cuda").half() * 0.01
    logits = many[-5:].reshape(5, -1) @ head
    for r, t in enumerate((22, 33, 44, 77, 88)):
        logits[r, t] = 30
    got = P.verify_drafts(logits, ids, torch.tensor([0, 5], **i32), torch.zeros(1, device="cuda"),
                          torch.rand(5, generator=g, device="cuda"), torch.rand(1, generator=g, device="cuda"))
    assert got[0].tolist() == [22, 33, 44, 77, -1] and got[1].tolist() == [4]


def test_paged_path_agrees_with_the_slot_cache(torch, P, D_slots=2):
    """One axis, the decoder's own tables and one token: the pages give what dial_decode_attention gives,
    whose norm and rotation round every step to f16 (at most 6 roundings of values up to 2 |x|)."""
    import dial_cuda as lib
    g = gen(torch, 31)
    hq, hkv, L = 32, 8, 333
    qkv = torch.randn((L, (hq + 2 * hkv) * D), generator=g, device="cuda").half()
    w = torch.ones(D, device="cuda").half()
    cos, sin = P.rope_tables(L, 1e6)
    pos = torch.arange(L, dtype=torch.int32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = P.PagedKVCache(8, hkv, 64, torch.float16)
    table = torch.arange(8, **i32).flip(0).view(1, 8).contiguous()
    cache.append(qkv[:L - 1], P.PagedBatch(table, torch.tensor([L - 1], **i32), torch.tensor([0, L - 1], **i32)), cos, sin,
                 pos[:L - 1], q_norm=w, k_norm=w)
    batch = P.PagedBatch(table, torch.tensor([L], **i32), torch.tensor([0, 1], **i32), max_q=1)
    q = cache.append(qkv[L - 1:], batch, cos, sin, pos[L - 1:], q_norm=w, k_norm=w)
    got = cache.attention(q, batch)
    kc = torch.zeros((1, hkv, 512, D), device="cuda").half()
    vc = torch.zeros_like(kc)
    qo = torch.empty((L, hq, D), device="cuda").half()
    ch, sh = cos.half(), sin.half()
    slots = torch.zeros(L, **i32)
    Lb = lib.lib()
    lib.check(Lb.dial_qk_norm_rope_kv_append(qkv.data_ptr(), w.data_ptr(), w.data_ptr(), ch.data_ptr(), sh.data_ptr(),
                                             pos.data_ptr(), slots.data_ptr(), qo.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                                             lib.F16, L, hq, hkv, D, 512, 1e-6, 1, lib.stream_ptr()), "append")
    out = torch.empty((L, hq, D), device="cuda").half()
    need = Lb.dial_attention_workspace_bytes(L, hq, L)
    ws = torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")
    lib.check(Lb.dial_attention(qo.data_ptr(), kc.data_ptr(), vc.data_ptr(), pos.data_ptr(), slots.data_ptr(), out.data_ptr(),
                                ws.data_ptr(), need, lib.F16, L, hq, hkv, D, 512, L, lib.stream_ptr()), "attention")
    k, v = cache.read(P.PagedBatch(table, torch.tensor([L], **i32), torch.tensor([0, L], **i32)), tokens=L)
    assert torch.equal(v, vc[0, :, :L].transpose(0, 1))
    size = kc.float().abs().max()
    assert (k.float() - kc[0, :, :L].transpose(0, 1).float()).abs().max() <= 6 * 2.0 ** -11 * 2 * size
    # a score moves by at most 12 u |q|.|k| scale <= 12 u 128^.5 * 1.5 (unit rms rows, some larger), an output by twice that
    assert (got[0].float() - out[L - 1].float()).abs().max() <= 2 * 12 * 2.0 ** -11 * 128 ** 0.5 * 1.5 * v.float().abs().max()


@pytest.mark.parametrize("q,kv", [([4], [300]), ([90], [300])])
@pytest.mark.parametrize("quant", [False, True])
def test_a_nan_score_reaches_its_rows_and_no_others(torch, P, q, kv, quant):
    """A NaN in one value of q or of an attended key: NaN in the rows that meet it, wherever in a tile it is."""
    s = Setup(torch, P, q, kv, "f16", quant, 64, 2)
    x = torch.randn((s.T, 8, D), generator=gen(torch, 4), device="cuda").half()
    good = s.cache.attention(x, s.batch)
    for t, h in ((0, 0), (q[0] - 1, 5), (q[0] // 2, 3)):
        keep = x[t, h, 77].clone()
        x[t, h, 77] = math.nan
        got = s.cache.attention(x, s.batch)
        x[t, h, 77] = keep
        assert torch.isnan(got[t, h]).all()
        got[t, h] = good[t, h]
        assert torch.equal(got, good)
    for at in (0, 1, 2, 3, 63, 126, 131, 200):  # (all tokens see these)
        page, row = s.host_table[0][at // 64], at % 64
        where = s.scales[0][page, 1, row] if quant else s.pages[0][page, 1, row, 5]
        keep = where.clone()
        where.fill_(math.nan)
        got = s.cache.attention(x, s.batch)
        where.copy_(keep)
        assert torch.isnan(got[:, 4:]).all(), at
        assert torch.equal(got[:, :4], good[:, :4])


@pytest.mark.parametrize("act,quant", [("f16", False), ("bf16", False), ("f16", True)])
def test_decoder_over_pages(torch, P, act, quant):
    """Two prompts in chunks of one batch, then their greedy continuations as drafts: the logits
    are those of the slot-cache decoder (1e-2 of the largest, the bound its own prefill and decode
    paths are held to; int8 caches twice that), and every draft that the target repeats is accepted."""
    from dial_cuda.model import Decoder, ModelConfig
    cfg = ModelConfig(n_layers=2, hidden=512, intermediate=1024, n_heads=8, n_kv_heads=2, vocab=2048, act_dtype=act)
    dec = Decoder(cfg, n_slots=2, max_seq=128)
    g = gen(torch, 77)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, n_new = (37, 20), 5
    seqs, slot_logits = [], []
    for b, n in enumerate(lens):
        ids = torch.randint(0, cfg.vocab, (n,), generator=g, **i32)
        nxt = dec.prefill(ids, slot=b)
        toks = [ids, nxt]
        for step in range(n_new - 1):
            out = torch.empty(1, **i32)
            dec.decode_step(toks[-1], torch.tensor([n + step], **i32), torch.tensor([b], **i32), n + step + 1, out)
            toks.append(out)
        seqs.append(torch.cat(toks))
        hidden = torch.empty((n + n_new - 1, cfg.hidden), device="cuda", dtype=dec.stage.dt)
        dec.stage.embed_tokens(seqs[b][:-1], hidden)
        T = n + n_new - 1
        dec.stage.layers_forward(hidden, torch.arange(T, **i32), torch.full((T,), b, **i32), T)
        lg = torch.empty((T, cfg.vocab), device="cuda", dtype=dec.stage.dt)
        dec.stage.head_forward(hidden, torch.empty(T, **i32), logits=lg)
        slot_logits.append(lg)
    caches = dec.stage.paged_caches(10, 16, quant)
    tables = P.rope_tables(128, cfg.rope_theta)
    table = torch.tensor([[4, 9, 1], [0, 7, 3]], **i32)
    one = P.PagedBatch(table[:1], torch.tensor([1], **i32), torch.tensor([0, 1], **i32))
    with pytest.raises(ValueError, match="caches"):
        dec.forward_paged(seqs[0][:1], torch.zeros(1, **i32), one, caches[:1], tables)
    with pytest.raises(TypeError, match="ids"):
        dec.forward_paged(seqs[0][:1].long(), torch.zeros(1, **i32), one, caches, tables)

    def chunk(spans):
        ids = torch.cat([seqs[b][lo:hi] for b, (lo, hi) in enumerate(spans)])
        pos = torch.cat([torch.arange(lo, hi, **i32) for lo, hi in spans])
        start = torch.tensor([0, spans[0][1] - spans[0][0], ids.numel()], **i32)
        batch = P.PagedBatch(table, torch.tensor([hi for _, hi in spans], **i32), start)
        return ids, batch, dec.forward_paged(ids, pos, batch, caches, tables)[0]

    bound = 1e-2 * (2 if quant else 1)
    worst = 0.0
    for spans in ([(0, 16), (0, 20)], [(16, 37), (20, 20)], [(37, 41), (20, 24)]):
        ids, batch, logits = chunk(spans)
        want = torch.cat([slot_logits[b][lo:hi] for b, (lo, hi) in enumerate(spans)])
        worst = max(worst, float((logits.float() - want.float()).abs().max() / want.float().abs().max()))
    assert worst <= bound, worst
    T, u = torch.zeros(2, device="cuda"), torch.rand(ids.numel() + 2, generator=g, device="cuda")
    out, count, _ = P.verify_drafts(logits, ids, batch.q_start, T, u[:-2].contiguous(), u[-2:].contiguous())
    best = logits.float().argmax(-1).tolist()
    got, s = out.tolist(), batch.q_start.tolist()
    for b in range(2):
        n = 0
        while True:  # accepted while the draft is the target's best token
            assert got[s[b] + n] == best[s[b] + n]
            n += 1
            if s[b] + n == s[b + 1] or int(ids[s[b] + n]) != best[s[b] + n - 1]:
                break
        assert int(count[b]) == n and all(x == -1 for x in got[s[b] + n:s[b + 1]])
