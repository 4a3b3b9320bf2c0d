"""The operators that serve from packed block formats against plain 64-bit arithmetic on the GPU.

Tolerances.  u(t) = finfo(t).eps / 2 is the largest relative error of one rounding to t.

Linear: x may be held as two binary16 pieces (each drops at most 2^-11 of what it takes, so 2^-22 of the value at least is
kept; 2^-21 is allowed), every sum of K products in fp32 adds at most K u(fp32) of the sum of magnitudes, and the result is
rounded once: |y - y64| <= (2^-21 + (K + 4) 2^-24) sum |x w| + u(t) |y64|.

Attention: a score is off by at most d = scale (2^-21 + (D + 4) 2^-24) sum |q k| + 2^-23 |s| (q in pieces, the products' sum in fp32,
the scaling); a weight p = exp(s - m) is then off by a factor within exp(2 d) of one, times 1 + 2^-21 for the exponential and,
where it is rounded for a 16-bit product, 1 + u(t).  Numerator and denominator each add (T + 4) 2^-24.  So with
e = 2 max d + 2^-21 + u(16-bit t) + (T + 4) 2^-24:  |o - o64| <= 2 e sum p |v| + u(t) |o64|.  Weights are held to an
absolute step as well.  They are binary16 values w = p 2^15, times the scale of V relative to the largest 2^E of a group of tokens:
below 2^-14 binary16 has a step of 2^-24, so a rounding moves w 2^(e - E) by up to 2^-25, which is 2^-40 of the row's largest
weight times 2^E, and two such roundings (of w and of the product) 2^-39, times the largest |v| of the block, for each of T tokens.
Where p is held in two pieces the same holds: the scale of V multiplies each piece by itself, so that what the first one's
rounding drops is not in the second.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def q():
    import mptorch_b200.quant as quant

    return quant


def half_ulp(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------------- packed values in 64 bits
def field_value(code, e_bits, m_bits):
    code = code.to(torch.int64)
    e, m = (code >> m_bits) & ((1 << e_bits) - 1), code & ((1 << m_bits) - 1)
    v = torch.where(e > 0, m + (1 << m_bits), m).double() * torch.exp2((e.clamp(min=1) - ((1 << (e_bits - 1)) - 1) - m_bits).double())
    return torch.where((code >> (e_bits + m_bits)) & 1 > 0, -v, v)


def e4m3_value(code):
    return torch.where((code & 127) == 127, math.nan, field_value(code, 4, 3))


def e8m0_value(code):
    return torch.where(code == 255, math.nan, torch.exp2(code.double() - 127))


def values(codes, scales, dim):
    """What rows of codes and E8M0 scales stand for."""
    if codes.shape[-1] == dim:
        v = e4m3_value(codes)
    else:
        v = torch.stack([field_value(codes & 15, 2, 1), field_value(codes >> 4, 2, 1)], -1).flatten(-2)
    return v * e8m0_value(scales).repeat_interleave(32, -1)


def random_rows(shape, dim, elem, g, low=118, high=128):
    """Random codes (no NaN) and scales."""
    codes = torch.randint(0, 256, shape + (dim if elem == "e4m3" else dim // 2,), device="cuda", generator=g, dtype=torch.uint8)
    if elem == "e4m3":
        codes = torch.where((codes & 127) == 127, codes - 1, codes)
    return codes, torch.randint(low, high, shape + (dim // 32,), device="cuda", generator=g, dtype=torch.uint8)


# ---------------------------------------------------------------------------------- linear
def pack(n, k, fmt, g):
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    v = torch.stack([field_value(codes & 15, 2, 1), field_value(codes >> 4, 2, 1)], -1).flatten(-2)
    if fmt == "mxfp4":
        scales = torch.randint(112, 126, (n, k // 32), device="cuda", generator=g, dtype=torch.uint8)
        return codes, scales, None, v * e8m0_value(scales).repeat_interleave(32, -1)
    scales = torch.randint(0, 127, (n, k // 16), device="cuda", generator=g, dtype=torch.uint8)
    glob = torch.tensor([0.0123], device="cuda")
    return codes, scales, glob, v * e4m3_value(scales).repeat_interleave(16, -1) * glob.double()


def linear(q, x, codes, scales, glob, bias=None):
    return q.mx_linear(x, codes, scales, bias) if glob is None else q.nvfp4_linear(x, codes, scales, glob, bias)


def check_linear(y, x, w, bias=None):
    k = w.shape[1]
    want = x.double() @ w.t()
    mag = x.double().abs() @ w.abs().t()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    tol = (2.0 ** -21 + (k + 4) * 2.0 ** -24) * mag + half_ulp(x.dtype) * want.abs()
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25                                   # half a step of its subnormal numbers
    assert y.dtype == x.dtype and y.shape == want.shape
    worst = ((y.double() - want).abs() - tol).max().item()
    assert worst <= 0, "off by %g more than allowed" % worst
    # roundings of random sign: sqrt(K) of them, each at most 2^-24 of a partial sum
    norm = ((y.double() - want).norm() / want.norm()).item()
    assert norm <= 2.0 ** -21 + (math.sqrt(k) + 4) * 2.0 ** -24 + half_ulp(x.dtype)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 32), (1, 17, 64), (1, 768, 768), (2, 33, 96), (3, 257, 160), (4, 64, 1024), (5, 2304, 768), (7, 100, 4096),
                                      (8, 129, 512), (9, 48, 2080), (16, 130, 288), (17, 65, 544), (32, 200, 1056), (33, 300, 64), (64, 515, 768),
                                      (65, 31, 128), (100, 513, 224), (127, 128, 256), (130, 260, 1568), (300, 1000, 768), (515, 129, 96)])
def test_linear(q, fmt, dtype, rows, n, k):
    g = gen(rows * 7 + n + k)
    codes, scales, glob, w = pack(n, k, fmt, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(dtype)
    bias = torch.randn(n, device="cuda", generator=g).to(dtype) if (rows + n) % 2 else None
    check_linear(linear(q, x, codes, scales, glob, bias), x, w, bias)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(24, 20000, 1568), (33, 130, 1536), (40, 700, 6400), (130, 2600, 3232), (200, 4000, 1792), (260, 200, 9632), (300, 9000, 2048)])
def test_linear_long_sums(q, fmt, dtype, rows, n, k):
    """Sums that are added up in memory piece by piece, in tiles that are cut and in whole ones, twice the same bits."""
    g = gen(rows + n + k)
    codes, scales, glob, w = pack(n, k, fmt, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(dtype)
    bias = torch.randn(n, device="cuda", generator=g).to(dtype)
    y = linear(q, x, codes, scales, glob, bias)
    check_linear(y, x, w, bias)
    for _ in range(2):
        assert torch.equal(linear(q, x, codes, scales, glob, bias), y)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows", [1, 3, 24, 200])
def test_linear_range_of_x(q, fmt, rows):
    """Values of x over many orders of magnitude, within a row and between rows, keep fp32's accuracy."""
    g = gen(rows)
    codes, scales, glob, w = pack(70, 256, fmt, g)
    x = torch.randn(rows, 256, device="cuda", generator=g) * torch.exp2(torch.randint(-8, 9, (rows, 256), device="cuda", generator=g).float())
    x = x * torch.exp2(torch.randint(-60, 60, (rows, 1), device="cuda", generator=g).float())
    y = linear(q, x, codes, scales, glob)
    want, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    assert ((y.double() - want).abs() <= (2.0 ** -21 + 260 * 2.0 ** -24) * mag + 2.0 ** -24 * want.abs()).all()
    one = x.clone()
    one[:] = 0
    one[:, 5] = 2.0 ** -100
    assert torch.equal(linear(q, one, codes, scales, glob).double(), (one.double() @ w.t()).float().double())
    zero = torch.zeros_like(x)
    assert torch.equal(linear(q, zero, codes, scales, glob), zero[:, :1].expand(rows, 70))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 5, 40, 150])
def test_linear_specials(q, fmt, dtype, rows):
    """NaN and infinities of x stay in their rows; a NaN scale in its output."""
    g = gen(3)
    codes, scales, glob, w = pack(40, 128, fmt, g)
    scales[7, 1] = 255 if fmt == "mxfp4" else 127
    x = torch.randn(rows, 128, device="cuda", generator=g).to(dtype)
    clean = linear(q, x, codes, scales, glob)
    assert clean[:, 7].isnan().all() and clean[:, :7].isfinite().all() and clean[:, 8:].isfinite().all()
    bad = x.clone()
    bad[-1, 3] = math.nan
    y = linear(q, bad, codes, scales, glob)
    assert y[-1].isnan().all() and torch.equal(y[:-1].nan_to_num(7), clean[:-1].nan_to_num(7))
    bad = x.clone()
    bad[0, 9] = math.inf
    y, want = linear(q, bad, codes, scales, glob), bad.float() @ torch.cat([w[:7], w[8:]]).float().t()
    y = torch.cat([y[:, :7], y[:, 8:]], 1)
    assert torch.equal(y[0].isnan(), want[0].isnan()) and torch.equal(y[0].float()[~want[0].isnan()], want[0][~want[0].isnan()])
    assert torch.equal(y[1:], torch.cat([clean[1:, :7], clean[1:, 8:]], 1))


def test_linear_extreme_scales(q):
    """E8M0 scales from end to end of their range, against rows of x that bring the products back into range."""
    codes = torch.full((3, 32), 0x22, device="cuda", dtype=torch.uint8)           # ones
    scales = torch.tensor([[0, 0], [127, 127], [254, 254]], device="cuda", dtype=torch.uint8)
    for e in (-100, 0, 100):
        for rows in (1, 20, 140):
            x = torch.full((rows, 64), 2.0 ** e, device="cuda")
            want = 64.0 * torch.tensor([2.0 ** -127, 1.0, 2.0 ** 127], device="cuda", dtype=torch.float64) * 2.0 ** e
            assert torch.equal(q.mx_linear(x, codes, scales), want.float().expand(rows, 3))


def test_linear_shapes_strides_and_quantizers(q):
    g = gen(11)
    w = torch.randn(96, 160, device="cuda", generator=g) * 0.02
    wq, scales, codes = q.mx_quantize(w, "e2m1", 32, return_scales=True, return_codes=True)
    nq, _, glob, ncodes, nscales = q.nvfp4_quantize(w, None, return_scales=True, return_codes=True)
    x = torch.randn(2, 3, 320, device="cuda", generator=g)[..., ::2]              # a strided view, three dimensions
    y = q.mx_linear(x, codes, scales)
    assert y.shape == (2, 3, 96)
    check_linear(y.flatten(0, 1), x.flatten(0, 1), wq.double())
    check_linear(q.nvfp4_linear(x, ncodes, nscales, glob).flatten(0, 1), x.flatten(0, 1), nq.double())
    assert torch.equal(q.nvfp4_linear(x, ncodes, nscales, glob), q.nvfp4_linear(x, ncodes, nscales, float(glob)))
    assert q.mx_linear(x[0, 0], codes, scales).shape == (96,)
    assert torch.equal(q.mx_linear(x[0, 0], codes, scales), q.mx_linear(x[0, :1], codes, scales)[0])
    assert q.mx_linear(x[:0], codes, scales).shape == (0, 3, 96)
    assert q.mx_linear(x, codes[:0], scales[:0]).shape == (2, 3, 0)
    odd = torch.randn(4 * 160 + 1, device="cuda", generator=g)[1:].view(4, 160)    # an address that is a multiple of 4 only
    assert torch.equal(q.mx_linear(odd, codes, scales), q.mx_linear(odd.clone(), codes, scales))
    odd = odd.bfloat16()
    pad = torch.empty(4 * 160 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(4, 160).copy_(odd)
    assert torch.equal(q.mx_linear(pad, codes, scales), q.mx_linear(odd, codes, scales))
    assert torch.equal(q.mx_linear(x, codes, scales), q.mx_linear(x, codes, scales))


@pytest.mark.parametrize("rows", [1, 5, 12, 40, 200])
def test_linear_slices_of_a_weight_and_no_inputs(q, rows):
    """Rows of a packed weight (scales that begin anywhere), one output, and no inputs at all."""
    g = gen(rows)
    for fmt, k in (("mxfp4", 96), ("mxfp4", 1120), ("nvfp4", 96), ("nvfp4", 544)):
        codes, scales, glob, w = pack(300, k, fmt, g)
        x = torch.randn(rows, k, device="cuda", generator=g)
        for lo, hi in ((1, 2), (7, 140), (131, 300)):
            check_linear(linear(q, x, codes[lo:hi], scales[lo:hi], glob), x, w[lo:hi])
    bias = torch.randn(9, device="cuda", generator=g)
    none = torch.zeros(9, 0, device="cuda", dtype=torch.uint8)
    assert torch.equal(q.mx_linear(torch.zeros(rows, 0, device="cuda"), none, none, bias), bias.expand(rows, 9))


# ---------------------------------------------------------------------------------- the cache
def place(lens, page, g, extra=2):
    """A page table over pages in random order (-1 behind the last one) and the number of pages."""
    counts = [-(-n // page) for n in lens]
    total, width = sum(counts) + extra, max(counts + [1])
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    pages, at = torch.full((len(lens), width), -1, device="cuda", dtype=torch.int32), 0
    for i, n in enumerate(counts):
        pages[i, :n] = order[at:at + n]
        at += n
    return pages, total


def i32(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


def cumulative(new):
    return i32([0] + list(torch.tensor(new).cumsum(0)))


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,page", [(32, 1, 8), (64, 3, 16), (96, 2, 64), (128, 4, 32), (256, 1, 256)])
def test_cache_write_and_read(q, elem, dtype, dim, heads, page):
    g = gen(dim)
    new, lens = [5, 1, 40, 0, 3], [5, 33, 40, 12, 2]                              # the last: one row stands before the first token
    pages, total = place(lens, page, g)
    cache = q.MXCache.empty(total, heads, dim, page, elem)
    for t in cache:
        t.random_(0, 256)
    before = [t.clone() for t in cache]
    qkv = torch.randn(49, heads * dim * 3, device="cuda", generator=g).to(dtype)  # k and v as views of one projection
    k, v = qkv[:, heads * dim:2 * heads * dim].view(49, heads, dim), qkv[:, 2 * heads * dim:].view(49, heads, dim)
    k[7, 0, 3] = math.inf
    v[8, heads - 1, dim - 1] = math.nan
    v[9] = 0
    k[10] *= 2.0 ** -14
    starts = cumulative(new)
    q.mx_cache_write(k, v, cache, pages, i32(lens), starts)
    kr, vr = q.mx_cache_read(cache, pages, i32(lens), 49, starts)
    hit = torch.zeros(total, heads, page, dtype=torch.bool, device="cuda")
    row = 0
    for s, (n, length) in enumerate(zip(new, lens)):
        for i in range(n):
            pos = length - n + i
            if pos >= 0:
                p, o = int(pages[s, pos // page]), pos % page
                hit[p, :, o] = True
                for x, codes, scales, back in ((k, cache[0], cache[1], kr), (v, cache[2], cache[3], vr)):
                    held, sc, cd = q.mx_quantize(x[row].float(), elem, 32, return_scales=True, return_codes=True)
                    assert torch.equal(codes[p, :, o], cd) and torch.equal(scales[p, :, o], sc)
                    assert torch.equal(back[row].nan_to_num(9), held.nan_to_num(9)) and torch.equal(back[row].isnan(), held.isnan())
            else:
                assert not kr[row].any() and not vr[row].any()
            row += 1
    for t, b in zip(cache, before):
        assert torch.equal(t[~hit], b[~hit])
    low = q.mx_cache_read(cache, pages, i32(lens), 49, starts, dtype=dtype)
    assert torch.equal(low[0].nan_to_num(9), kr.to(dtype).nan_to_num(9)) and low[1].dtype == dtype


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
def test_cache_uniform_padded_and_missing_pages(q, elem):
    g = gen(5)
    pages, total = place([24, 24, 24], 8, g)
    pages[1, 1], pages[2, 0] = -1, total + 5                                       # tokens 8..15 of one, 0..7 of the other: no page
    lens = i32([24, 24, 3])
    a, b = q.MXCache.empty(total, 2, 64, 8, elem), q.MXCache.empty(total, 2, 64, 8, elem)
    big = torch.randn(3, 2, 20, 65, device="cuda", generator=g)
    k, v = big[..., 1:].transpose(1, 2), big.flip(0)[..., :64].transpose(1, 2)     # [3, 20, 2, 64], rows that are not aligned
    q.mx_cache_write(k, v, a, pages, lens)
    q.mx_cache_write(k.contiguous(), v.contiguous(), b, pages, lens)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    kr, vr = q.mx_cache_read(a, pages, lens, 20)
    want = q.mx_quantize(k.contiguous(), elem, 32)
    want[1, 4:12] = 0
    want[2] = 0                                                                    # 17 rows before its first token, 3 in no page
    assert torch.equal(kr, want)
    # more tokens than the table has places for: those behind it are neither written nor read
    q.mx_cache_write(k[:1, :4], v[:1, :4], a, pages[:1], i32([26]))
    kr, _ = q.mx_cache_read(a, pages[:1], i32([26]), 4)
    assert torch.equal(kr[0, :2], q.mx_quantize(k[0, :2].contiguous(), elem, 32)) and not kr[0, 2:].any()
    # nothing at all
    q.mx_cache_write(k[:, :0], v[:, :0], a, pages, lens)
    assert q.mx_cache_read(a, pages, lens, 0)[0].shape == (3, 0, 2, 64)
    q.mx_cache_write(k[:0], v[:0], a, pages[:0], lens[:0])
    kr, vr = q.mx_cache_read(a, pages, lens, 7, i32([0, 2, 2, 4]))                 # rows behind the last sequence
    assert not kr[4:].any() and not vr[4:].any()


# ---------------------------------------------------------------------------------- attention
def reference(qry, cache, pages, lens, new, dim, scale, window=0, sinks=0):
    """Row by row in 64 bits: (outputs, allowed error) for rows in order; ``new`` rows of each sequence."""
    heads, group, page = cache[0].shape[1], qry.shape[1] // cache[0].shape[1], cache[0].shape[2]
    out, tol, at, u = torch.zeros(qry.shape, device="cuda", dtype=torch.float64), torch.zeros(qry.shape, device="cuda", dtype=torch.float64), 0, half_ulp(qry.dtype)
    for s, n in enumerate(new):
        if n == 0:
            continue
        length = min(int(lens[s]), pages.shape[1] * page)
        rows = qry[at:at + n].double()                                             # [n, heads * group, dim]
        pos = int(lens[s]) - n + torch.arange(n, device="cuda")[:, None]
        t = torch.arange(max(length, 0), device="cuda")
        table = pages[s].long()
        there = (table >= 0) & (table < cache[0].shape[0])
        slot = table.clamp(0, cache[0].shape[0] - 1)[t // page]
        seen = (t <= pos) & there[t // page]
        if window:
            seen &= (t > pos - window) | (t < sinks)
        for h in range(heads):
            k, v = (values(cache[i][slot, h, t % page], cache[i + 1][slot, h, t % page], dim) for i in (0, 2))
            for j in range(h * group, (h + 1) * group):
                x = rows[:, j]
                some = seen.any(1)
                sc = torch.where(seen, (x @ k.t()) * scale, -math.inf)
                p = torch.where(some[:, None], torch.softmax(sc, -1), 0.0)
                # a masked token takes no part, whatever it holds
                o = torch.stack([p[i][seen[i]] @ v[seen[i]] for i in range(n)])
                d = torch.where(seen, abs(scale) * (2.0 ** -21 + (dim + 4) * 2.0 ** -24) * (x.abs() @ k.abs().t()) + 2.0 ** -23 * sc.abs(), 0.0).amax(-1) if len(t) else torch.zeros(n, device="cuda", dtype=torch.float64)
                e = 2 * d + 2.0 ** -21 + (u if qry.dtype != torch.float32 else 0.0) + (len(t) + 4) * 2.0 ** -24
                out[at:at + n, j] = o
                step = len(t) * 2.0 ** -39
                most = v.abs().nan_to_num(0).unflatten(-1, (-1, 32)).amax((0, 2)).repeat_interleave(32) if len(t) else 0.0
                tol[at:at + n, j] = 2 * e[:, None] * torch.stack([p[i][seen[i]] @ v[seen[i]].abs() for i in range(n)]) + u * o.abs() + step * most
        at += n
    return out, tol + (2.0 ** -25 if qry.dtype == torch.float16 else 0.0)


def check_attention(got, want, tol):
    assert torch.equal(got.isnan(), want.isnan())
    worst = ((got.double() - want).abs() - tol).nan_to_num(0, 0, 0).max().item() if got.numel() else 0
    assert worst <= 0, "off by %g more than allowed" % worst


def setup(q, lens, new, heads, group, dim, page, elem, dtype, seed, uniform=False):
    g = gen(seed)
    pages, total = place(lens, page, g)
    cache = q.MXCache(*random_rows((total, heads, page), dim, elem, g), *random_rows((total, heads, page), dim, elem, g))
    shape = (len(new), new[0]) if uniform else (sum(new),)
    qry = (torch.randn(shape + (heads * group, dim), device="cuda", generator=g) * (0.05 if elem == "e4m3" else 1.0)).to(dtype)
    return qry, cache, pages, i32(lens), (None if uniform else cumulative(new))


SHAPES = [  # lens, new, kv heads, group, dim, page
    ([1, 7, 130, 0], [1, 1, 1, 1], 2, 1, 64, 16), ([300, 17, 64, 65, 1000], [1] * 5, 1, 8, 128, 64), ([129, 31], [1, 1], 3, 4, 96, 8),
    ([2100], [1], 2, 2, 32, 32), ([513, 200], [1, 1], 2, 3, 256, 128), ([77, 260, 5], [1] * 3, 1, 16, 192, 16), ([6000, 3], [1, 1], 1, 5, 64, 64)]
CHUNKS = [([40, 9, 300], [40, 2, 33], 2, 1, 64, 16), ([200], [200], 1, 4, 128, 64), ([700, 130, 1], [129, 130, 1], 2, 2, 128, 32),
          ([90, 0, 260], [64, 0, 128], 3, 1, 32, 8), ([150, 400], [17, 65], 1, 8, 96, 128), ([333], [300], 1, 2, 256, 16), ([260, 70], [200, 70], 1, 3, 192, 64)]


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(SHAPES)))
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_attention_one_token(q, elem, dtype, case, window, sinks):
    lens, new, heads, group, dim, page = SHAPES[case]
    qry, cache, pages, ln, starts = setup(q, lens, new, heads, group, dim, page, elem, dtype, case, uniform=True)
    got = q.mx_attention(qry, cache, pages, ln, window=window, sinks=sinks)
    want, tol = reference(qry.flatten(0, 1), cache, pages, lens, new, dim, 1 / math.sqrt(dim), window, sinks)
    check_attention(got.flatten(0, 1), want, tol)


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(CHUNKS)))
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5), (1, 0)])
def test_attention_chunks(q, elem, dtype, case, window, sinks):
    lens, new, heads, group, dim, page = CHUNKS[case]
    qry, cache, pages, ln, starts = setup(q, lens, new, heads, group, dim, page, elem, dtype, 50 + case)
    got = q.mx_attention(qry, cache, pages, ln, starts, scale=0.11, window=window, sinks=sinks)
    want, tol = reference(qry, cache, pages, lens, new, dim, 0.11, window, sinks)
    check_attention(got, want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group", [(64, 1), (96, 2), (128, 1), (192, 1), (256, 1)])
def test_attention_chunks_over_long_contexts(q, dtype, dim, group):
    """Many pieces of tokens for each row tile, in row tiles that are cut and in whole ones, twice the same bits."""
    lens, new = [2000, 1000, 333, 2600], [250, 300, 100, 129]
    qry, cache, pages, ln, starts = setup(q, lens, new, 4, group, dim, 16, "e4m3", dtype, dim)
    got = q.mx_attention(qry, cache, pages, ln, starts, scale=0.05)
    want, tol = reference(qry, cache, pages, lens, new, dim, 0.05)
    check_attention(got, want, tol)
    # errors of random sign: their norm stays well below the bound on each
    norm = ((got.double() - want).norm() / want.norm()).item()
    assert norm < (4e-6 if dtype == torch.float32 else 2 * half_ulp(dtype))
    for _ in range(3):
        assert torch.equal(q.mx_attention(qry, cache, pages, ln, starts, scale=0.05), got)


FORMS = [([70, 33], [1, 1], 1, 4), ([70, 33, 260], [9, 20, 130], 1, 2), ([190], [180], 2, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_masked_places_hold_anything(q, dtype, form, dim):
    """NaN scales and codes behind the last token, in pages that are not there and where a row's mask hides them change
    nothing; a NaN that a row sees makes that row NaN (in K all of it, in V the block)."""
    lens, new, heads, group = FORMS[form]
    qry, cache, pages, ln, starts = setup(q, lens, new, heads, group, dim, 16, "e4m3", dtype, 80 + form)
    clean = q.mx_attention(qry, cache, pages, ln, starts)
    used = torch.zeros(cache[0].shape[0], 16, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for t in range(n):
            used[pages[s, t // 16], t % 16] = True
    dirty = q.MXCache(*(torch.where(used[:, None, :, None], t, 255) for t in cache))
    assert torch.equal(q.mx_attention(qry, dirty, pages, ln, starts), clean)
    # the last token of the first sequence: NaN in K, then in one block of V
    p, o = int(pages[0, (lens[0] - 1) // 16]), (lens[0] - 1) % 16
    for which in (1, 3):
        bad = q.MXCache(*(t.clone() for t in cache))
        bad[which][p, 0, o, 1] = 255
        got = q.mx_attention(qry, bad, pages, ln, starts)
        want, tol = reference(qry, bad, pages, lens, new, dim, 1 / math.sqrt(dim))
        assert want.isnan().any() and not want.isnan().all()
        check_attention(got, want, tol)
        keep = ~want.isnan()
        assert torch.equal(got[keep], clean[keep])
    # the same in the middle, under a window that hides it from some rows
    p, o = int(pages[0, (lens[0] // 2) // 16]), (lens[0] // 2) % 16
    for which in (1, 3):
        bad = q.MXCache(*(t.clone() for t in cache))
        bad[which][p, 0, o, 0] = 255
        got = q.mx_attention(qry, bad, pages, ln, starts, window=20, sinks=2)
        want, tol = reference(qry, bad, pages, lens, new, dim, 1 / math.sqrt(dim), 20, 2)
        check_attention(got, want, tol)
    # a row of q with a NaN or an infinity
    for x in (math.nan, math.inf):
        bad = qry.clone()
        bad[-1, 1, 5] = x
        got = q.mx_attention(bad, cache, pages, ln, starts)
        assert got[-1, 1].isnan().all()
        assert torch.equal(got[:-1], clean[:-1]) and torch.equal(got[-1, 0], clean[-1, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 40, 150])
def test_attention_rows_that_see_nothing(q, dtype, new):
    lens = [0, new + 30, max(new - 25, 0), 17]
    qry, cache, pages, ln, _ = setup(q, [max(n, 1) for n in lens], [new] * 4, 2, 2, 64, 8, "e4m3", dtype, new, uniform=True)
    ln = i32(lens)
    pages[1, 1] = -1                                                              # a hole
    pages[3, :] = cache[0].shape[0]                                               # nothing there at all
    got = q.mx_attention(qry, cache, pages, ln)
    want, tol = reference(qry.flatten(0, 1), cache, pages, lens, [new] * 4, 64, 1 / 8)
    check_attention(got.flatten(0, 1), want, tol)
    assert not got[0].any() and not got[3].any() and got[1].any()
    # more tokens than the table has places for
    ln[1] = pages.shape[1] * 8 + 5
    got = q.mx_attention(qry, cache, pages, ln)
    want, tol = reference(qry.flatten(0, 1), cache, pages, [0, int(ln[1]), lens[2], 17], [new] * 4, 64, 1 / 8)
    check_attention(got.flatten(0, 1), want, tol)
    # rows behind the last sequence: zeros, or left as they were in a tensor of the caller's
    flat, starts = qry.flatten(0, 1), cumulative([new, 1, 0, 0])
    got = q.mx_attention(flat, cache, pages, ln, starts)
    assert not got[new + 1:].any()
    mine = torch.full_like(flat, 7)
    q.mx_attention(flat, cache, pages, ln, starts, out=mine)
    assert torch.equal(mine[:new + 1], got[:new + 1]) and (mine[new + 1:] == 7).all()
    assert q.mx_attention(flat[:0], cache, pages, ln, cumulative([0] * 4)).shape == (0, 4, 64)


@pytest.mark.parametrize("new", [1, 40, 150])
def test_attention_extreme_arguments(q, new):
    """A window and sinks of any size beside rows that stand nowhere, an empty cache, a table without places."""
    lens = [new + 200, max(new - 20, 0), new]
    qry, cache, pages, ln, _ = setup(q, [max(n, 1) for n in lens], [new] * 3, 2, 2, 64, 16, "e4m3", torch.float32, new, uniform=True)
    ln = i32(lens)
    plain = q.mx_attention(qry, cache, pages, ln)
    most = 2 ** 31 - 1
    assert torch.equal(q.mx_attention(qry, cache, pages, ln, window=most), plain)
    assert torch.equal(q.mx_attention(qry, cache, pages, ln, window=most, sinks=most), plain)
    got = q.mx_attention(qry, cache, pages, ln, window=7, sinks=most)
    want, tol = reference(qry.flatten(0, 1), cache, pages, lens, [new] * 3, 64, 1 / 8)
    check_attention(got.flatten(0, 1), want, tol)
    none = q.MXCache(*(t[:0] for t in cache))
    assert not q.mx_attention(qry, none, pages, ln).any() and not q.mx_cache_read(none, pages, ln, new)[0].any()
    q.mx_cache_write(qry[:, :, :2], qry[:, :, 2:], none, pages, ln)
    assert not q.mx_attention(qry, cache, pages[:, :0].contiguous(), ln).any()
    ragged = q.mx_attention(qry.flatten(0, 1), cache, pages[:0], ln[:0], i32([0]))   # no sequences: every row is behind the last
    assert not ragged.any()


def test_two_streams_at_once(q):
    """Calls that run at the same time share nothing: each stream gets the bits that it gets alone."""
    g = gen(4)
    codes, scales, glob, _ = pack(700, 512, "nvfp4", g)
    sets = [setup(q, [n + 900, n], [n] * 2, 2, 4, 128, 32, "e4m3", torch.bfloat16, n, uniform=True) + (torch.randn(n, 512, device="cuda", generator=g),) for n in (1, 7, 90, 300)]
    call = lambda s: (q.mx_attention(*s[:4]), q.nvfp4_linear(s[5], codes, scales, glob))  # noqa: E731
    alone = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(6):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(call(s))
    torch.cuda.synchronize()
    for want, results in zip(alone, got):
        assert all(torch.equal(x, y) for r in results for x, y in zip(r, want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 30, 140])
def test_attention_strides_and_order(q, dtype, new):
    qry, cache, pages, ln, _ = setup(q, [new + 40, new + 7, new], [new] * 3, 2, 2, 96, 16, "e2m1", dtype, 9, uniform=True)
    want = q.mx_attention(qry, cache, pages, ln)
    assert torch.equal(q.mx_attention(qry.transpose(1, 2).contiguous().transpose(1, 2), cache, pages, ln), want)   # heads outside
    wide = torch.zeros(3, new, 4, 97, device="cuda", dtype=dtype)
    wide[..., 1:] = qry
    assert torch.equal(q.mx_attention(wide[..., 1:], cache, pages, ln), want)                                     # rows not aligned
    assert torch.equal(q.mx_attention(qry.transpose(2, 3).contiguous().transpose(2, 3), cache, pages, ln), want)  # dimension outside
    assert torch.equal(q.mx_attention(qry.flatten(0, 1), cache, pages, ln, cumulative([new] * 3)).view_as(want), want)
    assert torch.equal(q.mx_attention(qry, cache, pages, ln, out=torch.empty_like(qry)), want)
    assert torch.equal(q.mx_attention(qry, tuple(cache), pages, ln, window=1 << 30), want)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
@pytest.mark.parametrize("new", [1, 20, 129])
def test_attention_scales(q, scale, new):
    """No scale, a negative one, and scores far apart."""
    qry, cache, pages, ln, starts = setup(q, [new + 90], [new], 1, 2, 64, 16, "e2m1", torch.float32, 4)
    got = q.mx_attention(qry, cache, pages, ln, starts, scale=scale)
    want, tol = reference(qry, cache, pages, [new + 90], [new], 64, scale)
    check_attention(got, want, tol)


@pytest.mark.parametrize("new", [1, 30, 140])
def test_attention_scales_of_v_far_apart(q, new):
    """Tokens whose V differs by many orders of magnitude, small ones with the large weights."""
    qry, cache, pages, ln, starts = setup(q, [new + 90], [new], 1, 2, 64, 16, "e4m3", torch.float32, 6)
    g = gen(8)
    cache.v_scales.copy_(torch.randint(100, 150, cache.v_scales.shape, device="cuda", generator=g, dtype=torch.uint8))
    got = q.mx_attention(qry, cache, pages, ln, starts, scale=0.05)
    want, tol = reference(qry, cache, pages, [new + 90], [new], 64, 0.05)
    check_attention(got, want, tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 130])
def test_offsets_past_32_bits(q, dtype, new):
    """A cache of more than 2^32 bytes of codes: pages at its far end."""
    cache = q.MXCache.empty(9000, 8, 256, 256)                                     # 4.7e9 bytes of codes each for K and V
    pages, ln = i32([[8999, 8500]]), i32([256 + 140])
    g = gen(1)
    k, v = torch.randn(1, 396, 8, 256, device="cuda", generator=g).to(dtype), torch.randn(1, 396, 8, 256, device="cuda", generator=g).to(dtype)
    q.mx_cache_write(k, v, cache, pages, ln)
    kr, vr = q.mx_cache_read(cache, pages, ln, 396)
    assert torch.equal(kr, q.mx_quantize(k.float(), "e4m3", 32)) and torch.equal(vr, q.mx_quantize(v.float(), "e4m3", 32))
    qry = torch.randn(1, new, 8, 256, device="cuda", generator=g).to(dtype)
    small = q.MXCache(*(t[pages[0].long()] for t in cache))
    got = q.mx_attention(qry, cache, pages, ln)
    want, tol = reference(qry[0], small, i32([[0, 1]]), [396], [new], 256, 1 / 16)
    check_attention(got[0], want, tol)


# ---------------------------------------------------------------------------------- streams, graphs, a run of them together
@pytest.mark.parametrize("new", [1, 150])
def test_streams_and_graphs(q, new):
    """Another stream than the default, and two captured graphs replayed with new inputs in turn: eager calls give the bits."""
    g = gen(2)
    lens = [new + 700, new + 41]
    codes, scales, glob, _ = pack(256, 256, "nvfp4", g)

    def step(qry, k, v, cache, pages, ln):
        q.mx_cache_write(k, v, cache, pages, ln)
        o = q.mx_attention(qry, cache, pages, ln)
        return o, q.nvfp4_linear(o.flatten(2), codes, scales, glob)

    def inputs(seed):
        qry, cache, pages, ln, _ = setup(q, lens, [new] * 2, 2, 2, 64, 16, "e4m3", torch.bfloat16, seed, uniform=True)
        h = gen(seed + 1)
        return [qry, torch.randn(2, new, 2, 64, device="cuda", generator=h).bfloat16(), torch.randn(2, new, 2, 64, device="cuda", generator=h).bfloat16(), cache, pages, ln]

    sets = [inputs(s) for s in (21, 22)]
    eager = []
    for a in sets:
        b = [*a[:3], q.MXCache(*(t.clone() for t in a[3])), *a[4:]]
        eager.append([t.clone() for t in step(*b)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*[*sets[0][:3], q.MXCache(*(t.clone() for t in sets[0][3])), *sets[0][4:]])
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, eager[0]))
    static = [[t.clone() for t in a[:3]] + [q.MXCache(*(t.clone() for t in a[3]))] + [t.clone() for t in a[4:]] for a in sets]
    graphs, outs = [], []
    for a in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(*a))
        graphs.append(gr)
    for _ in range(3):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    for o, e in zip(outs, eager):
        assert all(torch.equal(x, y) for x, y in zip(o, e))
    # new inputs in the first graph's tensors
    for t, s in zip(static[0][:3], sets[1][:3]):
        t.copy_(s)
    for t, s in zip(static[0][3], sets[1][3]):
        t.copy_(s)
    static[0][4].copy_(sets[1][4])
    static[0][5].copy_(sets[1][5])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs[0], eager[1]))


def test_both_routes_agree(q, monkeypatch):
    from mptorch_b200 import backend as be

    if be._ext is None:
        pytest.skip("the extension is not built")
    g = gen(6)
    codes, scales, glob, _ = pack(100, 256, "nvfp4", g)
    mcodes, mscales, _, _ = pack(100, 256, "mxfp4", g)
    x, bias = torch.randn(5, 256, device="cuda", generator=g), torch.randn(100, device="cuda", generator=g)
    qry, cache, pages, ln, starts = setup(q, [30, 170], [4, 140], 2, 2, 64, 16, "e4m3", torch.float32, 3)
    k = torch.randn(144, 2, 64, device="cuda", generator=g)

    def all_of_them():
        c = q.MXCache(*(t.clone() for t in cache))
        q.mx_cache_write(k, -k, c, pages, ln, starts)
        return [q.nvfp4_linear(x, codes, scales, glob, bias), q.mx_linear(x, mcodes, mscales, bias), *c, *q.mx_cache_read(c, pages, ln, 144, starts, torch.bfloat16),
                q.mx_attention(qry, c, pages, ln, starts), q.mx_attention(qry[:4].view(2, 2, 4, 64), c, pages, ln, window=9, sinks=1)]

    a = all_of_them()
    monkeypatch.setattr(be, "_ext", None)
    assert all(torch.equal(s, t) for s, t in zip(a, all_of_them()))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(q):
    dev = torch.device("cuda", 1)
    qry, cache, pages, ln, starts = setup(q, [30, 170], [4, 140], 2, 2, 64, 16, "e4m3", torch.float32, 3)
    want = q.mx_attention(qry, cache, pages, ln, starts)
    there = q.mx_attention(qry.to(dev), q.MXCache(*(t.to(dev) for t in cache)), pages.to(dev), ln.to(dev), starts.to(dev))
    assert there.device == dev and torch.equal(there.cpu(), want.cpu())
    with pytest.raises(RuntimeError, match="expected"):
        q.mx_attention(qry.to(dev), cache, pages, ln, starts)


# ---------------------------------------------------------------------------------- few rows of the products
@pytest.mark.parametrize("dtype,rows,k", [(torch.bfloat16, 10, 6944), (torch.bfloat16, 10, 7040), (torch.bfloat16, 10, 7072), (torch.float16, 11, 6304),
                                          (torch.float16, 11, 6400), (torch.float16, 11, 6432), (torch.bfloat16, 12, 5888), (torch.bfloat16, 12, 5920),
                                          (torch.bfloat16, 15, 4640), (torch.bfloat16, 15, 4736), (torch.bfloat16, 15, 4768), (torch.float32, 5, 7040),
                                          (torch.float32, 5, 7072), (torch.float32, 6, 5888), (torch.float32, 6, 5920), (torch.bfloat16, 16, 4384),
                                          (torch.bfloat16, 1, 65536), (torch.bfloat16, 2, 35840), (torch.bfloat16, 9, 7808)])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_linear_as_much_of_x_as_shared_memory_holds(q, fmt, dtype, rows, k):
    """Sizes on both sides of what the kernel for a few rows takes."""
    g = gen(rows + k)
    codes, scales, glob, w = pack(40, k, fmt, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(dtype)
    check_linear(linear(q, x, codes, scales, glob), x, w)


# Accuracy of long float32 sums.  The tensor cores cut their running sums off, by up to 2^-23 of the sum for each 16 products.  A kernel
# that adds partial sums of S products up in fp32 is off by at most (S / 16) 2^-23 of the sum of magnitudes for the cut sums, always in
# the same direction, and by roundings of random sign, sqrt(K / S) 2^-24, for the rest.  Of one sign, where nothing cancels, that is the
# result's relative error; 2^-21 comes on top for x and the weights of a softmax in two binary16 pieces.
def cut_off_bound(part, length):
    return (part / 16) * 2.0 ** -23 + (math.sqrt(length / part) + 4) * 2.0 ** -24 + 2.0 ** -21


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows,n,k", [(1, 33000, 9600), (2, 33000, 9600), (5, 4000, 6880), (7, 20000, 4096), (8, 40, 8160), (1, 300, 32768)])
def test_linear_few_rows_sums_of_one_sign(q, fmt, rows, n, k):
    """No longer sums than 128 products are left to the tensor cores; sums that ran through were up to 4.5e-5 off."""
    g = gen(rows + n)
    codes, scales, glob, _ = pack(n, k, fmt, g)
    codes &= 0x77
    w = torch.stack([field_value(codes & 15, 2, 1), field_value(codes >> 4, 2, 1)], -1).flatten(-2)
    w = w * (e8m0_value(scales).repeat_interleave(32, -1) if glob is None else e4m3_value(scales).repeat_interleave(16, -1) * glob.double())
    x = torch.randn(rows, k, device="cuda", generator=g).abs()
    want = x.double() @ w.t()
    assert ((linear(q, x, codes, scales, glob).double() - want).norm() / want.norm()).item() <= cut_off_bound(128, k)


@pytest.mark.parametrize("lens,heads,group,dim", [([20000] * 64, 8, 1, 64), ([20000] * 16, 4, 2, 128), ([30000, 20000], 1, 1, 256), ([9000] * 40, 8, 3, 96)])
def test_attention_tokens_over_long_contexts_of_one_sign(q, lens, heads, group, dim):
    """V of one sign, float32: no longer sums than 32 tokens are left to the tensor cores.  The weights are off by what the scores
    are: 2^-21 of sum |q k| for q in two pieces, and 2^-22 for the exponential; their error is of both signs and fades in the sum."""
    qry, cache, pages, ln, _ = setup(q, lens, [1] * len(lens), heads, group, dim, 64, "e4m3", torch.float32, dim, uniform=True)
    cache.v_codes.bitwise_and_(127)
    got = q.mx_attention(qry, cache, pages, ln, scale=0.02)
    off = norm = 0.0
    for s in range(0, len(lens), max(1, len(lens) // 4)):
        t = torch.arange(lens[s], device="cuda")
        slot = pages[s].long()[t // 64]
        for h in range(heads):
            k, v = (values(cache[i][slot, h, t % 64], cache[i + 1][slot, h, t % 64], dim) for i in (0, 2))
            rows = slice(h * group, (h + 1) * group)
            o = torch.softmax((qry[s, 0, rows].double() @ k.t()) * 0.02, -1) @ v
            off += (got[s, 0, rows].double() - o).square().sum().item()
            norm += o.square().sum().item()
    assert math.sqrt(off / norm) <= cut_off_bound(32, max(lens))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("new,window,dim,group", [(1, 50, 64, 1), (1, 50, 128, 4), (6, 50, 96, 2), (20, 0, 64, 1), (20, 33, 256, 1), (160, 0, 192, 1), (160, 40, 256, 2)])
def test_attention_large_values_in_masked_places(q, elem, dtype, new, window, dim, group):
    """V that a row does not see takes no bits from what it sees, however large it is: the row is as near to 64-bit arithmetic without
    those tokens as if they were not there.  A weight is held to 2^-26 of the row's largest where V's scales are up to 2^14 apart
    (binary16 has a step of 2^-24, and weights are scaled by 2^15 before and 2^-14 after), so that of each token's |v| is allowed."""
    length = new + 200
    qry, cache, pages, ln, _ = setup(q, [length], [new], 1, group, dim, 16, elem, dtype, 5 + dim, uniform=True)
    want, tol = reference(qry[0], cache, pages, [length], [new], dim, 1 / math.sqrt(dim), window)
    t = torch.arange(length, device="cuda")
    where = (pages[0].long()[t // 16], torch.zeros_like(t), t % 16)
    v = values(cache.v_codes[where], cache.v_scales[where], dim).abs()
    hidden = [length - 1] if new > 1 else []                       # by causality from all rows but the last
    if window:
        hidden += [length - new - window - 3, length - new - window]    # too old for every row
    for scale in (140, 200, 246):
        bad = q.MXCache(*(x.clone() for x in cache))
        for h in hidden:
            bad.v_scales[pages[0, h // 16], 0, h % 16] = scale
        got = q.mx_attention(qry, bad, pages, ln, window=window)
        rows = slice(0, new - 1 if new > 1 else 1)
        check_attention(got[0, rows], want[rows], tol[rows] + 2.0 ** -26 * v.sum(0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 12])
def test_attention_large_values_with_small_weights(q, dtype, new):
    """Tokens with tiny weights and V from 2^-27 to 2^127, all in one piece of 32 tokens, beside tokens with large weights and small V."""
    dim, length = 64, new + 70
    qry, cache, pages, ln, starts = setup(q, [length], [new], 1, 2, dim, 16, "e4m3", dtype, 3)
    qry.fill_(0.25)
    cache.k_scales.fill_(127)
    cache.k_codes.fill_(0xD0)                                      # -8: a score of -16 where it stays
    for i, t in enumerate((5, 11, 40, 62)):
        cache.k_codes[pages[0, t // 16], 0, t % 16] = 0x38 if i % 2 else 0x30         # 1 and 1/2
    g = gen(9)
    cache.v_scales.copy_(torch.randint(100, 240, cache.v_scales.shape, device="cuda", generator=g, dtype=torch.uint8))
    scale = 64.0                                                   # the other weights are e^-9216 and less: nothing, whatever V is
    for t in (5, 11, 40, 62):
        cache.v_scales[pages[0, t // 16], 0, t % 16] = 107
    got = q.mx_attention(qry, cache, pages, ln, starts, scale=scale)
    t = torch.tensor([11, 62], device="cuda")                      # score 1024, the halves 512
    slot = pages[0].long()[t // 16]
    v = values(cache.v_codes[slot, 0, t % 16], cache.v_scales[slot, 0, t % 16], dim)
    want = v.mean(0).expand(got.shape)
    tol = (2.0 ** -26 + 2.0 ** -20 + half_ulp(dtype)) * v.abs().sum(0) + (2.0 ** -24 if dtype == torch.float16 else 0.0)
    check_attention(got, want, tol.expand(got.shape))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("new,window", [(1, 0), (20, 0), (20, 25), (200, 0), (200, 64)])
def test_attention_values_beyond_fp32_in_masked_places(q, elem, dtype, new, window):
    """Scale bytes up to 254, with codes that take their values out of fp32's range, where a row does not see them."""
    length, dim = new + 90, 64
    qry, cache, pages, ln, _ = setup(q, [length], [new], 1, 2, dim, 16, elem, dtype, 12, uniform=True)
    want, tol = reference(qry[0], cache, pages, [length], [new], dim, 1 / 8, window)
    bad = q.MXCache(*(x.clone() for x in cache))
    for h in ([length - 1] if new > 1 else []) + ([length - new - window - 2] if window else []):
        for scales, codes in ((bad.k_scales, bad.k_codes), (bad.v_scales, bad.v_codes)):
            scales[pages[0, h // 16], 0, h % 16] = 254
            codes[pages[0, h // 16], 0, h % 16] = 0x7E if elem == "e4m3" else 0x77
    got = q.mx_attention(qry, bad, pages, ln, window=window)
    rows = slice(0, new - 1 if new > 1 else 1)
    t = torch.arange(length, device="cuda")
    where = (pages[0].long()[t // 16], torch.zeros_like(t), t % 16)
    v = values(cache.v_codes[where], cache.v_scales[where], dim).abs()
    check_attention(got[0, rows], want[rows], tol[rows] + 2.0 ** -26 * v.sum(0))      # as above


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 40, 200])
@pytest.mark.parametrize("x", [math.inf, -math.inf, math.nan])
def test_attention_infinite_rows_of_q(q, dtype, new, x):
    """Scores that are all minus infinity are no empty row: their softmax is NaN, as that of plus infinity.  A row that sees nothing
    gives zeros, whatever it holds."""
    qry, cache, pages, ln, _ = setup(q, [new], [new], 1, 2, 64, 16, "e4m3", dtype, 5, uniform=True)
    clean = q.mx_attention(qry, cache, pages, ln)
    cache.k_codes[pages[0, 0], 0, 0] = 0x38                        # the first token's K: ones
    cache.k_scales[pages[0, 0], 0, 0] = 127
    same = q.mx_attention(qry, cache, pages, ln)
    for where in (slice(None), 3):                                 # every element, or one beside finite ones
        bad = qry.clone()
        bad[0, 0, 0, where] = x
        bad[0, -1, 1, where] = x
        got = q.mx_attention(bad, cache, pages, ln)
        assert got[0, 0, 0].isnan().all() and got[0, -1, 1].isnan().all()
        got[0, 0, 0], got[0, -1, 1] = same[0, 0, 0], same[0, -1, 1]
        assert torch.equal(got, same)
    assert clean.isfinite().all()
    bad = torch.full_like(qry, x)
    assert not q.mx_attention(bad, cache, torch.full_like(pages, -1), ln).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 70, 96), (5, 70, 1120), (24, 300, 1024), (33, 1000, 2080), (40, 129, 6400), (200, 4000, 512), (300, 20000, 96)])
def test_linear_blocks_of_very_different_size(q, dtype, rows, n, k):
    """MXFP4 blocks far below their row's largest count in full, whatever the number of rows: x that is zero where the large ones are
    reads them out exactly, and together with others sums keep the bound of `test_linear`."""
    g = gen(rows + n + k)
    codes, scales, _, _ = pack(n, k, "mxfp4", g)
    some = torch.rand(n, 1, device="cuda", generator=g) < 0.3                     # rows with such blocks
    at = torch.randint(0, 2, scales.shape, device="cuda", generator=g).bool() & some
    at[:, 0], at[:, 1] = False, some[:, 0]
    low = (scales.int() - torch.randint(33, 100, scales.shape, device="cuda", generator=g)).clamp(min=0).to(torch.uint8)
    scales = torch.where(at, low, scales)
    zero = torch.rand(n, k // 32, device="cuda", generator=g) < 0.05               # and blocks of zeros, whose scale is the smallest
    scales = torch.where(zero, 0, scales).to(torch.uint8)
    codes = torch.where(zero.repeat_interleave(16, -1), 0, codes).to(torch.uint8)
    v = torch.stack([field_value(codes & 15, 2, 1), field_value(codes >> 4, 2, 1)], -1).flatten(-2)
    w = v * e8m0_value(scales).repeat_interleave(32, -1)
    x = torch.randn(rows, k, device="cuda", generator=g).to(dtype)
    bias = torch.randn(n, device="cuda", generator=g).to(dtype)
    check_linear(q.mx_linear(x, codes, scales, bias), x, w, bias)
    far = x.clone()
    far[:, :32] = 0
    far[:, 64:] = 0                                                               # the second block alone
    y = q.mx_linear(far, codes, scales)
    want, mag = far.double() @ w.t(), far.double().abs() @ w.abs().t()
    # float16 results have a step of 2^-24 at the least, float32 and bfloat16 sums one of 2^-149
    low = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -148
    assert ((y.double() - want).abs() <= (2.0 ** -21 + 36 * 2.0 ** -24) * mag + half_ulp(dtype) * want.abs() + low).all()
    unit = torch.zeros(rows, k, device="cuda", dtype=torch.float32)
    unit[:, 40] = 1
    assert torch.equal(q.mx_linear(unit, codes, scales).double(), w[:, 40].expand(rows, n))
    part = q.mx_linear(x, codes[17:60], scales[17:60], bias[17:60])
    check_linear(part, x, w[17:60], bias[17:60])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 4)])
def test_attention_chunks_after_a_wait_that_ran_out(q, dtype, dim, group):
    """Nothing is left unwritten or joined from old shares: what was computed before is right, all else is NaN.  (The library is told
    that a wait ran out; none does.)"""
    from mptorch_b200 import _cabi

    lens, new = [2000, 1000, 333, 2600, 150], [250, 300, 100, 129, 1]
    qry, cache, pages, ln, starts = setup(q, lens, new, 8, group, dim, 16, "e4m3", dtype, dim)
    clean = q.mx_attention(qry, cache, pages, ln, starts)
    assert clean.isfinite().all()
    held = []
    try:
        for part in (0, 1, 2):
            _cabi.lib().mpt_test_attention_wait_runs_out(part)
            out = torch.full_like(qry, 7)
            q.mx_attention(qry, cache, pages, ln, starts, out=out)
            row_nan = out.isnan().all(-1)
            assert torch.equal(row_nan, out.isnan().any(-1)) and torch.equal(out[~row_nan], clean[~row_nan])
            held.append(int((~row_nan).sum()))
    finally:
        _cabi.lib().mpt_test_attention_wait_runs_out(-1)
    assert held[0] == 0 and held[0] <= held[1] <= held[2]
    assert torch.equal(q.mx_attention(qry, cache, pages, ln, starts), clean)


@pytest.mark.parametrize("route", ["ext", "ctypes"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 20, 300])
def test_attention_into_the_memory_of_q(q, dtype, new, route, monkeypatch):
    """out is q, begins some rows before or behind it, or has its heads in another order."""
    from mptorch_b200 import backend as be

    if route == "ctypes":
        monkeypatch.setattr(be, "_ext", None)
    lens = [new + 300, new + 40, new]
    qry, cache, pages, ln, _ = setup(q, lens, [new] * 3, 2, 4, 64, 16, "e4m3", dtype, 7, uniform=True)
    want = q.mx_attention(qry, cache, pages, ln)
    mine = qry.clone()
    assert q.mx_attention(mine, cache, pages, ln, out=mine) is not None and torch.equal(mine, want)
    for shift in (-3, -1, 1, 2):
        room = torch.zeros(qry.numel() + 6 * 64, device="cuda", dtype=dtype)
        there = room[3 * 64:3 * 64 + qry.numel()].view_as(qry).copy_(qry)
        out = room[(3 + shift) * 64:(3 + shift) * 64 + qry.numel()].view_as(qry)
        q.mx_attention(there, cache, pages, ln, out=out)
        assert torch.equal(out, want)
    version = out._version
    q.mx_attention(qry, cache, pages, ln, out=out)
    assert out._version > version                                   # autograd learns of it
    turned = qry.transpose(1, 2).contiguous()                       # [sequences, heads, new, dim]
    out = turned.view(qry.shape)
    q.mx_attention(turned.transpose(1, 2), cache, pages, ln, out=out)
    assert torch.equal(out, want)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [32, 96, 1120, 4128, 8224])
def test_linear_one_row_finds_its_largest_value_anywhere(q, fmt, dtype, k):
    """A row is scaled by its largest magnitude, wherever it stands: a power of two beside zeros comes back exactly times the weight."""
    g = gen(k)
    codes, scales, glob, w = pack(24, k, fmt, g)
    for at in {0, 7, 8, 31, k // 2, k - 32, k - 9, k - 1}:
        x = torch.zeros(1, k, device="cuda", dtype=dtype)
        x[0, at] = 2.0 ** 60
        x[0, (at + 11) % k] = 2.0 ** 45
        want = x.double() @ w.t()
        got = linear(q, x, codes, scales, glob).double()
        assert ((got - want).abs() <= (2.0 ** -22 + half_ulp(dtype)) * want.abs() + 2.0 ** -22 * (x.double().abs() @ w.abs().t())).all()


@pytest.mark.parametrize("fmt,fold,rows,n,k", [("nvfp4", 1536, 300, 4000, 9152), ("nvfp4", 1536, 33, 18889, 9152), ("nvfp4", 1536, 130, 300, 9632),
                                               ("mxfp4", 4096, 300, 4000, 32768), ("mxfp4", 4096, 40, 20000, 20000)])
def test_linear_many_rows_sums_of_one_sign(q, fmt, fold, rows, n, k):
    """float32 rows: sums of the tile kernel are added up in memory after 1536 (NVFP4) or 4096 (MXFP4) products, where there are tiles
    enough for a CTA to have whole ones.  Sums that ran through were 2.2e-5 off after 9152 products and 6.9e-5 after 32768."""
    g = gen(rows + n)
    codes, scales, glob, _ = pack(n, k, fmt, g)
    codes &= 0x77
    w = torch.stack([field_value(codes & 15, 2, 1), field_value(codes >> 4, 2, 1)], -1).flatten(-2)
    w = w * (e8m0_value(scales).repeat_interleave(32, -1) if glob is None else e4m3_value(scales).repeat_interleave(16, -1) * glob.double())
    x = torch.randn(rows, k, device="cuda", generator=g).abs()
    want = x.double() @ w.t()
    assert ((linear(q, x, codes, scales, glob).double() - want).norm() / want.norm()).item() <= cut_off_bound(fold, k)


@pytest.mark.parametrize("dim,group", [(32, 1), (64, 1), (96, 2), (128, 1)])
def test_attention_chunks_over_long_contexts_of_one_sign(q, dim, group):
    """float32 chunks: sums are added up in registers after 512 tokens.  There are rows enough here for a CTA to have whole contexts."""
    lens, new, heads = [12000, 11000], [256, 300], 16 // group
    qry, cache, pages, ln, starts = setup(q, lens, new, heads, group, dim, 64, "e4m3", torch.float32, dim)
    cache.v_codes.bitwise_and_(127)
    got, at, off, norm = q.mx_attention(qry, cache, pages, ln, starts, scale=0.02), 0, 0.0, 0.0
    for s, n in enumerate(new):
        t = torch.arange(lens[s], device="cuda")
        slot = pages[s].long()[t // 64]
        hidden = t > lens[s] - n + torch.arange(n, device="cuda")[:, None]
        for h in range(0, heads, 3):
            k, v = (values(cache[i][slot, h, t % 64], cache[i + 1][slot, h, t % 64], dim) for i in (0, 2))
            for j in range(h * group, (h + 1) * group):
                o = torch.softmax(((qry[at:at + n, j].double() @ k.t()) * 0.02).masked_fill(hidden, -math.inf), -1) @ v
                off += (got[at:at + n, j].double() - o).square().sum().item()
                norm += o.square().sum().item()
        at += n
    assert math.sqrt(off / norm) <= cut_off_bound(512, max(lens))


@pytest.mark.parametrize("rows", [3, 24, 300])
def test_mxfp4_products_in_graphs_and_on_streams(q, rows):
    """Weights with and without far blocks: two captured graphs replayed in turn with new inputs, and calls on several streams at once."""
    g = gen(rows)
    sets = []
    for i in range(2):
        codes, scales, _, _ = pack(3000, 1056, "mxfp4", g)
        if i:
            scales[::7, 3] = 30
        sets.append([torch.randn(rows, 1056, device="cuda", generator=g), codes, scales])
    eager = [[q.mx_linear(x, c, s) for x in (sets[0][0], sets[1][0])] for _, c, s in sets]
    static = [[t.clone() for t in a] for a in sets]
    graphs, outs = [], []
    for a in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(q.mx_linear(*a))
        graphs.append(gr)
    for turn in range(3):
        for i, gr in enumerate(graphs):
            static[i][0].copy_(sets[turn % 2][0])
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, e[turn % 2]) for o, e in zip(outs, eager))
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [[] for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(q.mx_linear(sets[i & 1][0], *sets[i >> 1][1:]))
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        assert all(torch.equal(r, eager[i >> 1][i & 1]) for r in results)


@pytest.mark.parametrize("new", [1, 20])
def test_attention_of_blocks_of_zeros_and_single_large_values(q, new):
    """V with blocks of zeros (whose scale is the smallest) and with one token far above the others, each row against 64 bits."""
    dim, length = 96, new + 150
    for dtype in TYPES:
        qry, cache, pages, ln, starts = setup(q, [length], [new], 2, 2, dim, 16, "e4m3", dtype, 31)
        g = gen(new)
        zero = torch.rand(cache.v_scales.shape, device="cuda", generator=g) < 0.4
        cache.v_scales.masked_fill_(zero, 0)
        cache.v_codes.masked_fill_(zero.repeat_interleave(32, -1), 0)
        want, tol = reference(qry, cache, pages, [length], [new], dim, 1 / math.sqrt(dim))
        check_attention(q.mx_attention(qry, cache, pages, ln, starts), want, tol)
        for t, scale in ((3, 200), (90, 160), (91, 90)):
            cache.v_scales[pages[0, t // 16], 1, t % 16, 1] = scale
        got = q.mx_attention(qry, cache, pages, ln, starts)
        want, tol = reference(qry, cache, pages, [length], [new], dim, 1 / math.sqrt(dim))
        if dtype == torch.float16:                                  # (a result beyond its range is an infinity)
            got, want = got.float().clamp(-65504, 65504), want.clamp(-65504, 65504)
        check_attention(got, want, tol)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows,n,k", [(70000, 48, 32768), (70000, 32800, 64), (1, 300000, 32768), (20, 300000, 32768)])
def test_linear_offsets_past_32_bits(q, fmt, rows, n, k):
    """x, y, and packed weights of more than 2^31 elements or 2^32 bytes: places at the far end and in between."""
    g = gen(rows + n)
    codes, scales = torch.empty(n, k // 2, device="cuda", dtype=torch.uint8), torch.empty(n, k // (32 if fmt == "mxfp4" else 16), device="cuda", dtype=torch.uint8)
    for i in range(0, n, 20000):
        codes[i:i + 20000].random_(0, 256, generator=g)
        scales[i:i + 20000].random_(112, 126, generator=g) if fmt == "mxfp4" else scales[i:i + 20000].random_(0, 127, generator=g)
    if fmt == "mxfp4":
        scales[-1, 0] = 20                                          # a block of its own kernel, at the far end
    glob = None if fmt == "mxfp4" else torch.tensor([0.5], device="cuda")
    x = torch.empty(rows, k, device="cuda", dtype=torch.bfloat16)
    for i in range(0, rows, 10000):
        x[i:i + 10000].normal_(generator=g)
    y = linear(q, x, codes, scales, glob)
    at_m = torch.unique(torch.tensor([0, 1, rows // 3, rows - 2, rows - 1], device="cuda").clamp(0, rows - 1))
    at_n = torch.unique(torch.tensor([0, 17, n // 2, n - 3, n - 1], device="cuda"))
    c, s = codes[at_n], scales[at_n]
    v = torch.stack([field_value(c & 15, 2, 1), field_value(c >> 4, 2, 1)], -1).flatten(-2)
    w = v * (e8m0_value(s).repeat_interleave(32, -1) if glob is None else e4m3_value(s).repeat_interleave(16, -1) * glob.double())
    check_linear(y[at_m][:, at_n], x[at_m], w)
    # and that nothing is zero or left out on a larger part
    mean = y[-min(rows, 50):, -min(n, 1000):].float().abs().mean().item()
    assert 0.5 < mean / y[:min(rows, 50), :min(n, 1000)].float().abs().mean().item() < 2
