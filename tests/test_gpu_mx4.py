"""The MX4 operators on the GPU against their plain 64-bit forms."""
import threading

import numpy as np
import pytest

import _mx4 as mx
import simplang_amd as sa

pytestmark = pytest.mark.gpu

F, U = np.float32, np.uint8


def _dev(x, dev, pad=0, shift=0, fill=0):
    """x on the device in rows pad elements apart, the first shift elements into its memory."""
    import torch
    x = torch.from_numpy(np.ascontiguousarray(x))
    m, k = x.shape
    buf = torch.full((shift + m * (k + pad) + 1,), fill, dtype=x.dtype, device=dev)
    v = buf[shift:shift + m * (k + pad)].view(m, k + pad)[:, :k]
    v.copy_(x)
    return v


def _x(rng, m, k):
    """Values of very different sizes, zeros, whole blocks of zeros, borders and subnormals."""
    x = (rng.standard_normal((m, k)) * 2.0 ** rng.integers(-6, 7, (m, k))).astype(F)
    x[rng.random((m, k)) < 0.05] = 0
    half = np.concatenate([mx.VALUES, mx.MIDS, [7, 7.99, 5.0000005]])
    on = rng.random((m, k)) < 0.3
    x[on] = (half[rng.integers(0, len(half), on.sum())] * np.where(rng.random(on.sum()) < .5, -1, 1)).astype(F)
    for j in range(mx.blocks(k)):
        b = x[:, 32 * j:32 * j + 32]
        p = rng.integers(0, 12, m)
        b[p == 0] = 0
        b[p == 1] *= F(2.0 ** -120)
        b[p == 2] *= F(2.0 ** -60) * F(2.0 ** -70)
        b[p == 3] *= F(2.0 ** 110)
        b[p == 4] = F(-0.0)
        b[p == 5] = F(2.0 ** -149)
    return x


SIZES = [1, 2, 7, 31, 32, 33, 63, 64, 65, 100, 255, 256, 768, 1533, 3200]


@pytest.mark.parametrize("k", SIZES)
@pytest.mark.parametrize("m", [1, 5, 130])
def test_quantize_and_back(dev, m, k):
    import torch
    rng = np.random.default_rng(100 * k + m)
    x = _x(rng, m, k)
    codes, scales = mx.quantize(x)
    for pad, shift in ((0, 0), (3, 1), (32, 16)):
        dx = _dev(x, dev, pad, shift, 9)
        c = _dev(np.zeros_like(codes), dev, pad, shift, 77)
        s = _dev(np.zeros_like(scales), dev, pad, shift, 78)
        out = _dev(np.zeros_like(x), dev, pad, shift, 5)
        sa.quantize_mx4(dx, c, s)
        sa.dequantize_mx4(c, s, out)
        torch.cuda.synchronize()
        assert np.array_equal(s.cpu().numpy(), scales)
        assert np.array_equal(c.cpu().numpy(), codes)
        assert np.array_equal(out.cpu().numpy(), mx.values(codes, scales)[:, :k])
        for buf, n, f in ((c, codes.shape[1], 77), (s, scales.shape[1], 78), (out, k, 5)):
            whole = buf._base[shift:shift + m * (n + pad)].view(m, n + pad)
            assert (whole[:, n:] == f).all() and (buf._base[:shift] == f).all()


# sizes with more than 2^15 blocks of 32, in four blocks to a thread, the last workgroup's not all
# there: small rows and long ones, rows that end inside a block, a byte and four elements
MANY = [(717, 1533), (33000, 30), (1100, 1024), (5, 250007)]
# 2^24 elements and more, values past the caches where rows lie on 16 bytes: rows of 4099 elements 4100
# apart and of 4096; the same where the rows' stride or the first row is off 16 bytes
LARGE = [(4100, 4099, 1, 0), (4100, 4099, 5, 0), (4100, 4096, 0, 4), (4100, 4099, 2, 0), (4100, 4099, 1, 1),
         (4100, 4096, 0, 3), (17_000_000, 1, 3, 0)]


@pytest.mark.parametrize("m, k, pad, shift", [(m, k, *p) for m, k in MANY for p in ((0, 0), (3, 1), (32, 16))] + LARGE)
def test_quantize_and_back_of_many_blocks(dev, m, k, pad, shift):
    import torch
    rng = np.random.default_rng(m + k)
    some = min(m, 3000)  # rows of their own; the others repeat them
    x = _x(rng, some, k)
    codes, scales = mx.quantize(x)
    vals = mx.values(codes, scales)[:, :k].astype(F)
    idx = torch.from_numpy(rng.integers(0, some, m)).to(dev)

    def rows(v, fill):
        buf = torch.full((shift + m * (v.shape[1] + pad) + 1,), fill, dtype=torch.from_numpy(v).dtype, device=dev)
        return buf, buf[shift:-1].view(m, -1)[:, :v.shape[1]]

    _, dx = rows(x, 9)
    dx.copy_(torch.from_numpy(x).to(dev)[idx])
    outs = [rows(v, f) for v, f in ((codes, 77), (scales, 78), (vals, 5))]
    sa.quantize_mx4(dx, outs[0][1], outs[1][1])
    sa.dequantize_mx4(outs[0][1], outs[1][1], outs[2][1])
    for (buf, got), want, f in zip(outs, (codes, scales, vals), (77, 78, 5)):
        assert torch.equal(got, torch.from_numpy(want).to(dev)[idx])
        gaps = buf[shift:-1].view(m, -1)[:, want.shape[1]:]
        assert (gaps == f).all() and (buf[:shift] == f).all() and (buf[-1] == f).all()


def test_quantize_marks_blocks_that_are_not_finite(dev):
    import torch
    x = np.ones((6, 100), F)
    x[0, 3], x[1, 40], x[2, 99], x[3, 64:96] = np.nan, np.inf, -np.inf, np.nan
    x[4, 31] = np.float32(3.4e38)
    codes, scales = mx.quantize(x)
    c, s = (torch.zeros(v.shape, dtype=torch.uint8, device=dev) for v in (codes, scales))
    out = torch.zeros(x.shape, device=dev)
    sa.quantize_mx4(torch.from_numpy(x).to(dev), c, s)
    sa.dequantize_mx4(c, s, out)
    assert np.array_equal(s.cpu().numpy(), scales) and np.array_equal(c.cpu().numpy(), codes)
    assert (scales == 255).sum() == 4
    assert np.array_equal(out.cpu().numpy(), mx.values(codes, scales)[:, :100], equal_nan=True)


def test_dequantize_all_codes_and_scales(dev):
    import torch
    c = np.tile(np.arange(256, dtype=U), (256, 1))
    s = np.repeat(np.arange(256, dtype=U)[:, None], 16, 1)
    out = torch.zeros((256, 512), device=dev)
    sa.dequantize_mx4(torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev), out)
    with np.errstate(over="ignore"):
        want = mx.values(c, s).astype(F)
    assert np.array_equal(out.cpu().numpy(), want, equal_nan=True)


def _call(dev, gate, a, sa_, bs, pads=(0, 0), shifts=(0, 0), out_pad=0):
    """The product of A and the matrices bs on the device, out's gaps and ends checked."""
    import torch
    m, n = a.shape[0], bs[0][0].shape[0]
    args = []
    for c, s in ((a, sa_), *bs):
        # the bytes behind the rows are codes and scales that would show
        args += [_dev(c, dev, pads[0], shifts[0], 0x77), _dev(s, dev, pads[1], shifts[1], 255)]
    buf = torch.full((m + 2, n + out_pad), 12345.0, device=dev)
    out = buf[1:m + 1, :n]
    (sa.swiglu_mx4 if gate else sa.matmul_mx4)(*args, out)
    torch.cuda.synchronize()
    got = buf.cpu().numpy()
    assert (got[0] == 12345).all() and (got[-1] == 12345).all() and (got[:, n:] == 12345).all()
    return got[1:m + 1, :n]


def _check(got, want, tol):
    with np.errstate(all="ignore"):
        bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want))
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


def _want(gate, a, s, bs):
    g, tg = mx.product(a, s, *bs[0])
    return mx.gated(g, tg, *mx.product(a, s, *bs[1])) if gate else (g, tg)


MS = [1, 2, 3, 8, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 128, 129, 200, 257]
KBS = [1, 2, 8, 15, 16, 17, 32, 33, 48, 63, 64, 65, 80, 127, 128, 144, 208, 255, 256, 272, 384, 767, 1024]
NS = [1, 3, 15, 16, 17, 31, 32, 33, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300]


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("i", range(69))
def test_product_sizes(dev, gate, i):
    """Every row count, width and column count with several others, rows at any address."""
    m, kb, n = MS[i % len(MS)], KBS[i % len(KBS)], NS[(i * 7 + i // 19) % len(NS)]
    rng = np.random.default_rng(i)
    a, s = mx.codes(rng, m, kb)
    bs = [mx.codes(rng, n, kb) for _ in range(1 + gate)]
    got = _call(dev, gate, a, s, bs, *[((0, 0), (0, 0)), ((16, 16), (16, 16)), ((3, 1), (1, 1)), ((0, 2), (4, 2))][i % 4],
                out_pad=(0, 0, 1, 4)[i // 4 % 4])
    want, tol = _want(gate, a, s, bs)
    if not gate:
        assert np.array_equal(got, want)  # sums of these codes are exact in fp32
    _check(got, want, tol)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("lo, hi", [(100, 150), (60, 190), (0, 40), (200, 255), (0, 255)])
@pytest.mark.parametrize("m, kb, n", [(1, 400, 70), (16, 1000, 40), (40, 321, 65), (150, 640, 140), (300, 1024, 300)])
def test_product_of_scales_far_apart(dev, gate, lo, hi, m, kb, n):
    rng = np.random.default_rng(lo + hi + m)
    a, s = mx.codes(rng, m, kb, lo, hi)
    bs = [mx.codes(rng, n, kb, lo, hi) for _ in range(1 + gate)]
    got = _call(dev, gate, a, s, bs)
    want, tol = _want(gate, a, s, bs)
    with np.errstate(all="ignore"):
        # where a partial sum may pass fp32's range, infinities and what follows from them are right
        size = sum(np.abs(mx.values(a, s)) @ np.abs(mx.values(*b)).T for b in bs)
        if gate:
            size = np.maximum(size, np.abs(want) + tol)
    ok = size < 3e38
    _check(got[ok], want[ok], tol[ok])


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("m, kb, n", [(1, 100, 33), (20, 272, 65), (140, 256, 130), (300, 512, 300)])
def test_nan_scales_touch_their_rows_only(dev, gate, m, kb, n):
    rng = np.random.default_rng(m)
    a, s = mx.codes(rng, m, kb)
    bs = [mx.codes(rng, n, kb) for _ in range(1 + gate)]
    s[m // 2, -1] = 255
    bs[-1][1][n // 3, 0] = 255
    got = _call(dev, gate, a, s, bs)
    assert np.isnan(got[m // 2]).all() and np.isnan(got[:, n // 3]).all()
    s[m // 2, -1] = 0
    bs[-1][1][n // 3, 0] = 0
    want, tol = _want(gate, a, s, bs)
    keep = np.ix_(np.arange(m) != m // 2, np.arange(n) != n // 3)
    _check(got[keep], want[keep], tol[keep])


def _values64(codes, scales):
    """mx.values on the device."""
    import torch
    c = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1).int()
    v = torch.from_numpy(mx.VALUES).to(codes.device)[c & 7]
    v = torch.where(c > 7, -v, v)
    two = ((scales.long() - 127 + 1023) << 52).view(torch.float64)
    return v * two.repeat_interleave(32, 1)[:, :v.shape[1]]


# rows, code bytes of a row, columns, and the kernel that takes the product and the gate
FORMS = [
    (64, 1600, 2800, "ring64x2", "ring64x2"),
    (33, 2320, 3000, "skinny", "skinny"),
    (129, 2304, 1500, "ring64x2", "ring64x2"),
    (300, 1024, 3000, "ring64x2", "ring128"),
    (250, 912, 3000, "ring64x2", "ring128"),
    (100, 1088, 8200, "ring128", "ring64"),
    (257, 640, 8320, "ring64", "ring128"),
    (600, 272, 4100, "ring64", "ring128"),
    (513, 2448, 2050, "ring128", "ring64"),
    (900, 80, 9000, "ring128", "dma"),
    (130, 640, 9000, "ring128", "ring128"),
    (1100, 1104, 1100, "ring128", "ring64"),
    (1000, 144, 6000, "ring128", "dma"),
    (600, 2336, 2000, "ring128", "ring64"),
    (65, 6000, 1000, "ring64x2", "ring64x2"),
    (3000, 800, 2900, "ring128", "dma"),
    (2900, 1040, 3008, "dma", "dma"),
    (2817, 1088, 3089, "dma", "dma"),
    (3100, 1200, 2900, "dma", "dma"),
    (6000, 1024, 6000, "dma", "dma"),
    (3000, 2064, 2900, "dma", "dma"),
    (70, 2048, 4096, "ring64x2", "ring64x2"),
    (200, 768, 12000, "ring64", "ring128"),
    (150, 1600, 8200, "ring128", "ring128"),
    (300, 2400, 1500, "ring64x2", "ring64x2"),
]
# pad, shift: rows that do not lie on 16 bytes
ODD = [
    (600, 272, 4100, 1, 0, "ring64d", "ring128d"),
    (1000, 144, 6000, 1, 0, "ring128d", "ring128d"),
    (200, 768, 12000, 1, 0, "ring64d", "ring64d"),
    (250, 912, 3000, 3, 4, "ring64x2d", "ring128d"),
    (300, 2400, 1500, 3, 0, "ring64x2d", "ring64x2d"),
    (64, 1600, 2800, 1, 0, "ring64x2d", "ring64x2d"),
    (300, 1100, 2051, 0, 0, "ring64x2d", "ring128d"),
    (300, 1101, 2051, 0, 0, "ring64x2d", "ring128d"),
    (65, 2500, 3001, 0, 0, "ring64x2d", "ring64x2d"),
    (65, 6001, 1000, 0, 0, "ring64x2", "ring64x2"),
    (700, 767, 2051, 0, 0, "ring128d", "ring64d"),
    (700, 767, 2051, 2, 0, "ring128d", "ring64d"),
    (200, 1601, 4000, 0, 0, "ring64x2d", "ring128d"),
    (513, 2447, 2050, 0, 0, "ring128d", "ring64"),
    (100, 1087, 8200, 0, 4, "ring128d", "ring64d"),
    (33, 2319, 3000, 0, 0, "skinny", "skinny"),
    (2900, 1001, 3000, 0, 0, "dma", "dma"),
    (120, 17, 3000, 0, 0, "skinny", "skinny"),
    (120, 31, 3000, 0, 0, "skinny", "skinny"),
    (120, 16, 3000, 3, 0, "skinny", "skinny"),
    (120, 15, 3000, 0, 0, "skinny", "skinny"),
    (130, 385, 9000, 0, 0, "ring128d", "ring64d"),
    (20, 1451, 9000, 0, 0, "skinny", "skinny"),
    (200, 129, 5000, 0, 0, "ring64d", "ring64d"),
    (200, 1153, 5000, 0, 0, "ring128d", "ring64d"),
    (700, 767, 2051, 0, 1, "ring128", "ring64"),
    (200, 1601, 4000, 0, 3, "ring64x2", "ring128"),
    (300, 1100, 2051, 0, 2, "ring64x2", "ring128"),
    (2900, 1001, 3000, 0, 5, "dma", "dma"),
    (65, 1250, 3001, 0, 0, "ring64x2d", "ring64x2d"),
    (150, 1252, 3001, 0, 0, "ring64x2d", "ring128d"),
    (65, 1250, 3001, 1, 0, "ring64x2d", "ring64x2d"),
]


def _on_device(dev, seed, m, kb, n, gate, lo=126, hi=129, pad=0, shift=0):
    import torch
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def codes(r):
        out = []
        for w, a, b in ((kb, 0, 256), (-(-kb // 16), lo, hi)):
            buf = torch.randint(a, b, (shift + r * (w + pad) + 1,), generator=g, device=dev, dtype=torch.uint8)
            out.append(buf[shift:shift + r * (w + pad)].view(r, w + pad)[:, :w])
        return out

    return [codes(r) for r in (m, n, n)[:2 + gate]]


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("m, kb, n, pad, shift, plain, gated", ODD)
def test_every_form_of_odd_rows(dev, gate, m, kb, n, pad, shift, plain, gated):
    _form(dev, gate, m, kb, n, pad, shift, 1, gated if gate else plain)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("pad, shift, opad", [(0, 0, 0), (32, 16, 4), (3, 1, 1)])
@pytest.mark.parametrize("m, kb, n, plain, gated", FORMS)
def test_every_form(dev, gate, m, kb, n, plain, gated, pad, shift, opad):
    """Rows as they lie, padded, and at odd addresses."""
    _form(dev, gate, m, kb, n, pad, shift, opad, gated if gate else plain)


def _form(dev, gate, m, kb, n, pad, shift, opad, form):
    """Against 64 bits on the device, every output, by the form that is expected."""
    import torch
    a, *bs = _on_device(dev, m + kb, m, kb, n, gate, pad=pad, shift=shift)
    buf = torch.full((m + 2, n + opad), 5.0, device=dev)
    out = buf[1:-1, :n]
    f = sa.swiglu_mx4 if gate else sa.matmul_mx4
    f(*a, *[x for b in bs for x in b], out)  # (makes room for the scratch that the form takes)
    out.fill_(6)
    sa.timing(True)
    try:
        f(*a, *[x for b in bs for x in b], out)
        assert sa.timing_query("mx4_" + form)[1] == 1
    finally:
        sa.timing(False)
    assert (buf[0] == 5).all() and (buf[-1] == 5).all() and (buf[:, n:] == 5).all()
    want = [_values64(*a) @ _values64(*b).t().contiguous() for b in bs]
    if not gate:
        assert torch.equal(out.double(), want[0])  # the sums are exact in fp32
    else:
        w = want[0] / (1 + torch.exp(-want[0])) * want[1]
        assert ((out.double() - w).abs() <= mx.GATE * mx.EPS * w.abs() + 2.0 ** -119 * want[1].abs()).all()


@pytest.mark.parametrize("lo, hi", [(100, 150), (40, 200), (0, 40)])
@pytest.mark.parametrize("m, kb, n", [(129, 2304, 1500), (600, 272, 4100), (130, 640, 9000), (2900, 1040, 3008)])
def test_every_form_with_scales_far_apart(dev, m, kb, n, lo, hi):
    import torch
    a, b = _on_device(dev, m + lo, m, kb, n, False, lo, hi)
    a[1][m // 2, -1] = 255  # one row with a NaN
    out = sa.matmul_mx4(*a, *b, torch.empty((m, n), device=dev))
    assert out[m // 2].isnan().all()
    a[1][m // 2, -1] = 0
    va, vb = _values64(*a), _values64(*b)
    size = va.abs() @ vb.abs().t().contiguous()
    tol = (a[1].shape[1] + 20) * (mx.EPS * size + 2.0 ** -150)
    off = (out.double() - va @ vb.t().contiguous()).abs()
    off[m // 2] = 0
    # beyond fp32's range infinities and what follows from them are right
    assert ((off <= tol) | (size > 3e38)).all()


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("shifts", [(0, 0), (4, 0), (1, 0), (0, 3), (2, 8)])
@pytest.mark.parametrize("pads", [(0, 0), (1, 0), (2, 1), (3, 3), (4, 2)])
@pytest.mark.parametrize("m, kb, n", [(5, 97, 60), (20, 129, 40), (40, 130, 100), (130, 259, 300), (300, 388, 500)])
def test_codes_and_scales_at_addresses_of_their_own(dev, gate, m, kb, n, pads, shifts):
    rng = np.random.default_rng(m + kb)
    a, *bs = [mx.codes(rng, r, kb) for r in (m, n, n)[:2 + gate]]
    got = _call(dev, gate, *a, bs, pads, shifts, 3)
    want, tol = _want(gate, *a, bs)
    _check(got, want, tol)


def test_millions_of_rows(dev):
    import torch
    m, kb = 2_200_000, 3
    a, b = _on_device(dev, 1, m, kb, 300, False)
    out = sa.matmul_mx4(*a, *b, torch.empty((m, 300), device=dev))
    assert torch.equal(out[-5000:].double(), _values64(*[x[-5000:] for x in a]) @ _values64(*b).t().contiguous())
    assert torch.equal(out[:5000].double(), _values64(*[x[:5000] for x in a]) @ _values64(*b).t().contiguous())


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("m, n", [(1, 540_000_000), (1_080_000_000, 17)])
def test_more_blocks_than_a_launch_has(dev, gate, m, n):
    """Below K = 2 every sum is exact; the ends, the middle, and where a launch ends."""
    import torch
    if torch.cuda.mem_get_info()[0] < (100 << 30):
        pytest.skip("needs 100 GB")
    g = torch.Generator(device=dev).manual_seed(m)
    ops = [[torch.randint(0, 256, (r, 1), dtype=torch.uint8, device=dev, generator=g),
            torch.randint(122, 128, (r, 1), dtype=torch.uint8, device=dev, generator=g)]
           for r in ((m, n, n) if gate else (m, n))]
    f = sa.swiglu_mx4 if gate else sa.matmul_mx4
    out = f(*sum(ops, []), torch.full((m, n), float("nan"), device=dev))
    many = max(m, n)
    blocks = (2**31 - 1) // 64  # of a launch, of one wave
    for at in (0, many // 2, (16 * blocks if m == 1 else 64 * (blocks // 2)) - 500, many - 1000):
        cut = slice(at, at + 1000)
        rows, cols = (cut, slice(None)) if m > 1 else (slice(None), cut)
        h = [_values64(*[x[r] for x in o]) for o, r in zip(ops, (rows, cols, cols))]
        want = h[0] @ h[1].t().contiguous()
        got = out[rows, cols].double()
        if gate:
            want = want / (1 + torch.exp(-want)) * (h[0] @ h[2].t().contiguous())
            assert ((got - want).abs() <= mx.GATE * 2.0**-24 * want.abs()).all()
        else:
            assert torch.equal(got, want)


def test_product_of_nothing_is_zero(dev):
    import torch
    for m, n in ((1, 1), (20, 300)):
        e = lambda r: torch.zeros((r, 0), dtype=torch.uint8, device=dev)
        for f, k in ((sa.matmul_mx4, 1), (sa.swiglu_mx4, 2)):
            out = torch.full((m, n), 7.0, device=dev)
            f(e(m), e(m), *[x for _ in range(k) for x in (e(n), e(n))], out)
            assert (out == 0).all()


@pytest.mark.parametrize("m, k, h", [(1, 768, 2048), (5, 100, 333), (33, 512, 288), (200, 768, 2048)])
def test_feed_forward_block(dev, m, k, h):
    """quantize, swiglu_mx4, quantize, matmul_mx4, each on what the one before left."""
    import torch
    rng = np.random.default_rng(m)
    x = rng.standard_normal((m, k)).astype(F)
    w1, w3 = ((rng.standard_normal((h, k)) * 0.05).astype(F) for _ in range(2))
    w2 = (rng.standard_normal((k, h)) * 0.05).astype(F)

    def q(t):
        c = torch.empty((t.shape[0], (t.shape[1] + 1) // 2), dtype=torch.uint8, device=dev)
        s = torch.empty((t.shape[0], mx.blocks(t.shape[1])), dtype=torch.uint8, device=dev)
        return sa.quantize_mx4(t, c, s)

    on = lambda v: torch.from_numpy(v).to(dev)
    W1, W3, W2, X = q(on(w1)), q(on(w3)), q(on(w2)), q(on(x))
    hid = sa.swiglu_mx4(*X, *W1, *W3, torch.empty((m, h), device=dev))
    out = sa.matmul_mx4(*q(hid), *W2, torch.empty((m, k), device=dev))
    want, tol = mx.gated(*mx.product(*mx.quantize(x), *mx.quantize(w1)),
                         *mx.product(*mx.quantize(x), *mx.quantize(w3)))
    _check(hid.cpu().numpy(), want, tol)
    # the second half from the hidden values that the first half left: a code may lie on
    # either side of a border that the last bit of a hidden value crosses
    want, tol = mx.product(*mx.quantize(hid.cpu().numpy()), *mx.quantize(w2))
    _check(out.cpu().numpy(), want, tol)


@pytest.mark.parametrize("m, kb, n", [(1, 384, 300), (40, 384, 300), (200, 1024, 520), (2900, 1040, 1500)])
def test_gate_of_the_two_products(dev, m, kb, n):
    """The gate of what matmul_mx4 gives, and near the swiglu operator's (whose expf, sum,
    quotient and product are within 2 units, 2, 2.5 and 1 EPS)."""
    import torch
    a, *bs = _on_device(dev, m, m, kb, n, True, 116, 122)
    g, u, both, other = (torch.empty((m, n), device=dev) for _ in range(4))
    sa.matmul_mx4(*a, *bs[0], g)
    sa.matmul_mx4(*a, *bs[1], u)
    sa.swiglu_mx4(*a, *bs[0], *bs[1], both)
    sa.swiglu(g.view(-1), u.view(-1), other.view(-1), m * n)
    gd, ud = g.double(), u.double()
    want = gd / (1 + torch.exp(-gd)) * ud
    low = 2.0 ** -119 * ud.abs()
    assert ((both.double() - want).abs() <= mx.GATE * mx.EPS * want.abs() + low).all()
    assert ((both.double() - other.double()).abs() <= (mx.GATE + 10) * mx.EPS * want.abs() + low).all()


def test_gate_at_its_ends(dev):
    """Sums that are large, subnormal and infinite through the gate."""
    import torch
    # row i of A is 2^e_i in one element; W1's columns have +-1, W3's 1
    es = [-140, -126, -20, -1, 0, 3, 4, 5, 6, 6.5, 7, 20, 100, 120]
    m = len(es)
    a, s = np.zeros((m, 16), U), np.full((m, 1), 127, U)
    a[:, 0] = 2                                       # 1.0
    s[:, 0] = [max(int(e), -127) + 127 for e in es]
    w1, w3 = np.zeros((2, 16), U), np.zeros((2, 16), U)
    w1[:, 0], w3[:, 0] = [2, 10], 2
    t = np.full((2, 1), 127, U)
    got = _call(dev, True, a, s, [(w1, t), (w3, t)])
    want, tol = _want(True, a, s, [(w1, t), (w3, t)])
    ok = np.abs(want) < 3e38
    _check(got[ok], want[ok], tol[ok])
    assert (got[-1] == [np.inf, 0]).all() and (got[-2] == [np.inf, 0]).all()
    big = np.full((1, 1), 254, U)
    a[0, 0] = 7                                       # 6 * 2^127: infinite in fp32
    got = _call(dev, True, a[:1], big, [(w1[:1], t[:1]), (w3[:1], np.full((1, 1), 1, U))])
    assert np.isinf(got[0, 0]) and got[0, 0] > 0


def test_gate_where_exp_overflows(dev):
    """g = -96 to -80 in steps of 1/64, from binary digits in blocks of their own (exact)."""
    n = np.arange(80 * 64, 96 * 64 + 1)
    digits = n[:, None] >> np.arange(12, -1, -1) & 1
    a, s = np.zeros((len(n), 13 * 16), U), np.tile(127 + 6 - np.arange(13), (len(n), 1)).astype(U)
    a[:, ::16] = 2 * digits                           # 1.0
    w1, w3, t = np.zeros((1, 13 * 16), U), np.zeros((1, 13 * 16), U), np.full((1, 13), 127, U)
    w1[:, ::16], w3[:, 0] = 10, 2                     # -1.0; 64 (every n has that digit)
    for m in (len(n), 5):
        for at in range(0, len(n), m):
            cut = slice(at, at + m)
            got = _call(dev, True, a[cut], s[cut], [(w1, t), (w3, t)])[:, 0]
            g = -n[cut] / 64
            want = g / (1 + np.exp(-g)) * 64
            assert (np.abs(got - want) <= mx.GATE * mx.EPS * np.abs(want) + 2.0 ** -119 * 64).all()
            assert (got[g < -88.73] == 0).all()
            if at > 200:
                break


@pytest.mark.parametrize("m, n", [(5, 1), (1025, 1), (1025, 300), (1025, 6000)])
def test_gate_keeps_what_a_large_factor_brings_back(dev, m, n):
    """g = -96 to -80 as above with u = +-2^120: silu is 2^-108 to 2^-122 and normal in fp32, and zero
    only where exp(-g) overflows (-88.7228394).  The bound is the gate's own roundings, and
    two for the halves of the smallest subnormal in g / 4 and in silu."""
    import torch
    d = np.arange(80 * 64, 96 * 64 + 1)[-m:] if m > 5 else np.array([5595, 5620, 5650, 5678, 5679])
    digits = d[:, None] >> np.arange(12, -1, -1) & 1
    a, s = np.zeros((m, 13 * 16), U), np.tile(127 + 6 - np.arange(13), (m, 1)).astype(U)
    a[:, ::16] = 2 * digits                           # 1.0
    w1, w3 = np.zeros((n, 13 * 16), U), np.zeros((n, 13 * 16), U)
    t, t3 = np.full((n, 13), 127, U), np.full((n, 13), 127 + 114, U)
    sign = np.where(np.arange(n) % 3 == 1, -1, 1)
    w1[:, ::16], w3[:, 0] = 10, np.where(sign < 0, 10, 2)  # -1.0; 64 (every d has that digit) times 2^114
    on = [torch.from_numpy(v).to(dev) for v in (a, s, w1, t, w3, t3)]
    out = sa.swiglu_mx4(*on, torch.full((m, n), 3.0, device=dev)).double()
    g = torch.from_numpy(-d / 64).to(dev)
    u = torch.from_numpy(sign * 2.0 ** 120).to(dev)
    silu = g / (1 + torch.exp(-g)) * (g > -88.7228394)
    want = silu[:, None] * u
    assert ((out - want).abs() <= mx.GATE * mx.EPS * want.abs() + 2.0 ** -148 * u.abs()).all()


@pytest.mark.parametrize("m, n", [(3, 700), (1500, 700), (1500, 4000)])
def test_gate_over_its_range(dev, m, n):
    """g from -128 to 128 and down to 2^-36, u from 2^-100 to 2^19."""
    import torch
    rng = np.random.default_rng(m + n)
    # g = the sum of 13 digits times 2^(6 - j), exact; columns turn the sign and scale it by 2^-c
    d = rng.integers(0, 2 ** 13, m)
    a, s = np.zeros((m, 14 * 16), U), np.tile(127 + 6 - np.arange(14), (m, 1)).astype(U)
    a[:, :13 * 16:16] = 2 * (d[:, None] >> np.arange(12, -1, -1) & 1)
    a[:, 13 * 16], s[:, 13] = 2, 127                  # 1.0: u's
    w1, w3 = np.zeros((n, 14 * 16), U), np.zeros((n, 14 * 16), U)
    t, t3 = np.full((n, 14), 127, U), np.full((n, 14), 127, U)
    minus = rng.random(n) < 0.6
    c = rng.integers(0, 31, n) * (rng.random(n) < 0.7)
    w1[:, :13 * 16:16] = np.where(minus, 10, 2)[:, None]
    t[:] = 127 - c[:, None]
    e = rng.integers(-100, 20, n)
    w3[:, 13 * 16], t3[:] = 2, (127 + e)[:, None]
    on = [torch.from_numpy(v).to(dev) for v in (a, s, w1, t, w3, t3)]
    out = sa.swiglu_mx4(*on, torch.full((m, n), 3.0, device=dev)).double()
    g = torch.from_numpy(np.where(minus, -1, 1) * 2.0 ** -c * (d / 64)[:, None]).to(dev)
    u = torch.from_numpy(2.0 ** e).to(dev)
    want = g / (1 + torch.exp(-g)) * (g > -88.7228394) * u
    assert ((out - want).abs() <= mx.GATE * mx.EPS * want.abs() + 2.0 ** -148 * u.abs() + 2.0 ** -150).all()


def test_host_arrays(dev):
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((5, 100)).astype(F), rng.standard_normal((17, 100)).astype(F)
    q = lambda v: sa.quantize_mx4(v, np.empty((v.shape[0], 50), U), np.empty((v.shape[0], 4), U))
    X, W = q(x), q(w)
    for got, want in zip((*X, *W), (*mx.quantize(x), *mx.quantize(w))):
        assert np.array_equal(got, want)
    assert np.array_equal(sa.dequantize_mx4(*X, np.empty((5, 100), F)), mx.values(*X))
    _check(sa.matmul_mx4(*X, *W, np.empty((5, 17), F)), *mx.product(*X, *W))
    g, tg = mx.product(*X, *W)
    _check(sa.swiglu_mx4(*X, *W, *W, np.empty((5, 17), F)), *mx.gated(g, tg, g, tg))


@pytest.mark.parametrize("m, k", [(1, 64), (2, 32), (4, 64), (7, 100), (33, 3199), (700, 1533)])
@pytest.mark.parametrize("torch_tensors", [False, True])
def test_codes_and_scales_in_one_host_array(dev, m, k, torch_tensors):
    """Rows of codes and of scales between each other in plain host memory, either first, next to
    each other and apart: every row is there, and the bytes between them stay."""
    import torch
    rng = np.random.default_rng(m)
    x = _x(rng, m, k)
    codes, scales = mx.quantize(x)
    nc, ns = codes.shape[1], scales.shape[1]
    for at_c, at_s, width in ((0, nc, nc + ns), (ns, 0, nc + ns), (1, nc + 3, nc + ns + 8), (ns + 5, 2, nc + ns + 6)):
        before = rng.integers(0, 256, (m, width)).astype(U)
        buf = before.copy()
        c, s = buf[:, at_c:at_c + nc], buf[:, at_s:at_s + ns]
        want = before.copy()
        want[:, at_c:at_c + nc], want[:, at_s:at_s + ns] = codes, scales
        if torch_tensors:
            b = torch.from_numpy(buf)
            sa.quantize_mx4(torch.from_numpy(x), b[:, at_c:at_c + nc], b[:, at_s:at_s + ns])
        else:
            sa.quantize_mx4(x, c, s)
        assert np.array_equal(buf, want), (at_c, at_s, np.argwhere(buf != want)[:3])
        # and read from there, into rows of which the ends belong to someone else
        out = np.full((m, k + 3), 7, F)
        sa.dequantize_mx4(c, s, out[:, :k])
        assert np.array_equal(out[:, :k], mx.values(codes, scales)[:, :k]) and (out[:, k:] == 7).all()


@pytest.mark.parametrize("op", ["quantize", "dequantize", "product", "gate"])
def test_two_threads_into_parts_of_one_host_array(dev, op):
    """Each call writes its own columns of the rows that both share, in plain host memory, and
    nothing of the other's."""
    import torch
    m, k, n = 300, 1024, 400
    rng = np.random.default_rng(3)
    x = [_x(rng, m, k) for _ in range(2)]
    rows = [mx.codes(rng, r, k // 2) for r in (m, n, n)]
    gate = op == "gate"
    if op == "quantize":
        buf = np.zeros((m, 2, k // 2), U)
        want = [mx.quantize(v)[0] for v in x]
        calls = [lambda i=i: sa.quantize_mx4(x[i], buf[:, i], np.empty((m, k // 32), U)) for i in range(2)]
    elif op == "dequantize":
        q = [mx.quantize(v) for v in x]
        buf = np.zeros((m, 2, k), F)
        want = [mx.values(*v) for v in q]
        calls = [lambda i=i: sa.dequantize_mx4(*q[i], buf[:, i]) for i in range(2)]
    else:
        buf = np.zeros((m, 2, n), F)
        a, *bs = rows[:2 + gate]
        f = sa.swiglu_mx4 if gate else sa.matmul_mx4
        flat = [*a, *[v for b in bs for v in b]]
        want = [f(*flat, np.empty((m, n), F))] * 2  # (other tests say that it is right)
        calls = [lambda i=i: f(*flat, buf[:, i]) for i in range(2)]
    bad, meet = [], threading.Barrier(2)

    def work(i):
        torch.cuda.set_device(0)
        st = torch.cuda.Stream()
        sa.set_stream(st)
        try:
            for _ in range(30):
                buf[:, i] = 0
                meet.wait(60)
                calls[i]()
                if not np.array_equal(buf[:, i], want[i]):
                    bad.append(i)
                meet.wait(60)
                if not np.array_equal(buf[:, i], want[i]):
                    bad.append(i)
        except Exception as e:  # a thread's error is the test's
            bad.append(e)
            meet.abort()
        finally:
            sa.set_stream(None)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad, bad[:4]


def test_rows_far_apart(dev):
    """Rows whose offsets pass 32 bits, in every operand."""
    import torch
    rng = np.random.default_rng(8)
    far = (1 << 31) + 64
    big = torch.empty(3 * far, dtype=torch.uint8, device=dev)

    def spread(v, at):
        t = torch.as_strided(big, v.shape, (far, 1), at)
        t.copy_(torch.from_numpy(v))
        return t

    for m, n, kb in ((3, 3, 100), (3, 3, 256)):
        a, s = mx.codes(rng, m, kb)
        b, t = mx.codes(rng, n, kb)
        d = [spread(a, 0), spread(s, 1024), spread(b, 2048), spread(t, 4096)]
        out = torch.as_strided(big.view(torch.float32), (m, n), (far // 4, 1), 2048)
        want, _ = mx.product(a, s, b, t)
        sa.matmul_mx4(*d, out)
        assert np.array_equal(out.cpu().numpy(), want)
        x = torch.as_strided(big.view(torch.float32), (m, 2 * kb), (far // 4, 1), 8192)
        sa.dequantize_mx4(*d[:2], x)
        assert np.array_equal(x.cpu().numpy(), mx.values(a, s))
        x.copy_(torch.from_numpy(_x(rng, m, 2 * kb)))
        codes, scales = mx.quantize(x.cpu().numpy())
        sa.quantize_mx4(x, *d[:2])
        assert np.array_equal(d[0].cpu().numpy(), codes) and np.array_equal(d[1].cpu().numpy(), scales)


SHAPES = [(1, 400, 300), (16, 1080, 160), (40, 767, 65), (129, 2304, 1500), (700, 767, 2051), (130, 640, 9000),
          (2900, 1040, 3008), (2900, 1001, 3000)]


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("m, kb, n", SHAPES)
def test_captured_and_replayed(dev, gate, m, kb, n):
    """Replays on new inputs, with eager work between them, against eager results; another
    graph of the stream replayed in turn."""
    import torch
    rng = np.random.default_rng(m)
    f = sa.swiglu_mx4 if gate else sa.matmul_mx4
    sizes = (m, n, n) if gate else (m, n)
    new = lambda: [torch.from_numpy(v).to(dev) for r in sizes for v in mx.codes(rng, r, kb, 120, 125)]
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        sa.set_stream(st)
        try:
            t, t2 = new(), new()
            out, out2 = (torch.zeros((m, n), device=dev) for _ in range(2))
            f(*t, out)  # the warm-up call of this size
            st.synchronize()
            graphs = []
            for args in ((t, out), (t2, out2)):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=st):
                    f(*args[0], args[1])
                graphs.append(g)
            for _ in range(3):
                for a, b in zip(t + t2, new() + new()):
                    a.copy_(b)
                want = [f(*t, torch.empty_like(out)), f(*t2, torch.empty_like(out))]
                st.synchronize()
                for o in (out, out2):
                    o.fill_(9)
                for g in graphs:
                    g.replay()
                st.synchronize()
                assert torch.equal(out, want[0]) and torch.equal(out2, want[1])
        finally:
            sa.set_stream(torch.cuda.default_stream())


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("m, kb, n", [(9000, 1001, 9000), (9000, 2064, 9000)])
def test_captured_without_a_call_before(dev, gate, m, kb, n):
    """More scratch than any other test leaves: the captured call goes on without it."""
    import torch
    rng = np.random.default_rng(kb)
    f = sa.swiglu_mx4 if gate else sa.matmul_mx4
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        sa.set_stream(st)
        try:
            t = [torch.from_numpy(v).to(dev) for r in ((m, n, n) if gate else (m, n))
                 for v in mx.codes(rng, r, kb, 120, 122)]
            out, want = (torch.zeros((m, n), device=dev) for _ in range(2))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                f(*t, out)
            f(*t, want)
            for _ in range(3):
                out.fill_(9)
                g.replay()
                st.synchronize()
                # sums are multiples of 2^-16 (products of 2^-2 at least, times 2^-14) and
                # below 2^6 (36 * 2^-12 for each of 4128): exact in either order
                assert torch.equal(out, want)
        finally:
            sa.set_stream(torch.cuda.default_stream())


def test_two_threads_on_their_own_streams(dev):
    import torch
    rng = np.random.default_rng(9)
    jobs = []
    for m, kb, n in ((3, 767, 333), (260, 767, 333)):
        (a, s), (b, t) = mx.codes(rng, m, kb), mx.codes(rng, n, kb)
        jobs.append(([torch.from_numpy(v).to(dev) for v in (a, s, b, t)], mx.product(a, s, b, t)[0]))
    torch.cuda.synchronize()
    bad = []

    def work(job):
        torch.cuda.set_device(0)
        st = torch.cuda.Stream()
        sa.set_stream(st)
        try:
            with torch.cuda.stream(st):
                for _ in range(20):
                    out = torch.zeros(job[1].shape, device=dev)
                    sa.matmul_mx4(*job[0], out)
                    st.synchronize()
                    if not np.array_equal(out.cpu().numpy(), job[1]):
                        bad.append(job[1].shape)
        except Exception as e:  # a thread's error is the test's
            bad.append(e)
        finally:
            sa.set_stream(None)

    ts = [threading.Thread(target=work, args=(j,)) for j in jobs for _ in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad, bad


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("m, kb, n", SHAPES + [(2, 4320, 3200), (600, 272, 4100)])
def test_the_same_call_gives_the_same_bits(dev, gate, m, kb, n):
    import torch
    rng = np.random.default_rng(m)
    t = [torch.from_numpy(v).to(dev) for r in ((m, n, n) if gate else (m, n)) for v in mx.codes(rng, r, kb, 90, 150)]
    f = sa.swiglu_mx4 if gate else sa.matmul_mx4
    first = f(*t, torch.empty((m, n), device=dev))
    for _ in range(5):
        assert torch.equal(f(*t, torch.empty((m, n), device=dev)).nan_to_num(), first.nan_to_num())
