"""The 8-bit cache against numpy: codes and scales bit for bit, attention within the
rounding of fp32, eviction's choices exactly."""
import numpy as np
import pytest

import simplang_amd as sa
import _serve as S

pytestmark = pytest.mark.gpu


class Pair:
    """A cache on the GPU and the same in numpy, filled with garbage."""

    def __init__(self, dev, b, h, cap, hs, block, seed=0, layout="head"):
        import torch
        r = np.random.default_rng(seed)
        nb = -(-cap // block)
        kc, vc = (r.integers(-127, 128, (b, h, cap, hs)).astype(np.int8) for _ in range(2))
        ks, vs = ((r.random((b, h, nb)) * 0.05).astype(np.float32) for _ in range(2))
        self.np = S.Cache(kc, vc, ks, vs, block)

        def codes(x):
            t = torch.from_numpy(x).to(dev)
            if layout == "token":      # [batch, capacity, heads, head_size]
                return t.transpose(1, 2).contiguous().transpose(1, 2)
            if layout == "padded":     # rows of hs + 4 bytes, capacity + 3 rows
                w = torch.full((b, h, cap + 3, hs + 4), 99, dtype=torch.int8, device=dev)
                w[:, :, :cap, :hs] = t
                return w[:, :, :cap, :hs]
            return t
        self.t = [codes(kc), codes(vc)] + [torch.from_numpy(x).to(dev) for x in (ks, vs)]
        self.gpu = sa.KV8Cache(*self.t, block)
        self.dev = dev

    def same(self):
        for t, x in zip(self.t, (self.np.kc, self.np.vc, self.np.ks, self.np.vs)):
            got = t.cpu().numpy()
            assert np.array_equal(got, x, equal_nan=x.dtype.kind == "f"), np.argwhere(got != x)[:5]

    def up(self, *arrays):
        import torch
        return [torch.from_numpy(np.ascontiguousarray(a)).to(self.dev) for a in arrays]

    def append(self, k, v, lens, lengths, first=0):
        st, ln = S.starts(lens, first), np.asarray(lengths, np.int32)
        self.np.append(k, v, st, ln)
        self.gpu.append(*self.up(k, v, st, ln))


def _rows(n, h, hs, seed=0, amp=1.0):
    r = np.random.default_rng(seed + 100)
    return tuple((r.standard_normal((n, h, hs)) * amp).astype(np.float32) for _ in range(2))


@pytest.mark.parametrize("layout", ["head", "token", "padded"])
@pytest.mark.parametrize("h, hs, block", [(2, 64, 32), (3, 100, 16), (1, 128, 64), (2, 256, 128), (2, 20, 32)])
def test_append(dev, h, hs, block, layout):
    """Prompts, tokens one by one, pieces that start and end inside a block."""
    p = Pair(dev, 4, h, 300, hs, block, layout=layout)
    at = np.zeros(4, int)
    for i, new in enumerate([[1, 33, 0, 130], [1, 1, 1, 1], [40, 5, 150, 1], [1, 1, 0, 17], [200, 2, 70, 96]]):
        at = at + new
        p.append(*_rows(sum(new), h, hs, seed=i, amp=1 + i), new, at)
        p.same()


def test_append_raises_the_scale_of_a_block(dev):
    p = Pair(dev, 1, 2, 64, 64, 32)
    for i, amp in enumerate([0.1, 1, 0.5, 40, 3, 1e-3, 41]):
        p.append(*_rows(3, 2, 64, seed=i, amp=amp), [3], [3 * (i + 1)])
        p.same()


def test_append_zeros_ties_and_extremes(dev):
    p = Pair(dev, 1, 1, 128, 32, 16)
    k, v = np.zeros((64, 1, 32), np.float32), np.zeros((64, 1, 32), np.float32)
    k[16, 0, :] = np.arange(32) - 15.5          # the largest is 15.5
    k[17, 0, :] = 127                           # scale 1: the halves above are ties
    v[32:48] = 1e-45                            # the smallest number there is
    v[48:64] = 3.4e38
    v[0, 0, :] = (np.arange(32) - 16) * 2.0 ** -140
    p.append(k, v, [64], [64])
    p.same()
    p.append(*_rows(30, 1, 32), [30], [94])
    p.same()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_of_what_is_not_finite(dev, bad):
    """The block that gets it reads NaN, also after later tokens; its neighbours stay."""
    p = Pair(dev, 1, 2, 64, 32, 16)
    k, v = _rows(40, 2, 32)
    k[20, 1, 3] = bad
    p.append(k, v, [40], [40])
    got = p.gpu.read(*p.up(S.starts([40]), np.array([40], np.int32)),
                     *p.up(np.zeros_like(k), np.zeros_like(v)))[0].cpu().numpy()
    assert np.isnan(got[16:32, 1]).all() and np.isfinite(got[:, 0]).all()
    assert np.isfinite(got[:16, 1]).all() and np.isfinite(got[32:, 1]).all()
    assert (p.t[0][0, 1, 16:32] == 0).all()
    p.append(*_rows(3, 2, 32, seed=3), [3], [43])
    k, v = _rows(9, 2, 32, seed=4)
    p.append(k, v, [9], [28])                   # from 19 on, inside that block
    assert not np.isfinite(p.t[2][0, 1, 1].item()) and (p.t[0][0, 1, 16:28] == 0).all()


def test_append_outside_the_capacity(dev):
    p = Pair(dev, 3, 2, 50, 64, 16)
    p.append(*_rows(75, 2, 64), [30, 25, 20], [60, 10, -3])
    p.same()
    p.append(*_rows(9, 2, 64), [9, 0, 0], [2**31 - 1, 5, 5])
    p.same()


def test_append_rows_of_no_sequence(dev):
    p = Pair(dev, 2, 1, 64, 64, 16)
    p.append(*_rows(30, 1, 64), [10, 5], [12, 5], first=4)
    p.same()


def test_append_strided_rows(dev):
    import torch
    p = Pair(dev, 2, 2, 64, 64, 16)
    x = torch.randn((20, 9 * 64), device=dev)
    k, v = x[:, 320:448].unflatten(1, (2, 64)), x[:, 448:576].unflatten(1, (2, 64))
    st, ln = S.starts([13, 7]), np.array([13, 37], np.int32)
    p.np.append(k.cpu().numpy(), v.cpu().numpy(), st, ln)
    p.gpu.append(k, v, *p.up(st, ln))
    p.same()
    for off in (1, 2, 3):
        y = torch.randn(2 * 128 + 8, device=dev)
        k = y[off:off + 128].view(1, 2, 64)
        v = y[off + 128:off + 256].view(1, 2, 64)
        st, ln = S.starts([0, 1]), np.array([13, 37 + off], np.int32)
        p.np.append(k.cpu().numpy(), v.cpu().numpy(), st, ln)
        p.gpu.append(k, v, *p.up(st, ln))
        p.same()


@pytest.mark.parametrize("layout", ["head", "token", "padded"])
@pytest.mark.parametrize("h, hs, block", [(2, 64, 32), (3, 100, 16), (1, 256, 64), (2, 28, 128)])
def test_read(dev, h, hs, block, layout):
    import torch
    p = Pair(dev, 4, h, 200, hs, block, layout=layout)
    for lens, ln, first in ([3, 0, 150, 47], [3, 9, 160, 200], 0), ([1, 1, 1, 1], [1, 200, 64, 65], 2), \
            ([9, 5, 4, 3], [4, 203, 2**31 - 1, -1], 1):
        n = sum(lens) + first + 3
        st, ln = S.starts(lens, first), np.array(ln, np.int32)
        want = np.full((2, n, h, hs), 7, np.float32)
        p.np.read(st, ln, want[0], want[1])
        buf = torch.full((n, 2, h, hs), 7.0, device=dev)       # K and V rows side by side
        p.gpu.read(*p.up(st, ln), buf[:, 0], buf[:, 1])
        got = buf.cpu().numpy()
        assert np.array_equal(got[:, 0], want[0]) and np.array_equal(got[:, 1], want[1])


def _attend(p, q, lengths, scale=None, seen=None, in_place=False, fill=None):
    import torch
    lengths = np.asarray(lengths, np.int32)
    sc = p.np.kc.shape[3] ** -0.5 if scale is None else scale
    want, wseen, tol, stol = p.np.attention(q, lengths, sc, seen)
    out = torch.full(q.shape, 7.0, device=p.dev)
    qt, lt = p.up(q, lengths)
    if seen is None:
        p.gpu.attention(qt, lt, out, scale=scale)
    else:
        st, = p.up(seen)
        so = st if in_place else torch.full(seen.shape, 5.0, device=p.dev)
        p.gpu.attention(qt, lt, out, st, so, scale=scale)
        gs = so.cpu().numpy()
        for b, n in enumerate(lengths):
            n = min(max(n, 0), seen.shape[2])
            assert np.array_equal(gs[b, :, n:], seen[b, :, n:] if in_place else np.full_like(gs[b, :, n:], 5))
            bad = np.abs(gs[b, :, :n] - wseen[b, :, :n]) > stol[b, :, :n]
            assert not bad.any(), (b, np.argwhere(bad)[:4])
    got = out.cpu().numpy()
    bad = (np.abs(got - want) > tol[..., None]) | (np.isnan(got) != np.isnan(want))
    assert not bad.any(), (np.argwhere(bad)[:4], np.nanmax(np.abs(got - want) / np.maximum(tol[..., None], 1e-30)))
    return got


@pytest.mark.parametrize("layout", ["head", "token", "padded"])
@pytest.mark.parametrize("heads, h, hs, block", [(4, 2, 64, 32), (3, 3, 100, 16), (8, 1, 128, 64), (5, 1, 256, 128),
                                                 (12, 2, 80, 32), (2, 2, 16, 16), (4, 4, 20, 64)])
def test_attention(dev, heads, h, hs, block, layout):
    p = Pair(dev, 5, h, 600, hs, block, layout=layout)
    r = np.random.default_rng(9)
    q = r.standard_normal((5, heads, hs)).astype(np.float32)
    seen = r.random((5, h, 600)).astype(np.float32)
    _attend(p, q, [1, 600, 0, 65, 257], seen=seen)
    _attend(p, q, [64, 16, 15, 17, 700], seen=seen, in_place=True)
    _attend(p, q, [-5, 63, 128, 129, 599])


@pytest.mark.parametrize("heads, h", [(16, 1), (20, 1), (33, 1), (40, 2), (6, 3), (64, 4)])
def test_attention_groups(dev, heads, h):
    p = Pair(dev, 3, h, 200, 64, 32)
    r = np.random.default_rng(heads)
    _attend(p, r.standard_normal((3, heads, 64)).astype(np.float32), [200, 33, 150],
            seen=r.random((3, h, 200)).astype(np.float32))


@pytest.mark.parametrize("n, b, heads, h, hs, block", [(20000, 1, 8, 2, 128, 64), (5001, 2, 2, 2, 100, 16), (9000, 3, 4, 1, 64, 128)])
def test_attention_long(dev, n, b, heads, h, hs, block):
    """One row per head over many blocks: the work is split over the tokens."""
    p = Pair(dev, b, h, n + 7, hs, block)
    r = np.random.default_rng(n)
    _attend(p, r.standard_normal((b, heads, hs)).astype(np.float32), [n, 3, 700][:b],
            seen=r.random((b, h, n + 7)).astype(np.float32))


@pytest.mark.parametrize("n, h, cap, hs", [(64, 3, 600, 32), (65, 1, 600, 16), (200, 2, 3000, 16), (1, 1, 3000, 256),
                                           (4200, 1, 300, 16)])
def test_attention_many_sequences(dev, n, h, cap, hs):
    """More sequences than a wave has lanes, some empty, in one to several pieces each."""
    r = np.random.default_rng(n)
    lengths = r.integers(0, cap + 1, n).astype(np.int32)
    lengths[r.integers(0, n, n // 3)] = 0
    lengths[-1] = cap
    p = Pair(dev, n, h, cap, hs, 64, seed=n)
    q = r.standard_normal((n, 2 * h, hs)).astype(np.float32)
    _attend(p, q, lengths, seen=np.abs(r.standard_normal((n, h, cap))).astype(np.float32))


def test_attention_one_token_matters(dev):
    """A weight near one among thousands of nothing, and equal scores everywhere."""
    p = Pair(dev, 2, 1, 3000, 64, 32)
    r = np.random.default_rng(2)
    q = r.standard_normal((2, 2, 64)).astype(np.float32) * 30
    q[1] = 0
    _attend(p, q, [3000, 2999], seen=np.zeros((2, 1, 3000), np.float32))


def test_attention_scales(dev):
    """Blocks of very different scales, of scale zero, and the largest queries."""
    import torch
    p = Pair(dev, 2, 2, 256, 64, 16)
    r = np.random.default_rng(3)
    for z, t in ((p.np.ks, p.t[2]), (p.np.vs, p.t[3])):
        z *= (10.0 ** r.uniform(-6, 1, z.shape)).astype(np.float32)
        z[:, :, 3] = 0
        t.copy_(torch.from_numpy(z))
    q = r.standard_normal((2, 4, 64)).astype(np.float32)
    _attend(p, q, [256, 200], seen=r.random((2, 2, 256)).astype(np.float32))
    _attend(p, q * np.float32(1e-30), [256, 200])
    _attend(p, np.zeros_like(q), [256, 61])
    _attend(p, q, [256, 200], scale=0.0)
    _attend(p, q, [256, 200], scale=-1.0)
    _attend(p, q * np.float32(1e30), [256, 200], scale=1e-30)


def test_attention_behind_the_length_may_hold_anything(dev):
    p = Pair(dev, 2, 2, 160, 64, 32)
    r = np.random.default_rng(4)
    q = r.standard_normal((2, 4, 64)).astype(np.float32)
    want = _attend(p, q, [70, 96])
    for z in p.t[2:]:
        z[0, :, 3:] = float("nan")
        z[1, :, 3:] = float("inf")
    for c in p.t[:2]:
        c[0, :, 70:] = 77
        c[1, :, 96:] = -77
    out = p.up(np.zeros_like(q))[0]
    p.gpu.attention(*p.up(q, np.array([70, 96], np.int32)), out)
    assert np.array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_attention_over_a_bad_block(dev, which, bad):
    """A block whose scale is not finite makes the rows that read it NaN or infinite, no others."""
    p = Pair(dev, 2, 2, 160, 64, 32)
    p.t[which][1, 0, 2] = bad
    q = np.random.default_rng(4).standard_normal((2, 4, 64)).astype(np.float32)
    out = p.up(np.zeros_like(q))[0]
    p.gpu.attention(*p.up(q, np.array([160, 160], np.int32)), out)
    got = out.cpu().numpy()
    assert np.isfinite(got[0]).all() and np.isfinite(got[1, 2:]).all()
    assert not np.isfinite(got[1, :2]).any()


def test_attention_of_queries_that_are_not_finite(dev):
    p = Pair(dev, 1, 2, 160, 64, 32)
    q = np.random.default_rng(4).standard_normal((1, 4, 64)).astype(np.float32)
    want = _attend(p, q, [100])
    q[0, 1, 7], q[0, 2, 0] = np.nan, np.inf
    out = p.up(np.zeros_like(q))[0]
    p.gpu.attention(*p.up(q, np.array([100], np.int32)), out)
    got = out.cpu().numpy()
    assert np.isnan(got[0, 1:3]).all()
    assert np.array_equal(got[0, [0, 3]], want[0, [0, 3]])


def test_attention_strided(dev):
    import torch
    p = Pair(dev, 3, 2, 100, 64, 16)
    x = torch.randn((3, 700), device=dev)
    q = x[:, 5:261].unflatten(1, (4, 64))
    out = torch.full((3, 5, 70), 7.0, device=dev)
    seen = torch.rand((3, 2, 133), device=dev)
    was = seen.clone()
    ln = np.array([100, 40, 3], np.int32)
    p.gpu.attention(q, p.up(ln)[0], out[:, :4, :64], seen[:, :, :100], seen[:, :, :100])
    want, ws, tol, stol = p.np.attention(q.cpu().numpy(), ln, 0.125, was[:, :, :100].cpu().numpy())
    assert (np.abs(out[:, :4, :64].cpu().numpy() - want) <= tol[..., None]).all()
    assert (out[:, 4] == 7).all() and (out[:, :, 64:] == 7).all()
    assert (np.abs(seen[:, :, :100].cpu().numpy() - ws) <= stol).all()
    assert torch.equal(seen[:, :, 100:], was[:, :, 100:])


def _evict(p, to, lengths, seen, budget, recent, extra=0):
    import torch
    b, h = p.np.kc.shape[:2]
    ln = np.asarray(lengths, np.int32)
    kept, ns = np.zeros((b, h, budget), np.int32), np.full((b, h, budget + extra), 3, np.float32)
    p.np.evict(to.np, ln, seen, budget, recent, ns, kept)
    kt = torch.full((b, h, budget), 99, dtype=torch.int32, device=p.dev)
    nt = torch.full((b, h, budget + extra), 3.0, device=p.dev)
    p.gpu.evict(to.gpu, *p.up(ln, seen), nt, kt, budget, recent)
    assert np.array_equal(kt.cpu().numpy(), kept), np.argwhere(kt.cpu().numpy() != kept)[:5]
    assert np.array_equal(nt.cpu().numpy(), ns, equal_nan=True)
    to.same()


@pytest.mark.parametrize("layout", ["head", "token", "padded"])
@pytest.mark.parametrize("h, hs, block", [(2, 64, 32), (3, 100, 16), (1, 256, 128), (2, 20, 64)])
def test_evict(dev, h, hs, block, layout):
    p = Pair(dev, 5, h, 500, hs, block, layout=layout)
    r = np.random.default_rng(6)
    seen = (r.random((5, h, 500)) ** 8).astype(np.float32)
    for budget, recent, ln in ((100, 20, [500, 100, 101, 0, 333]), (65, 65, [64, 65, 66, 500, 1]),
                               (256, 0, [257, 500, 300, 10, 499]), (1, 0, [5, 1, 0, 500, 2]),
                               (17, 16, [500, 18, 17, 40, 9])):
        to = Pair(dev, 5, h, 256, hs, block, seed=8, layout=layout)
        _evict(p, to, ln, seen, budget, recent, extra=3)


def test_evict_ties_zeros_and_strange_weights(dev):
    p, to = Pair(dev, 1, 1, 3000, 32, 32), Pair(dev, 1, 1, 1500, 32, 32)
    r = np.random.default_rng(7)
    seen = r.integers(0, 3, (1, 1, 3000)).astype(np.float32)
    _evict(p, to, [3000], seen, 1500, 100)
    _evict(p, to, [2999], np.zeros_like(seen), 700, 0)
    seen[0, 0, ::7] = -0.0
    seen[0, 0, 1::7] = 0.0
    seen[0, 0, 2::7] = -1
    seen[0, 0, 3::7] = np.inf
    seen[0, 0, 4::7] = -np.inf
    seen[0, 0, 5::7] = 1e-42
    _evict(p, to, [3000], seen, 1300, 3)
    seen[0, 0, 100:104] = np.nan
    seen[0, 0, 200] = -np.nan
    _evict(p, to, [3000], seen, 300, 0)
    _evict(p, to, [2500], seen, 4, 0)


@pytest.mark.parametrize("n, budget", [(20000, 5000), (40001, 39999), (1025, 1024)])
def test_evict_long(dev, n, budget):
    p, to = Pair(dev, 1, 2, n, 16, 16), Pair(dev, 1, 2, budget, 16, 16)
    seen = (np.random.default_rng(n).random((1, 2, n)) * 20).astype(np.float32)
    _evict(p, to, [n], seen, budget, budget // 10)


def test_evict_bad_and_empty_blocks(dev):
    import torch
    p, to = Pair(dev, 1, 2, 200, 32, 16), Pair(dev, 1, 2, 100, 32, 16)
    for z, t in ((p.np.ks, p.t[2]), (p.np.vs, p.t[3])):
        z[0, 0, 3:6] = 0
        z[0, 1, 4] = np.nan
        t.copy_(torch.from_numpy(z))
    _evict(p, to, [200], np.zeros((1, 2, 200), np.float32), 100, 10)


def test_device_calls_refuse_caches_of_host_memory(dev):
    c = sa.KV8Cache(np.zeros((1, 1, 16, 16), np.int8), np.zeros((1, 1, 16, 16), np.int8),
                    np.zeros((1, 1, 1), np.float32), np.zeros((1, 1, 1), np.float32), 16)
    with pytest.raises(sa.SimpRTError, match="device memory"):
        c.append(*_rows(1, 1, 16), S.starts([1]), np.array([1], np.int32))


def test_host_rows(dev):
    """Rows, lengths and results in host memory: staged by the call."""
    p = Pair(dev, 2, 2, 64, 32, 16)
    k, v = _rows(20, 2, 32)
    st, ln = S.starts([15, 5]), np.array([20, 5], np.int32)
    p.np.append(k, v, st, ln)
    p.gpu.append(k, v, st, ln)
    p.same()
    got = p.gpu.read(st, ln, np.zeros_like(k), np.zeros_like(v))
    want = np.zeros_like(k), np.zeros_like(v)
    p.np.read(st, ln, *want)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    q = np.random.default_rng(1).standard_normal((2, 2, 32)).astype(np.float32)
    seen = np.ones((2, 2, 64), np.float32)
    ref, rs, tol, stol = p.np.attention(q, ln, 32 ** -0.5, seen)
    out = p.gpu.attention(q, ln, np.zeros_like(q), seen, seen)
    assert (np.abs(out - ref) <= tol[..., None]).all() and (np.abs(seen - rs) <= stol).all()


def test_offsets_beyond_32_bits(dev):
    """The last of the sequences lies more than 2^32 bytes into the cache."""
    import torch
    cap, hs, n = 1 << 18, 256, 70
    k = torch.zeros((n, 1, cap, hs), dtype=torch.int8, device=dev)
    v = torch.zeros_like(k)
    s = [torch.zeros((n, 1, cap // 128), device=dev) for _ in range(2)]
    c = sa.KV8Cache(k, v, *s, 128)
    x, y = (torch.randn((300, 1, hs), device=dev) for _ in range(2))
    lens = [0] * (n - 1) + [300]
    st = torch.tensor(S.starts(lens), device=dev)
    ln = torch.tensor([0] * (n - 1) + [cap - 5], dtype=torch.int32, device=dev)
    c.append(x, y, st, ln)
    a, b = torch.zeros_like(x), torch.zeros_like(y)
    c.read(st, ln, a, b)
    assert (x - a).abs().max() <= x.abs().max() / 127 * 0.51 and (y - b).abs().max() <= y.abs().max() / 127 * 0.51
    q = torch.randn((n, 2, hs), device=dev) * 30
    q[-1] = x[290] * 30
    out = torch.zeros_like(q)
    c.attention(q, ln, out)
    assert (out[:-1] == 0).all() and (out[-1] - b[290]).abs().max() < 1e-4
    assert (k[:-1].amax() == 0) and (k[-1, :, :cap - 5 - 300] == 0).all()


def test_graph_and_streams(dev):
    """A decode step captured once and replayed as the lengths grow, on another stream."""
    import torch
    B, H, heads, hs, cap = 3, 2, 6, 64, 96
    p = Pair(dev, B, H, cap, hs, 16)
    ref = Pair(dev, B, H, cap, hs, 16)
    at = np.array([5, 40, 0])
    k, v = _rows(45, H, hs)
    p.append(k, v, at, at)
    ref.append(k, v, at, at)
    st = torch.cuda.Stream()
    kt, vt, starts, ln = p.up(*_rows(B, H, hs), S.starts([1] * B), at.astype(np.int32))
    q, out = torch.zeros((B, heads, hs), device=dev), torch.zeros((B, heads, hs), device=dev)
    seen = torch.zeros((B, H, cap), device=dev)
    torch.cuda.synchronize()
    try:
        sa.set_stream(st)
        with torch.cuda.stream(st):
            p.gpu.attention(q, ln, out)                 # the size's warm-up call
            p.gpu.attention(q, ln, out, seen, seen)
        st.synchronize()
        seen.zero_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            p.gpu.append(kt, vt, starts, ln)
            p.gpu.attention(q, ln, out, seen, seen)
        total = np.zeros((B, H, cap))
        for i in range(20):
            at = at + 1
            r = np.random.default_rng(50 + i)
            nk, nv, nq = (r.standard_normal((B, n, hs)).astype(np.float32) for n in (H, H, heads))
            for a, b in ((kt, nk), (vt, nv), (q, nq), (ln, at.astype(np.int32))):
                a.copy_(torch.from_numpy(b))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            ref.np.append(nk, nv, S.starts([1] * B), at)
            want, ws, tol, stol = ref.np.attention(nq, at, hs ** -0.5, np.zeros((B, H, cap), np.float32))
            total += ws
            assert (np.abs(out.cpu().numpy() - want) <= tol[..., None]).all()
        assert np.abs(seen.cpu().numpy() - total).max() < 20 * (stol.max() + 20 * S.EPS)
        p.np = ref.np
        p.same()
    finally:
        sa.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("n", [3, 70])
def test_replays_with_other_lengths(dev, n):
    """One graph for short, long, empty and full sequences: the pieces follow the lengths."""
    import torch
    cap = 2900
    p = Pair(dev, n, 1, cap, 32, 64, seed=n)
    r = np.random.default_rng(n)
    q = r.standard_normal((n, 3, 32)).astype(np.float32)
    qt, ln = p.up(q, np.zeros(n, np.int32))
    out, seen = torch.zeros_like(qt), torch.zeros((n, 1, cap), device=dev)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        sa.set_stream(st)
        p.gpu.attention(qt, ln, out, seen, seen)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            p.gpu.attention(qt, ln, out, seen, seen)
        full, one = np.full(n, cap), np.ones(n)
        for lengths in (full, one, np.zeros(n), r.integers(0, cap + 1, n), np.where(r.random(n) < 0.8, 0, cap)):
            lengths = lengths.astype(np.int32)
            ln.copy_(torch.from_numpy(lengths))
            seen.zero_()
            out.fill_(3)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            want, ws, tol, stol = p.np.attention(q, lengths, 32 ** -0.5, np.zeros((n, 1, cap), np.float32))
            assert (np.abs(out.cpu().numpy() - want) <= tol[..., None]).all()
            assert (np.abs(seen.cpu().numpy() - ws) <= stol).all()
    finally:
        sa.set_stream(torch.cuda.current_stream())


def test_capture_without_a_warm_up_call_is_refused(dev):
    """The attention wants scratch, which a captured call does not allocate; the rest wants none."""
    import torch
    p = Pair(dev, 2, 1, 5000, 32, 16)
    q, out = torch.zeros((2, 2, 32), device=dev), torch.zeros((2, 2, 32), device=dev)
    k, v, st, ln = p.up(*_rows(2, 1, 32), S.starts([1, 1]), np.array([100, 7], np.int32))
    p.np.append(k.cpu().numpy(), v.cpu().numpy(), st.cpu().numpy(), [100, 7])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        sa.set_stream(stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            with pytest.raises(sa.SimpRTError, match="workspace"):
                p.gpu.attention(q, ln, out)
            p.gpu.append(k, v, st, ln)
        g.replay()
        torch.cuda.synchronize()
        p.same()
    finally:
        sa.set_stream(torch.cuda.current_stream())


def test_two_threads(dev):
    """Two threads at once on one stream: each finds its own results."""
    import threading
    import torch
    ps = [Pair(dev, 2, 2, 3000, 64, 32, seed=i) for i in range(2)]
    r = np.random.default_rng(1)
    qs = [r.standard_normal((2, 4, 64)).astype(np.float32) for _ in ps]
    ln = np.array([3000, 1700], np.int32)
    want = [p.np.attention(q, ln, 0.125) for p, q in zip(ps, qs)]
    fails = []

    def work(i):
        torch.cuda.set_device(0)
        sa.set_stream(torch.cuda.current_stream())
        q, lt = ps[i].up(qs[i], ln)
        for _ in range(30):
            out = torch.zeros_like(q)
            ps[i].gpu.attention(q, lt, out)
            torch.cuda.synchronize()
            if (np.abs(out.cpu().numpy() - want[i][0]) > want[i][2][..., None]).any():
                fails.append(i)
                return

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not fails


def test_read_into_parts_of_one_tensor(dev):
    """K and V between each other's rows, or heads."""
    import torch
    p = Pair(dev, 2, 3, 40, 32, 16)
    st, ln = S.starts([9, 20]), np.array([30, 33], np.int32)
    p.append(*_rows(29, 3, 32), [9, 20], ln)
    k, v = np.zeros((29, 3, 32), np.float32), np.zeros((29, 3, 32), np.float32)
    p.np.read(st, ln, k, v)
    for axis in (1, 2):
        x = torch.zeros((29, 2, 3, 32) if axis == 1 else (29, 3, 2, 32), device=dev)
        kt, vt = x.unbind(axis)
        p.gpu.read(*p.up(st, ln), kt, vt)
        assert np.array_equal(kt.cpu().numpy(), k) and np.array_equal(vt.cpu().numpy(), v)


def test_read_into_parts_of_one_host_array(dev):
    """The same in host memory: neither part's way back goes over the other."""
    import torch
    p = Pair(dev, 2, 3, 40, 32, 16)
    st, ln = S.starts([9, 20]), np.array([30, 33], np.int32)
    p.append(*_rows(29, 3, 32), [9, 20], ln)
    k, v = np.zeros((29, 3, 32), np.float32), np.zeros((29, 3, 32), np.float32)
    p.np.read(st, ln, k, v)
    for shape, axis in (((29, 2, 3, 32), 1), ((29, 3, 2, 32), 2)):
        x = np.full(shape[:-1] + (35,), 8, np.float32)  # three elements behind each head stay
        kt, vt = (np.moveaxis(x, axis, 0)[i][..., :32] for i in (0, 1))
        p.gpu.read(st, ln, kt, vt)
        assert np.array_equal(kt, k) and np.array_equal(vt, v) and (x[..., 32:] == 8).all()
        y = torch.full(shape, 8.0)
        p.gpu.read(torch.from_numpy(st), torch.from_numpy(ln), *y.unbind(axis)[::-1])
        assert np.array_equal(y.select(axis, 1).numpy(), k) and np.array_equal(y.select(axis, 0).numpy(), v)


def test_read_over_many_empty_sequences(dev):
    import torch
    n = 3000
    p = Pair(dev, n, 1, 16, 16, 16)
    lens = np.zeros(n, int)
    lens[[0, 1, 1500, n - 1]] = [3, 16, 5, 9]
    st, ln = S.starts(lens), np.full(n, 16, np.int32)
    k = np.zeros((33, 1, 16), np.float32)
    v = np.zeros_like(k)
    p.np.read(st, ln, k, v)
    kt, vt = torch.zeros((33, 1, 16), device=dev), torch.zeros((33, 1, 16), device=dev)
    p.gpu.read(*p.up(st, ln), kt, vt)
    assert np.array_equal(kt.cpu().numpy(), k) and np.array_equal(vt.cpu().numpy(), v)
    p.append(*_rows(33, 1, 16), lens, ln)
    p.same()


def test_a_serving_loop(dev):
    """Prompts in two chunks, decode steps, an eviction, more steps: the operators together,
    against the same loop in numpy."""
    import torch
    r = np.random.default_rng(11)
    heads, H, hs, block, cap, budget = 4, 2, 64, 16, 160, 64
    p, to = Pair(dev, 2, H, cap, hs, block), Pair(dev, 2, H, cap, hs, block, seed=5)
    f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    seen = np.zeros((2, H, cap), np.float32)
    seen_t = torch.zeros((2, H, cap), device=dev)
    at = np.zeros(2, int)
    for new in ([70, 33], [20, 50]):                # the second goes on after what is cached
        at = at + new
        k, v, q = f(sum(new), H, hs), f(sum(new), H, hs), f(sum(new), heads, hs)
        p.append(k, v, new, at)
        p.same()
        ks = S.starts(at)
        kk, vv = np.zeros((at.sum(), H, hs), np.float32), np.zeros((at.sum(), H, hs), np.float32)
        p.np.read(ks, at, kk, vv)
        kt, vt = p.gpu.read(*p.up(ks, at.astype(np.int32)), *p.up(np.zeros_like(kk), np.zeros_like(vv)))
        assert np.array_equal(kt.cpu().numpy(), kk) and np.array_equal(vt.cpu().numpy(), vv)
        out = torch.zeros(q.shape, device=dev)
        sa.attention_packed(p.up(q)[0], kt, vt, out, *p.up(S.starts(new), ks))
        want, tol = S.packed(q, kk, vv, S.starts(new), ks, hs ** -0.5, heads // H)
        assert (np.abs(out.cpu().numpy() - want) <= tol[..., None]).all()

    def step(c, seen, seen_t, at):
        k, v, q = f(2, H, hs), f(2, H, hs), f(2, heads, hs)
        c.append(k, v, [1, 1], at)
        want, ws, tol, stol = c.np.attention(q, at, hs ** -0.5, seen)
        out = torch.zeros(q.shape, device=dev)
        c.gpu.attention(*c.up(q, at.astype(np.int32)), out, seen_t, seen_t)
        assert (np.abs(out.cpu().numpy() - want) <= tol[..., None]).all()
        got = seen_t.cpu().numpy()
        assert (np.abs(got - ws) <= stol + 20 * S.EPS * np.abs(ws)).all()
        return got                                   # numpy goes on from the same weights

    for _ in range(12):
        at = at + 1
        seen = step(p, seen, seen_t, at)
    kept, ns = np.zeros((2, H, budget), np.int32), np.zeros((2, H, cap), np.float32)
    p.np.evict(to.np, at, seen, budget, 16, ns, kept)
    kt, nt = p.up(np.zeros_like(kept), np.zeros_like(ns))
    p.gpu.evict(to.gpu, *p.up(at.astype(np.int32)), seen_t, nt, kt, budget, 16)
    assert np.array_equal(kt.cpu().numpy(), kept) and np.array_equal(nt.cpu().numpy(), ns)
    to.same()
    at = np.minimum(at, budget)
    for _ in range(12):
        at = at + 1
        ns = step(to, ns, nt, at)
    to.same()
