"""attention_packed against 64-bit arithmetic: lengths, head layouts, strides, empty rows,
and what hidden keys may hold."""
import numpy as np
import pytest

import simplang_amd as sa
import _serve as S

pytestmark = pytest.mark.gpu


def _case(lens_q, lens_k, heads, kv, hs, seed=0, amp=1.0):
    r = np.random.default_rng(seed)
    f = lambda *s: (r.standard_normal(s) * amp).astype(np.float32)  # noqa: E731
    return (f(sum(lens_q), heads, hs), f(sum(lens_k), kv, hs), f(sum(lens_k), kv, hs),
            S.starts(lens_q), S.starts(lens_k))


def _run(dev, q, k, v, qs, ks, scale=None, out=None):
    import torch
    t = [torch.from_numpy(x).to(dev) for x in (q, k, v, qs, ks)]
    o = torch.full(q.shape, 7.0, device=dev) if out is None else out
    sa.attention_packed(*t[:3], o, t[3], t[4], scale)
    return o.cpu().numpy()


def _check(got, q, k, v, qs, ks, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    want, tol = S.packed(q, k, v, qs, ks, scale, q.shape[1] // k.shape[1])
    rows = np.zeros(q.shape[0], bool)
    rows[qs[0]:qs[-1]] = True
    assert (got[~rows] == 7.0).all()
    bad = np.abs(got - want) > tol[..., None]
    bad |= np.isnan(got) != np.isnan(want)
    assert not bad[rows].any(), (np.argwhere(bad & rows[:, None, None])[:4],
                                 np.nanmax(np.abs(got - want) / np.maximum(tol[..., None], 1e-30)))


LENS = [([1], [1]), ([16], [16]), ([17, 0, 1, 64], [17, 3, 1, 64]), ([65, 130], [65, 130]),
        ([5, 33], [200, 33]), ([1, 1, 1], [1, 77, 64]), ([3, 128], [515, 129])]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("heads, kv, hs", [(2, 2, 64), (4, 1, 32), (6, 2, 100), (3, 3, 128)])
def test_lengths_and_heads(dev, lens, heads, kv, hs):
    a = _case(*lens, heads, kv, hs)
    _check(_run(dev, *a), *a)


@pytest.mark.parametrize("hs", [1, 2, 3, 7, 16, 31, 33, 48, 65, 80, 96, 112, 127, 129, 160, 192, 250, 256])
def test_head_sizes(dev, hs):
    a = _case([70, 9], [70, 40], 4, 2, hs, seed=hs)
    _check(_run(dev, *a), *a)


@pytest.mark.parametrize("heads, kv", [(5, 1), (7, 7), (8, 1), (12, 4), (16, 1), (24, 2)])
def test_groups(dev, heads, kv):
    a = _case([100, 45, 3], [100, 60, 3], heads, kv, 64, seed=heads)
    _check(_run(dev, *a), *a)


@pytest.mark.parametrize("heads, kv, hs, nq, nk", [(8, 2, 128, 700, 700), (4, 4, 64, 1030, 1030), (2, 1, 256, 300, 450),
                                                   (8, 8, 100, 40, 2100), (16, 4, 64, 1, 3000)])
def test_long(dev, heads, kv, hs, nq, nk):
    a = _case([nq, 2], [nk, 2], heads, kv, hs, seed=nq)
    _check(_run(dev, *a), *a)


@pytest.mark.parametrize("heads, kv, hs, nq, nk", [(8, 1, 128, 500, 520), (8, 2, 64, 800, 800), (8, 1, 32, 450, 450),
                                                   (6, 1, 96, 600, 640), (4, 1, 192, 800, 811), (5, 1, 256, 650, 700),
                                                   (4, 1, 100, 801, 900), (4, 1, 63, 800, 830)])
def test_many_queries(dev, heads, kv, hs, nq, nk):
    """Enough queries to a key that K and V are taken apart once, ahead of the products."""
    a = _case([nq], [nk], heads, kv, hs, seed=nq)
    _check(_run(dev, *a), *a)


@pytest.mark.parametrize("heads, kv, hs, nq, nk", [(4, 1, 64, 2, 6000), (66, 2, 16, 1, 20000), (2, 1, 128, 33, 4000),
                                                   (3, 3, 7, 5, 3000), (1, 1, 256, 9, 2000), (300, 1, 2, 1, 2500)])
def test_few_queries_over_many_keys(dev, heads, kv, hs, nq, nk):
    """The keys are split over blocks, and the pieces joined."""
    a = _case([nq, 1, 0, 1], [nk, 1, 2, 0], heads, kv, hs, seed=nk)
    _check(_run(dev, *a), *a)


def test_fewer_keys_than_queries_leaves_rows_empty(dev):
    a = _case([40, 20, 5], [10, 0, 5], 4, 2, 64)
    got = _run(dev, *a)
    assert (got[:30] == 0).all() and (got[40:60] == 0).all()
    _check(got, *a)


def test_no_keys_at_all(dev):
    a = _case([33], [0], 4, 2, 64)
    assert (_run(dev, *a) == 0).all()


def test_rows_of_no_sequence_stay(dev):
    q, k, v, _, _ = _case([50], [60], 4, 2, 64)
    _check(_run(dev, q, k, v, S.starts([20, 5], 3), S.starts([20, 9], 2)), q, k, v,
           S.starts([20, 5], 3), S.starts([20, 9], 2))


def test_starts_outside_the_rows_are_cut_off(dev):
    q, k, v, _, _ = _case([50], [50], 2, 2, 64)
    got = _run(dev, q, k, v, np.array([-40, 20, 900], np.int32), np.array([-3, 20, 2**31 - 1], np.int32))
    _check(got, q, k, v, np.array([0, 20, 50]), np.array([0, 20, 50]))


def test_many_sequences(dev):
    r = np.random.default_rng(5)
    n = [int(x) for x in r.integers(0, 9, 300)]
    a = _case(n, n, 2, 1, 32)
    _check(_run(dev, *a), *a)


def test_strided_rows_of_a_fused_product(dev):
    import torch
    T, heads, kv, hs = 150, 6, 2, 64
    x = torch.randn((T, (heads + 2 * kv) * hs + 12), device=dev)
    parts = [x[:, a * hs:b * hs].view(T, -1, hs) if False else x[:, a * hs:b * hs].unflatten(1, (-1, hs))
             for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv))]
    o = torch.zeros((T, heads + 1, hs + 4), device=dev)
    qs = torch.tensor(S.starts([100, 50]), device=dev)
    sa.attention_packed(*parts, o[:, :heads, :hs], qs, qs)
    got = o.cpu().numpy()
    assert (got[:, heads] == 0).all() and (got[..., hs:] == 0).all()
    _check(got[:, :heads, :hs], *(p.cpu().numpy() for p in parts), qs.cpu().numpy(), qs.cpu().numpy())


@pytest.mark.parametrize("off", [1, 2, 3])
def test_unaligned(dev, off):
    import torch
    a = _case([75, 12], [75, 30], 4, 2, 64)
    t = []
    for x in a[:3]:
        buf = torch.zeros(x.size + 8, device=dev)
        buf[off:off + x.size] = torch.from_numpy(x).to(dev).reshape(-1)
        t.append(buf[off:off + x.size].view(x.shape))
    buf = torch.full((a[0].size + 8,), 7.0, device=dev)
    o = buf[off:off + a[0].size].view(a[0].shape)
    st = [torch.from_numpy(x).to(dev) for x in a[3:]]
    sa.attention_packed(*t, o, *st)
    _check(o.cpu().numpy(), *a)
    assert (buf[:off] == 7).all() and (buf[off + a[0].size:] == 7).all()


@pytest.mark.parametrize("n", [40, 400])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_hidden_keys_may_hold_anything(dev, which, bad, n):
    """Key n - 4 holds NaN or infinities: the queries before it do not see it."""
    a = _case([n, 30], [n, 30], 4, 2, 64)
    clean = _run(dev, *a)
    q, k, v, qs, ks = a
    (k if which == "k" else v)[n - 4, 0, 5:9] = bad
    got = _run(dev, q, k, v, qs, ks)
    want, tol = S.packed(*(np.where(np.isfinite(x), x, 0) for x in (q, k, v)), qs, ks, 0.125, 2)
    hurt = np.zeros(q.shape[:2], bool)
    hurt[n - 4:n, :2] = True
    assert (np.abs(got - want) <= tol[..., None])[~hurt].all()
    assert np.abs(clean - got)[~hurt].max() <= 2 * tol.max()
    if which == "k":
        assert np.isnan(got[n - 4:n, 0]).all() or not np.isnan(bad)
    else:
        assert not np.isfinite(got[n - 4:n, :2, 5:9]).any()
        assert np.isfinite(got[n - 4:n, :2, 9:]).all()


@pytest.mark.parametrize("nq, nk, heads", [(850, 850, 4), (40, 2500, 2)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, 1e30])
@pytest.mark.parametrize("which", ["k", "v"])
def test_hidden_keys_of_long_inputs(dev, which, bad, nq, nk, heads):
    """The same where the keys are taken apart ahead, and where they are split over blocks."""
    a = _case([nq], [nk], heads, 1, 64)
    q, k, v, qs, ks = a
    (k if which == "k" else v)[nk - 4, 0, 5:9] = bad
    got = _run(dev, *a)
    want, tol = S.packed(*(np.where(np.abs(x) < 1e20, x, 0) for x in (q, k, v)), qs, ks, 0.125, heads)
    assert (np.abs(got - want) <= tol[..., None])[:nq - 4].all()
    if which == "v":
        assert np.abs(got[nq - 4:, :, 5:9]).max() > 1e20 or not np.isfinite(got[nq - 4:, :, 5:9]).any()
        assert (np.abs(got - want)[..., 9:] <= tol[..., None]).all()


@pytest.mark.parametrize("nq, nk, heads", [(850, 850, 4), (40, 2500, 2), (90, 90, 2)])
@pytest.mark.parametrize("at", [0, 5, 31, 40])
def test_keys_of_zeros_and_tiny_keys(dev, nq, nk, heads, at):
    """Some keys and values are 0, some so small that they are next to nothing beside their
    neighbours: the queries that see only those get them in full."""
    q, k, v, qs, ks = _case([nq, 50], [nk, 50], heads, 1, 64)
    k[at:at + 3] = 0
    v[at:at + 2] = 0
    _check(_run(dev, q, k, v, qs, ks), q, k, v, qs, ks)
    v[:6] *= np.float32(1e-13)
    v[nk:nk + 7] *= np.float32(1e-30)
    got = _run(dev, q, k, v, qs, ks)
    _check(got, q, k, v, qs, ks)
    # relative to what the first queries see, not to the values they do not
    want, _ = S.packed(q, k, v, qs, ks, 0.125, heads)
    for r in [*range(0, 6 if nq == nk else 0), *range(nq, nq + 7)]:
        size = np.abs(want[r]).max()
        assert np.abs(got[r] - want[r]).max() <= 1e-5 * size, r


@pytest.mark.parametrize("size", [1e-36, 1e-33, 1e34])
@pytest.mark.parametrize("nq, nk, heads", [(850, 850, 4), (40, 2500, 2), (90, 90, 2)])
def test_tiny_and_huge_values_keep_their_bits(dev, nq, nk, heads, size):
    """The result is linear in V, and so is its bound as long as no value is subnormal (the
    smallest here are 5e-37): the bound at size 1, times the size."""
    q, k, v, qs, ks = _case([nq], [nk], heads, 1, 64)
    v[:] = (np.abs(v) + np.float32(0.5)) * np.float32(size)
    got = _run(dev, q, k, v, qs, ks).astype(np.float64)
    want, tol = S.packed(q, k, v / np.float64(np.float32(size)), qs, ks, 0.125, heads)
    assert (np.abs(got / np.float64(np.float32(size)) - want) <= tol[..., None]).all()


def test_large_and_small_values(dev):
    a = _case([90], [90], 2, 2, 64, amp=1.0)
    q, k, v, qs, ks = a
    for fq, fk, fv in ((30, 30, 1), (1e-20, 1e19, 1e30), (1e15, 1e-15, 1e-30), (1e-30, 1e-5, 1e5)):
        b = ((q * np.float32(fq)), (k * np.float32(fk)), (v * np.float32(fv)), qs, ks)
        _check(_run(dev, *b), *b)


def test_outliers_in_some_keys(dev):
    """Keys and values of very different sizes next to each other."""
    q, k, v, qs, ks = _case([300], [300], 2, 1, 64)
    r = np.random.default_rng(1)
    k *= (10.0 ** r.uniform(-4, 0, (300, 1, 64))).astype(np.float32)
    v *= (10.0 ** r.uniform(-6, 2, (300, 1, 64))).astype(np.float32)
    _check(_run(dev, q, k, v, qs, ks), q, k, v, qs, ks)


def test_infinite_scores(dev):
    """q . k beyond fp32: the row is NaN, as in fp32 arithmetic, and no other row is."""
    q, k, v, qs, ks = _case([20], [20], 2, 2, 64)
    q[7, 0] = 3e38
    q[9, 1, 3] = np.nan
    got = _run(dev, q, k, v, qs, ks)
    assert np.isnan(got[7, 0]).all() and np.isnan(got[9, 1]).all()
    ok = np.ones(q.shape[:2], bool)
    ok[7, 0] = ok[9, 1] = False
    assert np.isfinite(got[ok]).all()


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.5])
def test_scales(dev, scale):
    a = _case([60, 20], [60, 33], 4, 4, 32)
    _check(_run(dev, *a, scale), *a, scale)


def test_host_arrays(dev):
    q, k, v, qs, ks = _case([30, 5], [30, 9], 4, 2, 64)
    out = np.full(q.shape, 7, np.float32)
    sa.attention_packed(q, k, v, out, qs, ks)
    _check(out, q, k, v, qs, ks)


@pytest.mark.parametrize("n", [50, 900])
def test_another_stream_and_a_graph(dev, n):
    """Captured after one eager call of the size; every replay sees the inputs as they
    are then."""
    import torch
    a = _case([n, 7], [n, 7], 4, 2, 64)
    t = [torch.from_numpy(x).to(dev) for x in a]
    o = torch.zeros_like(t[0])
    st = torch.cuda.Stream()
    try:
        sa.set_stream(st)
        with torch.cuda.stream(st):
            sa.attention_packed(*t[:3], o, *t[3:])
        st.synchronize()
        _check(o.cpu().numpy(), *a)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            sa.attention_packed(*t[:3], o, *t[3:])
        for i in range(3):
            b = _case([n, 7], [n, 7], 4, 2, 64, seed=10 + i)
            for x, y in zip(t, b):
                x.copy_(torch.from_numpy(y))
            o.fill_(0)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            first = o.clone()
            _check(first.cpu().numpy(), *b)
            with torch.cuda.stream(st):
                sa.attention_packed(*t[:3], o, *t[3:])
            st.synchronize()
            assert torch.equal(first, o)
    finally:
        sa.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("nq, nk, heads", [(1700, 1700, 4), (41, 5200, 2)])
def test_replays_with_other_packings(dev, nq, nk, heads):
    """A graph of a call that takes the keys apart ahead, and of one that splits them: each
    replay with other sequences in the same rows, empty and overlong ones among them."""
    import torch
    q, k, v, _, _ = _case([nq], [nk], heads, 1, 32)
    t = [torch.from_numpy(x).to(dev) for x in (q, k, v)]
    qs, ks = torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    o = torch.zeros_like(t[0])
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        sa.set_stream(st)
        sa.attention_packed(*t, o, qs, ks)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            sa.attention_packed(*t, o, qs, ks)
        h = nq // 2
        for a, b in (([0, nq, nq], [0, nk, nk]), ([0, 0, nq], [0, 33, nk]), ([0, h, nq], [0, nk - 40, nk]),
                     ([0, h, h], [0, 5, nk]), ([0, nq, nq], [0, 1, nk])):
            a, b = np.array(a, np.int32), np.array(b, np.int32)
            qs.copy_(torch.from_numpy(a))
            ks.copy_(torch.from_numpy(b))
            o.fill_(4)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got = o.cpu().numpy()
            assert (got[a[-1]:] == 4).all()
            _check(got[:a[-1]], q[:a[-1]], k, v, a, b)
    finally:
        sa.set_stream(torch.cuda.current_stream())
