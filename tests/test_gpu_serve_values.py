"""The batch attention operators at values that only some of their forms meet: pieces of a
row in which every score is -inf, values that grow by many powers of
ten, queries that are tiny beside the keys."""
import numpy as np
import pytest

import simplang_amd as sa
import _serve as S

pytestmark = pytest.mark.gpu

# made in the block, taken apart ahead, split over blocks (made), split over blocks (wide)
FORMS = [(90, 300, 2, 1, 64), (850, 900, 4, 1, 64), (40, 2500, 2, 1, 64), (9, 2000, 1, 1, 256)]


def _inputs(nq, nk, heads, kv, hs, seed=0):
    r = np.random.default_rng(seed + nq + nk)
    f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    return f(nq, heads, hs), f(nk, kv, hs), f(nk, kv, hs)


def _run(dev, q, k, v, scale=None):
    import torch
    t = [torch.from_numpy(x).to(dev) for x in (q, k, v)]
    st = [torch.tensor([0, len(x)], dtype=torch.int32, device=dev) for x in (q, k)]
    out = torch.full(q.shape, 7.0, device=dev)
    sa.attention_packed(*t, out, *st, scale)
    return out.cpu().numpy()


def _want(q, k, v, gone, scale=None):
    """(out, bound) in 64 bits, with the keys in `gone` left out."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    nq, nk, group = len(q), len(k), q.shape[1] // k.shape[1]
    hidden = np.arange(nk)[None, :] > np.arange(nq)[:, None] + nk - nq
    hidden = hidden | gone[None, :]
    out, tol = np.zeros((*q.shape[:2], v.shape[2])), np.zeros(q.shape[:2])
    for h in range(q.shape[1]):
        x = [np.where(gone[:, None], 0, y[:, h // group]).astype(np.float64) for y in (k, v)]
        qq = q[:, h].astype(np.float64)
        out[:, h], _ = S.attention(qq, *x, scale, hidden)
        tol[:, h] = S.row_bound(qq, *x, scale, hidden)
    return out, tol


@pytest.mark.parametrize("where", ["first", "last"])
@pytest.mark.parametrize("gone", [192, 224, 400])
@pytest.mark.parametrize("how", ["channel", "overflow"])
@pytest.mark.parametrize("nq, nk, heads, kv, hs", FORMS)
def test_pieces_of_nothing_but_minus_infinity(dev, nq, nk, heads, kv, hs, how, gone, where):
    """Keys that score -inf have the weight 0, also where they fill a piece of the row:
    through a channel of -inf, and finite ones through products below -3.4e38."""
    gone = min(gone, nk - 64)
    q, k, v = _inputs(nq, nk, heads, kv, hs)
    at = np.zeros(nk, bool)
    at[:gone] = True
    if where == "last":
        at = np.roll(at, nk - gone)
    if how == "channel":
        q[..., 0], k[..., 0] = 1, 0
        k[at, :, 0] = -np.inf
    else:
        q = (np.abs(q) + np.float32(0.5)) * np.float32(1e19)
        k *= np.float32(1e-19)
        k[at] = -1e20
    got = _run(dev, q, k, v)
    want, tol = _want(q, k, v, at)
    seen = (~at)[None, :] & (np.arange(nk)[None, :] <= np.arange(nq)[:, None] + nk - nq)
    some = seen.any(1)
    assert np.isnan(got[~some]).all()
    assert (np.abs(got - want) <= tol[..., None])[some].all(), np.argwhere(~(np.abs(got - want) <= tol[..., None]))[:4]


@pytest.mark.parametrize("nq, nk, heads, kv, hs", FORMS)
def test_rows_of_nothing_but_minus_infinity(dev, nq, nk, heads, kv, hs):
    """No weight to share out: 0 / 0, in whichever form."""
    q, k, v = _inputs(nq, nk, heads, kv, hs)
    k[:] = -1e20
    assert np.isnan(_run(dev, (np.abs(q) + np.float32(0.5)) * np.float32(1e20), k, v)).all()
    k[..., 1:] = 0
    k[..., 0] = -np.inf
    q[..., 0] = 1
    assert np.isnan(_run(dev, q, k, v)).all()


@pytest.mark.parametrize("powers", [(-25, 25), (-30, -10, 10, 30), (-36, 35), (25, -25), (-3, 3)], ids=str)
@pytest.mark.parametrize("nq, heads, kv, hs", [(128, 2, 2, 64), (130, 1, 1, 100), (128, 2, 1, 192), (850, 4, 1, 64)])
def test_rows_before_much_larger_values(dev, nq, heads, kv, hs, powers):
    """Values that grow by many powers of ten every 32 keys: a row that sees only the first
    ones has them in full."""
    q, k, v = _inputs(nq, nq, heads, kv, hs)
    v = np.abs(v) + np.float32(0.5)
    step = np.minimum(np.arange(nq) // 32, len(powers) - 1)
    v *= (10.0 ** np.array(powers, np.float64)[step]).astype(np.float32)[:, None, None]
    got = _run(dev, q, k, v)
    want, _ = _want(q, k, v, np.zeros(nq, bool))
    # every value is above 0, so the bound of a row of ones is relative to the row
    _, tol = _want(q, k, np.ones_like(v), np.zeros(nq, bool))
    bad = np.abs(got - want) > tol[..., None] * want
    assert not bad.any(), np.argwhere(bad)[:4]


@pytest.mark.parametrize("size", [1e-30, 1e-34, 1e-36])
@pytest.mark.parametrize("heads", [2, 5])
def test_tiny_queries_keep_their_bits(dev, heads, size):
    """q . k is what counts, however the size is shared between them (values of 5e-38 and
    above, none subnormal)."""
    import torch
    from test_gpu_kv8 import Pair, _attend
    p = Pair(dev, 2, 1, 300, 64, 32)
    q = np.random.default_rng(5).standard_normal((2, heads, 64))
    q = (np.sign(q) * (np.abs(q) + 0.05) * size).astype(np.float32)
    p.np.ks *= np.float32(1 / size)
    p.t[2].copy_(torch.from_numpy(p.np.ks))
    _attend(p, q, [300, 77], seen=np.zeros((2, 1, 300), np.float32))


@pytest.mark.parametrize("heads", [2, 5])
def test_huge_queries_over_tiny_codes(dev, heads):
    """The largest element of a query may meet codes of 0 only: its size alone is no score."""
    import torch
    from test_gpu_kv8 import Pair, _attend
    p = Pair(dev, 2, 1, 300, 64, 32)
    p.np.kc[..., 0] = 0
    p.t[0].copy_(torch.from_numpy(p.np.kc))
    p.np.ks *= np.float32(1e5)
    p.t[2].copy_(torch.from_numpy(p.np.ks))
    q = np.zeros((2, heads, 64), np.float32)
    q[..., 0] = 1e36
    _attend(p, q, [300, 77], seen=np.zeros((2, 1, 300), np.float32))


@pytest.mark.parametrize("odd", [0, 3, 1 << 40])
def test_strides_of_one_row_and_one_head(dev, odd):
    """One row, one head: their strides are any number."""
    import torch
    from test_gpu_kv8 import Pair, _rows
    p = Pair(dev, 1, 1, 40, 64, 16)

    def one(x):
        return torch.as_strided(x, x.shape, (odd, odd, 1)) if odd < 99 else torch.as_strided(x, x.shape, (odd, odd + 1, 1))

    k, v = _rows(1, 1, 64)
    st, ln = np.array([0, 1], np.int32), np.array([21], np.int32)
    p.np.append(k, v, st, ln)
    up = p.up(k, v, st, ln)
    p.gpu.append(one(up[0]), one(up[1]), *up[2:])
    p.same()
    back = [torch.zeros((1, 1, 64), device=dev) for _ in range(2)]
    want = np.zeros((2, 1, 1, 64), np.float32)
    p.np.read(st, ln, *want)
    p.gpu.read(*up[2:], one(back[0]), one(back[1]))
    assert all(np.array_equal(b.cpu().numpy(), w) for b, w in zip(back, want))
    q = p.up(k)[0]
    out = torch.zeros_like(q)
    p.gpu.attention(one(q), up[3], one(out))
    ref, _, tol, _ = p.np.attention(k, ln, 0.125)
    assert (np.abs(out.cpu().numpy() - ref) <= tol[..., None]).all()
    out.fill_(7)
    sa.attention_packed(one(q), one(back[0]), one(back[1]), one(out), up[2], up[2])
    assert np.abs(out.cpu().numpy() - want[1]).max() <= 4 * S.EPS * np.abs(want[1]).max()


def test_capture_of_a_long_prompt_without_a_warm_up_call(dev):
    """Where the scratch for K and V taken apart ahead cannot be had, the blocks take them
    apart for themselves; after a warm-up call it is had."""
    import torch
    q, k, v = _inputs(900, 900, 4, 1, 64)
    more = _inputs(900, 900, 4, 1, 64, seed=1)
    want = [_want(*x, np.zeros(900, bool)) for x in ((q, k, v), more)]
    t = [torch.from_numpy(x).to(dev) for x in (q, k, v)]
    up = [torch.from_numpy(x).to(dev) for x in more]
    n = 32  # as many sequences of the same rows: enough blocks without splitting the keys
    wide = [x.repeat(n, 1, 1) for x in t]
    starts = torch.arange(0, 900 * n + 1, 900, dtype=torch.int32, device=dev)
    out = torch.zeros_like(wide[0])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        sa.set_stream(stream)
        g = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        for i in range(2):
            with torch.cuda.graph(g[i], stream=stream):
                sa.attention_packed(*wide, out, starts, starts)
            if i == 0:
                sa.attention_packed(*wide, out, starts, starts)
                stream.synchronize()
        for x, (ref, tol) in zip((t, up, t), (want[0], want[1], want[0])):
            for a, b in zip(wide, x):
                a.copy_(b.repeat(n, 1, 1))
            for y in g:
                out.fill_(5)
                torch.cuda.synchronize()
                y.replay()
                torch.cuda.synchronize()
                got = out.view(n, *q.shape).cpu().numpy()
                assert (np.abs(got - ref) <= tol[..., None]).all()
    finally:
        sa.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("size", [1e5, 1e9, 1e20])
@pytest.mark.parametrize("nq, nk, heads, kv, hs", FORMS + [(5, 5, 1, 1, 33), (70, 70, 2, 1, 2)])
def test_a_channel_that_masks_keys(dev, nq, nk, heads, kv, hs, size):
    """Channel 0 of a query is far above the others, and 0 in the keys that are not masked:
    what the others add up to counts in full."""
    q, k, v = _inputs(nq, nk, heads, kv, hs)
    gone = np.random.default_rng(3).random(nk) < 0.3
    gone[0] = False
    q[..., 0], k[..., 0] = size, 0
    k[gone, :, 0] = -1
    if size == 1e5:
        k[gone, :, 0] = -1e2
    got = _run(dev, q, k, v)
    want, tol = _want(q[..., 1:], k[..., 1:], v, gone, hs ** -0.5)
    assert (np.abs(got - want) <= tol[..., None]).all(), float(np.max(np.abs(got - want) / tol[..., None]))
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off < 2e-6, off


@pytest.mark.parametrize("power", [-12, -20, -28, -40, -60])
@pytest.mark.parametrize("nq, nk, heads, kv, hs", FORMS + [(800, 811, 4, 1, 192)])
def test_channels_far_below_the_others(dev, nq, nk, heads, kv, hs, power):
    """Some channels of V are 2^power of the rest: off by no more than 2^-38 of the largest
    value, besides what fp32 sums of their own size may be off.  So is the rest, by
    channels of K that are that small."""
    q, k, v = _inputs(nq, nk, heads, kv, hs)
    top = np.abs(v).max()
    small = np.arange(hs) % 7 == 3
    v[..., small] *= np.float32(2.0 ** power)
    k[..., np.arange(hs) % 5 == 2] *= np.float32(2.0 ** power)
    got = _run(dev, q, k, v)
    none = np.zeros(nk, bool)
    want, tol = _want(q, k, v, none)
    assert (np.abs(got - want) <= tol[..., None]).all()
    want, tol = _want(q, k, v[..., small], none)
    assert (np.abs(got[..., small] - want) <= tol[..., None] + 2.0 ** -38 * top).all()
    assert np.linalg.norm(got[..., small] - want) <= (2e-6 * np.linalg.norm(want) + 2.0 ** -39 * top * want.size ** 0.5)
