"""The batch attention at the ends of its sizes: rows far apart, many sequences, many heads,
and calls of two threads at once."""
import numpy as np
import pytest

import simplang_amd as sa
import _serve as S

pytestmark = pytest.mark.gpu


def _packed(dev, q, k, v, qs, ks, out=None):
    import torch
    out = torch.full_like(q, 7.0) if out is None else out
    sa.attention_packed(q, k, v, out, *(torch.from_numpy(np.asarray(x, np.int32)).to(dev) for x in (qs, ks)))
    return out


def _check(got, q, k, v, qs, ks):
    want, tol = S.packed(*(x.cpu().numpy() for x in (q, k, v)), qs, ks, q.shape[2] ** -0.5, q.shape[1] // k.shape[1])
    some = ~np.isnan(want)
    assert (np.abs(got.cpu().numpy() - want) <= tol[..., None])[some].all()


@pytest.mark.parametrize("heads, n", [(1, 150), (26, 150), (1, 700)])
def test_rows_more_than_32_bits_apart(dev, heads, n):
    """Rows of k and v nearly 2^23 elements apart, those of q and out 2^24: byte offsets up to
    2^34. Made in the block, taken apart ahead (26 heads over one), split over blocks."""
    import torch
    far, hs, nq = (1 << 23) - 4, 64, 130 if n < 700 else 20
    if heads > 1:
        nq = n
    base = [torch.empty(nq * 2 * far, device=dev) for _ in range(2)] + [torch.empty(n * far, device=dev) for _ in range(2)]
    q, out = (torch.as_strided(b, (nq, heads, hs), (2 * far, hs + 4, 1)) for b in base[:2])
    k, v = (torch.as_strided(b, (n, 1, hs), (far, hs, 1)) for b in base[2:])
    g = torch.Generator(device=dev)
    g.manual_seed(n)
    for x in (q, k, v):
        x.copy_(torch.randn(x.shape, device=dev, generator=g))
    st = [0, nq], [0, n]
    _packed(dev, q, k, v, *st, out=out)
    _check(out, q, k, v, *st)
    del base, q, k, v, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n, heads, kv", [(32767, 2, 1), (5000, 1, 1)])
def test_many_short_sequences(dev, n, heads, kv):
    import torch
    r = np.random.default_rng(n)
    nq, nk = r.integers(0, 3, n), r.integers(0, 4, n)
    nq[-1], nk[-1] = 3, 70
    g = torch.Generator(device=dev)
    g.manual_seed(n)
    q, k, v = (torch.randn((int(m.sum()) + 2, h, 16), device=dev, generator=g) for m, h in ((nq, heads), (nk, kv), (nk, kv)))
    st = S.starts(nq), S.starts(nk)
    got = _packed(dev, q, k, v, *st)
    assert (got[-2:] == 7).all()
    _check(got[:-2], q[:-2], k, v, *st)


@pytest.mark.parametrize("heads, kv, hs, nq, nk", [(65535, 65535, 4, 1, 3), (65535, 1, 4, 1, 5), (4096, 2, 16, 3, 700), (1000, 1000, 16, 2, 900)])
def test_many_heads(dev, heads, kv, hs, nq, nk):
    import torch
    g = torch.Generator(device=dev)
    g.manual_seed(heads)
    q, k, v = (torch.randn((m, h, hs), device=dev, generator=g) for m, h in ((nq, heads), (nk, kv), (nk, kv)))
    got = _packed(dev, q, k, v, [0, nq], [0, nk])
    pick = np.unique(np.linspace(0, heads - 1, 50).astype(int))
    of = pick * kv // heads
    for h, c in zip(pick, of):
        _check(got[:, h:h + 1], q[:, h:h + 1], k[:, c:c + 1], v[:, c:c + 1], [0, nq], [0, nk])


def test_many_heads_over_a_cache(dev):
    """4096 query heads to a kv head, and 32767 kv heads."""
    import torch
    from test_gpu_kv8 import Pair, _attend
    r = np.random.default_rng(0)
    p = Pair(dev, 1, 1, 300, 16, 16)
    _attend(p, r.standard_normal((1, 4096, 16)).astype(np.float32), [299], seen=np.zeros((1, 1, 300), np.float32))
    p = Pair(dev, 1, 32767, 20, 16, 16)
    q = r.standard_normal((1, 32767, 16)).astype(np.float32)
    k, v = (r.standard_normal((2, 32767, 16)).astype(np.float32) for _ in range(2))
    p.append(k, v, [2], [17])
    p.same()
    _attend(p, q, [17])


def test_two_threads_on_one_stream(dev):
    """Calls that write scratch with one launch and read it with the next, from two threads."""
    import threading
    import torch
    jobs = []
    for i, (nq, nk, heads, kv) in enumerate([(40, 2500, 2, 1), (850, 850, 8, 2)]):
        g = torch.Generator(device=dev)
        g.manual_seed(i)
        x = [torch.randn((m, h, 64), device=dev, generator=g) for m, h in ((nq, heads), (nk, kv), (nk, kv))]
        st = [torch.tensor([0, m], dtype=torch.int32, device=dev) for m in (nq, nk)]
        want = torch.zeros_like(x[0])
        sa.attention_packed(*x, want, *st)
        _check(want, *x, [0, nq], [0, nk])
        jobs.append((x, st, want))
    torch.cuda.synchronize()
    fails = []

    def work(x, st, want):
        torch.cuda.set_device(0)
        sa.set_stream(torch.cuda.current_stream())
        out = torch.zeros_like(want)
        for _ in range(50):
            out.zero_()
            sa.attention_packed(*x, out, *st)
            if not torch.equal(out, want):
                fails.append(len(want))
                return

    ts = [threading.Thread(target=work, args=j) for j in jobs for _ in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not fails
