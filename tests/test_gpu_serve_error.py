"""How close the batch attention is to 64-bit arithmetic in the 2-norm, next to the elementwise
worst cases of the other tests, which cannot see a low-order part go missing.

Bounds, from the arithmetic: with unit normal q and k and the scale 1 / sqrt(D) a score
is off by the root of D products' squared errors, each about 2^-23, and of some D / 16
roundings of a sum of order one: about 2 * 2^-23 in all, 2.4e-7.  The weights follow,
their errors are independent from key to key, and an fp32 sum over the keys adds
some 2^-24 a part: 2.5e-7 to 6e-7 are expected, and 1.5e-6 is the bound, for the forms
with few roundings and the long sums alike.  The model on the CPU shows that every part
of the operands is needed for that."""
import numpy as np
import pytest

BOUND = 1.5e-6


def _off(got, want):
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))


def _softmax(a):
    p = np.exp(a - a.max(-1, keepdims=True))
    return p / p.sum(-1, keepdims=True)


def _halves(x, axis):
    """x as two f16 parts below 2^15, scaled by a power of two per slice."""
    s = 2.0 ** (14 - np.floor(np.log2(np.abs(x).max(axis, keepdims=True))))
    hi = np.float16(x * s).astype(np.float64)
    lo = np.float16(x * s - hi).astype(np.float64)
    return hi / s, lo / s


def test_every_f16_part_counts():
    """attention_packed: hi hi + hi lo + lo hi of both products."""
    r = np.random.default_rng(0)
    q, k, v = (r.standard_normal((n, 128)).astype(np.float32).astype(np.float64) for n in (40, 700, 700))
    want = _softmax(q @ k.T * 128 ** -0.5) @ v
    (qh, ql), (kh, kl), (vh, vl) = _halves(q, 1), _halves(k, (0, 1)), _halves(v, (0, 1))

    def run(without):
        s = [qh @ kh.T, ql @ kh.T * (without != "q"), qh @ kl.T * (without != "k")]
        p = _softmax(sum(s) * 128 ** -0.5)
        ph, pl = _halves(p, 1)
        return ph @ vh + pl @ vh * (without != "p") + ph @ vl * (without != "v")

    assert _off(run(None), want) < BOUND / 4
    for name in "qkpv":
        assert _off(run(name), want) > 10 * BOUND, name


def test_every_byte_counts():
    """KV8Cache.attention: three bytes of q, and of the weights of 64 tokens."""
    r = np.random.default_rng(1)
    q = r.standard_normal((40, 128))
    k, v = (r.integers(-127, 128, (700, 128)) * 0.02 for _ in range(2))

    def whole(x, axis, byte):
        s = 8.35e6 / np.abs(x).max(axis, keepdims=True)
        u = np.rint(x * s)
        lost = {None: 0, 0: (u + 128) % 256 - 128, 1: ((u + 128) // 256 + 128) % 256 * 256 - 128 * 256}[byte]
        return (u - lost) / s

    def run(qb, pb):
        a = whole(q, 1, qb) @ k.T * 128 ** -0.5
        p = _softmax(a)
        o = sum(whole(p[:, t:t + 64], 1, pb) @ v[t:t + 64] for t in range(0, 700, 64))
        return o

    want = _softmax(q @ k.T * 128 ** -0.5) @ v
    assert _off(run(None, None), want) < BOUND / 4
    for lost in ((0, None), (1, None), (None, 0), (None, 1)):
        assert _off(run(*lost), want) > 1.5 * BOUND, lost


# (queries, keys, heads, kv heads, head_size, sequences): made in the block, the same with heads
# above 128, taken apart ahead with eight and four waves, split over blocks in each form
PACKED = [(200, 200, 4, 4, 64, 1), (40, 40, 16, 4, 20, 20), (130, 130, 12, 12, 128, 3), (512, 512, 8, 8, 96, 4),
          (300, 300, 16, 16, 192, 2), (300, 300, 16, 16, 256, 2), (1024, 1024, 32, 8, 64, 1), (1024, 1024, 32, 8, 128, 2),
          (800, 800, 32, 8, 192, 2), (800, 800, 32, 8, 256, 2), (40, 2500, 2, 1, 64, 1), (17, 6000, 4, 2, 100, 2),
          (9, 2000, 4, 4, 256, 1), (850, 900, 4, 1, 64, 1), (900, 3000, 4, 1, 128, 1), (1, 20000, 4, 1, 128, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("mean", [0, 1])
@pytest.mark.parametrize("nq, nk, heads, kv, hs, n", PACKED)
def test_packed_off_64_bits(dev, nq, nk, heads, kv, hs, n, mean):
    import torch
    import simplang_amd as sa
    g = torch.Generator(device=dev)
    g.manual_seed(nq + nk + hs)
    q, k, v = (torch.randn(s, device=dev, generator=g) for s in ((n, nq, heads, hs), (n, nk, kv, hs), (n, nk, kv, hs)))
    if mean:
        v = v * 0.1 + 1
    out = torch.zeros_like(q)
    qs, ks = (torch.arange(0, n * m + 1, m, dtype=torch.int32, device=dev) for m in (nq, nk))
    sa.attention_packed(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), out.flatten(0, 1), qs, ks)
    hidden = torch.ones((nq, nk), dtype=torch.bool, device=dev).triu(nk - nq + 1)
    err = size = 0.0
    for s in range(n):
        for h in range(heads):
            kk, vv = k[s, :, h * kv // heads].double(), v[s, :, h * kv // heads].double()
            a = (q[s, :, h].double() @ kk.T.contiguous() * hs ** -0.5).masked_fill(hidden, -float("inf"))
            want = torch.softmax(a, -1) @ vv
            err += (out[s, :, h].double() - want).square().sum().item()
            size += want.square().sum().item()
    off = (err / size) ** 0.5
    print(f"off {off:.3g}")
    assert off <= BOUND


# (tokens, heads, kv heads, head_size, sequences): four columns' bytes side by side up to groups of
# four, a column a head above; one piece and several
CACHED = [(50, 4, 4, 64, 3), (600, 8, 2, 128, 2), (2000, 4, 1, 256, 2), (2000, 2, 1, 192, 1), (20000, 8, 2, 128, 1),
          (600, 16, 2, 128, 2), (2000, 8, 1, 64, 2), (2000, 8, 1, 256, 1), (900, 33, 1, 100, 1), (5000, 5, 1, 192, 70)]


@pytest.mark.gpu
@pytest.mark.parametrize("mean", [0, 100])
@pytest.mark.parametrize("n, heads, kv, hs, batch", CACHED)
def test_cached_off_64_bits(dev, n, heads, kv, hs, batch, mean):
    import torch
    import simplang_amd as sa
    g = torch.Generator(device=dev)
    g.manual_seed(n + hs)
    nb, t = -(-n // 64), torch.arange(n, device=dev) // 64
    codes = [(torch.randn((batch, kv, n, hs), device=dev, generator=g) * (4 if m else 40) + m).round_().clamp_(-127, 127).to(torch.int8)
             for m in (0, mean)]
    scales = [(torch.rand((batch, kv, nb), device=dev, generator=g) + 0.5) * 0.02 for _ in range(2)]
    q = torch.randn((batch, heads, hs), device=dev, generator=g)
    out, seen, seen_out = torch.zeros_like(q), torch.zeros((batch, kv, n), device=dev), torch.zeros((batch, kv, n), device=dev)
    ln = torch.full((batch,), n, dtype=torch.int32, device=dev)
    sa.KV8Cache(*codes, *scales, 64).attention(q, ln, out, seen, seen_out)
    err, size = np.zeros(2), np.zeros(2)
    for b in range(batch):
        for h in range(kv):
            k, v = (c[b, h].double() * s[b, h].double()[t][:, None] for c, s in zip(codes, scales))
            rows = slice(h * heads // kv, (h + 1) * heads // kv)
            w = torch.softmax(q[b, rows].double() @ k.T.contiguous() * hs ** -0.5, -1)
            for i, (got, want) in enumerate(((out[b, rows], w @ v), (seen_out[b, h], w.sum(0)))):
                err[i] += (got.double() - want).square().sum().item()
                size[i] += want.square().sum().item()
    off = np.sqrt(err / size)
    print("off", off)
    assert (off <= BOUND).all(), off
