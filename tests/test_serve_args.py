"""Refusals of the batch attention entry points, on the CPU: every one of these calls
has to end before any device work."""
import numpy as np
import pytest

import simplang_amd as sa

F, I = np.float32, np.int32


def _prompt(tq=8, tk=8, heads=4, kv=2, hs=32, n=1):
    return dict(q=np.zeros((tq, heads, hs), F), k=np.zeros((tk, kv, hs), F), v=np.zeros((tk, kv, hs), F),
                out=np.zeros((tq, heads, hs), F), q_starts=np.zeros(n + 1, I), k_starts=np.zeros(n + 1, I))


@pytest.mark.parametrize("change, match", [
    (dict(out=np.zeros((8, 4, 31), F)), "shape mismatch"),
    (dict(v=np.zeros((7, 2, 32), F)), "shape mismatch"),
    (dict(k=np.zeros((8, 2, 16), F), v=np.zeros((8, 2, 16), F)), "shape mismatch"),
    (dict(k=np.zeros((8, 3, 32), F), v=np.zeros((8, 3, 32), F)), "no multiple"),
    (dict(q_starts=np.zeros(3, I)), "sequences"),
    (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"),
])
def test_prompt_refusals(change, match):
    with pytest.raises(sa.SimpRTError, match=match):
        sa.attention_packed(**{**_prompt(), **change})


def test_prompt_refuses_head_sizes_and_shared_memory():
    with pytest.raises(sa.SimpRTError, match="1..256"):
        sa.attention_packed(**_prompt(hs=257))
    a = _prompt()
    with pytest.raises(sa.SimpRTError, match="shares memory"):
        sa.attention_packed(**{**a, "out": a["q"]})
    with pytest.raises(sa.SimpRTError, match="shares memory"):
        sa.attention_packed(**{**_prompt(heads=2), "k": (x := np.zeros((8, 2, 32), F)), "out": x})


def test_prompt_refuses_types_and_strides():
    a = _prompt()
    with pytest.raises(TypeError, match="float32"):
        sa.attention_packed(**{**a, "q": a["q"].astype(np.float64)})
    with pytest.raises(TypeError, match="int32"):
        sa.attention_packed(**{**a, "q_starts": np.zeros(2, np.int64)})
    with pytest.raises(sa.SimpRTError, match="inner stride"):
        sa.attention_packed(**{**a, "q": np.zeros((8, 4, 64), F)[:, :, ::2]})


def test_prompt_of_nothing_is_no_error():
    sa.attention_packed(**_prompt(tq=0))
    sa.attention_packed(**_prompt(n=0))


def _cache(b=2, h=2, cap=40, hs=32, block=16, dt=np.int8):
    nb = -(-cap // block)
    return [np.zeros((b, h, cap, hs), dt), np.zeros((b, h, cap, hs), dt),
            np.zeros((b, h, nb), F), np.zeros((b, h, nb), F)]


def _rows(n=4, h=2, hs=32):
    return np.zeros((n, h, hs), F), np.zeros((n, h, hs), F)


def test_cache_shapes():
    with pytest.raises(TypeError, match="int8"):
        sa.KV8Cache(*_cache(dt=np.uint8), 16)
    a = _cache()
    with pytest.raises(ValueError, match="scales"):
        sa.KV8Cache(*a, 32)
    with pytest.raises(ValueError, match="head_size"):
        sa.KV8Cache(a[0], a[1][:, :, :39], a[2], a[3], 16)
    with pytest.raises(ValueError, match="innermost"):
        x = np.zeros((2, 2, 40, 64), np.int8)[..., ::2]
        sa.KV8Cache(x, x, a[2], a[3], 16)
    with pytest.raises(ValueError, match="same strides"):
        sa.KV8Cache(a[0], np.zeros((2, 2, 40, 64), np.int8)[..., :32], a[2], a[3], 16)


@pytest.mark.parametrize("make, match", [
    (lambda: sa.KV8Cache(*_cache(block=8), 8), "block"),
    (lambda: sa.KV8Cache(*_cache(hs=34), 16), "head_size"),
    (lambda: sa.KV8Cache(*_cache(hs=12), 16), "head_size"),
    (lambda: sa.KV8Cache(*_cache(hs=260), 16), "head_size"),
    (lambda: sa.KV8Cache(*[np.broadcast_to(x, (2, *x.shape[1:])) for x in _cache(b=1)], 16), "overlap"),
    (lambda: sa.KV8Cache(np.zeros((2, 2, 40, 34), np.int8)[..., :32], np.zeros((2, 2, 40, 34), np.int8)[..., :32],
                         *_cache()[2:], 16), "4-byte"),
])
def test_cache_refusals(make, match):
    c = make()
    k, v = _rows(hs=c.head_size)
    out = np.zeros((2, 4, c.head_size), F)
    with pytest.raises(sa.SimpRTError, match=match):
        c.append(k, v, np.zeros(3, I), np.zeros(2, I))
    with pytest.raises(sa.SimpRTError, match=match):
        c.read(np.zeros(3, I), np.zeros(2, I), k, v)
    with pytest.raises(sa.SimpRTError, match=match):
        c.attention(out.copy(), np.zeros(2, I), out)


@pytest.mark.parametrize("st, ln, shape, match", [
    (2, 2, (4, 2, 32), "starts"), (3, 3, (4, 2, 32), "lengths"), (3, 2, (4, 3, 32), "rows"),
    (3, 2, (4, 2, 28), "rows"),
])
def test_row_refusals(st, ln, shape, match):
    c = sa.KV8Cache(*_cache(), 16)
    k, v = np.zeros(shape, F), np.zeros(shape, F)
    with pytest.raises(sa.SimpRTError, match=match):
        c.append(k, v, np.zeros(st, I), np.zeros(ln, I))
    with pytest.raises(sa.SimpRTError, match=match):
        c.read(np.zeros(st, I), np.zeros(ln, I), k, v)


def test_attention_refusals():
    c = sa.KV8Cache(*_cache(), 16)
    q, ln = np.zeros((2, 4, 32), F), np.zeros(2, I)
    seen = np.zeros((2, 2, 40), F)
    for args, match in [
            ((np.zeros((2, 3, 32), F), ln, np.zeros((2, 3, 32), F)), "no multiple"),
            ((np.zeros((1, 4, 32), F), ln, np.zeros((1, 4, 32), F)), "batch, heads"),
            ((q, ln, np.zeros((2, 2, 32), F)), "batch, heads"),
            ((q, np.zeros(1, I), q.copy()), "lengths"),
            ((q, ln, q), "shares memory"),
            ((q, ln, q.copy(), seen[:, :, :39], seen[:, :, :39]), "capacity"),
            ((q, ln, q.copy(), seen, seen[:, :1]), "capacity"),
            ((q, ln, q.copy(), seen, seen, float("nan")), "finite")]:
        with pytest.raises(sa.SimpRTError, match=match):
            c.attention(*args)
    big = np.zeros(400, F)
    with pytest.raises(sa.SimpRTError, match="shares memory"):  # shifted by one: neither the same nor apart
        c.attention(q, ln, q.copy(), big[:160].reshape(2, 2, 40), big[1:161].reshape(2, 2, 40))
    with pytest.raises(ValueError, match="together"):
        c.attention(q, ln, q.copy(), seen)


def test_evict_refusals():
    src, dst = _cache(), _cache(cap=32)
    c, to = sa.KV8Cache(*src, 16), sa.KV8Cache(*dst, 16)
    ln, seen, ns, kept = np.zeros(2, I), np.zeros((2, 2, 40), F), np.zeros((2, 2, 32), F), np.zeros((2, 2, 20), I)
    for args, match in [
            ((to, ln, seen, ns, np.zeros((2, 2, 33), I), 33, 0), "budget"),
            ((to, ln, seen, ns, kept, 20, 21), "budget"),
            ((to, ln, seen, ns, kept, 20, -1), "budget"),
            ((to, ln, seen, ns, np.zeros((2, 2, 19), I), 20, 0), "kept"),
            ((to, ln, seen, ns[:, :, :19], kept, 20, 0), "new_seen"),
            ((to, ln, seen[:, :, :39], ns, kept, 20, 0), "seen"),
            ((sa.KV8Cache(*_cache(cap=32, block=32), 32), ln, seen, ns, kept, 20, 0), "differ"),
            ((sa.KV8Cache(*_cache(cap=32, h=1), 16), ln, seen, ns, kept, 20, 0), "differ"),
            ((c, ln, seen, np.zeros((2, 2, 40), F), kept, 20, 0), "shares memory"),
            ((to, ln, seen, seen, kept, 20, 0), "shares memory")]:
        with pytest.raises(sa.SimpRTError, match=match):
            c.evict(*args)
    with pytest.raises(TypeError, match="int32"):
        c.evict(to, ln, seen, ns, kept.astype(np.int64), 20)


def test_lists_and_outputs_in_one_memory_are_refused():
    a = _prompt(tq=8)
    flat = a["out"].reshape(-1).view(I)
    for name in ("q_starts", "k_starts"):
        with pytest.raises(sa.SimpRTError, match="shares memory"):
            sa.attention_packed(**{**a, name: flat[3:5]})
    arrays = _cache()
    c = sa.KV8Cache(*arrays, 16)
    k, v = _rows()
    with pytest.raises(sa.SimpRTError, match="shares memory"):
        c.read(np.zeros(3, I), np.zeros(2, I), k, k)
    with pytest.raises(sa.SimpRTError, match="shares memory"):
        c.read(v.reshape(-1).view(I)[:3], np.zeros(2, I), k, v)
    with pytest.raises(sa.SimpRTError, match="shares memory"):
        c.read(np.zeros(3, I), k.reshape(-1).view(I)[5:7], k, v)
    w = np.zeros((5, 2, 32), F)
    with pytest.raises(sa.SimpRTError, match="shares memory"):  # a row on
        c.read(np.zeros(3, I), np.zeros(2, I), w[:4], w[1:])
    w = np.zeros((4, 2, 96), F)
    with pytest.raises(sa.SimpRTError, match="shares memory"):  # the end of a head's row over the next one's
        c.read(np.zeros(3, I), np.zeros(2, I), w[..., :32], w[..., 31:63])
    q = np.zeros((2, 4, 32), F)
    out = q.copy()
    seen = np.zeros((2, 2, 40), F)
    with pytest.raises(sa.SimpRTError, match="shares memory"):
        c.attention(q, out.reshape(-1).view(I)[7:9], out)
    with pytest.raises(sa.SimpRTError, match="shares memory"):
        c.attention(q, seen.reshape(-1).view(I)[7:9], out, seen, seen)
    with pytest.raises(sa.SimpRTError, match="share memory"):
        c.append(k, v, np.zeros(3, I), arrays[2].reshape(-1).view(I)[:2])


def test_one_array_for_k_and_v_is_refused():
    a = _cache()
    k, v = _rows()
    for c in (sa.KV8Cache(a[0], a[0], a[2], a[3], 16), sa.KV8Cache(a[0], a[1], a[2], a[2], 16)):
        with pytest.raises(sa.SimpRTError, match="same memory"):
            c.append(k, v, np.zeros(3, I), np.zeros(2, I))


def test_far_rows_are_refused():
    """Strides beyond what the kernels' offsets hold, without the memory."""
    from numpy.lib.stride_tricks import as_strided
    a = _prompt(tq=2, tk=2)
    x = as_strided(np.zeros(1, F), (2, 2, 32), (4 << 23, 128, 4))
    with pytest.raises(sa.SimpRTError, match="2\\^23"):
        sa.attention_packed(**{**a, "k": x})
    with pytest.raises(sa.SimpRTError, match="2\\^23"):
        sa.attention_packed(**{**a, "v": x})
    y = as_strided(np.zeros(4, np.int8), (2, 2, 40, 32), (40 << 24, 32, 1 << 24, 1))
    z = as_strided(np.zeros(4, np.int8), (2, 2, 40, 32), (40 << 24, 32, 1 << 24, 1))
    with pytest.raises(sa.SimpRTError, match="2\\^24"):
        sa.KV8Cache(y, z, *_cache()[2:], 16).append(*_rows(), np.zeros(3, I), np.zeros(2, I))


def test_null_cache():
    from simplang_amd import host
    z = [None, None] + [0] * 7
    assert sa.lib.simp_rt_kv8_append(None, *z, *z, *host.desc1(np.zeros(1, I)), *host.desc1(np.zeros(1, I))) == -1
    assert "null" in sa.last_error()
