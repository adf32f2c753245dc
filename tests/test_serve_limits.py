"""Refusals of the batch attention entry points at the edge of what they take, on the CPU:
every refused call ends before any device work, and calls of no rows show that the rest
passes the checks."""
import numpy as np
import pytest

import simplang_amd as sa
from test_serve_args import F, I, _cache, _prompt, _rows


@pytest.mark.parametrize("scale", [1e300, -1e39, 3e38])
def test_scales_beyond_fp32_are_refused(scale):
    """Finite in 64 bits, infinite in the kernels' arithmetic (powers of two: times 1.44)."""
    with pytest.raises(sa.SimpRTError, match="finite"):
        sa.attention_packed(**_prompt(), scale=scale)
    c = sa.KV8Cache(*_cache(), 16)
    q = np.zeros((2, 4, 32), F)
    with pytest.raises(sa.SimpRTError, match="finite"):
        c.attention(q, np.zeros(2, I), q.copy(), scale=scale)


@pytest.mark.parametrize("scale", [0.0, 1e-300, -2e38])
def test_scales_within_fp32_pass(scale):
    sa.attention_packed(**_prompt(tq=0), scale=scale)


def _views(layout):
    """K and V of a cache in one tensor, and the offset of V's first element behind K's."""
    b, h, cap, hs = 2, 3, 40, 32
    if layout == "row":        # K and V rows in turn
        x = np.zeros((b, h, cap, 2, hs), np.int8)
        return x[:, :, :, 0], x[:, :, :, 1]
    if layout == "token":      # [batch, capacity, K and V, heads, head_size]
        x = np.zeros((b, cap, 2, h, hs), np.int8)
        return x[:, :, 0].transpose(0, 2, 1, 3), x[:, :, 1].transpose(0, 2, 1, 3)
    if layout == "head":       # a head's K, then its V
        x = np.zeros((b, h, 2, cap, hs), np.int8)
        return x[:, :, 0], x[:, :, 1]
    if layout == "seq":
        x = np.zeros((b, 2, h, cap, hs), np.int8)
        return x[:, 0], x[:, 1]
    x = np.zeros((2, b, h, cap, hs), np.int8)
    return x[0], x[1]


@pytest.mark.parametrize("layout", ["row", "token", "head", "seq", "apart"])
def test_k_and_v_between_each_other_pass(layout):
    k, v = _views(layout)
    s = np.zeros((2, 2, 3, 3), F)
    for x, y in ((k, v), (v, k)):
        c = sa.KV8Cache(x, y, s[0], s[1], 16)
        c.append(*_rows(n=0, h=3), np.zeros(3, I), np.zeros(2, I))


def _part(x, by):
    """x, its first element moved by so many bytes (the memory behind it is not touched)."""
    from numpy.lib.stride_tricks import as_strided
    whole = x.base if x.base is not None else x
    at = x.ctypes.data - whole.ctypes.data + by * x.itemsize
    flat = whole.reshape(-1).view(x.dtype)[at // x.itemsize:]
    return as_strided(flat[:1], x.shape, x.strides)


@pytest.mark.parametrize("by", [4, 28, -4, 32 * 40, 32, -32 * 40 * 3, 32 * 40 * 2 + 32 * 39])
def test_k_and_v_that_share_codes_are_refused(by):
    x = np.zeros((4, 3, 40, 32), np.int8)
    k = x[1:3]
    s = np.zeros((2, 2, 3, 3), F)
    with pytest.raises(sa.SimpRTError, match="same memory"):
        sa.KV8Cache(k, _part(k, by), s[0], s[1], 16).append(*_rows(h=3), np.zeros(3, I), np.zeros(2, I))


@pytest.mark.parametrize("layout, by", [("row", 4), ("row", -4), ("row", 96), ("token", 32), ("token", 100),
                                        ("head", 32 * 39), ("head", -32), ("seq", 32), ("seq", -4)])
def test_k_and_v_that_overlap_between_each_other_are_refused(layout, by):
    """One is between the other's rows, heads or sequences, and reaches into them."""
    k, v = _views(layout)
    s = np.zeros((2, 2, 3, 3), F)
    with pytest.raises(sa.SimpRTError, match="same memory"):
        sa.KV8Cache(k, _part(v, by), s[0], s[1], 16).append(*_rows(h=3), np.zeros(3, I), np.zeros(2, I))


def test_scales_that_share_memory_are_refused():
    k, v = _views("apart")
    s = np.zeros((4, 3, 3), F)
    for by in (1, 3, -3, 9):
        with pytest.raises(sa.SimpRTError, match="same memory"):
            sa.KV8Cache(k, v, s[1:3], _part(s[1:3], by), 16).append(*_rows(h=3), np.zeros(3, I), np.zeros(2, I))
    z = np.zeros((2, 3, 2, 3), F)
    sa.KV8Cache(k, v, z[:, :, 0], z[:, :, 1], 16).append(*_rows(n=0, h=3), np.zeros(3, I), np.zeros(2, I))
    with pytest.raises(sa.SimpRTError, match="same memory"):
        sa.KV8Cache(k, v, z[:, :, 0], _part(z[:, :, 1], 1), 16).append(*_rows(h=3), np.zeros(3, I), np.zeros(2, I))


@pytest.mark.parametrize("block", [0, -16, 8, 24, 256])
def test_blocks_that_are_none_are_refused(block):
    a = _cache()
    with pytest.raises(ValueError, match="block"):
        sa.KV8Cache(*a[:2], np.zeros((2, 2, 3), F), np.zeros((2, 2, 3), F), block).append(
            *_rows(n=0), np.zeros(3, I), np.zeros(2, I))


def test_strides_of_dimensions_of_one_element_say_nothing():
    """One sequence, one head, one block of scales, one row: numpy gives a new dimension the
    stride 0, and a part of a larger tensor keeps the larger one's."""
    k, v, ks, vs = _cache(b=1, h=1, cap=16)
    whole = np.zeros((1, 1, 7), F)
    c = sa.KV8Cache(k, v, whole[:, :, 3:4], vs[0, 0][None, None], 16)
    c.append(*_rows(n=0, h=1), np.zeros(2, I), np.zeros(1, I))
    c = sa.KV8Cache(k, v, np.zeros((1, 1, 9), F)[:, :, ::9], vs, 16)
    c.append(*_rows(n=0, h=1), np.zeros(2, I), np.zeros(1, I))
    q = np.zeros((4, 32), F)
    # as far as the first check behind the descriptors'
    a = dict(q=q[None], k=q[:2][None], v=q[:2][None], out=q.copy()[None], q_starts=np.zeros(2, I), k_starts=np.zeros(2, I))
    with pytest.raises(sa.SimpRTError, match="finite"):
        sa.attention_packed(**a, scale=float("nan"))
    a = dict(q=q[:, None], k=q[:, None], v=q[:, None], out=q.copy()[:, None], q_starts=np.zeros(2, I), k_starts=np.zeros(2, I))
    with pytest.raises(sa.SimpRTError, match="finite"):
        sa.attention_packed(**a, scale=float("nan"))
    for x in (q[None, :1], q[:1, None], q[:1][None]):
        with pytest.raises(sa.SimpRTError, match="finite"):
            c.attention(x, np.zeros(1, I), x.copy(), scale=float("nan"))


def test_read_of_one_row_between_the_heads():
    """K and V of one token, head by head in turn: as far as the cache's own check."""
    x = np.zeros((1, 2, 2, 32), F)
    c = sa.KV8Cache(*_cache(b=1), 16)
    st, ln = np.zeros(2, I), np.zeros(1, I)
    for k, v in ((x[:, :, 0], x[:, :, 1]), (x[0, :, 0][None], x[0, :, 1][None])):
        with pytest.raises(sa.SimpRTError) as e:
            c.read(st, ln, k, v)
        assert "shares memory" not in str(e.value)
        with pytest.raises(sa.SimpRTError, match="shares memory"):
            c.read(st, ln, k, _part(v, 1))


def test_lists_of_one_element_have_any_stride():
    x = np.zeros((5, 3), I)
    c = sa.KV8Cache(*_cache(b=1), 16)
    c.append(*_rows(n=0), np.zeros(2, I), x[2:3, 1])
    with pytest.raises(ValueError, match="contiguous"):
        c.append(*_rows(n=0), x[1:3, 1], x[2:3, 1])


def test_no_head_size_is_refused():
    with pytest.raises(sa.SimpRTError, match="1..256"):
        sa.attention_packed(**_prompt(hs=0))


def test_scales_whose_blocks_are_not_side_by_side_are_refused():
    k, v = _cache(b=1, h=1)[:2]
    s = np.zeros((1, 1, 6), F)
    for x in (s[:, :, ::2], s[:, :, 2::-1], np.broadcast_to(s[:, :, :1], (1, 1, 3))):
        with pytest.raises(ValueError, match="innermost"):
            sa.KV8Cache(k, v, x, x, 16)
