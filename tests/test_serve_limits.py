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
