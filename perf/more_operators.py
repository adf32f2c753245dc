"""Microscaled 4-bit floating point operators, as measurable cases.

MX4 rows hold E2M1 codes, two to a byte (low nibble = even element), and one power of two
for each block of 32 elements along the row, as a byte s that stands for 2^(s - 127).  A
feed-forward block on such operands is quantize, swiglu (both projections and the gate),
quantize, matmul.  Kinds:

  quant  fp32 rows [m, k] to codes and scales, and the values that they stand for back
  mm     out[m, n] = A B^T, A [m, k] and B [n, k] both MX4, fp32 out
  gate   out = silu(A W1^T) * (A W3^T), all three MX4, fp32 out
"""
import torch

own = False

DEV = "cuda:0"


def listed():
    return [
        # One token's activations of the 3B model: the smallest call.
        dict(name="quant_1x3200", kind="quant", m=1, k=3200),
        # A prompt of odd length, rows that end inside a block and inside a byte.
        dict(name="quant_odd_717x1533", kind="quant", m=717, k=1533),
        # A weight matrix, or the activations of many long prompts.
        dict(name="quant_8192x8192", kind="quant", m=8192, k=8192),
        # Decode: one token through the classifier of a 32000-token vocabulary.
        dict(name="mm_1x3200x32000", kind="mm", m=1, k=3200, n=32000),
        # Sixteen concurrent requests through the 3B model's down projection.
        dict(name="mm_16x8640x3200", kind="mm", m=16, k=8640, n=3200),
        # A 200-token prompt through its up projection.
        dict(name="mm_200x3200x8640", kind="mm", m=200, k=3200, n=8640),
        # Sizes that are no multiple of anything.
        dict(name="mm_odd_717x1533x2051", kind="mm", m=717, k=1533, n=2051),
        # The benchmark's largest square product.
        dict(name="mm_8192", kind="mm", m=8192, k=8192, n=8192),
        # Decode: one token of the 110M model, latency.
        dict(name="gate_1x768x2048", kind="gate", m=1, k=768, n=2048),
        # Sixteen concurrent requests of the 3B model.
        dict(name="gate_16x3200x8640", kind="gate", m=16, k=3200, n=8640),
        # A prompt of odd length through the 1B model's feed-forward.
        dict(name="gate_301x2048x8192", kind="gate", m=301, k=2048, n=8192),
        # Long prompts of the same model, packed.
        dict(name="gate_4096x2048x8192", kind="gate", m=4096, k=2048, n=8192),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _size(rng, lo, hi, step):
    """Log-uniform in [lo, hi]; two in three rounded to a multiple of step."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 1 / 3 else max(step, v // step * step)


def draw(rng):
    kind = rng.choice(["quant", "mm", "mm", "gate", "gate"])
    if kind == "quant":
        k = _size(rng, 32, 16384, 32)
        return dict(kind=kind, m=_log(rng, 1, min(16384, 8192 * 8192 // k)), k=k)
    k, n = _size(rng, 64, 8640, 64), _size(rng, 64, 32000, 64)
    # no more products than the largest listed case, and as many rows as such a batch has
    most = 8192 ** 3 // (k * n * (2 if kind == "gate" else 1))
    return dict(kind=kind, m=_log(rng, 1, max(1, min(8192, most))), k=k, n=n)


# ------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _activations(g, m, k):
    """Activations as norms and gates leave them: some channels several times the others."""
    amp = 0.5 + torch.rand((1, k), generator=g, device=DEV) ** 4 * 8
    return torch.randn((m, k), generator=g, device=DEV) * amp


def _weights(g, n, k):
    """Projection weights: rows of somewhat different sizes."""
    amp = 0.01 + 0.03 * torch.rand((n, 1), generator=g, device=DEV)
    return torch.randn((n, k), generator=g, device=DEV) * amp


def _inputs(case, seed):
    g = _gen(seed)
    x = _activations(g, case["m"], case["k"])
    if case["kind"] == "quant":
        return dict(x=x)
    s = dict(zip(("a", "sa"), _quantize(x)))
    for b, sb in (("b", "sb"),) if case["kind"] == "mm" else (("w1", "s1"), ("w3", "s3")):
        s[b], s[sb] = _quantize(_weights(g, case["n"], case["k"]))
    return s


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    m, k = case["m"], case["k"]
    if case["kind"] == "quant":
        s["codes"] = torch.empty((m, (k + 1) // 2), dtype=torch.uint8, device=DEV)
        s["scales"] = torch.empty((m, (k + 31) // 32), dtype=torch.uint8, device=DEV)
        s["out"] = torch.empty((m, k), device=DEV)
    else:
        s["out"] = torch.empty((m, case["n"]), device=DEV)
    if own:
        import simplang_amd as sa
        sa.set_stream(torch.cuda.current_stream())
    return s


# -------------------------------------------------------------- plain forms

def _quantize(x):
    """MX4 codes and scales of fp32 rows; x / 2^e in 64 bits, where it is exact."""
    m, k = x.shape
    blocks = (k + 31) // 32
    if k % 32:
        x = torch.cat([x, torch.zeros((m, 32 * blocks - k), device=x.device)], 1)
    x = x.view(m, blocks, 32)
    top = x.abs().amax(-1)
    e = torch.frexp(top)[1] - 3                    # floor(log2(top)) - 2
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)
    down = ((1023 - e.long()) << 52).view(torch.float64)
    v = x * down[..., None]
    a = v.abs()
    c = (a > 0.25).to(torch.uint8)
    for low in (1.25, 2.5, 5.0):                   # ties below an even code's value
        c += a > low
    for high in (0.75, 1.75, 3.5):                 # and above one's
        c += a >= high
    c += (v.signbit()).to(torch.uint8) * 8
    c = c.view(m, 16 * blocks, 2)
    codes = c[..., 0] | (c[..., 1] << 4)
    return codes[:, :(k + 1) // 2].contiguous(), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """The fp32 values of MX4 rows, two for every byte."""
    c = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1)
    mag = (c & 7).float()
    # codes 0 .. 4 count halves, 5 .. 7 are 3, 4, 6
    mag = torch.where(mag <= 4, mag * 0.5, torch.where(mag == 7, mag - 1, mag - 2))
    mag = torch.where(c > 7, -mag, mag)
    two = ((scales.int()) << 23).view(torch.float32).repeat_interleave(32, 1)[:, :c.shape[1]]
    return mag * two


def _product(a, b):
    return torch.matmul(_values(*a), _values(*b).t())


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        if kind == "quant":
            return _values(*_quantize(s["x"]))[:, :s["x"].shape[1]]
        a = s["a"], s["sa"]
        if kind == "mm":
            return _product(a, (s["b"], s["sb"]))
        g = _product(a, (s["w1"], s["s1"]))
        return g / (1 + torch.exp(-g)) * _product(a, (s["w3"], s["s3"]))
    import simplang_amd as sa
    if kind == "quant":
        sa.quantize_mx4(s["x"], s["codes"], s["scales"])
        return sa.dequantize_mx4(s["codes"], s["scales"], s["out"])
    if kind == "mm":
        return sa.matmul_mx4(s["a"], s["sa"], s["b"], s["sb"], s["out"])
    return sa.swiglu_mx4(s["a"], s["sa"], s["w1"], s["s1"], s["w3"], s["s3"], s["out"])


# --------------------------------------------------------------------- work

def work(case):
    m, k = case["m"], case["k"]
    row = (k + 1) // 2 + (k + 31) // 32
    if case["kind"] == "quant":
        # values in, codes and scales out and in again, values out
        return dict(bytes=m * (8 * k + 2 * row), flops=4 * m * k)
    mats, n = (2 if case["kind"] == "gate" else 1), case["n"]
    return dict(bytes=(m + mats * n) * row + 4 * m * n, flops=2 * mats * m * n * k)


# -------------------------------------------------------- the same in 64 bits

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values(codes, scales, k):
    """Block by block: a table by byte has both nibbles' values at once."""
    half = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=torch.float64, device=DEV)
    byte = torch.arange(256, device=DEV)
    pair = torch.stack([half[byte % 16], half[byte // 16]], -1)
    two = torch.tensor([2.0 ** (s - 127) for s in range(255)] + [float("nan")],
                       dtype=torch.float64, device=DEV)
    v = torch.empty((codes.shape[0], k), dtype=torch.float64, device=DEV)
    for j in range(scales.shape[1]):
        u = pair[codes[:, 16 * j:16 * j + 16].long()].reshape(codes.shape[0], -1)
        u *= two[scales[:, j].long()][:, None]
        v[:, 32 * j:32 * j + 32] = u[:, :k - 32 * j]
    return v


def _exact_quant(x):
    """Block by block: the exponent by searching among the powers of two, the value as the
    nearest of the eight, the one with the even code where two are as near."""
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    powers = torch.tensor([2.0 ** e for e in range(-149, 128)], dtype=torch.float64, device=DEV)
    table = torch.tensor(_E2M1, dtype=torch.float64, device=DEV)
    odd = torch.arange(8, device=DEV) % 2 * 1e-9
    for j in range(0, x.shape[1], 32):
        y = x[:, j:j + 32].double()
        top = y.abs().amax(1, keepdim=True)
        e = (torch.searchsorted(powers, top, right=True) - 1 - 149 - 2).clamp(min=-127)
        unit = powers[e + 149]
        # (fp32 values next to a midpoint are 2^-27 or more from it: 1e-9 only splits ties)
        near = ((y.abs() / unit)[..., None] - table).abs() + odd
        out[:, j:j + 32] = table[near.argmin(-1)] * unit * torch.where(y < 0, -1.0, 1.0)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "quant":
        return _exact_quant(s["x"])
    k = case["k"]
    a = _exact_values(s["a"], s["sa"], k)
    if case["kind"] == "mm":
        return a @ _exact_values(s["b"], s["sb"], k).t().contiguous()
    g = a @ _exact_values(s["w1"], s["s1"], k).t().contiguous()
    u = a @ _exact_values(s["w3"], s["s3"], k).t().contiguous()
    return u * g * torch.sigmoid(g)
