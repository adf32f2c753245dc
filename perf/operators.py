"""The attention operators of a serving loop, as measurable cases.

A batch of requests goes through four operators per layer: the prompts' attention
(`attention_packed`), the key/value rows into a cache of 8-bit codes with one
scale per block of tokens and head and back out of it (`KV8Cache.append`,
`.read`), each new token's attention over that cache (`.attention`), which also
adds up the weight every cached token has received, and the eviction of those that
received least (`.evict`).  Kinds:

  prompt  causal attention of packed prompts, each with `past` earlier tokens
  store   `new` tokens of each sequence stored behind its first `have`, and the
          values read back that the blocks they touched now stand for
  cached  one query per sequence over the cache, out and accumulated weights
  evict   each sequence cut to `budget` tokens per head, the last `recent` among
          them, and what is left read back

Lists (`past`, `new`, `have`, `lens`) are texts, one number per sequence.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"


def listed():
    return [
        # The 110M model, a prompt of a few words: the smallest call.
        dict(name="prompt_16_110m", kind="prompt", heads=12, kv_heads=12, head=64, past="0",
             new="16"),
        # Eight requests that arrived together, heads in groups of four (2048/512 dims).
        dict(name="prompt_8_ragged", kind="prompt", heads=32, kv_heads=8, head=64,
             past="0,0,0,0,0,0,0,0", new="1,7,300,64,129,511,33,200"),
        # The 3B model's heads of 100: two long prompts go on after what was cached.
        dict(name="prompt_chunks_3b", kind="prompt", heads=32, kv_heads=32, head=100,
             past="1500,803", new="256,17"),
        # One long document: the largest call.
        dict(name="prompt_4096", kind="prompt", heads=32, kv_heads=8, head=128, past="0",
             new="4096"),
        # A decode step of 32 requests, one token each.
        dict(name="store_step_32", kind="store", kv_heads=8, head=64, cap=2048, block=32,
             have=",".join(str(37 + 61 * i) for i in range(32)), new=",".join(["1"] * 32)),
        # Prompts of odd lengths stored behind what the sequences hold.
        dict(name="store_prompts", kind="store", kv_heads=8, head=128, cap=8192, block=64,
             have="0,0,1000,77,0", new="4096,2048,1000,513,31"),
        # One request of the 110M model at an ordinary length: latency.
        dict(name="cached_1_110m", kind="cached", heads=12, kv_heads=12, head=64, cap=1024,
             block=32, lens="200"),
        # Sixteen requests of very different lengths, grouped heads.
        dict(name="cached_16_ragged", kind="cached", heads=32, kv_heads=8, head=128, cap=4096,
             block=64, lens="4096,17,1,3333,64,2500,900,4000,129,3000,2047,1500,65,3700,700,2222"),
        # The 3B model's heads of 100, one key head per query head.
        dict(name="cached_8_3b", kind="cached", heads=32, kv_heads=32, head=100, cap=2048,
             block=16, lens="2048,300,1999,1024,77,1500,2000,511"),
        # One request over a very long context: one row per head, a long axis.
        dict(name="cached_1_131072", kind="cached", heads=32, kv_heads=8, head=128, cap=131072,
             block=128, lens="131072"),
        # A few chats of the 110M model over their budget by a little.
        dict(name="evict_4_110m", kind="evict", kv_heads=12, head=64, cap=1024, block=32,
             lens="600,513,1000,200", budget=512, recent=64),
        # Sixteen long requests cut to a quarter.
        dict(name="evict_16_long", kind="evict", kv_heads=8, head=128, cap=8192, block=64,
             lens="8192,8000,7777,6000,8192,5001,8100,4097,8192,8191,7000,6543,8192,8192,3000,1999",
             budget=2048, recent=256),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _texts(v):
    return ",".join(str(x) for x in v)


def _list(case, name):
    return [int(x) for x in case[name].split(",")]


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "store", "cached", "cached", "evict"])
    head = rng.choice([32, 48, 64, 64, 80, 96, 100, 128, 128, 192, 256])
    group = rng.choice([1, 1, 2, 4, 4, 5, 8])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    if kind != "prompt":
        block = rng.choice([16, 32, 64, 128])
    if kind == "prompt":
        heads = kv_heads * group
        n = _log(rng, 1, 16)
        longest = _log(rng, 16, 4096)
        new = [max(1, int(longest * rng.random() ** 2)) for _ in range(n - 1)] + [longest]
        past = [0] * n
        if rng.random() < 0.4:
            past = [_log(rng, 1, 4096) if rng.random() < 0.8 else 0 for _ in range(n)]
        # no more products, and no larger a padded score matrix, than the largest listed case
        while (sum(x * (p + x / 2) for p, x in zip(past, new)) * heads * head > 32 * 128 * 4096 * 2048
               or len(new) * max(new) * (max(new) + max(past)) * heads > 32 * 4096 * 4096):
            new = [max(1, x * 3 // 4) for x in new]
            past = [x * 3 // 4 for x in past]
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, head=head, past=_texts(past),
                    new=_texts(new))
    if kind == "store":
        n = _log(rng, 1, 64)
        top = max(1, min(4096, 9_000_000 // (n * kv_heads * head)))
        step = rng.random() < 0.4
        new = [1 if step else _log(rng, 1, top) for _ in range(n)]
        have = [rng.choice([0, _log(rng, 1, 2048)]) for _ in range(n)]
        # odd capacities too: a last block that is cut short
        cap = max(a + b for a, b in zip(have, new)) + rng.randint(0, 200)
        return dict(kind=kind, kv_heads=kv_heads, head=head, cap=cap, block=block,
                    have=_texts(have), new=_texts(new))
    n = _log(rng, 1, 64)
    top = max(64, min(65536, 100_000_000 // (n * kv_heads * head)))
    longest = _log(rng, 64, top)
    lens = [max(1, int(longest * rng.random())) for _ in range(n - 1)] + [longest]
    cap = longest + rng.randint(0, 200)
    if kind == "cached":
        return dict(kind=kind, heads=kv_heads * group, kv_heads=kv_heads, head=head, cap=cap,
                    block=block, lens=_texts(lens))
    budget = max(16, int(longest * rng.uniform(0.1, 0.9)))
    return dict(kind=kind, kv_heads=kv_heads, head=head, cap=cap, block=block, lens=_texts(lens),
                budget=budget, recent=int(budget * rng.choice([0, 0.1, 0.25, 0.5, 1])))


# ------------------------------------------------------------------- inputs

def _starts(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rows(g, *shape):
    """Activations as projections leave them: some channels several times the others."""
    x = torch.randn(shape, generator=g, device=DEV)
    return x * (0.5 + torch.rand(shape[-2:], generator=g, device=DEV) ** 4 * 4)


def _cache(g, n, case):
    """Codes and scales as stored rows leave them, in every slot, so also behind the lengths."""
    h, cap, d, t = case["kv_heads"], case["cap"], case["head"], case["block"]
    nb = -(-cap // t)
    amp = 0.5 + torch.rand((n, h, 1, d), generator=g, device=DEV) ** 4 * 2
    amp /= amp.amax(-1, keepdim=True)
    codes = (torch.randn((n, h, cap, d), generator=g, device=DEV) * (amp * 40)).round_()
    codes = codes.clamp_(-127, 127).to(torch.int8)
    return codes, (0.5 + torch.rand((n, h, nb), generator=g, device=DEV)) * 0.02


def _seen(g, n, case):
    """Attention weight received so far: a few tokens have most of it, and some have none."""
    u = torch.rand((n, case["kv_heads"], case["cap"]), generator=g, device=DEV)
    return torch.where(u < 0.1, torch.zeros_like(u), u ** 8 * 20)


def _inputs(case, seed):
    g = _gen(seed)
    kind, d = case["kind"], case["head"]
    if kind == "prompt":
        past, new = _list(case, "past"), _list(case, "new")
        tot = [p + x for p, x in zip(past, new)]
        return dict(q=_rows(g, sum(new), case["heads"], d), k=_rows(g, sum(tot), case["kv_heads"], d),
                    v=_rows(g, sum(tot), case["kv_heads"], d), q_starts=_starts(new),
                    k_starts=_starts(tot))
    lens = _list(case, "have" if kind == "store" else "lens")
    n, hk = len(lens), case["kv_heads"]
    kc, ks = _cache(g, n, case)
    vc, vs = _cache(g, n, case)
    s = dict(kc=kc, ks=ks, vc=vc, vs=vs)
    if kind == "store":
        new = _list(case, "new")
        first = [x - x % case["block"] for x in lens]
        s.update(k=_rows(g, sum(new), hk, d), v=_rows(g, sum(new), hk, d), starts=_starts(new),
                 lengths=_ints([a + b for a, b in zip(lens, new)]),
                 touched=_starts([a + b - f for a, b, f in zip(lens, new, first)]))
    elif kind == "cached":
        s.update(q=_rows(g, n, case["heads"], d), lengths=_ints(lens), seen=_seen(g, n, case))
    else:
        s.update(lengths=_ints(lens), seen=_seen(g, n, case),
                 left=_starts([min(x, case["budget"]) for x in lens]),
                 lengths2=_ints([min(x, case["budget"]) for x in lens]))
    return s


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    kind, d = case["kind"], case["head"]
    if kind == "prompt":
        s["out"] = torch.empty_like(s["q"])
    elif kind == "store":
        tail = int(s["touched"][-1])
        s["k_back"], s["v_back"] = (torch.empty((tail, case["kv_heads"], d), device=DEV)
                                    for _ in range(2))
    elif kind == "cached":
        s["out"], s["seen_out"] = torch.empty_like(s["q"]), torch.zeros_like(s["seen"])
    else:  # the cache that the next steps run on, blocks of the same size
        n, hk, b = len(s["lengths"]), case["kv_heads"], case["budget"]
        s["kc2"], s["vc2"] = (torch.zeros((n, hk, b, d), dtype=torch.int8, device=DEV)
                              for _ in range(2))
        s["ks2"], s["vs2"] = (torch.zeros((n, hk, -(-b // case["block"])), device=DEV)
                              for _ in range(2))
        s["seen2"] = torch.zeros((n, hk, b), device=DEV)
        s["kept"] = torch.empty((n, hk, b), dtype=torch.int32, device=DEV)
        s["k_back"], s["v_back"] = (torch.empty((int(s["left"][-1]), hk, d), device=DEV)
                                    for _ in range(2))
    if own:  # the handles that a serving loop keeps: addresses and sizes
        import simplang_amd as sa
        sa.set_stream(torch.cuda.current_stream())
        if kind != "prompt":
            s["cache"] = sa.KV8Cache(s["kc"], s["vc"], s["ks"], s["vs"], case["block"])
        if kind == "evict":
            s["cache2"] = sa.KV8Cache(s["kc2"], s["vc2"], s["ks2"], s["vs2"], case["block"])
    return s


# -------------------------------------------------------------- plain forms

def _seq_pos(starts, total):
    """Sequence and place in it of each packed row."""
    r = torch.arange(total, device=DEV)
    seq = torch.searchsorted(starts[1:].long(), r, right=True)
    return seq, r - starts.long()[seq]


def _padded(x, starts, longest):
    """Packed rows [total, H, D] as [sequences, H, longest, D]."""
    at = starts[:-1, None].long() + torch.arange(longest, device=DEV)
    return x[at.clamp(max=x.shape[0] - 1)].transpose(1, 2)


def _prompt(s):
    case = s["case"]
    hq, hk, d = case["heads"], case["kv_heads"], case["head"]
    new = _list(case, "new")
    lq, lk = max(new), max(p + x for p, x in zip(_list(case, "past"), new))
    n, g = len(new), hq // hk
    q = _padded(s["q"], s["q_starts"], lq).reshape(n, hk, g * lq, d)
    k = _padded(s["k"], s["k_starts"], lk)
    v = _padded(s["v"], s["k_starts"], lk)
    nq, nk = s["q_starts"].diff(), s["k_starts"].diff()
    last = torch.arange(lq, device=DEV) + (nk - nq)[:, None]  # the last key a query sees
    late = torch.arange(lk, device=DEV) > last[:, :, None]
    a = (torch.matmul(q, k.transpose(2, 3)) * (1 / math.sqrt(d))).view(n, hk, g, lq, lk)
    a.masked_fill_(late[:, None, None], -math.inf)
    a.sub_(a.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    o = torch.matmul(a.view(n, hk, g * lq, lk), v).view(n, hk, g, lq, d)
    o /= a.sum(-1, keepdim=True)
    seq, pos = _seq_pos(s["q_starts"], s["q"].shape[0])
    return o[seq, :, :, pos].reshape(-1, hq, d)


def _quotient(x, scale):
    """x / scale in 64 bits (a code is next to a border now and then) where the scale is
    above 0, else 0."""
    return torch.where(scale > 0, x.double() / scale.double(), 0.0)


def _store_one(x, codes, scales, seq, pos, row, fresh, block):
    """Stores packed rows x; the values of the rows (seq, pos), which are those of the
    blocks touched: row `row` of x where `fresh`, else codes that stay."""
    n, h, nb = scales.shape
    blk = seq * nb + pos // block
    new = x[row]                                              # [rows, H, D]
    top = torch.where(fresh[:, None], (new.abs().amax(-1).double() / 127).float(),
                      scales[seq, :, pos // block])           # old rows: their scale
    s = torch.zeros((n * nb, h), device=DEV)
    s.scatter_reduce_(0, blk[:, None].expand(-1, h), top, "amax")
    s = s[blk]                                                # [rows, H]
    old = codes[seq, :, pos]
    kept = (old * _quotient(scales[seq, :, pos // block], s)[..., None]).round()
    c = torch.where(fresh[:, None, None], _quotient(new, s[..., None]).round(), kept)
    c = c.clamp(-127, 127).to(torch.int8)
    codes[seq, :, pos] = c
    scales[seq, :, pos // block] = s
    return codes[seq, :, pos] * scales[seq, :, pos // block][..., None]


def _store(s):
    case = s["case"]
    t, st, tail = case["block"], s["starts"].long(), s["touched"].long()
    seq, at = _seq_pos(s["touched"], s["k_back"].shape[0])
    end = s["lengths"].long()
    pos = at + (end - tail.diff())[seq]
    row = st[1:][seq] - (end[seq] - pos)                      # below the sequence's first: old
    fresh = row >= st[seq]
    row = row.clamp(min=0)
    return tuple(_store_one(s[x], s[c], s[z], seq, pos, row, fresh, t)
                 for x, c, z in (("k", "kc", "ks"), ("v", "vc", "vs")))


def _cached(s):
    case = s["case"]
    n, hq, d = s["q"].shape
    hk, t, longest = case["kv_heads"], case["block"], max(_list(case, "lens"))
    nb = -(-longest // t)

    def values(c, z):
        z = z[:, :, :nb].repeat_interleave(t, 2)[:, :, :longest, None]
        return c[:, :, :longest] * z

    q = s["q"].view(n, hk, hq // hk, d)
    a = torch.matmul(q, values(s["kc"], s["ks"]).transpose(2, 3)) * (1 / math.sqrt(d))
    valid = (torch.arange(longest, device=DEV) < s["lengths"][:, None])[:, None, None]
    a = torch.where(valid, a, torch.full_like(a, -math.inf))
    a = (a - a.amax(-1, keepdim=True)).exp()
    a = a / a.sum(-1, keepdim=True)
    o = torch.matmul(a, values(s["vc"], s["vs"])).view(n, hq, d)
    seen = s["seen_out"]
    seen[:, :, :longest] = torch.where(valid[:, 0], s["seen"][:, :, :longest] + a.sum(2),
                                       seen[:, :, :longest])
    return o, seen


def _evict(s):
    case = s["case"]
    n, hk, cap = s["seen"].shape
    t, budget, recent = case["block"], case["budget"], case["recent"]
    longest = max(max(_list(case, "lens")), budget)
    idx = torch.arange(longest, device=DEV)
    length = s["lengths"].long()[:, None, None]
    rank = torch.full((n, hk, longest), -math.inf, device=DEV)
    rank[:, :, :min(cap, longest)] = s["seen"][:, :, :longest]
    rank = torch.where(idx >= length - recent, torch.full_like(rank, math.inf), rank)
    rank = torch.where(idx >= length, torch.full_like(rank, -math.inf), rank)
    kept = torch.argsort(rank, dim=-1, descending=True, stable=True)[:, :, :budget].sort(-1)[0]
    there = kept < length
    at = torch.where(there, kept, torch.zeros_like(kept))
    nb2 = -(-budget // t)
    out = []
    seq, pos = _seq_pos(s["left"], s["k_back"].shape[0])
    for c, z, c2, z2 in (("kc", "ks", "kc2", "ks2"), ("vc", "vs", "vc2", "vs2")):
        codes = torch.gather(s[c], 2, at[..., None].expand(-1, -1, -1, case["head"]))
        z1 = torch.where(there, torch.gather(s[z], 2, at // t), torch.zeros((), device=DEV))
        whole = torch.zeros((n, hk, nb2 * t), device=DEV)
        whole[:, :, :budget] = z1
        znew = whole.view(n, hk, nb2, t).amax(-1)
        ratio = _quotient(z1, znew.repeat_interleave(t, 2)[:, :, :budget])
        codes = (codes * ratio[..., None]).round().to(torch.int8)
        s[c2].copy_(torch.where(there[..., None], codes, s[c2]))
        filled = torch.arange(nb2, device=DEV) * t < length
        s[z2].copy_(torch.where(filled, znew, s[z2]))
        out.append(s[c2][seq, :, pos] * s[z2][seq, :, pos // t][..., None])
    seen = torch.where(there, torch.gather(s["seen"], 2, at), s["seen2"])
    s["seen2"].copy_(seen)
    s["kept"].copy_(torch.where(there, kept, torch.full_like(kept, -1)))
    return out[0], out[1], s["seen2"], s["kept"]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"prompt": _prompt, "store": _store, "cached": _cached, "evict": _evict}[kind](state)
    s = state
    if kind == "prompt":
        import simplang_amd as sa
        return sa.attention_packed(s["q"], s["k"], s["v"], s["out"], s["q_starts"], s["k_starts"])
    if kind == "store":
        s["cache"].append(s["k"], s["v"], s["starts"], s["lengths"])
        return s["cache"].read(s["touched"], s["lengths"], s["k_back"], s["v_back"])
    if kind == "cached":
        s["cache"].attention(s["q"], s["lengths"], s["out"], s["seen"], s["seen_out"])
        return s["out"], s["seen_out"]
    case = s["case"]
    s["cache"].evict(s["cache2"], s["lengths"], s["seen"], s["seen2"], s["kept"], case["budget"],
                     case["recent"])
    s["cache2"].read(s["left"], s["lengths2"], s["k_back"], s["v_back"])
    return s["k_back"], s["v_back"], s["seen2"], s["kept"]


# --------------------------------------------------------------------- work

def work(case):
    kind, d, hk = case["kind"], case["head"], case["kv_heads"]
    if kind == "prompt":
        past, new = _list(case, "past"), _list(case, "new")
        pairs = sum(x * p + x * (x + 1) // 2 for p, x in zip(past, new))
        rows = 2 * case["heads"] * sum(new) + 2 * hk * (sum(past) + sum(new))
        return dict(bytes=4 * d * rows, flops=4 * d * case["heads"] * pairs)
    t = case["block"]
    if kind == "store":
        have, new = _list(case, "have"), _list(case, "new")
        old = sum(x % t for x in have)
        # new rows in; old codes of the first blocks in; codes out; the touched blocks read
        # back: codes in, values out
        return dict(bytes=2 * hk * d * (4 * sum(new) + old + (old + sum(new)) * (1 + 1 + 4)),
                    flops=6 * hk * d * (old + sum(new)))
    lens = _list(case, "lens")
    blocks = sum(-(-x // t) for x in lens)
    if kind == "cached":
        return dict(bytes=hk * (2 * d + 8) * sum(lens) + 8 * hk * blocks
                    + 8 * d * case["heads"] * len(lens), flops=4 * d * case["heads"] * sum(lens))
    left = [min(x, case["budget"]) for x in lens]
    # the weights; codes of the tokens that stay in and out, and read back: in, and values
    # out; their scales, weights and places
    return dict(bytes=hk * (4 * sum(lens) + sum(left) * (2 * d * (1 + 1 + 1 + 4) + 8) + 24 * blocks),
                flops=6 * hk * d * sum(left))


# -------------------------------------------------------- the same in 64 bits

def _exact_prompt(case, s):
    new, hk = _list(case, "new"), case["kv_heads"]
    g, d = case["heads"] // hk, case["head"]
    q, k, v = (s[x].double() for x in "qkv")
    out = torch.empty_like(q)
    a = b = 0
    for x, p in zip(new, _list(case, "past")):
        hidden = torch.ones((x, p + x), dtype=torch.bool, device=DEV).triu(p + 1)
        for h in range(case["heads"]):
            kk, vv = k[b:b + p + x, h // g].contiguous(), v[b:b + p + x, h // g].contiguous()
            w = q[a:a + x, h].contiguous() @ kk.T.contiguous() / d ** 0.5
            out[a:a + x, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ vv
        a, b = a + x, b + p + x
    return out


def _exact_store(case, s):
    """Block by block: the stored scale is a 32-bit number, all else is in 64."""
    t, have, new = case["block"], _list(case, "have"), _list(case, "new")
    back = []
    for x, c, z in (("k", "kc", "ks"), ("v", "vc", "vs")):
        x, c, z = s[x].double().cpu().numpy(), s[c].cpu().numpy(), s[z].double().cpu().numpy()
        rows, r = [], 0
        for b, (m, n) in enumerate(zip(have, new)):
            for p in range(m - m % t, m + n, t):
                e = min(p + t, m + n)
                old = max(0, m - p)
                y = x[r + max(0, p - m):r + e - m]
                top = np.abs(y).max((0, 2))
                q0 = z[b, :, p // t]
                if old:
                    top = np.maximum(top, 127 * q0)
                scale = (top / 127).astype(np.float32).astype(np.float64)
                div = np.where(scale > 0, scale, 1)[:, None]
                kept = np.rint(c[b, :, p:p + old] * (q0[:, None] / div)[..., None])
                fresh = np.rint(y / div).transpose(1, 0, 2)
                rows.append((np.concatenate([kept, fresh], 1) * scale[:, None, None]).transpose(1, 0, 2))
            r += n
        back.append(torch.from_numpy(np.concatenate(rows)))
    return tuple(back)


def _exact_cached(case, s):
    t, hk = case["block"], case["kv_heads"]
    g, d = case["heads"] // hk, case["head"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    seen = torch.zeros(s["seen"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_list(case, "lens")):
        of = torch.arange(n, device=DEV) // t
        for h in range(hk):
            k = s["kc"][b, h, :n].double() * s["ks"][b, h].double()[of][:, None]
            v = s["vc"][b, h, :n].double() * s["vs"][b, h].double()[of][:, None]
            w = torch.softmax(s["q"][b, h * g:h * g + g].double() @ k.T.contiguous() / d ** 0.5, -1)
            out[b, h * g:h * g + g] = w @ v
            seen[b, h, :n] = s["seen"][b, h, :n].double() + w.sum(0)
    return out, seen


def _exact_evict(case, s):
    t, budget, recent = case["block"], case["budget"], case["recent"]
    seen, hk = s["seen"].double().cpu().numpy(), case["kv_heads"]
    lens = _list(case, "lens")
    seen2 = np.zeros((len(lens), hk, budget))
    kept = np.full((len(lens), hk, budget), -1, np.int64)
    for b, n in enumerate(lens):
        for h in range(hk):
            i = np.arange(n)
            at = np.sort(np.lexsort((i, -seen[b, h, :n], i < n - recent))[:budget])
            kept[b, h, :len(at)], seen2[b, h, :len(at)] = at, seen[b, h, at]
    back = []
    for c, z in (("kc", "ks"), ("vc", "vs")):
        c, z = s[c].cpu().numpy(), s[z].double().cpu().numpy()
        rows = []
        for b, n in enumerate(lens):
            m = min(n, budget)
            y = np.empty((m, hk, case["head"]))
            for h in range(hk):
                at = kept[b, h, :m]
                z1 = z[b, h, at // t]
                for p in range(0, m, t):
                    top = z1[p:p + t].max()
                    r = z1[p:p + t] / top if top > 0 else z1[p:p + t]
                    y[p:p + t, h] = np.rint(c[b, h, at[p:p + t]] * r[:, None]) * top
            rows.append(y)
        back.append(torch.from_numpy(np.concatenate(rows)))
    return back[0], back[1], torch.from_numpy(seen2), torch.from_numpy(kept)


def exact(case, seed):
    f = {"prompt": _exact_prompt, "store": _exact_store, "cached": _exact_cached,
         "evict": _exact_evict}[case["kind"]]
    return f(case, _inputs(case, seed))
