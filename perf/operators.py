"""Cases and plain forms of the serving-step operators: norm + rotation + cache append, the 4-bit KV cache read back,
attention over it, and sampling.

A 4-bit cache holds one row per (sequence, KV head, position): ``ceil(head_dim / 8)`` 32-bit words of 4-bit codes (dim
``8 w + i`` in bits ``4 i .. 4 i + 3`` of word w, tail codes zero) and one 32-bit word with two bfloat16 numbers, the step
in the low half and the lowest value ``lo`` in the high half.  A code stands for ``lo + code * step``.  K and V have their
own planes, ``[sequences, kv_heads, max_len, words]`` and ``[sequences, kv_heads, max_len]``.  The append is defined down
to its f32 roundings (f32 products and sums one by one, the norm's mean square in f64), so codes can be compared exactly.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5


def _case(name, op, **kw):
    return dict(name=name, op=op, **kw)


def listed():
    return [
        # one decode token of the repository's decoder (32 heads of 100, 640 positions), appended to the 4-bit cache
        _case("append4 one token", "append4", seqs=1, tokens=1, heads=32, kv=32, hd=100, lmax=640, start=576, norm=False),
        # 16 sequences' decode step with an f32 cache and norms of queries and keys
        _case("append32 decode 16", "append32", seqs=16, tokens=1, heads=32, kv=32, hd=100, lmax=640, start=575, norm=True),
        # a prompt of 512 tokens for each of 16 sequences, grouped KV heads, norms, 4-bit cache, read back for the prompt's own attention
        _case("append4 prompt 16x512", "append4", seqs=16, tokens=512, heads=32, kv=8, hd=128, lmax=640, start=0, norm=True),
        # a prompt's rows read back at the decoder's own shape
        _case("read 2x577", "read", seqs=2, rows=577, kv=32, hd=100, lmax=640),
        # long rows of a grouped cache read back
        _case("read 4x8192", "read", seqs=4, rows=8192, kv=8, hd=128, lmax=8192),
        # one sequence of the decoder, in the middle of its 128 decode steps
        _case("attn one sequence", "attn", seqs=1, t=1, heads=32, kv=32, hd=100, lmax=640, lo=577, hi=577),
        # 16 sequences of the decoder between the first and the last decode step
        _case("attn 16 sequences", "attn", seqs=16, t=1, heads=32, kv=32, hd=100, lmax=640, lo=513, hi=640),
        # five drafted tokens checked at once for four sequences
        _case("attn 4x5 drafted", "attn", seqs=4, t=5, heads=32, kv=8, hd=128, lmax=4096, lo=1501, hi=4001),
        # long ragged contexts with grouped KV heads
        _case("attn 8 long", "attn", seqs=8, t=1, heads=32, kv=8, hd=128, lmax=32768, lo=8191, hi=32768),
        # one sequence, the usual nucleus sampling over the decoder's vocabulary
        _case("sample one", "sample", n=1, vocab=32000, how="nucleus"),
        # a batch whose requests each bring their own settings
        _case("sample 16 mixed", "sample", n=16, vocab=32000, how="mixed"),
        # a large batch over a large vocabulary
        _case("sample 128 large", "sample", n=128, vocab=131072, how="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append4", "append32", "read", "attn", "attn", "sample"])
    if op == "sample":
        return dict(op=op, n=_log(rng, 1, 100), vocab=_log(rng, 500, 131072), how=rng.choice(["plain", "topk", "nucleus", "minp", "mixed"]))
    kv = rng.choice([1, 2, 4, 5, 8, 16, 32])
    hd = rng.choice([32, 64, 80, 96, 100, 104, 112, 124, 128, 128])
    if op == "read":
        rows = _log(rng, 1, 8192)
        return dict(op=op, seqs=rng.randint(1, 4), rows=rows, kv=min(kv, 8), hd=hd, lmax=_multiple(rows + rng.randint(0, 64)))
    heads = kv * rng.choice([1, 1, 2, 3, 4, 7, 8]) if kv <= 8 else kv
    if op == "attn":
        t = rng.choice([1, 1, 1, 2, 3, 5, 8])
        hi = _log(rng, 1, 32768 * 4 // max(4, t * heads // kv) if kv <= 8 else 2000)  # the products of the longest listed case at most
        return dict(op=op, seqs=_log(rng, 1, 8 if hi > 2000 else 32), t=t, heads=heads, kv=kv, hd=hd, lmax=_multiple(hi + rng.randint(0, 64)),
                    lo=rng.randint((hi + 1) // 2, hi), hi=hi)
    tokens = _log(rng, 1, 500)
    start = rng.randint(0, 100)
    return dict(op=op, seqs=rng.randint(1, 16), tokens=tokens, heads=heads, kv=min(kv, 8) if heads % min(kv, 8) == 0 else kv, hd=hd,
                lmax=_multiple(start + tokens + rng.randint(0, 40)), start=start, norm=rng.random() < 0.6)


def _multiple(n):
    return (n + 3) // 4 * 4


# ---- inputs ----------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _lens(case):
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    return [hi if n == 1 else lo + (hi - lo) * b // (n - 1) for b in range(n)]


def _planes(case, g):
    """A cache as a run of appends leaves it: every row quantised from values with a few wide channels."""
    wide = 1.0 + 3.0 * (torch.rand(case["kv"], 1, case["hd"], generator=g, device="cuda") < 0.05).float()
    out = {}
    for side in ("k", "v"):
        codes, steps = [], []
        for _ in range(case["seqs"]):
            c, s = _pack(*_quantise(_randn(g, case["kv"], case["lmax"], case["hd"]) * wide))
            codes.append(c)
            steps.append(s)
        out[side + "_codes"], out[side + "_steps"] = torch.stack(codes), torch.stack(steps)
    return out


def prepare(case, seed):
    g = _gen(seed)
    op, s = case["op"], {"case": case}
    if op == "sample":
        n, v = case["n"], case["vocab"]
        s["logits"] = _randn(g, n, v) * 2.5
        s["u"] = torch.rand(n, generator=g, device="cuda")
        rows = np.arange(n)
        hows = {"plain": 0, "topk": 1, "nucleus": 2, "minp": 3}
        kind = rows % 6 if case["how"] == "mixed" else np.full(n, hows[case["how"]])
        # 0 temperature alone, 1 top-k, 2 nucleus, 3 min-p, 4 all three, 5 greedy
        put = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
        s["temperature"] = put(np.where(kind == 5, 0.0, 0.6 + 0.1 * (rows % 8)), torch.float32)
        s["top_k"] = put(np.where((kind == 1) | (kind == 4), 20 + 10 * (rows % 7), 0), torch.int32)
        s["top_p"] = put(np.where((kind == 2) | (kind == 4), 0.8 + 0.03 * (rows % 6), 1.0), torch.float32)
        s["min_p"] = put(np.where((kind == 3) | (kind == 4), 0.02 + 0.01 * (rows % 5), 0.0), torch.float32)
        return s
    if op == "attn":
        s.update(_planes(case, g))
        s["q"] = _randn(g, case["seqs"], case["t"], case["heads"], case["hd"])
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
        return s
    if op == "read":
        s.update(_planes(case, g))
        b = torch.arange(case["seqs"], device="cuda")[:, None] * case["lmax"]
        s["rows"] = (b + torch.arange(case["rows"], device="cuda")[None, :]).reshape(-1)
        return s
    n, hd, half = case["seqs"] * case["tokens"], case["hd"], case["hd"] // 2
    s["qkv"] = _randn(g, n, (case["heads"] + 2 * case["kv"]) * hd)
    pos = torch.arange(case["start"], case["start"] + case["tokens"], device="cuda")
    s["positions"] = pos.repeat(case["seqs"]).to(torch.int32)
    s["rows"] = (torch.arange(case["seqs"], device="cuda")[:, None] * case["lmax"] + pos[None, :]).reshape(-1)
    ang = torch.arange(case["lmax"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    s["gq"] = 1.0 + 0.1 * _randn(g, hd) if case["norm"] else None
    s["gk"] = 1.0 + 0.1 * _randn(g, hd) if case["norm"] else None
    if op == "append32":
        s["k"] = _randn(g, case["seqs"], case["kv"], case["lmax"], hd)
        s["v"] = _randn(g, case["seqs"], case["kv"], case["lmax"], hd)
    else:
        w = (hd + 7) // 8
        for side in ("k", "v"):
            s[side + "_codes"] = torch.zeros(case["seqs"], case["kv"], case["lmax"], w, dtype=torch.int32, device="cuda")
            s[side + "_steps"] = torch.zeros(case["seqs"], case["kv"], case["lmax"], dtype=torch.int32, device="cuda")
    return s


# ---- plain forms -----------------------------------------------------------------------------

def _bf16_toward(x, up):
    """The bfloat16 neighbour of x at or above it (up) or at or below it, as f32."""
    i = x.view(torch.int32)
    cut = i & -65536
    away = (i != cut) & ((x > 0) if up else (x < 0))
    return (cut + away.to(torch.int32) * 65536).view(torch.float32)


def _quantise(x):
    """Rows of f32 values -> codes (f32 numbers 0..15), step and lo per row."""
    lo = _bf16_toward(x.amin(-1), False)
    step = _bf16_toward(((x.amax(-1) - lo) / torch.full_like(lo, 15.0)).clamp_min(2.0 ** -100), True)  # a true quotient, not times 1/15
    code = ((x - lo[..., None]) * (1.0 / step)[..., None]).round().clamp(0.0, 15.0)
    return code, step, lo


def _pack(code, step, lo):
    hd = code.shape[-1]
    c = torch.nn.functional.pad(code, (0, -hd % 8)).to(torch.int64).unflatten(-1, (-1, 8))
    words = (c << (4 * torch.arange(8, device=c.device))).sum(-1)
    both = ((step.view(torch.int32).to(torch.int64) >> 16) & 0xffff) | (lo.view(torch.int32).to(torch.int64) & -65536)
    return ((words + 2 ** 31) % 2 ** 32 - 2 ** 31).to(torch.int32), both.to(torch.int32)


def _values(codes, steps, hd):
    """Planes of a cache -> the f32 values they stand for."""
    nib = (codes[..., None] >> (4 * torch.arange(8, device=codes.device, dtype=torch.int32))) & 15
    step, lo = (steps << 16).view(torch.float32), (steps & -65536).view(torch.float32)
    return (nib.flatten(-2)[..., :hd].float() * step[..., None]) + lo[..., None]


def _normed(x, gamma):
    if gamma is None:
        return x
    eps = float(np.float32(EPS))
    inv = (1.0 / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()).float()
    return (x * inv) * gamma


def _rotated(x, c, s):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain_append(s):
    case = s["case"]
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    rows = s["qkv"].unflatten(-1, (h + 2 * kv, hd))
    pos = s["positions"].long()
    c, si = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _rotated(_normed(rows[:, :h], s["gq"]), c, si)
    return q, _rotated(_normed(rows[:, h:h + kv], s["gk"]), c, si), rows[:, h + kv:]


def _plain_attn(s):
    case = s["case"]
    hd, t, rep = case["hd"], case["t"], case["heads"] // case["kv"]
    k, v = _values(s["k_codes"], s["k_steps"], hd), _values(s["v_codes"], s["v_steps"], hd)
    b, _, length, _ = k.shape
    q = s["q"].unflatten(2, (case["kv"], rep)).permute(0, 2, 3, 1, 4).reshape(b, case["kv"], rep * t, hd)
    score = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    seen = s["lens"][:, None] - (t - 1) + torch.arange(t, device=q.device)  # positions query i may look at
    mask = torch.arange(length, device=q.device) < seen[:, None, None, :, None]
    mask = mask.expand(b, 1, rep, t, length).reshape(b, 1, rep * t, length)
    score = score.masked_fill(~mask, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    z = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(z == 0, torch.ones_like(z), z)
    return out.unflatten(2, (rep, t)).permute(0, 3, 1, 2, 4).reshape(b, t, case["heads"], hd)


def _plain_sample(s):
    # in 64 bits: which token a number falls on is decided by the last digits of long sums
    l = s["logits"].double()
    t = s["temperature"].double()[:, None]
    srt, order = torch.sort(l, dim=-1, descending=True, stable=True)
    x = (srt - srt[:, :1]) / torch.where(t > 0, t, torch.ones_like(t))
    w = x.exp()
    rank = torch.arange(l.shape[1], device=l.device)
    k = s["top_k"].long()[:, None]
    keep = (rank < torch.where(k > 0, k, l.shape[1])) & (x >= s["min_p"].double()[:, None].log())
    keep &= (t > 0) | (rank == 0)
    w = w * keep
    before = w.cumsum(-1) - w
    keep &= before < s["top_p"].double()[:, None] * w.sum(-1, keepdim=True)
    keep |= rank == 0
    w = torch.zeros_like(w).scatter_(-1, order, w * keep)
    cdf = w.cumsum(-1)
    token = (cdf <= s["u"].double()[:, None] * cdf[:, -1:]).sum(-1)
    p = w.gather(-1, token[:, None])[:, 0] / cdf[:, -1]
    return token, p.log().float()


def _run_plain(s):
    case = s["case"]
    op, hd = case["op"], case["hd"] if "hd" in case else 0
    if op == "attn":
        return _plain_attn(s)
    if op == "sample":
        return _plain_sample(s)
    at = (s["rows"] // case["lmax"], slice(None), s["rows"] % case["lmax"])
    if op in ("append4", "append32"):
        q, k, v = _plain_append(s)
        if op == "append32":
            s["k"][at], s["v"][at] = k, v
            return q, s["k"], s["v"]
        for side, x in (("k", k), ("v", v)):
            s[side + "_codes"][at], s[side + "_steps"][at] = _pack(*_quantise(x))
    read = [_values(s[side + "_codes"][at], s[side + "_steps"][at], hd) for side in ("k", "v")]
    return read if op == "read" else (q, *read)


def _run_own(s):
    from kore_b200 import serving

    case = s["case"]
    op = case["op"]
    if op == "sample":
        return serving.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                              return_logprobs=True)
    if op == "append32":
        q = serving.qknorm_rope_append(s["qkv"], s["positions"], s["rows"], s["cos"], s["sin"], (s["k"], s["v"]), case["heads"],
                                       q_gamma=s["gq"], k_gamma=s["gk"], eps=EPS)
        return q, s["k"], s["v"]
    if "cache" not in s:  # the handle that a program keeps beside its planes
        s["cache"] = serving.KV4Cache.from_planes(s["k_codes"], s["k_steps"], s["v_codes"], s["v_steps"], case["hd"])
    if op == "attn":
        return serving.attend(s["q"], s["cache"], s["lens"])
    if op == "append4":
        q = serving.qknorm_rope_append(s["qkv"], s["positions"], s["rows"], s["cos"], s["sin"], s["cache"], case["heads"],
                                       q_gamma=s["gq"], k_gamma=s["gk"], eps=EPS)
        return (q, *s["cache"].read(s["rows"]))
    return s["cache"].read(s["rows"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "sample":
        n = case["n"] * case["vocab"]
        return {"bytes": 4 * n + 32 * case["n"], "flops": 4 * n}
    hd = case["hd"]
    row = hd / 2 + 4  # codes, step and lo of one head's row
    if op == "attn":
        seen = sum(_lens(case))
        q = case["seqs"] * case["t"] * case["heads"] * hd
        return {"bytes": 2 * seen * case["kv"] * row + 8 * q, "flops": 4 * seen * case["t"] * case["heads"] * hd}
    if op == "read":
        n = case["seqs"] * case["rows"] * case["kv"]
        return {"bytes": 2 * n * (row + 4 * hd), "flops": 4 * n * hd}
    n = case["seqs"] * case["tokens"]
    moved = n * hd * 4 * (2 * case["heads"] + 2 * case["kv"])
    kept = 2 * n * case["kv"] * (4 * hd if op == "append32" else 2 * row + 4 * hd)  # written, or written, read and unpacked
    return {"bytes": moved + kept, "flops": 10 * n * hd * (case["heads"] + 2 * case["kv"])}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _r32(a):
    """one rounding to f32 of numbers held in 64 bits"""
    return a.astype(np.float32).astype(np.float64)


def _np_bf16(a, up):
    """nearest bfloat16 number not below (up) or not above a; a holds f32 numbers"""
    m, e = np.frexp(a)
    unit = np.ldexp(1.0, np.maximum(e, -125) - 8)
    return (np.ceil if up else np.floor)(a / unit) * unit


def _np_stored(x):
    lo = _np_bf16(x.min(-1), False)[..., None]
    step = _np_bf16(np.maximum(_r32(_r32(x.max(-1)[..., None] - lo) / 15.0), 2.0 ** -100), True)
    code = np.clip(np.rint(_r32(_r32(x - lo) * _r32(1.0 / step))), 0, 15)
    return _r32(lo + code * step)


def _unpacked(codes, steps, hd):
    """values of cache planes, in 64 bits: whole-number arithmetic on the words"""
    w, s = codes.long() % 2 ** 32, steps.long() % 2 ** 32
    nib = torch.stack([w // 16 ** i % 16 for i in range(8)], -1).reshape(*w.shape[:-1], -1)[..., :hd]
    step = (s % 65536).to(torch.int16).view(torch.bfloat16).double()
    lo = (s // 65536).to(torch.int16).view(torch.bfloat16).double()
    return nib.double() * step[..., None] + lo[..., None]


def _exact_append(case, s):
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    half = hd // 2
    x = s["qkv"].double().cpu().numpy().reshape(-1, h + 2 * kv, hd)
    cos, sin = (s[n].double().cpu().numpy()[s["positions"].cpu().numpy()][:, None] for n in ("cos", "sin"))

    def turned(y, gamma):
        if gamma is not None:  # the append's f32 roundings are part of its definition: they decide codes
            inv = _r32(1.0 / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(EPS))))
            y = _r32(_r32(y * inv) * gamma.double().cpu().numpy())
        a, b = y[..., :half], y[..., half:]
        return np.concatenate([_r32(_r32(a * cos) - _r32(b * sin)), _r32(_r32(a * sin) + _r32(b * cos))], -1)

    return turned(x[:, :h], s["gq"]), turned(x[:, h:h + kv], s["gk"]), x[:, h + kv:]


def _exact_attn(case, s):
    t, hd, rep = case["t"], case["hd"], case["heads"] // case["kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        for g in range(case["kv"]):
            k, v = (_unpacked(s[x + "_codes"][b, g, :n], s[x + "_steps"][b, g, :n], hd) for x in ("k", "v"))
            for i in range(t):
                m = n - (t - 1 - i)
                if m > 0:
                    a = torch.softmax(s["q"][b, i, g * rep:(g + 1) * rep].double() @ k[:m].T / math.sqrt(hd), -1)
                    out[b, i, g * rep:(g + 1) * rep] = a @ v[:m]
    return out


def _exact_sample(case, s):
    l, t, k, p, m, u = (s[n].double().cpu().numpy() for n in ("logits", "temperature", "top_k", "top_p", "min_p", "u"))
    tokens, logs = [], []
    for r in range(case["n"]):
        order = np.argsort(-l[r], kind="stable")
        if t[r] <= 0:
            tokens.append(int(order[0]))
            logs.append(0.0)
            continue
        x = (l[r][order] - l[r].max()) / t[r]
        n = min(int(k[r]) or len(x), len(x))
        if m[r] > 0:
            n = min(n, max(1, int(np.count_nonzero(x >= math.log(m[r])))))
        w = np.exp(x[:n])
        total = np.cumsum(w)
        n = 1 + int(np.searchsorted(total[:-1], p[r] * total[-1], side="left"))
        kept = np.sort(order[:n])
        z = np.cumsum(np.exp((l[r][kept] - l[r].max()) / t[r]))
        i = min(int(np.searchsorted(z, u[r] * z[-1], side="right")), n - 1)
        tokens.append(int(kept[i]))
        logs.append((l[r][kept[i]] - l[r].max()) / t[r] - math.log(z[-1]))
    return np.array(tokens), np.array(logs)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "attn":
        return _exact_attn(case, s)
    if op == "sample":
        return _exact_sample(case, s)
    lmax = case["lmax"]
    if op == "read":
        at = (s["rows"] // lmax, slice(None), s["rows"] % lmax)
        return [_unpacked(s[x + "_codes"][at], s[x + "_steps"][at], case["hd"]) for x in ("k", "v")]
    q, k, v = _exact_append(case, s)
    if op == "append4":
        return q, _np_stored(k), _np_stored(v)
    rows = s["rows"].cpu().numpy()
    out = [s[x].double().cpu().numpy() for x in ("k", "v")]
    for cache, x in zip(out, (k, v)):
        cache[rows // lmax, :, rows % lmax] = x
    return q, *out
