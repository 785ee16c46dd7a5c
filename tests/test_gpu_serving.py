"""Serving-step kernels against the 64-bit restatement: append, read-back and attention of the 4-bit KV cache, sampling,
and the decoder that runs them together."""
import numpy as np
import pytest

from oracle import decoder_ref as dr
from oracle import serving_ref as sr
from tests import cases

pytestmark = pytest.mark.gpu
f32 = np.float32


@pytest.fixture(scope="module")
def env():
    import torch

    from kore_b200 import KoreError, decoder, serving

    assert torch.cuda.is_available()
    dev = lambda a: torch.from_numpy(np.array(a)).cuda()
    return type("E", (), {"torch": torch, "serving": serving, "decoder": decoder, "KoreError": KoreError, "dev": staticmethod(dev)})


def tables(max_pos, hd):
    ang = np.arange(max_pos)[:, None] * 10000.0 ** (-np.arange(hd // 2) / (hd // 2))
    return np.cos(ang).astype(f32), np.sin(ang).astype(f32)


def planes_of(cache):
    return [t.cpu().numpy().view(np.uint32) for t in (cache.k_codes, cache.k_steps, cache.v_codes, cache.v_steps)]


def filled_cache(env, seqs, kv, lmax, hd, seed, scale=1.0):
    """A cache of quantised Gaussian rows, and its planes"""
    c = env.serving.KV4Cache(seqs, kv, lmax, hd)
    for side, s in (("k", 0), ("v", 1)):
        words, steps = sr.quantise(cases.gaussian(seed + s, (seqs, kv, c.max_len, hd), scale))
        getattr(c, side + "_codes").copy_(env.dev(words.view(np.int32)))
        getattr(c, side + "_steps").copy_(env.dev(steps.view(np.int32)))
    return c


# ---- append ------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,heads,kv,hd,norm", [(1, 32, 32, 100, False), (5, 8, 2, 128, True), (33, 6, 3, 4, True), (3, 4, 1, 36, False),
                                                (7, 4, 4, 124, True), (64, 2, 1, 64, True), (2, 5, 5, 8, False)])
def test_append_to_4_bits_is_exact(env, n, heads, kv, hd, norm):
    """codes, pairs and queries equal the restatement bit for bit; rows that no token names stay as they were"""
    rng = np.random.default_rng(n + hd)
    seqs, lmax = 3, 40
    qkv = (cases.gaussian(n * hd, (n, (heads + 2 * kv) * hd), 1.0) * np.exp(rng.uniform(-3, 3, (n, 1)))).astype(f32)
    gq, gk = ((1 + cases.gaussian(i, (hd,), 0.2)).astype(f32) if norm else None for i in (5, 6))
    cos, sin = tables(lmax, hd)
    rows = rng.choice(seqs * lmax, n, replace=False).astype(np.int64)
    pos = (rows % lmax).astype(np.int32)
    cache = filled_cache(env, seqs, kv, lmax, hd, 77)
    want = planes_of(cache)
    q = env.serving.qknorm_rope_append(env.dev(qkv), env.dev(pos), env.dev(rows), env.dev(cos), env.dev(sin), cache, heads,
                                       q_gamma=None if gq is None else env.dev(gq), k_gamma=None if gk is None else env.dev(gk), eps=1e-6)
    rq, rk, rv = sr.append(qkv, pos, cos, sin, heads, kv, hd, gq, gk, 1e-6)
    for at, x in ((0, rk), (2, rv)):
        want[at][rows // lmax, :, rows % lmax], want[at + 1][rows // lmax, :, rows % lmax] = sr.quantise(x)
    assert (q.cpu().numpy() == rq).all()
    for got, ref in zip(planes_of(cache), want):
        assert (got == ref).all()


@pytest.mark.parametrize("n,heads,kv,hd,norm", [(16, 32, 32, 100, True), (9, 4, 2, 30, True), (3, 3, 1, 2, False), (4, 8, 8, 128, False), (5, 2, 2, 6, True)])
def test_append_to_f32(env, n, heads, kv, hd, norm):
    rng = np.random.default_rng(hd)
    seqs, lmax = 2, 21
    qkv = cases.gaussian(n, (n, (heads + 2 * kv) * hd), 1.5)
    gq, gk = ((1 + cases.gaussian(i, (hd,), 0.2)).astype(f32) if norm else None for i in (5, 6))
    cos, sin = tables(lmax, hd)
    rows = rng.choice(seqs * lmax, n, replace=False).astype(np.int64)
    pos = (rows % lmax).astype(np.int32)
    k, v = (cases.gaussian(8 + i, (seqs, kv, lmax, hd), 1.0) for i in (0, 1))
    kd, vd = env.dev(k), env.dev(v)
    q = env.serving.qknorm_rope_append(env.dev(qkv), env.dev(pos), env.dev(rows), env.dev(cos), env.dev(sin), (kd, vd), heads,
                                       q_gamma=None if gq is None else env.dev(gq), k_gamma=None if gk is None else env.dev(gk))
    rq, rk, rv = sr.append(qkv, pos, cos, sin, heads, kv, hd, gq, gk)
    k[rows // lmax, :, rows % lmax], v[rows // lmax, :, rows % lmax] = rk, rv
    assert (q.cpu().numpy() == rq).all() and (kd.cpu().numpy() == k).all() and (vd.cpu().numpy() == v).all()


@pytest.mark.parametrize("heads,kv,hd,norm,odd", [(8, 2, 128, True, 0), (8, 2, 128, False, 0), (8, 2, 128, True, 1), (6, 3, 100, True, 0), (5, 1, 36, True, 0),
                                                  (3, 3, 4, False, 0), (4, 4, 124, True, 1)])
def test_append_of_many_tokens(env, heads, kv, hd, norm, odd):
    """groups of four heads (queries, keys and values in one group, and a last one that is not full), both caches, odd addresses"""
    n = 3000 // (heads + 2 * kv) + 5
    rng = np.random.default_rng(hd + heads)
    seqs, lmax = 4, (n + 3) // 4 * 4
    qkv = (cases.gaussian(hd, (n, (heads + 2 * kv) * hd), 1.0) * np.exp(rng.uniform(-3, 3, (n, 1)))).astype(f32)
    gq, gk = ((1 + cases.gaussian(i, (hd,), 0.2)).astype(f32) if norm else None for i in (5, 6))
    cos, sin = tables(lmax, hd)
    rows = rng.choice(seqs * lmax, n, replace=False).astype(np.int64)
    pos = (rows % lmax).astype(np.int32)
    src = env.torch.zeros((n, qkv.shape[1] + odd), device="cuda")[:, odd:]
    src.copy_(env.dev(qkv))
    rq, rk, rv = sr.append(qkv, pos, cos, sin, heads, kv, hd, gq, gk, 1e-6)
    cache = filled_cache(env, seqs, kv, lmax, hd, 78)
    want = planes_of(cache)
    pair = [cases.gaussian(8 + i, (seqs, kv, lmax, hd), 1.0) for i in (0, 1)]
    dev_pair = tuple(env.dev(x) for x in pair)
    for to in (cache, dev_pair):
        q = env.serving.qknorm_rope_append(src, env.dev(pos), env.dev(rows), env.dev(cos), env.dev(sin), to, heads,
                                           q_gamma=None if gq is None else env.dev(gq), k_gamma=None if gk is None else env.dev(gk), eps=1e-6)
        assert (q.cpu().numpy() == rq).all()
    for at, x in ((0, rk), (2, rv)):
        want[at][rows // lmax, :, rows % lmax], want[at + 1][rows // lmax, :, rows % lmax] = sr.quantise(x)
        pair[at // 2][rows // lmax, :, rows % lmax] = x
    for got, ref in zip(planes_of(cache), want):
        assert (got == ref).all()
    assert all((got.cpu().numpy() == ref).all() for got, ref in zip(dev_pair, pair))


def test_append_without_norm_is_the_rotation_of_kb_rope_kv(env):
    """on the f32 cache the operator without gammas gives the numbers of the framework's own append"""
    from kore_b200 import _cabi

    t, n, H, hd, lmax = env.torch, 6, 4, 100, 8
    cos, sin = tables(lmax, hd)
    qkv, pos = env.dev(cases.gaussian(3, (n, 3 * H * hd), 1.0)), t.arange(n, dtype=t.int32, device="cuda")
    rows = t.arange(n, dtype=t.int64, device="cuda")
    outs = []
    for own in (True, False):
        k, v, q = (t.zeros(s, device="cuda") for s in ((1, H, lmax, hd), (1, H, lmax, hd), (n, H, hd)))
        if own:
            env.serving.qknorm_rope_append(qkv, pos, rows, env.dev(cos), env.dev(sin), (k, v), H, q_out=q)
        else:
            c, s = env.dev(cos), env.dev(sin)
            _cabi.check(_cabi.lib().kb_rope_kv(qkv.data_ptr(), pos.data_ptr(), rows.data_ptr(), c.data_ptr(), s.data_ptr(), n, H, hd, lmax,
                                               q.data_ptr(), k.data_ptr(), v.data_ptr(), t.cuda.current_stream().cuda_stream))
            t.cuda.synchronize()
        outs.append([x.cpu() for x in (q, k, v)])
    assert all((a == b).all() for a, b in zip(*outs))


@pytest.mark.parametrize("four", [True, False])
def test_append_padding_strides_and_bad_rows(env, four):
    """padded tokens, rows and positions out of range append nothing; strided and odd-aligned rows give the same numbers"""
    t, heads, kv, hd, seqs, lmax = env.torch, 4, 2, 20, 2, 8
    n, width = 7, (4 + 2 * 2) * 20
    cos, sin = tables(lmax, hd)
    qkv = cases.gaussian(1, (n, width), 1.0)
    pos = np.array([0, 1, 2, 3, lmax, -1, 4], np.int32)
    rows = np.array([0, -1, seqs * lmax, 9, 2, 3, 1 << 40], np.int64)
    wide = t.zeros((n, width + 5), device="cuda")
    wide[:, 3:3 + width] = env.dev(qkv)
    for src in (env.dev(qkv), wide[:, 3:3 + width]):
        if four:
            cache = env.serving.KV4Cache(seqs, kv, lmax, hd)
        else:
            cache = tuple(t.zeros((seqs, kv, lmax, hd), device="cuda") for _ in range(2))
        q = env.serving.qknorm_rope_append(src, env.dev(pos), env.dev(rows), env.dev(cos), env.dev(sin), cache, heads).cpu().numpy()
        good = [0, 1, 2, 3, 6]
        rq, rk, rv = sr.append(qkv[good], pos[good], cos, sin, heads, kv, hd)
        assert (q[good] == rq).all() and np.isnan(q[[4, 5]]).all()
        k = cache.read(t.arange(seqs * lmax, device="cuda"))[0].view(seqs, lmax, kv, hd).transpose(1, 2) if four else cache[0]
        k = k.cpu().numpy()
        want = np.zeros((seqs, kv, lmax, hd), f32)
        for i, row in ((0, 0), (3, 9)):
            want[row // lmax, :, row % lmax] = sr.values(*sr.quantise(rk[good.index(i)]), hd) if four else rk[good.index(i)]
        assert (k == want).all()


def test_append_special_values(env):
    """rows with infinities, NaN or an overflowing range read back as NaN; constant, zero and subnormal rows stay what they are"""
    t, hd = env.torch, 8
    v = np.zeros((6, hd), f32)
    v[1], v[2, 3], v[3, 7], v[4, 0], v[4, 1], v[5] = 3.0, np.nan, np.inf, -3e38, 3e38, 1e-42
    qkv = np.zeros((6, 3 * hd), f32)
    qkv[:, 2 * hd:] = v
    qkv[2, 0] = np.nan  # a query: passed through
    cos, sin = tables(8, hd)
    cache = env.serving.KV4Cache(1, 1, 8, hd)
    idx = np.arange(6)
    q = env.serving.qknorm_rope_append(env.dev(qkv), env.dev(idx.astype(np.int32)), env.dev(idx), env.dev(cos), env.dev(sin), cache, 1)
    assert np.isnan(q.cpu().numpy()[2, 0]).any() and np.isfinite(q.cpu().numpy()[[0, 1, 3, 4, 5]]).all()
    words, steps = sr.quantise(v)
    got = planes_of(cache)
    assert (got[2][0, 0, :6] == words).all() and (got[3][0, 0, :6] == steps).all()
    read = cache.read(env.dev(idx))[1].cpu().numpy()[:, 0]
    assert np.isnan(read[2:5]).all() and (read[1] == 3.0).all() and (read[0] == 0).all()


# ---- read-back ---------------------------------------------------------------------------------
@pytest.mark.parametrize("seqs,kv,lmax,hd,n", [(2, 32, 64, 100, 50), (1, 1, 4, 4, 1), (3, 5, 36, 128, 1000), (2, 3, 8, 12, 9)])
def test_read_back(env, seqs, kv, lmax, hd, n):
    cache = filled_cache(env, seqs, kv, lmax, hd, 5)
    rows = np.random.default_rng(n).integers(-2, seqs * lmax + 2, n)  # the same row twice, and rows outside, are allowed
    kc, ks, vc, vs = planes_of(cache)
    ok = (rows >= 0) & (rows < seqs * lmax)
    at = (np.where(ok, rows, 0) // lmax, slice(None), np.where(ok, rows, 0) % lmax)
    for got, (w, s) in zip(cache.read(env.dev(rows)), ((kc, ks), (vc, vs))):
        want = np.where(ok[:, None, None], sr.values(w[at], s[at], hd), f32(0))
        assert (got.cpu().numpy() == want).all()


# ---- attention ---------------------------------------------------------------------------------
def check_attention(env, q, cache, lens, scale=0.0):
    """|error| <= (2 e + 2^-16) max|v|.  e bounds a score's error: products and sums of queries held to 22 bits and f32 accumulators
    that lose at most 2^-22 of the running sum at each of up to 16 steps, 2^-18 in all of scale * sum|q_d| (|lo| + 15 step); a
    softmax weight then moves by 2 e at most.  2^-16 covers weights held to 22 bits, their f32 sums (up to 64 steps of 2^-22 of the
    total) and the merge of partial results; an output is a mean of values, so all of it is relative to the largest."""
    planes = planes_of(cache)
    ref = sr.attention(q, *planes, lens, scale)
    got = env.serving.attend(env.dev(q), cache, env.dev(np.asarray(lens, np.int32)), scale=scale).cpu().numpy()
    heads, hd = q.shape[2], q.shape[3]
    rep = heads // cache.n_kv_heads
    for b, n in enumerate(np.clip(lens, 0, cache.max_len)):
        for h in range(heads):
            step, lo = (a.astype(np.float64)[:n] for a in sr.pair_of(planes[1][b, h // rep]))
            vstep, vlo = (a.astype(np.float64)[:n] for a in sr.pair_of(planes[3][b, h // rep]))
            if n == 0:
                assert (got[b, :, h] == 0).all()
                continue
            s = abs(scale) or 1 / np.sqrt(hd)
            e = 2.0 ** -18 * s * np.abs(q[b, :, h].astype(np.float64)).sum(-1) * (np.abs(lo) + 15 * step).max()
            tol = (2 * e + 2.0 ** -16) * (np.abs(vlo) + 15 * vstep).max()
            assert (np.abs(got[b, :, h] - ref[b, :, h]).max(-1) <= tol).all(), (b, h)
    return got


@pytest.mark.parametrize("seqs,t,heads,kv,hd,lmax,lens", [
    (1, 1, 32, 32, 100, 640, [577]), (3, 1, 8, 8, 100, 640, [1, 640, 33]), (4, 1, 8, 2, 128, 300, [0, 1, 2, 299]),
    (2, 5, 8, 2, 128, 300, [3, 297]), (2, 3, 7, 1, 64, 1000, [999, 64]), (1, 2, 4, 4, 4, 8, [8]), (2, 1, 16, 2, 36, 132, [131, 128]),
    (1, 1, 1, 1, 128, 5000, [4999]), (2, 17, 6, 3, 96, 200, [20, 199]), (1, 1, 64, 1, 104, 260, [257]), (2, 40, 2, 2, 8, 64, [64, 12]),
    (1, 1, 2, 1, 120, 36, [35]), (5, 4, 3, 3, 32, 16, [16, 0, 3, 4, 9]), (1, 1, 10, 2, 68, 1500, [1485])])
def test_attention(env, seqs, t, heads, kv, hd, lmax, lens):
    q = cases.gaussian(hd + t, (seqs, t, heads, hd), 1.0)
    check_attention(env, q, filled_cache(env, seqs, kv, lmax, hd, 11), lens)


@pytest.mark.parametrize("seqs,t,heads,kv,hd,lmax,longest", [(40, 1, 4, 2, 8, 1500, 1500), (50, 1, 16, 16, 8, 2000, 2000), (33, 4, 6, 2, 16, 800, 790),
                                                             (3, 2, 4, 4, 64, 20000, 20000)])
def test_attention_splits_of_many_unlike_sequences(env, seqs, t, heads, kv, hd, lmax, longest):
    """chunks are dealt over more sequences than a warp has lanes, over more units than the GPU holds CTAs, over one long among short"""
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, 60, seqs)
    lens[rng.choice(seqs, max(1, seqs // 8), replace=False)] = rng.integers(longest // 2, longest, max(1, seqs // 8))
    lens[seqs // 2] = longest
    q = cases.gaussian(seqs + t, (seqs, t, heads, hd), 1.0)
    check_attention(env, q, filled_cache(env, seqs, kv, lmax, hd, 15), list(lens))


def test_attention_scale_lens_and_squeezed_queries(env):
    """scale is used, lens beyond the cache or below zero are clamped, [seqs, heads, hd] is one token, strided queries"""
    t = env.torch
    cache = filled_cache(env, 3, 2, 40, 64, 12)
    q = cases.gaussian(4, (3, 1, 4, 64), 1.0)
    a = check_attention(env, q, cache, [100, -5, 7], scale=0.3)
    lens = env.dev(np.array([100, -5, 7], np.int32))
    b = env.serving.attend(env.dev(q[:, 0]), cache, lens, scale=0.3).cpu().numpy()
    wide = t.zeros((3, 1, 4, 70), device="cuda")
    wide[..., 2:66] = env.dev(q)
    c = env.serving.attend(wide[..., 2:66], cache, lens, scale=0.3).cpu().numpy()
    assert (a[:, 0] == b).all() and (a == c).all() and (a[1] == 0).all()


@pytest.mark.parametrize("t,heads", [(1, 4), (3, 8)])
def test_attention_ignores_what_it_does_not_see(env, t, heads):
    """NaN pairs and arbitrary codes at and behind a sequence's end change no bit; a NaN row that is seen shows"""
    cache = filled_cache(env, 2, 2, 200, 100, 13)
    q = cases.gaussian(4, (2, t, heads, 100), 1.0)
    lens = [70, 133]
    a = check_attention(env, q, cache, lens)
    for b, n in enumerate(lens):
        for x in (cache.k_codes, cache.v_codes):
            x[b, :, n:] = -1
        for x in (cache.k_steps, cache.v_steps):
            x[b, :, n:] = 0x7fc07fc0
    assert (check_attention(env, q, cache, lens) == a).all()
    cache.v_steps[0, 0, 5] = 0x7fc07fc0
    got = env.serving.attend(env.dev(q), cache, env.dev(np.array(lens, np.int32))).cpu().numpy()
    assert np.isnan(got[0, :, :heads // 2]).all() and (got[0, :, heads // 2:] == a[0, :, heads // 2:]).all() and (got[1] == a[1]).all()


def test_attention_values_of_unequal_size(env):
    """value rows from 2^-60 to 2^40, the largest weights on the smallest rows: each head keeps its own relative accuracy"""
    hd, n = 64, 500
    cache = env.serving.KV4Cache(1, 1, n, hd)
    rng = np.random.default_rng(3)
    k = rng.standard_normal((1, 1, n, hd)).astype(f32)
    for exps in (np.full(n, -60.0), np.full(n, 40.0), np.where(np.arange(n) < 250, -30.0, -33.0)):
        v = (rng.standard_normal((1, 1, n, hd)) * np.exp2(exps)[:, None]).astype(f32)
        for side, x in (("k", k), ("v", v)):
            w, s = sr.quantise(x)
            getattr(cache, side + "_codes").copy_(env.dev(w.view(np.int32)))
            getattr(cache, side + "_steps").copy_(env.dev(s.view(np.int32)))
        check_attention(env, cases.gaussian(9, (1, 1, 2, hd), 1.0), cache, [n])
    # one position carries nearly all the weight and its values are 2^-36 of the others': the result is that row to f32 accuracy
    q = np.zeros((1, 1, 1, hd), f32)
    q[0, 0, 0, 0] = 100.0 * 8
    k[0, 0, :, 0] = 0.0
    k[0, 0, 7, 0] = 1.0
    v = rng.standard_normal((1, 1, n, hd)).astype(f32)
    v[0, 0, 7] *= f32(2.0 ** -36)
    for side, x in (("k", k), ("v", v)):
        w, s = sr.quantise(x)
        getattr(cache, side + "_codes").copy_(env.dev(w.view(np.int32)))
        getattr(cache, side + "_steps").copy_(env.dev(s.view(np.int32)))
    got = env.serving.attend(env.dev(q), cache, env.dev(np.array([n], np.int32))).cpu().numpy()[0, 0, 0]
    ref = sr.attention(q, *planes_of(cache), [n])[0, 0, 0]
    # weights to 22 bits, sums of at most 500 terms: 2^-16 of the row's largest value
    assert np.abs(got - ref).max() <= 2.0 ** -16 * np.abs(ref).max()


def test_attention_repeats_bit_for_bit_on_streams_and_in_graphs(env):
    """two streams at once, a captured call replayed, two graphs replayed side by side: always the eager bits"""
    t = env.torch
    cache = filled_cache(env, 2, 2, 3000, 128, 14)
    q = env.dev(cases.gaussian(6, (2, 1, 8, 128), 1.0))
    lens = env.dev(np.array([2999, 1234], np.int32))
    ref = env.serving.attend(q, cache, lens)
    t.cuda.synchronize()
    outs, streams, graphs = [], [t.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with t.cuda.stream(s):
            outs += [env.serving.attend(q, cache, lens) for _ in range(5)]
    t.cuda.synchronize()
    for s in streams:
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g, stream=s):
            outs.append(env.serving.attend(q, cache, lens))
        graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with t.cuda.stream(s):
                g.replay()
    t.cuda.synchronize()
    assert all((o == ref).all() for o in outs)


def test_attention_workspaces_and_places_of_a_c_caller(env):
    """no workspace (eager and captured), one too small, queries and results at odd addresses, results over the queries"""
    from kore_b200 import _cabi

    t, lib = env.torch, _cabi.lib()
    seqs, heads, kv, hd, lmax = 3, 8, 2, 100, 4000
    cache = filled_cache(env, seqs, kv, lmax, hd, 16)
    q = env.dev(cases.gaussian(7, (seqs, 1, heads, hd), 1.0))
    lens = env.dev(np.array([4000, 17, 2600], np.int32))
    ref = env.serving.attend(q, cache, lens)
    need = int(lib.kb_attn_kv4_workspace_bytes(seqs, 1, heads, kv, hd, lmax))
    assert need > 0
    planes = [x.data_ptr() for x in (cache.k_codes, cache.k_steps, cache.v_codes, cache.v_steps)]
    ws = t.empty(need, dtype=t.uint8, device="cuda")

    def call(src, dst, space, size):
        return lib.kb_attn_kv4(src.data_ptr(), *planes, lens.data_ptr(), seqs, 1, heads, kv, hd, lmax, 0.0, dst.data_ptr(), space, size,
                               t.cuda.current_stream().cuda_stream)
    out = t.zeros_like(q)
    assert call(q, out, None, 0) == 0
    t.cuda.synchronize()
    assert (out == ref).all()
    out.zero_()
    assert call(q, out, ws.data_ptr(), need - 1) == _cabi.ERR_STORAGE
    t.cuda.synchronize()
    assert (out == 0).all()
    src, dst = (t.zeros(q.numel() + 3, device="cuda")[o:o + q.numel()] for o in (1, 3))
    src.copy_(q.view(-1))
    assert call(src, dst, ws.data_ptr(), need) == 0
    t.cuda.synchronize()
    assert (dst.view_as(ref) == ref).all()
    assert env.serving.attend(src.view_as(q), cache, lens, out=src.view_as(q)).data_ptr() == src.data_ptr()
    assert (src.view_as(ref) == ref).all()
    out.zero_()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g):
        assert call(q, out, None, 0) == 0
    for _ in range(3):
        g.replay()
    t.cuda.synchronize()
    assert (out == ref).all()


def test_attention_of_more_units_than_are_split(env):
    """1300 sequences of 8 KV heads: a CTA takes a unit whole, however long"""
    rng = np.random.default_rng(8)
    lens = rng.integers(0, 9, 1300)
    lens[[0, 700, 1299]] = 700, 671, 1
    check_attention(env, cases.gaussian(10, (1300, 1, 8, 4), 1.0), filled_cache(env, 1300, 8, 700, 4, 17), list(lens))


def test_a_cache_of_more_than_2_31_words(env):
    """the last rows of one sequence of 2^27 + 64 positions: appended, read back, attended to"""
    t, hd, lmax = env.torch, 128, (1 << 27) + 64
    if t.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 20 GB")
    cache = env.serving.KV4Cache(1, 1, lmax, hd)
    rows = np.array([0, (1 << 27) - 1, 1 << 27, lmax - 1], np.int64)
    x = cases.gaussian(18, (4, 3 * hd), 1.0)
    x[3, hd:2 * hd] = 4.0  # the last key
    one, zero = np.ones((1, hd // 2), f32), np.zeros((1, hd // 2), f32)
    q = env.serving.qknorm_rope_append(env.dev(x), t.zeros(4, dtype=t.int32, device="cuda"), env.dev(rows), env.dev(one), env.dev(zero), cache, 1)
    assert (q.cpu().numpy()[:, 0] == x[:, :hd]).all()
    k, v = (a.cpu().numpy()[:, 0] for a in cache.read(env.dev(rows)))
    for got, at in ((k, hd), (v, 2 * hd)):
        assert (got == sr.values(*sr.quantise(x[:, at:at + hd]), hd)).all()
    ask = np.full((1, 1, 1, hd), 0.5, f32)  # 256 times the scale with the last key: 22.6; 0 with the empty rows
    got = env.serving.attend(env.dev(ask), cache, env.dev(np.array([lmax], np.int32))).cpu().numpy()[0, 0, 0]
    w = np.exp(k.astype(np.float64) @ ask[0, 0, 0].astype(np.float64) / np.sqrt(hd))
    ref = (w @ v.astype(np.float64)) / (w.sum() + lmax - 4)
    # a weight of e^22.6 next to 2^27 of 1: scores to 2^-18 of 22.6, sums as in check_attention
    assert np.abs(got - ref).max() <= (2.0 ** -18 * 22.7 + 2.0 ** -16) * np.abs(v).max()
    del cache
    t.cuda.empty_cache()


# ---- the cache object --------------------------------------------------------------------------
def test_planes_stay_and_copies_are_their_own(env):
    """planes are written, not replaced; a deep copy has its own memory"""
    import copy

    t = env.torch
    cache = filled_cache(env, 2, 2, 8, 16, 19)
    with pytest.raises(AttributeError):
        cache.k_codes = t.zeros_like(cache.k_codes)
    other, before = copy.deepcopy(cache), planes_of(cache)
    x = env.dev(cases.gaussian(20, (1, 6 * 16), 1.0))
    i = lambda v, dt: t.full((1,), v, dtype=dt, device="cuda")
    cos, sin = tables(4, 16)
    env.serving.qknorm_rope_append(x, i(3, t.int32), i(3, t.int64), env.dev(cos), env.dev(sin), other, 2)
    assert all((a == b).all() for a, b in zip(planes_of(cache), before))
    assert any((a != b).any() for a, b in zip(planes_of(other), before))
    view = env.serving.KV4Cache.from_planes(cache.k_codes, cache.k_steps, cache.v_codes, cache.v_steps, 16)
    env.serving.qknorm_rope_append(x, i(3, t.int32), i(3, t.int64), env.dev(cos), env.dev(sin), view, 2)
    assert all((a == b).all() for a, b in zip(planes_of(cache), planes_of(other)))


def test_append_in_graphs_with_positions_moved_in_place(env):
    """what a decode step does: one captured append, replayed as the positions and rows advance"""
    t, heads, kv, hd, lmax = env.torch, 4, 2, 64, 16
    cos, sin = (env.dev(a) for a in tables(lmax, hd))
    xs = env.dev(cases.gaussian(21, (6, 3, (heads + 2 * kv) * hd), 1.0))
    eager, replayed = (env.serving.KV4Cache(3, kv, lmax, hd) for _ in range(2))
    pos, rows = t.zeros(3, dtype=t.int32, device="cuda"), t.arange(3, device="cuda") * lmax
    x, q = t.zeros_like(xs[0]), t.zeros((3, heads, hd), device="cuda")
    g = t.cuda.CUDAGraph()
    t.cuda.synchronize()
    with t.cuda.graph(g):
        env.serving.qknorm_rope_append(x, pos, rows, cos, sin, replayed, heads, q_out=q)
        pos.add_(1)
        rows.add_(1)
    for i in range(6):
        x.copy_(xs[i])
        g.replay()
        ref = env.serving.qknorm_rope_append(xs[i], t.full((3,), i, dtype=t.int32, device="cuda"), t.arange(3, device="cuda") * lmax + i, cos, sin,
                                             eager, heads)
        assert (q == ref).all()
    assert all((a == b).all() for a, b in zip(planes_of(eager), planes_of(replayed)))


# ---- sampling ----------------------------------------------------------------------------------
def check_sample(env, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    n = len(logits)
    put = lambda a, dt: None if a is None else env.dev(np.broadcast_to(np.asarray(a, dt), (n,)))
    tokens, logs = env.serving.sample(env.dev(logits) if isinstance(logits, np.ndarray) else logits, env.dev(np.asarray(u, f32)),
                                      temperature=put(temperature, f32), top_k=put(top_k, np.int32), top_p=put(top_p, f32),
                                      min_p=put(min_p, f32), return_logprobs=True)
    tokens, logs = tokens.cpu().numpy(), logs.cpu().numpy()
    host = logits if isinstance(logits, np.ndarray) else logits.cpu().numpy()
    at = lambda a, i, default: default if a is None else float(f32(np.broadcast_to(a, (n,))[i]))
    for i in range(n):
        tok, lp, margin = sr.sample_row(host[i], f32(u[i]), at(temperature, i, 1.0), int(at(top_k, i, 0)), at(top_p, i, 1.0), at(min_p, i, 0.0))
        # a weight is off by 2^-45 of the largest, a border by at most vocab of them (and 2^-50 for sums in f64)
        if margin > host.shape[1] * 2.0 ** -44:
            assert tokens[i] == tok, (i, tokens[i], tok, margin)
            # one f32 rounding of a logarithm whose share is off by vocab 2^-44
            assert np.isnan(lp) and np.isnan(logs[i]) or abs(logs[i] - lp) <= 2.0 ** -24 * abs(lp) + 1e-6
    return tokens


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1025, 32000, 50021])
def test_sample_settings(env, vocab):
    rng = np.random.default_rng(vocab)
    n = 24
    logits = (rng.standard_normal((n, vocab)) * 3).astype(f32)
    u = rng.random(n).astype(f32)
    check_sample(env, logits, u)
    check_sample(env, logits, u, temperature=rng.uniform(0.2, 2.5, n).astype(f32), top_k=rng.integers(0, 60, n))
    check_sample(env, logits, u, top_p=rng.uniform(0.05, 1.0, n).astype(f32))
    check_sample(env, logits, u, min_p=rng.uniform(0.0, 0.3, n).astype(f32), temperature=0.7)
    check_sample(env, logits, u, temperature=rng.uniform(0.2, 2.5, n).astype(f32), top_k=rng.integers(1, vocab + 2, n),
                 top_p=rng.uniform(0.3, 1.0, n).astype(f32), min_p=rng.uniform(0.0, 0.05, n).astype(f32))


def test_sample_ties_and_flat_rows(env):
    """equal logits go by index in every filter, across any number of them"""
    n, v = 8, 4096
    flat = np.zeros((n, v), f32)
    flat[1::2] = -0.0
    u = ((np.arange(n) + 0.5) / n).astype(f32)
    assert (check_sample(env, flat, u, top_k=100) < 100).all()
    assert (check_sample(env, flat, u, top_p=0.25) < v // 4).all()
    assert (check_sample(env, flat, u, top_p=0.5, top_k=10) < 5).all()
    two = np.where(np.arange(v) % 3 == 0, 2.0, 1.0).astype(f32)[None].repeat(n, 0)
    assert (check_sample(env, two, u, top_k=1500, top_p=0.9) >= 0).all()
    steps = np.round(cases.gaussian(3, (n, v), 2.0))  # a few dozen different logits
    check_sample(env, steps, u, top_k=[1, 2, 3, 5, 50, 500, 1000, 4000])
    check_sample(env, steps, u, top_p=[0.01, 0.1, 0.3, 0.5, 0.7, 0.9, 0.99, 0.999])


@pytest.mark.parametrize("vocab,spread", [(60000, 0.05), (131072, 1.0), (40000, 0.0), (9000, 0.2), (200003, 4.0)])
def test_sample_many_candidates(env, vocab, spread):
    """borders inside bins of hundreds to tens of thousands of elements, of unlike and of equal logits"""
    n = 6
    logits = cases.gaussian(vocab, (n, vocab), spread)
    u = ((np.arange(n) + 0.37) / n).astype(f32)
    check_sample(env, logits, u, top_p=[0.1, 0.5, 0.9, 0.99, 0.99999, 0.3])
    check_sample(env, logits, u, top_k=[300, 2999, 127, 129, vocab - 1, 20000 if vocab > 20000 else 5000])
    check_sample(env, logits, u, top_k=5000, top_p=0.7, temperature=1.7)
    check_sample(env, logits, u, temperature=[0.05, 0.3, 1.0, 3.0, 30.0, 1000.0], top_p=0.95, min_p=0.001)


def test_sample_special_rows_and_settings(env):
    """infinities, NaN, empty rows, greedy rows, settings outside their ranges"""
    n, v = 12, 300
    l = cases.gaussian(2, (n, v), 2.0)
    l[0] = -np.inf
    l[1] = np.nan
    l[2, ::2] = -np.inf
    l[3, 5], l[3, 9] = np.inf, np.inf
    l[4, 7] = np.nan
    l[5] = -np.inf
    l[5, 123] = -3e38
    l[6] = np.finfo(f32).min
    l[7, 10] = l[7, 20] = 50.0
    u = np.array([0.5] * 8 + [0.0, 1.0, -1.0, np.nan], f32)
    for kw in ({}, {"top_k": 3}, {"top_p": 0.9}, {"min_p": 0.1}, {"top_k": 40, "top_p": 0.5, "min_p": 0.01}, {"temperature": 0.0},
               {"temperature": 1e-38}, {"temperature": np.inf}, {"temperature": np.nan}, {"temperature": -1.0}, {"top_p": 0.0},
               {"top_p": -2.0}, {"top_p": 2.0}, {"min_p": 7.0}, {"min_p": -1.0}, {"top_k": -4}, {"top_k": v}, {"top_k": 2 ** 31 - 1}):
        got = check_sample(env, l, u, **kw)
        assert got[0] == 0 and got[1] == 0 and got[5] == 123 and got[4] != 7 and (got[2] % 2 == 1)
    assert check_sample(env, l, u, temperature=0.0)[7] == 10
    assert set(check_sample(env, l, u)[3:4]) <= {5, 9}


def test_sample_logits_further_apart_than_f32_reaches(env):
    """differences above the largest f32 number under large and infinite temperatures; the smallest numbers under the smallest ones"""
    n, v = 8, 2000
    u = ((np.arange(n) + 0.3) / n).astype(f32)
    far = (np.random.default_rng(5).uniform(-1, 1, (n, v)) * 3.4e38).astype(f32)
    far[:, 7], far[:, 9] = -np.inf, np.nan
    for temp in (1e38, 3e38, 3e37, np.inf):
        for kw in ({}, {"top_k": 5}, {"top_k": 700}, {"top_p": 0.5}, {"top_p": 0.02}, {"min_p": 0.2}, {"top_k": 1000, "top_p": 0.7}):
            check_sample(env, far, u, temperature=temp, **kw)
    near = (np.random.default_rng(6).integers(0, 40, (n, v)) * 1e-44).astype(f32)
    for temp in (1e-45, 1e-40, 1e-38, 1e-31):
        for kw in ({}, {"top_k": 5}, {"top_p": 0.5}, {"min_p": 0.2}, {"top_k": 1000, "top_p": 0.7}):
            assert (check_sample(env, near, u, temperature=temp, **kw) < v).all()


@pytest.mark.parametrize("temp,top", [(0.04, None), (0.02, None), (0.3, None), (0.03, 4.05), (0.02, 4.05), (0.03, 0.1)])
def test_sample_nuclei_next_to_the_whole(env, temp, top):
    """top_p so close to 1 that the border may be any of the last weights, among thousands of logits whose weight is 0"""
    n, v = 8, 60000
    logits = cases.gaussian(31, (n, v), 1.0)
    if top is not None:  # the largest just above a power of two, most of the others below it
        logits += f32(top) - logits.max(1, keepdims=True)
    u = np.array([0.0, 0.2, 0.5, 0.9, 0.99, 0.999, 0.9999, 0.99999], f32)
    for top_p in (0.9999, 0.99995, 0.99999, 0.9999999):
        check_sample(env, logits, u, temperature=temp, top_p=top_p)
        check_sample(env, logits, u, temperature=temp, top_p=top_p, min_p=1e-12)
        check_sample(env, logits, u, temperature=temp, top_p=top_p, top_k=30000)


def test_sample_on_streams_and_in_graphs(env):
    """two streams at once and captured calls give the eager tokens; settings changed in place take effect at the next replay"""
    t, n, v = env.torch, 40, 20000
    logits = env.dev(cases.gaussian(12, (n, v), 2.0))
    u = t.rand(n, device="cuda")
    kw = {"temperature": t.full((n,), 0.8, device="cuda"), "top_p": t.full((n,), 0.9, device="cuda"),
          "top_k": t.full((n,), 300, dtype=t.int32, device="cuda"), "min_p": t.zeros(n, device="cuda")}
    ref = env.serving.sample(logits, u, **kw)
    t.cuda.synchronize()
    streams, graphs, outs, captured = [t.cuda.Stream() for _ in range(2)], [], [], []
    for s in streams:
        with t.cuda.stream(s):
            outs += [env.serving.sample(logits, u, **kw) for _ in range(5)]
    t.cuda.synchronize()
    for s in streams:
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g, stream=s):
            captured.append(env.serving.sample(logits, u, **kw))
        graphs.append(g)

    def replay():
        for _ in range(3):
            for s, g in zip(streams, graphs):
                with t.cuda.stream(s):
                    g.replay()
        t.cuda.synchronize()
    replay()
    assert all((o == ref).all() for o in outs + captured)
    kw["temperature"].zero_()
    t.cuda.synchronize()
    replay()
    assert all((o == logits.argmax(1)).all() for o in captured)


def test_sample_strided_rows_and_largest_vocabulary(env):
    t = env.torch
    base = env.dev(cases.gaussian(4, (5, 1009), 2.0))
    u = np.array([0.1, 0.3, 0.5, 0.7, 0.9], f32)
    check_sample(env, base[:, 3:1000], u, top_p=0.9)
    check_sample(env, base.t()[:900], np.resize(u, 900), top_k=2)  # columns as rows: copied first
    g = t.Generator(device="cuda").manual_seed(1)
    check_sample(env, t.randn(2, 1 << 19, generator=g, device="cuda") * 2, u[:2], top_p=0.95, top_k=[0, 5000])
    with pytest.raises(env.KoreError):
        env.serving.sample(t.zeros((1, (1 << 19) + 1), device="cuda"), env.dev(u[:1]))
    assert env.serving.sample(t.zeros((0, 7), device="cuda"), t.zeros(0, device="cuda")).shape == (0,)


def test_sample_follows_the_distribution(env):
    """the numbers (i + 0.5) / n draw every token its share of n times, to within one"""
    n, v = 4000, 97
    l = cases.gaussian(8, (1, v), 1.5)
    tokens = env.serving.sample(env.dev(l).expand(n, v), env.dev(((np.arange(n) + 0.5) / n).astype(f32))).cpu().numpy()
    p = np.exp(l[0].astype(np.float64) - l.max())
    # the tokens run in index order, so a token's count is off by less than one; the f32 numbers move a border by 2^-24 n
    assert np.abs(np.bincount(tokens, minlength=v) - n * p / p.sum()).max() <= 1.01


# ---- refusals of the Python layer ----------------------------------------------------------------
def test_python_refusals(env):
    t, s = env.torch, env.serving
    cache = s.KV4Cache(2, 2, 10, 16)
    assert cache.max_len == 12 and cache.memory_bytes() == 2 * 2 * 2 * 12 * (2 + 1) * 4
    z = lambda *shape, dt=t.float32: t.zeros(shape, dtype=dt, device="cuda")
    i32, i64 = t.int32, t.int64
    bad = [lambda: cache.read(z(3, dt=i32)), lambda: cache.read(z(3, 1, dt=i64)), lambda: cache.read(z(3, dt=i64), k_out=z(3, 2, 15)),
           lambda: s.attend(z(2, 4, 16, dt=t.float16), cache, z(2, dt=i32)), lambda: s.attend(z(2, 4, 16), cache, z(3, dt=i32)),
           lambda: s.attend(z(2, 3, 16), cache, z(2, dt=i32)), lambda: s.attend(z(1, 4, 16), cache, z(2, dt=i32)),
           lambda: s.attend(z(2, 4, 16), cache, z(2, dt=i64)), lambda: s.attend(z(2, 4, 16), cache, z(2, dt=i32), out=z(2, 4, 15)),
           lambda: s.attend(z(2, 4, 16), cache, z(2, dt=i32), scale=float("nan")),
           lambda: s.qknorm_rope_append(z(3, 8 * 16), z(3, dt=i32), z(3, dt=i64), z(12, 8), z(12, 7), cache, 4),
           lambda: s.qknorm_rope_append(z(3, 8 * 16), z(3, dt=i64), z(3, dt=i64), z(12, 8), z(12, 8), cache, 4),
           lambda: s.qknorm_rope_append(z(3, 7 * 16), z(3, dt=i32), z(3, dt=i64), z(12, 8), z(12, 8), cache, 3),
           lambda: s.qknorm_rope_append(z(3, 8 * 16), z(3, dt=i32), z(3, dt=i64), z(12, 8), z(12, 8), cache, 4, q_gamma=z(15)),
           lambda: s.qknorm_rope_append(z(3, 8 * 16), z(3, dt=i32), z(3, dt=i64), z(12, 8), z(12, 8), (z(2, 2, 12, 16), z(2, 2, 12, 8)), 4),
           lambda: s.sample(z(2, 5), z(3)), lambda: s.sample(z(2, 5), z(2), top_k=z(2)), lambda: s.sample(z(2, 0), z(2)),
           lambda: s.sample(z(2, 5), z(2), tokens=z(2, dt=i32)), lambda: s.KV4Cache(1, 1, 8, 30)]
    for call in bad:
        with pytest.raises(env.KoreError):
            call()


def test_native_calls_and_what_they_decline(env):
    """plain arguments are answered by the native module, with the results of the way around it; others are declined, whatever they are"""
    t, s = env.torch, env.serving
    nat, f, i32 = s.native(), t.float32, t.int32
    cache = filled_cache(env, 2, 2, 12, 16, 40)
    z = lambda *shape, dt=f: t.zeros(shape, dtype=dt, device="cuda")
    q, lens = env.dev(cases.gaussian(41, (2, 3, 4, 16), 1.0)), env.dev(np.array([12, 5], np.int32))
    held = cache._held
    around = s.attend(t.cat([q, q], -1)[..., :16], cache, lens, scale=1)  # strided, an integer scale
    out = z(2, 3, 4, 16)
    got = nat.attend(held, 16, q, lens, 1.0, out)
    assert got is out and (out == around).all() and (nat.attend(held, 16, q, lens, 1.0, None) == around).all()
    rows = t.arange(24, device="cuda")
    k, v = nat.read(held, 16, rows, None, None)
    k2, v2 = z(24, 2, 16), z(24, 2, 16)
    assert nat.read(held, 16, rows, k2, v2)[1] is v2 and (k == k2).all() and (v == v2).all()
    logits, u = env.dev(cases.gaussian(42, (5, 90), 2.0)), t.rand(5, device="cuda")
    kw = dict(temperature=z(5) + 0.5, top_k=z(5, dt=i32) + 9, top_p=z(5) + 0.9, min_p=z(5) + 0.01)
    a = nat.sample(logits, u, *kw.values(), True, None)
    b = s.sample(t.nn.functional.pad(logits, (0, 7))[:, :90].t().contiguous().t(), u, return_logprobs=True, **kw)
    assert (a[0] == b[0]).all() and (a[1] == b[1]).all() and nat.sample(logits[:, 3:50], u, None, None, None, None, False, None) is not None
    x, pos, at = env.dev(cases.gaussian(43, (3, 8 * 16), 1.0)), z(3, dt=i32), t.arange(3, device="cuda")
    cos, sin = (env.dev(c) for c in tables(4, 16))
    pair = (z(2, 2, 12, 16), z(2, 2, 12, 16))
    for caches, hd in ((filled_cache(env, 2, 2, 12, 16, 44)._held, 16), (pair, 0)):
        good = [x, pos, at, cos, sin, caches, hd, 4, z(16) + 1, None, 1e-5, None]
        assert nat.append(*good).shape == (3, 4, 16)
        # arguments changed one at a time: types, shapes, orders, devices, kinds
        for i, bads in ((0, [x.double(), x[:, 1:], x.cpu(), x[0], None, x.t().contiguous().t()]), (1, [pos.long(), pos[:2], pos.cpu(), 7]),
                        (2, [at.int(), at[None], None]), (3, [cos[:, :3], cos.half(), cos.cpu(), z(0, 8)]), (4, [sin[:2], sin.t()]),
                        (5, [list(caches), caches[:1], (1, 2), None]), (7, [3, 4.0, -1, 1 << 70, "4"]), (8, [z(15), z(16, dt=t.float16)]),
                        (10, [1, None, -1.0]), (11, [z(3, 4, 15), x])):
            for bad in bads:
                assert nat.append(*good[:i], bad, *good[i + 1:]) is None, (i, bad)
        assert nat.append(*good[:-1]) is None and nat.append() is None
    assert nat.attend(held, 16, q[:1], lens, 1.0, None) is None and nat.attend(held, 16, q, lens.long(), 1.0, None) is None
    assert nat.attend(held, 16, q[:, :, :3].contiguous(), lens, 1.0, None) is None and nat.attend(held, 16, q, lens, float("nan"), None) is None
    assert nat.attend(held, 16, q[:, :0], lens, 1.0, None) is None and nat.attend(held[:3], 16, q, lens, 1.0, None) is None
    assert nat.read(held, 16, rows.int(), None, None) is None and nat.read(held, 16, rows, z(24, 2, 15), None) is None and nat.read(held, 16, rows[:0], None, None) is None
    assert nat.sample(logits, u[:4], None, None, None, None, False, None) is None and nat.sample(logits, u, None, z(5), None, None, False, None) is None
    assert nat.sample(logits, u, None, None, None, None, 0, None) is None and nat.sample(z(5, 0), u, None, None, None, None, False, None) is None
    # on another stream, and from several threads at once
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        assert (s.attend(q, cache, lens, scale=1.0) == around).all()
    import threading

    results = []

    def work():
        with t.cuda.stream(t.cuda.Stream()):
            r = [s.attend(q, cache, lens, scale=1.0) for _ in range(50)]
            t.cuda.current_stream().synchronize()
            results.append(all((y == around).all() for y in r))
    t.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(4)]
    [th.start() for th in threads]
    [th.join() for th in threads]
    assert results == [True] * 4


# ---- together: the decoder ------------------------------------------------------------------------
class Ref4(dr.DecoderRef):
    """the decoder's restatement with grouped heads, norms of queries and keys, and keys and values as the 4-bit cache stores them"""

    def forward(self, tokens):
        cfg, W, t = self.cfg, self.w, len(tokens)
        H, kv, hd = cfg.n_heads, cfg.kv_heads, cfg.head_dim
        hidden = W["embed"][np.asarray(tokens)].astype(f32)
        pos = np.arange(self.pos, self.pos + t)
        stored = (lambda x: sr.values(*sr.quantise(x), hd)) if cfg.kv_bits == 4 else (lambda x: x)
        for li, lw in enumerate(W["layers"]):
            xn = dr.rmsnorm(hidden, lw["norm1"], cfg.eps)
            qkv = np.concatenate([dr.project(lw[n], xn) for n in ("q", "k", "v")], 1)
            q, k, v = sr.append(qkv, pos, self.cos, self.sin, H, kv, hd, lw.get("q_norm"), lw.get("k_norm"), cfg.eps)
            self.k[li] = np.concatenate([self.k[li].reshape(-1, kv, hd), stored(k)])
            self.v[li] = np.concatenate([self.v[li].reshape(-1, kv, hd), stored(v)])
            a = dr.attention(q, self.k[li].repeat(H // kv, 1), self.v[li].repeat(H // kv, 1), self.pos).reshape(t, H * hd)
            hidden = dr.project(lw["o"], a, resid=hidden)
            xn = dr.rmsnorm(hidden, lw["norm2"], cfg.eps)
            hidden = dr.project(lw["down"], dr.silu_mul(dr.project(lw["gate"], xn), dr.project(lw["up"], xn)), resid=hidden)
        self.pos += t
        return (dr.rmsnorm(hidden[-1:], W["norm_f"], cfg.eps) @ W["lm_head"].T.astype(f32)).astype(f32)[0]


@pytest.mark.parametrize("batch,kv,bits,norm", [(2, 2, 4, True), (1, 4, 4, False), (3, 4, 32, True)])
def test_decoder_with_serving_operators(env, batch, kv, bits, norm):
    """prompt and steps (eager and from the graph) of a decoder with these operators against its restatement, then sampled steps"""
    t = env.torch
    cfg = env.decoder.DecoderConfig(n_layers=2, d_model=144, n_heads=4, d_ff=256, vocab=97, max_len=30, n_kv_heads=kv, qk_norm=norm,
                                    kv_bits=bits)
    weights = env.decoder.random_weights(cfg, seed=4100)
    if norm:
        for li, lw in enumerate(weights["layers"]):
            lw["q_norm"], lw["k_norm"] = ((1 + cases.gaussian(li * 2 + i, (cfg.head_dim,), 0.2)).astype(f32) for i in (0, 1))
    cos, sin = env.decoder.rope_tables(cfg)
    prompt = np.array([[5, 17, 3, 90, 41, 8], [1, 2, 3, 4, 5, 6], [9, 9, 8, 7, 60, 96]], np.int64)[:batch]
    dec = env.decoder.BitNetDecoder(cfg, weights, batch=batch)
    assert dec.persistent is None
    logits = dec.prefill(env.dev(prompt)).cpu().numpy()
    refs = [Ref4(cfg, weights, cos, sin) for _ in range(batch)]
    ref_logits = np.stack([r.forward(list(p)) for r, p in zip(refs, prompt)])
    # a last-bit difference in front of an 8-bit or 4-bit code can flip it: 3 % of the largest logit, as the f32 decoder's test
    # allows 2 % for its 8-bit codes; a 4-bit code that flips moves one of 144 values by 1/15 of its row's range
    tol = 0.03 * np.abs(ref_logits).max()
    assert np.abs(logits - ref_logits).max() <= tol
    toks = logits.argmax(axis=1)
    dec.tokens.copy_(env.dev(toks))
    for step in range(4):
        dec.decode_step(use_graph=step > 0)
        ref_logits = np.stack([r.forward([int(x)]) for r, x in zip(refs, toks)])
        got = dec.logits.cpu().numpy()
        assert np.abs(got - ref_logits).max() <= tol, step
        toks = dec.tokens.cpu().numpy()
        assert (toks == got.argmax(axis=1)).all()
    # sampled steps: the token is what the operator's restatement draws from the step's own logits and numbers
    dec.set_sampling(temperature=0.8, top_k=20, top_p=0.95, min_p=[0.01] * batch, seed=7)
    for step in range(4):
        if step == 3:
            dec.set_sampling(temperature=1.5, top_k=5, seed=8)  # in place, under the captured step
        dec.decode_step()
        got, u = dec.logits.cpu().numpy(), dec.uniform.cpu().numpy()
        for b in range(batch):
            kw = dict(temperature=f32(0.8), top_k=20, top_p=float(f32(0.95)), min_p=float(f32(0.01))) if step < 3 else dict(temperature=1.5, top_k=5)
            tok, _, margin = sr.sample_row(got[b], u[b], **kw)
            assert margin < 1e-9 or tok == int(dec.tokens[b])
    dec.set_sampling(None)
    dec.decode_step()
    assert (dec.tokens.cpu().numpy() == dec.logits.cpu().numpy().argmax(axis=1)).all()
    dec.close()


def test_decoder_sampling_behind_the_persistent_step(env):
    """one sequence with an f32 cache keeps its one-launch step; the draw follows it.  Equal seeds give equal texts"""
    cfg = env.decoder.DecoderConfig(n_layers=2, d_model=128, n_heads=4, d_ff=256, vocab=97, max_len=32)
    dec = env.decoder.BitNetDecoder(cfg, env.decoder.random_weights(cfg, seed=4000), batch=1)
    assert dec.persistent is not None
    prompt = env.dev(np.array([[5, 17, 3]], np.int64))
    texts = []
    for seed in (3, 3, 4):
        dec.set_sampling(temperature=2.0, seed=seed)
        texts.append(dec.generate(prompt, 12).cpu().numpy())
    assert (texts[0] == texts[1]).all() and (texts[0] != texts[2]).any()
    dec.set_sampling(None)
    greedy = dec.generate(prompt, 12).cpu().numpy()
    dec.set_sampling(temperature=0.0)
    assert (dec.generate(prompt, 12).cpu().numpy() == greedy).all()
    dec.close()


def test_decoder_refusals(env):
    for kw in (dict(kv_bits=8), dict(n_kv_heads=3, kv_bits=4), dict(n_kv_heads=2)):
        cfg = env.decoder.DecoderConfig(n_layers=1, d_model=128, n_heads=4, d_ff=256, vocab=50, max_len=16, **kw)
        with pytest.raises(env.KoreError):
            env.decoder.BitNetDecoder(cfg, {"layers": []}, batch=1)
