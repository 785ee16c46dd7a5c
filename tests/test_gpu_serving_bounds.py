"""Serving-step kernels where rare numbers meet: attention over the 4-bit cache at the ends of its ranges, borders of nuclei."""
import numpy as np
import pytest

from oracle import serving_ref as sr
from tests import cases
from tests.test_gpu_serving import check_attention, check_sample, env, filled_cache, tables  # noqa: F401

pytestmark = pytest.mark.gpu
f32 = np.float32


def cache_of(env, k, v):
    """A cache of these rows [seqs, kv, positions, hd]"""
    seqs, kv, n, hd = k.shape
    c = env.serving.KV4Cache(seqs, kv, n, hd)
    for side, x in (("k", k), ("v", v)):
        words, steps = sr.quantise(x)
        getattr(c, side + "_codes")[:, :, :n].copy_(env.dev(words.view(np.int32)))
        getattr(c, side + "_steps")[:, :, :n].copy_(env.dev(steps.view(np.int32)))
    return c


@pytest.mark.parametrize("n,t", [(1, 1), (2, 1), (40, 1), (40, 5), (700, 1), (3000, 2)])
def test_attention_of_the_largest_values(env, n, t):
    """values up to 2^119 / lens, as far as the header says they go"""
    hd, heads = 36, 4
    rng = np.random.default_rng(n)
    v = (rng.uniform(0, 0.99, (1, 2, n, hd)) * 2.0 ** 119 / n).astype(f32)
    v[:, 1] *= rng.choice([-1, 1], (1, n, hd))
    k = rng.standard_normal((1, 2, n, hd)).astype(f32)
    check_attention(env, cases.gaussian(n, (1, t, heads, hd), 1.0), cache_of(env, k, v), [n])


def test_attention_of_large_values_under_rising_weights(env):
    """weights that rise to 2^7.5 times the first ones without a new reference, on values of 2^110 behind values of 2^80"""
    hd, n = 64, 512
    late = np.arange(n) >= 128
    k = np.broadcast_to(np.where(late, 7.5 * np.log(2.0), 0.0)[:, None], (1, 1, n, hd)).astype(f32)  # 64 equal dims, queries of 1 / 8, scale 1 / 8
    v = (np.random.default_rng(1).uniform(-0.99, 0.99, (1, 1, n, hd)) * np.where(late, 2.0 ** 110, 2.0 ** 80)[:, None]).astype(f32)
    check_attention(env, np.full((1, 1, 1, hd), 1 / 8, f32), cache_of(env, k, v), [n])


@pytest.mark.parametrize("rows", ["constant", "spread"])
def test_attention_of_the_largest_scores(env, rows):
    """scale log2(e) sum|q| max|k| of 2^121.5: one position has all the weight"""
    hd, n, heads = 64, 300, 2
    rng = np.random.default_rng(4)
    q = np.abs(cases.gaussian(5, (1, 1, heads, hd), 30.0))
    if rows == "spread":
        q *= rng.choice([-1, 1], hd).astype(f32)
        k = rng.uniform(-0.9, 0.9, (1, heads, n, hd))
        k[0, :, 211] = np.sign(q[0, 0])
    else:
        k = np.broadcast_to((rng.permutation(n)[None, :, None] + 1.0) / n, (1, heads, n, hd))
    k = (k * 2.0 ** 121.5 * np.log(2.0) * np.sqrt(hd) / np.abs(q).sum(-1).max()).astype(f32)
    cache = cache_of(env, k, rng.standard_normal((1, heads, n, hd)).astype(f32))
    got = env.serving.attend(env.dev(q), cache, env.dev(np.array([n], np.int32)))[0, 0].cpu().numpy()
    at = 211 if rows == "spread" else int(k[0, 0, :, 0].argmax())
    value = cache.read(env.dev(np.array([at])))[1][0].cpu().numpy()
    # the next score is lower by far more than any rounding (1 / 300 of the largest at least): a weight of 1, held to 22 bits
    assert (np.abs(got - value) <= 2.0 ** -20 * np.abs(value).max()).all()


@pytest.mark.parametrize("side", ["k", "v"])
def test_rows_below_the_bfloat16_numbers(env, side):
    """-3.4e38 is an f32 number, but no bfloat16 number lies at or below it; the next row is an ordinary one"""
    hd = 8
    x = np.full((2, 3 * hd), -1.0, f32)
    x[0, slice(hd, 2 * hd) if side == "k" else slice(2 * hd, None)] = -3.4e38
    cache, one, zero = env.serving.KV4Cache(1, 1, 4, hd), np.ones((4, hd // 2), f32), np.zeros((4, hd // 2), f32)
    i = np.arange(2)
    env.serving.qknorm_rope_append(env.dev(x), env.dev(i.astype(np.int32)), env.dev(i), env.dev(one), env.dev(zero), cache, 1)
    for name, got in zip("kv", cache.read(env.dev(i))):
        got = got.cpu().numpy()[:, 0]
        assert (np.isnan(got[0]).all() if name == side else (got[0] == -1).all()) and (got[1] == -1).all()


# seeds of rows and top_p whose border, less the accuracy of the sums that look for it, lies where running sums in f64 of
# neighbouring threads do not meet: found by a search on the CPU over 2e8 rows
BETWEEN = [(38773736, 0.932712317), (65209376, 0.979467869), (186987744, 0.996985555), (74197353, 0.98854059), (171723530, 0.690360785),
           (57606035, 0.998813152), (28156044, 0.930305243), (52030044, 0.922126591), (61540356, 0.998595774), (124656509, 0.997032821),
           (187341261, 0.796574116), (175736678, 0.892285883), (213259238, 0.889294267)]


def test_sample_nuclei_that_end_between_two_sums(env):
    """rows of 20 to 60 equal logits every 1/32: every row gets its token"""
    rows = np.full((len(BETWEEN), 256 * 61), -np.inf, f32)
    for row, (state, _) in zip(rows, BETWEEN):
        row[0], at = 0.0, 1
        for b in range(256):
            state = (state * 1664525 + 1013904223) % 2 ** 32
            n = 20 + (state >> 16) % 41
            row[at:at + n] = -(b + 0.5) / 32
            at += n
    top_p = np.array([p for _, p in BETWEEN], f32)
    for u in (0.02, 0.37, 0.75, 0.99):
        check_sample(env, rows, np.full(len(rows), u, f32), top_p=top_p)


# ---- the decoder's count of its launches ----------------------------------------------------------
@pytest.mark.parametrize("batch,kv,bits,max_len", [(1, 4, 4, 32), (2, 2, 4, 4000), (6, 2, 4, 4000), (3, 4, 32, 32), (20, 4, 4, 32)])
def test_decoder_counts_its_launches(env, batch, kv, bits, max_len):
    """launches_per_step is the number of kernels of a captured step, and one more with sampling for the numbers drawn before it"""
    from cuda.bindings import runtime

    t = env.torch
    cfg = env.decoder.DecoderConfig(n_layers=2, d_model=128, n_heads=4, d_ff=256, vocab=97, max_len=max_len, n_kv_heads=kv, kv_bits=bits)
    dec = env.decoder.BitNetDecoder(cfg, env.decoder.random_weights(cfg, seed=4000), batch=batch)
    prompt = t.zeros((batch, 3), dtype=t.int64, device="cuda")
    assert dec.launches_per_step == 0
    for sampling in (False, True):
        dec.prefill(prompt)
        if sampling:
            dec.set_sampling(temperature=0.8)
        stream = t.cuda.Stream()
        stream.wait_stream(t.cuda.current_stream())
        with t.cuda.stream(stream):
            dec._decode_body()
        t.cuda.synchronize()
        g = t.cuda.CUDAGraph(keep_graph=True)
        with t.cuda.graph(g, stream=stream):
            dec._decode_body()
        raw = g.raw_cuda_graph()
        count = runtime.cudaGraphGetNodes(raw, 0)[2]
        nodes = runtime.cudaGraphGetNodes(raw, count)[1]
        kernels = sum(runtime.cudaGraphNodeGetType(x)[1] == runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel for x in nodes)
        assert dec.launches_per_step == kernels + sampling
        dec.generate(prompt, 3)  # a prompt and its first choice are no step
        assert dec.launches_per_step == kernels + sampling
    dec.close()


def test_decoder_counts_the_draw_behind_the_persistent_step(env):
    cfg = env.decoder.DecoderConfig(n_layers=2, d_model=128, n_heads=4, d_ff=256, vocab=97, max_len=32)
    dec = env.decoder.BitNetDecoder(cfg, env.decoder.random_weights(cfg, seed=4000), batch=1)
    assert dec.persistent is not None
    for temperature, launches in ((None, 1), (0.7, 3), (None, 1)):
        dec.set_sampling(temperature)
        dec.decode_step()
        assert dec.launches_per_step == launches
    dec.close()


# ---- without the native module ------------------------------------------------------------------
def test_results_without_the_native_module(env, monkeypatch):
    """the four operators by way of the interpreter: the same bits"""
    t, s = env.torch, env.serving
    hd, lmax = 64, 2000
    cos, sin = (env.dev(np.asarray(a, f32)) for a in (np.cos(np.arange(lmax))[:, None].repeat(hd // 2, 1), np.sin(np.arange(lmax))[:, None].repeat(hd // 2, 1)))
    x, q = env.dev(cases.gaussian(1, (6, 8 * hd), 1.0)), env.dev(cases.gaussian(2, (2, 3, 4, hd), 1.0))
    rows, lens = env.dev(np.array([0, 1, 2, lmax, lmax + 1, 2 * lmax - 1])), env.dev(np.array([3, lmax], np.int32))
    pos = (rows % lmax).int()
    logits, u = env.dev(cases.gaussian(3, (5, 3001), 2.0)), t.rand(5, device="cuda")

    def run():
        cache = s.KV4Cache(2, 2, lmax, hd)
        out = [s.qknorm_rope_append(x, pos, rows, cos, sin, cache, 4), *cache.read(rows), s.attend(q, cache, lens)]
        return out + list(s.sample(logits, u, top_p=t.full((5,), 0.9, device="cuda"), return_logprobs=True))
    with_module = run()
    monkeypatch.setattr(s, "_native", s._Declines)
    assert all((a == b).all() for a, b in zip(with_module, run()))


# ---- calls that the header allows --------------------------------------------------------------
@pytest.mark.parametrize("scale", [-0.2, 1e-3, 3.0])
@pytest.mark.parametrize("lmax", [300, 1500])
def test_attention_scales(env, scale, lmax):
    check_attention(env, cases.gaussian(70, (2, 2, 6, 44), 1.0), filled_cache(env, 2, 3, lmax, 44, 71), [lmax, lmax // 2 + 1], scale)


@pytest.mark.parametrize("n", [3, 700])
@pytest.mark.parametrize("which", ["q", "k"])
def test_append_with_one_gamma(env, n, which):
    """norms of queries alone or of keys alone, for few and for many tokens"""
    heads, kv, hd, lmax = 6, 2, 36, 704
    qkv = cases.gaussian(n, (n, (heads + 2 * kv) * hd), 2.0)
    gamma = (1 + cases.gaussian(7, (hd,), 0.2)).astype(f32)
    gq, gk = (gamma, None) if which == "q" else (None, gamma)
    cos, sin = tables(lmax, hd)
    i = np.arange(n)
    cache = env.serving.KV4Cache(1, kv, lmax, hd)
    q = env.serving.qknorm_rope_append(env.dev(qkv), env.dev(i.astype(np.int32)), env.dev(i), env.dev(cos), env.dev(sin), cache, heads,
                                       **{which + "_gamma": env.dev(gamma)})
    rq, rk, rv = sr.append(qkv, i, cos, sin, heads, kv, hd, gq, gk)
    assert (q.cpu().numpy() == rq).all()
    for got, x in zip(cache.read(env.dev(i)), (rk, rv)):
        assert (got.cpu().numpy() == sr.values(*sr.quantise(x), hd)).all()


def test_read_of_one_side(env):
    """a C caller may ask for keys or values alone, and then has no planes of the other"""
    from kore_b200 import _cabi

    t, seqs, kv, lmax, hd = env.torch, 2, 3, 40, 20
    cache = filled_cache(env, seqs, kv, lmax, hd, 72)
    rows = env.dev(np.array([0, 41, -1, 79, 80, 7]))
    both = cache.read(rows)
    stream = t.cuda.current_stream().cuda_stream
    for side, planes in enumerate(((cache.k_codes, cache.k_steps), (cache.v_codes, cache.v_steps))):
        out = t.full((6, kv, hd), 5.0, device="cuda")
        a, b = (x.data_ptr() for x in planes)
        args = (a, b, None, None) if side == 0 else (None, None, a, b)
        outs = (out.data_ptr(), None) if side == 0 else (None, out.data_ptr())
        _cabi.check(_cabi.lib().kb_kv4_read(*args, rows.data_ptr(), 6, kv, hd, seqs, lmax, *outs, stream))
        t.cuda.synchronize()
        assert (out == both[side]).all()


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_sample_rows_at_any_address(env, offset):
    """slices of a wider matrix, one row and several, whose rows start at every place of 16 bytes"""
    wide = env.dev(cases.gaussian(73, (3, 5011), 2.5))
    for n in (1, 3):
        view = wide[:n, offset:offset + 5003]
        check_sample(env, view, np.array([0.2, 0.6, 0.93][:n], f32), top_p=0.9)
        check_sample(env, view, np.array([0.2, 0.6, 0.93][:n], f32), top_k=30, temperature=0.7)
        check_sample(env, view, np.array([0.2, 0.6, 0.93][:n], f32), temperature=0.0)
