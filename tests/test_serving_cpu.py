"""Serving-step operators without a GPU: the restatement's own identities, and what the library refuses before any launch."""
import ctypes as C

import numpy as np
import pytest

from oracle import serving_ref as sr

f32 = np.float32


def test_quantiser_bounds_and_exact_rows():
    rng = np.random.default_rng(1)
    for hd in (4, 36, 100, 128):
        x = (rng.standard_normal((50, hd)) * np.exp(rng.uniform(-20, 20, (50, 1)))).astype(f32)
        words, steps = sr.quantise(x)
        step, lo = sr.pair_of(steps)
        assert words.shape == (50, (hd + 7) // 8)
        # half a step for the code; the f32 roundings of x - lo, of times 1 / step and of the sum come to a few 2^-24 of 15 steps and of |lo|
        slack = 2.0 ** -20 * (15 * step.astype(np.float64) + np.abs(lo))
        assert (np.abs(sr.values(words, steps, hd).astype(np.float64) - x) <= (0.5 * step.astype(np.float64) + slack)[:, None]).all()
        assert (lo <= x.min(-1)).all() and (step >= f32(2.0 ** -100)).all()
        if hd % 8:
            assert (words[:, -1] >> np.uint32(4 * (hd % 8)) == 0).all()  # tail codes are zero


def test_quantiser_special_rows():
    rows = np.zeros((6, 8), f32)
    rows[1] = 3.0  # constant, a bfloat16 number: comes back exactly
    rows[2, 3] = np.nan
    rows[3, 0] = -np.inf
    rows[4, 0], rows[4, 1] = -3e38, 3e38  # the range overflows
    rows[5] = np.float32(1e-42)  # subnormal
    words, steps = sr.quantise(rows)
    out = sr.values(words, steps, 8)
    assert (out[0] == 0).all() and (out[1] == 3).all()
    assert np.isnan(out[2:5]).all() and (words[2:5] == 0).all()
    assert (np.abs(out[5] - rows[5]) < 1e-40).all()


def test_sample_reference_keeps_what_it_says():
    l = np.array([1.0, 3.0, 3.0, 2.0, -np.inf, np.nan], f32)
    assert sr.sample_row(l, 0.99, top_k=1)[0] == 1  # equal logits: the lowest index
    assert sr.sample_row(l, 0.99, top_k=2)[0] == 2
    assert sr.sample_row(l, 0.99, top_p=0.0)[0] == 1
    assert sr.sample_row(l, 0.99, min_p=1.0)[0] == 2
    assert sr.sample_row(l, 0.99, temperature=0.0)[:2] == (1, 0.0)
    assert sr.sample_row(l, 0.0)[0] == 0
    assert sr.sample_row(np.full(3, -np.inf, f32), 0.5)[0] == 0
    got = [sr.sample_row(l, u)[0] for u in (np.arange(4000) + 0.5) / 4000]
    p = np.exp(l[:4].astype(np.float64) - 3)
    assert np.abs(np.bincount(got, minlength=6)[:4] / 4000 - p / p.sum()).max() <= 1 / 4000


@pytest.fixture(scope="module")
def lib():
    from kore_b200 import _cabi

    return _cabi.lib()


E_INVALID, E_UNSUPPORTED = 8, 9
P = 1 << 20  # stands for a device pointer: never dereferenced by a call that is refused


def _append4(lib, **kw):
    a = dict(qkv=P, ld=0, positions=P, rows=P, cos=P, sin=P, max_pos=8, gq=None, gk=None, eps=1e-5, n=0, heads=4, kv=2, hd=32, seqs=1,
             lmax=8, q=P, kc=P, ks=P, vc=P, vs=P)
    a.update(kw)
    a["eps"] = C.c_float(a["eps"])
    return lib.kb_qknorm_rope_kv4(*a.values(), None)


def _append32(lib, **kw):
    a = dict(qkv=P, ld=0, positions=P, rows=P, cos=P, sin=P, max_pos=8, gq=None, gk=None, eps=1e-5, n=0, heads=4, kv=2, hd=32, seqs=1,
             lmax=8, q=P, k=P, v=P)
    a.update(kw)
    a["eps"] = C.c_float(a["eps"])
    return lib.kb_qknorm_rope_kv(*a.values(), None)


def _read(lib, **kw):
    a = dict(kc=P, ks=P, vc=P, vs=P, rows=P, n=0, kv=2, hd=32, seqs=1, lmax=8, k=P, v=P)
    a.update(kw)
    return lib.kb_kv4_read(*a.values(), None)


def _attn(lib, **kw):
    a = dict(q=P, kc=P, ks=P, vc=P, vs=P, lens=P, batch=0, t=1, heads=4, kv=2, hd=32, lmax=8, scale=0.0, out=P, ws=None, wsb=0)
    a.update(kw)
    a["scale"] = C.c_float(a["scale"])
    return lib.kb_attn_kv4(*a.values(), None)


def _sample(lib, **kw):
    a = dict(logits=P, n=0, vocab=10, ld=0, t=None, k=None, p=None, m=None, u=P, tokens=P, logprobs=None)
    a.update(kw)
    return lib.kb_sample(*a.values(), None)


def test_empty_calls_do_nothing(lib):
    for call in (_append4, _append32, _read, _attn, _sample):
        assert call(lib) == 0
    assert _attn(lib, batch=3, t=0) == 0


@pytest.mark.parametrize("call,changes,code", [
    (_append4, dict(qkv=None), E_INVALID), (_append4, dict(vs=None), E_INVALID), (_append4, dict(heads=3), E_INVALID),
    (_append4, dict(kv=0), E_INVALID), (_append4, dict(hd=30), E_UNSUPPORTED), (_append4, dict(hd=132), E_UNSUPPORTED),
    (_append4, dict(lmax=10), E_UNSUPPORTED), (_append4, dict(ld=255), E_INVALID), (_append4, dict(eps=-1.0), E_INVALID),
    (_append4, dict(eps=float("nan")), E_INVALID), (_append4, dict(kc=P + 4), E_INVALID), (_append4, dict(n=1 << 40), E_UNSUPPORTED),
    (_append32, dict(k=None), E_INVALID), (_append32, dict(hd=31), E_UNSUPPORTED), (_append32, dict(hd=130), E_UNSUPPORTED),
    (_append32, dict(lmax=0), E_INVALID), (_append32, dict(heads=0), E_INVALID), (_append32, dict(ld=1), E_INVALID),
    (_read, dict(rows=None), E_INVALID), (_read, dict(k=None, v=None), E_INVALID), (_read, dict(kc=None), E_INVALID),
    (_read, dict(hd=6), E_UNSUPPORTED), (_read, dict(lmax=2), E_UNSUPPORTED), (_read, dict(v=P + 8), E_INVALID),
    (_attn, dict(lens=None), E_INVALID), (_attn, dict(heads=5), E_INVALID), (_attn, dict(hd=256), E_UNSUPPORTED),
    (_attn, dict(t=-1), E_INVALID), (_attn, dict(ws=P + 4), E_INVALID), (_attn, dict(lmax=7), E_UNSUPPORTED),
    (_attn, dict(batch=1 << 40), E_UNSUPPORTED), (_attn, dict(scale=float("inf")), E_INVALID),
    (_sample, dict(u=None), E_INVALID), (_sample, dict(vocab=0), E_INVALID), (_sample, dict(vocab=(1 << 19) + 1), E_UNSUPPORTED),
    (_sample, dict(ld=9), E_INVALID), (_sample, dict(n=1 << 40), E_UNSUPPORTED),
])
def test_refusals(lib, call, changes, code):
    assert call(lib, **changes) == code
    assert lib.kb_last_error()


@pytest.mark.parametrize("call", [_append4, _read, _attn])
def test_the_longest_cache(lib, call):
    """positions are 32-bit numbers with room for a chunk behind the last"""
    assert call(lib, lmax=1 << 30) == 0
    assert call(lib, lmax=(1 << 30) + 4) == E_UNSUPPORTED and call(lib, lmax=(1 << 31) - 4) == E_UNSUPPORTED


def test_row_words(lib):
    assert [int(lib.kb_kv4_row_words(h)) for h in (-1, 0, 4, 8, 100, 128)] == [0, 0, 1, 1, 13, 16]


def test_native_module_declines_without_a_gpu():
    """host tensors, wrong kinds and wrong numbers of arguments are left to the Python layer, nothing is touched"""
    import torch

    from kore_b200 import _build, serving

    _build.build_module()
    nat = serving.native()
    z = torch.zeros
    i32, i64 = torch.int32, torch.int64
    held = tuple(z(s, dtype=i32) for s in ((1, 1, 4, 2), (1, 1, 4), (1, 1, 4, 2), (1, 1, 4)))
    assert nat.sample(z(2, 5), z(2), None, None, None, None, False, None) is None
    assert nat.sample(None, None, None, None, None, None, None, None) is None and nat.sample() is None
    assert nat.read(held, 16, z(3, dtype=i64), None, None) is None and nat.read(1, 16, z(3, dtype=i64), None, None) is None
    assert nat.attend(held, 16, z(1, 2, 16), z(1, dtype=i32), 0.0, None) is None
    for caches in (held, (z(1, 1, 4, 16), z(1, 1, 4, 16)), (1, 2), "ab"):
        assert nat.append(z(1, 64), z(1, dtype=i32), z(1, dtype=i64), z(4, 8), z(4, 8), caches, 16, 2, None, None, 1e-5, None) is None
    with pytest.raises(TypeError):
        nat.setup(1, 2)


def test_python_layer_refuses_host_tensors():
    import torch

    from kore_b200 import KoreError, _build, serving

    _build.build_module()
    with pytest.raises(KoreError) as e:
        serving.sample(torch.zeros(2, 5), torch.zeros(2))
    assert "logits" in e.value.message
    with pytest.raises(KoreError):
        serving.KV4Cache(1, 1, 0, 32)
    with pytest.raises(KoreError):
        serving.KV4Cache(1, 1, (1 << 30) + 1, 32)
    z = torch.zeros((1, 1, 4, 4), dtype=torch.int32)
    with pytest.raises(KoreError):
        serving.KV4Cache.from_planes(z, z, z, z, 32)
    with pytest.raises(KoreError) as e:
        serving.KV4Cache.from_planes(z, z, z, z, 30)
    assert "head_dim" in e.value.message
