"""Attention over the 4-bit cache at the ends of its ranges and to the accuracy that its header states."""
import numpy as np
import pytest

from oracle import serving_ref as sr
from tests import cases
from tests.test_gpu_serving import check_attention, env  # noqa: F401

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
