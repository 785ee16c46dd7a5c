"""The bound of test_gpu_serving_accuracy.py tells real mistakes from rounding: planted here, in the restatement."""
import numpy as np
import pytest

from oracle import serving_ref as sr
from tests import cases
from tests.test_gpu_serving_accuracy import ACCURACY, SHAPES

SMALL = [s for s in SHAPES if max(s[6]) <= 5000]


def one_head(shape):
    """queries, keys and values of the first sequence's first head"""
    seqs, t, heads, kv, hd, lmax, lens = shape
    q = cases.gaussian(61, (seqs, t, heads, hd), 1.0)[0, -1, 0].astype(np.float64)
    k, v = (sr.values(*sr.quantise(cases.gaussian(60 + s, (seqs, kv, (lmax + 3) // 4 * 4, hd), 1.0)[0, 0, :lens[0]]), hd).astype(np.float64) for s in (0, 1))
    return q, k, v


def softmax_mean(s, v, weight=lambda p: p):
    p = weight(np.exp(s - s.max()))
    return p @ v / p.sum()


@pytest.mark.parametrize("shape", SMALL)
def test_planted_mistakes_exceed_the_bound(shape):
    q, k, v = one_head(shape)
    s = k @ q / np.sqrt(len(q))
    exact = softmax_mean(s, v)
    half = lambda x: x.astype(np.float16).astype(np.float64)
    one_term = softmax_mean(k @ half(q) / np.sqrt(len(q)), v)
    assert np.abs(one_term - exact).max() > ACCURACY
    assert np.abs(softmax_mean(s, v, half) - exact).max() > ACCURACY
    if len(v) <= 64:
        return
    for first in (0, 32, len(v) // 64 * 32, len(v) - 32):  # a tile left out
        rest = np.delete(np.arange(len(v)), np.arange(first, first + 32))
        assert np.abs(softmax_mean(s[rest], v[rest]) - exact).max() > 5 * ACCURACY
