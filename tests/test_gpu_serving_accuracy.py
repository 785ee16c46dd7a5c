"""Attention over the 4-bit cache: every position is read once, and results have the accuracy that the header states."""
import numpy as np
import pytest

from oracle import serving_ref as sr
from tests import cases
from tests.test_gpu_serving import env, filled_cache, planes_of  # noqa: F401

pytestmark = pytest.mark.gpu
f32 = np.float32

# sequences, query tokens, heads, KV heads, head_dim, capacity, lengths: whole and split ones, lengths next to the ends of tiles
# of 32 and of four warps' tiles, more sequences than a warp has lanes, more units than are split, prompts
SHAPES = [(1, 1, 4, 4, 100, 640, [577]), (4, 1, 8, 2, 128, 300, [299, 128, 33, 1]), (3, 1, 2, 2, 64, 640, [640, 97, 129]),
          (2, 5, 8, 2, 128, 1500, [1499, 700]), (2, 1, 7, 1, 104, 5000, [4999, 4097]), (2, 3, 4, 4, 68, 2000, [2000, 1025]),
          (40, 1, 4, 2, 64, 1500, [1500] + [33 * i + 1 for i in range(39)]), (3, 2, 4, 4, 64, 20000, [20000, 12801, 640]),
          (2, 300, 4, 2, 64, 520, [520, 301]), (1, 257, 6, 2, 36, 1100, [1100])]

# Unit-normal queries, keys and values.  Scores in units of log 2 come from sums of up to 8 steps of the matrix instruction, which
# lie below 16 (the codes count from a row's lowest value) and are cut off by half of 2^-19 a step: 2^-18 x 2 in the mean.
# If all of it went the way of the values it would move an output by ln 2 times that times the mean distance of the values from
# their mean, 0.8: 4.2e-6.  Queries and weights of 22 bits, the exponential's 2 units and the sums add 2^-21 each at most.
ACCURACY = 6e-6


@pytest.mark.parametrize("shape", SHAPES)
def test_attention_accuracy(env, shape):
    """one f16 term less in a query or a weight, or 32 positions less, would be seen (test_serving_accuracy_cpu.py)"""
    seqs, t, heads, kv, hd, lmax, lens = shape
    cache = filled_cache(env, seqs, kv, lmax, hd, 60)
    q = cases.gaussian(61, (seqs, t, heads, hd), 1.0)
    got = env.serving.attend(env.dev(q), cache, env.dev(np.array(lens, np.int32))).cpu().numpy()
    assert np.abs(got - sr.attention(q, *planes_of(cache), lens)).max() <= ACCURACY


@pytest.mark.parametrize("shape", SHAPES + [(1300, 1, 8, 8, 4, 700, [700, 671, 1] + [i % 9 for i in range(1297)]),
                                            (1, 1, 2, 1, 8, 100000, [99999]), (50, 1, 16, 16, 8, 2000, [40 * i for i in range(50)])])
def test_attention_reads_every_position_once(env, shape):
    """Queries of zero weigh all positions alike, and codes are whole numbers with a step of 1: sums are exact below 2^24 and an
    output is their mean, rounded once.  A position left out or read twice moves it by 0.5 / lens at least."""
    seqs, t, heads, kv, hd, lmax, lens = shape
    cache = filled_cache(env, seqs, kv, lmax, hd, 62)
    cache.v_steps.fill_(0x3f80)  # step 1, lo 0
    words = cache.v_codes.cpu().numpy().view(np.uint32)
    codes = ((words[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(*words.shape[:-1], -1)[..., :hd].astype(np.int64)
    sums = np.concatenate([np.zeros_like(codes[:, :, :1]), codes.cumsum(2)], 2)  # of the first n positions
    assert sums.max() < 2 ** 24
    got = env.serving.attend(env.torch.zeros((seqs, t, heads, hd), device="cuda"), cache, env.dev(np.array(lens, np.int32))).cpu().numpy()
    for b, length in enumerate(lens):
        seen = np.maximum(length - (t - 1) + np.arange(t), 0)
        mean = sums[b][:, seen] / np.maximum(seen, 1)[None, :, None]  # [kv, t, hd]
        want = mean.repeat(heads // kv, 0).transpose(1, 0, 2)
        assert (np.abs(got[b] - want) <= 2.0 ** -24 * want).all(), b
