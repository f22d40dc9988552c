"""CPU: the limit that the attention over the int8 K/V cache is held to (test_q8_attn_accuracy_gpu.py) passes a model of its
arithmetic, and fails that model with the lowest digit of the weights, or of the queries, left out."""
import numpy as np
import pytest

from helpers import rng
from q8_kv_ref import Cache
from test_q8_attn_accuracy_gpu import FACTOR, WEIGHTS, fp32, off
from test_q8_kv_gpu import rows

DIGITS = 0x7F7F7F


def held_in(n, bits):
    """Whole numbers of 24 bits, the lowest `24 - bits` left out."""
    step = 2.0 ** (24 - bits)
    return np.rint(n / step) * step


def model(ref, pos, q, q_bits, w_bits, step=64):
    """[B, rows, heads, hs]: queries and weights as integers of their row's and their step's largest, sums by steps."""
    kc, vc = (ref.codes[w][:, 0, :, :, :ref.hs].astype(np.float64) for w in "kv")
    sk, sv = (np.repeat(ref.scales[w][:, 0], ref.block, -1).astype(np.float64) for w in "kv")
    out = np.zeros(q.shape)
    mul = q.shape[2] // ref.H
    for b, i, h in np.ndindex(q.shape[:3]):
        T, g = pos[b] + i + 1, h // mul
        y = q[b, i, h].astype(np.float64)
        unit = 2.0 ** np.frexp(np.abs(y).max())[1] / DIGITS
        x = (kc[b, g, :T] @ held_in(np.rint(y / unit), q_bits) * unit * sk[b, g, :T] / np.sqrt(ref.hs)).astype(np.float32).astype(np.float64)
        w = np.exp(x - x.max())
        for t in range(0, T, step):
            of = w[t:t + step] * sv[b, g, t:min(t + step, T)]
            unit = 2.0 ** np.frexp(of.max())[1] / DIGITS
            out[b, i, h] += (held_in(np.rint(of / unit), w_bits) * unit) @ vc[b, g, t:min(t + step, T)]
        out[b, i, h] /= w.sum()
    return out


@pytest.mark.parametrize("hs,S", [(8, 301), (48, 301), (64, 300), (128, 500), (256, 301)])
def test_a_lost_digit_is_past_the_limit(hs, S):
    r = rng(hs)
    B, H, nt = 2, 3, 4
    ref = Cache(B, 1, H, hs, S, 32, r)
    ref.store(0, [0] * B, [S] * B, rows(r, B, S, H, hs), rows(r, B, S, H, hs))
    pos = [S - nt, S - nt - 20]
    q = r.standard_normal((B, nt, H, hs)).astype(np.float32)
    want, _ = ref.attend(0, pos, [nt] * B, nt, q, 1)
    limit = np.hypot(FACTOR * off(fp32(ref, pos, q, range(nt)), want), WEIGHTS)
    assert off(model(ref, pos, q, 24, 24), want) <= limit
    assert off(model(ref, pos, q, 24, 24, 256), want) <= limit
    for q_bits, w_bits in ((16, 24), (24, 16), (20, 24), (24, 20)):
        assert off(model(ref, pos, q, q_bits, w_bits), want) > 2 * limit, (q_bits, w_bits)
