"""GPU: how near the attention over the int8 K/V cache comes to 64 bits, beside fp32 over the same codes.

Limits go by an fp32 softmax in numpy over what the codes stand for: the root mean square over a call's rows of
|got - exact| / |exact| (2-norms) is at most FACTOR times numpy's.  Both forms round each score to fp32 (1/2 ulp, or more
for a sum of hs products), each weight (the exponential's ulp) and each sum.  The kernel adds an integer's rounding to the
query, at most 2^-25 of 2 to 16 times its median component, and one to each weight: together no more than what numpy's own sum of hs
products and its division add, so twice numpy's is what is expected at most, and half as much again is for the few rows of a call."""
import numpy as np
import pytest

from helpers import rng
from q8_kv_ref import Cache
from test_q8_kv_gpu import Device, rows

pytestmark = pytest.mark.gpu

FACTOR = 3.0
FORMS = [(4, 2, 1), (3, 2, 40), (2, 130, 70)]  # B, H, rows: one row a sequence, few rows, rows that fill the card


def fp32(ref, pos, q, some):
    """An fp32 softmax over the codes' values, [B, some, heads, hs]."""
    k, v = ref.values("k", 0), ref.values("v", 0)
    out = np.zeros((q.shape[0], len(some)) + q.shape[2:], np.float32)
    mul = q.shape[2] // ref.H
    for b in range(q.shape[0]):
        for j, i in enumerate(some):
            T = pos[b] + i + 1
            for h in range(q.shape[2]):
                x = k[b, h // mul, :T] @ q[b, i, h] / np.float32(np.sqrt(ref.hs))
                e = np.exp(x - x.max())
                out[b, j, h] = e @ v[b, h // mul, :T] / e.sum(dtype=np.float32)
    return out


def off(got, want):
    """Root mean square over the rows of the relative 2-norm error."""
    d = np.linalg.norm(got.astype(np.float64) - want, axis=-1) / np.linalg.norm(want, axis=-1)
    return float(np.sqrt(np.mean(d ** 2)))


def held(gpu, handle, ref, pos, q, what):
    """The call's rows (some of them, where they are many) within FACTOR of fp32."""
    B, nt, heads, hs = q.shape
    dev = Device(gpu, handle, ref)
    got = dev.attend(0, pos, None, q).reshape(q.shape)
    some = sorted({0, nt // 2, nt - 1} if heads > 8 else set(range(0, nt, 5)) | {nt - 1})
    want, _ = ref.attend(0, pos, [nt] * B, nt, q, heads // ref.H, some)
    want = want[:, some]
    mine, plain = off(got[:, some], want), off(fp32(ref, pos, q, some), want)
    assert mine <= FACTOR * plain, f"{what}: {mine:.3g} off, fp32 {plain:.3g}"


@pytest.mark.parametrize("power", [0, 25, 30, 33, 36, -30, -36])
@pytest.mark.parametrize("B,H,nt", FORMS)
def test_scores_of_queries_and_keys_far_apart(gpu, handle, power, B, H, nt):
    """Scores of ordinary size from queries of 10^power and keys of 10^-power, from the smallest normal numbers on."""
    r = rng(nt + 50 + power)
    hs, S = 64, 300
    ref = Cache(B, 1, H, hs, S, 32, r)
    k, v = r.standard_normal((B, S, H, hs)), rows(r, B, S, H, hs)
    q = (r.standard_normal((B, nt, H, hs)) * 10.0 ** power).astype(np.float32)
    ref.store(0, [0] * B, [S] * B, (k * 10.0 ** -power).astype(np.float32), v)
    held(gpu, handle, ref, [S - nt - 7 * b for b in range(B)], q, f"10^{power}")
