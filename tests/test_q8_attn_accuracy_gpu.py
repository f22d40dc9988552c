"""GPU: how near the attention over the int8 K/V cache comes to 64 bits, beside fp32 over the same codes.

A limit has two parts, added as squares: what fp32 costs, and what the kernel's integers add.

fp32: an fp32 softmax in numpy over what the codes stand for; the root mean square over a call's rows of
|got - exact| / |exact| (2-norms), times FACTOR.  Both forms round each score to fp32 (half a step, or more for a sum of hs
products), each weight (the exponential's step) and each sum.  The kernel's query adds at most half of 2^-24 of 2 to 16
times its median component, no more than what a sum of hs products adds: twice numpy's is what is expected
at most, and half as much again is for the few rows of a call.

integers: a weight times its value block's scale is n 2^-23 of its step's largest w_t 2^e_t, and the scale at least half of
2^e_t: off by up to half of 2^-22 of the largest weight times scale, 2^-22 / sqrt(12) in the mean.  A step has up to 256
keys of about the same codes: sqrt(256) 2^-22 / sqrt(12) = 1.1e-6 of what the largest key itself adds to the row, and the
row is no smaller than that where the values are of one size; where it is smaller, the weights have more digits."""
import numpy as np
import pytest

from helpers import rng
from q8_kv_ref import Cache
from test_q8_kv_gpu import Device, rows

pytestmark = pytest.mark.gpu

FACTOR = 3.0
WEIGHTS = 16 * 2.0 ** -22 / 12 ** 0.5
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
    """The call's rows (some of them, where they are many) within the limit."""
    B, nt, heads, hs = q.shape
    dev = Device(gpu, handle, ref)
    got = dev.attend(0, pos, None, q).reshape(q.shape)
    some = sorted({0, nt // 2, nt - 1} if heads > 8 else set(range(0, nt, 5)) | {nt - 1})
    want, _ = ref.attend(0, pos, [nt] * B, nt, q, heads // ref.H, some)
    want = want[:, some]
    mine, plain = off(got[:, some], want), off(fp32(ref, pos, q, some), want)
    assert mine <= np.hypot(FACTOR * plain, WEIGHTS), f"{what}: {mine:.3g} off, fp32 {plain:.3g}"


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


@pytest.mark.parametrize("score,part,at", [(8, 0.05, [0]), (10, 0.01, [0]), (12, 0.01, [130]), (12, 0, [0]), (16, 0, [0]), (20, 0, [77]),
                                           (12, 0, [0, 1, 2, 3]), (12, 0, [0, 64, 128, 192, 300])])
@pytest.mark.parametrize("hs", [24, 64, 128, 160, 256])
@pytest.mark.parametrize("B,H,nt", FORMS)
def test_most_of_the_weight_on_keys_of_small_values(gpu, handle, score, part, at, hs, B, H, nt):
    """Every row looks at one key, or a few, far more than at the others (a model's first token), and these have small
    values or none: what is left of a row are the others, at weights down to 2^-30 of the largest."""
    r = rng(nt + hs)
    H = H if hs < 160 or H < 100 else 66
    S = 600 if H < 100 else 400
    k, v = r.standard_normal((B, S, H, hs)), r.standard_normal((B, S, H, hs))
    q = r.standard_normal((B, nt, H, hs))
    d = r.standard_normal((1, 1, H, hs))
    d /= np.linalg.norm(d, axis=-1, keepdims=True)
    q += (4 - (q * d).sum(-1, keepdims=True)) * d
    k -= (k * d).sum(-1, keepdims=True) * d
    k[:, at] = d * score * np.sqrt(hs) / 4
    v[:, at] *= part
    ref = Cache(B, 1, H, hs, S, 32, r)
    ref.store(0, [0] * B, [S] * B, k.astype(np.float32), v.astype(np.float32))
    held(gpu, handle, ref, [S - nt - 7 * b for b in range(B)], q.astype(np.float32), f"{score}, values times {part}")


@pytest.mark.parametrize("B,H,nt", FORMS[1:])
def test_a_row_of_further_digits_leaves_its_neighbours(gpu, handle, B, H, nt):
    """Rows whose weights need more digits do not change a bit of the rows beside them."""
    r = rng(nt)
    hs, S = 64, 300
    k, v = r.standard_normal((B, S, H, hs)), r.standard_normal((B, S, H, hs))
    q = r.standard_normal((B, nt, H, hs)).astype(np.float32)
    v[:, 5] = 0
    ref = Cache(B, 1, H, hs, S, 32, r)
    ref.store(0, [0] * B, [S] * B, k.astype(np.float32), v.astype(np.float32))
    dev = Device(gpu, handle, ref)
    pos = [S - nt] * B
    before = dev.attend(0, pos, None, q).reshape(q.shape)
    some = [1, 18, nt - 2]
    q[:, some] += (k[:, 5] / (k[:, 5] ** 2).sum(-1, keepdims=True) * 13 * np.sqrt(hs))[:, None].astype(np.float32)
    got = dev.attend(0, pos, None, q).reshape(q.shape)
    want, _ = ref.attend(0, pos, [nt] * B, nt, q, 1, some)
    plain = off(fp32(ref, pos, q, some), want[:, some])
    assert off(got[:, some], want[:, some]) <= np.hypot(FACTOR * plain, WEIGHTS)
    rest = [i for i in range(nt) if i not in some]
    np.testing.assert_array_equal(got[:, rest], before[:, rest])


@pytest.mark.parametrize("first,rest", [(1e-30, 1e-30), (1e30, 1e30), (1e-30, 1e-28), (1e-37, 1e30), (1e30, 1e-5)])
@pytest.mark.parametrize("B,H,nt", FORMS)
def test_values_of_any_size(gpu, handle, first, rest, B, H, nt):
    """Small and large values, and values whose size changes on the way, cost the weights no bits."""
    r = rng(nt + int(np.log10(first * rest)) + 100)
    hs, S = 64, 500
    ref = Cache(B, 1, H, hs, S, 32, r)
    k, v = rows(r, B, S, H, hs), rows(r, B, S, H, hs)
    v[:, :300] *= np.float32(first)
    v[:, 300:] *= np.float32(rest)
    q = r.standard_normal((B, nt, H, hs)).astype(np.float32)
    ref.store(0, [0] * B, [S] * B, k, v)
    held(gpu, handle, ref, [S - nt - 7 * b for b in range(B)], q, f"{first} then {rest}")


@pytest.mark.parametrize("size,count,keys", [(20, 1, 0), (50, 1, 0), (50, 1, 1), (50, 3, 0), (1000, 1, 0), (1000, 1, 0.02), (1e5, 1, 0), (1e6, 2, 0)])
@pytest.mark.parametrize("hs", [64, 128, 192, 256])
@pytest.mark.parametrize("B,H,nt", FORMS)
def test_queries_of_a_few_large_components(gpu, handle, size, count, keys, hs, B, H, nt):
    """Components far larger than the rest, where the keys have little or nothing, take none of the others' bits."""
    r = rng(nt + hs + count)
    H = H if hs < 160 or H < 100 else 66
    S = 300
    k, v = r.standard_normal((B, S, H, hs)), r.standard_normal((B, S, H, hs))
    q = r.standard_normal((B, nt, H, hs))
    large = r.choice(hs, count, replace=False)
    q[..., large] = size
    k[..., large] *= keys
    ref = Cache(B, 1, H, hs, S, 32, r)
    ref.store(0, [0] * B, [S] * B, k.astype(np.float32), v.astype(np.float32))
    held(gpu, handle, ref, [S - nt - 7 * b for b in range(B)], q.astype(np.float32), f"{count} of {size}, keys times {keys}")


@pytest.mark.parametrize("size", [200, 2e4])
@pytest.mark.parametrize("hs,large", [(8, [0, 1, 5]), (16, [0, 2, 3]), (16, [1, 3, 7]), (24, [0, 1, 2, 17]), (40, [0, 1, 2, 3, 4, 5, 6])])
@pytest.mark.parametrize("B,H,nt", FORMS)
def test_small_heads_of_large_components(gpu, handle, size, hs, large, B, H, nt):
    """The same where the large components are a good part of a small head's."""
    r = rng(nt + hs + len(large))
    S = 300
    k, v = r.standard_normal((B, S, H, hs)), r.standard_normal((B, S, H, hs))
    q = r.standard_normal((B, nt, H, hs))
    q[..., large] = size
    k[..., large] = 0
    ref = Cache(B, 1, H, hs, S, 32, r)
    ref.store(0, [0] * B, [S] * B, k.astype(np.float32), v.astype(np.float32))
    held(gpu, handle, ref, [S - nt - 7 * b for b in range(B)], q.astype(np.float32), f"{large} of {size}")


@pytest.mark.parametrize("B,H,nt", FORMS[1:])
def test_a_row_of_large_components_leaves_its_neighbours(gpu, handle, B, H, nt):
    """Rows whose queries need more digits do not change a bit of the rows beside them."""
    r = rng(nt + 1)
    hs, S = 128, 300
    k, v = r.standard_normal((B, S, H, hs)), r.standard_normal((B, S, H, hs))
    q = r.standard_normal((B, nt, H, hs)).astype(np.float32)
    k[..., 7] = 0
    ref = Cache(B, 1, H, hs, S, 32, r)
    ref.store(0, [0] * B, [S] * B, k.astype(np.float32), v.astype(np.float32))
    dev = Device(gpu, handle, ref)
    pos = [S - nt] * B
    before = dev.attend(0, pos, None, q).reshape(q.shape)
    some = [1, 18, nt - 2]
    q[:, some, :, 7] = 1e4
    got = dev.attend(0, pos, None, q).reshape(q.shape)
    rest = [i for i in range(nt) if i not in some]
    np.testing.assert_array_equal(got[:, rest], before[:, rest])
    assert off(got[:, some], before[:, some].astype(np.float64)) < 1e-5  # the keys have nothing there


@pytest.mark.parametrize("S,block", [(301, 32), (1400, 128)])
@pytest.mark.parametrize("mul", [1, 3])
@pytest.mark.parametrize("hs", [8, 40, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("B,H,nt", FORMS)
def test_ordinary_rows(gpu, handle, S, block, mul, hs, B, H, nt):
    """Rows of a normal distribution, whose tokens and channels differ in size, at every number of 64-dimension steps."""
    if H > 100:  # the card is full from fewer heads on where they are shared
        H = 130 // mul if hs < 160 else 66 // mul
        if S > 1000 and hs > 64:
            S = 700
    r = rng(hs + S + mul)
    ref = Cache(B, 1, H, hs, S, block, r)
    ref.store(0, [0] * B, [S] * B, rows(r, B, S, H, hs), rows(r, B, S, H, hs))
    q = r.standard_normal((B, nt, H * mul, hs)).astype(np.float32)
    held(gpu, handle, ref, [S - nt - 7 * b for b in range(B)], q, "ordinary")
