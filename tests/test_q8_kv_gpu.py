"""GPU: the int8 K/V cache and the attention over it (include/thaDNN/thaDNN_q8_kv.hpp) against tests/q8_kv_ref.py.

Codes and scales are compared bit for bit, with everything that a store may not touch; what is read back is one
rounded product, so bit for bit too.  Attention is held to the bound that q8_kv_ref.Cache.attend derives."""
import ctypes as C

import numpy as np
import pytest

from helpers import rng
from q8_kv_ref import Cache

pytestmark = pytest.mark.gpu


class Device:
    """A Cache's twin on the device, mapped into one allocation."""

    def __init__(self, gpu, handle, ref):
        self.gpu, self.lib, self.handle, self.ref = gpu, gpu.lib(), handle, ref
        self.size = self.lib.thallama_q8_kv_bytes(*ref.sizes())
        self.mem = gpu.DevBuf(self.size)
        self.c = gpu.Q8KVCache()
        assert self.lib.thallama_q8_kv_map(C.byref(self.c), self.mem.ptr, *ref.sizes()) == 0
        self.parts = {"k": self.c.k, "v": self.c.v, "ks": self.c.ks, "vs": self.c.vs}
        self.upload()

    def upload(self):
        for w in "kv":
            self.mem.upload(self.ref.memory(w), self.parts[w] - self.mem.ptr)
            self.mem.upload(self.ref.scales[w], self.parts[w + "s"] - self.mem.ptr)

    def check(self, what):
        """Every byte of the cache is what the reference has."""
        self.gpu.sync()
        for w in "kv":
            got = self.mem.download(np.int8, self.ref.codes[w].size, self.parts[w] - self.mem.ptr)
            s = self.mem.download(np.float32, self.ref.scales[w].size, self.parts[w + "s"] - self.mem.ptr)
            np.testing.assert_array_equal(s.reshape(self.ref.scales[w].shape), self.ref.scales[w], f"{what}: scales of {w}")
            bad = self.ref.of_memory(w, got) != self.ref.codes[w]
            bad[..., self.ref.hs:] = False  # the lanes behind a head's end hold anything
            assert not bad.any(), f"{what}: codes of {w} differ at {np.argwhere(bad)[:4].tolist()}"

    def ints(self, x):
        return None if x is None else self.gpu.DevBuf.from_array(np.asarray(x, np.int32))

    def store(self, layer, pos, n, k, v, pad=0, shift=0):
        """k, v [B, n_tokens, H, hs], rows `pad` floats longer than they need, `shift` floats behind an aligned address."""
        B, nt = k.shape[:2]
        row = self.ref.H * self.ref.hs
        bufs = []
        for x in (k, v):
            full = np.full((B, nt, row + pad), np.nan, np.float32)
            full[:, :, :row] = x.reshape(B, nt, row)
            bufs.append(self.gpu.DevBuf.from_array(np.concatenate([np.full(shift, np.nan, np.float32), full.ravel()])))
        p, m = self.ints(pos), self.ints(n)
        rc = self.lib.thaDNN_q8_kv_store_batch(C.byref(self.handle), C.byref(self.c), layer, B, nt, p.ptr, m and m.ptr,
                                               bufs[0].ptr + 4 * shift, bufs[1].ptr + 4 * shift, row + pad)
        assert rc == 0
        self.gpu.sync()

    def load(self, layer, pos, n, nt, pad=0, shift=0, only=None):
        B, row = len(pos), self.ref.H * self.ref.hs
        mark = np.full(shift + B * nt * (row + pad), -77.0, np.float32)
        bufs = {w: self.gpu.DevBuf.from_array(mark) for w in "kv"}
        p, m = self.ints(pos), self.ints(n)
        at = {w: bufs[w].ptr + 4 * shift if only in (None, w) else None for w in "kv"}
        rc = self.lib.thaDNN_q8_kv_load_batch(C.byref(self.handle), C.byref(self.c), layer, B, nt, p.ptr, m and m.ptr,
                                              at["k"], at["v"], row + pad)
        assert rc == 0
        self.gpu.sync()
        return {w: bufs[w].download()[shift:].reshape(B, nt, row + pad) for w in "kv"}

    def attend(self, layer, pos, n, q, pad=0, shift=0, handle=None):
        """q [B, n_tokens, heads, hs] -> [B, n_tokens, heads * hs + pad], -77 where nothing was written."""
        B, nt, heads, hs = q.shape
        row = heads * hs
        full = np.full((B, nt, row + pad), np.nan, np.float32)
        full[:, :, :row] = q.reshape(B, nt, row)
        dq = self.gpu.DevBuf.from_array(np.concatenate([np.full(shift, np.nan, np.float32), full.ravel()]))
        out = self.gpu.DevBuf.from_array(np.full(shift + full.size, -77.0, np.float32))
        size = self.lib.thaDNN_q8_attention_workspace(C.byref(self.c), B, nt, heads)
        work = self.gpu.DevBuf.from_array(np.zeros(max(size, 1), np.uint8))
        p, m = self.ints(pos), self.ints(n)
        rc = self.lib.thaDNN_q8_attention_batch(C.byref(handle or self.handle), C.byref(self.c), layer, B, nt, p.ptr, m and m.ptr,
                                                heads, dq.ptr + 4 * shift, out.ptr + 4 * shift, row + pad, row + pad, work.ptr, size)
        assert rc == 0
        self.gpu.sync()
        return out.download()[shift:].reshape(B, nt, row + pad)


def rows(r, B, n, H, hs):
    """Keys or values whose tokens and channels differ in size."""
    x = r.standard_normal((B, n, H, hs)) * r.uniform(0.3, 2, (1, 1, H, hs)) * (1 + 3 * r.random((B, n, H, 1)) ** 6)
    return x.astype(np.float32)


def filled(gpu, handle, r, B, L, H, hs, S, block, upto, layer):
    """A cache whose sequences hold `upto[b]` tokens of `layer`, filled by the reference."""
    ref = Cache(B, L, H, hs, S, block, r)
    n = max(max(upto), 1)
    ref.store(layer, [0] * B, list(upto), rows(r, B, n, H, hs), rows(r, B, n, H, hs))
    return ref, Device(gpu, handle, ref)


# ------------------------------------------------------------------------------------------------ store and load
STORES = [  # B, L, H, hs, S, block, pos, n, n_tokens, pad, shift
    (1, 1, 1, 1, 1, 16, [0], [1], 1, 0, 0),
    (1, 2, 12, 64, 1024, 32, [300], [1], 1, 0, 0),
    (2, 1, 3, 128, 300, 64, [63, 64], [1, 1], 1, 0, 0),
    (3, 2, 5, 48, 500, 16, [211, 0, 17], [77, 5, 0], 77, 0, 0),
    (2, 1, 2, 256, 300, 128, [0, 120], [300, 150], 300, 0, 0),
    (1, 1, 2, 128, 257, 128, [1], None, 256, 0, 0),
    (2, 1, 3, 7, 100, 32, [30, 3], [40, 64], 64, 0, 0),
    (2, 1, 3, 40, 100, 64, [50, 99], [50, 1], 50, 4, 4),
    (2, 1, 3, 40, 100, 64, [50, 98], [50, 1], 50, 3, 1),
    (2, 1, 2, 16, 90, 16, [-3, 80], [10, 30], 30, 0, 0),      # rows before the first and behind the last position
    (2, 1, 2, 16, 90, 16, [95, 2147483647], [3, 3], 3, 0, 0),  # nothing inside
    (2, 1, 2, 16, 90, 16, [4, 5], [-1, 99], 6, 0, 0),          # counts outside 0 .. n_tokens
    (2, 1, 2, 33, 90, 32, [-2147483648, 1], [3, 0], 3, 0, 0),
]


@pytest.mark.parametrize("case", STORES, ids=[str(c[:9]) for c in STORES])
def test_store(gpu, handle, case):
    B, L, H, hs, S, block, pos, n, nt, pad, shift = case
    r = rng(sum(case[:6]))
    layer = L - 1
    ref, dev = filled(gpu, handle, r, B, L, H, hs, S, block, [min(max(p, 0), S) for p in pos], layer)
    k, v = rows(r, B, nt, H, hs), rows(r, B, nt, H, hs)
    k[0, :, 0] *= 5  # scales that grow
    dev.store(layer, pos, n, k, v, pad, shift)
    ref.store(layer, pos, [nt] * B if n is None else n, k, v)
    dev.check("store")
    back = dev.load(layer, pos, n, nt, pad, shift)
    row = H * hs
    for w in "kv":
        want = np.full((B, nt, row + pad), -77.0, np.float32)
        for b in range(B):
            for i in range(min(max(nt if n is None else n[b], 0), nt)):
                if 0 <= pos[b] + i < S:
                    want[b, i, :row] = ref.values(w, layer)[b, :, pos[b] + i].reshape(row)
        np.testing.assert_array_equal(back[w], want, f"load {w}")


def test_load_one_of_two(gpu, handle):
    r = rng(3)
    ref, dev = filled(gpu, handle, r, 2, 1, 3, 48, 100, 16, [90, 33], 0)
    both = dev.load(0, [3, 0], [80, 33], 80)
    for w, other in (("k", "v"), ("v", "k")):
        one = dev.load(0, [3, 0], [80, 33], 80, only=w)
        np.testing.assert_array_equal(one[w], both[w])
        assert (one[other] == -77).all()


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_token_by_token(gpu, handle, block):
    """One token a call, of growing and shrinking size: every growth makes the earlier codes anew."""
    r = rng(block)
    ref = Cache(2, 1, 2, 24, 200, block, r)
    dev = Device(gpu, handle, ref)
    for t in range(140):
        k, v = rows(r, 2, 1, 2, 24) * np.float32(1.02 ** t), rows(r, 2, 1, 2, 24) * np.float32(0.98 ** t)
        pos = [t, max(0, t - 40)]  # the second sequence begins anew at 0 again and again
        ref.store(0, pos, [1, 1], k, v)
        dev.store(0, pos, None, k, v)
    dev.check("token by token")


def test_small_scales(gpu, handle):
    """Blocks of zeros, of values around the smallest normal float, of the largest, and a division by a scale far
    from 1, in the first call and behind it."""
    r = rng(9)
    for top in (0.0, 1e-45, 1e-38, 1.4e-36, 1.6e-36, 1e-31, 1e-29, 1e29, 1e31, 3e38):
        ref = Cache(1, 1, 1, 16, 64, 16, r)
        dev = Device(gpu, handle, ref)
        x = (r.uniform(-1, 1, (1, 20, 1, 16)) * top).astype(np.float32)
        y = x * np.float32(0.5)
        y[0, 0, 0, 0] = x[0, 3, 0, 3] = top
        for pos, a, b in (([0], x, y), ([20], y, x), ([40], -x, -y), ([10], y, y)):
            ref.store(0, pos, [20], a, b)
            dev.store(0, pos, None, a, b)
            dev.check(f"{top} at {pos}")


def test_halves_round_away(gpu, handle):
    """Quotients that end in a half go away from zero; the largest value is 127 steps."""
    ref = Cache(1, 1, 1, 16, 64, 16, rng(1))
    dev = Device(gpu, handle, ref)
    x = np.zeros((1, 16, 1, 16), np.float32)
    x[0, :, 0, 0] = 127
    x[0, :, 0, 1:9] = np.arange(8) + 0.5
    x[0, :, 0, 9:] = -(np.arange(7) * 16 + 0.5)
    ref.store(0, [0], [16], x, x)
    assert ref.codes["k"][0, 0, 0, 0, :16].tolist() == [127, 1, 2, 3, 4, 5, 6, 7, 8, -1, -17, -33, -49, -65, -81, -97]
    dev.store(0, [0], None, x, x)
    dev.check("halves")


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_not_finite(gpu, handle, bad):
    """A value that is not finite makes its block's scale NaN, only that block's, until the block begins anew."""
    r = rng(2)
    ref, dev = filled(gpu, handle, r, 1, 1, 2, 32, 96, 16, [40], 0)
    x = rows(r, 1, 30, 2, 32)
    x[0, 3, 1, 5] = bad
    ref.store(0, [40], [30], x, x)
    dev.store(0, [40], None, x, x)
    assert np.isnan(ref.scales["k"][0, 0, 1, 2]) and np.isfinite(ref.scales["k"][0, 0, 0, :4]).all()
    dev.check("not finite")
    y = rows(r, 1, 4, 2, 32)
    for pos in ([44], [32]):
        ref.store(0, pos, [4], y, y)
        dev.store(0, pos, None, y, y)
        dev.check(f"behind it at {pos}")
    assert np.isfinite(ref.scales["k"][0, 0, 1, 2])


# ------------------------------------------------------------------------------------------------------ attention
ATTENDS = [  # B, L, H, mul, hs, S, block, pos, n, n_tokens, pad, shift
    (1, 1, 1, 1, 1, 1, 16, [0], [1], 1, 0, 0),
    (1, 2, 12, 1, 64, 1024, 32, [300], [1], 1, 0, 0),
    (3, 1, 2, 1, 128, 700, 64, [0, 63, 699], None, 1, 0, 0),
    (4, 1, 2, 4, 128, 600, 128, [64, 65, 127, 599], None, 1, 0, 0),
    (2, 1, 2, 8, 256, 400, 16, [399, 256], None, 1, 0, 0),
    (2, 2, 3, 3, 48, 333, 16, [200, 332], None, 1, 0, 0),
    (1, 1, 1, 32, 64, 300, 32, [299], None, 1, 0, 0),
    (2, 1, 1, 1, 8, 5000, 64, [4999, 1234], None, 1, 0, 0),
    (2, 1, 2, 1, 192, 260, 64, [200, 20], None, 2, 0, 0),
    (2, 1, 3, 2, 40, 200, 32, [100, 0], [7, 3], 9, 0, 0),
    (2, 1, 3, 2, 40, 200, 32, [100, 0], [7, 3], 9, 8, 4),
    (2, 1, 3, 2, 41, 200, 32, [100, 0], [7, 3], 9, 3, 1),
    (1, 1, 2, 1, 128, 400, 64, [0], None, 400, 0, 0),
    (3, 1, 2, 2, 64, 500, 128, [300, 0, 17], [130, 77, 0], 130, 0, 0),
    (1, 1, 1, 5, 96, 300, 16, [37], None, 200, 0, 0),
    (2, 1, 1, 1, 16, 300, 16, [250, 0], None, 33, 0, 0),
    (2, 1, 1, 2, 256, 300, 128, [100, 3], None, 50, 0, 0),
    (2, 1, 2, 1, 32, 90, 16, [-3, 80], [10, 30], 30, 0, 0),       # rows that see no key
    (2, 1, 2, 1, 32, 90, 16, [-1, 90], None, 1, 0, 0),
    (2, 1, 2, 2, 32, 90, 16, [2147483647, -2147483648], None, 3, 0, 0),
    (2, 1, 2, 1, 32, 90, 16, [4, 5], [-1, 99], 6, 0, 0),
] + [  # rows enough to fill the card: a few hundred tiles of 64
    (16, 1, 16, 1, 64, 200, 32, [7 * b for b in range(16)], [66 - 4 * b for b in range(16)], 66, 0, 0),
    (32, 2, 4, 3, 48, 700, 16, [20 * b for b in range(32)], None, 30, 0, 0),
    (64, 1, 4, 3, 48, 700, 16, [10 * b for b in range(64)], [30 - b % 9 for b in range(64)], 30, 4, 4),
    (64, 1, 2, 8, 128, 300, 64, [4 * b for b in range(64)], [b % 18 for b in range(64)], 17, 0, 0),
    (32, 1, 8, 5, 130, 350, 128, [9 * b for b in range(32)], None, 13, 2, 1),
    (64, 1, 4, 1, 200, 330, 32, [260, 3] * 32, [70, 65] * 32, 70, 4, 4),
    (64, 1, 4, 1, 256, 70, 16, [0, -5, 69, 70] * 16, None, 65, 0, 0),
    (64, 1, 4, 2, 8, 90, 64, [80, -40, -100, 2147483647] * 16, None, 33, 0, 0),
    (1, 1, 2, 2, 128, 4300, 64, [100], None, 4160, 0, 0),
]


def hold(got, want, bound, what):
    """got is within the bound of want, untouched (-77) where want is NaN."""
    none = np.isnan(want)
    assert (got[none] == -77).all(), f"{what}: rows that are not the call's were written"
    off = np.abs(got - want)[~none]
    assert np.isfinite(off).all(), f"{what}: not finite"
    over = off > bound[~none]
    assert not over.any(), f"{what}: {over.sum()} of {over.size} off by up to {off.max():.3g} (bound there {bound[~none][off.argmax()]:.3g})"


@pytest.mark.parametrize("case", ATTENDS, ids=[str(c[:10]) for c in ATTENDS])
def test_attention(gpu, handle, case):
    B, L, H, mul, hs, S, block, pos, n, nt, pad, shift = case
    r = rng(sum(case[:7]))
    layer = L - 1
    counts = [nt] * B if n is None else n
    upto = [min(max(p + c, 0), S) for p, c in zip(pos, counts)]
    ref, dev = filled(gpu, handle, r, B, L, H, hs, S, block, upto, layer)
    some = range(nt) if nt < 1000 else sorted({0, 1, nt - 1, *r.integers(0, nt, 40).tolist()})
    q = (r.standard_normal((B, nt, H * mul, hs)) * r.uniform(0.2, 3, (B, nt, H * mul, 1))).astype(np.float32)
    got = dev.attend(layer, pos, n, q, pad, shift)
    want, bound = ref.attend(layer, pos, counts, nt, q, mul, some)
    assert (got[:, :, H * mul * hs:] == -77).all(), "written behind a row's end"
    hold(got[:, some, :H * mul * hs].reshape(want[:, some].shape), want[:, some], bound[:, some], "attention")
    for b in range(B):
        assert np.isfinite(got[b, :max(counts[b], 0), :H * mul * hs]).all() and (got[b, max(counts[b], 0):] == -77).all()
    dev.check("attention leaves the cache")


@pytest.mark.parametrize("H,nt", [(2, 1), (2, 40), (90, 70)])  # the last fills the card
def test_attention_values_of_very_different_size(gpu, handle, H, nt):
    """Value blocks a million times smaller than others keep their share where the large ones' weights vanish, and so
    do blocks of zeros in the sum of the weights."""
    r = rng(nt)
    B, hs, S, block = 3, 64, 600, 16
    ref = Cache(B, 1, H, hs, S, block, r)
    k, v = rows(r, B, S, H, hs) * np.float32(0.2), rows(r, B, S, H, hs)
    v[:, 100:300] *= np.float32(1e-6)
    v[:, 300:400] *= np.float32(1e-30)
    v[:, 480:] = 0
    v[1] *= np.float32(1e-5)
    v[2] *= np.float32(1e30)
    q = r.standard_normal((B, nt, H, hs)).astype(np.float32)
    k[:, 100:200] += 3 * q[:, -1][:, None]  # the small blocks are where the rows look
    ref.store(0, [0] * B, [S] * B, k, v)
    dev = Device(gpu, handle, ref)
    pos = [S - nt] * B
    got = dev.attend(0, pos, None, q).reshape(q.shape)
    some = [0, nt - 1]
    want, bound = ref.attend(0, pos, [nt] * B, nt, q, 1, some)
    hold(got[:, some], want[:, some], bound[:, some], "different sizes")
    # That bound goes by the largest value, far above what the last row gets: hold it to its own size.  A weight times
    # its value block's scale, w_t = p_t sv_t, is held as n_t / 0x7f7f7f of 2^M with max w >= 2^M / 2, so it is off by
    # at most half a step, 2^M 2^-24 (1 + 2^-7) <= 2^-22 max w, times a code of at most 127; beside that each term is off by
    # its weight's own error, 2 (E + 8u |x|) + 32u of attend's bound and T u for each sum, all under 2^-15 here.
    for b in range(B):
        x = ref.values("k", 0, np.float64)[b, :, :pos[b] + nt] @ q[b, -1].astype(np.float64)[:, :, None] / 8.0
        e = np.exp(x - x.max(1, keepdims=True))
        p = e / e.sum(1, keepdims=True)
        w = p * np.repeat(ref.scales["v"][b, 0].astype(np.float64), block, -1)[:, :pos[b] + nt, None]
        v = np.abs(ref.values("v", 0, np.float64)[b, :, :pos[b] + nt])
        lim = 2.0 ** -15 * (p * v).sum(1) + x.shape[1] * 2.0 ** -22 * 127 * w.max(1)
        assert (np.abs(got[b, -1] - want[b, -1]) <= lim).all(), b


@pytest.mark.parametrize("first,rest", [(0.0, 1.0), (0.0, 1e4), (1e-37, 1.0), (1e-30, 1e8), (1e30, 1.0)])
@pytest.mark.parametrize("H,nt", [(2, 1), (2, 40), (130, 70)])  # the last fills the card
def test_attention_values_that_grow_or_shrink(gpu, handle, first, rest, H, nt):
    """The first 200 values are zeros, tiny or huge beside the others: the sum of the weights stays whole when the
    value scales' exponent moves by up to 2^130 from one step to the next."""
    r = rng(nt)
    B, hs, S = 2, 64, 400
    ref = Cache(B, 1, H, hs, S, 32, r)
    k, v = rows(r, B, S, H, hs) * np.float32(0.3), rows(r, B, S, H, hs)
    v[:, :200] *= np.float32(first)
    v[:, 200:] *= np.float32(rest)
    ref.store(0, [0] * B, [S] * B, k, v)
    dev = Device(gpu, handle, ref)
    q = r.standard_normal((B, nt, H, hs)).astype(np.float32)
    some = [0, nt - 1]
    got = dev.attend(0, [S - nt] * B, None, q).reshape(q.shape)
    want, bound = ref.attend(0, [S - nt] * B, [nt] * B, nt, q, 1, some)
    hold(got[:, some], want[:, some], bound[:, some], f"values {first} then {rest}")


@pytest.mark.parametrize("first", [0.0, 1e-37, 1e-30])
@pytest.mark.parametrize("H,nt", [(2, 40), (130, 70)])  # the last fills the card
def test_attention_rows_that_end_before_larger_values(gpu, handle, first, H, nt):
    """Rows that see only zeros, or tiny values, beside rows of the same call that see larger ones in the keys behind: each
    row's sum of the weights goes by the values that it sees itself.  Every row's last key falls into the turn from one to
    the other, at a tile's first key and inside a tile."""
    r = rng(nt)
    B, hs, S, block = 2, 64, 400, 32
    ref = Cache(B, 1, H, hs, S, block, r)
    k, v = rows(r, B, S, H, hs) * np.float32(0.3), rows(r, B, S, H, hs)
    ends = [384 - nt // 2, 352 - nt // 2]
    for b in range(B):
        v[b, 100:ends[b] + nt // 2] *= np.float32(first)
    ref.store(0, [0] * B, [S] * B, k, v)
    dev = Device(gpu, handle, ref)
    q = r.standard_normal((B, nt, H, hs)).astype(np.float32)
    got = dev.attend(0, ends, None, q).reshape(q.shape)
    some = range(nt) if H < 100 else range(0, nt, 9)
    want, bound = ref.attend(0, ends, [nt] * B, nt, q, 1, some)
    hold(got[:, some], want[:, some], bound[:, some], f"values {first}")


@pytest.mark.parametrize("parts", [(256, 256, 256), (128, 128, 768)])
@pytest.mark.parametrize("H,nt", [(2, 1), (2, 40), (130, 70)])  # the last fills the card
def test_attention_scores_that_make_up_for_the_values(gpu, handle, parts, H, nt):
    """Values of 1e-10, then of 1e30 under scores that leave them nothing (-200), then of 1 under scores of 300: the sum of
    the weights leaves fp32's range beside the second part's values, and comes back with the third's."""
    r = rng(nt)
    B, hs, S = 2, 64, sum(parts)
    ref = Cache(B, 1, H, hs, S, 64, r)
    v = rows(r, B, S, H, hs) * np.repeat(np.float32([1e-10, 1e30, 1.0]), parts)[None, :, None, None]
    k = np.ones((B, S, H, hs), np.float32) * (np.repeat(np.float32([0, -200, 300]), parts) / 8)[None, :, None, None]
    ref.store(0, [0] * B, [S] * B, k, v)
    dev = Device(gpu, handle, ref)
    q = np.ones((B, nt, H, hs), np.float32)
    some = [0, nt - 1]
    for seen in (S, parts[0] + parts[1]):  # the third part's keys in sight, and not
        pos = [seen - nt] * B
        got = dev.attend(0, pos, None, q).reshape(q.shape)
        want, bound = ref.attend(0, pos, [nt] * B, nt, q, 1, some)
        far = 2.0 ** -64 * np.abs(v[:, :seen]).max()
        hold(got[:, some], want[:, some], bound[:, some] + far, f"{seen} keys")


def test_attention_scores_of_any_size(gpu, handle):
    """Scores far below anything a sum starts from (-1e33), and as far above.

    A score is known to 8u of its own size (q8_kv_ref.Cache.attend), u = 2^-24: 1e33 to 5e26, where 1 is a factor of e in
    its weight.  Every weight from 0 to 1 so lies within the bound, and what is left of it is that a row is some mean of
    the values: between the least and the largest, up to 400u of the largest for 100 weights held in 24 bits and their sums."""
    r = rng(1)
    ref = Cache(2, 1, 1, 64, 100, 16, r)
    k, v = np.ones((2, 100, 1, 64), np.float32), rows(r, 2, 100, 1, 64)
    ref.store(0, [0, 0], [100, 100], k, v)
    dev = Device(gpu, handle, ref)
    q = np.full((2, 1, 1, 64), 1e32, np.float32)
    q[0] *= -1
    got = dev.attend(0, [99, 99], None, q).reshape(2, 64)
    seen = ref.values("v", 0, np.float64)[:, 0, :100]
    lim = 400 * 2.0 ** -24 * np.abs(v).max()
    assert ((got >= seen.min(1) - lim) & (got <= seen.max(1) + lim)).all()
    assert (np.abs(got).max(1) > 0).all()  # a mean of nothing would be zeros


@pytest.mark.parametrize("nt", [1, 20])
def test_attention_sees_nothing_behind_its_position(gpu, handle, nt):
    """NaN scales and any codes behind the last key leave a row's result bit for bit as it was; a NaN block in sight
    makes the rows that see it NaN, and only those."""
    r = rng(nt + 5)
    B, H, mul, hs, S, block = 2, 2, 2, 48, 400, 16
    pos = [177, 64]
    ref, dev = filled(gpu, handle, r, B, 1, H, hs, S, block, [p + nt for p in pos], 0)
    q = r.standard_normal((B, nt, H * mul, hs)).astype(np.float32)
    before = dev.attend(0, pos, None, q)
    for w in "kv":
        for b in range(B):
            ref.codes[w][b, 0, :, pos[b] + nt:] = r.integers(-128, 128, ref.codes[w][b, 0, :, pos[b] + nt:].shape)
            ref.scales[w][b, 0, :, -(-(pos[b] + nt) // block):] = np.nan
    dev.upload()
    np.testing.assert_array_equal(dev.attend(0, pos, None, q), before)
    for w in "kv":
        kept = ref.scales[w].copy()
        ref.scales[w][0, 0, 1, 180 // block] = np.nan  # tokens 176 .. 191 of one head of one sequence
        dev.upload()
        got = dev.attend(0, pos, None, q).reshape(B, nt, H, mul, hs)
        assert np.isnan(got[0, :, 1]).all(), w
        got[0, :, 1] = before.reshape(got.shape)[0, :, 1]
        np.testing.assert_array_equal(got, before.reshape(got.shape), w)
        ref.scales[w][:] = kept
    if nt > 16:  # rows 0 .. 14 end before token 192, whose block is NaN now
        ref.scales["v"][0, 0, 0, 192 // block] = np.nan
        dev.upload()
        got = dev.attend(0, pos, None, q).reshape(B, nt, H, mul, hs)
        seen = np.arange(nt) + pos[0] >= 192
        assert np.isnan(got[0, seen, 0]).all()
        np.testing.assert_array_equal(got[0, ~seen], before.reshape(got.shape)[0, ~seen])


@pytest.mark.parametrize("B,H,mul", [(2, 2, 2), (64, 4, 4)])
@pytest.mark.parametrize("hs", [48, 128])
def test_attention_rows_before_a_bad_block(gpu, handle, B, H, mul, hs):
    """A NaN block in the middle of what a row tile sees leaves the tile's earlier rows as they were."""
    r = rng(B + hs)
    S, block, nt, pos = 100, 16, 20, 40
    ref, dev = filled(gpu, handle, r, B, 1, H, hs, S, block, [60] * B, 0)
    q = r.standard_normal((B, nt, H * mul, hs)).astype(np.float32)
    before = dev.attend(0, [pos] * B, None, q).reshape(B, nt, H, mul, hs)
    for w in "kv":
        kept = ref.scales[w].copy()
        ref.scales[w][:, 0, 1, 3] = np.nan  # tokens 48 .. 63 of one head
        dev.upload()
        got = dev.attend(0, [pos] * B, None, q).reshape(before.shape)
        assert np.isnan(got[:, 8:, 1]).all(), w
        got[:, 8:, 1] = before[:, 8:, 1]
        np.testing.assert_array_equal(got, before, w)
        ref.scales[w][:] = kept


@pytest.mark.parametrize("B,H,nt", [(2, 2, 1), (2, 2, 20), (64, 4, 20)])  # the last fills the card
def test_attention_queries_not_finite(gpu, handle, B, H, nt):
    """A query with a NaN or an infinity has a NaN result; the rows beside it keep theirs."""
    r = rng(nt)
    mul, hs, S = 4, 64, 200
    ref, dev = filled(gpu, handle, r, B, 1, H, hs, S, 32, [150] * B, 0)
    q = r.standard_normal((B, nt, H * mul, hs)).astype(np.float32)
    pos = [100 + 20 * (b & 1) for b in range(B)]
    before = dev.attend(0, pos, None, q).reshape(q.shape)
    q[0, 0, 3, 5] = np.nan
    q[1, nt - 1, 6, 63] = np.inf
    got = dev.attend(0, pos, None, q).reshape(q.shape)
    assert np.isnan(got[0, 0, 3]).all() and np.isnan(got[1, nt - 1, 6]).all()
    got[0, 0, 3], got[1, nt - 1, 6] = before[0, 0, 3], before[1, nt - 1, 6]
    np.testing.assert_array_equal(got, before)


@pytest.mark.parametrize("nt", [1, 20])
def test_attention_zero_and_large_queries(gpu, handle, nt):
    """A query of zeros takes the mean; scores in the hundreds pick one key; tiny queries and keys lose nothing."""
    r = rng(nt)
    B, H, hs, S = 4, 1, 64, 300
    ref = Cache(B, 1, H, hs, S, 64, r)
    k, v = rows(r, B, 250, H, hs), rows(r, B, 250, H, hs)
    q = r.standard_normal((B, nt, H, hs)).astype(np.float32)
    q[0] = 0
    q[1] *= 100
    q[2] *= np.float32(1e-30)
    k[2] *= np.float32(1e30)
    q[3] *= np.float32(1e25)
    k[3] *= np.float32(1e-25)
    ref.store(0, [0] * B, [250] * B, k, v)
    dev = Device(gpu, handle, ref)
    got = dev.attend(0, [200] * B, None, q).reshape(q.shape)
    want, bound = ref.attend(0, [200] * B, [nt] * B, nt, q, 1)
    hold(got, want, bound, "queries")


# ------------------------------------------------------------------------------------------------------- together
class Hip:
    """The runtime that libthallama.so is linked to: streams' captures as graphs."""

    def __init__(self):
        self.lib = C.CDLL("libamdhip64.so.7")

    def __call__(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, f"{name}: {rc}"

    def capture(self, stream, work):
        graph, run = C.c_void_p(), C.c_void_p()
        self("hipStreamBeginCapture", C.c_void_p(stream), 0)
        work()
        self("hipStreamEndCapture", C.c_void_p(stream), C.byref(graph))
        self("hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
        self("hipGraphDestroy", graph)
        return run


def test_prompt_then_tokens(gpu, handle):
    """A ragged batch of prompts and the tokens behind them, as a decoder would run them, against the reference, and
    the prompt's attention in one call against the same in pieces."""
    r = rng(77)
    B, L, H, mul, hs, S, block = 3, 2, 2, 4, 64, 256, 32
    ref = Cache(B, L, H, hs, S, block, r)
    dev = Device(gpu, handle, ref)
    pos, count, nt = [0, 0, 0], [60, 33, 1], 60
    for step in range(6):
        for layer in range(L):
            k, v = rows(r, B, nt, H, hs), rows(r, B, nt, H, hs)
            q = r.standard_normal((B, nt, H * mul, hs)).astype(np.float32)
            ref.store(layer, pos, count, k, v)
            dev.store(layer, pos, count, k, v)
            got = dev.attend(layer, pos, count, q).reshape(q.shape)
            want, bound = ref.attend(layer, pos, count, nt, q, mul)
            hold(got, want, bound, f"step {step} layer {layer}")
        dev.check(f"step {step}")
        pos = [p + c for p, c in zip(pos, count)]
        nt, count = 1, [1, 1, step % 2]


def test_captured_decode_step(gpu):
    """A decode step (store, then attention) captured once and replayed while the positions on the device move, each
    replay against the eager calls on a second cache, with other work on the stream between."""
    handle = gpu.new_handle()
    r = rng(5)
    B, H, mul, hs, S, block = 2, 2, 2, 64, 1500, 64
    ref, dev = filled(gpu, handle, r, B, 1, H, hs, S, block, [900, 40], 0)
    eager = Device(gpu, handle, ref)
    row = H * hs
    hip = Hip()
    size = dev.lib.thaDNN_q8_attention_workspace(C.byref(dev.c), B, 1, H * mul)
    pos = dev.ints([900, 40])
    k, v, q = gpu.DevBuf(B * row * 4), gpu.DevBuf(B * row * 4), gpu.DevBuf(B * row * mul * 4)
    out, work = gpu.DevBuf(B * row * mul * 4), gpu.DevBuf.from_array(np.zeros(size, np.uint8))

    def step():
        h, c = C.byref(handle), C.byref(dev.c)
        assert dev.lib.thaDNN_q8_kv_store_batch(h, c, 0, B, 1, pos.ptr, None, k.ptr, v.ptr, row) == 0
        assert dev.lib.thaDNN_q8_attention_batch(h, c, 0, B, 1, pos.ptr, None, H * mul, q.ptr, out.ptr, row * mul, row * mul,
                                                 work.ptr, size) == 0

    graph = hip.capture(handle.calc_stream, step)
    for t in range(6):
        at = [900 + t, 40 + 7 * t]
        x, y = rows(r, B, 1, H, hs), rows(r, B, 1, H, hs)
        z = r.standard_normal((B, 1, H * mul, hs)).astype(np.float32)
        for buf, a in ((k, x), (v, y), (q, z), (pos, np.asarray(at, np.int32))):
            buf.upload(a)
        gpu.sync()
        hip("hipGraphLaunch", graph, C.c_void_p(handle.calc_stream))
        gpu.sync()
        got = out.download().reshape(z.shape)
        ref.store(0, at, [1, 1], x, y)
        eager.store(0, at, None, x, y)
        np.testing.assert_array_equal(got, eager.attend(0, at, None, z).reshape(z.shape), f"replay {t}")
    dev.check("replays")
    eager.check("eager")
    hip("hipGraphExecDestroy", graph)
    assert gpu.lib().thablasDestroy(handle) == 0


def test_two_streams_at_once(gpu):
    """Attention on one cache from two streams at once, a workspace each."""
    r = rng(8)
    B, H, hs, S = 2, 4, 128, 1000
    handles = [gpu.new_handle() for _ in range(2)]
    ref, dev = filled(gpu, handles[0], r, B, 1, H, hs, S, 64, [1000, 700], 0)
    qs = [r.standard_normal((B, 1, H, hs)).astype(np.float32) for _ in range(2)]
    alone = [dev.attend(0, [999, 600], None, q) for q in qs]
    size = dev.lib.thaDNN_q8_attention_workspace(C.byref(dev.c), B, 1, H)
    pos = dev.ints([999, 600])
    bufs = [[gpu.DevBuf.from_array(q), gpu.DevBuf(q.nbytes), gpu.DevBuf.from_array(np.zeros(size, np.uint8))] for q in qs]
    gpu.sync()
    for _ in range(20):
        for h, (q, out, work) in zip(handles, bufs):
            assert dev.lib.thaDNN_q8_attention_batch(C.byref(h), C.byref(dev.c), 0, B, 1, pos.ptr, None, H, q.ptr, out.ptr, H * hs,
                                                     H * hs, work.ptr, size) == 0
    gpu.sync()
    for (_, out, _), want in zip(bufs, alone):
        np.testing.assert_array_equal(out.download(), want.ravel())
    for h in handles:
        assert dev.lib.thablasDestroy(h) == 0


def test_same_bits_again(gpu, handle):
    """The same call gives the same bits, however often it runs."""
    r = rng(12)
    ref, dev = filled(gpu, handle, r, 2, 1, 2, 128, 1500, 64, [1400, 1200], 0)
    for nt in (1, 70):
        q = r.standard_normal((2, nt, 8, 128)).astype(np.float32)
        first = dev.attend(0, [1400 - nt, 1100], None, q)
        for _ in range(5):
            np.testing.assert_array_equal(dev.attend(0, [1400 - nt, 1100], None, q), first)


def test_offsets_past_32_bits(gpu, handle):
    """A cache of over 4 GiB of key codes: its last sequence's last layer lies past 2^32."""
    B, L, H, hs, S, block = 5, 8, 8, 256, 65536, 128
    size = gpu.lib().thallama_q8_kv_bytes(B, L, H, hs, S, block)
    mem = gpu.DevBuf(size)
    c = gpu.Q8KVCache()
    assert gpu.lib().thallama_q8_kv_map(C.byref(c), mem.ptr, B, L, H, hs, S, block) == 0
    r = rng(4)
    nt = 200
    small = Cache(B, 1, H, hs, 256, block, r)
    k, v = rows(r, B, nt, H, hs), rows(r, B, nt, H, hs)
    n = [0] * (B - 1) + [nt]
    small.store(0, [0] * B, n, k, v)
    # the same rows at the very end of the last layer of the last sequence, their block's start on the same offset
    dev = object.__new__(Device)
    dev.gpu, dev.lib, dev.handle, dev.ref, dev.mem, dev.c = gpu, gpu.lib(), handle, small, mem, c
    dev.store(L - 1, [0] * (B - 1) + [S - 256], n, k, v)
    back = dev.load(L - 1, [0] * (B - 1) + [S - 256], n, nt)
    for w in "kv":
        np.testing.assert_array_equal(back[w][B - 1], small.values(w, 0)[B - 1, :, :nt].transpose(1, 0, 2).reshape(nt, -1))
        assert (back[w][:B - 1] == -77).all()


def test_fewer_sequences_than_the_cache_holds(gpu, handle):
    """A call works on the first sequences alone, in the order of the cache's."""
    r = rng(3)
    ref, dev = filled(gpu, handle, r, 4, 2, 2, 32, 150, 32, [60, 70, 80, 90], 1)
    x, y = rows(r, 2, 9, 2, 32), rows(r, 2, 9, 2, 32)
    ref.store(1, [60, 70], [9, 9], x, y)
    dev.store(1, [60, 70], None, x, y)
    dev.check("two of four")
    q = r.standard_normal((2, 9, 4, 32)).astype(np.float32)
    want, bound = ref.attend(1, [60, 70], [9, 9], 9, q, 2)
    hold(dev.attend(1, [60, 70], None, q).reshape(q.shape), want, bound, "two of four")
    back = dev.load(1, [0, 5], None, 40)
    for w in "kv":
        all_of = ref.values(w, 1)
        for b, first in enumerate([0, 5]):
            np.testing.assert_array_equal(back[w][b].reshape(40, 2, 32), all_of[b, :, first:first + 40].transpose(1, 0, 2))
