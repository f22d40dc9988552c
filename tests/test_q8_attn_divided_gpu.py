"""GPU: attention over the int8 K/V cache where a row tile's keys are divided among workgroups that have several tiles a wave, and in
caches past 4 GiB, against tests/q8_kv_ref.py."""
import ctypes as C

import numpy as np
import pytest

from helpers import rng
from q8_kv_ref import Cache
from test_q8_attn_accuracy_gpu import FACTOR, WEIGHTS, fp32, off
from test_q8_kv_gpu import Device, hold, rows

pytestmark = pytest.mark.gpu

# B, H, mul, hs, S, block, rows a sequence; a wave's tiles are its keys / 64 / (4 waves * workgroups a row tile)
DIVIDED = [
    (4, 8, 1, 32, 9000, 64, 1),     # 32 row tiles, 8 workgroups each: 4 to 5 tiles a wave
    (1, 8, 3, 128, 9000, 32, 11),   # 33 rows, three row tiles: 24 units, 10 workgroups each
    (2, 4, 2, 48, 12000, 128, 30),  # 60 rows, four row tiles, 8 workgroups
    (3, 5, 1, 200, 7000, 16, 1),    # 15 units, 17 workgroups
    (8, 8, 1, 16, 16500, 64, 1),    # one row tile each and long: twice the workgroups, 8 instead of 4
    (6, 8, 4, 64, 20600, 128, 1),   # the same, 10 instead of 5, and shared heads
    (2, 2, 1, 256, 3000, 64, 20),   # two row tiles, 12 workgroups with one tile a wave, at most
]


@pytest.mark.parametrize("case", DIVIDED, ids=[str(c) for c in DIVIDED])
def test_divided(gpu, handle, case):
    """Ragged rows at the ends of long contexts, down to a third of them and to nothing."""
    B, H, mul, hs, S, block, nt = case
    r = rng(sum(case))
    pos = [S - nt - (2 * S * b) // (3 * max(1, B - 1)) if B > 1 else S - nt - 1 for b in range(B)]
    if B > 3:
        pos[1] = 70
    ref = Cache(B, 1, H, hs, S, block, r)
    upto = [p + nt for p in pos]
    ref.store(0, [0] * B, upto, rows(r, B, S, H, hs), rows(r, B, S, H, hs))
    dev = Device(gpu, handle, ref)
    q = r.standard_normal((B, nt, H * mul, hs)).astype(np.float32)
    got = dev.attend(0, pos, None, q).reshape(q.shape)
    some = sorted({0, nt // 2, nt - 1})
    want, bound = ref.attend(0, pos, [nt] * B, nt, q, mul, some)
    hold(got[:, some], want[:, some], bound[:, some], "divided")
    mine, plain = off(got[:, some], want[:, some]), off(fp32(ref, pos, q, some), want[:, some])
    assert mine <= np.hypot(FACTOR * plain, WEIGHTS), f"{mine:.3g} off, fp32 {plain:.3g}"


@pytest.mark.parametrize("mul,nt", [(1, 1), (2, 9), (8, 56)])  # the last has row tiles of 64 enough to fill the card
def test_offsets_past_32_bits(gpu, handle, mul, nt):
    """The last sequence's last layer of a cache of over 4 GiB of codes each begins past 2^32."""
    B, L, H, hs, S, block = 5, 8, 8, 256, 65536, 128
    size = gpu.lib().thallama_q8_kv_bytes(B, L, H, hs, S, block)
    mem = gpu.DevBuf(size)
    c = gpu.Q8KVCache()
    assert gpu.lib().thallama_q8_kv_map(C.byref(c), mem.ptr, B, L, H, hs, S, block) == 0
    r = rng(mul)
    T = 230
    small = Cache(B, 1, H, hs, 256, block, r)
    k, v = rows(r, B, T, H, hs), rows(r, B, T, H, hs)
    n = [0] * (B - 1) + [T]
    small.store(0, [0] * B, n, k, v)
    dev = object.__new__(Device)
    dev.gpu, dev.lib, dev.handle, dev.ref, dev.mem, dev.c = gpu, gpu.lib(), handle, small, mem, c
    dev.store(L - 1, [0] * B, n, k, v)
    q = r.standard_normal((B, nt, H * mul, hs)).astype(np.float32)
    pos, count = [0] * (B - 1) + [T - nt], [0] * (B - 1) + [nt]
    got = dev.attend(L - 1, pos, count, q).reshape(q.shape)
    some = sorted({0, nt // 2, nt - 1})
    want, bound = small.attend(0, pos, count, nt, q, mul, some)
    hold(got[:, some], want[:, some], bound[:, some], "past 2^32")
    assert (got[:B - 1] == -77).all() and np.isfinite(got[B - 1]).all()
