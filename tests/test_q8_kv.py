"""CPU: the int8 K/V cache's sizes, its parts in one allocation, and every refusal of its operators (they return
before anything is launched, so no device is needed)."""
import ctypes as C

import numpy as np
import pytest

from helpers import rng
from q8_kv_ref import Cache

INVALID, UNSUPPORTED, NULL_HANDLE, OK = 3, 7, 9, 0
AT = 1 << 20  # an aligned address that nothing reads


@pytest.mark.parametrize("sizes", [(1, 1, 1, 1, 1, 16), (2, 3, 5, 48, 500, 16), (8, 32, 32, 128, 2048, 64), (3, 1, 2, 200, 65, 128),
                                   (1, 1, 1, 256, 64, 64)])
def test_bytes_and_parts(tl, sizes):
    B, L, H, hs, S, block = sizes
    unit = max(64, block)
    slots, lanes = -(-S // unit) * unit, -(-hs // 16) * 16
    codes = -(-B * L * H * slots * lanes // 256) * 256
    scales = -(-B * L * H * slots // block * 4 // 256) * 256
    assert tl.lib().thallama_q8_kv_bytes(*sizes) == 2 * codes + 2 * scales
    c = tl.Q8KVCache()
    assert tl.lib().thallama_q8_kv_map(C.byref(c), AT, *sizes) == 0
    assert (c.k, c.v, c.ks, c.vs) == (AT, AT + codes, AT + 2 * codes, AT + 2 * codes + scales)
    assert (c.n_batches, c.n_layers, c.n_kv_heads, c.head_size, c.seq_len, c.block) == sizes


@pytest.mark.parametrize("sizes", [(0, 1, 1, 64, 64, 16), (1, 0, 1, 64, 64, 16), (1, 1, 0, 64, 64, 16), (1, 1, 1, 0, 64, 16),
                                   (1, 1, 1, 64, 0, 16), (1, 1, 1, 64, 64, 0), (1, 1, 1, 257, 64, 16), (1, 1, 1, 64, 64, 8),
                                   (1, 1, 1, 64, 64, 48), (1, 1, 1, 64, 64, 256), (-1, 1, 1, 64, 64, 16),
                                   (1, 1, 1, 64, 0x7fffffff, 16), (1, 1, 1, 64, 0x40000001, 16), (1 << 30, 1 << 30, 1 << 20, 64, 64, 16),
                                   (1, 1, 1 << 30, 64, 64, 16)])
def test_no_such_cache(tl, sizes):
    assert tl.lib().thallama_q8_kv_bytes(*sizes) == 0
    assert tl.lib().thallama_q8_kv_map(C.byref(tl.Q8KVCache()), AT, *sizes) == -1


def test_map_refuses_addresses(tl):
    sizes = (1, 1, 1, 64, 64, 16)
    assert tl.lib().thallama_q8_kv_map(None, AT, *sizes) == -1
    assert tl.lib().thallama_q8_kv_map(C.byref(tl.Q8KVCache()), None, *sizes) == -1
    assert tl.lib().thallama_q8_kv_map(C.byref(tl.Q8KVCache()), AT + 128, *sizes) == -1


GOOD = dict(gpu=0, B=2, L=3, H=4, hs=64, S=100, block=32, k=AT, v=AT, ks=AT, vs=AT, layer=1, nb=2, n=5, pos=AT, num=AT, x=AT, y=AT,
            stride=256, heads=8, ostride=512, handle=True, cache=True, work=AT, size=1 << 40)
BAD = [(dict(handle=False), NULL_HANDLE), (dict(cache=False), INVALID), (dict(gpu=-1), INVALID), (dict(layer=-1), INVALID),
       (dict(layer=3), INVALID), (dict(nb=3), INVALID), (dict(nb=-1), INVALID), (dict(n=-1), INVALID), (dict(pos=None), INVALID),
       (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(ks=None), INVALID), (dict(vs=None), INVALID), (dict(k=AT + 8), INVALID),
       (dict(v=AT + 1), INVALID), (dict(ks=AT + 2), INVALID), (dict(vs=AT + 1), INVALID), (dict(pos=AT + 1), INVALID),
       (dict(num=AT + 2), INVALID), (dict(hs=257), UNSUPPORTED), (dict(block=24), UNSUPPORTED), (dict(block=256), UNSUPPORTED),
       (dict(hs=0), INVALID), (dict(S=0), INVALID), (dict(block=0), INVALID), (dict(B=0), INVALID), (dict(L=-2), INVALID),
       (dict(H=-4), INVALID), (dict(B=1 << 30, L=1 << 30, H=1 << 20, nb=1), INVALID), (dict(nb=0), OK), (dict(n=0), OK),
       (dict(nb=0, pos=None, x=None, y=None), OK), (dict(x=AT + 2), INVALID), (dict(y=AT + 1), INVALID)]
BIG = dict(B=1 << 24, L=1, H=64, hs=256, S=16, block=16, nb=1 << 24, layer=0, n=16)  # more workgroups than a launch holds


def call(tl, op, **change):
    a = dict(GOOD, **change)
    h = C.byref(tl.Handle(a["gpu"], None, None)) if a["handle"] else None
    c = C.byref(tl.Q8KVCache.make(*(a[n] for n in ("B", "L", "H", "hs", "S", "block", "k", "v", "ks", "vs")))) if a["cache"] else None
    head = (h, c, a["layer"], a["nb"], a["n"], a["pos"], a["num"])
    if op == "attention":
        return tl.lib().thaDNN_q8_attention_batch(*head, a["heads"], a["x"], a["y"], a.get("qstride", 512), a["ostride"], a["work"], a["size"])
    return getattr(tl.lib(), f"thaDNN_q8_kv_{op}_batch")(*head, a["x"], a["y"], a["stride"])


@pytest.mark.parametrize("op", ["store", "load", "attention"])
@pytest.mark.parametrize("change,status", BAD, ids=[str(c) for c, _ in BAD])
def test_refusals(tl, op, change, status):
    assert call(tl, op, **change) == status


@pytest.mark.parametrize("op,change,status", [
    ("store", dict(x=None), INVALID), ("store", dict(y=None), INVALID), ("store", dict(stride=255), INVALID),
    ("store", dict(stride=-1), INVALID), ("load", dict(stride=255), INVALID), ("load", dict(x=None, y=None), OK),
    ("store", dict(BIG, stride=16384), UNSUPPORTED), ("load", dict(BIG, B=1 << 30, nb=1 << 30, H=1, hs=16, stride=16), UNSUPPORTED),
    ("attention", dict(x=None), INVALID), ("attention", dict(y=None), INVALID), ("attention", dict(qstride=511), INVALID),
    ("attention", dict(ostride=511), INVALID), ("attention", dict(heads=0), INVALID), ("attention", dict(heads=6), INVALID),
    ("attention", dict(heads=-4), INVALID), ("attention", dict(BIG, heads=64, qstride=16384, ostride=16384, n=1 << 20), UNSUPPORTED)])
def test_refusals_of_one(tl, op, change, status):
    assert call(tl, op, **change) == status


@pytest.mark.parametrize("op,change", [
    ("store", dict(B=1 << 25, nb=1 << 25, hs=256)), ("load", dict(B=1 << 23, nb=1 << 23, hs=16)),
    ("attention", dict(B=1 << 24, nb=1 << 24, hs=16)), ("attention", dict(B=1 << 23, nb=1 << 23, n=32, hs=16)), ("attention", dict(B=1 << 20, nb=1 << 20, H=1 << 20, heads=1 << 20, hs=1, n=1 << 30))])
def test_more_than_a_launch(tl, op, change):
    """A launch has less than 2^32 threads; rows and heads whose product leaves 64 bits count as more than that."""
    a = dict(dict(L=1, H=1, S=64, block=16, layer=0, n=1, heads=1), **change)
    assert call(tl, op, **dict(a, stride=1 << 20, qstride=1 << 20, ostride=1 << 20)) == UNSUPPORTED
    if op == "attention":
        cache = tl.Q8KVCache.make(*([a[n] for n in ("B", "L", "H", "hs", "S", "block")] + [AT] * 4))
        assert tl.lib().thaDNN_q8_attention_workspace(C.byref(cache), a["nb"], a["n"], a["heads"]) == 0


def test_workspace(tl):
    """One size serves every call of a cache: it does not shrink with fewer rows or sequences."""
    size = lambda **c: tl.lib().thaDNN_q8_attention_workspace(  # noqa: E731
        C.byref(tl.Q8KVCache.make(2, 1, 4, c.get("hs", 64), 100, c.get("block", 32), AT, AT, AT, AT)), c.get("nb", 2), c.get("n", 5), c.get("heads", 8))
    assert size() > 0 and size(nb=1, n=1, heads=4) == size() == size(n=1000)
    for bad in (dict(nb=3), dict(nb=0), dict(n=0), dict(heads=6), dict(heads=0), dict(hs=300), dict(block=20)):
        assert size(**bad) == 0, bad
    assert tl.lib().thaDNN_q8_attention_workspace(None, 1, 1, 4) == 0


@pytest.mark.parametrize("change", [dict(work=None), dict(work=AT + 4), dict(size=64)])
def test_attention_needs_its_workspace(tl, change):
    """Few rows over many keys are divided: the call wants the workspace, aligned and whole."""
    assert call(tl, "attention", **dict(dict(S=4000, n=1), **change)) == INVALID


def test_reference_scale_grows():
    """The oracle itself: a token of twice the size halves the earlier codes, a smaller one leaves them."""
    c = Cache(1, 1, 1, 2, 16, 16, rng(0))
    x = np.zeros((1, 1, 1, 2), np.float32)
    for pos, top in enumerate([1.0, 2.0, 0.5]):
        x[:] = top, -top
        c.store(0, [pos], [1], x, x)
    assert c.codes["k"][0, 0, 0, :3, :2].tolist() == [[64, -64], [127, -127], [32, -32]]
    assert c.scales["k"][0, 0, 0, 0] == np.float32(2) / np.float32(127)
