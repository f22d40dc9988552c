"""GPU: the workspace of the attention over the int8 K/V cache: zeroed as its header says, and left to calls of any shape."""
import ctypes as C

import numpy as np
import pytest

from helpers import rng
from test_q8_kv_gpu import Hip, filled, hold

pytestmark = pytest.mark.gpu


def test_memset_is_done_when_it_returns(gpu):
    """A stream that does not wait for the legacy one reads what thallama_memset has just written."""
    handle, hip, size = gpu.new_handle(), Hip(), 1 << 30
    buf, back = gpu.DevBuf(size), gpu.DevBuf(4096)
    for value in (0x11, 0x22, 0x33):
        assert gpu.lib().thallama_memset(buf.ptr, value, size) == 0
        hip("hipMemcpyAsync", C.c_void_p(back.ptr), C.c_void_p(buf.ptr + size - 4096), C.c_size_t(4096), 3, C.c_void_p(handle.calc_stream))
        hip("hipStreamSynchronize", C.c_void_p(handle.calc_stream))
        assert (back.download(np.uint8) == value).all(), hex(value)
    assert gpu.lib().thablasDestroy(handle) == 0


@pytest.mark.parametrize("how", ["thallama_memset", "hipMemsetAsync"])
def test_zeroed_as_documented(gpu, how):
    """Memory that held anything, zeroed in either of the documented ways, serves a call whose keys are divided."""
    handle, hip = gpu.new_handle(), Hip()
    r = rng(3)
    B, H, hs, S = 1, 4, 64, 3000
    ref, dev = filled(gpu, handle, r, B, 1, H, hs, S, 64, [S], 0)
    q = r.standard_normal((B, 1, H, hs)).astype(np.float32)
    want, bound = ref.attend(0, [S - 1], [1], 1, q, 1)
    size = dev.lib.thaDNN_q8_attention_workspace(C.byref(dev.c), B, 1, H)
    pos, dq = dev.ints([S - 1]), gpu.DevBuf.from_array(q)
    out = gpu.DevBuf.from_array(np.full(q.size, -77.0, np.float32))
    work = gpu.DevBuf.from_array(np.full(size, 0x5a, np.uint8))
    gpu.sync()
    if how == "thallama_memset":
        assert dev.lib.thallama_memset(work.ptr, 0, size) == 0
    else:
        hip("hipMemsetAsync", C.c_void_p(work.ptr), 0, C.c_size_t(size), C.c_void_p(handle.calc_stream))
    assert dev.lib.thaDNN_q8_attention_batch(C.byref(handle), C.byref(dev.c), 0, B, 1, pos.ptr, None, H, dq.ptr, out.ptr, H * hs, H * hs,
                                             work.ptr, size) == 0
    gpu.sync()
    hold(out.download().reshape(q.shape), want, bound, how)
    assert dev.lib.thablasDestroy(handle) == 0


def test_one_workspace_for_calls_of_any_shape(gpu, handle):
    """Calls of differing heads, rows and lengths, ragged and full, one after another on one workspace of the documented
    size: each agrees with the reference, and nothing behind the workspace is written."""
    r = rng(11)
    B, H, hs, S = 3, 4, 64, 5000
    ref, dev = filled(gpu, handle, r, B, 1, H, hs, S, 64, [S] * B, 0)
    size = dev.lib.thaDNN_q8_attention_workspace(C.byref(dev.c), 1, 1, H)
    guard = 1 << 16
    work = gpu.DevBuf(size + guard)
    work.upload(np.concatenate([np.zeros(size, np.uint8), np.full(guard, 0xA5, np.uint8)]))
    shapes = [(1, 1, 1, [4999]), (3, 5, 2, [4000, 17, 2500]), (2, 1, 8, [4999, 300]), (3, 70, 1, [4000, 4100, 0]), (1, 3, 1, [100]),
              (3, 1, 1, [4999, 4998, 64]), (2, 40, 4, [3000, 1]), (1, 1, 2, [4999]), (3, 300, 2, [1000, 0, 4700])]
    for nb, nt, mul, pos in shapes * 2:
        q = r.standard_normal((nb, nt, H * mul, hs)).astype(np.float32)
        p, dq = dev.ints(pos), gpu.DevBuf.from_array(q)
        out = gpu.DevBuf.from_array(np.full(q.size, -77.0, np.float32))
        assert dev.lib.thaDNN_q8_attention_batch(C.byref(handle), C.byref(dev.c), 0, nb, nt, p.ptr, None, H * mul, dq.ptr, out.ptr, H * mul * hs,
                                                 H * mul * hs, work.ptr, size) == 0
        gpu.sync()
        some = sorted({0, nt // 2, nt - 1})
        want, bound = ref.attend(0, pos, [nt] * nb, nt, q, mul, some)
        hold(out.download().reshape(q.shape)[:, some], want[:, some], bound[:, some], f"{nb} x {nt} x {mul}")
        assert (work.download(np.uint8, guard, size) == 0xA5).all()
