"""Rows that start between the boundaries of the kernels' vector loads and stores are refused, not read."""
import ctypes

import pytest
import torch

from helpers import make_engine, randn

pytestmark = pytest.mark.gpu


def _at(shape, floats, fill=0.0):
    """A contiguous f32 tensor that starts `floats` elements behind a 256-byte boundary."""
    n = 1
    for d in shape:
        n *= d
    return torch.full((n + 64,), fill, device="cuda")[floats:floats + n].view(shape)


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16", "f32"])
@pytest.mark.parametrize("heads", [(8, 2), (16, 2)])
def test_decode_rows(kv_dtype, heads):
    from oomllama_b200._lib import PACKED_STRIDE, OomAttnError
    eng = make_engine(*heads, [40], kv_dtype=kv_dtype)
    k = randn((40, 2, 128), 1).cuda()
    eng.kv_write(0, 0, k, k)
    shape = (1, heads[0], 128)
    good = randn(shape, 2).cuda()
    want = eng.decode(0, [0], good)

    def refused(f):
        with pytest.raises(OomAttnError) as e:
            f()
        assert e.value.code == 1

    for off in (1, 2, 3):
        q, out = _at(shape, off), _at(shape, off, 7.0)
        q.copy_(good)
        if off == 2 and kv_dtype == "bf16":  # its q is read by 8-byte loads
            assert torch.equal(eng.decode(0, [0], q), want)
        else:
            refused(lambda: eng.decode(0, [0], q))
            refused(lambda: eng.decode_packed(0, [0], q))
        refused(lambda: eng.decode(0, [0], good, out=out))
        refused(lambda: eng.decode_packed(0, [0], good, out=_at((1, heads[0], PACKED_STRIDE), off)))
        assert (out == 7).all()
    q = _at(shape, 4)
    q.copy_(good)
    assert torch.equal(eng.decode(0, [0], q, out=_at(shape, 8)), want)
    eng.sync()
    eng.close()


@pytest.mark.parametrize("kv_dtype", ["q4", "bf16", "f32"])
def test_static_scratch_pools(lib, kv_dtype):
    from oomllama_b200 import _lib
    code = {"f32": _lib.DTYPE_F32, "bf16": _lib.DTYPE_BF16, "q4": _lib.DTYPE_Q4}[kv_dtype]
    pool = torch.zeros(4 << 20, dtype=torch.uint8, device="cuda")
    bt, q, out = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), *(torch.zeros(1, 4, 128, device="cuda") for _ in "qo")
    err, arr = ctypes.create_string_buffer(256), lambda x: (ctypes.c_int32 * len(x))(*x)
    p = lambda t, off=0: ctypes.c_void_p(t.data_ptr() + off)  # noqa: E731
    v_at = _lib.Q4_CHUNK if kv_dtype == "q4" else 1 << 20
    for off in (4, 8):
        for k_off, v_off in ((off, v_at + off), (0, v_at + off)):
            assert lib.oomattn_decode_static_scratch(
                0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), code, p(pool, k_off), p(pool, v_off), 4, p(bt), 4,
                4, 1, ctypes.c_float(0.0), 1, arr([0]), arr([20]), p(q), p(out), None, err, 256) == 1, err.value
    torch.cuda.synchronize()


def test_fused_projection():
    from oomllama_b200._lib import OomAttnError
    H = 256
    eng = make_engine(2, 1, [40, 40], kv_dtype="bf16", hidden=H)
    x, wq, wk = randn((3, H), 1).cuda(), randn((256, H), 2).cuda(), randn((128, H), 3).cuda()
    odd = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)  # noqa: E731
    for args in ((odd(x), wq, wk, wk), (x, odd(wq), wk, wk), (x, wq, odd(wk), wk), (x, wq, wk, odd(wk))):
        with pytest.raises(OomAttnError) as e:
            eng.qkv_rope_append(0, [0], *args)
        assert e.value.code == 1
    assert eng.seq_len(0, 0) == 0
    eng.qkv_rope_append(0, [0], x, wq, wk, wk)
    eng.sync()
    assert eng.seq_len(0, 0) == 3
    eng.close()
