"""Host-side checks of the KV cache and rope entry points that need no GPU: argument blocks of the
documented size, and refusals that come before any device call."""
import ctypes as C

import numpy as np

from rusty_engine_b200 import _lib


def desc(**kw):
    d = _lib.KvDesc()
    d.n_blocks, d.block_size, d.n_kv_heads, d.head_dim, d.code, d.device = 4, 16, 2, 64, 0, 0
    for k, v in kw.items():
        setattr(d, k, v)
    h = C.c_void_p()
    st = _lib.load().rmoe_kv_create(C.byref(d), C.byref(h))
    return st, _lib.load().rmoe_last_error().decode()


def test_argument_blocks_have_the_header_sizes():
    """A 64-bit C compiler's sizes of the structs in include/rmoe.h."""
    assert (_lib.ROPE_ARGS.size, _lib.KV_EXTEND_ARGS.size, _lib.KV_RELEASE_ARGS.size) == (152, 104, 64)
    assert (_lib.KV_APPEND_ARGS.size, _lib.KV_ATTEND_ARGS.size) == (160, 128)
    assert (C.sizeof(_lib.RopeDesc), C.sizeof(_lib.KvDesc)) == (72, 56)


def test_kv_create_refusals():
    I, U = _lib.RMOE_ERR_INVALID, _lib.RMOE_ERR_UNSUPPORTED
    for kw, want, word in ((dict(block_size=24), U, "block size"), (dict(head_dim=96), U, "head_dim"),
                           (dict(code=2), U, "code"), (dict(n_blocks=0), I, "blocks"), (dict(n_kv_heads=0), I, "heads"),
                           (dict(n_blocks=1 << 30), U, "2^31"), (dict(k=4096), I, "all of"),
                           (dict(k=4097, v=4096, k_scale=4096, v_scale=4096), I, "aligned"),
                           (dict(k=4096, v=4096, k_scale=4098, v_scale=4096), I, "aligned")):
        st, msg = desc(**kw)
        assert st == want and word in msg, (kw, st, msg)
    L = _lib.load()
    h = C.c_void_p()
    assert L.rmoe_kv_create(None, C.byref(h)) == I and L.rmoe_kv_create(C.byref(_lib.KvDesc()), None) == I


def test_rope_create_refusals():
    I = _lib.RMOE_ERR_INVALID
    L = _lib.load()
    ff = np.array([1.0, np.nan], dtype=np.float32)
    for kw in (dict(rot_dim=7), dict(rot_dim=0), dict(max_pos=0), dict(base=0.0), dict(base=float("inf")), dict(layout=2),
               dict(scaling=3), dict(scaling=1, factor=0.5), dict(scaling=2, factor=2.0, orig_ctx=0),
               dict(scaling=2, factor=float("nan"), orig_ctx=64), dict(mscale=float("nan")),
               dict(rot_dim=4, freq_factors=ff.ctypes.data)):
        d = _lib.RopeDesc()
        d.rot_dim, d.max_pos, d.base, d.factor = 8, 4, 1e4, 1.0
        for k, v in kw.items():
            setattr(d, k, v)
        h = C.c_void_p()
        assert L.rmoe_rope_create(C.byref(d), C.byref(h)) == I, kw
        assert not h.value


def test_null_handles_and_arguments():
    I, U = _lib.RMOE_ERR_INVALID, _lib.RMOE_ERR_UNSUPPORTED
    L = _lib.load()
    for st in (L.rmoe_rope_apply(None, None, None), L.rmoe_rope_status(None), L.rmoe_kv_status(None),
               L.rmoe_kv_append(None, None, None), L.rmoe_kv_read(None, None, 0, 0, None, None, None),
               L.rmoe_kv_attend(None, None, None), L.rmoe_kv_extend(None, None), L.rmoe_kv_release(None, None),
               L.rmoe_kv_buffers(None, None)):
        assert st == I
    L.rmoe_rope_destroy(None)
    L.rmoe_kv_destroy(None)
    # extend's and release's sizes are checked before their pointers
    assert L.rmoe_kv_extend(_lib.KV_EXTEND_ARGS.pack(*[0] * 10, 1, 4, 1, 24, 0, 0), None) == U
    assert L.rmoe_kv_extend(_lib.KV_EXTEND_ARGS.pack(*[0] * 10, 20000, 4, 1, 16, 0, 0), None) == U
    assert L.rmoe_kv_extend(_lib.KV_EXTEND_ARGS.pack(*[0] * 10, 1, 1 << 31, 1, 16, 0, 0), None) == U
    assert L.rmoe_kv_extend(_lib.KV_EXTEND_ARGS.pack(*[0] * 10, 1, 4, 1, 16, 0, 0), None) == I
    p = [4096] * 10
    p[8] = p[1] = 8192  # lens_out is lens
    assert L.rmoe_kv_extend(_lib.KV_EXTEND_ARGS.pack(*p, 1, 4, 1, 16, 0, 0), None) == I
    assert L.rmoe_kv_release(_lib.KV_RELEASE_ARGS.pack(*[0] * 6, 1, 4, 16, 0), None) == I
