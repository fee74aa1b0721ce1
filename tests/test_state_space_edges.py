"""State-space operators without a GPU: sizes of one."""
import ctypes

from scanscam_b200 import _native


# ---- one channel ----------------------------------------------------------------------------------------
def test_one_packed_channel_lies_either_way(native):
    """The stride of an axis of one channel says nothing: no layout of it is refused."""
    conv = _native.ShortConv(dtype=_native.F32, batch=1, channels=1, steps=10, width=4, sequences=2, offsets=0x1000,
                             x=_native.View(0x1000, (ctypes.c_int64 * 4)(10, 10, 1, 0)))
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_BAD_ARG
    assert b"weight is NULL" in native.ssb_last_error()
    conv.weight = 0x1000
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_BAD_ARG
    assert b"out is NULL" in native.ssb_last_error()
    grads = _native.ShortConvGrads(gout=conv.x, gx=conv.x)
    assert native.ssb_short_conv_bwd(ctypes.byref(conv), ctypes.byref(grads), None, 0, None) == _native.ERR_BAD_ARG
    assert b"gweight is NULL" in native.ssb_last_error()
    conv.channels = 2
    assert native.ssb_short_conv_fwd(ctypes.byref(conv), None) == _native.ERR_UNSUPPORTED
