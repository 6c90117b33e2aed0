"""ctypes binding of the C-ABI's calls on a cache held in 4 bits (include/zentorch_hip.h)."""
import ctypes

import zt_capi as C

_vp, _i64, _i32, _sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t


class KvCacheMxfp4(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scales", _vp), ("v_scales", _vp), ("pages", _i64), ("heads", _i64),
                ("page_size", _i64), ("head_dim", _i64), ("k_strides", _i64 * 3), ("v_strides", _i64 * 3),
                ("k_scale_strides", _i64 * 3), ("v_scale_strides", _i64 * 3)]


def lib():
    L = C.lib()
    pc, pi = ctypes.POINTER(KvCacheMxfp4), ctypes.POINTER(_i64)
    L.zt_rotary_cache_append_mxfp4.argtypes = [_vp, _i32, _i64, _i64, pi, _vp, pi, _vp, pi, _vp, _vp, _i64, _i64,
                                               _i64, _i32, _vp, pc, _vp, _vp]
    L.zt_cache_read_mxfp4.argtypes = [pc, _vp, _i64, _i32, _vp, _vp, _vp]
    L.zt_paged_attention_mxfp4.argtypes = [_vp, _i32, _i64, _i64, _i64, _i64, pc, _vp, _i64, _i64, _vp, _vp, _i64,
                                           _i32, _i64, ctypes.c_float, _vp, _vp, _sz, _vp]
    L.zt_paged_attention_mxfp4_workspace_size.argtypes = [_i64, _i64, _i32, pc, _i64, _i64, _i64]
    L.zt_paged_attention_mxfp4_workspace_size.restype = _sz
    return L
