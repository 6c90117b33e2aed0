"""ctypes binding of the paged-cache part of the C-ABI (include/zentorch_hip.h)."""
import ctypes

import zt_capi as C

_vp, _i64, _i32, _sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t


class KvCache(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("dtype", _i32), ("pages", _i64), ("heads", _i64),
                ("page_size", _i64), ("head_dim", _i64), ("k_strides", _i64 * 3),
                ("v_strides", _i64 * 3)]


def lib():
    L = C.lib()
    pc, pi = ctypes.POINTER(KvCache), ctypes.POINTER(_i64)
    L.zt_rotary_embedding.argtypes = [_vp, _i32, _i64, _i64, _i64, _i64, _i64, _vp, _vp, _i64, _i64,
                                      _i64, _i32, _vp, _vp]
    L.zt_rotary_cache_append.argtypes = [_vp, _i64, _i64, pi, _vp, pi, _vp, pi, _vp, _vp, _i64, _i64,
                                         _i64, _i32, _vp, pc, _vp, _vp]
    L.zt_paged_attention.argtypes = [_vp, _i64, _i64, _i64, _i64, pc, _vp, _i64, _i64, _vp, _vp, _i64,
                                     _i32, _i64, ctypes.c_float, _vp, _vp, _sz, _vp]
    L.zt_paged_attention_workspace_size.argtypes = [_i64, _i64, pc, _i64, _i64, _i64]
    L.zt_paged_attention_workspace_size.restype = _sz
    L.zt_cache_extend.argtypes = [_vp] * 4 + [_i64] * 5 + [_vp] * 6
    L.zt_cache_fork.argtypes = [_vp] * 4 + [_i64] * 4 + [_vp] * 5
    L.zt_cache_compact.argtypes = [_vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _sz, _vp]
    L.zt_cache_compact_workspace_size.argtypes = [_i64]
    L.zt_cache_compact_workspace_size.restype = _sz
    L.zt_cache_copy_pages.argtypes = [ctypes.POINTER(_vp), _i64, _i64, _i64, _i64, _vp, _i64, _vp]
    return L
