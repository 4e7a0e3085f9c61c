"""ctypes view of the paged 4-bit KV cache (include/ckb200_cache.h): argument types of its entry points.  Pointers are passed as integers
(`tensor.data_ptr()`), streams as handles."""
from __future__ import annotations

import ctypes as C

_P, _I, _L, _Z = C.c_void_p, C.c_int, C.c_longlong, C.c_size_t
_CACHE_API = {
    # function: (result, arguments)
    "ckb200_init": (_I, [_I]),
    "ckb200_last_error_message": (C.c_char_p, []),
    "ckb200_kv_q4_page_bytes": (_Z, [_I] * 3),
    "ckb200_kv_q4_row_offset": (_L, [_P] + [_I] * 7),
    "ckb200_dev_kv_cache_store_q4": (_I, [_P] * 4 + [_L] * 2 + [_P, _I, _P] + [_I] * 6 + [_P]),
    "ckb200_dev_kv_cache_load_q4": (_I, [_P] * 2 + [_L] * 2 + [_P] * 3 + [_I, _P] + [_I] * 6 + [_P]),
    "ckb200_dev_rope_kv_store_q4": (_I, [_P] * 7 + [_I, _P, _I, _P] + [_I] * 6 + [_P]),
    "ckb200_attention_q4cache_workspace_bytes": (_Z, [_I] * 5),
    "ckb200_dev_attention_q4cache": (_I, [_P, _L, _P, _P, _P, _L, _P, _I, _P] + [_I] * 8 + [_P, _Z, _P]),
    "ckb200_kv_pages_workspace_bytes": (_Z, [_I] * 3),
    "ckb200_dev_kv_pages_copy": (_I, [_P, _I, _L, _L, _P, _P, _I, _I, _P]),
    "ckb200_dev_kv_pages_resize": (_I, [_P, _I, _P, _P, _P, _I, _I, _I, _P, _I, _L, _L, _P, _P, _Z, _P]),
    "ckb200_dev_kv_pages_fork": (_I, [_P, _I, _P, _P, _P, _I, _I, _I, _P, _Z, _P]),
    "ckb200_dev_kv_pages_compact": (_I, [_P, _I, _P, _P, _I, _I, _I, _P, _I, _L, _L, _P, _P, _Z, _P]),
}


def bind_cache_api(lib):
    """Declare argument and result types of the paged cache's functions on a ctypes handle of libckb200.so."""
    for name, (res, args) in _CACHE_API.items():
        f = getattr(lib, name)
        f.restype, f.argtypes = res, args
