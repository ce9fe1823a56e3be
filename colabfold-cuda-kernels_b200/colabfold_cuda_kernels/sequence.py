"""ctypes binding of the sequence operators: rotary positions, the paged cache in 8 bits and the attention over it.

Tensors are device pointers with strides in elements, so that it works beside any array library; a stream is its handle
(`torch.cuda.current_stream().cuda_stream`). The descriptors (Rows, Rotation, Cache, Batch) can be kept as long as the buffers they
point to; a call reads them before it returns and only enqueues work. What each field and argument means is in include/cck_b200.h.
A call that is refused raises ValueError (arguments, types, workspace) or RuntimeError (device, launch) with the library's message.

    cache = Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, page_tokens, heads, dim)
    batch = Batch(sequences, rows, max_new, max_len, table.shape[1], first.data_ptr(), lengths.data_ptr(), table.data_ptr())
    cache_append(stream, cache, batch, k_rows, v_rows, rotation, q_rows, q_rows)   # queries rotated in place
    cache_attention(stream, cache, batch, q_rows, out_rows, dim ** -0.5, ws, ws_bytes)
"""
import ctypes

import colabfold_cuda_kernels as _cck

__all__ = ["Rows", "Rotation", "Cache", "Batch", "rotary", "cache_append", "cache_attention", "cache_attention_workspace_bytes", "cache_bytes"]

DTYPES = {"bf16": 0, "f16": 1, "f32": 2}
_i32, _i64, _ptr = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


class Rows(ctypes.Structure):
    """A tensor [rows][heads][dim], the last dimension contiguous."""

    _fields_ = [("data", _ptr), ("row_stride", _i64), ("head_stride", _i64), ("dtype", _i32), ("heads", _i32)]

    def __init__(self, data, dtype, heads, row_stride, head_stride):
        super().__init__(data, row_stride, head_stride, DTYPES[dtype], heads)


class Rotation(ctypes.Structure):
    """Rotary positions: `sections` pairs for each axis, freq f32 [dims / 2], pos i32 [axes][rows]."""

    _fields_ = [("dims", _i32), ("axes", _i32), ("adjacent", _i32), ("section", _i32 * 4), ("freq", _ptr), ("pos", _ptr), ("pos_stride", _i64)]

    def __init__(self, dims, sections, freq, pos, pos_stride=0, adjacent=False):
        if len(sections) > 4:
            raise ValueError("a rotation has up to four axes")
        super().__init__(dims, len(sections), int(bool(adjacent)), (_i32 * 4)(*sections), freq, pos, pos_stride)


class Cache(ctypes.Structure):
    """Codes (e4m3, see the layout in the header) and scales (f32 [pages][heads]) of keys and values."""

    _fields_ = [("k", _ptr), ("v", _ptr), ("k_scale", _ptr), ("v_scale", _ptr), ("pages", _i32), ("page_tokens", _i32), ("heads", _i32), ("dim", _i32)]


class Batch(ctypes.Structure):
    """The sequences of a call: first i32 [sequences + 1], len i32 [sequences], table i32 [sequences][table_pages]."""

    _fields_ = [("sequences", _i32), ("rows", _i32), ("max_new", _i32), ("max_len", _i32), ("table_pages", _i32), ("first", _ptr), ("len", _ptr), ("table", _ptr),
                ("table_stride", _i64)]

    def __init__(self, sequences, rows, max_new, max_len, table_pages, first, len, table, table_stride=None):
        super().__init__(sequences, rows, max_new, max_len, table_pages, first, len, table, table_pages if table_stride is None else table_stride)


def cache_bytes(pages, page_tokens, heads, dim):
    """(bytes of the codes of the keys, and as many of the values; bytes of the scales of the keys, and as many of the values)."""
    return pages * page_tokens * heads * dim, 4 * pages * heads


def _load():
    lib = ctypes.CDLL(_cck.library_path("cache_attention", 100))
    lib.cck_last_error.restype = ctypes.c_char_p
    rows, rotation, cache, batch = (ctypes.POINTER(t) for t in (Rows, Rotation, Cache, Batch))
    lib.cck_rotary.argtypes = [_ptr, rotation, ctypes.c_int, ctypes.c_int, rows, rows, ctypes.c_int]
    lib.cck_cache_append.argtypes = [_ptr, cache, batch, rows, rows, rotation, rows, rows, _ptr]
    lib.cck_cache_attention.argtypes = [_ptr, cache, batch, rows, rows, _ptr, ctypes.c_float, ctypes.c_int, ctypes.c_int, _ptr, ctypes.c_size_t]
    lib.cck_cache_attention_workspace_bytes.argtypes = [cache, batch, ctypes.c_int]
    lib.cck_cache_attention_workspace_bytes.restype = ctypes.c_size_t
    return lib


_lib = _load()


def _check(rc):
    if rc:
        message = _lib.cck_last_error().decode()
        raise (RuntimeError if rc in (5, 6) else ValueError)(message)


def rotary(stream, rotation, rows, dim, x, y, inverse=False):
    """y = R(pos) x, or R(-pos) x with `inverse`: the gradient of the former."""
    _check(_lib.cck_rotary(stream, rotation, rows, dim, x, y, inverse))


def cache_append(stream, cache, batch, k, v, rotation=None, q=None, q_out=None, status=None):
    """The batch's rows of k and v into the cache, keys rotated; q rotated into q_out."""
    _check(_lib.cck_cache_append(stream, cache, batch, k, v, rotation, q, q_out, status))


def cache_attention_workspace_bytes(cache, batch, q_heads):
    return _lib.cck_cache_attention_workspace_bytes(cache, batch, q_heads)


def cache_attention(stream, cache, batch, q, out, softmax_scale, ws=None, ws_bytes=0, causal=True, window=0, lse=None):
    """out = softmax(softmax_scale q K^T) V for the batch's rows."""
    _check(_lib.cck_cache_attention(stream, cache, batch, q, out, lse, softmax_scale, causal, window, ws, ws_bytes))
