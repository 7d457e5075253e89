"""The four-bit operators of the C ABI: `Kv4Cache` (a paged four-bit key/value cache and the attention over it) and `W4`
(a linear layer's weights in four bits). The stored format is described in include/tabicl_b200.h.

Buffers are device pointers (e.g. torch tensors' data_ptr()); `stream` is a cudaStream_t handle (None: the context's own
stream, 1: the legacy default stream). The caller keeps the buffers alive.
"""
import ctypes

F32, F16, BF16 = 0, 1, 2

_int, _i32, _i64, _size, _void, _float = (ctypes.c_int, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p,
                                          ctypes.c_float)
_REFUSED = ctypes.c_size_t(-1).value


class _Kv4(ctypes.Structure):
    _fields_ = [("pool", _void), ("pages", _i64), ("heads", _i32), ("width", _i32), ("page", _i32), ("group", _i32)]


class _Batch(ctypes.Structure):
    _fields_ = [("seqs", _i32), ("rows", _i32), ("max_rows", _i32), ("max_len", _i32), ("starts", _void), ("lens", _void),
                ("table", _void), ("table_stride", _i64)]


class _W4(ctypes.Structure):
    _fields_ = [("codes", _void), ("scales", _void), ("n", _i32), ("k", _i32), ("group", _i32)]


def signatures():
    p = ctypes.POINTER
    copy = [_void, p(_Kv4), _int, _int, _void, _void, _i64, _i64, _void, _i64, _i64, _void]
    return {
        "tcu_kv4_page_bytes": (_size, [_int, _int, _int, _int]),
        "tcu_kv4_store_device": (_int, copy),
        "tcu_kv4_load_device": (_int, copy),
        "tcu_kv4_attend_workspace": (_size, [_void, p(_Kv4), p(_Batch), _int, _int]),
        "tcu_kv4_attend_device": (_int, [_void, p(_Kv4), p(_Batch), _int, _int, _void, _i64, _i64, _void, _i64, _i64, _float,
                                         _int, _int, _void, _void, _size, _void]),
        "tcu_w4_code_bytes": (_size, [_int, _int]),
        "tcu_w4_scale_bytes": (_size, [_int, _int, _int]),
        "tcu_w4_pack_device": (_int, [_void, _int, _int, _int, _int, _void, _i64, _void, _void, _void]),
        "tcu_w4_linear_workspace": (_size, [_void, p(_W4), _int, _int]),
        "tcu_w4_linear_device": (_int, [_void, p(_W4), _int, _int, _void, _i64, _void, _i64, _void, _int, _void, _i64, _void,
                                        _size, _void]),
        "tcu_label_logprobs_device": (_int, [_void, _int, _void, _int, _int, _i64, _void, _int, _void, _void, _int, _void,
                                             _void, ctypes.c_double, _void]),
    }


_loaded = None


def _lib():
    """The library (kept here: a call's own time on the host is a few microseconds)."""
    global _loaded
    if _loaded is None:
        from . import lib
        _loaded = lib()
    return _loaded


class Kv4Cache:
    """A four-bit key/value cache in pages, over the caller's pool of `pages` * page_bytes() bytes."""

    def __init__(self, gpu, pool_ptr, pages, *, heads, width, page, group):
        self.gpu = gpu
        self._c = _Kv4(pool_ptr, pages, heads, width, page, group)

    @staticmethod
    def page_bytes(heads, width, page, group):
        """Bytes of one page; 0 when the sizes are not taken."""
        return _lib().tcu_kv4_page_bytes(heads, width, page, group)

    def store(self, dtype, tokens, slots_ptr, k_ptr, k_row, k_head, v_ptr, v_row, v_head, stream=None):
        """Quantise rows of keys and values ([heads][width] by row and head strides) into their slots (int64; negative:
        skipped)."""
        r = _lib().tcu_kv4_store_device(self.gpu._h, self._c, dtype, tokens, slots_ptr, k_ptr, k_row, k_head, v_ptr, v_row,
                                        v_head, stream)
        return r if r == 0 else self.gpu.check(r)

    def load(self, dtype, tokens, slots_ptr, k_ptr, k_row, k_head, v_ptr, v_row, v_head, stream=None):
        """The numbers that the slots' keys and values stand for (zeros for a negative slot)."""
        r = _lib().tcu_kv4_load_device(self.gpu._h, self._c, dtype, tokens, slots_ptr, k_ptr, k_row, k_head, v_ptr, v_row,
                                       v_head, stream)
        return r if r == 0 else self.gpu.check(r)

    @staticmethod
    def batch(seqs, max_rows, max_len, lens_ptr, table_ptr, table_stride, starts_ptr=None, rows=None):
        """What a step attends over: `seqs` sequences of lens[s] tokens on the pages table[s * table_stride + ...], with
        max_rows query rows each, or (starts) rows starts[s]..starts[s + 1] of `rows` in all."""
        return _Batch(seqs, seqs * max_rows if rows is None else rows, max_rows, max_len, starts_ptr, lens_ptr, table_ptr,
                      table_stride)

    def attend_workspace(self, batch, q_heads, dtype):
        """Bytes of working memory that `attend` needs for such a batch (zeroed before its first use)."""
        n = _lib().tcu_kv4_attend_workspace(self.gpu._h, self._c, batch, q_heads, dtype)
        if n == _REFUSED:
            self.gpu.check(-1)
        return n

    def attend(self, batch, dtype, q_heads, q_ptr, q_row, q_head, out_ptr, o_row, o_head, scale, causal=False, window=0,
               lse=None, work=None, work_bytes=0, stream=None):
        """Softmax attention of the batch's query rows; lse (optional): f32 [rows][q_heads]."""
        r = _lib().tcu_kv4_attend_device(self.gpu._h, self._c, batch, dtype, q_heads, q_ptr, q_row, q_head, out_ptr, o_row,
                                         o_head, scale, causal, window, lse, work, work_bytes, stream)
        return r if r == 0 else self.gpu.check(r)


class W4:
    """A weight matrix [n][k] in four bits, over the caller's buffers of code_bytes() and scale_bytes() bytes."""

    def __init__(self, gpu, n, k, group, codes_ptr, scales_ptr):
        self.gpu = gpu
        self._w = _W4(codes_ptr, scales_ptr, n, k, group)

    @staticmethod
    def code_bytes(n, k):
        return _lib().tcu_w4_code_bytes(n, k)

    @staticmethod
    def scale_bytes(n, k, group):
        return _lib().tcu_w4_scale_bytes(n, k, group)

    def pack(self, dtype, w_ptr, ldw, stream=None):
        """Quantise the matrix at w_ptr (row stride ldw) into the codes and scales."""
        w = self._w
        return self.gpu.check(_lib().tcu_w4_pack_device(self.gpu._h, dtype, w.n, w.k, w.group, w_ptr, ldw, w.codes, w.scales,
                                                        stream))

    def linear_workspace(self, rows, dtype):
        """Bytes of working memory that `linear` needs for so many rows (zeroed before its first use)."""
        n = _lib().tcu_w4_linear_workspace(self.gpu._h, self._w, rows, dtype)
        if n == _REFUSED:
            self.gpu.check(-1)
        return n

    def linear(self, dtype, rows, x_ptr, ldx, y_ptr, ldy, bias=None, act=0, residual=None, ldr=0, work=None, work_bytes=0,
               stream=None):
        """y = act(x W^T + bias) + residual; act 1 is GELU, the residual may be y itself."""
        r = _lib().tcu_w4_linear_device(self.gpu._h, self._w, dtype, rows, x_ptr, ldx, y_ptr, ldy, bias, act, residual, ldr, work,
                                        work_bytes, stream)
        return r if r == 0 else self.gpu.check(r)
