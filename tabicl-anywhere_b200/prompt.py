"""A prompt's operators of the C ABI: `Fp4` (a matrix in microscaled four-bit floating point, and products of two) and `Packed`
(attention of packed rows over keys and values as they are). The stored format is described in include/tabicl_b200.h.

Buffers are device pointers (e.g. torch tensors' data_ptr()); `stream` is a cudaStream_t handle (None: the context's own
stream, 1: the legacy default stream). The caller keeps the buffers alive.
"""
import ctypes

from .fourbit import _REFUSED, _float, _i32, _i64, _int, _lib, _size, _void

MX, NV = 0, 1


class _Fp4(ctypes.Structure):
    _fields_ = [("codes", _void), ("scales", _void), ("rows", _i32), ("k", _i32), ("format", _i32), ("unit", _float)]


class _Packed(ctypes.Structure):
    _fields_ = [("seqs", _i32), ("q_rows", _i32), ("k_rows", _i32), ("max_q", _i32), ("max_k", _i32), ("q_starts", _void),
                ("k_starts", _void)]


def signatures():
    m, b = ctypes.POINTER(_Fp4), ctypes.POINTER(_Packed)
    rows = [_void, _i64, _i64]
    return {
        "tcu_fp4_code_bytes": (_size, [_int, _int]),
        "tcu_fp4_scale_bytes": (_size, [_int, _int, _int]),
        "tcu_fp4_pack_device": (_int, [_void, m, _int, _void, _i64, _void]),
        "tcu_fp4_load_device": (_int, [_void, m, _int, _void, _i64, _void]),
        "tcu_fp4_linear_workspace": (_size, [_void, m, m, _int]),
        "tcu_fp4_linear_device": (_int, [_void, m, m, _int, _void, _i64, _void, _int, _void, _i64, _void, _size, _void]),
        "tcu_packed_attend_workspace": (_size, [_void, b, _int, _int, _int, _int]),
        "tcu_packed_attend_device": (_int, [_void, b, _int, _int, _int, _int, *rows, *rows, *rows, *rows, _float, _int, _int, _void, _void,
                                            _size, _void]),
    }


class Fp4:
    """A matrix [rows][k] in microscaled four-bit floating point (format MX or NV), over the caller's buffers of code_bytes()
    and scale_bytes() bytes. unit: what a scale of 1 times a number of 1 stands for (1 for MX)."""

    def __init__(self, gpu, rows, k, format, codes_ptr, scales_ptr, unit=1.0):
        self.gpu = gpu
        self._m = _Fp4(codes_ptr, scales_ptr, rows, k, format, unit)

    @staticmethod
    def code_bytes(rows, k):
        """Bytes of the codes; 0 when the sizes are not taken."""
        return _lib().tcu_fp4_code_bytes(rows, k)

    @staticmethod
    def scale_bytes(rows, k, format):
        """Bytes of the scales; 0 when the sizes are not taken."""
        return _lib().tcu_fp4_scale_bytes(rows, k, format)

    def pack(self, dtype, x_ptr, ldx, stream=None):
        """Quantise the rows at x_ptr (row stride ldx) into the codes and scales."""
        r = _lib().tcu_fp4_pack_device(self.gpu._h, self._m, dtype, x_ptr, ldx, stream)
        return r if r == 0 else self.gpu.check(r)

    def load(self, dtype, y_ptr, ldy, stream=None):
        """The numbers that the matrix stands for, into the rows at y_ptr (row stride ldy)."""
        r = _lib().tcu_fp4_load_device(self.gpu._h, self._m, dtype, y_ptr, ldy, stream)
        return r if r == 0 else self.gpu.check(r)

    def linear_workspace(self, x, dtype):
        """Bytes of working memory that `linear` needs for the rows of x (zeroed before its first use)."""
        n = _lib().tcu_fp4_linear_workspace(self.gpu._h, self._m, x._m, dtype)
        if n == _REFUSED:
            self.gpu.check(-1)
        return n

    def linear(self, x, dtype, y_ptr, ldy, bias=None, act=0, residual=None, ldr=0, work=None, work_bytes=0, stream=None):
        """y = act(x W^T + bias) + residual with this matrix as W, x another Fp4; act 1 is GELU, the residual may be y itself."""
        r = _lib().tcu_fp4_linear_device(self.gpu._h, self._m, x._m, dtype, y_ptr, ldy, bias, act, residual, ldr, work, work_bytes,
                                         stream)
        return r if r == 0 else self.gpu.check(r)


class Packed:
    """`seqs` sequences of different lengths, one behind the other: query rows q_starts[s]..q_starts[s + 1] of `q_rows` and keys and
    values k_starts[s]..k_starts[s + 1] of `k_rows` (int32 on the device; k_starts_ptr None: the queries' own), at most max_q and
    max_k each."""

    def __init__(self, gpu, seqs, q_rows, k_rows, max_q, max_k, q_starts_ptr, k_starts_ptr=None):
        self.gpu = gpu
        self._p = _Packed(seqs, q_rows, k_rows, max_q, max_k, q_starts_ptr, k_starts_ptr)

    def attend_workspace(self, dtype, q_heads, heads, width):
        """Bytes of working memory that `attend` needs (zeroed before its first use)."""
        n = _lib().tcu_packed_attend_workspace(self.gpu._h, self._p, dtype, q_heads, heads, width)
        if n == _REFUSED:
            self.gpu.check(-1)
        return n

    def attend(self, dtype, q_heads, heads, width, q_ptr, q_row, q_head, k_ptr, k_row, k_head, v_ptr, v_row, v_head, out_ptr, o_row, o_head,
               scale, causal=False, window=0, lse=None, work=None, work_bytes=0, stream=None):
        """Softmax attention of the query rows over their sequences' keys and values; lse (optional): f32 [q_rows][q_heads]."""
        r = _lib().tcu_packed_attend_device(self.gpu._h, self._p, dtype, q_heads, heads, width, q_ptr, q_row, q_head, k_ptr, k_row, k_head,
                                            v_ptr, v_row, v_head, out_ptr, o_row, o_head, scale, causal, window, lse, work, work_bytes,
                                            stream)
        return r if r == 0 else self.gpu.check(r)
