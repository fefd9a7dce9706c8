"""Block-scaled 4-bit matrices for Python callers: descriptors and sizes.  The arithmetic is in
libb200const.so (b200c_mx_quantize, b200c_mx_dequantize, b200c_mx_matmul; formats and storage in include/b200const.h) and is called
through the backend: CudaBackend.mx_quantize / mx_dequantize / mx_matmul.  No counterpart in the reference, whose
narrowest weights are int4 with one scale per channel."""
import ctypes as C

from . import _cabi as A
from .const import raise_for


def sizes(fmt, rows, cols, layout=A.MX_SCALES_TILED):
    """(bytes between rows of codes, bytes of all codes, bytes of all scales) of a rows x cols matrix."""
    lib = A.load()
    ld, codes, scales = C.c_int64(), C.c_size_t(), C.c_size_t()
    raise_for(lib.b200c_mx_sizes(fmt, layout, rows, cols, C.byref(ld), C.byref(codes), C.byref(scales)), lib.b200c_last_error())
    return ld.value, codes.value, scales.value


class MxMatrix:
    """One matrix: its format and shape, and the device pointers of its codes, scales and (nvfp4) tensor scale.  The
    memory stays the caller's."""

    def __init__(self, fmt, rows, cols, codes, scales, tensor_scale=None, ld=None, layout=A.MX_SCALES_TILED):
        if ld is None:
            ld = sizes(fmt, rows, cols, layout)[0]
        self.c = A.b200c_mx_matrix(fmt, layout, rows, cols, ld, codes, scales, tensor_scale)
        self.ref = C.byref(self.c)

    @property
    def shape(self):
        return self.c.rows, self.c.cols

    def __repr__(self):
        name = {A.MXFP4: "mxfp4", A.NVFP4: "nvfp4"}[self.c.format]
        return f"MxMatrix({name}, {self.c.rows} x {self.c.cols}, {'tiled' if self.c.scale_layout else 'row'} scales)"
