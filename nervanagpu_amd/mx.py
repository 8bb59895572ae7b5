"""
Block-scaled ("MX") matrices: 4 or 8 bits a value and one power of two for every
block of 32 values along one axis (the OCP microscaling formats MXFP4 and MXINT8).

    W4 = ng.mx_array(W)                        # (nOut, nIn), blocks along the inputs
    ng.mx_dot(W4, x, y, relu=True)             # fp16 activations
    x4 = ng.mx_quantize(x, ng.mx_empty(x.shape, axis=0))
    ng.mx_dot(W4, x4, y)                       # both operands in 4 bits

No counterpart in the reference, whose narrowest storage is fp16 with stochastic
rounding (nervanagpu/float_ew.py:182-201); the tensors are made and used like its
GPUTensors (nervanagpu/nervanagpu.py:30-466).
"""
import numpy as np

from . import _lib

MX_BLOCK = 32
_FORMATS = {"fp4": (_lib.NG_MX_FP4, 16), "int8": (_lib.NG_MX_INT8, 32)}


def code_pitch(fmt, depth):
    """bytes of codes of a line of `depth` values"""
    return -(-depth // MX_BLOCK) * _FORMATS[fmt][1]


def scale_pitch(depth):
    """bytes of scales of a line: one a block, rounded up to a multiple of 8"""
    blocks = -(-depth // MX_BLOCK)
    return -(-blocks // 8) * 8


class MXTensor(object):
    """
    A block-scaled matrix on the device.

    shape: (rows, cols) of the matrix it stands for
    fmt:   "fp4" (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) or "int8" (code / 64)
    axis:  the axis the blocks of 32 run along; a line is one run of that axis
    codes, scales: uint8 GPUTensors to use instead of new ones, of (lines,
           code_pitch) and (lines, scale_pitch); codes beyond the last value of a
           line must be zero
    rounding: non-zero: mx_quantize rounds stochastically into this tensor (right on
           average; int8 values above 127/64 of their block's power of two saturate)
    """

    def __init__(self, backend, shape, fmt="fp4", axis=1, codes=None, scales=None, rounding=0, name=None):
        if fmt not in _FORMATS:
            raise ValueError("unknown block-scaled format %r (fp4, int8)" % (fmt,))
        if axis not in (0, 1):
            raise ValueError("bad axis for an MXTensor")
        self.shape = tuple(int(extent) for extent in shape)
        assert len(self.shape) == 2 and min(self.shape) >= 0, "block-scaled tensors are matrices"
        assert max(self.shape) < 2 ** 31, "extents of block-scaled tensors stay below 2^31"
        self.backend, self.fmt, self.axis = backend, fmt, axis
        self.rounding, self.name = rounding, name
        self.size = self.shape[0] * self.shape[1]
        # lines and their length
        self.lines, self.depth = self.shape[1 - axis], self.shape[axis]
        dims = ((self.lines, code_pitch(fmt, self.depth)), (self.lines, scale_pitch(self.depth)))
        if codes is None and scales is None:
            codes, scales = (backend.empty(d, dtype=np.uint8) for d in dims)
        for given, d, what in ((codes, dims[0], "codes"), (scales, dims[1], "scales")):
            assert given is not None and given.dtype.type is np.uint8 and given.shape == d and given.is_contiguous, \
                "%s of this MXTensor are a contiguous uint8 tensor of %s" % (what, d)
            assert not self.size or given.ptr % 16 == 0, "%s must be 16-byte aligned" % what
        # fixed for the tensor's life, like a GPUTensor's memory
        self._codes, self._scales = codes, scales
        self.nbytes = codes.nbytes + scales.nbytes
        self._operand = _lib.MxOperand(self.fmt_code, 1, 0, codes.ptr if self.size else None, scales.ptr if self.size else None)

    def __str__(self):
        return "MXTensor(%s) name:%s shape:%s axis:%d rounding:%s" % (self.fmt, self.name, self.shape, self.axis, self.rounding)

    __repr__ = __str__

    def __len__(self):
        return self.shape[0]

    @property
    def fmt_code(self):
        return _FORMATS[self.fmt][0]

    @property
    def T(self):
        """the transposed matrix on the same memory"""
        return MXTensor(self.backend, self.shape[::-1], self.fmt, 1 - self.axis, self.codes, self.scales,
                        self.rounding, self.name)

    def set(self, ary):
        """convert a host array on the device; returns self"""
        ary = np.asarray(ary)
        assert ary.shape == self.shape
        dtype = np.float16 if ary.dtype == np.float16 else np.float32
        self.backend.mx_quantize(self.backend.array(ary, dtype=dtype), self)
        return self

    def get(self):
        """the values as a host array (fp32, which holds all of them)"""
        out = self.backend.empty(self.shape, dtype=np.float32)
        if self.size:
            self.backend.mx_dequantize(self, out)
        return out.get()

    @property
    def codes(self):
        return self._codes

    @property
    def scales(self):
        return self._scales

    def operand(self):
        """this tensor as an operand of ng_mx_gemm"""
        return self._operand
