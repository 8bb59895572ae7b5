"""
NervanaGPU / GPUTensor / OpTreeNode: the Python surface of the reference
(nervanagpu/nervanagpu.py:30-1321) on top of the HIP shared library.

Same class names, methods, argument order, defaults and return values as the
reference so that callers are drop-in; pycuda is replaced by the ctypes binding
in `_lib`, the cubin loaders by compiled-in entry points, and the clock-seeded
random pool by a counter-based stream (`seed`, launch counter) so stochastic
rounding is reproducible.
"""
import ctypes
import os
import sys
from ctypes import c_void_p

import numpy as np

from . import _lib
from .mx import MXTensor
from .float_ew import call_compensated_sum, call_compound_kernel

_none_slice = slice(None, None, None)

_DTYPE_CODE = {np.dtype(np.float16): _lib.NG_F16, np.dtype(np.float32): _lib.NG_F32,
               np.dtype(np.uint8): _lib.NG_U8, np.dtype(np.int8): _lib.NG_I8}


_FLOATS = (np.float16, np.float32)
_ACT_CODE = {"relu": 0, "sig": 1, "tanh": 2, "silu": 3, "gelu": 4}


def _contiguous_strides(shape):
    """Element (not byte) strides of a row-major array (nervanagpu.py:1323-1331)."""
    if shape:
        strides = [1]
        for s in shape[:0:-1]:
            strides.append(strides[-1] * s)
        return tuple(strides[::-1])
    return ()


class GPUTensor(object):
    """Row-major strided view of device memory (nervanagpu/nervanagpu.py:30-466)."""

    def __init__(self, backend, shape,
                 dtype=np.float16,
                 allocator=_lib.mem_alloc,
                 base=None,
                 gpudata=None,
                 strides=None,
                 take_array=None,
                 is_trans=False,
                 name=None,
                 rounding=0):

        assert dtype in (np.float16, np.float32, np.uint8, np.int8, np.uint16, np.int16, np.uint32, np.int32)
        # an integer stands for a one-dimensional shape
        if isinstance(shape, (int, np.integer)):
            shape = (shape,)
        self.shape = tuple(int(extent) for extent in shape)
        self.size = 1
        for extent in self.shape:
            self.size *= extent
        self.dtype = np.dtype(dtype)
        self.nbytes = self.size * self.dtype.itemsize
        # row-major unless a view says otherwise; strides count elements, not bytes
        self.strides = _contiguous_strides(self.shape) if strides is None else tuple(int(s) for s in strides)

        # where the memory comes from: a fresh allocation, or (views) the
        # allocation of `base` addressed through `gpudata`
        self.backend, self.allocator, self.base = backend, allocator, base
        if gpudata is not None:
            self.gpudata = gpudata
        else:
            assert base is None
            self.gpudata = allocator(self.nbytes) if self.size else None

        # view / expression attributes
        self.take_array = take_array      # (int32 index tensor, axis) of a lazy gather
        self.is_trans = is_trans
        self.name = name
        self.rounding = rounding          # mantissa bits of stochastic stores, 0 = nearest
        self.kahan_count = self.kahan_reset = 0

    def __str__(self):
        return ("Array(0x%x) name:%s dtype:%s shape:%s strides:%s "
                " is_trans:%s" % (int(self.gpudata) if self.gpudata is not None else 0, self.name,
                                  self.dtype, self.shape, self.strides, self.is_trans))

    def __repr__(self):
        return self.__str__()

    def __int__(self):
        return int(self.gpudata)

    # tensors are dictionary keys by identity; == builds an expression node
    __hash__ = object.__hash__

    @property
    def ptr(self):
        return int(self.gpudata)

    def __len__(self):
        """Return the size of the leading dimension of self."""
        if len(self.shape):
            return self.shape[0]
        return 0

    @property
    def is_contiguous(self):
        return not self.take_array and self.strides == _contiguous_strides(self.shape)

    def set(self, ary):
        """copy a contiguous host array to the device; returns self"""
        assert ary.size == self.size
        assert self.is_contiguous, "Array in set() must be contiguous"
        if ary.dtype != self.dtype:
            ary = ary.astype(self.dtype)
        ary = np.ascontiguousarray(ary)
        if self.size:
            _lib.memcpy_htod(self.gpudata, ary, self.backend.stream)
        return self

    def get(self, stream=None):
        """copy the device array to a new host numpy array"""
        assert self.is_contiguous, "Array in get() must be contiguous"
        ary = np.empty(self.shape, self.dtype)
        if self.size:
            _lib.memcpy_dtoh(ary, self.gpudata, stream if stream is not None else self.backend.stream)
        return ary

    def asnumpyarray(self):
        """alias of get()"""
        return self.get()

    def asbuffer(self):
        """host copy of the raw bytes (the device pointer is not host addressable)"""
        return self.get().tobytes()

    def take(self, indices, axis, out=None):
        """rows (axis 0) or columns (axis 1) selected by an int32 index vector, as
        a lazy view; with `out` the gather is executed into it"""
        picked = self[:, indices] if axis == 1 else self[indices, :]
        return out._assign(picked) if out else picked

    def _view(self, shape, strides, byte_offset=0, **changes):
        """a tensor of the same class on the same allocation"""
        fields = dict(backend=self.backend, shape=tuple(shape), dtype=self.dtype, allocator=self.allocator,
                      base=self, gpudata=self.gpudata, strides=tuple(strides), name=self.name,
                      rounding=self.rounding)
        if byte_offset:
            fields["gpudata"] = (int(self.gpudata) if self.gpudata is not None else 0) + byte_offset
        fields.update(changes)
        return self.__class__(**fields)

    def _index_vector(self, entry):
        """the device int32 vector behind a fancy-index entry"""
        if isinstance(entry, (list, tuple)):
            entry = np.array(entry, dtype=np.int32)
        if isinstance(entry, np.ndarray):
            entry = self.__class__(self.backend, entry.shape, dtype=np.int32).set(entry)
        if max(entry.shape) != entry.size:
            raise IndexError("Fancy indexing only currently supported for dim > 1 in a single dimension.")
        if entry.dtype.type is not np.int32:
            raise IndexError("Fancy indexing only currently supported with int32 types.")
        return entry

    def __getitem__(self, index):
        """View selected by integers, slices, one Ellipsis and at most one index
        vector (list / ndarray / int32 tensor: a gather along that axis, resolved
        when the view is used in an expression).  No data moves."""
        if isinstance(index, slice) and index == _none_slice:
            return self                       # the common a[:]
        entries = list(index) if isinstance(index, tuple) else [index]

        # an Ellipsis stands for as many full slices as it takes to reach every axis
        dots = [i for i, e in enumerate(entries) if e is Ellipsis]
        if len(dots) > 1:
            raise IndexError("more than one ellipsis not allowed in index")
        if dots:
            missing = len(self.shape) - (len(entries) - 1)
            if missing < 0:
                raise IndexError("invalid use of ellipsis in index")
            entries[dots[0]:dots[0] + 1] = [_none_slice] * missing
        if len(entries) > len(self.shape):
            raise IndexError("too many axes in index")
        entries += [_none_slice] * (len(self.shape) - len(entries))

        shape, strides, elements, gather = [], [], 0, None
        for axis, (entry, extent, stride) in enumerate(zip(entries, self.shape, self.strides)):
            if isinstance(entry, slice):
                first, stop, step = entry.indices(extent)
                shape.append(max(-((first - stop) // step), 0))
                strides.append(step * stride)
                elements += first * stride
            elif isinstance(entry, (int, np.integer)):
                position = int(entry) + extent if entry < 0 else int(entry)
                if not 0 <= position < extent:
                    raise IndexError("subindex in axis %d out of range" % axis)
                elements += position * stride           # the axis disappears
            elif isinstance(entry, (GPUTensor, np.ndarray, list, tuple)):
                if gather is not None:
                    raise IndexError("Fancy indexing only currently supported for one axis at a time.")
                vector = self._index_vector(entry)
                gather = (vector, axis)
                shape.append(vector.size)
                strides.append(stride)
            else:
                raise IndexError("invalid subindex in axis %d" % axis)
        return self._view(shape, strides, elements * self.dtype.itemsize, take_array=gather)

    def _assign(self, value):
        """self[...] = value.  Plain fills and plain copies use the memory
        primitives; everything else becomes an "assign" expression."""
        if isinstance(value, np.ndarray):
            return self.set(value)
        if not isinstance(value, (int, float, GPUTensor, OpTreeNode)):
            raise TypeError("Invalid type for assignment: %s" % type(value))
        stream = self.backend.stream
        if isinstance(value, (int, float)) and self.is_contiguous:
            if self.size:
                # the scalar's bit pattern in this dtype, replicated
                bits = int.from_bytes(np.array(value).astype(self.dtype).tobytes(), sys.byteorder)
                _lib.memset(self.gpudata, bits, self.size, self.dtype.itemsize, stream)
            return self
        if isinstance(value, GPUTensor) and self._is_plain_copy_of(value):
            if self.size:
                _lib.memcpy_dtod(self.gpudata, value.gpudata, self.nbytes, stream)
            return self
        OpTreeNode.build("assign", self, value)
        return self

    def _is_plain_copy_of(self, other):
        return (self.dtype == other.dtype and self.size == other.size
                and self.is_contiguous and other.is_contiguous
                and not self.is_trans and not other.is_trans)

    def __setitem__(self, index, value):
        self.__getitem__(index)._assign(value)

    def fill(self, value):
        return self._assign(value)

    def copy(self, a):
        return self._assign(a)

    def copy_from(self, a):
        """alias of set"""
        return self.set(a)

    def _same_memory(self, what, shape):
        if not self.is_contiguous:
            raise TypeError("%s of non-contigous arrays is not yet supported" % what)
        return tuple(int(d) for d in shape), _contiguous_strides(shape)

    def reshape(self, *shape):
        """the same elements under another shape (contiguous tensors only)"""
        if len(shape) == 1 and isinstance(shape[0], (tuple, list)):
            shape = tuple(shape[0])
        if shape == self.shape:
            return self
        if int(np.prod(shape, dtype=np.int64)) != self.size:
            raise ValueError("total size of new array must be unchanged")
        shape, strides = self._same_memory("reshaping", shape)
        return self._view(shape, strides)

    def share(self, shape, dtype=None, name=None):
        """a tensor of any shape and dtype with at most as many elements, laid over
        the start of this allocation: how temporaries share one buffer"""
        if int(np.prod(shape, dtype=np.int64)) > self.size:
            raise ValueError("total size of new array must <= size of parent")
        shape, strides = self._same_memory("sharing", shape)
        return self._view(shape, strides, name=name, dtype=self.dtype if dtype is None else np.dtype(dtype))

    @property
    def T(self):
        """Transposed view: the axes reverse, except that a tensor of more than two
        dimensions keeps its first (batch) axis in place, which is what the 3-D
        operands of batched_dot need.  Every .T flips is_trans."""
        rank = len(self.shape)
        order = list(range(rank - 1, -1, -1)) if rank <= 2 else [0] + list(range(rank - 1, 0, -1))
        return self._view([self.shape[a] for a in order], [self.strides[a] for a in order],
                          is_trans=not self.is_trans)

    def transpose(self, out=None):
        """transposed view, or a transposed copy into out"""
        if out:
            return OpTreeNode.build("assign", out, self.T)
        return self.T

    # arithmetic and comparison operators build expression nodes: see _install_operators


class NervanaGPU(object):

    def __init__(self, stochastic_round=False, bench=False,
                 cubin_path=os.path.join("kernels", "cubin"),
                 scratch_size=9 * 1024 * 1024, default_dtype=np.float16,
                 seed=None, device=0):
        """
        NervanaGPU: the primary interface class and factory for GPUTensors
        (nervanagpu/nervanagpu.py:471-492).

        stochastic_round: number of mantissa bits to stochastically round to
                          (True = 10); zero/False disables stochastic rounding.
        bench: set to 1 to print performance data for most kernel calls.
        cubin_path: accepted and ignored (kernels are compiled into the library).
        scratch_size: initial size of the shared scratch arena, in 4-byte words;
                      it grows on demand.
        seed: seed of the counter-based random stream used by stochastic rounding
              and `rand` (default: drawn from numpy's global generator, so
              np.random.seed() makes a run reproducible).
        """
        if stochastic_round:
            if stochastic_round is True:
                stochastic_round = 10
        else:
            stochastic_round = 0

        self.scratch_size = scratch_size
        self.round_mode = stochastic_round
        self.cubin_path = cubin_path
        self.bench = bench
        self.stream = None
        self.default_dtype = default_dtype
        self.device = device
        if seed is None:
            seed = int(np.random.randint(0, 2 ** 31 - 1))
        self.rng_seed = int(seed) & 0xFFFFFFFF
        self.rng_counter = 0
        self._scratch = None
        self._scratch_bytes = 0
        self._events = None
        _lib.set_default_device(device)

    # ---- random stream / scratch / events -------------------------------------

    def _next_rng_stream(self):
        """(seed, stream id) for the next launch that consumes random bits"""
        self.rng_counter = (self.rng_counter + 1) & 0xFFFFFFFF
        return self.rng_seed, self.rng_counter

    def _get_scratch(self, nbytes):
        """the one scratch arena shared by conv bprop/update, pooling and split GEMMs
        (nervanagpu/nervanagpu.py:1333-1335); grows when a layer needs more"""
        nbytes = max(int(nbytes), self.scratch_size * 4)
        if self._scratch is None or self._scratch_bytes < nbytes:
            if self._scratch is not None:
                _lib.stream_sync(self.stream)
            self._scratch = _lib.mem_alloc(nbytes)
            self._scratch_bytes = nbytes
        return self._scratch, self._scratch_bytes

    def _get_events(self):
        if self._events is None:
            self._events = (_lib.Event(), _lib.Event())
        return self._events

    # ---- factory ---------------------------------------------------------------

    def empty(self, shape, dtype=None, name=None, allocator=_lib.mem_alloc):
        """allocate the space for a GPUTensor"""
        dtype = self.default_dtype if dtype is None else dtype
        return GPUTensor(self, shape, dtype, allocator=allocator, name=name, rounding=self.round_mode)

    def array(self, ary, dtype=None, name=None, allocator=_lib.mem_alloc):
        """converts a numpy array to a GPUTensor"""
        dtype = self.default_dtype if dtype is None else dtype
        return GPUTensor(self, ary.shape, dtype, allocator=allocator, name=name,
                         rounding=self.round_mode).set(ary)

    def zeros(self, shape, dtype=None, name=None, allocator=_lib.mem_alloc):
        """array of the given shape and dtype filled with 0's"""
        dtype = self.default_dtype if dtype is None else dtype
        return GPUTensor(self, shape, dtype, allocator=allocator, name=name,
                         rounding=self.round_mode)._assign(0)

    def ones(self, shape, dtype=None, name=None, allocator=_lib.mem_alloc):
        """array of the given shape and dtype filled with 1's"""
        dtype = self.default_dtype if dtype is None else dtype
        return GPUTensor(self, shape, dtype, allocator, name=name, rounding=self.round_mode)._assign(1)

    def empty_like(self, other_ary, name=None):
        return GPUTensor(self, other_ary.shape, other_ary.dtype, other_ary.allocator,
                         name=name, rounding=self.round_mode)

    def zeros_like(self, other_ary, name=None):
        return GPUTensor(self, other_ary.shape, other_ary.dtype, other_ary.allocator,
                         name=name, rounding=self.round_mode)._assign(0)

    # ---- convolution -------------------------------------------------------------

    def conv_layer(self, dtype,
                   N, C, K,
                   D=1, H=1, W=1,
                   T=1, R=1, S=1,
                   pad_d=0, pad_h=0, pad_w=0,
                   str_d=1, str_h=1, str_w=1,
                   grid_P=0, grid_Q=0, update_size=None):
        """
        Create a new ConvLayer parameter object, passed to all convolution
        operations (nervanagpu/nervanagpu.py:540-589).

        N: minibatch size; C / K: input / output feature maps
        D,H,W: input depth/height/width; T,R,S: filter depth/height/width
        padding: zero-padding around each edge; strides: filter step
        grid_P, grid_Q, update_size: tuning hints of the reference's update
        kernels; accepted and ignored (update always accumulates in fp32 with a
        fixed-order reduction).
        """
        from .layers import ConvLayer
        return ConvLayer(self, dtype, N, C, K, D, H, W, T, R, S,
                         pad_d, pad_h, pad_w, str_d, str_h, str_w, grid_P, grid_Q, update_size)

    def deconv_layer(self, dtype,
                     N, C, K,
                     P, Q,
                     R=1, S=1,
                     pad_d=0, pad_h=0, pad_w=0,
                     str_d=1, str_h=1, str_w=1,
                     grid_P=0, grid_Q=0, update_size=None):
        """DeconvLayer parameter object (nervanagpu/nervanagpu.py:591-639):
        C output feature maps, K input feature maps, P,Q the input extent."""
        from .layers import DeconvLayer
        return DeconvLayer(self, dtype, N, C, K, P, Q, R, S,
                           pad_d, pad_h, pad_w, str_d, str_h, str_w, grid_P, grid_Q, update_size)

    def fprop_conv(self, layer, I, F, O, alpha=1.0, relu=False, repeat=1):
        assert layer.sizeI == I.size
        assert layer.sizeF == F.size
        assert layer.sizeO == O.size
        return self._execute_conv(layer, "fprop", I, F, O, alpha, relu, repeat)

    def bprop_conv(self, layer, F, E, grad_I, alpha=1.0, repeat=1, relu_mask=None):
        """relu_mask (not in the reference; unit strides only): the activations of
        the layer below, shaped like grad_I.  grad_I is also multiplied by
        (relu_mask > 0), the rectifier derivative that layer applies to its
        incoming error (nervanagpu/layers.py:89-91), inside the kernel's store."""
        assert layer.sizeF == F.size
        assert layer.sizeO == E.size
        assert layer.sizeI == grad_I.size
        if relu_mask is not None:
            assert relu_mask.size == grad_I.size and relu_mask.dtype == grad_I.dtype and relu_mask.is_contiguous
        return self._execute_conv(layer, "bprop", E, F, grad_I, alpha, False, repeat, relu_mask)

    def update_conv(self, layer, I, E, grad_F, alpha=1.0, repeat=1):
        assert layer.sizeI == I.size
        assert layer.sizeO == E.size
        assert layer.sizeF == grad_F.size
        return self._execute_conv(layer, "updat", I, E, grad_F, alpha, False, repeat)

    def _execute_conv(self, layer, op, A, B, C, alpha, relu, repeat, relu_mask=None):
        """A,B,C: (I,F,O) for fprop, (E,F,grad_I) for bprop, (I,E,grad_F) for update
        (nervanagpu/nervanagpu.py:671-734)."""
        int8_in = A.dtype.type in (np.uint8, np.int8) and op in ("fprop", "updat")
        assert int8_in or A.dtype == B.dtype
        for t in (A, B, C):
            assert t.is_contiguous, "convolution operands must be contiguous"

        plan = layer._get_plan()
        ws, ws_bytes = self._get_scratch(layer._workspace_bytes())
        flags = _lib.FLAG_RELU if relu else 0
        stream = self.stream

        if op == "fprop":
            assert B.dtype == C.dtype == layer.np_dtype
            def launch():
                _lib.call("ng_conv_fprop", plan, _DTYPE_CODE[A.dtype], c_void_p(A.ptr), c_void_p(B.ptr),
                          c_void_p(C.ptr), alpha, flags, c_void_p(int(ws)), ws_bytes, stream)
        elif op == "bprop":
            assert A.dtype == C.dtype == layer.np_dtype
            def launch():
                _lib.call("ng_conv_bprop", plan, c_void_p(B.ptr), c_void_p(A.ptr), c_void_p(C.ptr),
                          alpha, c_void_p(relu_mask.ptr if relu_mask is not None else None),
                          c_void_p(int(ws)), ws_bytes, stream)
        else:
            assert B.dtype == layer.np_dtype
            assert C.dtype.type in (np.float32, np.float16)
            def launch():
                _lib.call("ng_conv_update", plan, _DTYPE_CODE[A.dtype], _DTYPE_CODE[C.dtype],
                          c_void_p(A.ptr), c_void_p(B.ptr), c_void_p(C.ptr),
                          alpha, c_void_p(int(ws)), ws_bytes, stream)

        if repeat > 1:
            for r in range(max(repeat // 10, 1)):
                launch()
        if self.bench or repeat > 1:
            start, end = self._get_events()
            start.record(stream)
        for r in range(repeat):
            launch()
        if self.bench or repeat > 1:
            end.record(stream)
            end.synchronize()
            msecs = end.time_since(start) / repeat
            gflops = layer.flops / (msecs * 1000000.0)
            print("%7.3f msecs %8.3f gflops %6.0f (%s: %s)" %
                  (msecs, gflops, layer.flops / 1000000.0, op, layer))
            return msecs, gflops
        return 0, 0

    # ---- pooling -------------------------------------------------------------------

    def pool_layer(self, dtype,
                   op, N, C,
                   D=1, H=1, W=1,
                   J=1, T=1, R=1, S=1,
                   pad_j=0, pad_d=0, pad_h=0, pad_w=0,
                   str_j=None, str_d=None, str_h=None, str_w=None):
        """
        Create a new PoolLayer parameter object (nervanagpu/nervanagpu.py:736-771).

        op: "max", "avg" or "l2" pooling (l2: forward only)
        N: minibatch; C,D,H,W: input feature maps / depth / height / width
        J,T,R,S: window over feature maps (maxout) / depth / height / width
        padding: around each edge; strides default to the window (no overlap)
        """
        from .layers import PoolLayer
        if str_j is None: str_j = J
        if str_d is None: str_d = T
        if str_h is None: str_h = R
        if str_w is None: str_w = S
        return PoolLayer(self, dtype, op, N, C, D, H, W, J, T, R, S,
                         pad_j, pad_d, pad_h, pad_w, str_j, str_d, str_h, str_w)

    def fprop_pool(self, layer, I, O, repeat=1):
        assert layer.sizeI == I.size
        assert layer.sizeO == O.size
        return self._execute_pool(layer, I, O, None, 0, repeat)

    def bprop_pool(self, layer, I, E, grad_I, repeat=1, relu_mask=False):
        """relu_mask (max pooling only, not in the reference): also multiply
        grad_I by (I > 0), the rectifier derivative the layer that produced I
        applies to its incoming error (nervanagpu/layers.py:89-91); the pooling
        kernel already reads I, so the separate elementwise pass is saved."""
        assert layer.sizeI == I.size
        assert layer.sizeO == E.size
        assert layer.sizeI == grad_I.size
        assert I.dtype == grad_I.dtype
        return self._execute_pool(layer, I, E, grad_I, 1, repeat, relu_mask)

    def _execute_pool(self, layer, I, O, B, mode, repeat, relu_mask=False):
        assert I.dtype == O.dtype
        assert I.is_contiguous and O.is_contiguous and (B is None or B.is_contiguous)
        if layer.op not in ("max", "avg", "l2"):
            raise ValueError("pooling op %r is not implemented (max, avg, l2)" % (layer.op,))
        if layer.op == "l2" and mode:
            raise ValueError("l2 pooling has no backward pass: the reference defines none (benchmarks/pool_test.py:142-146)")
        op = {"max": 0, "avg": 1, "l2": 2}[layer.op]
        params = layer._params()
        code = _DTYPE_CODE[I.dtype]
        stream = self.stream
        if mode:
            ws, ws_bytes = self._get_scratch(layer._workspace_bytes())
            def launch():
                _lib.call("ng_pool_bprop", ctypes.byref(params), code, op, c_void_p(I.ptr), c_void_p(O.ptr),
                          c_void_p(B.ptr), _lib.FLAG_RELU if relu_mask else 0, c_void_p(int(ws)), ws_bytes, stream)
        else:
            def launch():
                _lib.call("ng_pool_fprop", ctypes.byref(params), code, op, c_void_p(I.ptr), c_void_p(O.ptr), stream)

        if repeat > 1:
            for r in range(max(repeat // 10, 1)):
                launch()
        if self.bench or repeat > 1:
            start, end = self._get_events()
            start.record(stream)
        for r in range(repeat):
            launch()
        if self.bench or repeat > 1:
            end.record(stream)
            end.synchronize()
            msecs = end.time_since(start) / repeat
            print("%7.3f msecs (%s)" % (msecs, layer))
            if repeat > 1:
                return msecs

    # ---- GEMM ------------------------------------------------------------------------

    def _gemm(self, A, B, C, m, n, k, lda, ldb, ldc, alpha, beta, relu, repeat,
              batch_grid, ldaz, ldbz, ldcz, batch_loops):
        if C.dtype.type is np.float16:
            clss, code = "hgemm", _lib.NG_F16
        elif C.dtype.type is np.float32:
            clss, code = "sgemm", _lib.NG_F32
        else:
            raise TypeError("Only floating point dot currently supported.")
        op = ("t" if A.is_trans else "n") + ("t" if B.is_trans else "n")
        assert op != "tt"

        flags = 0
        if C.rounding:
            flags |= 1 | (int(C.rounding) << 16)
        if relu:
            flags |= 2
        stream = self.stream
        ws, ws_bytes = self._get_scratch(0)
        state = {}

        def launch():
            seed, sid = self._next_rng_stream() if C.rounding else (0, 0)
            state["sid"] = sid
            _lib.call("ng_gemm", code, int(A.is_trans), int(B.is_trans), m, n, k,
                      c_void_p(A.ptr), lda, c_void_p(B.ptr), ldb, c_void_p(C.ptr), ldc,
                      alpha, beta, flags, seed, sid,
                      batch_grid, ldaz, ldbz, ldcz, batch_loops,
                      c_void_p(int(ws)), ws_bytes, stream)

        if repeat > 1:
            for r in range(max(repeat // 10, 1)):
                launch()
        if self.bench or repeat > 1:
            start, end = self._get_events()
            start.record(stream)
        for r in range(repeat):
            launch()
        if self.bench or repeat > 1:
            end.record(stream)
            end.synchronize()
            msecs = end.time_since(start) / repeat
            gflops = (batch_loops * batch_grid * m * n * k * 2.0) / (msecs * 1000000.0)
            print("%7.3f msecs %4.0f gflops (%s_%s: %d,%d,%d) grid:%d loops:%d" %
                  (msecs, gflops, clss, op, m, n, k, batch_grid, batch_loops))
            if repeat > 1:
                return gflops
        return C

    def batched_dot(self, A, B, C, alpha=1.0, beta=0.0, relu=False, repeat=1, size=None):
        """batched GEMM (nervanagpu/nervanagpu.py:820-957): A and/or B are 3-D
        (batch, ., .).  3-D C: one product per batch (2-D operands broadcast);
        2-D C: the products are summed over the batch.  `size` is accepted as a
        hint and ignored."""
        assert A.dtype.type == B.dtype.type == C.dtype.type

        def split(t):
            """(batch count or None, batch stride, the 2-D matrix part)"""
            if len(t.shape) == 3:
                return t.shape[0], t.strides[0], (t.shape[1:], t.strides[1:])
            return None, 0, (t.shape, t.strides)

        batch_a, ldaz, (shape_a, strides_a) = split(A)
        batch_b, ldbz, (shape_b, strides_b) = split(B)
        batch_c, ldcz, (shape_c, strides_c) = split(C)
        assert batch_a is not None or batch_b is not None, "Tensor A or B must have 3 dims to use batched_dot"
        batches = {b for b in (batch_a, batch_b, batch_c) if b is not None}
        assert len(batches) == 1, "batched operands disagree on the batch count"
        count = batches.pop()
        # a batched C takes one product per batch entry (a 2-D operand is reused
        # for all of them: batch stride 0); a 2-D C receives the sum over the batch
        batch_grid, batch_loops = (count, 1) if batch_c is not None else (1, count)

        (m, k), n = shape_a, shape_b[1]
        assert shape_c == (m, n) and shape_b[0] == k
        return self._gemm(A, B, C, m, n, k, max(strides_a), max(strides_b), max(strides_c),
                          alpha, beta, relu, repeat, batch_grid, ldaz, ldbz, ldcz, batch_loops)

    def dot(self, A, B, C, alpha=1.0, beta=0.0, relu=False, repeat=1, size=None):
        """
        C = alpha * A * B   + beta * C
        C = alpha * A.T * B + beta * C
        C = alpha * A * B.T + beta * C

        relu: if true applied before output (and prior to beta addition)
        size: tile hint of the reference ("128x64" ...); accepted and ignored.
        (nervanagpu/nervanagpu.py:959-1105)
        """
        assert A.dtype.type == B.dtype.type == C.dtype.type

        # one dimension must be contiguous
        assert min(A.strides) == 1
        assert min(B.strides) == 1
        assert min(C.strides) == 1

        lda = max(A.strides)
        ldb = max(B.strides)
        ldc = max(C.strides)

        m = A.shape[0]
        n = B.shape[1]
        k = A.shape[1]

        assert m == C.shape[0]
        assert n == C.shape[1]
        assert k == B.shape[0]

        return self._gemm(A, B, C, m, n, k, lda, ldb, ldc, alpha, beta, relu, repeat, 1, 0, 0, 0, 1)

    # ---- block-scaled matrices and 8-bit checkpoints (not in the reference) -------------

    def mx_empty(self, shape, fmt="fp4", axis=1, name=None, rounding=None):
        """allocate a block-scaled matrix (see mx.MXTensor); rounding: stochastic
        when true, default as this backend stores its other tensors"""
        return MXTensor(self, shape, fmt, axis, name=name, rounding=self.round_mode if rounding is None else rounding)

    def mx_array(self, ary, fmt="fp4", axis=1, name=None, rounding=None):
        """a host matrix converted to a block-scaled one"""
        return self.mx_empty(ary.shape, fmt, axis, name, rounding).set(ary)

    @staticmethod
    def _mx_dense(A, axis, what):
        """(pitch, whether lines along `axis` are contiguous) of a dense 2-D tensor"""
        shape, strides = A.shape, A.strides
        assert len(shape) == 2 and not A.take_array, "%s must be a 2-D tensor" % what
        inner, outer = strides[axis], strides[1 - axis]
        depth, lines = shape[axis], shape[1 - axis]
        # the C interface takes extents as ints
        assert (depth | lines) < 2 ** 31, "%s has an extent of 2^31 or more" % what
        if inner == 1:
            if outer >= depth:
                return outer, 1
            if lines <= 1:
                return depth, 1
        if outer == 1:
            if inner >= lines:
                return inner, 0
            if depth <= 1:
                return lines, 0
        assert not A.size, "one dimension of %s must be contiguous" % what
        return depth, 1

    def mx_quantize(self, A, out):
        """out = A in blocks of 32 values that share a power of two.  A: fp16 or fp32
        matrix with one contiguous dimension.  Rounds to the nearest code (ties to
        even), or stochastically if out.rounding is set: then every value is right on
        average, but for int8 values above the last code (127/64 of the block's power of
        two, at most 128/64), which become 127/64 in either mode.  A block with an
        infinity or a NaN becomes NaN.  Returns out."""
        assert type(out) is MXTensor and A.shape == out.shape
        if A.dtype.type not in _FLOATS:
            raise TypeError("Only floating point tensors can be quantized.")
        ld, along = self._mx_dense(A, out.axis, "A")
        if out.size:
            flags, (seed, sid) = (_lib.FLAG_SR, self._next_rng_stream()) if out.rounding else (0, (0, 0))
            _lib.call("ng_mx_quantize", out.fmt_code, _DTYPE_CODE[A.dtype], A.ptr, ld, along, out.lines, out.depth,
                      out.codes.ptr, out.scales.ptr, flags, seed, sid, self.stream)
        return out

    def mx_dequantize(self, A, out):
        """out (fp16 or fp32) = the values of the block-scaled A, rounded to the nearest
        whatever out.rounding says; returns out"""
        assert type(A) is MXTensor and A.shape == out.shape
        if out.dtype.type not in _FLOATS:
            raise TypeError("Only floating point tensors can be dequantized into.")
        ld, along = self._mx_dense(out, A.axis, "out")
        if A.size:
            _lib.call("ng_mx_dequantize", A.fmt_code, A.codes.ptr, A.scales.ptr, A.lines, A.depth, _DTYPE_CODE[out.dtype],
                      out.ptr, ld, along, self.stream)
        return out

    def _mx_side(self, X, axis, what):
        """an operand of mx_dot whose contraction is its axis `axis`"""
        if type(X) is MXTensor:
            if X.axis != axis:
                raise ValueError("the blocks of %s must run along the contraction (axis %d)" % (what, axis))
            return X.operand()
        assert X.dtype.type is np.float16, "a dense operand of mx_dot must be fp16"
        ld, along = self._mx_dense(X, axis, what)
        return _lib.MxOperand(_lib.NG_MX_NONE, along, ld, X.ptr if X.size else None, None)

    def mx_dot(self, A, B, C, alpha=1.0, beta=0.0, relu=False, repeat=1):
        """
        C = relu(alpha * A * B) + beta * C for block-scaled operands

        A (m, k), B (k, n): both fp4, or one of them fp4 or int8 and the other a dense
        fp16 tensor (any order of its axes; the values of the block-scaled one are then
        taken as fp16: exact if they came from fp16, else far ones overflow or vanish).
        Blocks run along k: A has axis 1, B has axis 0.
        C: fp16 or fp32, rows or columns contiguous, on memory of its own; stochastic
        rounding as in dot.  relu keeps NaN, unlike dot's: a block that is marked NaN
        stays visible.
        """
        if type(A) is MXTensor:
            if type(B) is MXTensor and not A.fmt == B.fmt == "fp4":
                raise TypeError("block-scaled operands must both be fp4, or one operand a dense fp16 tensor")
        elif type(B) is not MXTensor:
            raise TypeError("mx_dot needs a block-scaled operand (dot multiplies dense ones)")
        if C.dtype.type not in _FLOATS:
            raise TypeError("Only floating point dot currently supported.")
        a, b = self._mx_side(A, 1, "A"), self._mx_side(B, 0, "B")
        (m, k), n = A.shape, B.shape[1]
        assert C.shape == (m, n) and B.shape[0] == k
        ldc, by_rows = self._mx_dense(C, 1, "C")
        assert ldc < 2 ** 31, "rows of C are too far apart"
        if not by_rows:
            # columns contiguous: the transposed product
            m, n, a, b = n, m, b, a
        if not C.size:
            return C
        code = _DTYPE_CODE[C.dtype]
        rounding = C.rounding
        flags = (1 | (int(rounding) << 16) if rounding else 0) | (2 if relu else 0)
        stream, c_ptr, gemm = self.stream, C.ptr, _lib.load().ng_mx_gemm

        def launch():
            seed, sid = self._next_rng_stream() if rounding else (0, 0)
            ws, ws_bytes = self._get_scratch(0)
            status = gemm(code, m, n, k, a, b, c_ptr, ldc, alpha, beta, flags, seed, sid, int(ws), ws_bytes, stream)
            if status == _lib.NG_MX_WORKSPACE:
                # nothing has been launched: the arena grows and the call is made again
                ws, ws_bytes = self._get_scratch(_lib.load().ng_mx_gemm_workspace_bytes(code, m, n, k, a, b))
                status = gemm(code, m, n, k, a, b, c_ptr, ldc, alpha, beta, flags, seed, sid, int(ws), ws_bytes, stream)
            if status:
                _lib.check(status)

        if repeat > 1:
            for r in range(max(repeat // 10, 1)):
                launch()
        if self.bench or repeat > 1:
            start, end = self._get_events()
            start.record(stream)
        for r in range(repeat):
            launch()
        if self.bench or repeat > 1:
            end.record(stream)
            end.synchronize()
            msecs = end.time_since(start) / repeat
            gflops = (m * n * k * 2.0) / (msecs * 1000000.0)
            print("%7.3f msecs %4.0f gflops (mx_dot: %d,%d,%d)" % (msecs, gflops, m, n, k))
            if repeat > 1:
                return gflops
        return C

    def _act_operands(self, op, dense, saved):
        """(op code, dtype code, rows, cols, codes, scales, pitches) of an activation
        function's operands, all checked"""
        code = _ACT_CODE.get(op)
        if code is None:
            raise ValueError("unknown activation function %r (%s)" % (op, ", ".join(sorted(_ACT_CODE))))
        first = dense[0]
        if first.dtype.type not in _FLOATS:
            raise TypeError("Only floating point activations are supported.")
        lds = []
        for X in dense:
            assert X.shape == first.shape and X.dtype == first.dtype, "activation operands must match"
            ld, along = self._mx_dense(X, 1, "an activation operand")
            assert along, "rows of activation operands must be contiguous"
            lds.append(ld)
        codes = scales = None
        if saved is not None:
            assert type(saved) is MXTensor and saved.shape == first.shape, "the checkpoint must match the operands"
            if saved.fmt != "int8" or saved.axis != 1:
                raise ValueError("a checkpoint of activations is an int8 MXTensor with axis 1")
            if saved.size:
                codes, scales = saved.codes.ptr, saved.scales.ptr
        return code, _DTYPE_CODE[first.dtype], first.shape[0], first.shape[1], codes, scales, lds

    def fprop_act(self, op, I, O, saved=None):
        """
        O = op(I), and saved (an MXTensor, fmt "int8", axis 1) = I rounded to the
        nearest, in one pass.

        op: "relu", "sig", "tanh", "silu" (x sig(x)) or "gelu" (x times the normal
        distribution function of x); I, O: fp16 or fp32 matrices, rows contiguous; O may
        be I.  Stored rounded to the nearest, whatever O.rounding says.
        """
        code, dtype, rows, cols, codes, scales, (ldi, ldo) = self._act_operands(op, (I, O), saved)
        if I.size:
            _lib.call("ng_act_fprop", code, dtype, rows, cols, I.ptr, ldi, O.ptr, ldo, codes, scales, self.stream)
        return O

    def bprop_act(self, op, saved, E, grad_I):
        """grad_I = E * op'(saved): the derivative is taken at the values the 8-bit
        checkpoint of fprop_act stands for, NaN where its block holds an infinity or
        a NaN (under relu too).  grad_I may be E."""
        assert saved is not None, "bprop_act needs the checkpoint of fprop_act"
        code, dtype, rows, cols, codes, scales, (lde, ldg) = self._act_operands(op, (E, grad_I), saved)
        if E.size:
            _lib.call("ng_act_bprop", code, dtype, rows, cols, codes, scales, E.ptr, lde, grad_I.ptr, ldg, self.stream)
        return grad_I

    def compensated_sum(self, sum_tensor, cmp_tensor, add_tensor, cmp_scale=1.0, add_scale=1.0):
        """Kahan-compensated low-precision accumulate
        (nervanagpu/nervanagpu.py:1107-1126, nervanagpu/float_ew.py:1430-1482):
            y = add*add_scale - cmp*cmp_scale; t = round(sum + y);
            cmp = round_nearest((t - sum) - y); sum = t"""
        if cmp_tensor.kahan_reset and cmp_tensor.kahan_count > cmp_tensor.kahan_reset:
            cmp_scale = 0
            cmp_tensor.kahan_count = 0
        assert sum_tensor.dtype.type == cmp_tensor.dtype.type == add_tensor.dtype.type
        cmp_tensor.kahan_count += 1

        # one kernel: reads sum, cmp and add, writes sum and cmp; no temporary.
        # With stochastic rounding it draws one random stream per call.
        call_compensated_sum(self, sum_tensor, cmp_tensor, add_tensor, float(cmp_scale), float(add_scale))

    # The elementwise wrappers (add, subtract, ..., sqrt, ..., equal, ..., maximum,
    # minimum) are installed from the tables below the class: every one of them
    # only records a node, `out=` executes it.

    def reciprocal(self, a, out=None):
        return OpTreeNode.build("div", 1, a, out=out)

    def clip(self, a, a_min, a_max, out=None):
        return self.minimum(self.maximum(a, a_min), a_max, out=out)

    def _reduce(self, op, a, axis, partial, out):
        """one reduction along axis 0 or 1; axis None reduces the rows into
        `partial` (shape (rows, 1)) first and that column into `out` second, two
        kernels (nervanagpu/nervanagpu.py:1167-1171)"""
        if axis is not None:
            return OpTreeNode.build(op, a, None, axis=axis, out=out)
        assert partial is not None
        rows = OpTreeNode.build(op, a, None, axis=1, out=partial)
        return OpTreeNode.build(op, rows, None, axis=0, out=out)

    def sum(self, a, axis=None, partial=None, out=None, keepdims=True):
        return self._reduce("sum", a, axis, partial, out)

    def max(self, a, axis=None, partial=None, out=None, keepdims=True):
        return self._reduce("max", a, axis, partial, out)

    def min(self, a, axis=None, partial=None, out=None, keepdims=True):
        return self._reduce("min", a, axis, partial, out)

    def argmax(self, a, axis=1, out=None, keepdims=True):
        return OpTreeNode.build("argmax", a, None, axis=axis, out=out)

    def argmin(self, a, axis=1, out=None, keepdims=True):
        return OpTreeNode.build("argmin", a, None, axis=axis, out=out)

    def mean(self, a, axis=None, partial=None, out=None, keepdims=True):
        """sum times the reciprocal of the number of elements reduced"""
        extent = OpTreeNode.shape(a)
        count = extent[0] * extent[1] if axis is None else extent[axis]
        total = self._reduce("sum", a, axis, partial, None)
        return OpTreeNode.build("mul", total, 1.0 / count, out=out)

    def var(self, a, axis=None, partial=None, out=None, keepdims=True):
        """population variance: mean((a - mean(a))^2); the full reduction keeps its
        intermediate mean in the first element of `partial`"""
        if axis is None:
            assert partial is not None
            centre = self.mean(a, partial=partial, out=partial[0:1, 0:1])
        else:
            centre = self.mean(a, axis=axis)
        return self.mean(self.square(a - centre), axis=axis, partial=partial, out=out)

    def std(self, a, axis=None, partial=None, out=None, keepdims=True):
        # The reference passes `out` to var() and wraps the result in a lazy sqrt
        # that is never executed, leaving the variance in `out`
        # (nervanagpu/nervanagpu.py:1210-1211); here the sqrt is part of the
        # assignment so `out` receives the standard deviation.
        return self.sqrt(self.var(a, axis=axis, partial=partial), out=out)

    def rand(self, out=None):
        return OpTreeNode.build("rand", None, None, out=out)

    def dropout(self, keep=0.5, out=None):
        """mask that is 1 with probability `keep`"""
        return self.less_equal(self.rand(), keep, out=out)

    def take(self, a, indices, axis, out=None):
        return a.take(indices, axis, out)

    def onehot(self, indices, axis, out=None):
        if axis not in (0, 1):
            raise ValueError("bad axis for onehot")
        return OpTreeNode.build("onehot", None, None, idx=indices, axis=axis, out=out)


# public name -> op of the expression generator (nervanagpu/nervanagpu.py:1128-1162)
_BINARY_WRAPPERS = {
    "add": "add", "subtract": "sub", "multiply": "mul", "divide": "div", "true_divide": "div", "power": "pow",
    "equal": "eq", "not_equal": "ne", "less": "lt", "less_equal": "le", "greater": "gt", "greater_equal": "ge",
    "maximum": "maximum", "minimum": "minimum",
}
_UNARY_WRAPPERS = {
    "negative": "neg", "sgn": "sgn", "absolute": "abs", "fabs": "abs", "sqrt": "sqrt", "square": "sqr",
    "exp": "exp", "exp2": "exp2", "log": "log", "log2": "log2", "sig": "sig", "sig2": "sig2",
    "tanh": "tanh", "tanh2": "tanh2", "finite": "finite",
}


def _install_wrappers():
    def binary(op):
        def method(self, a, b, out=None):
            return OpTreeNode.build(op, a, b, out=out)
        return method

    def unary(op):
        def method(self, a, out=None):
            return OpTreeNode.build(op, a, None, out=out)
        return method

    for name, op in _BINARY_WRAPPERS.items():
        setattr(NervanaGPU, name, binary(op))
    for name, op in _UNARY_WRAPPERS.items():
        setattr(NervanaGPU, name, unary(op))


_install_wrappers()


class OpTreeNode(tuple):
    """Node of a lazy expression: (op description dict, left operand, right
    operand).  Operands are tensors, Python / numpy scalars, other nodes, or None
    for the missing side of a unary or zero-argument op.  Nothing runs until the
    expression is assigned (`out[:] = expr`, `out=`, `+=` ...): then the tree is
    flattened to a postfix stack and handed to the kernel generator
    (nervanagpu/nervanagpu.py:1227-1321)."""

    _OPERAND_TYPES = (int, float, np.integer, np.floating, GPUTensor, type(None))

    def __new__(cls, *args):
        return tuple.__new__(cls, args)

    # identity hashing: == is an expression builder, and the op dict is unhashable
    __hash__ = object.__hash__

    @staticmethod
    def build(op, a, b, out=None, **kwargs):
        """node for `op(a, b)`; an "assign" op or an `out` tensor executes at once"""
        if not all(isinstance(x, OpTreeNode._OPERAND_TYPES + (OpTreeNode,)) for x in (a, b)):
            return NotImplemented
        node = OpTreeNode(dict(kwargs, op=op), a, b)
        if op == "assign":
            return node.execute()
        if out is not None:
            return OpTreeNode({"op": "assign"}, out, node).execute()
        return node

    def execute(self):
        stack = self.traverse([])
        backend = next((x.backend for x in stack if isinstance(x, GPUTensor)), None)
        return call_compound_kernel(backend, *stack)

    def traverse(self, stack):
        """append this subtree to `stack` in postfix order: operands, then the op"""
        description, left, right = self
        for operand in (left, right):
            if type(operand) is OpTreeNode:
                operand.traverse(stack)
            elif operand is not None:
                stack.append(operand)
        stack.append(description)
        return stack

    @staticmethod
    def shape(node):
        """2-D shape an expression broadcasts to: per axis the largest extent of
        any tensor in it; scalars count as (1, 1)"""
        if type(node) is GPUTensor:
            return node.shape
        if type(node) is not OpTreeNode:
            return (1, 1)
        tensors = [x for x in node.traverse([]) if type(x) is GPUTensor]
        return tuple(max([1] + [t.shape[axis] for t in tensors]) for axis in (0, 1))


def _install_operators(cls, in_place):
    """Python operators of tensors and expression nodes: each one only records
    an op (names as in nervanagpu/nervanagpu.py:438-464, 1296-1321); the
    in-place forms of tensors execute into the tensor itself."""
    def forward(op):
        return lambda self, other: OpTreeNode.build(op, self, other)

    def reflected(op):
        return lambda self, other: OpTreeNode.build(op, other, self)

    def into_self(op):
        return lambda self, other: OpTreeNode.build(op, self, other, out=self)

    def unary(op):
        return lambda self: OpTreeNode.build(op, self, None)

    for method, op in (("add", "add"), ("sub", "sub"), ("mul", "mul"), ("div", "div"), ("truediv", "div"),
                       ("pow", "pow")):
        setattr(cls, "__%s__" % method, forward(op))
        setattr(cls, "__r%s__" % method, reflected(op))
        if in_place:
            setattr(cls, "__i%s__" % method, into_self(op))
    for op in ("eq", "ne", "lt", "le", "gt", "ge"):
        setattr(cls, "__%s__" % op, forward(op))
    for op in ("abs", "neg"):
        setattr(cls, "__%s__" % op, unary(op))


_install_operators(GPUTensor, in_place=True)
_install_operators(OpTreeNode, in_place=False)
