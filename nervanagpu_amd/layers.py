"""
Layer objects: the geometry carriers every convolution / pooling call takes
(`ConvLayer`, `DeconvLayer`, `PoolLayer`) and the small training driver built
on them (`DataLayer`, `FullLayer`, `Inception`, `Layer.create`), with the public
surface of nervanagpu/layers.py:26-778 of the reference.

What a caller may rely on, as in the reference:

* geometry attributes `N C K M P Q`, `NCK TRS/JTRS DHW MPQ padding strides`,
  tensor shapes `dimI dimF dimO` (CHWN / CTRSK / KMPQN), their 2-D views
  `dimI2 dimF2 dimO2`, element counts `sizeI sizeF sizeO`, `nOut`, `flops`;
* buffers `fprop_in fprop_out bprop_out weights updat_out` created by
  `init_activations / init_deltas / init_weights`, with the sharing rules of the
  benchmark driver (two alternating delta buffers, one update buffer);
* `fprop(x, scale_weights=0)`, `bprop(err)`: rectified forward, rectifier
  derivative, data gradient, weight gradient, SGD step;
* `Layer.create(lib, conf, prev_layer, dtype)` chaining layers from config dicts.

Nothing here knows launch geometry: the reference precomputes grids, magic
division constants and argument lists for its Maxwell kernels at this point
(nervanagpu/layers.py:327-481); here a convolution layer owns a plan of the HIP
library instead, created on first use.
"""
import ctypes
from math import ceil

import numpy as np

from . import _lib


def _count(shape):
    """number of elements of a shape"""
    n = 1
    for extent in shape:
        n *= int(extent)
    return n


def _out_extent(size, window, pad, stride):
    """outputs along one axis: ceil((size - window + 1 + 2 pad) / stride)
    (nervanagpu/layers.py:297-301, 566-569)"""
    return int(ceil(float(size - window + 1 + 2 * pad) / stride))


# (reduction of the library, attribute holding the tensor, attribute holding the
# partial-result buffer, attribute holding the 2-D view shape, needs weights)
_STAT_SOURCES = {
    "activation": ("fprop_out", "act_stats", "dimO2", False),
    "delta":      ("bprop_out", "delta_stats", "dimI2", False),
    "update":     ("updat_out", "weight_stats", "dimF2", True),
    "weight":     ("weights", "weight_stats", "dimF2", True),
}


class Layer(object):
    """Common state of all layers and the pieces of the training step they share."""

    def __init__(self, lib, dtype, N, dtypeU=None):
        self.lib = lib
        self.N = N
        self.dtype = dtype
        # weight gradients may be kept wider than the weights (fp32 for convolutions)
        self.dtypeU = dtypeU if dtypeU is not None else dtype
        self.flops = 0
        self.sizeI = self.sizeO = self.sizeF = 0
        self.weights = self.fprop_in = self.fprop_out = self.bprop_out = None
        self.learning_rate = 0.0
        # Not in the reference.  A network builder sets this when the layer above
        # applies this layer's rectifier derivative inside its own backward kernel
        # (max pooling via PoolLayer.relu_below, unit-stride convolution via
        # ConvLayer.relu_mask_below); bprop_relu then has nothing left to do.
        self.relu_done_above = False

    # -- buffers ---------------------------------------------------------------

    def _stat_buffer(self, shape2):
        return self.lib.empty((shape2[0], 1), dtype=np.float32)

    def init_activations(self):
        self.fprop_out = self.lib.empty(self.dimO, dtype=self.dtype)
        self.act_stats = self._stat_buffer(self.dimO2)

    def init_deltas(self, shared=None):
        """own error buffer, or a view of shared[0]; the list is then flipped in
        place so that the next layer takes the other buffer"""
        if shared is not None:
            self.bprop_out = shared[0].share(self.dimI)
            shared.reverse()
        else:
            self.bprop_out = self.lib.empty(self.dimI, dtype=self.dtype)
        self.delta_stats = self._stat_buffer(self.dimI2)

    def init_weights(self, loc=0.0, scale=0.1, shared=None, zeros=False):
        if self.sizeF <= 0:
            return
        if zeros:
            self.weights = self.lib.zeros(self.dimF, dtype=self.dtype)
        else:
            self.weights = self.lib.array(np.random.normal(loc, scale, self.dimF), dtype=self.dtype)
        self.updat_out = (self.lib.empty(self.dimF, dtype=self.dtypeU) if shared is None
                          else shared.share(self.dimF, dtype=self.dtypeU))
        self.weight_stats = self._stat_buffer(self.dimF2)

    # -- training step -----------------------------------------------------------

    def fprop(self, fprop_in, scale_weights=0):
        """base behaviour: remember the input (viewed in this layer's shape) the
        first time one is given"""
        if self.fprop_in is None and fprop_in:
            self.fprop_in = fprop_in.reshape(self.dimI)
        return self.fprop_in

    def bprop(self, bprop_in):
        return bprop_in

    def bprop_relu(self, bprop_in):
        """derivative of the rectifier that the forward kernels apply to fprop_out"""
        if not self.relu_done_above:
            bprop_in *= self.fprop_out > 0
        return bprop_in

    def grad_descent(self):
        self.weights += self.updat_out * self.learning_rate

    def scale_weights(self, scale):
        """rescale the weights so that the mean |activation| becomes `scale`"""
        self.weights *= scale / self.get_activation_mean()

    def _rerun_scaled(self, fprop_in, scale_weights):
        # used by the weighted layers after their first forward pass
        if scale_weights:
            self.scale_weights(scale_weights)
            self.fprop(fprop_in)

    # -- statistics ----------------------------------------------------------------

    def _stat(self, source, reduction):
        tensor_attr, buffer_attr, shape_attr, needs_weights = _STAT_SOURCES[source]
        if needs_weights and self.sizeF <= 0:
            return 0
        tensor, buf = getattr(self, tensor_attr), getattr(self, buffer_attr)
        flat = abs(tensor.reshape(getattr(self, shape_attr)))
        reduce_fn = getattr(self.lib, reduction)
        return float(reduce_fn(flat, partial=buf, out=buf[0:1, 0:1]).get()[0, 0])

    def fprop_stats(self):
        print("fprop:%10.5f mean %11.5f max %s" % (self.get_activation_mean(), self.get_activation_max(), self))

    def bprop_stats(self):
        if self.bprop_out is not None:
            print("bprop:%10.5f mean %11.5f max %s" % (self.get_delta_mean(), self.get_delta_max(), self))
        if self.weights is None:
            return
        update = (self.get_update_mean(), self.get_update_max())
        weight = (self.get_weight_mean(), self.get_weight_max())
        print("updat:%10.5f mean %11.5f max %s" % (update + (self,)))
        print("weigh:%10.5f mean %11.5f max" % weight)
        print("ratio:%10.5f mean %11.5f max" % tuple(0.0001 * u / w for u, w in zip(update, weight)))

    # -- construction from configuration dicts ------------------------------------------

    @staticmethod
    def create(lib, conf, prev_layer, dtype):
        """Build `conf["layer"]` from a config dict.  Keys that are numpy dtypes
        hold overrides for that dtype, "common" holds keys shared by several
        configs; N and the input extents come from the layer below."""
        settings = {k: v for k, v in conf.items() if k != "layer"}
        kind = conf["layer"]
        settings["dtype"] = dtype
        settings.update(settings.pop(dtype, {}))
        settings.update(settings.pop("common", {}))
        if prev_layer is not None:
            _inherit_extents(lib, kind, settings, prev_layer, dtype)
        # whatever dtype-keyed overrides are left belong to other dtypes
        return kind(lib, **{k: v for k, v in settings.items() if isinstance(k, str)})


def _add_stat_getters():
    def getter(source, reduction):
        return lambda self: self._stat(source, reduction)
    for source in _STAT_SOURCES:
        for reduction in ("mean", "max"):
            setattr(Layer, "get_%s_%s" % (source, reduction), getter(source, reduction))


_add_stat_getters()


def _inherit_extents(lib, kind, settings, below, dtype):
    """what a layer takes over from the one below it (Layer.create)"""
    settings["N"] = below.N
    if kind is FullLayer:
        settings["nIn"] = below.nOut
        return
    if kind is PoolLayer and type(below) is FullLayer:
        settings["C"] = below.nOut           # pooling over the outputs of a dense layer
        return
    settings["C"], settings["H"], settings["W"] = below.K, below.P, below.Q
    if kind is not Inception:
        return
    # every branch is a chain hanging off the layer below; the module's output
    # stacks the branch outputs along K, so their maps must agree
    branches, K = [], 0
    for branch_confs in settings.pop("partitions"):
        chain, tail = [], below
        for layer_conf in branch_confs:
            tail = Layer.create(lib, layer_conf, tail, dtype)
            chain.append(tail)
        branches.append(chain)
        K += tail.K
        if "P" in settings:
            assert (settings["P"], settings["Q"]) == (tail.P, tail.Q)
        else:
            settings["M"], settings["P"], settings["Q"] = tail.M, tail.P, tail.Q
    settings["partitions"] = branches
    settings["K"] = K


class DataLayer(Layer):
    """Input of a network: its output buffer holds the minibatch."""

    def __init__(self, lib, dtype, N, C, D=1, H=1, W=1):
        super(DataLayer, self).__init__(lib, dtype, N)
        self.C = self.K = C
        self.M, self.P, self.Q = D, H, W
        self.DHW = (D, H, W)
        self.dimI = self.dimO = (C, D, H, W, N)
        self.nOut = C * D * H * W
        self.dimI2 = self.dimO2 = (self.nOut, N)
        self.sizeI = self.sizeO = _count(self.dimO)

    def init_data(self, ary=None):
        if ary is not None:
            self.fprop_out.set(ary)
        else:
            self.fprop_out.fill(0)

    def init_deltas(self, shared=None):
        pass    # nothing flows back into the data

    def init_weights(self, loc=0.0, scale=0.1, shared=None, zeros=False):
        pass

    def fprop(self, fprop_in, scale_weights=0):
        return self.fprop_out

    def __str__(self):
        return "DataLayer: NCK: (%d, %d, %d) DHW:%s" % (self.N, self.C, self.K, self.DHW)


class FullLayer(Layer):
    """Dense layer on (features, N) matrices: three GEMMs per training step
    (nervanagpu/layers.py:254-273).

    Not in the reference, fp16 layers only, off by default:

    mx4     y = W x and dx = W^T e multiply 4-bit block-scaled copies of W, x and e
            (blocks along the contraction of each product, made in every step; they
            round stochastically if the backend does).  The weights themselves and
            their gradient stay as they are.  Pays from minibatches of about a thousand
            on (9216 -> 4096: a step of 4096 images 903 -> 659 us, of 128 108 -> 154).
    save8   the input is kept for the backward pass in 8 bits (saved_in): the weight
            gradient, and with relu_below the rectifier derivative of the layer
            below, are computed from what those stand for: NaN for the 32 values of a
            block that holds an infinity or a NaN.  The fp16 input may be overwritten
            once fprop has returned, so layers may share activation
            buffers (init_activations(shared=...)).
    """

    def __init__(self, lib, dtype, N, nIn, nOut, mx4=False, save8=False):
        super(FullLayer, self).__init__(lib, dtype, N)
        self.nIn, self.nOut = nIn, nOut
        self.dimI = self.dimI2 = (nIn, N)
        self.dimO = self.dimO2 = (nOut, N)
        self.dimF = self.dimF2 = (nOut, nIn)
        self.sizeI, self.sizeO, self.sizeF = nIn * N, nOut * N, nIn * nOut
        self.flops = N * nIn * nOut * 2.0
        if mx4 or save8:
            assert np.dtype(dtype).type is np.float16, "block-scaled layers are fp16 layers"
        self.mx4, self.save8 = mx4, save8
        self.relu_below = False         # with save8: apply (input > 0) to the error passed down
        self.saved_in = None
        self._mx = {}

    def _mx_copy(self, name, source, axis):
        """the 4-bit copy of `source` for one product, in a tensor kept for it"""
        if name not in self._mx:
            self._mx[name] = self.lib.mx_empty(source.shape, "fp4", axis)
        return self.lib.mx_quantize(source, self._mx[name])

    def init_activations(self, shared=None):
        """own output buffer, or a view of shared[0]; the list is then flipped, as
        in init_deltas.  Sharing needs save8 on every layer that reads a shared
        buffer, and relu_below there (the rectifier of an overwritten output is
        known from its 8-bit copy alone)."""
        if shared is None:
            return super(FullLayer, self).init_activations()
        self.fprop_out = shared[0].share(self.dimO)
        self.act_stats = self._stat_buffer(self.dimO2)
        shared.reverse()

    def fprop(self, fprop_in, scale_weights=0):
        x = super(FullLayer, self).fprop(fprop_in)
        if self.mx4:
            self.lib.mx_dot(self._mx_copy("W", self.weights, 1), self._mx_copy("x", x, 0), self.fprop_out, relu=True)
        else:
            self.lib.dot(self.weights, x, self.fprop_out, relu=True)        # y = relu(W x)
        if self.save8:
            if self.saved_in is None:
                self.saved_in = self.lib.mx_empty(self.dimI, "int8", 1, rounding=0)
            self.lib.mx_quantize(x, self.saved_in)
        self._rerun_scaled(x, scale_weights)
        return self.fprop_out

    def bprop(self, bprop_in):
        assert self.save8 or not self.relu_below, "relu_below of a dense layer needs save8"
        err = self.bprop_relu(bprop_in)
        if self.mx4:
            self.lib.mx_dot(self._mx_copy("W^T", self.weights, 0).T, self._mx_copy("e", err, 0), self.bprop_out)
        else:
            self.lib.dot(self.weights.T, err, self.bprop_out)               # dx = W^T e
        if self.save8:
            self.lib.mx_dot(err, self.saved_in.T, self.updat_out)
            if self.relu_below:
                self.lib.bprop_act("relu", self.saved_in, self.bprop_out, self.bprop_out)
        else:
            self.lib.dot(err, self.fprop_in.T, self.updat_out)              # dW = e x^T
        self.grad_descent()
        return self.bprop_out

    def __str__(self):
        return "FullLayer: N, nIn, nOut: (%d, %d, %d)" % (self.N, self.nIn, self.nOut)


class _PlanHandle(object):
    """owns a convolution plan of the HIP library"""

    def __init__(self, params, dtype_code):
        self.handle = ctypes.c_void_p()
        _lib.init()
        _lib.call("ng_conv_plan_create", ctypes.byref(params), dtype_code, ctypes.byref(self.handle))
        self.workspace_bytes = int(_lib.load().ng_conv_plan_workspace_bytes(self.handle))

    def __del__(self):
        try:
            if self.handle:
                _lib.load().ng_conv_plan_destroy(self.handle)
                self.handle = None
        except Exception:
            pass


class ConvLayer(Layer):
    """Geometry of one direct convolution: I (C,D,H,W,N) * F (C,T,R,S,K) ->
    O (K,M,P,Q,N) (nervanagpu/layers.py:279-326).  grid_P, grid_Q and update_size
    are accepted and ignored: in the reference they traded parallelism against
    fp32 accumulation depth of the weight-gradient kernels, here that gradient is
    always accumulated in fp32 and summed in a fixed order."""

    def __init__(self, lib, dtype,
                 N, C, K,
                 D=1, H=1, W=1,
                 T=1, R=1, S=1,
                 pad_d=0, pad_h=0, pad_w=0,
                 str_d=1, str_h=1, str_w=1,
                 grid_P=0, grid_Q=0, update_size=None):
        super(ConvLayer, self).__init__(lib, dtype, N, np.float32)
        assert N % 8 == 0, "N dim must be multiple of 8"
        assert K % 8 == 0, "K dim must be multiple of 8"
        self.np_dtype = np.dtype(dtype)
        assert self.np_dtype.type in (np.float16, np.float32), "conv filters must be fp16 or fp32"

        self.padding = (pad_d, pad_h, pad_w)
        self.strides = (str_d, str_h, str_w)
        self.DHW, self.TRS = (D, H, W), (T, R, S)
        self.MPQ = tuple(_out_extent(size, win, pad, strd)
                         for size, win, pad, strd in zip(self.DHW, self.TRS, self.padding, self.strides))
        assert min(self.MPQ) > 0, "filter does not fit the padded input"
        self.C, self.K = C, K
        self.M, self.P, self.Q = self.MPQ
        self.NCK = (N, C, K)

        self.dimI = (C,) + self.DHW + (N,)
        self.dimF = (C,) + self.TRS + (K,)
        self.dimFb = (K,) + self.TRS + (C,)
        self.dimO = (K,) + self.MPQ + (N,)
        taps, pixels_in, pixels_out = _count(self.TRS), _count(self.DHW), _count(self.MPQ)
        self.dimI2 = (C * pixels_in, N)
        self.dimF2, self.dimF2t = (C * taps, K), (K, C * taps)
        self.dimO2 = (K * pixels_out, N)
        self.sizeI, self.sizeF, self.sizeO = _count(self.dimI), _count(self.dimF), _count(self.dimO)
        self.nOut = pixels_out * K
        # multiply-adds counted twice, as the reference's benchmarks do (layers.py:422)
        self.flops = pixels_out * K * N * C * taps * 2.0

        self.grid_P, self.grid_Q, self.update_size = grid_P, grid_Q, update_size
        self._plan = None

    # -- the library's plan ---------------------------------------------------------

    def _params(self):
        return _lib.ConvParams(*(self.NCK + self.DHW + self.TRS + self.MPQ + self.padding + self.strides))

    def _get_plan(self):
        if self._plan is None:
            self._plan = _PlanHandle(self._params(),
                                     _lib.NG_F16 if self.np_dtype.type is np.float16 else _lib.NG_F32)
        return self._plan.handle

    def _workspace_bytes(self):
        self._get_plan()
        return self._plan.workspace_bytes

    # -- training step -----------------------------------------------------------------

    def fprop(self, fprop_in, scale_weights=0):
        x = super(ConvLayer, self).fprop(fprop_in)
        self.lib.fprop_conv(self, x, self.weights, self.fprop_out, relu=True)
        self._rerun_scaled(x, scale_weights)
        return self.fprop_out

    def bprop(self, bprop_in):
        err = self.bprop_relu(bprop_in)
        if self.bprop_out is not None:      # the first weighted layer has nothing below to feed
            self.lib.bprop_conv(self, self.weights, err, self.bprop_out,
                                relu_mask=getattr(self, "relu_mask_below", None))
        self.lib.update_conv(self, self.fprop_in, err, self.updat_out)
        self.grad_descent()
        return self.bprop_out

    def __str__(self):
        return "ConvLayer: NCK: (%d, %d, %d) DHW:%s TRS:%s MPQ:%s" % \
            (self.N, self.C, self.K, self.DHW, self.TRS, self.MPQ)


class DeconvLayer(ConvLayer):
    """A convolution described by its OUTPUT map P x Q (2-D only): the input
    extent is the smallest H x W that yields it.  Running the layer backwards
    (bprop_conv as the forward pass) is the deconvolution
    (nervanagpu/layers.py:509-537)."""

    def __init__(self, lib, dtype,
                 N, C, K,
                 P, Q,
                 R=1, S=1,
                 pad_d=0, pad_h=0, pad_w=0,
                 str_d=1, str_h=1, str_w=1,
                 grid_P=0, grid_Q=0, update_size=None):
        H = str_h * (P - 1) + R - 2 * pad_h
        W = str_w * (Q - 1) + S - 2 * pad_w
        super(DeconvLayer, self).__init__(
            lib, dtype, N, C, K, 1, H, W, 1, R, S,
            pad_d, pad_h, pad_w, str_d, str_h, str_w, grid_P, grid_Q, update_size)

    def __str__(self):
        return "DeconvLayer: NCK: (%d, %d, %d) DHW:%s TRS:%s MPQ:%s" % \
            (self.N, self.C, self.K, self.DHW, self.TRS, self.MPQ)


class PoolLayer(Layer):
    """Pooling window (J over feature maps, T,R,S over space) with its own pads
    and strides; a stride left out equals the window, i.e. the windows tile
    (nervanagpu/layers.py:540-590).  `overlap` is the number of windows covering
    an input element when they do overlap, else 0."""

    def __init__(self, lib, dtype,
                 op, N, C,
                 D=1, H=1, W=1,
                 J=1, T=1, R=1, S=1,
                 pad_j=0, pad_d=0, pad_h=0, pad_w=0,
                 str_j=None, str_d=None, str_h=None, str_w=None):
        super(PoolLayer, self).__init__(lib, dtype, N)
        self.op = op
        self.JTRS = (J, T, R, S)
        self.strides = tuple(win if strd is None else strd
                             for win, strd in zip(self.JTRS, (str_j, str_d, str_h, str_w)))
        self.padding = (pad_j, pad_d, pad_h, pad_w)
        self.DHW = (D, H, W)
        if any(strd < win for win, strd in zip(self.JTRS, self.strides)):
            self.overlap = 1.0
            for win, strd in zip(self.JTRS, self.strides):
                self.overlap *= ceil(float(win) / strd)
        else:
            self.overlap = 0.0

        extents = tuple(_out_extent(size, win, pad, strd)
                        for size, win, pad, strd in zip((C, D, H, W), self.JTRS, self.padding, self.strides))
        assert min(extents) > 0, "window does not fit the padded input"
        self.C = C
        self.K, self.M, self.P, self.Q = extents
        self.MPQ = extents[1:]

        self.dimI = (C, D, H, W, N)
        self.dimO = extents + (N,)
        self.dimF2 = None
        self.dimI2 = (C * D * H * W, N)
        self.nOut = _count(extents)
        self.dimO2 = (self.nOut, N)
        self.sizeI, self.sizeO = _count(self.dimI), _count(self.dimO)

    def _params(self):
        return _lib.PoolParams(*((self.N, self.C) + self.DHW + self.JTRS + (self.K,) + self.MPQ
                                 + self.padding + self.strides))

    def _workspace_bytes(self):
        # one argmax byte per output element, only for max pooling
        if self.op != "max":
            return 0
        params = self._params()
        return int(_lib.load().ng_pool_workspace_bytes(ctypes.byref(params), 0, 0))

    def fprop(self, fprop_in, scale_weights=0):
        x = super(PoolLayer, self).fprop(fprop_in)
        self.lib.fprop_pool(self, x, self.fprop_out)
        return self.fprop_out

    def bprop(self, bprop_in):
        self.lib.bprop_pool(self, self.fprop_in, bprop_in, self.bprop_out,
                            relu_mask=getattr(self, "relu_below", False))
        return self.bprop_out

    def __str__(self):
        return "PoolLayer: NCK: (%d, %d, %d) DHW:%s JTRS:%s MPQ:%s op: %s " % \
            (self.N, self.C, self.K, self.DHW, self.JTRS, self.MPQ, self.op)


class Inception(Layer):
    """Parallel branches (lists of layers) over one input whose outputs are
    stacked along K (nervanagpu/layers.py:643-755).  The tail of each branch
    writes straight into its K-slice of the module's output; the head of each
    branch writes the module's error buffer."""

    def __init__(self, lib, dtype, partitions,
                 N, C, K,
                 D=1, H=1, W=1,
                 M=1, P=1, Q=1):
        super(Inception, self).__init__(lib, dtype, N)
        self.partitions = partitions
        self.C, self.K = C, K
        self.M, self.P, self.Q = M, P, Q
        self.NCK, self.DHW, self.MPQ = (N, C, K), (D, H, W), (M, P, Q)
        self.dimI, self.dimO = (C, D, H, W, N), (K, M, P, Q, N)
        self.dimI2, self.dimO2 = (C * D * H * W, N), (K * M * P * Q, N)
        self.sizeI, self.sizeO = _count(self.dimI), _count(self.dimO)
        self.nOut = K * M * P * Q
        # flops add up; sizeF / dimF describe the largest filter inside (what a
        # shared weight-gradient buffer must hold)
        inner = self._inner_layers()
        self.flops = sum(layer.flops for layer in inner)
        self.sizeF = 0
        for layer in inner:
            if layer.sizeF and layer.sizeF >= self.sizeF:
                self.sizeF, self.dimF = layer.sizeF, layer.dimF

    def _inner_layers(self, backwards=False):
        if backwards:
            return [layer for branch in reversed(self.partitions) for layer in reversed(branch)]
        return [layer for branch in self.partitions for layer in branch]

    def init_activations(self):
        super(Inception, self).init_activations()
        first = 0
        for branch in self.partitions:
            for layer in branch[:-1]:
                layer.init_activations()
            tail = branch[-1]
            tail.fprop_out = self.fprop_out[first:first + tail.K, ...]
            tail.act_stats = self.lib.empty((tail.dimO2[0], 1), dtype=np.float32)
            first += tail.K

    def init_deltas(self, shared=None):
        super(Inception, self).init_deltas(shared)
        inside = shared[1:3]        # two more buffers alternate inside the module
        for branch in self.partitions:
            branch[0].bprop_out, branch[0].delta_stats = self.bprop_out, self.delta_stats
            for layer in branch[1:]:
                layer.init_deltas(shared=inside)

    def init_weights(self, loc=0.0, scale=0.1, shared=None, zeros=False):
        for layer in self._inner_layers():
            layer.init_weights(loc, scale, shared, zeros)

    def fprop(self, fprop_in, scale_weights=0):
        x = super(Inception, self).fprop(fprop_in)
        for branch in self.partitions:
            y = x
            for layer in branch:
                y = layer.fprop(y, scale_weights)
        return self.fprop_out

    def bprop(self, bprop_in):
        last = self.K
        for branch in reversed(self.partitions):
            width = branch[-1].K
            err = bprop_in[last - width:last, ...]
            last -= width
            for layer in reversed(branch):
                err = layer.bprop(err)
        return self.bprop_out

    def fprop_stats(self):
        for layer in self._inner_layers():
            layer.fprop_stats()

    def bprop_stats(self):
        for layer in self._inner_layers(backwards=True):
            layer.bprop_stats()

    def __str__(self):
        lines = ["Inception: NCK: (%d, %d, %d) DHW:%s MPQ:%s" % (self.N, self.C, self.K, self.DHW, self.MPQ)]
        for number, branch in enumerate(self.partitions, 1):
            lines.append("  Part%d:" % number)
            lines.extend("    %s" % layer for layer in branch)
        return "\n".join(lines)


def _magic32(nmax, d):
    """Magic number and shift for unsigned division by d of numerators <= nmax:
    n // d == (n * magic) >> shift  (Hacker's Delight magicgu;
    nervanagpu/layers.py:757-768)."""
    # With magic = ceil(2^shift / d) the product overshoots n/d by n*err/(d*2^shift),
    # err = magic*d - 2^shift.  The quotient stays exact as long as the worst
    # numerator (the largest n <= nmax with n % d == d-1) keeps that overshoot
    # below 1/d, i.e. worst * err < 2^shift.  Take the smallest such shift.
    worst = ((nmax + 1) // d) * d - 1
    for shift in range(2 * max(int(nmax).bit_length(), 1) + 1):
        magic = -((-1 << shift) // d)
        err = magic * d - (1 << shift)
        if worst * err < (1 << shift):
            return (magic, shift)
    raise ValueError("Can't find magic number for division")


def _flatten(lst):
    """flatten a nested list of lists or values"""
    return sum(([x] if not isinstance(x, (list, tuple)) else _flatten(x) for x in lst), [])


def _get_sm_count():
    """number of compute units of the current device"""
    return _lib.device_attr(0)
