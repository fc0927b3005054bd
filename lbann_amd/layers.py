"""Host-side mirror of the LBANN layer classes (layer norm, batch norm, softmax, log-softmax,
channelwise softmax; instance norm, entry-wise batch norm, cross entropy and the two scale/bias
layers) and of the operators around a transformer's residual stream and logits (dropout,
residual norm, logits adjustment), over the C ABI.

Each class of a reference layer keeps that layer's constructor parameters, its member
matrices and its two compute hooks, `fp_compute()` and `bp_compute()`
(include/lbann/layers/layer.hpp:835,852), and forwards them to liblbnorm.so; residual norm and
logits adjustment, which have no layer there, have forward() and backward() only.
A harness plays the role of data_type_layer::forward_prop / back_prop_impl_
(src/layers/data_type_layer.cpp:170-275, :292-376): it binds the input
matrices, sizes the outputs (left uninitialised, as the reference does) and
calls the hooks.

PyTorch is used for device memory and the HIP stream only; no arithmetic on the
path is done by torch, and there is no fallback when the library is missing.
"""
import functools
import operator
import weakref

import numpy as np
import torch

from . import capi
from .capi import LBN_STATS_REFERENCE_ORDER, LBN_STATS_SUMSQ, LBN_STATS_TWO_PASS, LbnError, call  # noqa: F401


def _prod(xs):
    return functools.reduce(operator.mul, xs, 1)


class DeviceMatrix:
    """Column-major matrix in device memory: Height/Width/LDim/Buffer of El::Matrix<T,GPU>.

    Backed by a torch tensor of shape (width, ldim); element (r, c) is tensor[c, r].
    """

    def __init__(self, height, width, dtype=torch.float32, ldim=None, device="cuda", fill=None):
        self.height, self.width = int(height), int(width)
        self.ldim = int(ldim) if ldim is not None else max(self.height, 1)
        assert self.ldim >= self.height
        self.tensor = torch.empty((max(self.width, 1), self.ldim), dtype=dtype, device=device)
        if fill is not None:
            self.tensor.fill_(fill)

    @classmethod
    def attach(cls, tensor, height):
        """View of a (width, ldim) tensor that someone else owns (El::Matrix::Attach); no copy."""
        if tensor.dim() != 2 or tensor.shape[1] < height or (tensor.shape[1] > 1 and tensor.stride(1) != 1):
            raise ValueError("attach takes a (width, ldim) tensor whose columns are contiguous and hold `height` entries")
        m = cls.__new__(cls)
        m.height, m.width = int(height), tensor.shape[0]
        m.ldim = int(tensor.stride(0)) if tensor.shape[0] > 1 else max(tensor.shape[1], 1)
        if m.ldim < m.height:
            raise ValueError("attach: columns overlap")
        m.tensor = tensor
        return m

    # El::Matrix vocabulary
    def Height(self):
        return self.height

    def Width(self):
        return self.width

    def LDim(self):
        return self.ldim

    def Buffer(self):
        return capi.vp(self.tensor.data_ptr())

    LockedBuffer = Buffer

    @property
    def dtype(self):
        return self.tensor.dtype

    @classmethod
    def from_numpy(cls, a, dtype=None, ldim=None, device="cuda"):
        """`a` has shape (height, width) (any memory order)."""
        a = np.asarray(a)
        h, w = a.shape
        tdt = dtype or {np.dtype("float32"): torch.float32, np.dtype("float16"): torch.float16,
                        np.dtype("float64"): torch.float64}[a.dtype]
        m = cls(h, w, dtype=tdt, ldim=ldim, device=device)
        if ldim is not None and ldim > h:
            m.tensor.fill_(float("nan"))  # padding rows must never be read or matter
        if w > 0 and h > 0:
            m.tensor[:w, :h] = torch.from_numpy(np.ascontiguousarray(a.T)).to(device=device, dtype=tdt)
        return m

    def to_numpy(self):
        """Returns an (height, width) array.  Results are consumed here: a wait between
        workgroups that ran out in any call since the last check raises ClusterWaitTimedOut."""
        check_cluster_waits()
        t = self.tensor[: self.width, : self.height]
        if t.dtype in (torch.float16, torch.bfloat16):
            t = t.float()
        return np.asfortranarray(t.cpu().numpy().T)


class _Vector:
    """Weights / gradient vector in device memory (fp32; binary64 for a layer of doubles)."""

    def __init__(self, n, device="cuda", values=None, dtype=torch.float32):
        if values is None:
            self.tensor = torch.empty(max(int(n), 1), dtype=dtype, device=device)
        else:
            npdt = np.float64 if dtype == torch.float64 else np.float32
            self.tensor = torch.as_tensor(np.asarray(values, dtype=npdt)).to(device).contiguous()
        self.n = int(n)

    def Buffer(self):
        return capi.vp(self.tensor.data_ptr())

    def to_numpy(self):
        check_cluster_waits()
        return self.tensor[: self.n].cpu().numpy()


_STORAGE = {torch.float32: "f32", torch.float16: "f16", torch.float64: "f64"}


def _storage(owner, types, *matrices):
    """Suffix of the entry points for the storage type that every matrix of a call has (None: no such matrix).  A type
    that the layer has no kernels for, bfloat16 among them, is refused: read as another type it would reach past its end."""
    kinds = {m.dtype for m in matrices if m is not None}
    if len(kinds) != 1:
        raise TypeError(f"{type(owner).__name__}: matrices of different types {sorted(map(str, kinds))}")
    suffix = _STORAGE.get(kinds.pop())
    if suffix not in types:
        raise TypeError(f"{type(owner).__name__}: storage is {' or '.join(types)}, not "
                        f"{next(m.dtype for m in matrices if m is not None)}")
    return suffix


def _stream():
    return capi.vp(torch.cuda.current_stream().cuda_stream)


def _null():
    return capi.vp(None)


class ClusterWaitTimedOut(LbnError):
    """A kernel in which workgroups wait for each other gave up on a wait (the sticky error
    word of a workspace is raised): the results of that call are undefined."""

    def __init__(self, where):
        RuntimeError.__init__(self, f"a bounded wait between workgroups ran out ({where}); "
                                    "results of that call are undefined")
        self.status = None


# Workspaces handed to a compute call since the last check: their error words are read where
# results are consumed (DeviceMatrix.to_numpy, which waits for the device anyway), so that a
# wait that ran out surfaces as an exception instead of as silently wrong numbers.  With
# LBN_CHECK_CLUSTER_WAITS=1 in the environment every fp_compute()/bp_compute() checks its own
# workspace right after the call (this synchronises: a debugging mode).
_PENDING = {}
_CHECK_EVERY_CALL = bool(int(__import__("os").environ.get("LBN_CHECK_CLUSTER_WAITS", "0") or 0))


def check_cluster_waits():
    """Raises ClusterWaitTimedOut if any workspace used since the last check has its error
    word raised; clears the word, so that the next use of the workspace starts clean."""
    pending = list(_PENDING.values())
    _PENDING.clear()
    for ws in pending:
        if ws.buf is None:
            continue
        flag = capi.cint(0)
        call("lbn_workspace_timed_out", _stream(), capi.vp(ws.buf.data_ptr()), flag)
        if flag.value:
            ws.buf[:64].zero_()
            raise ClusterWaitTimedOut(f"workspace of {ws.owner}")


def _after_call():
    """The debugging mode's check after a compute call.  It waits for the device, which a stream
    that is being captured into a HIP graph does not allow: calls recorded into a graph are
    checked where their results are consumed, like every call outside the debugging mode."""
    if _CHECK_EVERY_CALL and not torch.cuda.is_current_stream_capturing():
        check_cluster_waits()


class _Workspace:
    """Scratch memory owned by a layer, grown on demand (never shrunk).  The first 64 bytes
    (the error word of the kernels that wait across workgroups) are cleared when the memory
    is allocated: recycled device memory may hold anything."""

    def __init__(self, owner="a layer", header=True):
        self.buf = None
        self.owner = owner
        self.header = header  # False: scratch of a layer none of whose kernels wait across workgroups

    def get(self, nbytes, device):
        nbytes = int(nbytes)
        if nbytes == 0:
            return _null(), 0
        if self.buf is None or self.buf.numel() < nbytes:
            self.buf = torch.empty(max(nbytes, 64), dtype=torch.uint8, device=device)
            self.buf[:64].zero_()
        if self.header:
            _PENDING[id(self)] = self
        return capi.vp(self.buf.data_ptr()), nbytes


class _Layer:
    """Members every data_type_layer hands to its compute hooks."""

    def __init__(self, device="cuda"):
        self.device = device
        self.prev_activations = None    # input x
        self.activations = None         # output y
        self.prev_error_signals = None  # dL/dy
        self.error_signals = None       # dL/dx
        self._ws = _Workspace(type(self).__name__)

    # what fp_setup_inputs/outputs and bp_setup_gradient_wrt_inputs do
    def bind_forward(self, x, in_place=False):
        self.prev_activations = x
        if in_place:
            self.activations = x
        else:
            self.activations = DeviceMatrix(x.height, x.width, dtype=x.dtype, ldim=x.ldim, device=self.device)

    def bind_backward(self, dy, in_place=False):
        self.prev_error_signals = dy
        if in_place:
            self.error_signals = dy
        else:
            self.error_signals = DeviceMatrix(dy.height, dy.width, dtype=dy.dtype, ldim=dy.ldim, device=self.device)

    # fp_call()/bp_call() return (entry point name, argument tuple) of the C-ABI call
    # that is the body of the reference's fp_compute()/bp_compute().
    def fp_compute(self):
        name, args = self.fp_call()
        call(name, *args)
        _after_call()

    def bp_compute(self):
        name, args = self.bp_call()
        call(name, *args)
        _after_call()

    def forward(self, x, in_place=False):
        self.bind_forward(x, in_place)
        self.fp_compute()
        if in_place and _SAVED:
            _wrote_over(x)
        return self.activations

    def backward(self, dy, in_place=False):
        self.bind_backward(dy, in_place)
        self.bp_compute()
        if in_place and _SAVED:
            _wrote_over(dy)
        return self.error_signals


class layer_norm_layer(_Layer):
    """lbann::layer_norm_layer (include/lbann/layers/regularizers/layer_norm.hpp:53-143)."""

    def __init__(self, dims, epsilon=1e-5, scale=False, bias=False, start_dim=0,
                 scale_values=None, bias_values=None, stats_mode=LBN_STATS_TWO_PASS, device="cuda",
                 datatype=torch.float32):
        """datatype: the reference's TensorDataType; torch.float64 selects the _f64 entry points
        (weights, statistics and their gradients are then doubles as well)."""
        super().__init__(device)
        self.datatype = wt = torch.float64 if datatype == torch.float64 else torch.float32
        self.dims = tuple(int(d) for d in dims)
        self.m_epsilon, self.m_scale, self.m_bias, self.m_start_dim = float(epsilon), bool(scale), bool(bias), int(start_dim)
        sd = self.m_start_dim if self.m_start_dim >= 0 else len(self.dims) + self.m_start_dim
        if sd < 0 or sd >= len(self.dims):
            raise ValueError(f"layer norm start dimension {start_dim} does not match tensor dimensionality {len(self.dims)}")
        # get_normdims (layer_norm.hpp:362-405)
        self.num_normalized = _prod(self.dims[:sd])
        self.normalization_size = _prod(self.dims[sd:])
        self.normalization_stride = self.normalization_size
        n = self.normalization_size
        self.weights = []
        if self.m_scale:
            self.weights.append(_Vector(n, device, scale_values if scale_values is not None else np.ones(n), wt))
        if self.m_bias:
            self.weights.append(_Vector(n, device, bias_values if bias_values is not None else np.zeros(n), wt))
        self.m_scale_gradient = _Vector(n, device, dtype=wt) if self.m_scale else None
        self.m_bias_gradient = _Vector(n, device, dtype=wt) if self.m_bias else None
        self.m_statistics = None
        self.m_statistics_gradient = None
        self.stats_mode = stats_mode

    def _suffix(self, *matrices):
        return _storage(self, ("f64",) if self.datatype == torch.float64 else ("f32", "f16"), *matrices)

    def _scratch(self):
        """One scratch buffer for both directions, sized for the larger need, so that neither
        call's bound pointer is invalidated by the other growing it."""
        x = self.prev_activations
        G, n = self.num_normalized, self.normalization_size
        esize = 2 if x.dtype == torch.float16 else 4
        lib = capi.lib()
        if self.datatype == torch.float64:
            self._ws.header = False
            return self._ws.get(lib.lbn_layer_norm_bwd_workspace_bytes_f64(G, n, x.width, int(self.m_scale or self.m_bias)),
                                self.device)
        need = max(lib.lbn_layer_norm_fwd_workspace_bytes(G, n, x.width, esize),
                   lib.lbn_layer_norm_bwd_workspace_bytes(G, n, x.width, int(self.m_scale or self.m_bias), esize))
        return self._ws.get(need, self.device)

    def fp_call(self):
        x, y = self.prev_activations, self.activations
        suffix = self._suffix(x, y)
        G, n = self.num_normalized, self.normalization_size
        if self.m_statistics is None or self.m_statistics.width != x.width:
            self.m_statistics = DeviceMatrix(2 * G, x.width, dtype=self.datatype, device=self.device)
        scale = self.weights[0].Buffer() if self.m_scale else _null()
        bias = self.weights[-1].Buffer() if self.m_bias else _null()
        ws, nb = self._scratch()
        if self.datatype == torch.float64:  # no forward scratch
            return ("lbn_layer_norm_fwd_f64",
                    (_stream(), G, n, self.normalization_stride, x.width,
                     self.m_epsilon, x.Buffer(), x.ldim, y.Buffer(), y.ldim, self.m_statistics.Buffer(),
                     self.m_statistics.ldim, scale, bias, self.stats_mode))
        return (f"lbn_layer_norm_fwd_{suffix}",
                (_stream(), G, n, self.normalization_stride, x.width,
                 self.m_epsilon, x.Buffer(), x.ldim, y.Buffer(), y.ldim, self.m_statistics.Buffer(),
                 self.m_statistics.ldim, scale, bias, ws, nb, self.stats_mode))

    def bp_call(self):
        x, dy, dx = self.prev_activations, self.prev_error_signals, self.error_signals
        suffix = self._suffix(x, dy, dx)
        G, n = self.num_normalized, self.normalization_size
        if self.m_statistics_gradient is None or self.m_statistics_gradient.width != x.width:
            self.m_statistics_gradient = DeviceMatrix(2 * G, x.width, dtype=self.datatype, device=self.device)
        scale = self.weights[0].Buffer() if self.m_scale else _null()
        dscale = self.m_scale_gradient.Buffer() if self.m_scale else _null()
        dbias = self.m_bias_gradient.Buffer() if self.m_bias else _null()
        ws, nb = self._scratch()
        return (f"lbn_layer_norm_bwd_{suffix}",
                (_stream(), G, n, self.normalization_stride, x.width,
                 self.m_epsilon, x.Buffer(), x.ldim, dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim,
                 self.m_statistics.Buffer(), self.m_statistics.ldim, self.m_statistics_gradient.Buffer(),
                 self.m_statistics_gradient.ldim, scale, dscale, dbias, ws, nb))


class instance_norm_layer(_Layer):
    """lbann::instance_norm_layer (include/lbann/layers/regularizers/instance_norm.hpp):
    channels = leading output dimension, every (sample, channel) slab normalised on its own."""

    def __init__(self, dims, epsilon=1e-5, device="cuda"):
        super().__init__(device)
        self.dims = tuple(int(d) for d in dims)
        self.m_epsilon = float(epsilon)
        self.num_channels = self.dims[0]
        self.channel_size = _prod(self.dims) // self.num_channels
        self.m_workspace = None  # (2*channels x width): means, then variances
        self._ws_fwd = _Workspace("instance_norm_layer (forward)")  # forward scratch of its own: backward's holds the statistics gradients

    def fp_call(self):
        x, y = self.prev_activations, self.activations
        _storage(self, ("f32",), x, y)
        if self.m_workspace is None or self.m_workspace.width != x.width:
            self.m_workspace = DeviceMatrix(2 * self.num_channels, x.width, device=self.device)
        ws, nb = self._ws_fwd.get(capi.lib().lbn_instance_norm_fwd_workspace_bytes(
            self.num_channels, self.channel_size, x.width), self.device)
        return ("lbn_instance_norm_fwd_f32",
                (_stream(), self.num_channels, self.channel_size, x.width, self.m_epsilon, x.Buffer(),
                 x.ldim, y.Buffer(), y.ldim, self.m_workspace.Buffer(), self.m_workspace.ldim, ws, nb))

    def bp_call(self):
        x, dy, dx = self.prev_activations, self.prev_error_signals, self.error_signals
        _storage(self, ("f32",), x, dy, dx)
        ws, nb = self._ws.get(capi.lib().lbn_instance_norm_bwd_workspace_bytes(
            self.num_channels, self.channel_size, x.width), self.device)
        return ("lbn_instance_norm_bwd_f32",
                (_stream(), self.num_channels, self.channel_size, x.width, self.m_epsilon, x.Buffer(),
                 x.ldim, dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim, self.m_workspace.Buffer(),
                 self.m_workspace.ldim, ws, nb))


class entrywise_batch_normalization_layer(_Layer):
    """lbann::entrywise_batch_normalization_layer
    (include/lbann/layers/regularizers/entrywise_batch_normalization.hpp): per-entry statistics
    over the mini-batch; weights[0] running mean, weights[1] running variance.

    `comm_allreduce(matrix)` stands for the reference's comm.allreduce over the mini-batch's
    ranks (entrywise_batch_normalization.cpp:97-100, :301-303): when given, it is called on the
    (height x 2) matrix of local sums, which it must replace by their sum over the ranks, and
    `statistics_count` is the global mini-batch size (input.Width() there); the layer then
    runs the split entry points around it."""

    def __init__(self, dims, decay=0.9, epsilon=1e-5, device="cuda", comm_allreduce=None, statistics_count=None):
        super().__init__(device)
        self.dims = tuple(int(d) for d in dims)
        self.m_decay, self.m_epsilon = float(decay), float(epsilon)
        self.comm_allreduce, self.statistics_count = comm_allreduce, statistics_count
        h = _prod(self.dims)
        # default weights (entrywise_batch_normalization.hpp:159-176): mean 0, variance 1
        self.weights = [_Vector(h, device, np.zeros(h)), _Vector(h, device, np.ones(h))]
        self.m_batch_statistics = DeviceMatrix(h, 2, device=device)
        self.m_batch_statistics_gradient = DeviceMatrix(h, 2, device=device)
        self.training = True
        self._ws = _Workspace(type(self).__name__, header=False)  # partial sums only: no kernel of this layer waits

    def _scratch(self):
        x = self.prev_activations
        return self._ws.get(capi.lib().lbn_entrywise_batch_norm_workspace_bytes(x.height, x.width), self.device)

    def fp_call(self):
        x, y = self.prev_activations, self.activations
        _storage(self, ("f32",), x, y)
        st = self.m_batch_statistics
        ws, nb = self._scratch()
        return ("lbn_entrywise_batch_norm_fwd_f32",
                (_stream(), x.height, x.width, self.m_decay, self.m_epsilon, int(self.training), x.Buffer(),
                 x.ldim, y.Buffer(), y.ldim, st.Buffer(), st.ldim, self.weights[0].Buffer(),
                 self.weights[1].Buffer(), ws, nb))

    def bp_call(self):
        x, dy, dx = self.prev_activations, self.prev_error_signals, self.error_signals
        _storage(self, ("f32",), x, dy, dx)
        st, sg = self.m_batch_statistics, self.m_batch_statistics_gradient
        ws, nb = self._scratch()
        return ("lbn_entrywise_batch_norm_bwd_f32",
                (_stream(), x.height, x.width, self.m_epsilon, int(self.training), x.Buffer(), x.ldim,
                 dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim, st.Buffer(), st.ldim, sg.Buffer(), sg.ldim,
                 self.weights[1].Buffer(), ws, nb))

    def _col(self, m, j):
        return capi.vp(m.tensor.data_ptr() + 4 * j * m.ldim)

    def fp_compute(self):
        if self.comm_allreduce is None:
            return super().fp_compute()
        x, y, st = self.prev_activations, self.activations, self.m_batch_statistics
        _storage(self, ("f32",), x, y)
        if self.training:
            count = int(self.statistics_count if self.statistics_count is not None else x.width)
            call("lbn_entrywise_batch_norm_fwd_sums_f32", _stream(), x.height, x.width, x.Buffer(), x.ldim,
                 st.Buffer(), st.ldim)
            self.comm_allreduce(st)
            call("lbn_entrywise_batch_norm_fwd_stats_f32", _stream(), x.height, count, self.m_decay, st.Buffer(),
                 st.ldim, self.weights[0].Buffer(), self.weights[1].Buffer())
            mean, var = self._col(st, 0), self._col(st, 1)
        else:
            mean, var = self.weights[0].Buffer(), self.weights[1].Buffer()
        call("lbn_entrywise_batch_norm_fwd_apply_f32", _stream(), x.height, x.width, self.m_epsilon, x.Buffer(), x.ldim,
             y.Buffer(), y.ldim, mean, var)

    def bp_compute(self):
        if self.comm_allreduce is None or not self.training:
            return super().bp_compute()
        x, dy, dx = self.prev_activations, self.prev_error_signals, self.error_signals
        _storage(self, ("f32",), x, dy, dx)
        st, sg = self.m_batch_statistics, self.m_batch_statistics_gradient
        count = int(self.statistics_count if self.statistics_count is not None else x.width)
        if count > 1:
            call("lbn_entrywise_batch_norm_bwd_sums_f32", _stream(), x.height, x.width, self.m_epsilon, x.Buffer(),
                 x.ldim, dy.Buffer(), dy.ldim, st.Buffer(), st.ldim, sg.Buffer(), sg.ldim)
            self.comm_allreduce(sg)
        call("lbn_entrywise_batch_norm_bwd_apply_f32", _stream(), x.height, x.width, count, self.m_epsilon, x.Buffer(),
             x.ldim, dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim, st.Buffer(), st.ldim, sg.Buffer(), sg.ldim)


class batch_normalization_layer(_Layer):
    """lbann::batch_normalization_layer (include/lbann/layers/regularizers/batch_normalization.hpp:130-199),
    local statistics (statistics_group_size == 1)."""

    def __init__(self, dims, decay=0.9, epsilon=1e-5, bessel_correction=True, scale_values=None,
                 bias_values=None, stats_mode=LBN_STATS_TWO_PASS, device="cuda", datatype=torch.float32):
        super().__init__(device)
        self.datatype = wt = torch.float64 if datatype == torch.float64 else torch.float32
        self.dims = tuple(int(d) for d in dims)
        self.m_decay, self.m_epsilon, self.m_bessel_correction = float(decay), float(epsilon), bool(bessel_correction)
        self.num_channels = self.dims[0]
        self.channel_size = _prod(self.dims[1:])
        C = self.num_channels
        # weights 0..3: scale, bias, running mean, running variance (defaults 1, 0, 0, 1)
        self.weights = [
            _Vector(C, device, scale_values if scale_values is not None else np.ones(C), wt),
            _Vector(C, device, bias_values if bias_values is not None else np.zeros(C), wt),
            _Vector(C, device, np.zeros(C), wt),
            _Vector(C, device, np.ones(C), wt),
        ]
        # m_mean_and_var / m_mean_and_var_gradient: C x 2, column 0 mean, column 1 variance
        self.m_mean_and_var = DeviceMatrix(C, 2, dtype=wt, device=device)
        self.m_mean_and_var_gradient = DeviceMatrix(C, 2, dtype=wt, device=device)
        self.m_scale_gradient = _Vector(C, device, dtype=wt)
        self.m_bias_gradient = _Vector(C, device, dtype=wt)
        self.training = True
        self.stats_mode = stats_mode

    def _col(self, m, j):
        return capi.vp(m.tensor.data_ptr() + m.tensor.element_size() * j * m.ldim)

    def _scratch(self, width):
        C, cs = self.num_channels, self.channel_size
        if self.datatype == torch.float64:
            self._ws.header = False
            return self._ws.get(capi.lib().lbn_batch_norm_workspace_bytes_f64(C, cs, width), self.device)
        return self._ws.get(capi.lib().lbn_batch_norm_workspace_bytes(C, cs, width), self.device)

    def _suffix(self, *matrices):
        return _storage(self, ("f64",) if self.datatype == torch.float64 else ("f32", "f16"), *matrices)

    def fp_call(self):
        x, y = self.prev_activations, self.activations
        suffix = self._suffix(x, y)
        C, cs = self.num_channels, self.channel_size
        ws, nb = self._scratch(x.width)
        return (f"lbn_batch_norm_fwd_{suffix}",
                (_stream(), C, cs, x.width, int(self.m_bessel_correction),
                 self.m_epsilon, self.m_decay, int(self.training), x.Buffer(), x.ldim, y.Buffer(), y.ldim,
                 self._col(self.m_mean_and_var, 0), self._col(self.m_mean_and_var, 1),
                 self.weights[0].Buffer(), self.weights[1].Buffer(), self.weights[2].Buffer(),
                 self.weights[3].Buffer(), ws, nb, self.stats_mode))

    def bp_call(self):
        x, dy, dx = self.prev_activations, self.prev_error_signals, self.error_signals
        suffix = self._suffix(x, dy, dx)
        C, cs = self.num_channels, self.channel_size
        ws, nb = self._scratch(x.width)
        name = f"lbn_batch_norm_bwd_{suffix}"
        if self.stats_mode & LBN_STATS_REFERENCE_ORDER and self.datatype != torch.float64:  # parity tests: the reference's order of summation
            _storage(self, ("f32",), x)
            name = "lbn_batch_norm_bwd_reference_order_f32"
        return (name,
                (_stream(), C, cs, x.width, int(self.m_bessel_correction),
                 self.m_epsilon, int(self.training), x.Buffer(), x.ldim, dy.Buffer(), dy.ldim, dx.Buffer(),
                 dx.ldim, self._col(self.m_mean_and_var, 0), self._col(self.m_mean_and_var, 1),
                 self.weights[2].Buffer(), self.weights[3].Buffer(), self.weights[0].Buffer(),
                 self.m_scale_gradient.Buffer(), self.m_bias_gradient.Buffer(),
                 self._col(self.m_mean_and_var_gradient, 0), self._col(self.m_mean_and_var_gradient, 1), ws, nb))


class _softmax_like(_Layer):
    _name = None

    def _suffix(self, *matrices):
        return _storage(self, ("f32", "f16", "f64"), *matrices)

    def fp_call(self):
        x, y = self.prev_activations, self.activations
        suffix = self._suffix(x, y)
        if x.dtype == torch.float64:  # TensorDataType = double: no scratch
            return (f"lbn_{self._name}_fwd_f64", (_stream(), x.height, x.width, x.Buffer(), x.ldim, y.Buffer(), y.ldim))
        ws, nb = self._ws.get(capi.lib().lbn_softmax_workspace_bytes(x.height, x.width), self.device)
        return (f"lbn_{self._name}_fwd_{suffix}",
                (_stream(), x.height, x.width, x.Buffer(), x.ldim, y.Buffer(), y.ldim, ws, nb))

    def bp_call(self):
        y, dy, dx = self.activations, self.prev_error_signals, self.error_signals
        suffix = self._suffix(y, dy, dx)
        if y.dtype == torch.float64:
            return (f"lbn_{self._name}_bwd_f64",
                    (_stream(), y.height, y.width, y.Buffer(), y.ldim, dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim))
        ws, nb = self._ws.get(capi.lib().lbn_softmax_workspace_bytes(y.height, y.width), self.device)
        return (f"lbn_{self._name}_bwd_{suffix}",
                (_stream(), y.height, y.width, y.Buffer(), y.ldim, dy.Buffer(), dy.ldim, dx.Buffer(),
                 dx.ldim, ws, nb))


class softmax_layer(_softmax_like):
    """lbann::softmax_layer, data-parallel layout, softmax_mode::INSTANCE
    (include/lbann/layers/activations/softmax.hpp:85-262)."""
    _name = "softmax"

    def __init__(self, mode="instance", device="cuda"):
        super().__init__(device)
        if mode != "instance":
            # the reference's CPU path rejects every other mode (openmp/softmax.hpp:61-63)
            raise ValueError("Unsupported softmax mode")


class log_softmax_layer(_softmax_like):
    """lbann::log_softmax_layer (include/lbann/layers/activations/log_softmax.hpp)."""
    _name = "log_softmax"


class channelwise_softmax_layer(_Layer):
    """lbann::channelwise_softmax_layer (include/lbann/layers/misc/channelwise_softmax.hpp:50-107)."""

    def __init__(self, dims, dim=0, single_dim_mode=False, device="cuda"):
        super().__init__(device)
        self.dims = tuple(int(d) for d in dims)
        nd = len(self.dims)
        if dim < -nd or dim >= nd:
            raise ValueError(f"Dimension {dim} is out of bounds for Channelwise Softmax layer on tensor with {nd} dimensions.")
        if not single_dim_mode and dim not in (0, -nd, nd - 1, -1):
            raise ValueError("Channelwise softmax with all dimensions is only supported for the first or last tensor dimensions.")
        self.m_dim, self.m_single_dim_mode = int(dim), bool(single_dim_mode)

    def get_channel_size_and_stride(self):
        """(channel_size, channel_stride, num_channels), channelwise_softmax_impl.hpp:58-104."""
        dims = self.dims
        d = self.m_dim + len(dims) if self.m_dim < 0 else self.m_dim
        total = _prod(dims)
        if self.m_single_dim_mode:
            cs = dims[d]
            return cs, _prod(dims[d:]), total // cs
        cs = total // dims[d]
        return cs, (cs if d == 0 else 1), dims[d]

    def fp_call(self):
        x, y = self.prev_activations, self.activations
        _storage(self, ("f32", "f64"), x, y)
        cs, stride, C = self.get_channel_size_and_stride()
        if x.dtype == torch.float64:
            return ("lbn_channelwise_softmax_fwd_f64",
                    (_stream(), C, cs, stride, x.width, x.Buffer(), x.ldim, y.Buffer(), y.ldim))
        ws, nb = self._ws.get(capi.lib().lbn_channelwise_softmax_workspace_bytes(C, cs, x.width), self.device)
        return ("lbn_channelwise_softmax_fwd_f32",
                (_stream(), C, cs, stride, x.width, x.Buffer(), x.ldim, y.Buffer(), y.ldim, ws, nb))

    def bp_call(self):
        y, dy, dx = self.activations, self.prev_error_signals, self.error_signals
        _storage(self, ("f32", "f64"), y, dy, dx)
        cs, stride, C = self.get_channel_size_and_stride()
        if y.dtype == torch.float64:
            return ("lbn_channelwise_softmax_bwd_f64",
                    (_stream(), C, cs, stride, y.width, y.Buffer(), y.ldim, dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim))
        ws, nb = self._ws.get(capi.lib().lbn_channelwise_softmax_workspace_bytes(C, cs, y.width), self.device)
        return ("lbn_channelwise_softmax_bwd_f32",
                (_stream(), C, cs, stride, y.width, y.Buffer(), y.ldim, dy.Buffer(), dy.ldim, dx.Buffer(),
                 dx.ldim, ws, nb))


class _scale_bias_layer(_Layer):
    """Shared state of the two scale/bias layers: one weights matrix (n x 2), column 0 scale
    (default 1), column 1 bias (default 0), and m_weights_gradient of the same shape."""

    def _setup_weights(self, n, device):
        self.weights = DeviceMatrix(n, 2, device=device)
        self.weights.tensor[0].fill_(1.0)
        self.weights.tensor[1].fill_(0.0)
        self.m_weights_gradient = DeviceMatrix(n, 2, device=device)

    def set_weights(self, scale, bias):
        n = self.weights.height
        self.weights.tensor[0, :n] = torch.as_tensor(np.asarray(scale, np.float32).reshape(-1)).to(self.device)
        self.weights.tensor[1, :n] = torch.as_tensor(np.asarray(bias, np.float32).reshape(-1)).to(self.device)


class entrywise_scale_bias_layer(_scale_bias_layer):
    """lbann::entrywise_scale_bias_layer (include/lbann/layers/learning/entrywise_scale_bias.hpp:57-203)."""

    def __init__(self, dims, device="cuda"):
        super().__init__(device)
        self.dims = tuple(int(d) for d in dims)
        self._setup_weights(_prod(self.dims), device)

    def fp_call(self):
        x, y, wt = self.prev_activations, self.activations, self.weights
        _storage(self, ("f32",), x, y)
        return ("lbn_entrywise_scale_bias_fwd_f32",
                (_stream(), x.height, x.width, x.Buffer(), x.ldim, y.Buffer(), y.ldim, wt.Buffer(), wt.ldim))

    def bp_call(self):
        x, dy, dx = self.prev_activations, self.prev_error_signals, self.error_signals
        _storage(self, ("f32",), x, dy, dx)
        wt, wg = self.weights, self.m_weights_gradient
        self._ws.header = False
        ws, nb = self._ws.get(capi.lib().lbn_entrywise_scale_bias_bwd_workspace_bytes(x.height, x.width),
                              self.device)
        return ("lbn_entrywise_scale_bias_bwd_f32",
                (_stream(), x.height, x.width, x.Buffer(), x.ldim, dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim,
                 wt.Buffer(), wt.ldim, wg.Buffer(), wg.ldim, ws, nb))


class channelwise_scale_bias_layer(_scale_bias_layer):
    """lbann::channelwise_scale_bias_layer (include/lbann/layers/learning/channelwise_scale_bias.hpp:60-206)."""

    def __init__(self, dims, device="cuda"):
        super().__init__(device)
        self.dims = tuple(int(d) for d in dims)
        self.num_channels = self.dims[0]
        self.channel_size = _prod(self.dims[1:])
        self._setup_weights(self.num_channels, device)

    def fp_call(self):
        x, y, wt = self.prev_activations, self.activations, self.weights
        _storage(self, ("f32",), x, y)
        return ("lbn_channelwise_scale_bias_fwd_f32",
                (_stream(), self.num_channels, self.channel_size, x.width, x.Buffer(), x.ldim, y.Buffer(), y.ldim,
                 wt.Buffer(), wt.ldim))

    def bp_call(self):
        x, dy, dx = self.prev_activations, self.prev_error_signals, self.error_signals
        _storage(self, ("f32",), x, dy, dx)
        wt, wg = self.weights, self.m_weights_gradient
        C, cs = self.num_channels, self.channel_size
        self._ws.header = False
        ws, nb = self._ws.get(capi.lib().lbn_channelwise_scale_bias_bwd_workspace_bytes(C, cs, x.width), self.device)
        return ("lbn_channelwise_scale_bias_bwd_f32",
                (_stream(), C, cs, x.width, x.Buffer(), x.ldim, dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim,
                 wt.Buffer(), wt.ldim, wg.Buffer(), wg.ldim, ws, nb))


class cross_entropy_layer:
    """lbann::cross_entropy_layer (include/lbann/layers/loss/cross_entropy.hpp:75-190): two
    parents (prediction, ground truth), output of dims {1}.  `dims` are the prediction's
    dimensions; with use_labels the ground truth has dims (1, dims[1:]) and holds class
    indices (cross_entropy_impl.hpp:59-133)."""

    def __init__(self, dims, use_labels=False, device="cuda"):
        self.device = device
        self.dims = tuple(int(d) for d in dims)
        self.m_use_labels = bool(use_labels)
        if self.m_use_labels and len(self.dims) < 2:
            raise ValueError("cross entropy layer expects both input tensors to have the same number of "
                             "dimensions and have >2 dimensions when use_labels is enabled.")
        self.spatial_sample_size = _prod(self.dims[1:])
        self.prev_activations = [None, None]
        self.activations = None
        self.prev_error_signals = None
        self.error_signals = [None, None]
        self._ws = _Workspace("cross_entropy_layer", header=False)

    def _suffix(self, *matrices):
        """fp32 or fp16 storage (the reference instantiates the layer for both,
        cross_entropy.cpp:157-166); every matrix of a call has the layer's one data type."""
        return _storage(self, ("f32", "f16"), *matrices)

    def fp_call(self):
        x, t, y = self.prev_activations[0], self.prev_activations[1], self.activations
        suffix = self._suffix(x, t, y)
        ws, nb = self._ws.get(capi.lib().lbn_cross_entropy_fwd_workspace_bytes(x.height, x.width), self.device)
        return (f"lbn_cross_entropy_fwd_{suffix}",
                (_stream(), x.height, x.width, int(self.m_use_labels), self.spatial_sample_size, x.Buffer(), x.ldim,
                 t.Buffer(), t.ldim, y.Buffer(), y.ldim, ws, nb))

    def bp_call(self):
        x, t, dy = self.prev_activations[0], self.prev_activations[1], self.prev_error_signals
        dx, dt = self.error_signals
        return (f"lbn_cross_entropy_bwd_{self._suffix(x, t, dy, dx, dt)}",
                (_stream(), x.height, x.width, int(self.m_use_labels), self.spatial_sample_size, x.Buffer(), x.ldim,
                 t.Buffer(), t.ldim, dy.Buffer(), dy.ldim, dx.Buffer(), dx.ldim,
                 dt.Buffer() if dt is not None else _null(), dt.ldim if dt is not None else 0))

    def fp_compute(self):
        name, args = self.fp_call()
        call(name, *args)
        _after_call()

    def bp_compute(self):
        name, args = self.bp_call()
        call(name, *args)
        _after_call()

    def forward(self, prediction, ground_truth):
        self.prev_activations = [prediction, ground_truth]
        self.activations = DeviceMatrix(1, prediction.width, dtype=prediction.dtype, device=self.device)
        self.fp_compute()
        return self.activations

    def backward(self, dy):
        """dy: (1 x width) gradient w.r.t. the loss.  Returns [dL/dprediction, dL/dground_truth];
        the second is None with use_labels (the reference leaves that error signal untouched)."""
        x, t = self.prev_activations
        self.prev_error_signals = dy
        self.error_signals = [DeviceMatrix(x.height, x.width, dtype=x.dtype, ldim=x.ldim, device=self.device),
                              None if self.m_use_labels else DeviceMatrix(t.height, t.width, dtype=t.dtype,
                                                                          ldim=t.ldim, device=self.device)]
        self.bp_compute()
        return self.error_signals


def softmax_cross_entropy_forward(softmax, cross_entropy, x, ground_truth):
    """Forward of a softmax_layer whose only child is a cross_entropy_layer, in one call
    (lbn_softmax_cross_entropy_fwd_f32): what softmax.forward(x) followed by
    cross_entropy.forward(y, ground_truth) computes, with both layers' members bound as
    those two calls bind them, so each layer's backward runs unchanged afterwards.
    Returns (y, loss).  fp32 storage only."""
    _storage(softmax, ("f32",), x, ground_truth)
    softmax.bind_forward(x)
    y = softmax.activations
    cross_entropy.prev_activations = [y, ground_truth]
    cross_entropy.activations = DeviceMatrix(1, x.width, device=cross_entropy.device)
    loss = cross_entropy.activations
    ws, nb = softmax._ws.get(capi.lib().lbn_softmax_cross_entropy_fwd_workspace_bytes(x.height, x.width), softmax.device)
    call("lbn_softmax_cross_entropy_fwd_f32", _stream(), x.height, x.width, int(cross_entropy.m_use_labels),
         cross_entropy.spatial_sample_size, x.Buffer(), x.ldim, ground_truth.Buffer(), ground_truth.ldim,
         y.Buffer(), y.ldim, loss.Buffer(), loss.ldim, ws, nb)
    _after_call()
    return y, loss


def softmax_cross_entropy_backward(softmax, cross_entropy, dloss, want_dtruth=False):
    """Backward of the pair in one call (lbn_softmax_cross_entropy_bwd_f32): what
    cross_entropy.backward(dloss) followed by softmax.backward(dprediction) computes, without
    the gradient with respect to the prediction ever being written.  The layers must have run
    their forward (together or one after the other).  Returns dx; cross_entropy.error_signals
    becomes [None, dtruth or None]."""
    y, truth = cross_entropy.prev_activations
    if y is not softmax.activations:
        raise ValueError("the softmax layer's output is not the cross-entropy layer's prediction")
    _storage(cross_entropy, ("f32",), y, truth, dloss)
    cross_entropy.prev_error_signals = dloss
    dtruth = None
    if want_dtruth and not cross_entropy.m_use_labels:
        dtruth = DeviceMatrix(truth.height, truth.width, ldim=truth.ldim, device=cross_entropy.device)
    cross_entropy.error_signals = [None, dtruth]
    softmax.prev_error_signals = None
    softmax.error_signals = DeviceMatrix(y.height, y.width, ldim=y.ldim, device=softmax.device)
    dx = softmax.error_signals
    ws, nb = softmax._ws.get(capi.lib().lbn_softmax_workspace_bytes(y.height, y.width), softmax.device)
    call("lbn_softmax_cross_entropy_bwd_f32", _stream(), y.height, y.width, int(cross_entropy.m_use_labels),
         cross_entropy.spatial_sample_size, y.Buffer(), y.ldim, truth.Buffer(), truth.ldim, dloss.Buffer(), dloss.ldim,
         dx.Buffer(), dx.ldim, dtruth.Buffer() if dtruth is not None else _null(),
         dtruth.ldim if dtruth is not None else 0, ws, nb)
    _after_call()
    return dx


_SUFFIX = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}
_ENTRIES = {}


def _entry(name, dtype):
    """The entry point of `name` for a storage type (a decoding step makes these calls in a row
    on a few microseconds' work each, so nothing here is looked up twice)."""
    f = _ENTRIES.get((name, dtype))
    if f is None:
        if dtype not in _SUFFIX:
            raise TypeError(f"storage is fp32, fp16 or bfloat16, not {dtype}")
        full = f"{name}_{_SUFFIX[dtype]}"
        entry = getattr(capi.lib(), full)

        def f(*args):
            status = entry(*args)
            if status:
                raise LbnError(full, status, capi.lib().lbn_status_string(status).decode())
        _ENTRIES[name, dtype] = f
    return f


def _same_kind(like, height, width, **matrices):
    """Every given matrix has the shape, the storage type and the device of `like`."""
    t = like.tensor
    dtype, index = t.dtype, t.get_device()
    for name, m in matrices.items():
        if m is None:
            continue
        u = m.tensor
        if m.height != height or m.width != width or u.dtype is not dtype or u.get_device() != index:
            raise ValueError(f"{name} is {m.height} x {m.width} {m.dtype} on {u.device}; expected "
                             f"{height} x {width} {dtype} on {t.device}")


def _share_memory(a, b):
    """Whether two matrices have an entry in common.  Rows of one buffer that lie beside each other have none; of
    matrices with different leading dimensions only the extents are looked at."""
    if not (a.width and a.height and b.width and b.height):
        return False
    size_a, size_b = a.tensor.element_size(), b.tensor.element_size()
    ld_a, ld_b = a.ldim * size_a, b.ldim * size_b
    rows_a, rows_b = a.height * size_a, b.height * size_b
    ahead = b.tensor.data_ptr() - a.tensor.data_ptr()
    if not -((b.width - 1) * ld_b + rows_b) < ahead < (a.width - 1) * ld_a + rows_a:
        return False
    if ld_a != ld_b or a.width == 1 or b.width == 1:
        return True
    columns, rows = divmod(ahead, ld_a)  # b starts `rows` bytes into the column `columns` of a
    return (rows < rows_a and -b.width < columns < a.width) or (rows + rows_b > ld_a and -b.width < columns + 1 < a.width)


_SAVED = {}  # by id: residual norm layers (weak references) whose backward has matrices of the last forward to read


def _wrote_over(m, by=None):
    """A call (of the layer `by`) has written over its input m: backward of the layers that still read that memory is
    refused from here on."""
    for key, ref in list(_SAVED.items()):
        layer = ref()
        if layer is None or layer is by:
            continue
        if any(saved is not None and _share_memory(saved, m) for saved in layer._read_by_backward()):
            layer._overwritten = True
            _SAVED.pop(key, None)


def _stream_for(m):
    """The current stream, as an address.  Kernels go to the current device: refuse matrices of
    another one."""
    index = m.tensor.get_device()  # negative for host memory
    if index < 0:
        raise ValueError(f"matrix on {m.tensor.device}; expected device memory")
    if index != torch.cuda.current_device():
        raise ValueError(f"matrix on {m.tensor.device}; the current device is cuda:{torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(index)


def _matrix_beside(like, height, width, dtype=None):
    """An uninitialised matrix on the device of `like`, of its storage type unless another is given."""
    m = DeviceMatrix.__new__(DeviceMatrix)
    m.height, m.width, m.ldim = height, width, height or 1
    shape = width or 1, height or 1
    m.tensor = like.tensor.new_empty(shape) if dtype is None else like.tensor.new_empty(shape, dtype=dtype)
    return m


def _pointer(t):
    return None if t is None else t.data_ptr()


def _buffer(m):
    """(address, leading dimension) of an optional matrix."""
    return (None, 0) if m is None else (m.tensor.data_ptr(), m.ldim)


def _device_values(t, n, dtype, what, like):
    """Address of an optional device vector of at least n entries."""
    if t is None:
        return None
    t = getattr(t, "tensor", t)
    if t.dtype != dtype or t.dim() != 1 or t.numel() < n or (n > 1 and t.stride(0) != 1) or t.get_device() != like.tensor.get_device():
        raise ValueError(f"{what}: expected {n} contiguous {dtype} values on {like.tensor.device}")
    return t.data_ptr()


class _Dropout:
    """Where the random bits of a layer's calls come from: key `seed`, counter `offset`.  A
    training-mode forward without an explicit offset takes the next one (0, 1, ...; explicit ones do not count).

    The mask is a function of these numbers alone, so that another object with the same seed repeats it (recomputation,
    other ranks).  Layers that are to drop independently need seeds of their own: the default is the same for all."""

    def __init__(self, keep_prob, seed):
        if not 0.0 < keep_prob <= 1.0:
            raise ValueError(f"keep_prob is {keep_prob}; it must be in (0, 1]")
        self.m_keep_prob = float(keep_prob)
        self.m_seed = int(seed) & 0xFFFFFFFFFFFFFFFF
        self.m_offset = 0           # of the last forward, which backward repeats
        self.m_column_offset = 0    # global index of the first column of this process's mini-batch
        self.m_step = None          # int64 device tensor of one value added to the offset when a kernel runs
        self.m_kept = 1.0           # keep probability of the last forward (1 outside training)
        self._next = 0

    def _start(self, training, offset):
        if offset is None and training and self.m_keep_prob < 1.0:
            offset = self._next
            self._next = offset + 1 & 0xFFFFFFFFFFFFFFFF
        if offset is not None:
            self.m_offset = int(offset) & 0xFFFFFFFFFFFFFFFF
        self.m_kept = self.m_keep_prob if training else 1.0

    def _drop_args(self, like):
        step = None
        if self.m_step is not None:
            step = _device_values(self.m_step, 1, torch.int64, "m_step", like)
        return self.m_kept, self.m_seed, self.m_offset, step, self.m_column_offset


class dropout_layer(_Layer, _Dropout):
    """Dropout (LBANN's dropout layer: include/lbann/layers/regularizers/dropout.hpp) from a
    counter-based generator: the mask is a function of (seed, offset, row, column) and is never
    stored; backward forms it again."""

    def __init__(self, keep_prob=0.5, seed=0, device="cuda"):
        _Layer.__init__(self, device)
        _Dropout.__init__(self, keep_prob, seed)
        self.m_kept = self.m_keep_prob

    def forward(self, x, in_place=False, training=True, offset=None):
        before = self.m_offset, self.m_kept, self._next
        self._start(training, offset)
        try:
            return super().forward(x, in_place)
        except Exception:
            self.m_offset, self.m_kept, self._next = before  # backward still repeats the last forward
            raise

    def bind_forward(self, x, in_place=False):
        self.prev_activations = x
        self.activations = x if in_place else _matrix_beside(x, x.height, x.width)

    def bind_backward(self, dy, in_place=False):
        self.prev_error_signals = dy
        self.error_signals = dy if in_place else _matrix_beside(dy, dy.height, dy.width)

    def _run(self, name, x, y):
        _same_kind(x, x.height, x.width, output=y)
        _entry(name, x.tensor.dtype)(_stream_for(x), x.height, x.width, *self._drop_args(x), *_buffer(x), *_buffer(y))

    def fp_compute(self):
        self._run("lbn_dropout_fwd", self.prev_activations, self.activations)

    def bp_compute(self):
        self._run("lbn_dropout_bwd", self.prev_error_signals, self.error_signals)


class residual_norm_layer(_Dropout):
    """The residual stream between two transformer blocks in one call each way:

        u = N1(branch);  v = dropout(u);  h = a * residual + b * gate * v;  y = N2(h)

    with N1 (`branch_norm`) and N2 (`output_norm`) "none", "rms" or "layer".  scale / bias arguments
    are arrays or tensors of `size` values, None for no such weight (a scale of one, a bias of zero, and no
    gradient); contiguous fp32 tensors on the device are used where they are, so that an optimizer's updates
    are seen, others are copied.  branch, residual, h and y share one storage type: fp32, fp16 or bfloat16.

    forward(branch, residual, gate) returns y (None without an output norm) and keeps the new
    stream in `residual`; backward(dy, dresidual) returns (dbranch, dresidual of the old stream)
    and leaves the weights' gradients in m_{branch,output}_{scale,bias}_gradient and
    m_gate_gradient."""

    _gradients = [(name, f"m_{name}_gradient") for name in ("branch_scale", "branch_bias", "output_scale", "output_bias")]
    KINDS = {"none": capi.LBN_NORM_NONE, "rms": capi.LBN_NORM_RMS, "layer": capi.LBN_NORM_LAYER}

    def __init__(self, size, branch_norm="none", output_norm="rms", epsilon=1e-5, residual_multiplier=1.0,
                 branch_multiplier=1.0, branch_scale=None, branch_bias=None, output_scale=None, output_bias=None,
                 keep_prob=1.0, seed=0, device="cuda"):
        super().__init__(keep_prob, seed)
        for kind in (branch_norm, output_norm):
            if kind not in self.KINDS:
                raise ValueError(f"unknown norm {kind!r}; expected one of {sorted(self.KINDS)}")
        self.device = device
        self.size = int(size)
        self.m_branch_norm, self.m_output_norm = branch_norm, output_norm
        self.m_epsilon = float(epsilon)
        self.m_residual_multiplier, self.m_branch_multiplier = float(residual_multiplier), float(branch_multiplier)
        self._kinds = self.KINDS[branch_norm], self.KINDS[output_norm]
        self.weights = {}
        for name, value, kind in (("branch_scale", branch_scale, branch_norm), ("branch_bias", branch_bias, branch_norm),
                                  ("output_scale", output_scale, output_norm), ("output_bias", output_bias, output_norm)):
            if value is None:
                self.weights[name] = None
            elif kind == "none":
                raise ValueError(f"{name} without a norm to scale")
            else:
                t = value if isinstance(value, torch.Tensor) else torch.as_tensor(np.asarray(value, np.float32))
                self.weights[name] = t.to(device=device, dtype=torch.float32).contiguous()
                if t.dim() != 1 or t.numel() != self.size:
                    raise ValueError(f"{name} has shape {tuple(t.shape)}; expected ({self.size},)")
        self.branch = self.h = self.gate = self.residual = self.activations = self.m_statistics = None
        self.m_has_residual = self._overwritten = False
        self.m_gate_gradient = None
        self._scratch = None, 0  # a shape of backward and the scratch it takes
        for _, attribute in self._gradients:
            setattr(self, attribute, None)

    def _check_gate(self, gate, like):
        if gate is None:
            return
        if gate.height != self.size or gate.width < 1 or like.width % gate.width or gate.tensor.dtype != torch.float32 \
                or gate.tensor.get_device() != like.tensor.get_device():
            raise ValueError(f"gate is {gate.height} x {gate.width} {gate.dtype}; expected {self.size} rows of fp32 on "
                             f"{like.tensor.device} and a number of columns that divides {like.width}")

    def _check_weights(self, like):
        index, n, fp32 = like.tensor.get_device(), self.size, torch.float32
        for name, t in self.weights.items():
            if t is None or t.get_device() == index and t.numel() == n and t.dtype is fp32 and t.is_contiguous():
                continue
            raise ValueError(f"{name}: {t.numel()} {t.dtype} values on {t.device}; expected {n} contiguous ones of fp32 on {like.tensor.device}")

    def forward(self, branch, residual=None, gate=None, training=True, offset=None, in_place=False):
        """in_place: the new stream overwrites `residual`, and outside training, where no backward
        needs it, y overwrites `branch`.  training=False: no dropout, no statistics.

        In training, `residual` must not be what another layer's backward is still to read: a layer with an
        output norm reads the stream that it returned.  A layer whose matrices were written over refuses backward."""
        n, w, kinds, wt = self.size, branch.width, self._kinds, self.weights
        _same_kind(branch, n, w, branch=branch, residual=residual)
        stream = _stream_for(branch)
        self._check_weights(branch)
        self._check_gate(gate, branch)
        if in_place:
            self._check_places(branch, residual, gate, training)
        h = residual if in_place and residual is not None else _matrix_beside(branch, n, w)
        y = None
        if kinds[1]:
            y = branch if in_place and not training else _matrix_beside(branch, n, w)
        statistics = _matrix_beside(branch, 4, w, torch.float32) if training else None
        before = self.m_offset, self.m_kept, self._next
        self._start(training, offset)
        try:
            _entry("lbn_residual_norm_fwd", branch.tensor.dtype)(
                stream, n, w, *kinds, self.m_epsilon, self.m_residual_multiplier, self.m_branch_multiplier, *_buffer(branch),
                *_buffer(residual), *_buffer(gate), 0 if gate is None else gate.width, _pointer(wt["branch_scale"]),
                _pointer(wt["branch_bias"]), _pointer(wt["output_scale"]), _pointer(wt["output_bias"]), *self._drop_args(branch),
                *_buffer(h), *_buffer(y), *_buffer(statistics))
        except Exception:
            self.m_offset, self.m_kept, self._next = before  # backward still repeats the last forward
            raise
        # only now: a call that was refused leaves the last one's matrices, statistics and dropout together
        self.branch, self.gate, self.m_has_residual, self.m_statistics = branch, gate, residual is not None, statistics
        self.h = self.residual = h
        self.activations = y
        if not training or self._overwritten or id(self) not in _SAVED:
            self._keep(training)
        if in_place and _SAVED:
            if residual is not None:
                _wrote_over(residual, self)
            if y is branch:
                _wrote_over(branch, self)
        return y

    def _check_places(self, branch, residual, gate, training):
        """Two outputs, or one and what is read again after it was written, need memory of their own."""
        again = training and (self._kinds[0] or gate is not None)  # backward reads the branch
        y_too = not training and self._kinds[1]                    # y takes the branch's place
        o = branch.tensor.data_ptr() if branch.width else None
        r = None if residual is None else residual.tensor.data_ptr()
        clash = o is not None and o == r and (again or y_too)
        if gate is not None and branch.width and (training or gate.width < branch.width):
            clash = clash or gate.tensor.data_ptr() in (r, o if y_too else None)
        if clash:
            raise ValueError("in_place: branch, residual and gate need memory of their own")

    def _keep(self, training):
        self._overwritten = False
        key = id(self)
        if not training:
            _SAVED.pop(key, None)
        elif key not in _SAVED:
            _SAVED[key] = weakref.ref(self, lambda _, saved=_SAVED: saved.pop(key, None))

    def _read_by_backward(self):
        """The matrices of the last forward (or bind_saved) that backward reads."""
        branch = self.branch if self._kinds[0] or self.gate is not None else None
        return branch, self.h if self._kinds[1] else None, self.gate

    def bind_saved(self, branch, h, statistics, gate=None, has_residual=True, offset=0, training=True):
        """What an earlier forward left behind, for a backward without one in this object
        (recomputation, pipelines): its block output, new stream, statistics, gate and dropout offset."""
        if statistics is None:
            raise ValueError("bind_saved takes the statistics of a training-mode forward")
        self._check_gate(gate, statistics)
        self.branch, self.h, self.m_statistics, self.gate = branch, h, statistics, gate
        self.residual, self.m_has_residual = h, bool(has_residual)
        self._start(training, offset)
        self._keep(True)

    def backward(self, dy=None, dresidual=None):
        like = dy if dy is not None else dresidual
        if like is None or (dy is not None) != bool(self._kinds[1]):
            raise ValueError("backward takes dy exactly if there is an output norm, and dresidual if there is none")
        if self.m_statistics is None:
            raise ValueError("backward needs a training-mode forward (or bind_saved) first")
        if self._overwritten:
            raise ValueError("a later call with in_place has overwritten the stream, branch or gate that backward reads")
        n, w, kinds, wt, gate = self.size, like.width, self._kinds, self.weights, self.gate
        _same_kind(like, n, w, dy=dy, dresidual=dresidual, branch=self.branch, h=self.h)
        st = self.m_statistics
        if st.height != 4 or st.width != w or st.tensor.dtype != torch.float32 or st.tensor.get_device() != like.tensor.get_device():
            raise ValueError("the statistics are a (4 x width) fp32 matrix")
        stream = _stream_for(like)
        self._check_weights(like)
        dbranch = _matrix_beside(like, n, w)
        dres = _matrix_beside(like, n, w) if self.m_has_residual else None
        wanted = sum(wt[name] is not None for name, _ in self._gradients)
        if wanted > 1:  # rows of one allocation: four take 3.1 us, four allocations 5.5
            rows = iter(like.tensor.new_empty((wanted, n), dtype=torch.float32).unbind(0))
        elif wanted:
            rows = iter((like.tensor.new_empty((n,), dtype=torch.float32),))
        grads = []
        for name, attribute in self._gradients:
            g = None
            if wt[name] is not None:
                g = _Vector.__new__(_Vector)
                g.n, g.tensor = n, next(rows)
            setattr(self, attribute, g)
            grads.append(None if g is None else g.tensor.data_ptr())
        gates = 0 if gate is None else gate.width
        self.m_gate_gradient = dgate = None if gate is None else _matrix_beside(like, n, gates, torch.float32)
        if w == 0:  # nothing is launched then; sums over no columns are zero
            for m in (dgate, *(getattr(self, attribute) for _, attribute in self._gradients)):
                if m is not None:
                    m.tensor.zero_()
        key = w, gates, like.tensor.dtype, wanted > 0
        last, need = self._scratch  # replaced as one, so that a thread beside this one sees both or neither
        if last != key:
            need = capi.lib().lbn_residual_norm_bwd_workspace_bytes(n, w, int(wanted > 0), gates, like.tensor.element_size())
            self._scratch = key, need
        # scratch of this call alone: nothing that another stream or a recorded graph could share
        ws = like.tensor.new_empty((need,), dtype=torch.uint8) if need else None
        _entry("lbn_residual_norm_bwd", like.tensor.dtype)(
            stream, n, w, *kinds, self.m_epsilon, self.m_residual_multiplier, self.m_branch_multiplier, *_buffer(self.branch),
            *(_buffer(self.h) if kinds[1] else (None, 0)), *_buffer(gate), gates, _pointer(wt["branch_scale"]),
            _pointer(wt["branch_bias"]), _pointer(wt["output_scale"]), *self._drop_args(like), *_buffer(st), *_buffer(dy),
            *_buffer(dresidual), *_buffer(dbranch), *_buffer(dres), *_buffer(dgate), *grads, _pointer(ws), need)
        return dbranch, dres


class logits_adjust_layer:
    """Penalties for repeated tokens, bias lists and grammar masks on the logits of a decoding
    step, in front of the softmax layer.  One column per sequence; see lbn_logits_adjust_* in
    include/lbnorm.h for the formula.  Forward only."""

    def __init__(self, vocabulary, device="cuda"):
        self.vocabulary = int(vocabulary)
        self.device = device
        self.activations = None

    @staticmethod
    def _matrix(m, width, dtype, what, like, height=None):
        if m is None:
            return None, 0, 0
        if m.tensor.dtype != dtype or m.tensor.get_device() != like.tensor.get_device() or (width is not None and m.width != width) \
                or (height is not None and m.height != height):
            raise ValueError(f"{what} is {m.height} x {m.width} {m.dtype} on {m.tensor.device}")
        return m.tensor.data_ptr(), m.ldim, m.height

    def forward(self, x, tokens=None, lengths=None, prompt_lengths=None, repetition=None, presence=None, frequency=None,
                bias_tokens=None, bias_values=None, mask=None, mask_index=None, in_place=False):
        """x: (vocabulary x sequences).  tokens: (max_tokens x sequences) int32, lengths and
        prompt_lengths int32 vectors; repetition, presence, frequency fp32 vectors; bias_tokens
        (int32) and bias_values (fp32): (entries x sequences); mask: (ceil(vocabulary / 32) x
        grammars) int32 words, mask_index an int32 vector.  Everything but x is optional."""
        w = x.width
        _same_kind(x, self.vocabulary, w, logits=x)
        stream = _stream_for(x)
        y = x if in_place else _matrix_beside(x, self.vocabulary, w)
        if (bias_tokens is None) != (bias_values is None):
            raise ValueError("bias_tokens and bias_values go together")
        words = (self.vocabulary + 31) // 32
        tok, ld_tok, max_tokens = self._matrix(tokens, w, torch.int32, "tokens", x)
        bt, ld_bt, biases = self._matrix(bias_tokens, w, torch.int32, "bias_tokens", x)
        bv, ld_bv, _ = self._matrix(bias_values, w, torch.float32, "bias_values", x, biases or None)
        mk, ld_mk, _ = self._matrix(mask, None, torch.int32, "mask", x, words)
        _entry("lbn_logits_adjust", x.tensor.dtype)(
            stream, self.vocabulary, w, *_buffer(x), *_buffer(y), tok, ld_tok, max_tokens,
            _device_values(lengths, w, torch.int32, "lengths", x),
            _device_values(prompt_lengths, w, torch.int32, "prompt_lengths", x),
            _device_values(repetition, w, torch.float32, "repetition", x),
            _device_values(presence, w, torch.float32, "presence", x),
            _device_values(frequency, w, torch.float32, "frequency", x), bt, ld_bt, bv, ld_bv, biases, mk, ld_mk,
            0 if mask is None else mask.width, _device_values(mask_index, w, torch.int32, "mask_index", x))
        if in_place and _SAVED:
            _wrote_over(x)
        self.activations = y
        return y


class gradient_buffer:
    """The optimizer's gradient buffer as the layers see it: optimizer::add_to_gradient and
    get_gradient_buffer (include/lbann/optimizers/optimizer_impl.hpp:207-288) with their status
    machine (include/lbann/optimizers/optimizer.hpp:54-70), for one process (RedundantSize = 1,
    so a needed synchronisation changes the status and nothing else).

    `gradient` is a (height x width) DeviceMatrix.  It starts `cleared`: the first contribution
    overwrites it without reading it, later ones accumulate."""

    READY, CLEARED, SYNC_NEEDED = "ready", "cleared", "sync_needed"

    def __init__(self, height, width=1, device="cuda"):
        self.gradient = DeviceMatrix(height, width, device=device)
        self.status = self.CLEARED

    def clear(self):
        self.status = self.CLEARED

    def _scales(self, sync_needed):
        # (buf_scale, in_scale) and the status transition of get_gradient_buffer
        if self.status == self.READY:
            if sync_needed:
                self.status = self.SYNC_NEEDED
            return 1.0, 1.0
        if self.status == self.CLEARED:
            self.status = self.SYNC_NEEDED if sync_needed else self.READY
            return 0.0, 1.0
        if self.status == self.SYNC_NEEDED:
            return 1.0, 1.0
        raise ValueError(f"unexpected gradient status ({self.status})")

    def add_to_gradient(self, contrib, scale=1.0, sync_needed=False, ldim=None):
        """contrib: a DeviceMatrix of the buffer's shape, or a _Vector / torch tensor holding one column
        (then `ldim` is its leading dimension when the buffer has several columns)."""
        g = self.gradient
        if (contrib.tensor if hasattr(contrib, "tensor") else contrib).dtype != torch.float32:
            raise TypeError("gradient contributions are fp32")
        buf_scale, in_scale = self._scales(sync_needed)
        if isinstance(contrib, DeviceMatrix):
            if (contrib.height, contrib.width) != (g.height, g.width):
                raise ValueError("gradient contribution has the wrong shape")
            ptr, ld = contrib.Buffer(), contrib.ldim
        else:
            t = contrib.tensor if hasattr(contrib, "tensor") else contrib
            ld = int(ldim) if ldim is not None else g.height
            if t.numel() < (g.width - 1) * ld + g.height:
                raise ValueError("gradient contribution is too small")
            ptr = capi.vp(t.data_ptr())
        call("lbn_gradient_sink_f32", _stream(), g.height, g.width, buf_scale, in_scale * float(scale), ptr, ld,
             g.Buffer(), g.ldim)

    def finish_sync(self):
        """What the all-reduce completes on several processes; here the values are already final."""
        if self.status == self.SYNC_NEEDED:
            self.status = self.READY
