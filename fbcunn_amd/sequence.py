"""Layers that networks over sequences have around their convolutions, in the protocol of the other modules
(updateOutput, updateGradInput, accGradParameters; gradients of parameters are assigned)."""
import ctypes

import torch

from . import _lib
from ._lib import RecurrenceDesc, ResidualNormDesc, Rows, Steps, check, lib
from .tensors import TYPES, Workspace, _ptr, is_capturing, signature, stream_on

__all__ = ["GatedLinearRecurrence", "GatedResidualNorm"]


def _check_activation(t, name, like=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s: CUDA support only!" % name)
    if t.dtype not in TYPES:
        raise TypeError("%s must be float32, bfloat16 or float16" % name)
    if like is not None:
        if t.dtype != like.dtype:
            raise TypeError("%s must be %s" % (name, like.dtype))
        if t.shape != like.shape:
            raise ValueError("%s has the wrong shape" % name)
        if t.device != like.device:
            raise ValueError("%s is on another device" % name)


def _parameter(t, name, channels, index):
    """The address of a parameter or its gradient; None for an absent one.  Looked at in each call, since any tensor may have
    been assigned to it."""
    if t is None:
        return None
    try:
        if t.dtype is torch.float32 and t.numel() == channels and t.is_contiguous() and t.get_device() == index:
            return t.data_ptr()
    except AttributeError:
        raise TypeError("%s must be a tensor" % name) from None
    if t.dtype is not torch.float32:
        raise TypeError("%s must be float32" % name)
    if t.get_device() != index:
        raise ValueError("%s is on another device than the inputs" % name)
    raise ValueError("%s must be %d contiguous numbers" % (name, channels))


class _Call:
    """What a module's calls on inputs of one signature share, and the results that it makes for them."""

    def __init__(self, like, results):
        self.shape, self.dtype, self.device, self.index = like.shape, like.dtype, like.device, like.device.index
        self.captured = self.capturing = False   # into any graph so far; now
        self._made = [(None, 0, 0)] * results
        self._written, self._kept = [False] * results, []   # which of them a graph writes to; those that were replaced

    def result(self, i, places=()):
        """Result i, the tensor of the last call unless one of `places`, the addresses of what this call reads, lies in it: an
        input that is a module's last result, or a view of it, keeps its values, which backward, or its other half, reads."""
        t, at, end = self._made[i]
        if t is None:
            return self._make(i)
        for p in places:
            if at <= p < end:
                return self._make(i)
        if self.capturing:
            self._written[i] = True
        return t

    def _make(self, i):
        if self._written[i]:
            self._kept.append(self._made[i][0])
        shape, dtype = self._like(i)
        t = torch.empty(shape, dtype=dtype, device=self.device)
        at = t.data_ptr()
        self._made[i] = t, at, at + t.numel() * t.element_size()
        self._written[i] = self.capturing
        return t

    def _like(self, i):
        return self.shape, self.dtype


class _Calls:
    """A module's call for the inputs that it was last given.  One that a graph was captured from is kept with its results,
    which the graph writes to whenever it is replayed."""

    def __init__(self, kind, *more):
        self._kind, self._more, self._signature, self._call, self._captured = kind, more, None, None, []

    @property
    def used(self):
        return self._call is not None

    def of(self, net, inputs):
        now = signature(*inputs)
        if now != self._signature:
            call = self._kind(net, inputs, *self._more)
            if self._call is not None and self._call.captured:
                self._captured.append(self._call)
            self._call, self._signature = call, now
        call = self._call
        call.capturing = is_capturing()
        call.captured |= call.capturing
        return call


class _RecurrenceCall(_Call):
    """Of the recurrence: checked sizes and descriptors.  Results: the output, the gradients of x and gate, the last state and the
    gradient of the first, the states that backward begins at."""

    def __init__(self, net, input, dims):
        x, gate = input
        channels = net.nChannels
        _check_activation(x, "x")
        _check_activation(gate, "gate", x)
        if x.dim() != dims or x.size(-1) != channels:
            raise ValueError("x must be (%s%d)" % ("batch, steps, " if dims == 3 else "batch, ", channels))
        super().__init__(x, 6)
        self.batch, steps = x.size(0), x.size(1) if dims == 3 else 1
        desc = RecurrenceDesc(self.batch, channels, steps, TYPES[x.dtype])
        self.desc = ctypes.byref(desc)
        self.checkpointBytes = lib().fbfc_recurrence_checkpoint_bytes(self.desc)
        self.workspaceBytes = lib().fbfc_recurrence_workspace_bytes(self.desc)
        whole = (steps * channels, channels, 1)
        strides = [t.stride() if dims == 3 else (t.stride(0), 0, t.stride(1)) for t in (x, gate)]
        # x, gate, output, gradients of x and gate, gradient of the output (its strides are those of each call)
        self.steps = [Steps(0, *s) for s in (strides[0], strides[1], whole, whole, whole, whole)]
        self.refs = [ctypes.byref(s) for s in self.steps]

    def _like(self, i):
        if i < 3:
            return self.shape, self.dtype
        return ((self.batch, self.shape[-1]), torch.float32) if i < 5 else ((self.checkpointBytes,), torch.uint8)


class GatedLinearRecurrence:
    """a_t = sigmoid(gate_t + bias), state = a_t state + (1 - a_t) x_t, output_t = state, for every sequence and channel.

    updateOutput takes [x, gate], both (batch, steps, nChannels), float32, bfloat16 or float16, of any strides, and gives the
    output, of the same shape; self.state is then the state behind the last step (batch, nChannels) in float32.
    `state`: the state before the first step, zeros where it is None.  `lengths`: an int32 CUDA tensor with the steps of each
    sequence; what lies behind them has no effect, and outputs and gradients there are zero.  backward (and its halves
    updateGradInput and accGradParameters) follows an updateOutput of the same inputs, from which the module keeps the
    state before every 128 steps; after evaluate() it keeps none and cannot go backward.  step advances sequences by one
    token.  As in the other modules the outputs are the module's own tensors, which its next call on inputs of the same
    shape writes again, unless they are its inputs; a `state` that is its self.state is advanced in place."""

    def __init__(self, nChannels, device="cuda"):
        if not isinstance(nChannels, int) or nChannels < 1:
            raise ValueError("nChannels must be a positive number")
        self.nChannels = nChannels
        self.device = torch.device(device)
        self.bias = torch.zeros(nChannels, device=self.device)
        self.gradBias = torch.zeros(nChannels, device=self.device)
        self.train = True
        self.output = self.state = self.gradInput = self.gradState = None
        self._begin()

    def _begin(self):
        self._workspace = Workspace()
        self._calls = {dims: _Calls(_RecurrenceCall, dims) for dims in (2, 3)}   # of step and updateOutput
        self._forward = None   # (shape, type, lengths, checkpoints) of the updateOutput that backward may follow

    def cleanupBuffers(self):
        """Waits for the device and gives back all memory but the last results.  No graph that was captured with the module may
        be replayed from then on."""
        if any(c.used for c in self._calls.values()):
            torch.cuda.synchronize()
        self._begin()

    def training(self):
        self.train = True

    def evaluate(self):
        self.train = False

    def parameters(self):
        return [self.bias], [self.gradBias]

    def zeroGradParameters(self):
        self.gradBias.zero_()

    def _call(self, input, dims):
        if len(input) != 2:
            raise ValueError("the input is [x, gate]")
        call = self._calls[dims].of(self, input)
        places = input[0].data_ptr(), input[1].data_ptr()
        call.steps[0].data, call.steps[1].data = places
        return call, places, stream_on(call.index)

    def _check_state(self, t, name, call):
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError("%s: CUDA support only!" % name)
        if t.dtype != torch.float32:
            raise TypeError("%s must be float32" % name)
        if t.shape != (call.batch, self.nChannels) or not t.is_contiguous() or t.device != call.device:
            raise ValueError("%s must be a contiguous (%d, %d) tensor on the inputs' device" % (name, call.batch, self.nChannels))
        return t.data_ptr()

    @staticmethod
    def _check_lengths(t, call):
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError("lengths: CUDA support only!")
        if t.dtype != torch.int32:
            raise TypeError("lengths must be int32")
        if t.shape != (call.batch,) or not t.is_contiguous() or t.device != call.device:
            raise ValueError("lengths must be %d contiguous numbers on the inputs' device" % call.batch)
        return t.data_ptr()

    def updateOutput(self, input, state=None, lengths=None):
        call, places, stream = self._call(input, 3)
        bias = _parameter(self.bias, "bias", self.nChannels, call.index)
        first, sizes = self._check_state(state, "state", call), self._check_lengths(lengths, call)
        self.output = call.result(0, places + (first or 0,))
        self.state = call.result(3, places)
        kept = call.result(5) if self.train else None
        call.steps[2].data = self.output.data_ptr()
        self._forward = None
        check(lib().fbfc_recurrence_forward(call.desc, *call.refs[:2], bias, first, sizes, call.refs[2],
                                            self.state.data_ptr(), kept.data_ptr() if self.train else None,
                                            self._workspace.take(call.workspaceBytes, call.device, stream, call.capturing).data_ptr(),
                                            stream))
        if self.train:
            self._forward = (call.shape, call.dtype, lengths, kept)
        return self.output

    forward = updateOutput

    def step(self, input, state):
        """One token of each sequence: [x, gate] of (batch, nChannels); advances `state` in place and gives the output."""
        call, places, stream = self._call(input, 2)
        if state is None:
            raise TypeError("step needs the state that it advances")
        bias, at = _parameter(self.bias, "bias", self.nChannels, call.index), self._check_state(state, "state", call)
        self.output = call.result(0, places)
        call.steps[2].data = self.output.data_ptr()
        check(lib().fbfc_recurrence_forward(call.desc, *call.refs[:2], bias, at, None, call.refs[2], at, None,
                                            None, stream))
        return self.output

    def _backward(self, input, gradOutput, gradState, inputs, weights, scale):
        call, places, stream = self._call(input, 3)
        shape, dtype, lengths, kept = self._forward or (None, None, None, None)
        if shape != call.shape or dtype != call.dtype or kept.device != call.device:
            raise ValueError("backward follows an updateOutput of the same inputs, not after evaluate()")
        _check_activation(gradOutput, "gradOutput", call)
        last = self._check_state(gradState, "gradState", call)
        bias = _parameter(self.bias, "bias", self.nChannels, call.index)
        gradBias = _parameter(self.gradBias, "gradBias", self.nChannels, call.index) if weights else None
        of = call.steps[5]
        of.data = at = gradOutput.data_ptr()
        of.stride_batch, of.stride_step, of.stride_channel = gradOutput.stride()
        grads, first = (None, None), None
        if inputs:
            places += (at, last or 0)
            self.gradInput = [call.result(1, places), call.result(2, places)]
            call.steps[3].data, call.steps[4].data = (t.data_ptr() for t in self.gradInput)
            grads = call.refs[3:5]
            self.gradState = call.result(4, places)
            first = self.gradState.data_ptr()
        check(lib().fbfc_recurrence_backward(call.desc, *call.refs[:2], bias, _ptr(lengths), kept.data_ptr(),
                                             call.refs[5], last, *grads, gradBias, scale, first,
                                             self._workspace.take(call.workspaceBytes, call.device, stream, call.capturing).data_ptr(),
                                            stream))

    def updateGradInput(self, input, gradOutput, gradState=None):
        """[gradient of x, gradient of gate]; self.gradState is the gradient of the state before the first step.  `gradState`:
        the gradient of the state behind the last one."""
        self._backward(input, gradOutput, gradState, True, False, 1.0)
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0, gradState=None):
        self._backward(input, gradOutput, gradState, False, True, scale)

    def backward(self, input, gradOutput, scale=1.0, gradState=None):
        """updateGradInput and accGradParameters in one pass over the inputs."""
        self._backward(input, gradOutput, gradState, True, True, scale)
        return self.gradInput


class _NormCall(_Call):
    """Of the norms: checked sizes and descriptors.  Results: output, normed, the gradients of the inputs."""

    def __init__(self, net, input):
        residual = input[0]
        _check_activation(residual, "residual")
        if residual.dim() < 1 or residual.size(-1) != net.nChannels:
            raise ValueError("residual must have %d channels last" % net.nChannels)
        for t, name in zip(input[1:], net._names[1:]):
            _check_activation(t, name, residual)
        super().__init__(residual, 2 + len(input))
        self.sizes = ResidualNormDesc(residual.numel() // net.nChannels, net.nChannels, TYPES[residual.dtype], net.eps)
        self.desc = ctypes.byref(self.sizes)
        self.workspaceBytes = lib().fbfc_residual_norm_workspace_bytes(self.desc)
        # residual, branch, gate; output, normed; their gradients; the inputs' gradients
        self.rows = [Rows(0, net.nChannels) for _ in range(10)]
        self.refs = [ctypes.byref(r) for r in self.rows]
        for rows, t, name in zip(self.rows, input, net._names):
            rows.stride = net._row_stride(t, name)
        self.inputs = self.refs[:len(input)] + [None] * (3 - len(input))

    def at(self, i, t):
        """Descriptor i, now of tensor t; None for an absent one."""
        if t is None:
            return None
        self.rows[i].data = t.data_ptr()
        return self.refs[i]


class GatedResidualNorm:
    """The norms before and after a block, with the block's gate and residual scale, in one pass:

        output = residual + scale * sigmoid(gate) * postWeight * branch / rms(branch)
        normed = preWeight * output / rms(output),      rms(x) = sqrt(mean x^2 + eps) over the last dimension

    updateOutput takes [residual, branch, gate] and gives [output, normed].  Without `gate` the input is [residual,
    branch]; without `branch` it is [residual], and the output is the residual itself (the norm before the first block);
    without `norm` normed is None (behind the last block).  Inputs are float32, bfloat16 or float16 of one shape (...,
    nChannels) with the channels side by side.  backward takes [gradOutput, gradNormed], either of which may be None,
    and the inputs as they were.  The parameters have 32 bits."""

    def __init__(self, nChannels, eps=1e-6, branch=True, gate=True, norm=True, device="cuda"):
        if not isinstance(nChannels, int) or nChannels < 1:
            raise ValueError("nChannels must be a positive number")
        if not branch and not norm:
            raise ValueError("without a branch and without a norm nothing is left")
        self.nChannels, self.eps = nChannels, eps
        self.hasGate, self.hasBranch, self.hasNorm = bool(gate and branch), bool(branch), bool(norm)
        self.device = torch.device(device)
        one = lambda on: torch.ones(nChannels, device=self.device) if on else None   # noqa: E731
        zero = lambda on: torch.zeros(nChannels, device=self.device) if on else None   # noqa: E731
        self.postWeight, self.scale, self.preWeight = one(branch), one(branch), one(norm)
        self.gradPostWeight, self.gradScale, self.gradPreWeight = zero(branch), zero(branch), zero(norm)
        self.output, self.gradInput = None, None
        self._names = ("residual", "branch", "gate")[:1 + self.hasBranch + self.hasGate]
        self._begin()

    def _begin(self):
        self._workspace = Workspace()
        self._calls = _Calls(_NormCall)

    def cleanupBuffers(self):
        """Waits for the device and gives back all memory but the last results.  No graph that was captured with the module may
        be replayed from then on."""
        if self._calls.used:
            torch.cuda.synchronize()
        self._begin()

    def parameters(self):
        pairs = [(self.postWeight, self.gradPostWeight), (self.scale, self.gradScale), (self.preWeight, self.gradPreWeight)]
        return [p for p, _ in pairs if p is not None], [g for _, g in pairs if g is not None]

    def zeroGradParameters(self):
        for g in self.parameters()[1]:
            g.zero_()

    # the stride between the rows of a tensor
    def _row_stride(self, t, name):
        if t.is_contiguous():
            return self.nChannels
        try:
            t = t.view(-1, self.nChannels)
        except RuntimeError:
            raise ValueError("%s must be rows of channels, one stride apart" % name) from None
        if self.nChannels > 1 and t.stride(1) != 1:
            raise ValueError("the channels of %s must lie side by side" % name)
        return t.stride(0)

    def _call(self, input):
        if isinstance(input, torch.Tensor):
            input = [input]
        if len(input) != len(self._names):
            raise ValueError("the input is [%s]" % ", ".join(self._names))
        call = self._calls.of(self, input)
        call.sizes.eps = self.eps
        places = []
        for rows, t in zip(call.rows, input):
            rows.data = p = t.data_ptr()
            places.append(p)
        return call, input, places, stream_on(call.index)

    def updateOutput(self, input):
        call, input, places, stream = self._call(input)
        weights = self._weights(call)
        output = call.result(0, places) if self.hasBranch else None
        normed = call.result(1, places) if self.hasNorm else None
        check(lib().fbfc_residual_norm_forward(call.desc, *call.inputs, *weights, call.at(3, output), call.at(4, normed),
                                               stream))
        self.output = [output if self.hasBranch else input[0], normed]
        return self.output

    forward = updateOutput

    def _weights(self, call):
        n, index = self.nChannels, call.index
        return (_parameter(self.postWeight, "postWeight", n, index), _parameter(self.scale, "scale", n, index),
                _parameter(self.preWeight, "preWeight", n, index))

    def _gradWeights(self, call):
        n, index = self.nChannels, call.index
        return (_parameter(self.gradPostWeight, "gradPostWeight", n, index), _parameter(self.gradScale, "gradScale", n, index),
                _parameter(self.gradPreWeight, "gradPreWeight", n, index))

    def _backward(self, input, gradOutput, inputs, weights, scale):
        call, input, places, stream = self._call(input)
        gr, gn = gradOutput
        if gr is None and gn is None:
            raise ValueError("gradOutput is [gradOutput, gradNormed], and one of them is needed")
        if gn is not None and not self.hasNorm:
            raise ValueError("there is no norm behind the block to have a gradient")
        for i, t, name in ((5, gr, "gradOutput"), (6, gn, "gradNormed")):
            if t is not None:
                _check_activation(t, name, call)
                call.rows[i].stride = self._row_stride(t, name)
                places.append(t.data_ptr())
        values, params = self._weights(call), self._gradWeights(call) if weights else [None] * 3
        grads = [None] * 3
        if inputs:
            self.gradInput = [call.result(2 + i, places) for i in range(len(input))]
            grads[:len(input)] = [call.at(7 + i, t) for i, t in enumerate(self.gradInput)]
        ws = self._workspace.take(call.workspaceBytes, call.device, stream, call.capturing).data_ptr() if weights else None
        check(lib().fbfc_residual_norm_backward(call.desc, *call.inputs, *values, call.at(5, gr), call.at(6, gn), *grads,
                                                *params, scale, ws, stream))

    def updateGradInput(self, input, gradOutput):
        self._backward(input, gradOutput, True, False, 1.0)
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0):
        self._backward(input, gradOutput, False, True, scale)

    def backward(self, input, gradOutput, scale=1.0):
        """updateGradInput and accGradParameters in one pass over the inputs."""
        self._backward(input, gradOutput, True, True, scale)
        return self.gradInput
