"""Layers that networks over sequences have around their convolutions, in the protocol of the other modules
(updateOutput, updateGradInput, accGradParameters; gradients of parameters are assigned)."""
import ctypes

import torch

from . import _lib
from ._lib import RecurrenceDesc, ResidualNormDesc, Rows, Steps, check, lib
from .tensors import TYPES, Workspace, _ptr, _stream

__all__ = ["GatedLinearRecurrence", "GatedResidualNorm"]


def _check_activation(t, name, like=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s: CUDA support only!" % name)
    if t.dtype not in TYPES:
        raise TypeError("%s must be float32, bfloat16 or float16" % name)
    if t.device.index != torch.cuda.current_device():
        raise ValueError("%s is not on the current device" % name)
    if like is not None:
        if t.dtype != like.dtype:
            raise TypeError("%s must be %s" % (name, like.dtype))
        if t.shape != like.shape:
            raise ValueError("%s has the wrong shape" % name)


def _like(old, t):
    """`old` where it can take what has the shape and the type of t, else a new tensor."""
    if old is not None and old.shape == t.shape and old.dtype == t.dtype and old.device == t.device:
        return old
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _steps(t):
    return None if t is None else ctypes.byref(Steps(t.data_ptr(), *t.stride()))


class GatedLinearRecurrence:
    """a_t = sigmoid(gate_t + bias), state = a_t state + (1 - a_t) x_t, output_t = state, for every sequence and channel.

    updateOutput takes [x, gate], both (batch, steps, nChannels), float32, bfloat16 or float16, of any strides, and gives the
    output, of the same shape; self.state is then the state behind the last step (batch, nChannels) in float32.
    `state`: the state before the first step, zeros where it is None.  `lengths`: an int32 CUDA tensor with the steps of each
    sequence; behind them nothing is read, and outputs and gradients are zero.  backward (and its halves updateGradInput
    and accGradParameters) follows an updateOutput of the same inputs, from which the module keeps the state before every
    128 steps; after evaluate() it keeps none and cannot go backward.  step advances sequences by one token."""

    def __init__(self, nChannels, device="cuda"):
        if not isinstance(nChannels, int) or nChannels < 1:
            raise ValueError("nChannels must be a positive number")
        self.nChannels = nChannels
        self.device = torch.device(device)
        self.bias = torch.zeros(nChannels, device=self.device)
        self.gradBias = torch.zeros(nChannels, device=self.device)
        self.train = True
        self.output = self.state = self.gradInput = self.gradState = None
        self._workspace, self._checkpoints = Workspace(), Workspace()
        self._forward = None   # (shape, type, lengths, checkpoints) of the updateOutput that backward may follow

    def training(self):
        self.train = True

    def evaluate(self):
        self.train = False

    def parameters(self):
        return [self.bias], [self.gradBias]

    def zeroGradParameters(self):
        self.gradBias.zero_()

    def _inputs(self, input):
        if len(input) != 2:
            raise ValueError("the input is [x, gate]")
        x, gate = input
        _check_activation(x, "x")
        _check_activation(gate, "gate", x)
        if x.dim() != 3 or x.size(2) != self.nChannels:
            raise ValueError("x must be (batch, steps, %d)" % self.nChannels)
        return x, gate, ctypes.byref(RecurrenceDesc(x.size(0), self.nChannels, x.size(1), TYPES[x.dtype]))

    def _check_state(self, t, name, batch):
        if t is None:
            return
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError("%s: CUDA support only!" % name)
        if t.dtype != torch.float32:
            raise TypeError("%s must be float32" % name)
        if tuple(t.shape) != (batch, self.nChannels) or not t.is_contiguous() or t.device.index != torch.cuda.current_device():
            raise ValueError("%s must be a contiguous (%d, %d) tensor on the current device" % (name, batch, self.nChannels))

    @staticmethod
    def _check_lengths(t, batch):
        if t is None:
            return
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError("lengths: CUDA support only!")
        if t.dtype != torch.int32:
            raise TypeError("lengths must be int32")
        if tuple(t.shape) != (batch,) or not t.is_contiguous() or t.device.index != torch.cuda.current_device():
            raise ValueError("lengths must be %d contiguous numbers on the current device" % batch)

    def updateOutput(self, input, state=None, lengths=None):
        x, gate, desc = self._inputs(input)
        batch = x.size(0)
        self._check_state(state, "state", batch)
        self._check_lengths(lengths, batch)
        self.output = _like(self.output, x)
        if self.state is None or self.state.size(0) != batch or self.state.device != x.device:
            self.state = torch.empty(batch, self.nChannels, device=x.device)
        kept = None
        if self.train:
            kept = self._checkpoints.take(lib().fbfc_recurrence_checkpoint_bytes(desc), x.device)
        ws = self._workspace.take(lib().fbfc_recurrence_workspace_bytes(desc), x.device)
        self._forward = None
        check(lib().fbfc_recurrence_forward(desc, _steps(x), _steps(gate), _ptr(self.bias), _ptr(state), _ptr(lengths),
                                            _steps(self.output), _ptr(self.state), _ptr(kept), _ptr(ws), _stream()))
        if self.train:
            self._forward = (x.shape, x.dtype, lengths, kept)
        return self.output

    forward = updateOutput

    def step(self, input, state):
        """One token of each sequence: [x, gate] of (batch, nChannels); advances `state` in place and gives the output."""
        if len(input) != 2:
            raise ValueError("the input is [x, gate]")
        x, gate = input
        _check_activation(x, "x")
        _check_activation(gate, "gate", x)
        if x.dim() != 2 or x.size(1) != self.nChannels:
            raise ValueError("x must be (batch, %d)" % self.nChannels)
        if state is None:
            raise TypeError("step needs the state that it advances")
        self._check_state(state, "state", x.size(0))
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        tensors = [ctypes.byref(Steps(t.data_ptr(), t.stride(0), 0, t.stride(1))) for t in (x, gate, out)]
        desc = RecurrenceDesc(x.size(0), self.nChannels, 1, TYPES[x.dtype])
        check(lib().fbfc_recurrence_forward(ctypes.byref(desc), tensors[0], tensors[1], _ptr(self.bias), _ptr(state), None,
                                            tensors[2], _ptr(state), None, None, _stream()))
        return out

    def _backward(self, input, gradOutput, gradState, inputs, weights, scale):
        x, gate, desc = self._inputs(input)
        if self._forward is None or self._forward[:2] != (x.shape, x.dtype):
            raise ValueError("backward follows an updateOutput of the same inputs, not after evaluate()")
        _check_activation(gradOutput, "gradOutput", x)
        self._check_state(gradState, "gradState", x.size(0))
        grads, first = [None, None], None
        if inputs:
            old = self.gradInput or [None, None]
            self.gradInput = [_like(old[0], x), _like(old[1], x)]
            grads = [_steps(t) for t in self.gradInput]
            if self.gradState is None or self.gradState.size(0) != x.size(0) or self.gradState.device != x.device:
                self.gradState = torch.empty(x.size(0), self.nChannels, device=x.device)
            first = self.gradState
        ws = self._workspace.take(lib().fbfc_recurrence_workspace_bytes(desc), x.device)
        check(lib().fbfc_recurrence_backward(desc, _steps(x), _steps(gate), _ptr(self.bias), _ptr(self._forward[2]),
                                             _ptr(self._forward[3]), _steps(gradOutput), _ptr(gradState), *grads,
                                             _ptr(self.gradBias if weights else None), scale, _ptr(first), _ptr(ws), _stream()))

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
        self._workspace = Workspace()

    def parameters(self):
        pairs = [(self.postWeight, self.gradPostWeight), (self.scale, self.gradScale), (self.preWeight, self.gradPreWeight)]
        return [p for p, _ in pairs if p is not None], [g for _, g in pairs if g is not None]

    def zeroGradParameters(self):
        for g in self.parameters()[1]:
            g.zero_()

    # rows of a tensor for the C ABI; None is an absent one
    def _rows(self, t, name):
        if t is None:
            return None
        try:
            t = t.view(-1, self.nChannels)
        except RuntimeError:
            raise ValueError("%s must be rows of channels, one stride apart" % name) from None
        if self.nChannels > 1 and t.stride(1) != 1:
            raise ValueError("the channels of %s must lie side by side" % name)
        return ctypes.byref(Rows(t.data_ptr(), t.stride(0)))

    def _inputs(self, input):
        names = ("residual", "branch", "gate")[:1 + self.hasBranch + self.hasGate]
        if isinstance(input, torch.Tensor):
            input = [input]
        if len(input) != len(names):
            raise ValueError("the input is [%s]" % ", ".join(names))
        residual = input[0]
        _check_activation(residual, "residual")
        if residual.dim() < 1 or residual.size(-1) != self.nChannels:
            raise ValueError("residual must have %d channels last" % self.nChannels)
        for t, name in zip(input[1:], names[1:]):
            _check_activation(t, name, residual)
        desc = ResidualNormDesc(residual.numel() // self.nChannels, self.nChannels, TYPES[residual.dtype], self.eps)
        return ctypes.byref(desc), residual, [self._rows(t, n) for t, n in zip(input, names)] + [None] * (3 - len(names))

    def updateOutput(self, input):
        desc, residual, rows = self._inputs(input)
        old = self.output or [None, None]
        # without a branch the first output is the caller's tensor, never one to write into
        output = _like(old[0], residual) if self.hasBranch else None
        normed = _like(old[1], residual) if self.hasNorm else None
        check(lib().fbfc_residual_norm_forward(desc, *rows, _ptr(self.postWeight), _ptr(self.scale), _ptr(self.preWeight),
                                               self._rows(output, "output"), self._rows(normed, "normed"), _stream()))
        self.output = [output if self.hasBranch else residual, normed]
        return self.output

    forward = updateOutput

    def _backward(self, input, gradOutput, inputs, weights, scale):
        desc, residual, rows = self._inputs(input)
        gr, gn = gradOutput
        if gr is None and gn is None:
            raise ValueError("gradOutput is [gradOutput, gradNormed], and one of them is needed")
        if gn is not None and not self.hasNorm:
            raise ValueError("there is no norm behind the block to have a gradient")
        for t, name in ((gr, "gradOutput"), (gn, "gradNormed")):
            if t is not None:
                _check_activation(t, name, residual)
        grads = [None] * 3
        if inputs:
            old = self.gradInput or [None] * 3
            n = 1 + self.hasBranch + self.hasGate
            self.gradInput = [_like(old[i], residual) for i in range(n)]
            grads = [self._rows(t, "gradInput") for t in self.gradInput] + [None] * (3 - n)
        ws, params = None, [None] * 3
        if weights:
            ws = self._workspace.take(lib().fbfc_residual_norm_workspace_bytes(desc), residual.device)
            params = [self.gradPostWeight, self.gradScale, self.gradPreWeight]
        check(lib().fbfc_residual_norm_backward(desc, *rows, _ptr(self.postWeight), _ptr(self.scale), _ptr(self.preWeight),
                                                self._rows(gr, "gradOutput"), self._rows(gn, "gradNormed"), *grads,
                                                *map(_ptr, params), scale, _ptr(ws), _stream()))

    def updateGradInput(self, input, gradOutput):
        self._backward(input, gradOutput, True, False, 1.0)
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0):
        self._backward(input, gradOutput, False, True, scale)

    def backward(self, input, gradOutput, scale=1.0):
        """updateGradInput and accGradParameters in one pass over the inputs."""
        self._backward(input, gradOutput, True, True, scale)
        return self.gradInput
