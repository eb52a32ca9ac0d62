"""Layers that networks over sequences have around their convolutions, in the protocol of the other modules
(updateOutput, updateGradInput, accGradParameters; gradients of parameters are assigned)."""
import ctypes

import torch

from . import _lib
from ._lib import ResidualNormDesc, Rows, check, lib
from .tensors import TYPES, Workspace, _ptr, _stream

__all__ = ["GatedResidualNorm"]


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

    @staticmethod
    def _like(old, t):
        """`old` where it can take what has the shape and the type of t, else a new tensor."""
        if old is not None and old.shape == t.shape and old.dtype == t.dtype and old.device == t.device:
            return old
        return torch.empty(t.shape, dtype=t.dtype, device=t.device)

    def updateOutput(self, input):
        desc, residual, rows = self._inputs(input)
        old = self.output or [None, None]
        # without a branch the first output is the caller's tensor, never one to write into
        output = self._like(old[0], residual) if self.hasBranch else None
        normed = self._like(old[1], residual) if self.hasNorm else None
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
            self.gradInput = [self._like(old[i], residual) for i in range(n)]
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
