"""Steps of the parameters of a network: what follows accGradParameters in a training step."""
import ctypes

import torch

from . import _lib
from ._lib import AdamwConfig, AdamwTensor, check, lib
from .tensors import TYPES, _ptr, _stream

__all__ = ["AdamW"]


class AdamW:
    """One AdamW step over many tensors at once (fbfc_adamw_step), in place:

        m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weightDecay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

    `params` and `grads` are lists of contiguous CUDA tensors of the same sizes, the parameters all of one type and the
    gradients all of one type (float32, bfloat16 or float16).  The optimizer steps these very tensors: gradients are
    written into them before each step, as the modules' accGradParameters does.  With stateBits = 32 the states `m` and
    `v` are float32, with 8 they are float8_e4m3fn with a float32 scale per 256 elements (`mScale`, `vScale`), rounded
    at random (from `seed` and the number of the step).  In the states every tensor begins at a multiple of 256 elements.
    `lr` and `weightDecay` may be changed between steps.  A step captured into a graph is a new step at each replay,
    for as long as the optimizer lives."""

    def __init__(self, params, grads, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weightDecay=1e-2, stateBits=32, seed=0):
        self._handle = ctypes.c_void_p(0)
        params, grads = list(params), list(grads)
        if not params or len(params) != len(grads):
            raise ValueError("as many gradients as parameters are needed, and at least one")
        for kind, tensors in (("parameter", params), ("gradient", grads)):
            for t in tensors:
                if not isinstance(t, torch.Tensor) or not t.is_cuda:
                    raise TypeError("%s: CUDA support only!" % kind)
                if t.dtype not in TYPES:
                    raise TypeError("%ss must be float32, bfloat16 or float16" % kind)
                if t.dtype != tensors[0].dtype:
                    raise TypeError("%ss must be of one type" % kind)
                if t.device != params[0].device:
                    raise ValueError("all tensors must be on one device")
                if not t.is_contiguous():
                    raise ValueError("%ss must be contiguous" % kind)
        for p, g in zip(params, grads):
            if p.shape != g.shape:
                raise ValueError("gradient of shape %s for a parameter of shape %s" % (tuple(g.shape), tuple(p.shape)))
        if stateBits not in (8, 32):
            raise ValueError("states have 8 or 32 bits")
        self.params, self.grads = params, grads
        self.lr, self.weightDecay, self.stateBits = lr, weightDecay, stateBits
        self.device = params[0].device
        table = (AdamwTensor * len(params))(*[(p.data_ptr(), g.data_ptr(), p.numel()) for p, g in zip(params, grads)])
        n = lib().fbfc_adamw_state_elements(table, len(params))
        self.mScale = self.vScale = None
        if stateBits == 32:
            self.m, self.v = (torch.zeros(n, device=self.device) for _ in range(2))
        else:
            self.m, self.v = (torch.zeros(n, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn) for _ in range(2))
            self.mScale, self.vScale = (torch.zeros(n // 256, device=self.device) for _ in range(2))
        config = AdamwConfig(TYPES[params[0].dtype], TYPES[grads[0].dtype], stateBits, seed & 0xFFFFFFFF, betas[0], betas[1], eps)
        with torch.cuda.device(self.device):
            check(lib().fbfc_adamw_create(ctypes.byref(config), table, len(params), _ptr(self.m), _ptr(self.v),
                                          _ptr(self.mScale), _ptr(self.vScale), ctypes.byref(self._handle)))

    @classmethod
    def fromModules(cls, modules, **kw):
        """An optimizer of all the parameters of the modules."""
        params, grads = [], []
        for module in modules:
            p, g = module.parameters()
            params += p
            grads += g
        return cls(params, grads, **kw)

    def step(self, scale=1.0):
        """One step with the gradients times `scale`, on the current stream."""
        if torch.cuda.current_device() == self.device.index:
            check(lib().fbfc_adamw_step(self._handle, self.lr, self.weightDecay, scale, _stream()))
            return
        with torch.cuda.device(self.device):
            check(lib().fbfc_adamw_step(self._handle, self.lr, self.weightDecay, scale, _stream()))

    @property
    def t(self):
        """The number of steps taken; waits for the current stream."""
        with torch.cuda.device(self.device):
            n = ctypes.c_long(0)
            check(lib().fbfc_adamw_get_step(self._handle, ctypes.byref(n), _stream()))
            return n.value

    def loadState(self, m, v, mScale=None, vScale=None, t=0):
        """Copies states that another optimizer of the same tensors held after `t` steps."""
        given, mine = (m, v, mScale, vScale), (self.m, self.v, self.mScale, self.vScale)
        for x, y, name in zip(given, mine, ("m", "v", "mScale", "vScale")):
            if (x is None) != (y is None):
                raise ValueError("%s does not go with %d-bit states" % (name, self.stateBits))
            if x is not None and not isinstance(x, torch.Tensor):
                raise TypeError("%s must be a tensor" % name)
            if x is not None and (x.dtype != y.dtype or x.shape != y.shape):
                raise ValueError("%s must be %s of shape %s" % (name, y.dtype, tuple(y.shape)))
        with torch.cuda.device(self.device):
            check(lib().fbfc_adamw_set_step(self._handle, t, _stream()))   # refuses a number of steps before anything is copied
        for x, y in zip(given, mine):
            if x is not None:
                y.copy_(x)

    def close(self):
        if self._handle:
            lib().fbfc_adamw_destroy(self._handle)
            self._handle = ctypes.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
