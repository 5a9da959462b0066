# coding: utf-8
"""AdamW over many tensors in one launch, with moments in 32 or in 8 bits."""
import ctypes

import torch

from .core import _LIB, _call_and_throw_if_error
from .lookup import _tensors

__all__ = ["AdamW"]

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Param(ctypes.Structure):
    _fields_ = [("param", ctypes.c_void_p), ("size", ctypes.c_int64), ("type", ctypes.c_int)]


class _Config(ctypes.Structure):
    _fields_ = [("beta1", ctypes.c_double), ("beta2", ctypes.c_double), ("eps", ctypes.c_double),
                ("weight_decay", ctypes.c_double), ("state_bits", ctypes.c_int), ("seed", ctypes.c_uint),
                ("moment1", ctypes.c_void_p), ("moment2", ctypes.c_void_p), ("scale1", ctypes.c_void_p),
                ("scale2", ctypes.c_void_p), ("master", ctypes.c_void_p)]


class AdamW(object):
    """Adam with decoupled weight decay on a list of CUDA tensors::

        m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

    params: contiguous float32 / bfloat16 / float16 tensors of one device, of any sizes, none
    sharing memory with another.  eps: 0 or at least 2^-126.  Arithmetic is float32; ``master=True`` keeps a float32 copy of
    the parameters that the steps update, and stores it rounded in the parameters.

    The moments of tensor k lie at elements ``slots[k] ..`` of the flat tensors ``moment1`` and
    ``moment2`` (and ``master``); a slot starts at a multiple of 128.  ``state_bits=8``: both are
    ``float8_e4m3fn`` numbers that ``scale1`` / ``scale2`` (one power of two for 128 elements)
    multiply, and ``moment2`` holds the SQUARE ROOT of the second moment.  They are rounded with a
    dither keyed by (element, step, ``seed``), so that small changes survive on average.

    ``grads``: gradient tensors that the program fills in place for every step; ``step()`` then
    needs no argument.  A step is one launch (one for every 2048 tensors), enqueued on the current
    stream of the device; the step count lives on the device, so a captured step counts every
    replay.  Steps of one optimizer must follow each other on the device.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 master=False, grads=None, seed=0):
        params = list(params)
        if not params:
            raise ValueError("params is empty")
        for p in params:
            if not isinstance(p, torch.Tensor) or p.dtype not in _TYPE:
                raise TypeError("a parameter must be a float32, bfloat16 or float16 tensor")
            if not p.is_contiguous():
                raise ValueError("a parameter is not contiguous")
        extents = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
        for a, b in zip(extents, extents[1:]):
            if b[0] < a[1]:
                raise ValueError("two parameters share memory")
        config = _Config(float(betas[0]), float(betas[1]), float(eps), float(weight_decay), int(state_bits),
                         int(seed) & 0xFFFFFFFF)
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self.lr = self._rate(lr)
        self.params = params
        self.slots, end = [], 0
        for p in params:
            self.slots.append(end)
            end += (p.numel() + 127) // 128 * 128
        table = (_Param * len(params))(*[_Param(p.data_ptr(), p.numel(), _TYPE[p.dtype]) for p in params])
        length, size = ctypes.c_int64(0), ctypes.c_int64(0)
        _call_and_throw_if_error(_LIB.AAdamWBytes(table, len(params), ctypes.byref(length), ctypes.byref(size)))
        assert length.value == end
        for p in params:
            if p.device.type != "cuda":
                raise ValueError("the parameters must be CUDA tensors")
            if p.device != params[0].device:
                raise ValueError("a parameter is on %s, the others are on %s" % (p.device, params[0].device))
        self.device = params[0].device
        state = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        zeros = lambda n, t: torch.zeros(n, dtype=t, device=self.device)  # noqa: E731
        self.moment1, self.moment2 = zeros(end, state), zeros(end, state)
        self.scale1 = self.scale2 = self.master = None
        if state_bits == 8:
            self.scale1, self.scale2 = zeros(end // 128, torch.float32), zeros(end // 128, torch.float32)
        if master:
            self.master = zeros(end, torch.float32)
            for p, at in zip(params, self.slots):
                self.master[at:at + p.numel()].copy_(p.detach().reshape(-1))
        workspace = zeros(size.value, torch.uint8)
        torch.cuda.current_stream(self.device).synchronize()  # the library uploads its table on its own
        self._optimizer = _tensors.adamw(params, bytes(config), (self.moment1, self.moment2, self.scale1, self.scale2,
                                                                 self.master, workspace), grads)

    @staticmethod
    def _rate(lr):
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.numel() != 1:
                raise TypeError("lr must be a number or a float32 tensor of one element")
            return lr
        return float(lr)

    def step(self, grads=None, lr=None, grad_scale=None):
        """One step.  grads: one tensor, or None (that parameter and its moments stay as they are),
        for every parameter; by default the tensors given at construction.  lr: a number or a
        float32 CUDA tensor of one element, by default the constructor's.  grad_scale: a float32
        CUDA tensor of one element that multiplies every gradient (clipping, loss scaling)."""
        _tensors.adamw_step(self._optimizer, grads, self.lr if lr is None else lr, grad_scale)

    @property
    def steps(self):
        """Steps taken so far (waits for the current stream)."""
        return _tensors.adamw_count(self._optimizer, None)

    def state_dict(self):
        """The step count and the buffers themselves (no copies)."""
        out = {"step": self.steps, "moment1": self.moment1, "moment2": self.moment2}
        if self.scale1 is not None:
            out.update(scale1=self.scale1, scale2=self.scale2)
        if self.master is not None:
            out["master"] = self.master
        return out

    def load_state_dict(self, state):
        """Copies a state of the same layout (``state_dict``) into this optimizer."""
        mine = [k for k in ("moment1", "moment2", "scale1", "scale2", "master") if getattr(self, k) is not None]
        if sorted(state) != sorted(mine + ["step"]):
            raise ValueError("the state must hold %s" % ", ".join(["step"] + mine))
        for k in mine:
            x, y = getattr(self, k), state[k]
            if x.shape != y.shape or x.dtype != y.dtype:
                raise ValueError("%s must be %d elements of %s" % (k, x.numel(), x.dtype))
        _tensors.adamw_count(self._optimizer, int(state["step"]))  # refuses a bad count before anything is copied
        for k in mine:
            getattr(self, k).copy_(state[k])

    def moments(self, k):
        """First and second moment of parameter ``k`` as float32 tensors of its shape."""
        p, at = self.params[k], self.slots[k]
        cut = lambda x: x[at:at + p.numel()].view(p.shape)  # noqa: E731
        if self.scale1 is None:
            return cut(self.moment1).clone(), cut(self.moment2).clone()
        wide = lambda x, s: (x.float().view(-1, 128) * s[:, None]).view(-1)  # noqa: E731
        return cut(wide(self.moment1, self.scale1)), cut(wide(self.moment2, self.scale2)).square()
