# coding: utf-8
"""AdamW over many tensors in one launch, with moments in 32 or in 8 bits."""
import ctypes

import torch

from .core import _LIB, _call_and_throw_if_error
from .lookup import _TYPE, _extent, _float_type, _memory, _one_device, _stream, _tensor

__all__ = ["AdamW"]


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
    sharing memory with another.  Arithmetic is float32; ``master=True`` keeps a float32 copy of
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
            _float_type(_tensor(p, "a parameter"), "a parameter")
            if not p.is_contiguous():
                raise ValueError("a parameter is not contiguous")
        extents = sorted(_extent(p) for p in params if p.numel())
        for a, b in zip(extents, extents[1:]):
            if b[0] < a[1]:
                raise ValueError("two parameters share memory")
        self._config = _Config(float(betas[0]), float(betas[1]), float(eps), float(weight_decay), int(state_bits),
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
        index = None
        for p in params:
            index = _one_device(params[0], parameter=p)
        self.device = params[0].device
        self._index = index
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
        self._grads = None if grads is None else self._pointers(grads)
        self._bound = None if grads is None else list(grads)
        self._versions = [p for p in params if p.requires_grad]
        self._stream = _stream(index)
        self._workspace = _memory(size.value, self.device)
        for name in ("moment1", "moment2", "scale1", "scale2", "master"):
            buf = getattr(self, name)
            setattr(self._config, name, None if buf is None else buf.data_ptr())
        torch.cuda.current_stream(self.device).synchronize()  # the library uploads its table on its own
        self._handle = ctypes.c_void_p()
        _call_and_throw_if_error(_LIB.AAdamWCreate(table, len(params), ctypes.byref(self._config),
                                                   self._workspace.data_ptr(), index, ctypes.byref(self._handle)))

    def __del__(self):
        handle = getattr(self, "_handle", None)
        if handle is not None and _LIB is not None:
            _LIB.AFreeAdamW(handle)
            self._handle = None

    @staticmethod
    def _rate(lr):
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.numel() != 1:
                raise TypeError("lr must be a number or a float32 tensor of one element")
            return lr
        return float(lr)

    def _pointers(self, grads):
        """(address array, all float32?) of one gradient, or None, for every parameter."""
        if len(grads) != len(self.params):
            raise ValueError("%d gradients for %d parameters" % (len(grads), len(self.params)))
        same, single, at = True, True, []
        for g, p in zip(grads, self.params):
            if g is None:
                at.append(None)
                continue
            if not isinstance(g, torch.Tensor) or g.shape != p.shape or not g.is_contiguous():
                raise ValueError("a gradient must be a contiguous tensor of its parameter's shape")
            if g.device != p.device:
                raise ValueError("a gradient is on %s, its parameter on %s" % (g.device, p.device))
            if g.dtype != torch.float32:
                single = False
            if g.dtype != p.dtype:
                same = False
            at.append(g.data_ptr())
        if not same and not single:
            raise TypeError("gradients must have their parameters' types, or all be float32")
        return (ctypes.c_void_p * len(at))(*at), not same

    def step(self, grads=None, lr=None, grad_scale=None):
        """One step.  grads: one tensor, or None (that parameter and its moments stay as they are),
        for every parameter; by default the tensors given at construction.  lr: a number or a
        float32 CUDA tensor of one element, by default the constructor's.  grad_scale: a float32
        CUDA tensor of one element that multiplies every gradient (clipping, loss scaling)."""
        if grads is None:
            if self._grads is None:
                raise ValueError("no gradients: pass grads to step() or to the constructor")
            pointers, single = self._grads
        else:
            pointers, single = self._pointers(grads)
        lr = self.lr if lr is None else self._rate(lr)
        lr_at = scale_at = None
        if isinstance(lr, torch.Tensor):
            _one_device(self.params[0], lr=lr)
            lr, lr_at = 0.0, lr.data_ptr()
        if grad_scale is not None:
            if not isinstance(grad_scale, torch.Tensor) or grad_scale.dtype != torch.float32 or grad_scale.numel() != 1:
                raise TypeError("grad_scale must be a float32 tensor of one element")
            _one_device(self.params[0], grad_scale=grad_scale)
            scale_at = grad_scale.data_ptr()
        stream = _stream(self._index)
        if stream != self._stream:
            self._on_another_stream()
        _call_and_throw_if_error(_LIB.AAdamWStep(self._handle, pointers, len(self.params), int(single), lr, lr_at,
                                                 scale_at, stream))
        if self._versions:  # autograd sees that they changed
            torch.autograd.graph.increment_version(self._versions)

    def _on_another_stream(self):
        """The optimizer's memory must not be handed out again before that stream is done with it."""
        current = torch.cuda.current_stream(self.device)
        for x in (self.moment1, self.moment2, self.scale1, self.scale2, self.master, self._workspace):
            if x is not None:
                x.record_stream(current)

    @property
    def steps(self):
        """Steps taken so far (waits for the current stream)."""
        n = ctypes.c_int64(0)
        _call_and_throw_if_error(_LIB.AAdamWGetStep(self._handle, ctypes.byref(n), _stream(self._index)))
        return n.value

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
        for k in mine:
            getattr(self, k).copy_(state[k])
        _call_and_throw_if_error(_LIB.AAdamWSetStep(self._handle, int(state["step"]), _stream(self._index)))

    def moments(self, k):
        """First and second moment of parameter ``k`` as float32 tensors of its shape."""
        p, at = self.params[k], self.slots[k]
        cut = lambda x: x[at:at + p.numel()].view(p.shape)  # noqa: E731
        if self.scale1 is None:
            return cut(self.moment1).clone(), cut(self.moment2).clone()
        wide = lambda x, s: (x.float().view(-1, 128) * s[:, None]).view(-1)  # noqa: E731
        return cut(wide(self.moment1, self.scale1)), cut(wide(self.moment2, self.scale2)).square()
