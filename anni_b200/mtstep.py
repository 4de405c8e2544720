"""AdamW over a list of tensors (``include/anni_mtstep.h``): the step of ``engine.OptStep`` for tensors
that lie wherever their owner put them, with moments in 32 bits or in 8.

torch provides device memory and streams; all arithmetic of a step happens inside ``libanni_b200.so``.
"""
import ctypes as C

import torch

from . import capi
from .capi import DT_BF16, DT_F32, DT_Q8, MT_BLOCK, SEG_TWIN_BF16, SEG_WD, check

_GRAD_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16}
_TOP_M, _TOP_V = 448.0, 57344.0


class Tensor(C.Structure):
    """anni_mt_tensor."""
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("m", C.c_void_p), ("v", C.c_void_p),
                ("m_scale", C.c_void_p), ("v_scale", C.c_void_p), ("twin_bf16", C.c_void_p),
                ("n", C.c_int64), ("flags", C.c_uint32)]


def lib():
    """The library with this object's entry points typed."""
    L = capi.lib()
    i, vp = C.c_int, C.c_void_p
    L.anni_mtstep_create.restype = i
    L.anni_mtstep_create.argtypes = [C.POINTER(Tensor), i, i, i, C.POINTER(vp)]
    L.anni_mtstep_destroy.restype = None
    L.anni_mtstep_destroy.argtypes = [vp]
    L.anni_mtstep_set_grads.restype = i
    L.anni_mtstep_set_grads.argtypes = [vp, C.POINTER(vp), vp]
    L.anni_mtstep_step.restype = i
    L.anni_mtstep_step.argtypes = [vp, C.POINTER(capi.Hyper), C.c_uint64, vp]
    L.anni_mtstep_status_read.restype = i
    L.anni_mtstep_status_read.argtypes = [vp, C.POINTER(capi.Status), vp]
    return L


def _blocks(n):
    return -(-n // MT_BLOCK)


def encode(x, kind):
    """fp32 moments as 8-bit numbers of ``kind`` (torch.float8_e4m3fn for m, torch.float8_e5m2 for v) and the
    scale of each block of 256 elements, rounded to nearest as a step rounds them: for loading 32-bit moments."""
    x = x.reshape(-1).float()
    top = _TOP_M if kind == torch.float8_e4m3fn else _TOP_V
    pad = torch.nn.functional.pad(x, (0, -x.numel() % MT_BLOCK)).view(-1, MT_BLOCK)
    amax = pad.abs().amax(1, keepdim=True)
    some = ~(amax < 2.0 ** -100)
    y = (pad * torch.where(some, top / amax, 0.0)).clamp(-top, top).to(kind)
    if kind == torch.float8_e5m2:
        y = torch.maximum(y.view(torch.uint8), ((pad > 0) & some).to(torch.uint8)).view(kind)
    return y.view(-1)[:x.numel()].clone(), torch.where(some, amax / top, 0.0).view(-1)


def decode(codes, scale):
    """8-bit moments and their scales as fp32: for checkpoints."""
    x = codes.reshape(-1).float()
    return x * scale.repeat_interleave(MT_BLOCK)[:x.numel()]


class MultiStep:
    """The step over ``params``, a list of contiguous fp32 CUDA tensors.

    ``grads``: one tensor per parameter, all fp32 or all bf16, or None for a tensor that sits out; they may
    be replaced by ``set_grads`` (or ``step(..., grads=)``) whenever their owner reallocates them.
    ``decay``: per tensor, whether decoupled decay applies (default: to all).  ``twins``: bf16 tensors that
    receive the rounded parameters, or None.  ``state_dtype``: DT_F32 (``m``, ``v`` fp32) or DT_Q8 (``m``
    float8_e4m3fn, ``v`` float8_e5m2, ``m_scale`` and ``v_scale`` fp32 per 256 elements); zeroed state is
    made here unless ``moments=(m, v)`` and, for DT_Q8, ``scales=(m_scale, v_scale)`` hand it in.

    Calls on one object, this one among them, belong on one stream.  Every call works on the list's device.  Gradients given to a call with
    ``stream=`` stay allocated until that stream has finished with them, also when others have replaced them; those
    that a captured step reads are the caller's to keep for as long as it is replayed.
    """

    def __init__(self, params, *, grads=None, state_dtype=DT_F32, grad_dtype=None, decay=None, twins=None,
                 moments=None, scales=None):
        self.h = None
        params = list(params)
        if not params:
            raise ValueError("MultiStep: the list of tensors is empty")
        if state_dtype == DT_Q8 and moments is not None and scales is None:
            raise ValueError("MultiStep: 8-bit moments come with their scales")
        n = len(params)
        grads = [None] * n if grads is None else list(grads)
        if grad_dtype is None:
            kinds = {g.dtype for g in grads if g is not None}
            if len(kinds) > 1 or not kinds <= set(_GRAD_DT):
                raise TypeError(f"MultiStep: gradients are all float32 or all bfloat16, got {sorted(map(str, kinds))}")
            grad_dtype = _GRAD_DT[kinds.pop()] if kinds else DT_F32
        self.params, self.grad_dtype, self.state_dtype = params, grad_dtype, state_dtype
        self.counts = [p.numel() for p in params]
        self.device = params[0].device
        if self.device.type != "cuda":
            raise RuntimeError("anni_b200 needs a CUDA device: there is no CPU path")
        if state_dtype not in (DT_F32, DT_Q8):
            raise ValueError("MultiStep: state_dtype is DT_F32 or DT_Q8")
        eight = state_dtype == DT_Q8
        if moments is None:
            kinds = (torch.float8_e4m3fn, torch.float8_e5m2) if eight else (torch.float32, torch.float32)
            moments = [[torch.zeros(p.numel(), dtype=torch.uint8 if eight else k, device=self.device).view(k) for p in params]
                       for k in kinds]
        if scales is None and eight:
            scales = [[torch.zeros(_blocks(p.numel()), dtype=torch.float32, device=self.device) for p in params] for _ in range(2)]
        self.m, self.v = map(list, moments)
        self.m_scale, self.v_scale = map(list, scales) if eight else (None, None)
        self.twins = list(twins) if twins is not None else [None] * n
        decay = [True] * n if decay is None else list(decay)
        self._check("params", params, torch.float32)
        self._check("m", self.m, torch.float8_e4m3fn if eight else torch.float32)
        self._check("v", self.v, torch.float8_e5m2 if eight else torch.float32)
        if eight:
            blocks = [_blocks(k) for k in self.counts]
            self._check("m_scale", self.m_scale, torch.float32, blocks)
            self._check("v_scale", self.v_scale, torch.float32, blocks)
        self._check("twins", self.twins, torch.bfloat16, none=True)
        self._check_grads(grads)
        if len(decay) != n:
            raise ValueError("MultiStep: decay needs one entry per parameter")
        arr = (Tensor * n)()
        # of entries without elements the library looks at nothing but the count
        for field, xs in (("param", params), ("grad", grads), ("m", self.m), ("v", self.v), ("m_scale", self.m_scale),
                          ("v_scale", self.v_scale), ("twin_bf16", self.twins)):
            for t, x in zip(arr, xs or ()):
                if x is not None and x.numel():
                    setattr(t, field, x.data_ptr())
        for t, k, wd, twin in zip(arr, self.counts, decay, self.twins):
            t.n, t.flags = k, (SEG_WD if wd else 0) | (SEG_TWIN_BF16 if twin is not None else 0)
        self.grads, self.grads_on = grads, None
        self.L = lib()
        h = C.c_void_p()
        with torch.cuda.device(self.device):
            check("anni_mtstep_create", self.L.anni_mtstep_create(arr, n, grad_dtype, state_dtype, C.byref(h)))
        self.h = h

    def _check(self, what, xs, dtype, counts=None, none=False):
        if len(xs) != len(self.params):
            raise ValueError(f"MultiStep: {what} needs one entry per parameter")
        dev = self.device.index
        for k, (x, n) in enumerate(zip(xs, self.counts if counts is None else counts)):
            if none and x is None:
                continue
            if x.dtype is not dtype or x.get_device() != dev or not x.is_contiguous():
                raise TypeError(f"MultiStep: {what}[{k}] must be a contiguous {dtype} tensor on {self.device}")
            if x.numel() != n:
                raise ValueError(f"MultiStep: {what}[{k}] has {x.numel()} elements, not {n}")

    def _check_grads(self, grads):
        self._check("grads", grads, torch.bfloat16 if self.grad_dtype == DT_BF16 else torch.float32, none=True)

    def _stream(self, stream):
        s = torch.cuda.current_stream(self.device) if stream is None else stream
        return C.c_void_p(s.cuda_stream)

    def _hold_grads(self, stream):
        """The gradients' memory is not handed out again before `stream` has done what is queued on it when they go."""
        if stream is not None and self.grads_on != stream.cuda_stream:
            for g in self.grads:
                if g is not None:
                    g.record_stream(stream)
            self.grads_on = stream.cuda_stream

    def set_grads(self, grads, stream=None):
        """New gradient tensors (None: sits out) for the steps queued after this call on the same stream."""
        grads = list(grads)
        self._check_grads(grads)
        arr = (C.c_void_p * len(grads))(*[g.data_ptr() if g is not None and g.numel() else None for g in grads])
        check("anni_mtstep_set_grads", self.L.anni_mtstep_set_grads(self.h, arr, self._stream(stream)))
        self.grads, self.grads_on = grads, None
        self._hold_grads(stream)

    def step(self, hp, *, seed=0, grads=None, stream=None):
        """One step (``hp`` from ``OptStep.hyper``); ``seed`` chooses the random bits of STEP_STOCHASTIC."""
        if grads is not None:
            self.set_grads(grads, stream)
        check("anni_mtstep_step", self.L.anni_mtstep_step(self.h, C.byref(hp), seed & (2 ** 64 - 1), self._stream(stream)))
        self._hold_grads(stream)

    def status(self, stream=None):
        st = capi.Status()
        check("anni_mtstep_status_read", self.L.anni_mtstep_status_read(self.h, C.byref(st), self._stream(stream)))
        return st

    def moments(self):
        """m and v as lists of fp32 tensors of the parameters' shapes (copies in the 8-bit form)."""
        if self.state_dtype == DT_F32:
            return tuple([x.view(p.shape) for x, p in zip(xs, self.params)] for xs in (self.m, self.v))
        return ([decode(x, s).view(p.shape) for x, s, p in zip(self.m, self.m_scale, self.params)],
                [decode(x, s).view(p.shape) for x, s, p in zip(self.v, self.v_scale, self.params)])

    def close(self):
        """Releases the handle's device tables; steps still queued must have finished."""
        if getattr(self, "h", None):
            self.L.anni_mtstep_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
