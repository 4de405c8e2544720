"""Loss of a language model's head and its gradients (``include/anni_head.h``).

``head_loss`` and ``head_loss_grad`` take torch tensors, allocate their workspace from torch for the length of
the call and run on the current stream; nothing is kept between calls.  With ``stream=`` they run there: the caller
orders the two streams, and all tensors of the call stay allocated until that stream has finished with them.  The
results carry no autograd history: the gradients are ``head_loss_grad``'s.
"""
import contextlib
import ctypes as C

import torch

from . import capi
from .capi import DT_BF16, DT_F32, check

HEAD_ACCUMULATE = 1
_GRAD_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16}


class Call(C.Structure):
    """anni_head_call."""
    _fields_ = [("x", C.c_void_p), ("ldx", C.c_int64), ("w", C.c_void_p), ("ldw", C.c_int64),
                ("bias", C.c_void_p), ("target", C.c_void_p), ("tokens", C.c_int64), ("d_model", C.c_int32),
                ("vocab", C.c_int32), ("nll", C.c_void_p), ("lse", C.c_void_p), ("weight", C.c_void_p),
                ("grad_scale", C.c_double), ("grad_dtype", C.c_int), ("flags", C.c_int), ("dx", C.c_void_p),
                ("lddx", C.c_int64), ("dw", C.c_void_p), ("lddw", C.c_int64), ("dbias", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


_L = None


def lib():
    """The library with these entry points typed."""
    global _L
    if _L is None:
        L = capi.lib()
        P = C.POINTER(Call)
        L.anni_head_workspace.restype = C.c_int
        L.anni_head_workspace.argtypes = [P, C.c_int, C.POINTER(C.c_size_t)]
        L.anni_lm_adam_head_call.restype = C.c_int
        L.anni_lm_adam_head_call.argtypes = [C.c_void_p, C.c_int, C.c_int, P]
        for f in (L.anni_head_loss, L.anni_head_loss_grad):
            f.restype = C.c_int
            f.argtypes = [P, C.c_void_p]
        _L = L
    return _L


def _rows(name, t, rows, cols, dtype, device):
    """Address and row stride of a matrix whose rows are contiguous."""
    if t.dtype != dtype or t.device != device or t.dim() != 2 or t.shape != (rows, cols):
        raise TypeError(f"head: {name} must be a {dtype} tensor of shape ({rows}, {cols}) on {device}")
    if cols > 1 and t.stride(1) != 1 or rows > 1 and t.stride(0) < cols:
        raise ValueError(f"head: the rows of {name} must be contiguous and apart")
    return t.data_ptr(), (t.stride(0) if rows > 1 else cols)


def _flat(name, t, n, dtype, device):
    if t.dtype != dtype or t.device != device or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise TypeError(f"head: {name} must be a contiguous {dtype} tensor of {n} elements on {device}")
    return t.data_ptr()


def _call(x, w, target, bias):
    if not x.is_cuda:
        raise RuntimeError("anni_b200 needs a CUDA device: there is no CPU path")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[0]:
        raise ValueError("head: x is (tokens, d_model), w is (d_model, vocab)")
    c = Call()
    (c.tokens, c.d_model), c.vocab = x.shape, w.shape[1]
    c.x, c.ldx = _rows("x", x, *x.shape, torch.bfloat16, x.device)
    c.w, c.ldw = _rows("w", w, *w.shape, torch.bfloat16, x.device)
    c.target = _flat("target", target, c.tokens, torch.int32, x.device)
    if bias is not None:
        c.bias = _flat("bias", bias, c.vocab, torch.float32, x.device)
    return c


def _here(device, stream):
    """A context in which `device` and `stream` are current; nothing to do where they are already."""
    if stream is None and device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    both = contextlib.ExitStack()
    both.enter_context(torch.cuda.device(device))
    both.enter_context(torch.cuda.stream(stream))       # None: no change
    return both


def _used_on(stream, *tensors):
    """The memory of these tensors is not handed out again before `stream` has done what is queued on it when they die."""
    if stream is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _run(name, c, grad, device):
    L = lib()
    need = C.c_size_t()
    check("anni_head_workspace", L.anni_head_workspace(c, grad, need))
    # the allocator hands the block to later work of this stream only: no other call can hold it meanwhile
    ws = torch.empty(need.value, dtype=torch.uint8, device=device)
    c.workspace, c.workspace_bytes = ws.data_ptr(), need.value
    check(name, getattr(L, name)(c, torch.cuda.current_stream(device).cuda_stream))


def head_loss(x, w, target, *, bias=None, stream=None):
    """Rows of (nll, lse): x bf16 (tokens, d_model), w bf16 (d_model, vocab), target int32 (tokens), bias fp32
    (vocab) or None.  A target below 0 is ignored (nll 0), one beyond the vocabulary gives NaN."""
    c = _call(x, w, target, bias)
    caller = None if stream is None else torch.cuda.current_stream(x.device)
    with _here(x.device, stream):
        nll, lse = torch.empty(2, c.tokens, dtype=torch.float32, device=x.device).unbind(0)
        c.nll, c.lse = nll.data_ptr(), lse.data_ptr()
        _run("anni_head_loss", c, 0, x.device)
    _used_on(stream, x, w, target, bias)
    _used_on(caller, nll)               # lse is of the same storage; both were allocated on `stream`
    return nll, lse


def head_loss_grad(x, w, target, lse, *, bias=None, weight=None, grad_scale=1.0, dx=None, dw=None, dbias=None,
                   accumulate=False, stream=None):
    """Gradients of ``grad_scale * sum(weight * nll)`` into those of ``dx`` (tokens, d_model), ``dw`` (d_model,
    vocab), ``dbias`` (vocab) that are given, all fp32 or all bf16; with ``accumulate`` dw and dbias are added to.
    ``lse`` is ``head_loss``'s of the same x, w and bias; ``weight`` fp32 (tokens) or None."""
    c = _call(x, w, target, bias)
    kinds = {t.dtype for t in (dx, dw, dbias) if t is not None}
    if len(kinds) > 1 or not kinds <= set(_GRAD_DT):
        raise TypeError("head: gradients are all float32 or all bfloat16")
    kind = kinds.pop() if kinds else torch.float32
    c.grad_dtype, c.grad_scale, c.flags = _GRAD_DT[kind], grad_scale, HEAD_ACCUMULATE if accumulate else 0
    c.lse = _flat("lse", lse, c.tokens, torch.float32, x.device)
    if weight is not None:
        c.weight = _flat("weight", weight, c.tokens, torch.float32, x.device)
    if dx is not None:
        c.dx, c.lddx = _rows("dx", dx, c.tokens, c.d_model, kind, x.device)
    if dw is not None:
        c.dw, c.lddw = _rows("dw", dw, c.d_model, c.vocab, kind, x.device)
    if dbias is not None:
        c.dbias = _flat("dbias", dbias, c.vocab, kind, x.device)
    with _here(x.device, stream):
        _run("anni_head_loss_grad", c, 1, x.device)
    _used_on(stream, x, w, target, lse, bias, weight, dx, dw, dbias)
