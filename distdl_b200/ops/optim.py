"""Fused AdamW step and sum-of-squares kernels on flat fp32 buffers; the norm of many gradients and their clipping."""
from __future__ import annotations

import array
import ctypes
import functools

import torch

from .. import _native
from ._util import call_on, ordinary, ptr, stream_ptr, use_native

_native.declare("dd_grad_norm_parts", [ctypes.c_int])
_native.declare("dd_grad_norm", [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p,
                                 ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_double, ctypes.c_int, ctypes.c_int,
                                 ctypes.c_void_p])


def adamw_step_(master, m, v, grad, param_bf16, *, lr, beta1, beta2, eps, weight_decay, step,
                grad_scale_tensor=None, grad_scale=1.0, zero_grad=True):
    """In-place AdamW on flat fp32 ``master``/``m``/``v`` with fp32 ``grad``;
    refreshes the bf16 working copy and clears the gradient in the same pass."""
    n = master.numel()
    if n == 0:
        return
    if use_native(master):
        _native.call("dd_adamw", master.data_ptr(), m.data_ptr(), v.data_ptr(), grad.data_ptr(), ptr(param_bf16), n,
                     lr, beta1, beta2, eps, weight_decay, step, ptr(grad_scale_tensor), grad_scale, int(zero_grad),
                     stream_ptr())
        return
    # library-kernel path (CPU plumbing and the baseline arm): processed in slices so
    # that the temporaries stay small next to the optimizer state
    bc1 = 1 - beta1 ** step
    bc2 = 1 - beta2 ** step
    chunk = 1 << 26
    for lo in range(0, n, chunk):
        sl = slice(lo, min(n, lo + chunk))
        g = grad[sl] * grad_scale
        if grad_scale_tensor is not None:
            g = g * grad_scale_tensor
        m[sl].mul_(beta1).add_(g, alpha=1 - beta1)
        v[sl].mul_(beta2).addcmul_(g, g, value=1 - beta2)
        denom = (v[sl] / bc2).sqrt_().add_(eps)
        master[sl].mul_(1 - lr * weight_decay).addcdiv_(m[sl], denom, value=-lr / bc1)
        if zero_grad:
            grad[sl].zero_()
        if param_bf16 is not None:
            param_bf16[sl].copy_(master[sl])


def sumsq_(x: torch.Tensor, out: torch.Tensor) -> None:
    """out[0] += sum(x**2) for a flat fp32 tensor."""
    if x.numel() == 0:
        return
    if use_native(x):
        _native.call("dd_sumsq_f32", x.data_ptr(), x.numel(), out.data_ptr(), stream_ptr())
    else:
        for lo in range(0, x.numel(), 1 << 26):
            c = x[lo:lo + (1 << 26)]
            out += (c.float() * c.float()).sum()


def accumulate_f32_(acc: torch.Tensor, g: torch.Tensor, scale: float = 1.0) -> None:
    """``acc += scale * g`` with a flat fp32 accumulator and a gradient of any
    float dtype (one fused cast-and-add kernel for contiguous bf16 on a GPU)."""
    if use_native(g) and g.dtype == torch.bfloat16 and g.is_contiguous() and acc.is_contiguous():
        _native.call("dd_cast_bf16_f32", g.data_ptr(), acc.data_ptr(), g.numel(), float(scale), 1, stream_ptr())
    else:
        acc.add_(g.reshape(-1).to(acc.dtype), alpha=scale)


_Parameter = torch.nn.Parameter
_TYPES = {torch.Tensor, _Parameter}             # (others may hold their elements elsewhere)
_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements of ``t`` fill a piece of memory without holes and without sharing any, in whatever order."""
    if t.is_contiguous():
        return True
    need = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != need:
            return False
        need *= n
    return True


def _tensors(tensors, norm=None):
    """(addresses, sizes, type codes) of the tensors as C arrays, or None where the kernels do not take them (CUDA, bf16 /
    fp16 / fp32, dense)."""
    device = tensors[0].device
    where = device.index if device.type == "cuda" else -1
    if any([t.get_device() != where for t in tensors]):
        raise ValueError(f"gradients on {device} and elsewhere: a norm is of one device's tensors")
    if any([t.layout is not torch.strided for t in tensors]):
        raise ValueError("gradients are dense tensors")
    codes = [_CODES.get(t.dtype, 9) for t in tensors]
    if 9 in codes:
        for t in tensors:
            if not t.is_floating_point():
                raise ValueError(f"gradients are floating-point tensors, not {t.dtype}")
        return None
    if not use_native(tensors[0]) or not ordinary(tensors[0], norm) \
            or not _TYPES.issuperset([type(t) for t in tensors]) or not all([t.is_contiguous() or _dense(t) for t in tensors]):
        return None
    return (array.array("Q", [t.data_ptr() for t in tensors]), array.array("q", [t.numel() for t in tensors]),
            array.array("B", codes))


def _parts(tensors, norm=None):
    """(tensors that the kernels take, their :func:`_tensors` or None, the others)."""
    lists = _tensors(tensors, norm)
    if lists is not None:
        return tensors, lists, []
    taken = [t.dtype in _CODES and type(t) in _TYPES and _dense(t) for t in tensors]
    if any(taken) and not all(taken):
        mine = [t for t, own in zip(tensors, taken) if own]
        lists = _tensors(mine, norm)
        if lists is not None:
            return mine, lists, [t for t, own in zip(tensors, taken) if not own]
    return [], None, tensors


def _flat(tensors):
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    return [t for t in tensors if t is not None]


def gradients_of(tensors):
    """The gradients meant by ``tensors`` (one, or an iterable): of a parameter, trained or frozen, its ``.grad``, of which there
    may be none; anything else as it is."""
    return _flat([t.grad if (t.requires_grad and t.is_leaf) or (type(t) is not torch.Tensor and isinstance(t, _Parameter)) else t
                  for t in _flat(tensors)])


def _plain_sumsq(tensors):
    return torch.stack([t.detach().double().square().sum() for t in tensors]).sum()


@functools.lru_cache(maxsize=256)
def _norm_parts(device: int, count: int) -> int:
    with torch.cuda.device(device):
        return _native.lib().dd_grad_norm_parts(count)


def _grad_norm(tensors, lists, norm, squared, max_norm, given, clip):
    p, n, code = (a.buffer_info()[0] for a in lists)
    parts = 0 if given else _norm_parts(tensors[0].get_device(), len(tensors))
    scratch = None if given else torch.empty(parts, dtype=torch.float64, device=tensors[0].device)
    call_on(tensors[0], "dd_grad_norm", p, n, code, len(tensors), ptr(scratch), parts, ptr(norm), ptr(squared), max_norm,
            int(given), int(clip))


def grad_norm(tensors, squared: bool = False) -> torch.Tensor:
    """The 2-norm of all elements of ``tensors`` (one tensor, or an iterable; None is passed over) as an fp32 scalar on their
    device, or with ``squared`` the sum of squares in fp64 (to be added over workers).  Squares and sums are formed in 64
    bits, in an order that does not change from run to run.  bf16, fp16 and fp32, mixed as they come, run on the kernels;
    fp64, subclasses and views with holes among them by torch's operators."""
    tensors = _flat(tensors)
    if not tensors:
        return torch.zeros((), dtype=torch.float64 if squared else torch.float32)
    mine, lists, others = _parts(tensors)
    if others:
        total = _plain_sumsq(others)
        if mine:
            total = total + grad_norm(mine, squared=True)
        return total if squared else total.sqrt().float()
    out = torch.empty((), dtype=torch.float64 if squared else torch.float32, device=tensors[0].device)
    _grad_norm(tensors, lists, None if squared else out, out if squared else None, 0.0, False, False)
    return out


def clip_grad_norm_(tensors, max_norm: float, norm: torch.Tensor = None) -> torch.Tensor:
    """Scales gradients in place by ``min(1, max_norm / (norm + 1e-6))``, ``norm`` being their 2-norm, which is returned (an
    fp32 scalar on their device; nothing waits for it).  ``tensors``: gradients, or parameters (and other leaves that require
    a gradient), whose ``.grad`` is meant, also where they are frozen; None is passed over.  ``norm`` given (an fp32 scalar
    on their device, say of the gradients of all workers): that norm is taken.  Where the norm is not above ``max_norm``
    nothing is written; one that is not a number makes all gradients so.  The tensors must not share memory with one
    another."""
    tensors = gradients_of(tensors)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, and a number: {max_norm}")
    if norm is not None and (norm.numel() != 1 or norm.dtype != torch.float32):
        raise ValueError(f"norm must be an fp32 scalar, not {tuple(norm.shape)} {norm.dtype}")
    if not tensors:
        return torch.zeros((), dtype=torch.float32) if norm is None else norm
    if norm is not None and norm.device != tensors[0].device:
        raise ValueError(f"the norm is on {norm.device}, the gradients on {tensors[0].device}")
    mine, lists, others = _parts(tensors, norm)
    if others and norm is None:
        norm = grad_norm(tensors)
    if mine:
        given = norm is not None
        if not given:
            norm = torch.empty((), dtype=torch.float32, device=mine[0].device)
        _grad_norm(mine, lists, norm, None, max_norm, given, True)
        torch.autograd.graph.increment_version(mine)          # (passes over tensors of inference mode)
    if others:
        with torch.no_grad():
            scale = (max_norm / (norm + 1e-6)).clamp(max=1.0).reshape(())
            for t in others:
                t.copy_(t * scale if t.dtype == torch.float64 else t.float() * scale)
    return norm
