"""Rotary positions in their usual variants, and the norm of every query and key head with the rotation in the same pass
(kernels in ``csrc/heads.cu``).  New relative to the reference, which has no attention code."""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from dataclasses import dataclass, fields
from typing import Optional

import torch

from .. import _native
from ._util import call_on, main_grad_now, ordinary, ordinary_gradient, ptr, use_native

_native.declare("dd_heads", [ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p])
_native.declare("dd_heads_parts", [])
# struct HeadsCall of csrc/heads.cu: ten addresses, nine long numbers, eleven numbers, three fp32 values
_CALL = struct.Struct("=10Q9q11i3f")
_SECOND = struct.Struct("=2q")                  # and what may follow it
_ROTATE, _FORWARD, _BACKWARD = 0, 1, 2

_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_SCALINGS = (None, "linear", "ntk", "yarn", "bands")


@dataclass(frozen=True)
class Rotary:
    """How positions turn the pairs of a head's components: pair ``i`` at position ``p`` by the angle ``p * f_i``,
    ``f_i = theta^(-2 i / dim)``.

    ``dim``: the leading components that turn (an even number; None: the whole head).  ``interleaved``: neighbours
    ``(2 i, 2 i + 1)`` are a pair, instead of ``(i, i + dim / 2)``.  ``scaling`` stretches the frequencies for contexts
    ``factor`` times longer than the ``original`` one:

    * ``"linear"``: ``f_i / factor``;
    * ``"ntk"``: ``theta * factor^(dim / (dim - 2))`` in the place of ``theta``;
    * ``"bands"``: with ``n_i = original f_i / (2 pi)`` turns over the original context, pairs with ``n_i > high`` stay, those
      with ``n_i < low`` get ``f_i / factor``, between them a weighted mean;
    * ``"yarn"``: the same from the pair that turns ``fast`` times (stays) to the one that turns ``slow`` times, along the
      pairs' numbers, and all results times ``magnitude`` (None: ``0.1 ln(factor) + 1``).

    ``magnitude`` (1 where it is None, but for ``"yarn"``) multiplies what is turned; components behind ``dim`` stay as
    they are."""
    theta: float = 500000.0
    dim: Optional[int] = None
    interleaved: bool = False
    scaling: Optional[str] = None
    factor: float = 1.0
    original: Optional[int] = None
    low: float = 1.0
    high: float = 4.0
    fast: float = 32.0
    slow: float = 1.0
    magnitude: Optional[float] = None

    def __post_init__(self):
        if not (math.isfinite(self.theta) and self.theta > 1.0):
            raise ValueError(f"theta must be finite and above 1, not {self.theta}")
        if self.dim is not None and (self.dim < 0 or self.dim % 2):
            raise ValueError(f"dim must be even, not {self.dim}")
        if self.scaling not in _SCALINGS:
            raise ValueError(f"scaling must be one of {_SCALINGS}, not {self.scaling!r}")
        if self.scaling is not None and not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError(f"factor must be finite and at least 1, not {self.factor}")
        if self.scaling in ("yarn", "bands") and (self.original is None or self.original < 1):
            raise ValueError(f"scaling {self.scaling!r} needs the original context length")
        if self.scaling == "bands" and not 0 <= self.low < self.high:
            raise ValueError(f"bands need 0 <= low < high, not {self.low} and {self.high}")
        if self.scaling == "yarn" and not 0 < self.slow < self.fast:
            raise ValueError(f"yarn needs 0 < slow < fast, not {self.slow} and {self.fast}")
        if self.magnitude is not None and not math.isfinite(self.magnitude):
            raise ValueError("magnitude must be finite")

    def rotated(self, head_dim: int) -> int:
        """The leading components of a head that turn."""
        dim = head_dim - head_dim % 2 if self.dim is None else self.dim
        if self.dim is None and head_dim % 2:
            raise ValueError(f"heads of {head_dim} components: say how many of them turn (dim)")
        if dim > head_dim:
            raise ValueError(f"{dim} components are to turn, the heads have {head_dim}")
        if self.scaling == "ntk" and dim == 2:
            raise ValueError("scaling 'ntk' needs more than one pair")
        return dim

    def _plan(self, head_dim: int):
        """(components that turn, neighbours?, address of the frequencies in turns per position, what multiplies) for the
        kernels, kept with the settings (the array that holds the frequencies as its last entry)."""
        plans = self.__dict__.get("_plans")
        if plans is None:
            plans = self.__dict__.setdefault("_plans", {})
        plan = plans.get(head_dim)
        if plan is None:
            dim = self.rotated(head_dim)
            arr = (ctypes.c_double * max(1, dim // 2))(*(f / (2 * math.pi) for f in _frequencies(self, dim)))
            # (the first of several threads' stays: its address may be in use)
            plan = plans.setdefault(head_dim, (dim, int(self.interleaved), ctypes.addressof(arr), self.scale, arr))
        return plan

    def __getstate__(self):                 # (copies and pickles hold the settings; addresses are this process's)
        return {f.name: getattr(self, f.name) for f in fields(self)}

    def __setstate__(self, state):
        self.__dict__.update(state)

    @property
    def scale(self) -> float:
        """What multiplies the turned components."""
        if self.magnitude is not None:
            return float(self.magnitude)
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "yarn" else 1.0

    def frequencies(self, head_dim: int) -> tuple:
        """``f_i`` of the pairs of a head, in radians per position (64 bits)."""
        return _frequencies(self, self.rotated(head_dim))


@functools.lru_cache(maxsize=256)
def _frequencies(rotary: Rotary, dim: int) -> tuple:
    theta, factor = float(rotary.theta), float(rotary.factor)
    if rotary.scaling == "ntk" and dim:
        theta *= factor ** (dim / (dim - 2))
    out = []
    for i in range(dim // 2):
        f = theta ** (-2.0 * i / dim)
        if rotary.scaling == "linear":
            f /= factor
        elif rotary.scaling == "bands":
            keep = (rotary.original * f / (2 * math.pi) - rotary.low) / (rotary.high - rotary.low)
            keep = min(1.0, max(0.0, keep))
            f = keep * f + (1.0 - keep) * f / factor
        elif rotary.scaling == "yarn":
            first, last = (dim * math.log(rotary.original / (2 * math.pi * turns)) / (2 * math.log(theta))
                           for turns in (rotary.fast, rotary.slow))
            first, last = max(math.floor(first), 0), min(math.ceil(last), dim - 1)
            slowed = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
            f = (1.0 - slowed) * f + slowed * f / factor
        out.append(f)
    return tuple(out)


def _place_of_ranges(ranges, tokens, seq, device):
    """(positions or None, offset, second) of a local sequence made of several ranges ``((start, length), ...)``: up to two of
    them travel with the call, ``second = (first place of the second, what its positions are ahead of the first's)``; of more
    the positions are listed on the device.  Nothing is kept: what one call makes belongs to its stream, mode and graph."""
    runs = []
    for a, n in ranges:
        a, n = int(a), int(n)
        if n < 0:
            raise ValueError(f"a range of positions has a length that is not negative, not {n}")
        if n and runs and runs[-1][0] + runs[-1][1] == a:
            runs[-1] = (runs[-1][0], runs[-1][1] + n)
        elif n:
            runs.append((a, n))
    n = sum(r[1] for r in runs)
    if n != seq:
        raise ValueError(f"the ranges hold {n} positions, a sequence has {seq} tokens")
    if tokens % max(1, n) or (n == 0 and tokens):
        raise ValueError(f"{tokens} tokens are not whole sequences of {n}")
    if len(runs) > 2:
        return torch.cat([torch.arange(a, a + m, dtype=torch.int64, device=device) for a, m in runs]), 0, None
    if not runs:
        return None, 0, None
    (a, n), second = runs[0], None
    if len(runs) == 2:
        second = (n, runs[1][0] - n - a)
    return None, a, second


def _where(qkv, rotary, seq, offset, ranges, positions):
    """The arguments that say how ``qkv [tokens, heads, head_dim]`` is turned: (rotary, positions or None, seq, offset,
    second): the position of a token of place ``i`` (its index modulo ``seq``) is ``positions[i]``, or ``offset + i``, and from
    the place ``second[0]`` on ``second[1]`` more."""
    if rotary is None:
        return None, None, 1, 0, None
    if not isinstance(rotary, Rotary):
        raise TypeError(f"rotary must be an ops.Rotary, not {type(rotary).__name__}")
    if ranges is not None:
        if positions is not None or offset:
            raise ValueError("give positions, ranges or an offset, not several of them")
        positions, offset, second = _place_of_ranges(ranges, qkv.shape[0], seq, qkv.device)
        return rotary, positions, max(1, int(seq)), offset, second
    if positions is None:
        if seq < 1:
            raise ValueError(f"a sequence has at least one token, not {seq}")
        return rotary, None, int(seq), int(offset), None
    if offset:
        raise ValueError("give positions or an offset, not both")
    if positions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"positions must be int64 or int32, not {positions.dtype}")
    if positions.device != qkv.device:
        raise ValueError(f"positions are on {positions.device}, the heads on {qkv.device}")
    n, tokens = positions.numel(), qkv.shape[0]
    if n != tokens and n != seq or (n == 0 and tokens) or (n and tokens % n):
        raise ValueError(f"{n} positions for {tokens} tokens in sequences of {seq}: one per token, or one per place in a "
                         f"sequence")
    if positions.dim() != 1 or not positions.is_contiguous():
        positions = positions.reshape(-1).contiguous()
    return rotary, positions, max(1, n), 0, None


def _angles(qkv, where):
    """(cos, sin) [tokens, 1, dim / 2] times the magnitude, fp32 from 64 bits (plain path)."""
    rotary, positions, seq, offset, second = where
    f = torch.tensor(rotary.frequencies(qkv.shape[2]), dtype=torch.float64, device=qkv.device)
    at = torch.arange(qkv.shape[0], device=qkv.device) % seq
    if positions is not None:
        at = positions[at]
    elif second is not None:
        at = torch.where(at < second[0], at, at + second[1]) + offset
    else:
        at = at + offset
    angle = (at.double().unsqueeze(1) * f).unsqueeze(1)
    wide = torch.float64 if qkv.dtype == torch.float64 else torch.float32
    return (rotary.scale * angle.cos()).to(wide), (rotary.scale * angle.sin()).to(wide)


def _rotated(x, cos, sin, dim, interleaved):
    if interleaved:
        a, b = x[..., 0:dim:2], x[..., 1:dim:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :dim // 2], x[..., dim // 2:dim]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., dim:]], dim=-1)


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _plain_rope(qkv, nheads, where, sign=1.0):
    rotary = where[0]
    cos, sin = _angles(qkv, where)
    sin = sign * sin
    y = _rotated(_wide(qkv[:, :nheads]), cos, sin, rotary.rotated(qkv.shape[2]), rotary.interleaved)
    return torch.cat([y.to(qkv.dtype), qkv[:, nheads:]], dim=1)


def _native_ok(qkv, *others):
    return use_native(qkv) and qkv.dtype in _DTYPE and 1 <= qkv.shape[2] <= 512 and ordinary(qkv, *others)


def _unit(t):
    """``t`` with its components next to one another."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _call(kind, x, out, hq, hkv, where, sign=1.0, wq=None, wk=None, eps=0.0, dy=None, dwq=None, dwk=None, partial=None,
          accumulate=False):
    """One call of the kernels on ``[tokens, heads, head_dim]`` tensors."""
    tokens, heads, hd = x.shape
    xs, os = x.stride(), out.stride()
    ds = xs if dy is None else dy.stride()
    rotary, positions, seq, offset, second = where
    dim, near, address, scale = (0, 0, 0, 1.0) if rotary is None else rotary._plan(hd)[:4]
    w = wk if wq is None else wq
    call = _CALL.pack(
        x.data_ptr(), 0 if dy is None else dy.data_ptr(), out.data_ptr(), ptr(wq), ptr(wk), ptr(dwq), ptr(dwk), ptr(partial),
        0 if positions is None else positions.data_ptr(), address, xs[0], xs[1], ds[0], ds[1], os[0], os[1], tokens, offset, seq,
        kind, _DTYPE[x.dtype], hq, hkv, heads - hq - hkv, hd, dim, near, w is not None and w.dtype == torch.float32,
        positions is not None and positions.dtype == torch.int64, accumulate, scale, sign, eps)
    if second is not None:
        call += _SECOND.pack(*second)
    call_on(x, "dd_heads", call, len(call))


def _rotated_copy(qkv, nheads, where, sign):
    src = _unit(qkv)
    out = torch.empty_like(src, memory_format=torch.contiguous_format)
    _call(_ROTATE, src, out, nheads, 0, where, sign)
    return out


class _RopeFn(torch.autograd.Function):
    """The rotation into a new tensor; its gradient is the rotation backwards, a call of the same function."""

    @staticmethod
    def forward(ctx, qkv, cfg):
        nheads, where, sign = cfg
        if where[1] is not None:
            ctx.save_for_backward(where[1])
        ctx.cfg = cfg
        return _rotated_copy(qkv, nheads, where, sign)

    @staticmethod
    def backward(ctx, d):
        nheads, where, sign = ctx.cfg
        return _turned_back(ctx, d, nheads, where, -sign), None


def _turned_back(ctx, d, nheads, where, sign):
    if where[1] is not None:
        where = (where[0], ctx.saved_tensors[0], *where[2:])     # (which says whether they have been changed since)
    if not ordinary_gradient(d):            # under a function transform: elementary operations
        return _plain_rope(d, nheads, where, sign)
    if torch.is_grad_enabled():             # differentiated itself
        return _RopeFn.apply(d, (nheads, where, sign))
    return _rotated_copy(d, nheads, where, sign)


class _RopeInPlaceFn(torch.autograd.Function):
    """The rotation in place of ``qkv``, which is read in the layout ``[tokens, heads, head_dim]``.  (The gradient is turned
    into a new tensor: the incoming one may be the caller's own.)"""

    @staticmethod
    def forward(ctx, qkv, cfg):
        layout, nheads, where = cfg
        ctx.mark_dirty(qkv)
        if where[1] is not None:
            ctx.save_for_backward(where[1])
        ctx.cfg = cfg
        t = qkv.view(layout)
        _call(_ROTATE, t, t, nheads, 0, where)
        return qkv

    @staticmethod
    def backward(ctx, d):
        layout, nheads, where = ctx.cfg
        return _turned_back(ctx, d.reshape(layout), nheads, where, -1.0).reshape(d.shape), None


def _check_heads(qkv, nheads):
    if qkv.dim() != 3 or not qkv.is_floating_point():
        raise ValueError(f"heads come as a floating-point tensor [tokens, heads, head_dim], not {tuple(qkv.shape)} "
                         f"{qkv.dtype}")
    if not 0 <= nheads <= qkv.shape[1]:
        raise ValueError(f"{nheads} heads are asked for, there are {qkv.shape[1]}")


def _overlaps(t):
    """Whether elements of ``t [tokens, heads, head_dim]`` may share memory (as those of an expanded tensor do)."""
    if t.is_contiguous():
        return False
    need = 1
    for stride, n in sorted(zip(t.stride(), t.shape)):
        if n > 1:
            if stride < need:
                return True
            need = stride * (n - 1) + need
    return False


def rope(qkv: torch.Tensor, seq: int, nheads: int, *, rotary: Rotary, offset: int = 0, ranges=None,
         positions=None) -> torch.Tensor:
    """``qkv [tokens, heads, head_dim]`` with its first ``nheads`` heads turned by their positions, the others copied; ``qkv``
    itself stays as it is (:func:`distdl_b200.ops.rope_` turns it in place).

    A token's position is ``offset`` plus its index modulo ``seq``, or comes from ``ranges = ((start, length), ...)``
    adding up to ``seq``, or from ``positions`` (int64 or int32, on the device): one per token, or one per place in a
    sequence of ``seq``.  bf16, fp16 and fp32 heads of up to 512 components run on the kernel, at any strides with unit
    stride inside a head; the angles are formed in 64 bits, so that positions may be as far as 2^31.  Differentiable any
    number of times."""
    _check_heads(qkv, nheads)
    if rotary is None:
        raise ValueError("rope needs a Rotary")
    where = _where(qkv, rotary, seq, offset, ranges, positions)
    rotary._plan(qkv.shape[2])
    if not _native_ok(qkv, where[1]):
        return _plain_rope(qkv, nheads, where)
    if qkv.requires_grad and torch.is_grad_enabled():
        return _RopeFn.apply(qkv, (nheads, where, 1.0))
    return _rotated_copy(qkv, nheads, where, 1.0)


def rope_in_place(qkv, seq, nheads, rotary, offset=0, ranges=None, positions=None, layout=None):
    """:func:`distdl_b200.ops.rope_` with a :class:`Rotary`."""
    if layout is None:
        shape, read = tuple(qkv.shape), qkv
    else:
        shape = tuple(int(v) for v in layout)
        if qkv.numel() != math.prod(shape):
            raise ValueError(f"a tensor {tuple(qkv.shape)} cannot be read as {shape}")
        try:
            read = qkv.detach().view(shape)
        except RuntimeError:                # its strides do not allow it
            read = None
    held = read is not None                 # in memory as it is read
    if not held:
        read = qkv.detach().reshape(shape)
    _check_heads(read, nheads)
    where = _where(read, rotary, seq, offset, ranges, positions)
    rotary._plan(shape[2])
    native = _native_ok(read, where[1])
    if not held or _overlaps(read) or (native and read.stride(2) != 1 and shape[2] > 1):
        raise ValueError("a tensor that is turned in place must have its heads in memory of their own (for the kernels, their "
                         "components next to one another): use ops.rope")
    if qkv.requires_grad and torch.is_grad_enabled() and qkv.is_leaf:
        raise RuntimeError("a leaf that requires a gradient cannot be turned in place: use ops.rope, or torch.no_grad()")
    if not native:
        return qkv.copy_(_plain_rope(qkv.reshape(shape), nheads, where).reshape(qkv.shape))
    if qkv.requires_grad and torch.is_grad_enabled():
        return _RopeInPlaceFn.apply(qkv, (shape, nheads, where))
    _call(_ROTATE, read, read, nheads, 0, where)
    torch.autograd.graph.increment_version(qkv)               # (passes over tensors of inference mode)
    return qkv


# ------------------------------------------------------------------------------- norm of the heads and rotation
def _weight_ok(w, qkv):
    return w is None or (w.dtype in (qkv.dtype, torch.float32) and w.device == qkv.device)


def _plain_qk_norm_rope(qkv, hq, hkv, wq, wk, eps, where):
    nh = hq + hkv
    x = _wide(qkv[:, :nh])
    u = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    parts = [u[:, :hq] if wq is None else u[:, :hq] * wq.to(x.dtype), u[:, hq:] if wk is None else u[:, hq:] * wk.to(x.dtype)]
    y = torch.cat(parts, dim=1)
    rotary = where[0]
    if rotary is not None:
        cos, sin = _angles(qkv, where)
        y = _rotated(y, cos, sin, rotary.rotated(qkv.shape[2]), rotary.interleaved)
    return torch.cat([y.to(qkv.dtype), qkv[:, nh:]], dim=1)


def _normed_copy(qkv, hq, hkv, wq, wk, eps, where):
    src = _unit(qkv)
    out = torch.empty_like(src, memory_format=torch.contiguous_format)
    _call(_FORWARD, src, out, hq, hkv, where, 1.0, wq, wk, eps)
    return out


@functools.lru_cache(maxsize=64)
def _parts(device: int) -> int:
    """CTAs of the backward kernel at most, each with a row of sums."""
    with torch.cuda.device(device):
        return _native.lib().dd_heads_parts()


def _norm_backward(x, dy, wq, wk, hq, hkv, eps, where, want, main=(None, None)):
    """(dx, dwq, dwk) of :func:`qk_norm_rope`; ``want``: which weights' gradients; ``main``: fp32 accumulators that they are
    added to instead (both that are wanted, or neither)."""
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    accumulate = main[0] is not None or main[1] is not None
    dwq, dwk, partial = main[0], main[1], None
    if want[0] or want[1]:
        partial = torch.empty(_parts(x.get_device()) * 2 * x.shape[2], dtype=torch.float32, device=x.device)
        if not accumulate:
            dwq = torch.empty_like(wq) if want[0] else None
            dwk = torch.empty_like(wk) if want[1] else None
    _call(_BACKWARD, x, dx, hq, hkv, where, 1.0, wq, wk, eps, dy, dwq, dwk, partial, accumulate)
    return (dx, None, None) if accumulate else (dx, dwq, dwk)


class _QKNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, wq, wk, cfg):
        hq, hkv, eps, where = cfg
        ctx.save_for_backward(qkv, wq, wk, where[1])
        ctx.refs = (wq, wk)
        ctx.cfg = cfg
        return _normed_copy(qkv, hq, hkv, wq, wk, eps, where)

    @staticmethod
    def backward(ctx, dy):
        qkv, wq, wk, positions = ctx.saved_tensors
        hq, hkv, eps, where = ctx.cfg
        where = (where[0], positions, *where[2:])
        need = ctx.needs_input_grad
        if torch.is_grad_enabled() or not ordinary_gradient(dy):
            # differentiated itself, or under a function transform: elementary operations
            leaves = [t for t, n in zip((qkv, wq, wk), need) if n]
            with torch.enable_grad():
                out = _plain_qk_norm_rope(qkv, hq, hkv, wq, wk, eps, where)
                got = iter(torch.autograd.grad(out, leaves, dy, create_graph=True))
            return (*(next(got) if n else None for n in need[:3]), None)
        want = need[1:3]
        main = (None, None)
        if hasattr(ctx.refs[0], "main_grad") or hasattr(ctx.refs[1], "main_grad"):
            # gathered weights collect their gradient in fp32 beside them
            main = [main_grad_now(getattr(r, "main_grad", None), getattr(r, "main_grad_owner", None), ctx, k) if n else None
                    for k, r, n in ((1, ctx.refs[0], want[0]), (2, ctx.refs[1], want[1]))]
            if any(m is None for m, n in zip(main, want) if n) or main[0] is main[1]:
                main = (None, None)         # (one weight for both kinds: autograd adds)
        return (*_norm_backward(_unit(qkv), _unit(dy), wq, wk, hq, hkv, eps, where, want, main), None)


def _norm_args(qkv, hq, hkv, wq, wk, rotary, seq, offset, ranges, positions):
    """(where, whether the kernels take it, wq, wk): the weights as rows."""
    _check_heads(qkv, hq + hkv)
    if hq < 0 or hkv < 0:
        raise ValueError(f"numbers of heads are not negative: {hq}, {hkv}")
    for w in (wq, wk):
        if w is not None and (w.numel() != qkv.shape[2] or not w.is_floating_point()):
            raise ValueError(f"a weight of the norm has one value per component ({qkv.shape[2]}), not {tuple(w.shape)}")
    where = _where(qkv, rotary, seq, offset, ranges, positions)
    if rotary is not None:
        rotary._plan(qkv.shape[2])
    native = (_native_ok(qkv, where[1], wq, wk) and _weight_ok(wq, qkv) and _weight_ok(wk, qkv)
              and (wq is None or wk is None or wq.dtype == wk.dtype))
    # (a weight that is a row already stays the tensor that it is: its accumulator is an attribute of it)
    if wq is not None and (wq.dim() != 1 or not wq.is_contiguous()):
        wq = wq.reshape(-1).contiguous()
    if wk is not None and (wk.dim() != 1 or not wk.is_contiguous()):
        wk = wk.reshape(-1).contiguous()
    return where, native, wq, wk


def qk_norm_rope(qkv: torch.Tensor, seq: int, hq: int, hkv: int, q_weight=None, k_weight=None, *, rotary: Rotary = None,
                 offset: int = 0, ranges=None, positions=None, eps: float = 1e-6) -> torch.Tensor:
    """The RMS norm of every query and key head, and the rotation by their positions in the same pass: the first ``hq`` heads
    of ``qkv [tokens, heads, head_dim]`` become ``R(u * q_weight)``, ``u = x / sqrt(mean x^2 + eps)`` over a head, the next
    ``hkv`` the same with ``k_weight``; the heads behind (the values) are copied.  Weights ``[head_dim]`` of ``qkv``'s type or
    in fp32, or None; ``rotary`` None: the norm alone.  Positions as for :func:`rope`.

    The result is a new tensor and the backward pass reads ``qkv`` again, so that it stays as it is;
    :func:`qk_norm_rope_` works in place where no gradient is wanted."""
    where, native, wq, wk = _norm_args(qkv, hq, hkv, q_weight, k_weight, rotary, seq, offset, ranges, positions)
    if not native:
        return _plain_qk_norm_rope(qkv, hq, hkv, wq, wk, eps, where)
    if torch.is_grad_enabled() and (qkv.requires_grad or (wq is not None and wq.requires_grad)
                                    or (wk is not None and wk.requires_grad)):
        return _QKNormRopeFn.apply(qkv, wq, wk, (hq, hkv, float(eps), where))
    return _normed_copy(qkv, hq, hkv, wq, wk, float(eps), where)


def qk_norm_rope_(qkv: torch.Tensor, seq: int, hq: int, hkv: int, q_weight=None, k_weight=None, *, rotary: Rotary = None,
                  offset: int = 0, ranges=None, positions=None, eps: float = 1e-6) -> torch.Tensor:
    """:func:`qk_norm_rope` in place, for inference: refused where a gradient would be wanted."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (qkv, q_weight, k_weight)):
        raise RuntimeError("qk_norm_rope_ overwrites what its gradient would need: use qk_norm_rope, or torch.no_grad()")
    where, native, wq, wk = _norm_args(qkv, hq, hkv, q_weight, k_weight, rotary, seq, offset, ranges, positions)
    if _overlaps(qkv):
        raise ValueError("a tensor that is changed in place must not overlap itself: use ops.qk_norm_rope")
    if native and (qkv.stride(2) == 1 or qkv.shape[2] == 1):
        _call(_FORWARD, qkv, qkv, hq, hkv, where, 1.0, wq, wk, float(eps))
        torch.autograd.graph.increment_version(qkv)
        return qkv
    with torch.no_grad():
        qkv.copy_(_plain_qk_norm_rope(qkv, hq, hkv, wq, wk, eps, where))
    return qkv
