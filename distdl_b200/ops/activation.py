"""SwiGLU, GELU and rotary-embedding kernels (new relative to the reference,
which has no activation or attention code; they are required by the
GPT-2 / Llama / Mixtral model shapes)."""
from __future__ import annotations


import torch

from .. import _native
from ._util import _modes, stream_ptr, use_native


class _SwiGLUFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        F = gu.shape[-1] // 2
        g2 = gu.reshape(-1, 2 * F)
        if not g2.is_contiguous():
            g2 = g2.contiguous()
        out = torch.empty(g2.shape[0], F, dtype=gu.dtype, device=gu.device)
        _native.call("dd_swiglu_fwd", g2.data_ptr(), out.data_ptr(), g2.shape[0], F, stream_ptr())
        ctx.save_for_backward(g2)
        ctx.shape = gu.shape
        return out.view(*gu.shape[:-1], F)

    @staticmethod
    def backward(ctx, dout):
        (g2,) = ctx.saved_tensors
        F = g2.shape[-1] // 2
        d2 = dout.reshape(-1, F)
        if not d2.is_contiguous():
            d2 = d2.contiguous()
        dgu = torch.empty_like(g2)
        _native.call("dd_swiglu_bwd", d2.data_ptr(), g2.data_ptr(), dgu.data_ptr(), g2.shape[0], F, stream_ptr())
        return dgu.view(ctx.shape)


def swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for a tensor whose last dimension is ``[gate | up]``."""
    F = gate_up.shape[-1] // 2
    if use_native(gate_up) and gate_up.dtype == torch.bfloat16 and F % 8 == 0:
        return _SwiGLUFn.apply(gate_up)
    g, u = gate_up[..., :F], gate_up[..., F:]
    return torch.nn.functional.silu(g) * u


class _GeluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        xc = x.contiguous()
        y = torch.empty_like(xc)
        _native.call("dd_gelu_fwd", xc.data_ptr(), y.data_ptr(), xc.numel(), stream_ptr())
        ctx.save_for_backward(xc)
        return y

    @staticmethod
    def backward(ctx, dy):
        (xc,) = ctx.saved_tensors
        dyc = dy.contiguous()
        dx = torch.empty_like(xc)
        _native.call("dd_gelu_bwd", dyc.data_ptr(), xc.data_ptr(), dx.data_ptr(), xc.numel(), stream_ptr())
        return dx


def gelu(x: torch.Tensor) -> torch.Tensor:
    """tanh-approximated GELU (the GPT-2 activation)."""
    if use_native(x) and x.dtype == torch.bfloat16 and x.numel() % 8 == 0:
        return _GeluFn.apply(x)
    return torch.nn.functional.gelu(x, approximate="tanh")


_rope_cache = {}


def _host_table(seq, head_dim, theta):
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64, device="cpu") / head_dim))
    ang = torch.outer(torch.arange(seq, dtype=torch.float64, device="cpu"), inv)
    return torch.stack([ang.cos(), ang.sin()], dim=-1).float()


def _kept_table(key, make, device):
    """The table of ``key``, copied from the host when it is first asked for: the copy has ended when this returns, so that
    every stream may read it.  Fake tensors get a fake one, which is not kept."""
    t = _rope_cache.get(key)
    if t is None or (_modes() and torch._guards.detect_fake_mode() is not None):
        with torch.inference_mode(False):
            t = make().to(device).contiguous()
        if type(t) is torch.Tensor:
            _rope_cache[key] = t
    return t


def rope_table(seq: int, head_dim: int, theta: float, device) -> torch.Tensor:
    """[seq, head_dim/2, 2] fp32 table of (cos, sin)."""
    return _kept_table((seq, head_dim, theta, str(device)), lambda: _host_table(seq, head_dim, theta), device)


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, table, seq, nheads, layout):
        # qkv: contiguous, read as [tokens, heads_total, hd] = layout; rotates heads [0, nheads) in place.
        ctx.mark_dirty(qkv)
        tokens, ht, hd = layout
        _native.call("dd_rope", qkv.data_ptr(), table.data_ptr(), tokens, seq, ht, nheads, hd, 1.0, stream_ptr())
        ctx.table, ctx.seq, ctx.nheads, ctx.layout = table, seq, nheads, layout
        return qkv

    @staticmethod
    def backward(ctx, d):
        # the incoming gradient belongs to this node alone (the rotated tensor has one producer and
        # its consumers' gradients were summed into a fresh tensor): rotate it back in place
        d = d.contiguous()
        tokens, ht, hd = ctx.layout
        _native.call("dd_rope", d.data_ptr(), ctx.table.data_ptr(), tokens, ctx.seq, ht, ctx.nheads, hd, -1.0,
                     stream_ptr())
        return d, None, None, None, None


def rope_table_ranges(ranges, head_dim: int, theta: float, device) -> torch.Tensor:
    """Table for a local sequence made of several position ranges ``((start, length), ...)``."""
    key, last = (tuple(ranges), head_dim, theta, str(device)), max(a + n for a, n in ranges)
    if key not in _rope_cache and torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing():
        full = rope_table(last, head_dim, theta, device)      # (a piece of the graph's own)
        return torch.cat([full[a:a + n] for a, n in ranges])

    def make():
        full = _host_table(last, head_dim, theta)
        return torch.cat([full[a:a + n] for a, n in ranges])

    return _kept_table(key, make, device)


def rope_(qkv: torch.Tensor, seq: int, nheads: int, theta: float = 500000.0, offset: int = 0,
          ranges=None, layout=None, *, rotary=None, positions=None) -> torch.Tensor:
    """Applies rotary position embedding (rotate-half convention) to the first
    ``nheads`` heads of ``qkv`` [tokens, heads_total, head_dim]; position of a
    token is ``offset`` plus its index modulo ``seq`` (``offset`` > 0 for a worker that holds a
    later block of a sequence split across workers), or, with ``ranges = ((start, length), ...)``
    adding up to ``seq``, the positions of those ranges one after the other.  In place on CUDA.

    ``layout = (tokens, heads_total, head_dim)``: ``qkv`` is the projection's own output in
    whatever shape it has (say ``[batch, seq, heads_total * head_dim]``) and is only READ in that
    layout.  Prefer this form: rotating a reshaped VIEW in place makes autograd copy the whole
    gradient twice in the backward pass.

    ``rotary`` (an :class:`~distdl_b200.ops.Rotary`, in the place of ``theta``): other pairings, a part of the head, long
    contexts.  ``positions`` (int64 or int32, on the device of ``qkv``): a position per token, or per place in a sequence.
    With either of them ``qkv`` itself is turned and returned, on every device: bf16, fp16 and fp32 heads on CUDA by the
    kernels, at any strides with unit stride inside a head.  It must not be a leaf that requires a gradient;
    :func:`~distdl_b200.ops.rope` leaves its input alone."""
    if rotary is not None or positions is not None:
        from .rotary import Rotary, rope_in_place
        return rope_in_place(qkv, seq, nheads, Rotary(theta=theta) if rotary is None else rotary, offset, ranges, positions,
                             layout)
    if layout is not None:
        if use_native(qkv) and qkv.dtype == torch.bfloat16 and layout[2] % 16 == 0 and qkv.is_contiguous():
            tokens, ht, hd = (int(v) for v in layout)
            if ranges is not None:
                table = rope_table_ranges(tuple((int(a), int(n)) for a, n in ranges), hd, theta, qkv.device)
            else:
                table = rope_table(offset + seq, hd, theta, qkv.device)
                if offset:
                    table = table[offset:]
            return _RopeFn.apply(qkv, table, seq, nheads, (tokens, ht, hd))
        shape = qkv.shape
        return rope_(qkv.reshape(layout), seq, nheads, theta, offset, ranges).reshape(shape)
    tokens, ht, hd = qkv.shape
    if ranges is not None:
        table = rope_table_ranges(tuple((int(a), int(n)) for a, n in ranges), hd, theta, qkv.device)
    else:
        table = rope_table(offset + seq, hd, theta, qkv.device)
        if offset:
            table = table[offset:]                            # rows [offset, offset + seq)
    if use_native(qkv) and qkv.dtype == torch.bfloat16 and hd % 16 == 0 and qkv.is_contiguous():
        return _RopeFn.apply(qkv, table, seq, nheads, (tokens, ht, hd))
    pos = torch.arange(tokens, device=qkv.device) % seq
    cos = table[pos, :, 0].unsqueeze(1)
    sin = table[pos, :, 1].unsqueeze(1)
    x = qkv[:, :nheads].float()
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    rot = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(qkv.dtype)
    return torch.cat([rot, qkv[:, nheads:]], dim=1)
