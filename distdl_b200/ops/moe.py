"""Mixture-of-experts token routing ops (slot assignment, permuted scatter,
weighted gather) with autograd; CUDA kernels in ``csrc/moe.cu``.  New relative to
the reference (its expert layers expect already-routed ``[expert, capacity,
...]`` tensors, ``src/distdl/nn/linear_ag_expert.py:393-422``)."""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from .. import _native
from ._util import call_on, ordinary, ordinary_gradient, ptr, stream_ptr, use_native

_v, _i, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
_native.declare("dd_moe_assign", [_v, _i, _i, _i, _v, _v, _v])
_native.declare("dd_moe_chunks", [_i])


def _counters(items: int, E: int, device):
    """Scratch of the slot assignment: [0, E) receives the pairs per expert, the rest holds the
    per-chunk histograms."""
    chunks = _native.lib().dd_moe_chunks(int(items))
    return torch.empty((chunks + 1) * E, dtype=torch.int32, device=device)
_native.declare("dd_moe_scatter_rows", [_v, _v, _v, _v, _v, _i, _i, _i, _i, _v])
_native.declare("dd_moe_gather_rows", [_v, _v, _v, _v, _v, _i, _i, _i, _i, _v])
_native.declare("dd_moe_pair_dot", [_v, _v, _v, _v, _v, _i, _i, _i, _i, _v])


_native.declare("dd_moe_router_fwd", [_v, _i, _i, _i, _i, _i, _v, _v, _v, _v, _v, _v])
_native.declare("dd_moe_router_bwd", [_v, _i, _i, _i, _i, _v, _v, _v, _v, _v, _v])


class _RouterFn(torch.autograd.Function):
    """Softmax over the experts, top-k, renormalised weights and the column sums of the probabilities
    in one kernel, the slots (arrival order = pair index, so overflow drops the same pairs in every
    run) in a second one; one more kernel for the backward pass."""

    @staticmethod
    def forward(ctx, logits, E, k, capacity):
        T, ld = logits.shape
        dev = logits.device
        ids = torch.empty(T * k, dtype=torch.int32, device=dev)
        w = torch.empty(T, k, dtype=torch.float32, device=dev)
        slot = torch.empty(T * k, dtype=torch.int32, device=dev)
        scratch = _counters(T, E, dev)
        counts = scratch[:E]
        prob_sum = torch.zeros(E, dtype=torch.float32, device=dev)
        _native.call("dd_moe_router_fwd", logits.data_ptr(), ld, T, E, k, capacity, ids.data_ptr(), w.data_ptr(),
                     slot.data_ptr(), scratch.data_ptr(), prob_sum.data_ptr(), stream_ptr())
        ctx.save_for_backward(logits, ids, w)
        ctx.cfg = (E, k)
        ctx.mark_non_differentiable(ids, slot, counts)
        ctx.set_materialize_grads(False)
        return w, prob_sum, ids, slot, counts

    @staticmethod
    def backward(ctx, dw, dprob, _dids, _dslot, _dcounts):
        logits, ids, w = ctx.saved_tensors
        E, k = ctx.cfg
        T, ld = logits.shape
        dlogits = torch.empty_like(logits)
        dwc = None if dw is None else dw.float().contiguous()
        dpc = None if dprob is None else dprob.float().contiguous()
        _native.call("dd_moe_router_bwd", logits.data_ptr(), ld, T, E, k, ids.data_ptr(), w.data_ptr(), ptr(dwc),
                     ptr(dpc), dlogits.data_ptr(), stream_ptr())
        return dlogits, None, None, None


_native.declare("dd_route_words", [_i, _i])
_native.declare("dd_route_fwd", [ctypes.c_char_p, _i, _v])
_ROUTE_CALL = struct.Struct("=8Qq11if")           # struct RouteCall of csrc/router.cu
_native.declare("dd_route_bwd", [_v, _i, _i, _i, _i, _i, _i, _i, _f, _v, _v, _v, _v, _v, _v])
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_MOST_EXPERTS, _MOST_CHOICES, _MOST_GROUPS = 512, 32, 32


def _route_forward(logits, E, k, capacity, how):
    score, bias, groups, top_groups, group_score, renormalize, scale = how
    T, ld = logits.shape
    dev = logits.device
    # (pieces of their own: whoever changes one of them in place must not seem to change what the backward pass has kept)
    ids = torch.empty(T * k, dtype=torch.int32, device=dev)
    slot = torch.empty_like(ids)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    w = torch.empty(T, k, dtype=torch.float32, device=dev)
    prob_sum = torch.empty(E, dtype=torch.float32, device=dev)
    words = _native.lib().dd_route_words(T, E)
    scratch = torch.empty(words, dtype=torch.int32, device=dev)
    call_on(logits, "dd_route_fwd", _ROUTE_CALL.pack(
        logits.data_ptr(), ptr(bias), ids.data_ptr(), w.data_ptr(), slot.data_ptr(), counts.data_ptr(), prob_sum.data_ptr(),
        scratch.data_ptr(), words, ld, _DTYPE[logits.dtype], T, E, k, capacity, groups, top_groups, group_score == "top2",
        score == "sigmoid", renormalize, scale), _ROUTE_CALL.size)
    return w, prob_sum, ids, slot, counts


class _RouteFn(torch.autograd.Function):
    """:func:`route` in its general form: two kernels, and one for the backward pass."""

    @staticmethod
    def forward(ctx, logits, E, k, capacity, how):
        w, prob_sum, ids, slot, counts = _route_forward(logits, E, k, capacity, how)
        ctx.save_for_backward(logits, ids, w)
        ctx.cfg = (E, k, how)
        ctx.mark_non_differentiable(ids, slot, counts)
        ctx.set_materialize_grads(False)
        return w, prob_sum, ids, slot, counts

    @staticmethod
    def backward(ctx, dw, dprob, _dids, _dslot, _dcounts):
        logits, ids, w = ctx.saved_tensors
        E, k, how = ctx.cfg
        if dw is None and dprob is None:
            return None, None, None, None, None
        if torch.is_grad_enabled() or not all([g is None or ordinary_gradient(g) for g in (dw, dprob)]):
            # differentiated itself, or under a function transform: elementary operations, with the experts as they are
            with torch.enable_grad():
                outs = _route_weights(logits, E, ids.reshape(-1, k), how)
                outs, grads = zip(*[(o, g) for o, g in zip(outs, (dw, dprob)) if g is not None])
                (d,) = torch.autograd.grad(outs, logits, grads, create_graph=True)
            return d, None, None, None, None
        if dw is not None and (dw.dtype != torch.float32 or not dw.is_contiguous()):
            dw = dw.float().contiguous()
        if dprob is not None and (dprob.dtype != torch.float32 or not dprob.is_contiguous()):
            dprob = dprob.float().contiguous()
        dlogits = torch.empty_like(logits)
        call_on(logits, "dd_route_bwd", logits.data_ptr(), logits.shape[1], _DTYPE[logits.dtype], logits.shape[0], E, k,
                int(how[0] == "sigmoid"), int(how[5]), how[6], ids.data_ptr(), w.data_ptr(), ptr(dw), ptr(dprob),
                dlogits.data_ptr())
        return dlogits, None, None, None, None


def _scores(logits, E, score):
    """(scores, what they are over their sum) in the type of ``logits``; zeros in rows without an expert."""
    l = logits[:, :E]
    none = (l == -math.inf).all(-1, keepdim=True)
    l = torch.where(none, torch.zeros_like(l), l)
    if score == "softmax":
        s = torch.softmax(l, -1)
        p = s
    else:
        s = torch.sigmoid(l)
        p = torch.softmax(torch.nn.functional.logsigmoid(l), -1)         # s / sum s, however small they are
    return s.masked_fill(none, 0.0), p.masked_fill(none, 0.0)


def _route_weights(logits, E, ids, how):
    """Weights ``[tokens, k]`` and sums of probabilities for chosen experts ``ids`` (-1: none), fp32."""
    score, _bias, _groups, _top, _by, renormalize, scale = how
    wide = logits.double()
    s, p = _scores(wide, E, score)
    at = ids.long().clamp(min=0)
    here = ids >= 0
    if renormalize:
        l = wide[:, :E].gather(1, at)
        l = (l if score == "softmax" else torch.nn.functional.logsigmoid(l)).masked_fill(~here, -math.inf)
        some = here.any(-1, keepdim=True)
        w = torch.softmax(torch.where(some, l, torch.zeros_like(l)), -1)
    else:
        w = s.gather(1, at)
    w = (scale * w).masked_fill(~here, 0.0)
    bad = _bad(wide[:, :E], score)
    w = torch.where(bad & here, torch.full_like(w, math.nan), w)
    p = torch.where(bad, torch.full_like(p, math.nan), p)
    return w.float(), p.sum(0).float()


def _bad(l, score):
    return (torch.isnan(l) | ((l == math.inf) if score == "softmax" else torch.zeros_like(l, dtype=torch.bool))).any(
        -1, keepdim=True)


def _choose(logits, E, k, how):
    """The experts ``[tokens, k]`` of :func:`route` (-1: none left), in 64 bits."""
    score, bias, groups, top_groups, group_score, _renormalize, _scale = how
    l = logits[:, :E].detach().double()
    best = torch.isnan(l) if score == "sigmoid" else torch.isnan(l) | (l == math.inf)     # no numbers: the best
    c = _scores(l.masked_fill(best, -math.inf), E, score)[0]
    if bias is not None:
        c = c + bias.double()
    elif group_score == "max" or top_groups == groups or groups == E:
        c = l                                               # the same order, also where scores are no longer told apart
    c = c.clamp(max=torch.finfo(torch.float64).max)         # (+inf of a sigmoid or a bias: below what is no number)
    c = c.masked_fill((l == -math.inf) | torch.isnan(c), -math.inf).masked_fill(best, math.inf)
    if top_groups < groups:
        by = c.reshape(len(c), groups, E // groups).sort(dim=-1, descending=True).values
        value = by[..., 0]
        if group_score == "top2" and E > groups:
            value = torch.where((by[..., 1] > -math.inf) & (value < math.inf),
                                (value + by[..., 1]).clamp(max=torch.finfo(torch.float64).max), value)
        kept = value.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
        live = torch.zeros_like(value, dtype=torch.bool).scatter(1, kept, True)
        c = c.masked_fill(~live.repeat_interleave(E // groups, dim=1), -math.inf)
    top = c.sort(dim=-1, descending=True, stable=True)
    ids = top.indices[:, :k].masked_fill(top.values[:, :k] == -math.inf, -1)
    return ids.to(torch.int32).contiguous()


def route(logits: torch.Tensor, num_experts: int, k: int, capacity: int, *, score: str = "softmax", bias=None,
          groups: int = 1, top_groups: int = None, group_score: str = "max", renormalize: bool = True, scale: float = 1.0):
    """Top-k routing of ``logits [tokens, >= num_experts]`` (extra columns are padding).

    Returns ``(weights [tokens, k] fp32, prob_sum [E] fp32, ids [tokens * k] int32, slot
    [tokens * k] int32, counts [E] int32)``: the weights of the chosen experts, the sum over tokens
    of the probabilities (for a load-balancing loss), the chosen experts in falling order, each pair's slot in its
    expert's capacity buffer (-1 = dropped) and the number of pairs routed to every expert.  ``weights`` and
    ``prob_sum`` carry gradients back to ``logits``.

    * ``score``: ``"softmax"`` of the logits, or ``"sigmoid"``; the probabilities are the scores over their sum.
    * ``bias`` (fp32 ``[num_experts]``): added to the scores for the choice alone (balance without a loss:
      :func:`balance_bias_`); it carries no gradient.
    * ``groups``: the experts lie in as many groups of equal size; only those of the ``top_groups`` best are chosen from.  A
      group counts what its best expert does (``group_score="max"``) or its two best together (``"top2"``).
    * ``renormalize``: the weights of a token add up to ``scale``; else they are ``scale`` times the scores.

    Equal scores go to the lowest expert, and scores are told apart as exact arithmetic would.  An expert with a logit or a
    bias of -inf is never chosen; where fewer than ``k`` are left the places have id -1, slot -1 and weight 0, and a row of -inf (a
    padding token) routes nowhere and adds nothing to ``prob_sum``.  A NaN makes the token's weights NaN.  bf16, fp16 and
    fp32 logits of up to 512 experts, with 32 choices and 32 groups at most, run on the kernels."""
    E = num_experts
    if score == "softmax" and bias is None and groups == 1 and renormalize and scale == 1.0 and use_native(logits) \
            and logits.dtype == torch.bfloat16 and E <= 64 and k <= 8 and logits.is_contiguous() and logits.numel():
        return _RouterFn.apply(logits, E, k, capacity)        # (a thread per token, csrc/moe.cu)
    how = _route_check(logits, E, k, score, bias, groups, top_groups, group_score, renormalize, scale)
    if use_native(logits) and logits.dtype in _DTYPE and E <= _MOST_EXPERTS and k <= _MOST_CHOICES \
            and groups <= _MOST_GROUPS and logits.numel() and logits.shape[0] * k < 2 ** 31 and ordinary(logits, how[1]):
        logits = logits if logits.is_contiguous() else logits.contiguous()
        capacity = min(int(capacity), 2 ** 31 - 1)
        if torch.is_grad_enabled() and logits.requires_grad:
            return _RouteFn.apply(logits, E, k, capacity, how)
        return _route_forward(logits, E, k, capacity, how)
    ids = _choose(logits, E, k, how)
    w, prob_sum = _route_weights(logits, E, ids, how)
    slot, counts = _slots_in_order(ids.reshape(-1), E, capacity)
    return w, prob_sum, ids.reshape(-1), slot, counts


def _route_check(logits, E, k, score, bias, groups, top_groups, group_score, renormalize, scale):
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"logits come as a floating-point matrix [tokens, experts], not {tuple(logits.shape)} {logits.dtype}")
    if not 1 <= E <= logits.shape[1]:
        raise ValueError(f"{E} experts, {logits.shape[1]} logits per token")
    if not 1 <= k <= E:
        raise ValueError(f"between 1 and {E} experts per token, not {k}")
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"score must be 'softmax' or 'sigmoid', not {score!r}")
    if group_score not in ("max", "top2"):
        raise ValueError(f"group_score must be 'max' or 'top2', not {group_score!r}")
    if groups < 1 or E % groups:
        raise ValueError(f"{E} experts do not lie in {groups} equal groups")
    top_groups = groups if top_groups is None else top_groups
    if not 1 <= top_groups <= groups:
        raise ValueError(f"between 1 and {groups} groups are chosen from, not {top_groups}")
    if k > top_groups * (E // groups):
        raise ValueError(f"{top_groups} groups of {E // groups} experts have no {k} to choose")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, not {scale}")
    if bias is not None:
        if bias.numel() != E or bias.device != logits.device or not bias.is_floating_point():
            raise ValueError(f"the bias has one value per expert ({E}), on the device of the logits")
        bias = bias.detach().reshape(-1)
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.float().contiguous()
    return score, bias, int(groups), int(top_groups), group_score, bool(renormalize), float(scale)


@torch.no_grad()
def balance_bias_(bias: torch.Tensor, counts: torch.Tensor, rate: float) -> torch.Tensor:
    """One step towards equal load without a loss: the bias of every expert with fewer pairs than the mean of ``counts``
    (pairs per expert, summed over all workers) grows by ``rate``, that of one with more shrinks by it."""
    if bias.numel() != counts.numel():
        raise ValueError(f"{bias.numel()} values of the bias, {counts.numel()} counts")
    c = counts.reshape(bias.shape).double()
    return bias.add_((torch.sign(c.mean() - c) * rate).to(bias.dtype))


def _slots_in_order(flat, E, capacity):
    """(slots, counts) for ids in pair order, -1 among them, by a stable sort (any number of experts, any device)."""
    here = flat >= 0
    key = torch.where(here, flat, torch.full_like(flat, E)).long()
    counts = torch.zeros(E + 1, dtype=torch.int64, device=flat.device).scatter_add(0, key, torch.ones_like(key))
    order = key.sort(stable=True).indices
    rank = torch.empty_like(key)
    rank[order] = torch.arange(key.numel(), device=key.device) - (counts.cumsum(0) - counts)[key[order]]
    slot = torch.where(here & (rank < capacity), rank, torch.full_like(rank, -1))
    return slot.to(torch.int32), counts[:E].to(torch.int32)


def assign_slots(ids: torch.Tensor, num_experts: int, capacity: int):
    """ids [pairs] int32 -> (slot [pairs] int32 with -1 for dropped pairs, counts [E] int32)."""
    flat = ids.reshape(-1).to(torch.int32).contiguous()
    if use_native(flat):
        scratch = _counters(flat.numel(), num_experts, flat.device)
        slot = torch.empty_like(flat)
        _native.call("dd_moe_assign", flat.data_ptr(), flat.numel(), num_experts, capacity, scratch.data_ptr(),
                     slot.data_ptr(), stream_ptr())
        return slot, scratch[:num_experts]
    onehot = torch.nn.functional.one_hot(flat.long(), num_experts)
    pos = (onehot.cumsum(0) - 1)[torch.arange(flat.numel()), flat.long()]
    slot = torch.where(pos < capacity, pos, torch.full_like(pos, -1)).to(torch.int32)
    return slot, onehot.sum(0).to(torch.int32)


def _scatter(src, ids, slot, w, E, C, k):
    d = src.shape[-1]
    dst = torch.zeros(E, C, d, dtype=src.dtype, device=src.device)
    if use_native(src) and src.dtype == torch.bfloat16 and d % 8 == 0:
        _native.call("dd_moe_scatter_rows", src.data_ptr(), ids.data_ptr(), slot.data_ptr(), ptr(w), dst.data_ptr(),
                     ids.numel(), k, C, d, stream_ptr())
        return dst
    keep = slot >= 0
    rows = src[torch.arange(ids.numel(), device=src.device) // k]
    if w is not None:
        rows = rows * w.reshape(-1, 1).to(rows.dtype)
    dst[ids[keep].long(), slot[keep].long()] = rows[keep]
    return dst


def _gather(src, ids, slot, w, tokens, k):
    E, C, d = src.shape
    if use_native(src) and src.dtype == torch.bfloat16 and d % 8 == 0:
        dst = torch.empty(tokens, d, dtype=src.dtype, device=src.device)
        _native.call("dd_moe_gather_rows", src.data_ptr(), ids.data_ptr(), slot.data_ptr(), ptr(w), dst.data_ptr(),
                     tokens, k, C, d, stream_ptr())
        return dst
    keep = (slot >= 0).reshape(tokens, k, 1)
    rows = src[ids.long().clamp(min=0), slot.long().clamp(min=0)].reshape(tokens, k, d).float()
    if w is not None:
        rows = rows * w.reshape(tokens, k, 1)
    return rows.masked_fill(~keep, 0.0).sum(1).to(src.dtype)


def _pair_dot(a, b, ids, slot, k):
    E, C, d = b.shape
    n = ids.numel()
    if use_native(a) and a.dtype == torch.bfloat16 and d % 8 == 0:
        out = torch.empty(n, dtype=torch.float32, device=a.device)
        _native.call("dd_moe_pair_dot", a.data_ptr(), b.data_ptr(), ids.data_ptr(), slot.data_ptr(), out.data_ptr(),
                     n, k, C, d, stream_ptr())
        return out
    rows = b[ids.long().clamp(min=0), slot.long().clamp(min=0)].float()
    av = a[torch.arange(n, device=a.device) // k].float()
    return (rows * av).sum(-1).masked_fill(slot < 0, 0.0)


class DispatchFn(torch.autograd.Function):
    """x [T, d] -> per-expert capacity buffers [E, C, d] (unused slots zero)."""

    @staticmethod
    def forward(ctx, x, ids, slot, E, C, k):
        ctx.save_for_backward(ids, slot)
        ctx.cfg = (x.shape[0], k)
        return _scatter(x.contiguous(), ids, slot, None, E, C, k)

    @staticmethod
    def backward(ctx, g):
        ids, slot = ctx.saved_tensors
        T, k = ctx.cfg
        return _gather(g.contiguous(), ids, slot, None, T, k), None, None, None, None, None


class CombineFn(torch.autograd.Function):
    """y[t] = sum_c w[t, c] * buf[ids[t, c], slot[t, c]]."""

    @staticmethod
    def forward(ctx, buf, w, ids, slot, T, k):
        bufc, wc = buf.contiguous(), w.reshape(-1).float().contiguous()
        ctx.save_for_backward(bufc, wc, ids, slot)
        ctx.cfg = (T, k, w.shape, w.dtype)
        return _gather(bufc, ids, slot, wc, T, k)

    @staticmethod
    def backward(ctx, dy):
        buf, w, ids, slot = ctx.saved_tensors
        T, k, wshape, wdtype = ctx.cfg
        E, C, d = buf.shape
        dyc = dy.contiguous()
        dbuf = _scatter(dyc, ids, slot, w, E, C, k)
        dw = _pair_dot(dyc, buf, ids, slot, k).reshape(wshape).to(wdtype)
        return dbuf, dw, None, None, None, None


def dispatch(x, ids, slot, num_experts, capacity, k):
    return DispatchFn.apply(x, ids, slot, num_experts, capacity, k)


def combine(buf, weights, ids, slot, tokens, k):
    return CombineFn.apply(buf, weights, ids, slot, tokens, k)
