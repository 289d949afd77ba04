"""Routed experts: top-k routing, grouped products with ragged groups, SwiGLU with an 8-bit checkpoint, combination.

The operators of a mixture-of-experts feed-forward in which a token is computed by its ``top_k`` experts only
(``BatchedExpertMoE(routed=True)`` calls them; ``expert_mlp`` is the whole block):

* ``route_topk(logits, top_k)`` -> ``ExpertRoute``: the chosen experts, their softmax weights, and the rows of the
  (token, choice) pairs sorted by expert;
* ``grouped_linear(x, weight, bias, route=... | offsets=...)``: every row times its group's weight on tcgen05, rows
  gathered from the tokens (``route``) or already in group order (``offsets``);
* ``swiglu(x, checkpoint=None | "e4m3")``: ``up * silu(gate)``; with a checkpoint the backward pass reads an 8-bit
  copy of the input instead of the input;
* ``combine_rows(z, route, weights)``: the experts' rows back to their tokens, weighted.

Layout: logits ``[slots, tokens, experts]`` (or ``[tokens, experts]``: one slot); token ``t = slot * tokens + b``;
the experts of slot ``s`` are groups ``s * experts .. (s + 1) * experts - 1``.  A route is made and used on the
device: nothing is read back, and every call can be captured into a CUDA graph.

An expert whose logit is -inf is never chosen; a token with fewer than ``top_k`` other experts has fewer rows (its
remaining choices are -1 with weight 0), down to none: its output is then zero.  Rows behind the last group are
zeros in every output.  Nothing here uses floating-point atomics: a call gives the same bits every time.

CUDA tensors run the native kernels (``csrc/experts.cu``, ``csrc/grouped_gemm.cu``); CPU tensors run the plain
formulas below, which are the oracle of the numerics tests.  The reference computes every expert for every token
and picks afterwards (src/flare/jax/layers/token_mix.py).
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from .._native import DEFAULT_TIMEOUT_NS, default_status, native, on_cuda

MAX_EXPERTS = 512   # of one slot
MAX_TOP_K = 32
MAX_ROUTE_GROUPS = 65536  # slots * experts of one route
MAX_GROUPS = 2048   # of one grouped product
GROUP = 32          # columns that share one power-of-two scale of the 8-bit checkpoint

_STATUS: dict[int, int] = {}


def _status(x: torch.Tensor) -> int:
    """Address of the status word of x's device (looked up once a device: a serving step pays for every call).  The word
    is not made inside a capture: its zeros would be part of the graph, and nothing would clear it before a replay."""
    at = _STATUS.get(x.get_device())
    if at is None:
        if x.get_device() not in _native._STATUS and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first call on a device cannot be captured into a CUDA graph: make one before the capture")
        at = _STATUS[x.get_device()] = default_status(x.device).ptr
    return at


class ExpertRoute(NamedTuple):
    """Where tokens go.  ``k`` choices a token, ``R = tokens * k`` row places in all.  The five belong together: the
    operators check their types and sizes, not that ``rows``, ``row_of`` and ``offsets`` say the same."""

    experts: torch.Tensor  # int32 [.., tokens, k]: the chosen experts by falling logit, -1 where there is none
    weights: torch.Tensor  # float32 [.., tokens, k]: softmax over the chosen logits, 0 where there is none
    offsets: torch.Tensor  # int32 [groups + 1]: group g owns rows offsets[g] .. offsets[g + 1]
    rows: torch.Tensor     # int32 [R]: the token of each row, -1 behind the last group
    row_of: torch.Tensor   # int32 [.., tokens, k]: the row of each choice, -1 where there is none


# -------------------------------------------------------------------- routing
def route_topk_reference(logits: torch.Tensor, top_k: int) -> ExpertRoute:
    """The routing in plain torch (any device, differentiable in the weights)."""
    lg = logits if logits.dim() == 3 else logits.unsqueeze(0)
    S, B, E = lg.shape
    dev = lg.device
    val = lg if lg.dtype == torch.float64 else lg.float()
    # NaN sorts above everything, as in torch.topk; equal logits keep the order of the experts
    idx = torch.sort(val.detach(), dim=-1, descending=True, stable=True).indices[..., :top_k]
    picked = val.gather(-1, idx)
    live = ~torch.isneginf(picked.detach())
    top = torch.where(live[..., :1], picked[..., :1], torch.zeros_like(picked[..., :1])).detach()
    e = torch.where(live, torch.exp(torch.where(live, picked - top, torch.zeros_like(picked))), torch.zeros_like(picked))
    weights = torch.where(live, e / torch.where(live[..., :1], e.sum(-1, keepdim=True), torch.ones_like(top)), torch.zeros_like(e))
    slot = torch.arange(S, device=dev).view(S, 1, 1)
    group = torch.where(live, idx + slot * E, S * E).reshape(-1)
    order = torch.sort(group, stable=True).indices
    counts = torch.bincount(group, minlength=S * E + 1)[:S * E]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.arange(group.numel(), device=dev)
    rows = torch.where(place < offsets[-1], order // top_k, -1)
    row_of = torch.where(live.reshape(-1), torch.empty_like(place).scatter_(0, order, place), -1)
    shape = (*logits.shape[:-1], top_k)
    i32 = torch.int32
    return ExpertRoute(torch.where(live, idx, -1).to(i32).view(shape), weights.to(torch.float32 if lg.dtype != torch.float64 else lg.dtype).view(shape),
                       offsets.to(i32), rows.to(i32), row_of.to(i32).view(shape))


def route_topk(logits: torch.Tensor, top_k: int) -> ExpertRoute:
    """Route every token to its ``top_k`` experts of largest logit (ties: the lowest expert; NaN above all).

    ``weights`` is the softmax over the chosen logits in float32 and is differentiable; the gradient of a logit
    that was not chosen is zero.
    """
    if logits.is_cuda:
        return ExpertRoute(*native().route_topk(logits, top_k))
    if logits.dim() not in (2, 3):
        raise ValueError(f"logits must be [tokens, experts] or [slots, tokens, experts], got {tuple(logits.shape)}")
    if not 1 <= top_k <= min(logits.shape[-1], MAX_TOP_K):
        raise ValueError(f"top_k must be from 1 to the number of experts ({logits.shape[-1]}) and {MAX_TOP_K}, got {top_k}")
    return route_topk_reference(logits, top_k)


# ------------------------------------------------------------ grouped products
def grouped_linear_reference(x, weight, bias=None, *, offsets, rows=None):
    """A loop over the groups in the operands' own types (any device, differentiable)."""
    w = weight.reshape(-1, *weight.shape[-2:])
    b = bias.reshape(w.shape[0], -1) if bias is not None else None
    off = offsets.tolist()
    n = rows.numel() if rows is not None else x.shape[0]
    parts, at = [], 0

    def zeros(k):
        return x.new_zeros(k, w.shape[2])

    for g in range(w.shape[0]):
        lo, hi = min(max(off[g], at), n), min(max(off[g + 1], at), n)
        if lo > at:
            parts.append(zeros(lo - at))
        if hi > lo:
            xg = x[rows[lo:hi].long()] if rows is not None else x[lo:hi]
            y = xg @ w[g].to(x.dtype)
            parts.append(y if b is None else y + b[g].to(x.dtype))
        at = max(hi, lo)
    parts.append(zeros(n - at))
    return torch.cat(parts)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                   offsets: torch.Tensor | None = None, route: ExpertRoute | None = None) -> torch.Tensor:
    """Every row times its group's weight: ``y[r] = x[r] @ weight[g] + bias[g]`` for the rows of group ``g``.

    Exactly one of ``route`` and ``offsets`` is given.  With ``route`` the rows are gathered, ``x`` is ``[tokens,
    in]`` and row ``r`` is token ``route.rows[r]``; with ``offsets`` (int32 ``[groups + 1]``, on the device) ``x`` is
    ``[R, in]`` in group order.  ``weight`` is ``[.., in, out]`` with ``groups`` matrices in all, ``bias`` ``[.., out]``;
    they may be float32 (the weight is rounded to x's type; gradients come back in the types of the operands).  On CUDA
    ``x`` is bfloat16 or float16, and ``in`` and ``out`` are multiples of 8.  Returns ``[R, out]``; a row of no group is
    zero.  Offsets that fall, or leave ``0 .. R``, are reported by ``default_status(device).check()``; they are clamped to the rows,
    and a group starts at the largest offset up to its own: no row belongs to two groups.

    Sums are in float32 and rounded once.  For the backward pass the gathered rows and the rounded weight are kept; a
    token's input gradient is summed over its rows in float32.
    """
    rows = row_of = None
    if (offsets is None) == (route is None):
        raise ValueError("give exactly one of route and offsets")
    if route is not None:
        offsets, rows, row_of = route.offsets, route.rows, route.row_of
    if x.is_cuda:
        # a parameter bound to a flat fused optimizer (``_flare_grad``: its fp32 view of the gradient buffer) gets its
        # gradient added there by the kernel, as in the layers of ``models.layers``
        return native().grouped_linear(x, weight, bias, offsets, rows, row_of, getattr(weight, "_flare_grad", None),
                                       getattr(bias, "_flare_grad", None), _status(x), DEFAULT_TIMEOUT_NS)
    on_cuda(x, weight, offsets, *(t for t in (bias, rows) if t is not None))  # refuses a mixture of devices
    if x.dim() != 2 or weight.dim() < 3 or weight.shape[-2] != x.shape[1]:
        raise ValueError(f"x must be [rows, in] and weight [.., in, out], got {tuple(x.shape)} and {tuple(weight.shape)}")
    K, N = weight.shape[-2:]
    groups = weight.numel() // max(K * N, 1)
    if route is not None and (row_of.numel() != rows.numel() or row_of.numel() != x.shape[0] * row_of.shape[-1]):
        raise ValueError(f"route of {rows.numel()} rows does not fit {x.shape[0]} tokens")
    if offsets.dtype != torch.int32 or offsets.shape != (groups + 1,):
        raise ValueError(f"offsets must be int32 [{groups + 1}] for {groups} groups, got {offsets.dtype} {tuple(offsets.shape)}")
    if bias is not None and (bias.shape[-1] != N or bias.numel() != groups * N):
        raise ValueError(f"bias must be [.., {N}] for {groups} groups, got {tuple(bias.shape)}")
    return grouped_linear_reference(x, weight, bias, offsets=offsets, rows=rows)


# -------------------------------------------------------------------- SwiGLU
def e4m3_checkpoint_reference(x: torch.Tensor) -> torch.Tensor:
    """The values that the 8-bit checkpoint of ``x [rows, 2h]`` stands for.

    Either half is cut into groups of 32 columns.  A group's scale is the power of two that puts its largest finite
    magnitude in (224, 448] (at least 2^-126); the values divided by it are rounded to e4m3 (3 bits of mantissa, ties
    to even).  Infinities become NaN, which e4m3 has.
    """
    R, n = x.shape
    h = n // 2
    v = x.float().view(R, 2, h)
    g = -(-h // GROUP)
    v = torch.nn.functional.pad(v, (0, g * GROUP - h)).view(R, 2, g, GROUP)
    mag = v.abs()
    top = torch.where(torch.isfinite(mag), mag, torch.zeros_like(mag)).amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(m), torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126))
    q = torch.where(torch.isinf(v), torch.full_like(v, float("nan")), v / scale).to(torch.float8_e4m3fn).float() * scale
    return q.view(R, 2, g * GROUP)[:, :, :h].reshape(R, n)


def _swiglu_plain(x):
    h = x.shape[1] // 2
    xf = x.double()  # a sigmoid below float32's range times a large value need not be small
    up, gate = xf[:, :h], xf[:, h:]
    return (up * (gate * torch.sigmoid(gate))).to(x.dtype)


class _SwigluPlainFn(torch.autograd.Function):
    """The same on the CPU: the gradient is the formula's at what was kept."""

    @staticmethod
    def forward(ctx, x, keep):
        ctx.save_for_backward(e4m3_checkpoint_reference(x) if keep else x)
        return _swiglu_plain(x)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x = ctx.saved_tensors[0].double()
        h = x.shape[1] // 2
        up, gate, s = x[:, :h], x[:, h:], torch.sigmoid(x[:, h:])
        d = dy.double()
        return torch.cat([d * (gate * s), d * (up * (s * (1 + gate * (1 - s))))], 1).to(dy.dtype), None


def swiglu(x: torch.Tensor, *, checkpoint: str | None = None) -> torch.Tensor:
    """``up * gate * sigmoid(gate)`` of ``x [rows, 2h] = [up | gate]``: ``[rows, h]``.

    For the backward pass x itself is kept, or with ``checkpoint="e4m3"`` an 8-bit copy (half a 16-bit x and 1/32; see
    ``e4m3_checkpoint_reference`` for its values), so that x can be freed after the call: the gradient is then the
    formula's at the values of the copy.  The result does not depend on ``checkpoint``.
    """
    if checkpoint not in (None, "e4m3"):
        raise ValueError(f"checkpoint must be None or 'e4m3', got {checkpoint!r}")
    if x.is_cuda:
        return native().swiglu(x, checkpoint is not None)
    if x.dim() != 2 or x.shape[1] % 2:
        raise ValueError(f"x must be [rows, 2h], got {tuple(x.shape)}")
    return _SwigluPlainFn.apply(x, checkpoint is not None)


# --------------------------------------------------------------- combination
def combine_rows_reference(z, route: ExpertRoute, weights=None):
    """Plain torch (any device, differentiable), in z's type or float32 if that has more bits."""
    acc = z.dtype if z.dtype == torch.float64 else torch.float32
    k = route.row_of.shape[-1]
    at = route.row_of.reshape(-1, k).long()
    on = (at >= 0).unsqueeze(-1)
    zf = torch.cat([z.to(acc), z.new_zeros(1, z.shape[1], dtype=acc)])
    picked = torch.where(on, zf[torch.where(at >= 0, at, z.shape[0])], torch.zeros((), dtype=acc, device=z.device))
    if weights is not None:
        w = weights.reshape(-1, k, 1).to(acc)
        picked = picked * torch.where(on, w, torch.zeros_like(w))  # what stands where there is no choice is not used
    return picked.sum(1).to(z.dtype)


def combine_rows(z: torch.Tensor, route: ExpertRoute, weights: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = sum_j weights[t, j] * z[row_of[t, j]]``: rows ``[R, n]`` of a route back to its tokens ``[tokens, n]``.

    ``weights`` (``route.weights``, or any ``[.., tokens, k]``) may be left out for the plain sum.  Sums are in float32, in
    order of ``j``; a token without rows gets zeros.
    """
    if z.is_cuda:
        return native().combine_rows(z, weights, route.offsets, route.row_of)
    if z.dim() != 2 or z.shape[0] != route.row_of.numel():
        raise ValueError(f"z must be [{route.row_of.numel()}, n] for this route, got {tuple(z.shape)}")
    if route.offsets.dtype != torch.int32 or route.offsets.dim() != 1 or not route.offsets.numel():
        raise ValueError(f"offsets must be int32 [groups + 1], got {route.offsets.dtype} {tuple(route.offsets.shape)}")
    if weights is not None and (weights.numel() != route.row_of.numel() or weights.shape[-1:] != route.row_of.shape[-1:]):
        raise ValueError(f"weights must have the shape {tuple(route.row_of.shape)}, got {tuple(weights.shape)}")
    on_cuda(z, route.row_of, *(() if weights is None else (weights,)))  # refuses a mixture of devices
    return combine_rows_reference(z, route, weights)


# ------------------------------------------------------------ the whole block
def expert_mlp(x: torch.Tensor, logits: torch.Tensor, w_up: torch.Tensor, b_up: torch.Tensor | None, w_down: torch.Tensor,
               b_down: torch.Tensor | None, *, top_k: int, checkpoint: str | None = None) -> torch.Tensor:
    """A routed mixture of SwiGLU experts: ``y[t] = sum_j w_tj (swiglu(x[t] W_up[e_tj] + b_up) W_down[e_tj] + b_down)``.

    ``x [.., d]`` and ``logits [.., experts]`` have the same leading shape (``[tokens]`` or ``[slots, tokens]``); weights
    ``[.., d, 2h]`` and ``[.., h, d]``, biases ``[.., 2h]`` and ``[.., d]``, a matrix for each expert of each slot.  On CUDA
    the limits are those of ``grouped_linear``: 16-bit x, widths in multiples of 8, at most ``MAX_GROUPS`` experts over all
    slots.  Float32 weights are rounded in every call; where that counts (a serving step of a few tokens), pass 16-bit ones.
    """
    if x.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"x and logits must have the same tokens, got {tuple(x.shape)} and {tuple(logits.shape)}")
    route = route_topk(logits, top_k)
    h = grouped_linear(x.reshape(-1, x.shape[-1]), w_up, b_up, route=route)
    z = grouped_linear(swiglu(h, checkpoint=checkpoint), w_down, b_down, offsets=route.offsets)
    return combine_rows(z, route, route.weights).view(*x.shape[:-1], w_down.shape[-1])


__all__ = ["ExpertRoute", "combine_rows", "combine_rows_reference", "e4m3_checkpoint_reference", "expert_mlp", "grouped_linear",
           "grouped_linear_reference", "route_topk", "route_topk_reference", "swiglu"]
