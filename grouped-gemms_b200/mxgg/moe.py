"""Mixture-of-experts layer on the mxgg kernels (forward).

    logits -> top-2 routing -> quantise-on-dispatch (gather + to_mx, one pass)
    -> up projection (d_model -> d_ff) per expert, to_mx fused into its epilogue
    -> down projection (d_ff -> d_model) per expert -> weighted top-2 combine

Expert weights are MXFP8, or MXFP4 (e2m1) with MXFP8 activations.  Each
expert's rows are padded to a multiple of 32 (zero rows), the group alignment
the weight-gradient kernels and the inbox transfers need.  With a
`FusedExpertParallel`, rank r hosts its placement's experts: rows travel to
the hosting rank by peer copies, the up projection reads them in place, and
the down projection stores its tiles straight to the rows' owners.  In
`MoELayer` the routing is small torch ops; the GEMMs, the quantisers and the
final weighted sum are the sm_100a kernels.

For training, and for routing without a host synchronisation, the pieces stand
alone: `route_topk` (any top-k, with per-expert counts, a balance loss and a z
loss), `dispatch_plan` (the layout built on the GPU, capturable),
`combine_topk`, and their gradients `route_topk_backward`,
`combine_topk_backward` and `dispatch_backward`.  Like the GEMMs, they are
plain functions: a gradient is a call, not an autograd node.
"""

import ctypes
from dataclasses import dataclass
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from .ep import ExpertPlacement, FusedExpertParallel
from .ops import (_IN_DTYPES, _addr, _as, _on, _one_device, _ptr, _raw_stream, _scratch, _stream, grouped_mm_mx,
                  grouped_mm_segments, to_mx, to_mx_fp4)

PAD = 32


def route_top2(logits: Tensor):
    """Softmax over experts, the two largest, renormalised: (experts (T, 2), weights (T, 2) fp32)."""
    probs = torch.softmax(logits.float(), dim=-1)
    w, e = torch.topk(probs, 2, dim=-1)
    return e, w / w.sum(-1, keepdim=True)


@dataclass
class DispatchLayout:
    row_index: Tensor     # (P,) int32 source token of every padded row, -1 for padding
    counts: list          # (E,) padded rows per expert (multiples of PAD)
    pair_pos: Tensor      # (T, 2) int64 padded row of each (token, choice)


def dispatch_layout(experts: Tensor, n_experts: int, pad: int = PAD) -> DispatchLayout:
    """Rows sorted by expert, every expert's rows padded to a multiple of `pad`."""
    T, k = experts.shape
    flat = experts.reshape(-1).to(torch.int64)      # route_topk's choices are int32
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=n_experts)
    padded = (counts + pad - 1) // pad * pad
    start_pad = torch.cumsum(padded, 0) - padded
    start = torch.cumsum(counts, 0) - counts
    e_sorted = flat[order]
    pos_sorted = start_pad[e_sorted] + (torch.arange(flat.numel(), device=flat.device) - start[e_sorted])
    P = int(padded.sum())
    row_index = torch.full((P,), -1, dtype=torch.int32, device=flat.device)
    row_index[pos_sorted] = (order // k).to(torch.int32)
    pair_pos = torch.empty_like(flat)
    pair_pos[order] = pos_sorted
    return DispatchLayout(row_index=row_index, counts=padded.tolist(), pair_pos=pair_pos.reshape(T, k))


def quantize_gather(x: Tensor, row_index: Tensor):
    """(scales, q) of to_mx(x[row_index]) with zero rows where row_index < 0, in one pass."""
    x = x.contiguous()
    P, C = row_index.numel(), x.shape[1]
    q = torch.empty((P, C), dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty((P, C // 32), dtype=torch.uint8, device=x.device)
    _lib.check(_lib.load().mxgg_quantize_mx_gather(_ptr(x), _IN_DTYPES[x.dtype], x.shape[0], _ptr(row_index), P, C,
                                                   _ptr(q), _ptr(s), _stream(x.device)), "mxgg_quantize_mx_gather")
    return s, q


def combine_top2(y: Tensor, layout: DispatchLayout, weights: Tensor, out_dtype=torch.bfloat16) -> Tensor:
    """out[t] = sum_k weights[t, k] * y[pair_pos[t, k]] (fp32 sum in choice order, one pass)."""
    if out_dtype != torch.bfloat16 or y.dtype != torch.bfloat16:
        raise TypeError("combine_top2 takes and returns bf16 rows")
    y = y.contiguous()
    T, k = layout.pair_pos.shape
    N = y.shape[1]
    out = torch.empty((T, N), dtype=torch.bfloat16, device=y.device)
    pos = layout.pair_pos.to(torch.int64).contiguous()
    w = weights.to(torch.float32).contiguous()
    _lib.check(_lib.load().mxgg_combine_topk(_ptr(y), y.shape[0], _ptr(pos), _ptr(w), T, N, k, _ptr(out),
                                             _stream(y.device)), "mxgg_combine_topk")
    return out


class Routing(NamedTuple):
    experts: Tensor        # (T, k) int32, -1 where there is no choice
    weights: Tensor        # (T, k) fp32
    counts: Tensor         # (E,) int32 choices of each expert
    balance_loss: Tensor   # () fp32: E * sum_e f_e P_e
    z_loss: Tensor         # () fp32: mean of logsumexp^2
    buffer: Tensor         # int32: the allocation the fields are views of; the backward pass reads it, so leave it as it is
    renormalise: bool

    @property
    def stats(self) -> Tensor:
        """(T, 2) fp32: largest logit and log sum exp(logit - it)."""
        T, k = self.experts.shape
        return self.buffer.view(torch.float32).as_strided((T, 2), (2, 1), _routing_parts(T, k, self.counts.shape[0])[2])

    @property
    def tokens(self) -> Tensor:
        """() int32: tokens that count."""
        return self.buffer.as_strided((), (), _routing_parts(*self.experts.shape, self.counts.shape[0])[4] + 2)


def _routing_parts(T: int, k: int, E: int) -> tuple:
    """Offsets, in 4-byte elements, of a Routing buffer's 16-byte aligned parts: experts, weights, stats, counts,
    (balance, z, tokens), scratch."""
    tk, st, e = (T * k + 3) & ~3, (2 * T + 3) & ~3, (E + 3) & ~3
    return 0, tk, 2 * tk, 2 * tk + st, 2 * tk + st + e, 2 * tk + st + e + 4


@lru_cache(maxsize=256)
def _routing_sizes(T: int, k: int, E: int) -> Tuple[tuple, int]:
    """A Routing buffer's parts and the bytes of its scratch (negative: no such size); they follow from the
    sizes alone, and asking for them anew takes 1.5 us of a call's host time."""
    return _routing_parts(T, k, E), _lib.load().mxgg_route_workspace_size(T, E)


def route_topk(logits: Tensor, k: int, token_mask: Optional[Tensor] = None, renormalise: bool = True) -> Routing:
    """Softmax router: the k largest of each row of `logits` ((T, E) bf16 / fp16 / fp32, any row stride),
    the lowest expert first among equals, with their softmax weights (over their sum with `renormalise`),
    per-expert counts, the balance loss E * sum_e f_e P_e (f_e the share of the choices, P_e the mean
    softmax) and the z loss (mean logsumexp^2).

    `token_mask` (T,) bool: tokens where it is false get experts -1 and weights 0 and take no part in
    counts or losses, whatever their logits hold.  A logit of -inf switches an expert off for a token; a
    token with no logit above it is treated like a masked one.  E <= 1024, k <= 16."""
    what = "mxgg.moe.route_topk"
    dev = _one_device(what, logits, token_mask)
    if logits.dtype not in _IN_DTYPES:
        raise TypeError(f"{what}: unsupported logits dtype {logits.dtype}")
    if logits.dim() != 2:
        raise ValueError(f"{what}: logits must be (tokens, experts), got {tuple(logits.shape)}")
    T, E = logits.shape
    logits, ld = _rows(logits)
    if token_mask is not None:
        if token_mask.dtype != torch.bool or token_mask.shape != (T,):
            raise ValueError(f"{what}: token_mask must be a bool ({T},) tensor")
        token_mask = token_mask.contiguous()
    if not 1 <= k <= E:
        raise ValueError(f"{what}: k = {k} of {E} experts")
    lib = _lib.load()
    # One allocation for every output and the scratch: an allocation costs 2.4 us of host time, a view of it
    # 1 us, the kernel of a decode step 6 us.
    at, ws_bytes = _routing_sizes(T, k, E)
    with _on(dev):
        ints = torch.empty(at[5] + max(ws_bytes, 0) // 4, dtype=torch.int32, device=dev)
        floats = ints.view(torch.float32)
        p = ints.data_ptr()
        _lib.check(lib.mxgg_route_topk(_addr(logits), _IN_DTYPES[logits.dtype], ld, _addr(token_mask), T, E, k,
                                       int(renormalise), p, p + 4 * at[1], p + 4 * at[2], p + 4 * at[3],
                                       p + 4 * at[4], p + 4 * at[4] + 8, p + 4 * at[5], ws_bytes, _raw_stream(dev)),
                   "mxgg_route_topk")
    return Routing(ints.as_strided((T, k), (k, 1), 0), floats.as_strided((T, k), (k, 1), at[1]),
                   ints.as_strided((E,), (1,), at[3]), floats.as_strided((), (), at[4]),
                   floats.as_strided((), (), at[4] + 1), ints, bool(renormalise))


def _rows(t: Tensor) -> Tuple[Tensor, int]:
    """A 2-D `t` with contiguous rows that do not overlap, and the elements between them (kept as it comes
    where that is so already)."""
    T, E = t.shape
    if (E > 1 and t.stride(1) != 1) or (T > 1 and t.stride(0) < E):
        t = t.contiguous()
    return t, (t.stride(0) if T > 1 else E)


def _routing_record(what: str, routing: Routing) -> Tuple[int, int, int, tuple]:
    """(T, k, E, parts) of a Routing whose buffer is what route_topk wrote, or an error."""
    buf, choices, counts = routing.buffer, routing.experts.shape, routing.counts.shape
    if len(choices) != 2 or len(counts) != 1:
        raise ValueError(f"{what}: routing holds experts {tuple(choices)} and counts {tuple(counts)}, not (tokens, k) "
                         "and (experts,)")
    (T, k), E = choices, counts[0]
    at, ws_bytes = _routing_sizes(T, k, E)
    # the whole size: a record of more tokens than the fields have lies otherwise
    if buf.dtype != torch.int32 or buf.shape != (at[5] + max(ws_bytes, 0) // 4,) or not buf.is_contiguous():
        raise ValueError(f"{what}: routing.buffer must be the int32 tensor of route_topk for ({T}, {k}) choices of {E} "
                         f"experts, got {buf.dtype} {tuple(buf.shape)}")
    if not buf.is_inference() and buf._version != 0:
        raise ValueError(f"{what}: a tensor of routing was changed in place; the gradient is that of route_topk's own "
                         "weights, counts and choices, so change a copy")
    return T, k, E, at


def route_topk_backward(logits: Tensor, routing: Routing, grad_weights: Optional[Tensor] = None,
                        grad_balance_loss: Union[Tensor, float, None] = None,
                        grad_z_loss: Union[Tensor, float, None] = None) -> Tensor:
    """Gradient to the logits of `route_topk(logits, ...) -> routing` ((T, E), the logits' dtype), for the
    gradients of its weights ((T, k) fp32) and of its two losses (a float, or a one-element fp32 tensor on
    the GPU).  None: no gradient there.  Choices and counts are constants.  Zero rows for tokens that do
    not count.  All it needs of `routing` it reads from `routing.buffer`: a Routing with other tensors in the
    fields' places gives the same gradient, and one whose tensors were changed in place is refused."""
    what = "mxgg.moe.route_topk_backward"
    T, k, E, at = _routing_record(what, routing)
    scalars = [g if isinstance(g, Tensor) else None for g in (grad_balance_loss, grad_z_loss)]
    dev = _one_device(what, logits, routing.buffer, grad_weights, *scalars)
    if logits.dtype not in _IN_DTYPES:
        raise TypeError(f"{what}: unsupported logits dtype {logits.dtype}")
    if logits.shape != (T, E):
        raise ValueError(f"{what}: logits must be ({T}, {E}), got {tuple(logits.shape)}")
    logits, ld = _rows(logits)
    if grad_weights is not None:
        if grad_weights.shape != (T, k):
            raise ValueError(f"{what}: grad_weights must be ({T}, {k}), got {tuple(grad_weights.shape)}")
        grad_weights = _as(grad_weights, torch.float32)
    for i, g in enumerate(scalars):
        if g is not None:
            if g.numel() != 1:
                raise ValueError(f"{what}: a loss gradient is a float or a one-element tensor")
            scalars[i] = g.to(torch.float32)
    coef = [1.0 if isinstance(g, Tensor) else float(g or 0.0) for g in (grad_balance_loss, grad_z_loss)]
    p = routing.buffer.data_ptr()
    grad = logits.new_empty((T, E))
    with _on(dev):
        _lib.check(_lib.load().mxgg_route_topk_backward(
            logits.data_ptr(), _IN_DTYPES[logits.dtype], ld, T, E, k, int(routing.renormalise),
            p, p + 4 * at[1], p + 4 * at[2], p + 4 * at[3], p + 4 * at[4] + 8, _addr(grad_weights), _addr(scalars[0]), coef[0], _addr(scalars[1]), coef[1],
            grad.data_ptr(), _raw_stream(dev)), "mxgg_route_topk_backward")
    return grad


class DispatchPlan(NamedTuple):
    offs: Tensor        # (E,) int32 cumulative padded group ends, the grouped GEMMs' offsets
    counts: Tensor      # (E,) int32 rows in use per expert
    row_index: Tensor   # (P,) int32 source token of every row, -1 in padding
    pair_pos: Tensor    # (T, k) int64 row of each (token, choice), -1 for one that takes no part


def dispatch_plan(experts: Tensor, n_experts: int, pad: int = PAD) -> DispatchPlan:
    """`dispatch_layout` built on the GPU: rows sorted by expert (stable in (token, choice) order), every
    expert's rows padded to a multiple of `pad`.  Nothing travels to the host, so the call can be captured
    into a CUDA graph; row_index is as long as the most any choice can need (its rows at or past offs[-1]
    are -1, and the grouped GEMMs leave such rows unwritten).  Experts outside [0, n_experts) (the -1 of a
    masked token) take no part.  n_experts <= 1024."""
    what = "mxgg.moe.dispatch_plan"
    dev = _one_device(what, experts)
    if experts.dim() != 2 or experts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: experts must be an int32 or int64 (tokens, k) tensor")
    T, k = experts.shape
    if experts.dtype == torch.int64:
        # a value that int32 does not hold must not wrap into the range
        experts = torch.where((experts >= 0) & (experts < n_experts), experts, -1)
    experts = _as(experts, torch.int32)
    lib = _lib.load()
    rows = int(lib.mxgg_dispatch_plan_rows(T, k, n_experts, pad))
    ws_bytes = int(lib.mxgg_dispatch_plan_workspace_size(T, k, n_experts))
    if rows < 0 or ws_bytes < 0:
        raise ValueError(f"{what}: unsupported sizes (tokens {T}, k {k}, experts {n_experts}, pad {pad})")
    # one allocation, as in route_topk: pair_pos, then the int32 parts
    with _on(dev):
        longs = torch.empty(T * k + n_experts + (rows + 1) // 2 + (ws_bytes + 23) // 8, dtype=torch.int64, device=dev)
        ints = longs.view(torch.int32)
        o_off = 2 * T * k
        o_row = o_off + 2 * n_experts
        o_ws = (o_row + rows + 3) & ~3
        p = longs.data_ptr()
        _lib.check(lib.mxgg_dispatch_plan(_addr(experts), T, k, n_experts, pad, p + 4 * o_off,
                                          p + 4 * (o_off + n_experts), p + 4 * o_row, rows, p, p + 4 * o_ws, ws_bytes,
                                          _raw_stream(dev)), "mxgg_dispatch_plan")
    return DispatchPlan(ints.as_strided((n_experts,), (1,), o_off), ints.as_strided((n_experts,), (1,), o_off + n_experts),
                        ints.as_strided((rows,), (1,), o_row), longs.as_strided((T, k), (k, 1), 0))


def _check_pairs(what: str, rows: Tensor, pair_pos: Tensor) -> None:
    if rows.dim() != 2 or rows.dtype != torch.bfloat16:
        raise TypeError(f"{what}: rows must be a 2-D bf16 tensor, got {rows.dtype} {tuple(rows.shape)}")
    if pair_pos.dim() != 2 or pair_pos.dtype != torch.int64:
        raise TypeError(f"{what}: pair_pos must be an int64 (tokens, k) tensor")


def combine_topk(y: Tensor, pair_pos: Tensor, weights: Tensor) -> Tensor:
    """out[t] = sum_j weights[t, j] * y[pair_pos[t, j]] for any k: bf16 rows, fp32 sum in choice order, bf16
    out; positions outside y (the -1 of a masked token) contribute nothing."""
    what = "mxgg.moe.combine_topk"
    dev = _one_device(what, y, pair_pos, weights)
    _check_pairs(what, y, pair_pos)
    if weights.shape != pair_pos.shape:
        raise ValueError(f"{what}: weights must be {tuple(pair_pos.shape)}, got {tuple(weights.shape)}")
    y, pair_pos, weights = y.contiguous(), pair_pos.contiguous(), _as(weights, torch.float32)
    (T, k), (rows, N) = pair_pos.shape, y.shape
    if rows == 0 or k == 0:
        return torch.zeros((T, N), dtype=torch.bfloat16, device=dev)
    with _on(dev):
        out = torch.empty((T, N), dtype=torch.bfloat16, device=dev)
        _lib.check(_lib.load().mxgg_combine_topk(_addr(y), rows, _addr(pair_pos), _addr(weights), T, N, k, _addr(out),
                                                 _raw_stream(dev)), "mxgg_combine_topk")
    return out


def combine_topk_backward(grad_out: Tensor, y: Tensor, pair_pos: Tensor, weights: Tensor,
                          row_index: Tensor) -> Tuple[Tensor, Tensor]:
    """Gradients of `combine_topk`: (grad_y, grad_weights).  grad_y is bf16 like y, with zeros in the rows
    no choice lies in (the padding, whose products a weight gradient must not see); grad_weights is (T, k)
    fp32, 0 where a choice has no row.  pair_pos and row_index come from `dispatch_plan` or
    `dispatch_layout` (no row belongs to two choices)."""
    what = "mxgg.moe.combine_topk_backward"
    dev = _one_device(what, grad_out, y, pair_pos, weights, row_index)
    _check_pairs(what, y, pair_pos)
    (T, k), (rows, N) = pair_pos.shape, y.shape
    if grad_out.dtype != torch.bfloat16 or grad_out.shape != (T, N):
        raise ValueError(f"{what}: grad_out must be a bf16 ({T}, {N}) tensor")
    if weights.shape != (T, k):
        raise ValueError(f"{what}: weights must be ({T}, {k}), got {tuple(weights.shape)}")
    if row_index.dtype != torch.int32 or row_index.shape != (rows,):
        raise ValueError(f"{what}: row_index must be an int32 ({rows},) tensor")
    grad_out, y, pair_pos = grad_out.contiguous(), y.contiguous(), pair_pos.contiguous()
    weights, row_index = _as(weights, torch.float32), row_index.contiguous()
    if k == 0:
        return torch.zeros_like(y), torch.zeros((T, 0), dtype=torch.float32, device=dev)
    with _on(dev):
        grad_y = y.new_empty((rows, N))
        grad_w = weights.new_empty((T, k))
        _lib.check(_lib.load().mxgg_combine_topk_backward(
            _addr(grad_out), _addr(y), rows, _addr(pair_pos), _addr(weights), _addr(row_index), T, N, k, _addr(grad_y),
            _addr(grad_w), _raw_stream(dev)), "mxgg_combine_topk_backward")
    return grad_y, grad_w


def dispatch_backward(grad_rows: Tensor, pair_pos: Tensor) -> Tensor:
    """Gradient of the dispatch (row pair_pos[t, j] holds token t): grad_x[t] = sum_j
    grad_rows[pair_pos[t, j]], bf16 rows, fp32 sum in choice order, bf16 out."""
    what = "mxgg.moe.dispatch_backward"
    dev = _one_device(what, grad_rows, pair_pos)
    _check_pairs(what, grad_rows, pair_pos)
    grad_rows, pair_pos = grad_rows.contiguous(), pair_pos.contiguous()
    (T, k), (rows, N) = pair_pos.shape, grad_rows.shape
    if k == 0:
        return torch.zeros((T, N), dtype=torch.bfloat16, device=dev)
    with _on(dev):
        out = torch.empty((T, N), dtype=torch.bfloat16, device=dev)
        _lib.check(_lib.load().mxgg_dispatch_backward(_addr(grad_rows), rows, _addr(pair_pos), T, N, k, _addr(out),
                                                      _raw_stream(dev)), "mxgg_dispatch_backward")
    return out


def _quantize_weights(w: Tensor, fp4: bool):
    L, N, K = w.shape
    w2 = w.reshape(L * N, K)
    if fp4:
        s, q = to_mx_fp4(w2, _lib.SCALE_ROW_MAJOR)
        return q.view(torch.uint8).reshape(L, N, K // 2).view(torch.float4_e2m1fn_x2), s.reshape(L, N, K // 32)
    s, q = to_mx(w2, _lib.QUANT_ROWS, _lib.SCALE_ROW_MAJOR)
    return q.reshape(L, N, K), s.reshape(L, N, K // 32)


class MoELayer:
    """Top-2 MoE FFN forward with `experts` hosted on this rank.

    w_up (L, d_ff, d_model) and w_down (L, d_model, d_ff) bf16 are the hosted
    experts' weights (quantised once here); `placement`/`ep` select expert
    parallelism (None: every expert on this GPU)."""

    def __init__(self, w_up: Tensor, w_down: Tensor, n_experts: int, weights_fp4: bool = False,
                 placement: Optional[ExpertPlacement] = None, ep: Optional[FusedExpertParallel] = None):
        self.n_experts = n_experts
        self.placement = placement
        self.ep = ep
        self.d_ff, self.d_model = w_up.shape[1], w_up.shape[2]
        self.fp4 = weights_fp4
        self.up_q, self.up_s = _quantize_weights(w_up, weights_fp4)
        self.down_q, self.down_s = _quantize_weights(w_down, weights_fp4)

    def forward(self, x: Tensor, logits: Tensor) -> Tensor:
        experts, weights = route_top2(logits)
        if self.ep is None:
            # the plan stays on the GPU: no host synchronisation, and the call can be captured
            lay = dispatch_plan(experts, self.n_experts)
            a_s, a_q = quantize_gather(x, lay.row_index)
            seg_e = torch.arange(self.n_experts, dtype=torch.int32, device=x.device)
            # the up projection's epilogue writes to_mx of its bf16 output
            h_s, h_q, _, _, _ = grouped_mm_mx(a_q, self.up_q, a_s, self.up_s, lay.offs, seg_e, torch.bfloat16, False)
            y = grouped_mm_segments(h_q, self.down_q, h_s, self.down_s, lay.offs, seg_e, torch.bfloat16)
            return combine_topk(y, lay.pair_pos, weights)
        layout = dispatch_layout(experts, self.n_experts)
        a_s, a_q = quantize_gather(x, layout.row_index)
        # rows stream into the hosts' receive buffers while the up projection
        # consumes them; the down projection sends its rows to their owners
        ep = self.ep
        plan = ep.plan(layout.counts, self.placement)
        ep.dispatch(plan, a_q, a_s)
        h_q = torch.empty((plan.rows_recv, self.d_ff), dtype=torch.float8_e4m3fn, device=x.device)
        h_s = torch.empty((plan.rows_recv, self.d_ff // 32), dtype=torch.uint8, device=x.device)
        ep.gemm_received(plan, self.d_model, self.up_q, self.up_s, torch.bfloat16, local_mx=(h_q, h_s))
        ep.gemm_local(plan, h_q, h_s, self.down_q, self.down_s, torch.bfloat16)
        y = ep.finish(plan, self.d_model, torch.bfloat16)
        return combine_top2(y, layout, weights)

    def flops(self, tokens: int) -> float:
        """Useful FLOPs of one forward over `tokens` tokens (padding excluded)."""
        return 2.0 * (2 * tokens) * self.d_model * self.d_ff * 2
