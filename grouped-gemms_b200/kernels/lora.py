"""Low-rank adapters of many requests (or experts) beside a grouped projection.

``lora_grouped_mm`` adds ``scaling_l (x A_l^T) B_l^T`` to the rows of each
segment: the segments are the groups of ``triton_mxfp8_grouped_mm``, or any
other cumulative row ends (requests), or single rows (a decode step).
``lora_grouped_mm_backward`` gives its gradients.  bf16 operands, fp32 sums;
no counterpart in the reference.
"""

from typing import Optional

import torch

import mxgg

from ._common import _UNAVAILABLE_MSG, _mxfp8_available


def lora_grouped_mm(
    x: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    group_end_offsets: Optional[torch.Tensor],
    adapter: Optional[torch.Tensor] = None,
    scaling: Optional[torch.Tensor] = None,
    base: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    out_dtype: torch.dtype = None,
    return_v: bool = False,
):
    """``base + scaling[l] * (x @ lora_a[l]^T) @ lora_b[l]^T``, ``l`` the row's adapter.

    Args:
        x: ``(M, K)`` bf16 (the unquantised input of the projection).
        lora_a: ``(L, R, K)`` bf16; lora_b: ``(L, N, R)`` bf16.  K, N and R multiples of 8, R <= 128.
        group_end_offsets: ``(S,)`` int32 / int64 cumulative row ends of the segments (at most 1024; cut at M),
            or ``None``: every row is a segment of its own.  That form is for a decode step: a row looks for its
            adapter's others among 1024, and thousands of rows take ten times as long as in segments.
        adapter: ``(S,)`` int32 / int64 adapter of each segment; a value outside ``[0, L)`` (say -1) means
            none.  ``None``: segment s carries adapter s.
        scaling: ``(L,)`` fp32 factor of each adapter, ``None``: 1.
        base: ``(M, N)`` the projection's output to add to (any row stride); ``None``: zeros.
        out: instead of ``base``: a bf16 / fp16 / fp32 ``(M, N)`` tensor that the product is added into in
            place; it is returned.
        out_dtype: of the result: ``base``'s dtype, or bf16, when not given.
        return_v: also return the scaled intermediate ``lora_grouped_mm_backward`` takes.

    Rows without an adapter are ``base``'s (zeros without one); rows at or past the last end are left
    unwritten, like ``triton_mxfp8_grouped_mm``'s.

    The intermediate ``v = scaling x lora_a^T`` is an fp32 sum kept in two bf16 halves, 16 bits of mantissa: an fp32
    result carries an error of up to 2^-17 of ``sum |v lora_b|``, not fp32's own.
    """
    if not _mxfp8_available:
        raise NotImplementedError(_UNAVAILABLE_MSG)
    if out is not None:
        if base is not None:
            raise ValueError("lora_grouped_mm: base and out are two ways to say what is added to; give one")
        if out_dtype not in (None, out.dtype):
            raise ValueError(f"lora_grouped_mm: out is {out.dtype}, out_dtype {out_dtype}")
        v = mxgg.ops.lora_mm_add(x, lora_a, lora_b, group_end_offsets, adapter, scaling, out, return_v)
        return (out, v) if return_v else out
    if out_dtype is None:
        out_dtype = base.dtype if base is not None else torch.bfloat16
    f = mxgg.ops.lora_mm_v if return_v else mxgg.ops.lora_mm
    return f(x, lora_a, lora_b, group_end_offsets, adapter, scaling, base, out_dtype)


def lora_grouped_mm_backward(
    grad_out: torch.Tensor,
    x: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    v: torch.Tensor,
    group_end_offsets: torch.Tensor,
    adapter: Optional[torch.Tensor] = None,
    scaling: Optional[torch.Tensor] = None,
    grad_base: Optional[torch.Tensor] = None,
    grad_x_dtype: torch.dtype = None,
    grad_w_dtype: torch.dtype = torch.bfloat16,
    need=(True, True, True),
):
    """Gradients of ``lora_grouped_mm``: ``(grad_x, grad_a, grad_b)``.

    ``grad_out`` is ``(M, N)`` bf16, ``v`` what the forward returned with ``return_v``; the other arguments
    are the forward's.  ``grad_x = grad_base + scaling[l] * (grad_out @ lora_b[l]) @ lora_a[l]`` where
    ``grad_base`` ``(M, K)`` is the gradient that reaches x through the projection itself (``None``: zeros),
    of ``grad_x_dtype`` (``grad_base``'s dtype, or bf16); rows at or past the last end are left unwritten.
    ``grad_a`` ``(L, R, K)`` and ``grad_b`` ``(L, N, R)`` of ``grad_w_dtype`` (bf16, fp16 or fp32) sum over
    every row that carries the adapter (zeros where none does), in an order that does not depend on timing.
    ``need`` says which of the three are wanted; the others come back empty.
    Infinite elements give the formula's infinities, except that at ranks above 32 those of ``x`` in ``grad_a`` and of
    ``grad_out`` in ``grad_b`` may give NaN instead.
    """
    if not _mxfp8_available:
        raise NotImplementedError(_UNAVAILABLE_MSG)
    if group_end_offsets is None:
        raise ValueError("lora_grouped_mm_backward: the gradients take segments, not single rows")
    if grad_x_dtype is None:
        grad_x_dtype = grad_base.dtype if grad_base is not None else torch.bfloat16
    return mxgg.ops.lora_mm_backward(grad_out, x, lora_a, lora_b, v, group_end_offsets, adapter, scaling, grad_base,
                                     grad_x_dtype, grad_w_dtype, [bool(n) for n in need])
