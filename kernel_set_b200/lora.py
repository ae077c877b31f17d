"""Low-rank adapters of many requests at once beside a projection that they share, and their gradient.

Row ``t`` of the batch has adapter ``a(t)`` or none; ``s`` is the adapter's scale, ``A [rank, K]`` and ``B [N, rank]`` its
factors: ``out[t] = base[t] + s B (A x[t])``. The rows are taken in the order of a plan, sorted by adapter, which is
made once for a step and serves all of its layers::

    sorted_ids, offsets = lora.plan(adapter_ids, num_adapters)
    y = dispatch.w4a16(x, ...)                                     # the shared projection
    lora.apply(y, y, x, a, b, scales, sorted_ids, offsets)         # in place

For training, ``apply(..., h=h)`` keeps ``A x`` and :func:`backward` gives the gradients. Rows sorted by expert
(``moe.permute``) take an adapter per expert with ``sorted_ids=None`` and the experts' offsets. The reference has no
operator of this kind."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._lib import by_address as lib, check
from ._tensor import TensorLike, default_stream, dtype_to_ks, f32_ptr, i32_ptr, on_device_of, ptr, same_dtype, stream_ptr


def plan(adapter_ids: torch.Tensor, num_adapters: int, sorted_ids: Optional[torch.Tensor] = None,
         offsets: Optional[torch.Tensor] = None, stream: TensorLike = None):
    """The rows sorted by adapter. ``adapter_ids [tokens]`` int32, an id outside ``[0, num_adapters)`` stands for
    "none". Returns ``(sorted_ids [tokens], offsets [num_adapters + 2])``, both int32, in the given buffers if any."""
    if adapter_ids.dtype != torch.int32:
        raise ValueError(f"adapter_ids must be int32; got {adapter_ids.dtype}")
    tokens = adapter_ids.numel()
    if sorted_ids is None:
        sorted_ids = torch.empty(tokens, dtype=torch.int32, device=adapter_ids.device)
    if offsets is None:
        offsets = torch.empty(int(num_adapters) + 2, dtype=torch.int32, device=adapter_ids.device)
    _sizes(num_adapters=(offsets.numel(), int(num_adapters) + 2), tokens=(sorted_ids.numel(), tokens))
    with on_device_of(adapter_ids):
        check(lib.ks_lora_plan(i32_ptr(sorted_ids, name="sorted_ids"), i32_ptr(offsets, name="offsets"),
                               i32_ptr(adapter_ids, name="adapter_ids"), tokens, int(num_adapters),
                               default_stream(stream, adapter_ids)), "ks_lora_plan")
    return sorted_ids, offsets


def _sizes(**pairs) -> None:
    for what, (got, want) in pairs.items():
        if got != want:
            raise ValueError(f"{what}: {got} where {want} is expected")


def _rows(t: torch.Tensor, name: str, rows: int, cols: int):
    """Address and leading dimension of a matrix whose rows are contiguous."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (got device {t.device}); kernel_set operates on device memory")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols:
        raise ValueError(f"{name} must be [{rows}, {cols}]; got {list(t.shape)}")
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    ld = t.stride(0) if rows > 1 else cols
    if ld < cols:
        raise ValueError(f"the rows of {name} overlap")
    return t.data_ptr(), ld


def _problem(x, a, b, scales, sorted_ids, offsets):
    if a.dim() != 3 or b.dim() != 3 or x.dim() != 2:
        raise ValueError("x must be [tokens, K], a [adapters, rank, K], b [adapters, N, rank]")
    adapters, rank, k = a.shape
    n = b.shape[1]
    tokens = x.shape[0]
    _sizes(b=(tuple(b.shape), (adapters, n, rank)), scales=(scales.numel(), adapters))
    if offsets.numel() < adapters + 1:
        raise ValueError(f"offsets: {offsets.numel()} entries where at least {adapters + 1} are expected")
    if sorted_ids is not None:
        _sizes(sorted_ids=(sorted_ids.numel(), tokens))
    if scales.dtype != torch.float32:
        raise ValueError(f"scales must be float32; got {scales.dtype}")
    for name, t in (("sorted_ids", sorted_ids), ("offsets", offsets)):
        if t is not None and t.dtype != torch.int32:
            raise ValueError(f"{name} must be int32; got {t.dtype}")
    return tokens, adapters, rank, k, n


def apply(out: torch.Tensor, base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor,
          sorted_ids: Optional[torch.Tensor], offsets: torch.Tensor, h: Optional[torch.Tensor] = None,
          stream: TensorLike = None) -> torch.Tensor:
    """``out = base + s B (A x)`` row by row; rows without an adapter get their ``base``.

    ``x [tokens, K]``, ``base`` and ``out [tokens, N]`` (``out`` may be ``base``; rows contiguous, any distance apart,
    so a slice of a fused projection's columns will do), ``a [adapters, rank, K]``, ``b [adapters, N, rank]``, all f16 or bf16;
    ``scales [adapters]`` fp32; ``h [tokens, rank]`` fp32 receives ``A x`` for :func:`backward`."""
    tokens, adapters, rank, k, n = _problem(x, a, b, scales, sorted_ids, offsets)
    same_dtype(x, out=out, base=base, a=a, b=b)
    out_ptr, ld_out = _rows(out, "out", tokens, n)
    base_ptr, ld_base = _rows(base, "base", tokens, n)
    x_ptr, ld_x = _rows(x, "x", tokens, k)
    if h is not None:
        if h.dtype != torch.float32:
            raise ValueError(f"h must be float32; got {h.dtype}")
        _sizes(h=(tuple(h.shape), (tokens, rank)))
    with on_device_of(x):
        check(lib.ks_lora_apply(out_ptr, ld_out, base_ptr, ld_base, f32_ptr(h, name="h"), x_ptr, ld_x, ptr(a, name="a"),
                                ptr(b, name="b"), f32_ptr(scales, name="scales"), i32_ptr(sorted_ids, name="sorted_ids"),
                                i32_ptr(offsets, name="offsets"), tokens, adapters, rank, k, n, dtype_to_ks(x.dtype),
                                default_stream(stream, x)), "ks_lora_apply")
    return out


def backward_workspace(tokens: int, adapters: int, rank: int, k: int, n: int) -> int:
    """Bytes of workspace that :func:`backward` needs for these sizes."""
    size = ctypes.c_size_t()
    check(lib.ks_lora_backward_workspace(ctypes.byref(size), int(tokens), int(adapters), int(rank), int(k), int(n)),
          "ks_lora_backward_workspace")
    return size.value


def backward(d_x: torch.Tensor, d_a: torch.Tensor, d_b: torch.Tensor, d_x_base: torch.Tensor, d_out: torch.Tensor,
             x: torch.Tensor, h: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor,
             sorted_ids: Optional[torch.Tensor], offsets: torch.Tensor, workspace: Optional[torch.Tensor] = None,
             stream: TensorLike = None):
    """Gradient of :func:`apply`: with ``g = s B^T d_out`` per row, ``d_x = d_x_base + A^T g`` (``d_x`` may be
    ``d_x_base``, the gradient through the shared projection), ``d_a = sum g x^T`` and ``d_b = s sum d_out h^T`` over each
    adapter's rows, zeros for an adapter without rows. ``h`` is what the forward pass kept. ``d_out`` is the gradient of
    ``base`` as it is. Types and shapes as in :func:`apply`; ``workspace``: uint8, allocated if not given.
    Returns ``(d_x, d_a, d_b)``."""
    tokens, adapters, rank, k, n = _problem(x, a, b, scales, sorted_ids, offsets)
    same_dtype(x, d_x=d_x, d_a=d_a, d_b=d_b, d_x_base=d_x_base, d_out=d_out, a=a, b=b)
    _sizes(d_a=(tuple(d_a.shape), tuple(a.shape)), d_b=(tuple(d_b.shape), tuple(b.shape)),
           h=(tuple(h.shape), (tokens, rank)))
    if h.dtype != torch.float32:
        raise ValueError(f"h must be float32; got {h.dtype}")
    d_x_ptr, ld_d_x = _rows(d_x, "d_x", tokens, k)
    d_x_base_ptr, ld_d_x_base = _rows(d_x_base, "d_x_base", tokens, k)
    d_out_ptr, ld_d_out = _rows(d_out, "d_out", tokens, n)
    x_ptr, ld_x = _rows(x, "x", tokens, k)
    if workspace is None:
        workspace = torch.empty(backward_workspace(tokens, adapters, rank, k, n), dtype=torch.uint8, device=x.device)
        if stream is not None:   # it goes back to its pool when this returns
            workspace.record_stream(torch.cuda.ExternalStream(stream_ptr(stream), device=x.device))
    with on_device_of(x):
        check(lib.ks_lora_backward(d_x_ptr, ld_d_x, ptr(d_a, name="d_a"), ptr(d_b, name="d_b"), d_x_base_ptr, ld_d_x_base,
                                   d_out_ptr, ld_d_out, x_ptr, ld_x, f32_ptr(h, name="h"), ptr(a, name="a"), ptr(b, name="b"),
                                   f32_ptr(scales, name="scales"), i32_ptr(sorted_ids, name="sorted_ids"),
                                   i32_ptr(offsets, name="offsets"), tokens, adapters, rank, k, n,
                                   ptr(workspace, name="workspace"), workspace.numel() * workspace.element_size(),
                                   dtype_to_ks(x.dtype), default_stream(stream, x)), "ks_lora_backward")
    return d_x, d_a, d_b
