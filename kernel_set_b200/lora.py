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
import functools
from typing import Optional

import torch

from ._lib import by_address as lib, check
from ._tensor import TensorLike, allocating_on, default_stream, dtype_to_ks, i32_ptr, on_device_of, ptr, same_device


def plan(adapter_ids: torch.Tensor, num_adapters: int, sorted_ids: Optional[torch.Tensor] = None,
         offsets: Optional[torch.Tensor] = None, stream: TensorLike = None):
    """The rows sorted by adapter. ``adapter_ids [tokens]`` int32, an id outside ``[0, num_adapters)`` stands for
    "none". Returns ``(sorted_ids [tokens], offsets [num_adapters + 2])``, both int32, in the given buffers if any. With ``stream``,
    buffers that it makes belong to that stream, as if they had been made with it as the current one."""
    for name, given in (("adapter_ids", adapter_ids), ("sorted_ids", sorted_ids), ("offsets", offsets)):
        if given is not None and given.dtype != torch.int32:
            raise ValueError(f"{name} must be int32; got {given.dtype}")
    same_device(adapter_ids, sorted_ids=sorted_ids, offsets=offsets)
    tokens = adapter_ids.numel()
    if sorted_ids is None or offsets is None:
        with allocating_on(stream, adapter_ids.device):
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


def _ld(t: torch.Tensor, rows: int, cols: int) -> int:
    """Elements from a row of ``t`` to the next; -1 where its rows are not contiguous or overlap."""
    ld, inner = t.stride()
    if inner != 1 and cols > 1:
        return -1
    return cols if rows <= 1 else (ld if ld >= cols else -1)


def _refuse(rows: dict, flat: dict, sorted_ids, offsets, adapters: int) -> None:
    """The message for a call that the wrappers' quick test does not let through: ``rows`` are matrices with contiguous
    rows (tensor, shape, dtype), ``flat`` contiguous tensors."""
    for name, (t, shape, dtype) in {**rows, **flat}.items():
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} must be {list(shape)}; got {list(t.shape)}")
        if t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}; got {t.dtype}")
    if offsets.numel() < adapters + 1:
        raise ValueError(f"offsets: {offsets.numel()} entries where at least {adapters + 1} are expected")
    if offsets.dtype != torch.int32:
        raise ValueError(f"offsets must be int32; got {offsets.dtype}")
    for name, (t, shape, dtype) in rows.items():
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (got device {t.device}); kernel_set operates on device memory")
        if _ld(t, *shape) < 0:
            raise ValueError(f"the rows of {name} must be contiguous and apart")
    for name, (t, shape, dtype) in flat.items():
        ptr(t, name=name)
    ptr(offsets, name="offsets")
    same_device(rows["x"][0], offsets=offsets, **{name: t for name, (t, shape, dtype) in {**rows, **flat}.items()})
    raise AssertionError("unreachable")


def _dims(x: torch.Tensor, b: torch.Tensor):
    if x.dim() != 2 or b.dim() != 3:
        raise ValueError("x must be [tokens, K], a [adapters, rank, K], b [adapters, N, rank]")
    return (*x.shape, *b.shape)


def _plan_ok(sorted_ids, offsets, tokens: int, adapters: int, dev: int) -> bool:
    return (offsets.dtype is torch.int32 and offsets.get_device() == dev and offsets.is_contiguous() and offsets.numel() > adapters
            and (sorted_ids is None or (sorted_ids.dtype is torch.int32 and sorted_ids.get_device() == dev and sorted_ids.is_contiguous()
                                        and sorted_ids.numel() == tokens)))


def apply(out: torch.Tensor, base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor,
          sorted_ids: Optional[torch.Tensor], offsets: torch.Tensor, h: Optional[torch.Tensor] = None,
          stream: TensorLike = None) -> torch.Tensor:
    """``out = base + s B (A x)`` row by row; rows without an adapter get their ``base``.

    ``x [tokens, K]``, ``base`` and ``out [tokens, N]`` (``out`` may be ``base``; rows contiguous, any distance apart,
    so a slice of a fused projection's columns will do), ``a [adapters, rank, K]``, ``b [adapters, N, rank]``, all f16 or bf16;
    ``scales [adapters]`` fp32; ``h [tokens, rank]`` fp32 receives ``A x`` for :func:`backward`."""
    tokens, k, adapters, n, rank = _dims(x, b)
    dt, dev = x.dtype, x.get_device()
    # one quick test of everything: the smallest calls are bound by the host's path
    if not (out.shape == base.shape == (tokens, n) and a.shape == (adapters, rank, k) and scales.shape == (adapters,)
            and out.dtype is base.dtype is a.dtype is b.dtype is dt and scales.dtype is torch.float32
            and out.get_device() == base.get_device() == a.get_device() == b.get_device() == scales.get_device() == dev >= 0
            and (ld_out := _ld(out, tokens, n)) >= 0 and (ld_base := _ld(base, tokens, n)) >= 0 and (ld_x := _ld(x, tokens, k)) >= 0
            and a.is_contiguous() and b.is_contiguous() and scales.is_contiguous() and _plan_ok(sorted_ids, offsets, tokens, adapters, dev)
            and (h is None or (h.shape == (tokens, rank) and h.dtype is torch.float32 and h.get_device() == dev and h.is_contiguous()))):
        flat = {"a": (a, (adapters, rank, k), dt), "b": (b, (adapters, n, rank), dt), "scales": (scales, (adapters,), torch.float32)}
        if sorted_ids is not None:
            flat["sorted_ids"] = (sorted_ids, (tokens,), torch.int32)
        if h is not None:
            flat["h"] = (h, (tokens, rank), torch.float32)
        _refuse({"out": (out, (tokens, n), dt), "base": (base, (tokens, n), dt), "x": (x, (tokens, k), dt)}, flat, sorted_ids, offsets,
                adapters)
    with on_device_of(x):
        check(lib.ks_lora_apply(out.data_ptr(), ld_out, base.data_ptr(), ld_base, None if h is None else h.data_ptr(), x.data_ptr(), ld_x,
                                a.data_ptr(), b.data_ptr(), scales.data_ptr(), None if sorted_ids is None else sorted_ids.data_ptr(),
                                offsets.data_ptr(), tokens, adapters, rank, k, n, dtype_to_ks(dt), default_stream(stream, x)),
              "ks_lora_apply")
    return out


@functools.lru_cache(maxsize=256)
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
    ``base`` as it is. Types and shapes as in :func:`apply`; ``workspace``: uint8, allocated (from
    ``stream``'s pool) if not given.
    Returns ``(d_x, d_a, d_b)``."""
    tokens, k, adapters, n, rank = _dims(x, b)
    dt, dev = x.dtype, x.get_device()
    if not (d_x.shape == d_x_base.shape == (tokens, k) and d_out.shape == (tokens, n) and a.shape == d_a.shape == (adapters, rank, k)
            and d_b.shape == (adapters, n, rank) and h.shape == (tokens, rank) and scales.shape == (adapters,)
            and d_x.dtype is d_x_base.dtype is d_out.dtype is a.dtype is d_a.dtype is b.dtype is d_b.dtype is dt
            and h.dtype is scales.dtype is torch.float32
            and d_x.get_device() == d_x_base.get_device() == d_out.get_device() == a.get_device() == d_a.get_device() == b.get_device()
            == d_b.get_device() == h.get_device() == scales.get_device() == dev >= 0 and a.is_contiguous() and d_a.is_contiguous() and b.is_contiguous() and d_b.is_contiguous()
            and h.is_contiguous() and scales.is_contiguous()
            and (ld_d_x := _ld(d_x, tokens, k)) >= 0 and (ld_d_x_base := _ld(d_x_base, tokens, k)) >= 0
            and (ld_d_out := _ld(d_out, tokens, n)) >= 0 and (ld_x := _ld(x, tokens, k)) >= 0
            and _plan_ok(sorted_ids, offsets, tokens, adapters, dev)):
        flat = {"a": (a, (adapters, rank, k), dt), "d_a": (d_a, (adapters, rank, k), dt), "b": (b, (adapters, n, rank), dt),
                "d_b": (d_b, (adapters, n, rank), dt), "h": (h, (tokens, rank), torch.float32),
                "scales": (scales, (adapters,), torch.float32)}
        if sorted_ids is not None:
            flat["sorted_ids"] = (sorted_ids, (tokens,), torch.int32)
        _refuse({"d_x": (d_x, (tokens, k), dt), "d_x_base": (d_x_base, (tokens, k), dt), "d_out": (d_out, (tokens, n), dt),
                 "x": (x, (tokens, k), dt)}, flat, sorted_ids, offsets, adapters)
    same_device(x, workspace=workspace)
    if workspace is None:
        with allocating_on(stream, x.device):   # (it goes back to that stream's pool when this returns: later calls there come behind)
            workspace = torch.empty(backward_workspace(tokens, adapters, rank, k, n), dtype=torch.uint8, device=x.device)
    with on_device_of(x):
        check(lib.ks_lora_backward(d_x.data_ptr(), ld_d_x, d_a.data_ptr(), d_b.data_ptr(), d_x_base.data_ptr(), ld_d_x_base,
                                   d_out.data_ptr(), ld_d_out, x.data_ptr(), ld_x, h.data_ptr(), a.data_ptr(), b.data_ptr(),
                                   scales.data_ptr(), None if sorted_ids is None else sorted_ids.data_ptr(), offsets.data_ptr(), tokens,
                                   adapters, rank, k, n, ptr(workspace, name="workspace"),
                                   workspace.numel() * workspace.element_size(), dtype_to_ks(dt), default_stream(stream, x)),
              "ks_lora_backward")
    return d_x, d_a, d_b
