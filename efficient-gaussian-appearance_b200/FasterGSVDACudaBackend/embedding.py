"""Embedding lookup with scaling: rows of a table (latents shared by Gaussians, per-view embeddings, a vocabulary) by
index, and the table's gradient from the sorted indices (csrc/embedding.cu)."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import lib, check, ptr

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _launch(device: torch.device, fn, *args) -> None:
    """Runs a library call with the device's current stream as its last argument, on that device."""
    if device.index == torch.cuda.current_device():
        check(fn(*args, torch.cuda.current_stream().cuda_stream))
    else:
        with torch.cuda.device(device):
            check(fn(*args, torch.cuda.current_stream().cuda_stream))


def _lookup(table: torch.Tensor, indices: torch.Tensor, scale: float, padding: int) -> torch.Tensor:
    rows, width = table.shape[0], table.shape[1:].numel()
    out = torch.empty((*indices.shape, *table.shape[1:]), dtype=table.dtype, device=table.device)
    _launch(table.device, lib.fgs_embedding_lookup, ptr(table), rows, width, _TYPES[table.dtype], ptr(indices), indices.numel(),
            indices.element_size(), scale, padding, ptr(out))
    return out


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table: torch.Tensor, indices: torch.Tensor, scale: float, padding: int) -> torch.Tensor:
        ctx.save_for_backward(indices)
        ctx.table = (table.shape, table.dtype, scale, padding)
        return _lookup(table, indices, scale, padding)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out: torch.Tensor):
        indices, = ctx.saved_tensors
        shape, dtype, scale, padding = ctx.table
        grad_out = grad_out.to(dtype).contiguous()
        width = shape[1:].numel()
        grad = torch.empty(shape, dtype=dtype, device=grad_out.device)
        n = indices.numel()
        space = torch.empty(_lib.size_out(lib.fgs_embedding_workspace_bytes, n, shape[0], width), dtype=torch.uint8, device=grad.device)
        _launch(grad.device, lib.fgs_embedding_grad, ptr(indices), n, indices.element_size(), ptr(grad_out), _TYPES[dtype], shape[0], width, scale,
                padding, ptr(grad), ptr(space), space.numel())
        return grad, None, None, None


def embedding_lookup(table: torch.Tensor, indices: torch.Tensor, scale: float = 1.0, padding_index: int | None = None) -> torch.Tensor:
    """scale * table[indices]: [*indices.shape, *table.shape[1:]], computed in float32 and rounded once to the table's type.

    `table` [rows, ...]: contiguous CUDA float32, bfloat16 or float16; `indices`: int64 or int32 of any shape on the same
    device. A negative index, or `padding_index`, stands for no row: zeros, and no gradient. An index past the table is
    not read: its output is NaN, and it adds to no gradient (nothing is copied to the host to raise an error).

    Differentiable in `table` (once). The gradient is dense, scale * the sum of the output gradients of each row's
    indices: summed in float32 in an order that depends only on the inputs, so the same inputs give the same bits. Both
    directions may be captured into CUDA graphs."""
    if not table.is_cuda or table.dtype not in _TYPES or not table.is_contiguous() or table.dim() < 1:
        raise RuntimeError('table must be a contiguous CUDA float32, bfloat16 or float16 tensor [rows, ...]')
    if indices.dtype not in (torch.int64, torch.int32) or indices.device != table.device:
        raise RuntimeError('indices must be an int64 or int32 tensor on the device of the table')
    if padding_index is not None and not 0 <= padding_index < table.shape[0]:
        raise ValueError('padding_index must be a row of the table (negative indices are padding anyway)')
    indices = indices.contiguous()
    padding = -1 if padding_index is None else int(padding_index)
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbeddingLookup.apply(table, indices, float(scale), padding)
    return _lookup(table, indices, float(scale), padding)
