"""Embedding lookup with scaling: rows of a table (latents shared by Gaussians, per-view embeddings, a vocabulary) by
index, and the table's gradient from the sorted indices (csrc/embedding.cu; checks and autograd node in csrc/host.cpp)."""
import torch

from ._lib import host


def embedding_lookup(table: torch.Tensor, indices: torch.Tensor, scale: float = 1.0, padding_index: int | None = None) -> torch.Tensor:
    """scale * table[indices]: [*indices.shape, *table.shape[1:]], computed in float32 and rounded once to the table's type.

    `table` [rows, ...]: contiguous CUDA float32, bfloat16 or float16; `indices`: int64 or int32 of any shape on the same
    device. A negative index, or `padding_index`, stands for no row: zeros, and no gradient. An index past the table is
    not read: its output is NaN, and it adds to no gradient (nothing is copied to the host to raise an error).

    Differentiable in `table` (once, backward only). The gradient is dense, scale * the sum of the output gradients of
    each row's indices: summed in float32 in an order that depends only on the inputs (and the alignment of the
    gradient's address), so the same inputs give the same bits. Both directions may be captured into CUDA graphs (the
    backward not while an eager graph of the table, made on the default stream, lives: RuntimeError).

    Tracers (torch.jit.trace, torch.fx, torch.export), fake tensors and function transforms are refused (RuntimeError): they
    would not see what the kernels write. torch.compile leaves the call out of its graph."""
    return host().embedding_lookup(table, indices, scale, padding_index)
