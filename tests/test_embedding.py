"""embedding_lookup without a GPU: what it and its C entries refuse."""
import ctypes

import pytest
import torch


def test_refuses_host_tensors_and_types():
    import FasterGSVDACudaBackend as F
    with pytest.raises(RuntimeError, match='contiguous CUDA'):
        F.embedding_lookup(torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize('args,match', [
    ((-1, 4, 0, 5, 8, 64), 'dimensions'), ((1 << 31, 4, 0, 5, 8, 64), 'dimensions'), ((4, -1, 0, 5, 8, 64), 'dimensions'),
    ((4, 4, 3, 5, 8, 64), 'dtype'), ((4, 4, 0, -5, 8, 64), 'indices'), ((4, 4, 0, 1 << 31, 8, 64), 'indices'), ((4, 4, 0, 5, 2, 64), 'bytes'),
    ((4, 4, 0, 5, 8, None), 'NULL')])
def test_c_entries_refuse(args, match):
    """Bad shapes, types and pointers come back as an error status with a message, before any launch."""
    from FasterGSVDACudaBackend._lib import lib, check
    rows, width, dtype, n, size, p = args
    with pytest.raises(RuntimeError, match=match):
        check(lib.fgs_embedding_lookup(64, rows, width, dtype, 64, n, size, 1.0, -1, p, None))
    with pytest.raises(RuntimeError, match=match):
        check(lib.fgs_embedding_grad(64, n, size, 64, dtype, rows, width, 1.0, -1, p, 64, 1 << 40, None))


def test_workspace_size():
    from FasterGSVDACudaBackend._lib import lib, check, size_out
    assert 0 < size_out(lib.fgs_embedding_workspace_bytes, 100, 50, 8) < size_out(lib.fgs_embedding_workspace_bytes, 100_000, 50, 8)
    need = size_out(lib.fgs_embedding_workspace_bytes, 100, 50, 8)
    with pytest.raises(RuntimeError, match='workspace'):
        check(lib.fgs_embedding_grad(64, 100, 8, 64, 0, 50, 8, 1.0, -1, 64, 64, need - 1, None))
    with pytest.raises(RuntimeError, match='indices'):
        size_out(lib.fgs_embedding_workspace_bytes, -1, 50, 8)
