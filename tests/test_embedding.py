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


def _trace(kind, f, *args):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    if kind == 'jit.trace':
        return torch.jit.trace(f, args)
    if kind == 'fake':
        with FakeTensorMode(allow_non_fake_inputs=True):
            return f(*args)
    return make_fx(f, tracing_mode=kind)(*args)


@pytest.mark.parametrize('kind', ['jit.trace', 'real', 'fake', 'symbolic'])
def test_tracers_refused(kind):
    """A tracer would record the allocation of the output and none of the kernel's writes to it."""
    import FasterGSVDACudaBackend as F
    table, idx = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match='cannot be traced'):
        _trace(kind, lambda t, i: F.embedding_lookup(t, i) + 1.0, table, idx)


def test_tensors_without_memory_refused():
    """Fake tensors out of their mode, and tensors of function transforms."""
    import FasterGSVDACudaBackend as F
    from torch._subclasses.fake_tensor import FakeTensorMode
    table, idx = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    with FakeTensorMode() as mode:
        fake = mode.from_tensor(table)
    for call in (lambda: F.embedding_lookup(fake, idx), lambda: torch.func.grad(lambda t: F.embedding_lookup(t, idx).sum())(table),
                 lambda: torch.func.vmap(lambda t: F.embedding_lookup(t, idx))(table[None]),
                 lambda: torch.func.functionalize(lambda t: F.embedding_lookup(t, idx))(table)):
        with pytest.raises(RuntimeError, match='plain tensor'):
            call()


def test_dependent_kernels_promise_nothing_about_what_they_read():
    """A kernel that may start before its predecessor has ended must not declare what it reads const and __restrict__: that
    lets the compiler move the read in front of the wait."""
    import re
    from pathlib import Path
    csrc = Path(__file__).resolve().parent.parent / 'efficient-gaussian-appearance_b200' / 'csrc'
    dependent = {}
    for source in csrc.glob('*.cu'):
        for kernel in source.read_text().split('__global__')[1:]:
            head, _, body = kernel.partition(') {')
            body = body.split('\n}\n')[0]
            if 'wait_dependency()' in body:
                name = re.search(r'(\w+_kernel|radix_\w+)\(', head).group(1)
                dependent[name] = re.findall(r'const [\w: <>]+\*\s*__restrict__\s+(\w+)', head)
    assert {'radix_downsweep', 'radix_row_scan', 'clip_kernel', 'sum_kernel', 'join_kernel', 'clear_kernel', 'adamw_kernel'} <= set(dependent)
    assert not any(dependent.values()), dependent


@pytest.mark.parametrize('place', [{'table': 66}, {'out': 65}, {'indices': 68}, {'workspace': 72}])
def test_c_entries_refuse_misaligned_pointers(place):
    """A kernel would fault on an address that is no multiple of its elements' size."""
    from FasterGSVDACudaBackend._lib import lib, check
    a = {'table': 64, 'out': 64, 'indices': 64, 'workspace': 64, **place}
    with pytest.raises(RuntimeError, match='aligned'):
        check(lib.fgs_embedding_grad(a['indices'], 5, 8, a['table'], 0, 4, 4, 1.0, -1, a['out'], a['workspace'], 1 << 40, None))
    if 'workspace' not in place:
        with pytest.raises(RuntimeError, match='aligned'):
            check(lib.fgs_embedding_lookup(a['table'], 4, 4, 0, a['indices'], 5, 8, 1.0, -1, a['out'], None))
