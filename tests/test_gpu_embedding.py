"""embedding_lookup and its gradient on the GPU against the formula in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24  # half a float32 step, relative
HALF_STEP = {torch.float32: E32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _np(t):
    return t.detach().double().cpu().numpy()


def _check_rows(out, table, idx, scale, padding=None):
    """The scale's conversion and the product: two float32 roundings, then the type's own."""
    t, i, o = _np(table).reshape(table.shape[0], -1), idx.cpu().numpy().reshape(-1), _np(out)
    o = o.reshape(i.size, t.shape[1])
    none = (i < 0) | (i == (padding if padding is not None else -1))
    bad = i >= t.shape[0]
    assert (o[none] == 0).all() and np.isnan(o[bad & ~none]).all()
    live = ~none & ~bad
    want = scale * t[i[live]]
    err = np.abs(o[live] - want)
    assert (err <= (2.01 * E32 + (0 if out.dtype == torch.float32 else 1.01 * HALF_STEP[out.dtype])) * np.abs(want) + SMALLEST[out.dtype]).all()


def _check_grad(grad, g, idx, scale, padding=None):
    """A row of k tokens: at most k - 1 float32 additions in any order, each off by half a step of a partial sum, which is
    at most the sum of the magnitudes; then the scale's conversion, the product, and the type's own rounding."""
    rows = grad.shape[0]
    i = idx.cpu().numpy().reshape(-1)
    g = _np(g).reshape(i.size, -1)
    live = (i >= 0) & (i < rows) & (i != (padding if padding is not None else -1))
    want, size, count = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1])), np.zeros(rows)
    np.add.at(want, i[live], g[live])
    np.add.at(size, i[live], np.abs(g[live]))
    np.add.at(count, i[live], 1)
    got = _np(grad).reshape(rows, -1)
    assert (got[count == 0] == 0).all()
    err = np.abs(got - scale * want)
    tol = 1.01 * abs(scale) * E32 * np.maximum(count - 1, 0)[:, None] * size
    tol = tol + (2.01 * E32 + (0 if grad.dtype == torch.float32 else 1.01 * HALF_STEP[grad.dtype])) * (np.abs(scale * want) + tol) + SMALLEST[grad.dtype]
    assert (err <= tol).all(), float((err - tol).max())


def _inputs(cuda, rows, width, tokens, dtype, kind, index_type, seed=0):
    r = torch.Generator().manual_seed(seed)
    table = (torch.randn(rows, *width, generator=r) if isinstance(width, tuple) else torch.randn(rows, width, generator=r)).to(dtype).to(cuda)
    if kind == 'even':
        idx = torch.randint(0, rows, (tokens,), generator=r)
    elif kind == 'one':
        idx = torch.full((tokens,), rows - 1)
    elif kind == 'skewed':
        idx = (torch.rand(tokens, generator=r) ** 4 * rows).long().clamp(max=rows - 1)
    else:  # sorted runs, with gaps
        idx = torch.arange(tokens) * rows // max(tokens, 1) // 3 * 3
        idx = idx.clamp(max=rows - 1)
    absent = torch.rand(tokens, generator=r)
    if kind != 'one':
        idx = torch.where(absent < 0.1, -1, idx)
        idx = torch.where(absent > 0.97, rows + (absent * 100).long(), idx)
    g = torch.randn(tokens, *(width if isinstance(width, tuple) else (width,)), generator=r).to(dtype).to(cuda)
    return table, idx.to(index_type).to(cuda), g


# rows, width, tokens: one of each; odd and even widths around the access and lane counts; rows that cross chunks;
# more chunks than one joining CTA looks at; a row longer than one CTA's part
SIZES = [(1, 1, 1), (5, 1, 7), (3, 2, 100), (1000, 3, 1), (17, 4, 33), (9, 5, 2000), (300, 32, 5000), (4096, 45, 3000), (40, 64, 4097), (2, 127, 640),
         (700, 128, 257), (3, 129, 1000), (60, 1000, 300), (11, 4099, 50), (70_000, 8, 9000), (4, (15, 3), 777), (6, 8200, 9)]


@pytest.mark.parametrize('dtype', DTYPES, ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('kind', ['even', 'one', 'skewed', 'runs'])
@pytest.mark.parametrize('size', SIZES, ids=[str(s) for s in SIZES])
def test_lookup_and_gradient(cuda, size, kind, dtype):
    import FasterGSVDACudaBackend as F
    rows, width, tokens = size
    index_type = torch.int64 if tokens % 2 else torch.int32
    table, idx, g = _inputs(cuda, rows, width, tokens, dtype, kind, index_type)
    scale = 1.0 if kind == 'one' else 5.7
    table.requires_grad_(True)
    out = F.embedding_lookup(table, idx, scale=scale)
    assert out.shape == idx.shape + table.shape[1:] and out.dtype == dtype
    _check_rows(out, table, idx, scale)
    out.backward(g)
    assert table.grad.shape == table.shape and table.grad.dtype == dtype
    _check_grad(table.grad, g, idx, scale)
    with torch.no_grad():
        assert torch.equal(F.embedding_lookup(table, idx, scale=scale).nan_to_num(9.0), out.nan_to_num(9.0))


def test_many_tokens_of_few_rows(cuda):
    """Rows over hundreds of chunks, summed by the joining kernel."""
    import FasterGSVDACudaBackend as F
    for rows, width in ((1, 8), (3, 33), (37, 16)):
        table, idx, g = _inputs(cuda, rows, width, 300_001, torch.float32, 'even', torch.int32)
        table.requires_grad_(True)
        F.embedding_lookup(table, idx).backward(g)
        _check_grad(table.grad, g, idx, 1.0)


def test_index_shapes_padding_and_strides(cuda):
    import FasterGSVDACudaBackend as F
    table, idx, g = _inputs(cuda, 50, 24, 210, torch.bfloat16, 'even', torch.int64)
    idx = idx.clamp(max=49).view(6, 35)
    table.requires_grad_(True)
    out = F.embedding_lookup(table, idx.t(), scale=-0.5, padding_index=7)
    assert out.shape == (35, 6, 24)
    _check_rows(out, table, idx.t().contiguous(), -0.5, padding=7)
    # a gradient in another order, and one that is broadcast
    go = g.view(6, 35, 24).transpose(0, 1)
    out.backward(go, retain_graph=True)
    _check_grad(table.grad, go.contiguous(), idx.t().contiguous(), -0.5, padding=7)
    table.grad = None
    out.sum().backward()
    _check_grad(table.grad, torch.ones(35, 6, 24, dtype=torch.bfloat16), idx.t().contiguous(), -0.5, padding=7)
    single = F.embedding_lookup(table.detach(), torch.tensor(3, device=cuda))
    assert single.shape == (24,) and torch.equal(single, table.detach()[3])


def test_odd_addresses(cuda):
    """A table and gradients that start one element past an aligned address take the narrow accesses."""
    import FasterGSVDACudaBackend as F
    for dtype in DTYPES:
        base = torch.randn(1 + 30 * 16, device=cuda).to(dtype)
        table = base[1:].view(30, 16).requires_grad_(True)
        idx = torch.randint(0, 30, (99,), device=cuda)
        out = F.embedding_lookup(table, idx, scale=2.0)
        _check_rows(out, table, idx, 2.0)
        g = torch.randn(1 + 99 * 16, device=cuda).to(dtype)[1:].view(99, 16)
        grad, = torch.autograd.grad(out, table, g)
        _check_grad(grad, g, idx, 2.0)


def test_empty(cuda):
    import FasterGSVDACudaBackend as F
    table = torch.randn(4, 3, device=cuda, requires_grad=True)
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    out = F.embedding_lookup(table, none)
    assert out.shape == (0, 3)
    out.sum().backward()
    assert not table.grad.any()
    table.grad = None
    F.embedding_lookup(table, torch.full((5,), -1, device=cuda)).sum().backward()
    assert not table.grad.any()
    empty = torch.empty(0, 3, device=cuda, requires_grad=True)
    out = F.embedding_lookup(empty, torch.tensor([-1, 0], device=cuda))
    assert (out[0] == 0).all() and out[1].isnan().all()
    out.sum().backward()
    assert empty.grad.shape == (0, 3)
    assert F.embedding_lookup(torch.empty(4, 0, device=cuda), torch.tensor([1], device=cuda)).shape == (1, 0)
    wide = torch.empty(4, 0, device=cuda, requires_grad=True)
    F.embedding_lookup(wide, torch.tensor([1], device=cuda)).sum().backward()


def test_gradient_against_differences(cuda):
    import FasterGSVDACudaBackend as F
    r = torch.Generator().manual_seed(3)
    table = torch.randn(6, 5, generator=r).to(cuda).requires_grad_(True)
    idx = torch.tensor([0, 3, 3, -1, 5, 3, 0], device=cuda)
    w = torch.randn(7, 5, generator=r).to(cuda)
    loss = lambda t: (F.embedding_lookup(t, idx, scale=1.5).double().square() * w.double()).sum()  # noqa: E731
    loss(table).backward()
    step = 2.0 ** -6  # the loss is quadratic: central differences are exact up to the rounding of the rows
    for i in range(6):
        for j in range(5):
            d = torch.zeros_like(table)
            d[i, j] = step
            with torch.no_grad():
                got = float(loss(table + d) - loss(table - d)) / (2 * step)
            # each of the 4 values squared per entry: rows off by 3 roundings of at most 8, over 2 * step
            assert abs(got - float(table.grad[i, j])) <= 4 * 2 * 3 * E32 * 64 * float(w.abs().max()) / step


@pytest.mark.parametrize('dtype', DTYPES, ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('tokens', [65_536, 65_537, 200_000])
def test_around_and_beyond_one_cluster(cuda, tokens, dtype):
    """The longest list that one cluster sorts, the next longer one, and one of several tiles; an odd width; rows in use
    and out of use; absent tokens whose gradients are NaN."""
    import FasterGSVDACudaBackend as F
    for rows, width, kind in ((1000, 7, 'skewed'), (300_000, 4, 'even'), (2, 16, 'even')):
        table, idx, g = _inputs(cuda, rows, width, tokens, dtype, kind, torch.int64)
        g = (g.float() * 0.01).to(dtype)
        g[(idx < 0) | (idx >= rows)] = float('nan')
        table.requires_grad_(True)
        out = F.embedding_lookup(table, idx, scale=0.25)
        _check_rows(out, table, idx, 0.25)
        out.backward(g)
        _check_grad(table.grad, g, idx, 0.25)
        none = torch.full_like(idx, -1)
        none[tokens // 2] = rows - 1
        grad, = torch.autograd.grad(F.embedding_lookup(table, none), table, torch.ones_like(g))
        assert (grad[rows - 1] == 1).all() and not grad[:rows - 1].any()


def test_extreme_indices_and_tables_of_one_dimension(cuda):
    import FasterGSVDACudaBackend as F
    table = torch.randn(9, device=cuda, requires_grad=True)
    idx = torch.tensor([[2 ** 40, -2 ** 40, 8], [0, 2 ** 32 + 1, 9], [-1, 3, 3]], device=cuda)
    out = F.embedding_lookup(table, idx, scale=2.0)
    assert out.shape == (3, 3)
    _check_rows(out.reshape(-1, 1), table.reshape(-1, 1), idx.reshape(-1), 2.0)
    out.nan_to_num().sum().backward()
    want = torch.zeros(9)
    want[8], want[0], want[3] = 2.0, 2.0, 4.0
    assert torch.equal(table.grad.cpu(), want)
    with torch.inference_mode():
        assert torch.equal(F.embedding_lookup(table, idx[2]), torch.stack([table.new_zeros(()), table[3], table[3]]))
    big = torch.tensor([2 ** 31 - 1, -2 ** 31, 4], dtype=torch.int32, device=cuda)
    out = F.embedding_lookup(table.detach(), big)
    assert out[0].isnan() and out[1] == 0 and out[2] == table[4]


def test_more_than_2_31_elements(cuda):
    """A table, an output and a gradient whose offsets pass 32 bits."""
    import FasterGSVDACudaBackend as F
    rows, width = 2 ** 21 + 5, 1032
    table = torch.zeros(rows, width, dtype=torch.bfloat16, device=cuda)
    at = torch.tensor([0, 2 ** 21 - 3, 2 ** 21 + 4, 2 ** 21 + 4, 77], device=cuda)
    r = torch.Generator().manual_seed(0)
    table[at] = torch.randn(5, width, generator=r).bfloat16().to(cuda)
    table.requires_grad_(True)
    out = F.embedding_lookup(table, at, scale=3.0)
    _check_rows(out, table.detach()[at], torch.arange(5), 3.0)
    g = torch.randn(5, width, generator=r).bfloat16().to(cuda)
    grad, = torch.autograd.grad(out, table, g)
    want = torch.zeros(3, width, dtype=torch.float64)
    want[0], want[1], want[2] = g[0].double().cpu(), g[1].double().cpu(), (g[2].double() + g[3].double()).cpu()
    got = grad[at[:3]].double().cpu()
    assert ((got - 3.0 * want).abs() <= 2.0 ** -7 * (3.0 * want).abs() + 2.0 ** -20).all()
    assert int(torch.count_nonzero(grad).item()) == int(torch.count_nonzero(grad[at[[0, 1, 2, 4]]]).item())
    del out, grad
    short = table.detach()[:1000]
    many = torch.arange(2 ** 21 + 5, device=cuda) % 1000
    out = F.embedding_lookup(short, many)
    assert torch.equal(out[-3:], short[many[-3:]]) and torch.equal(out[2 ** 21 - 2], short[many[2 ** 21 - 2]])


def test_same_bits_on_any_stream(cuda):
    import FasterGSVDACudaBackend as F
    table, idx, g = _inputs(cuda, 90, 40, 20_000, torch.float32, 'skewed', torch.int64)
    table.requires_grad_(True)
    first, = torch.autograd.grad(F.embedding_lookup(table, idx), table, g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    grads = []
    for s in streams:  # several calls at once, each with its own workspace
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            grads.append(torch.autograd.grad(F.embedding_lookup(table, idx), table, g)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in grads)


@pytest.mark.parametrize('rows,tokens', [(200, 5000), (200, 70_000), (400_000, 5000)], ids=['short', 'radix passes', 'cleared beside the sort'])
def test_captured_and_replayed(cuda, rows, tokens):
    """Both directions in one graph, replayed on other indices and gradients; a second graph lives beside it."""
    import FasterGSVDACudaBackend as F
    table, idx, g = _inputs(cuda, rows, 48, tokens, torch.bfloat16, 'even', torch.int64)
    table.requires_grad_(True)

    def both():
        out = F.embedding_lookup(table, idx, scale=3.0)
        return out.detach(), torch.autograd.grad(out, table, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both()
        graphs.append((graph, outs))
    for seed, kind in ((1, 'one'), (2, 'skewed')):
        t2, i2, g2 = _inputs(cuda, rows, 48, tokens, torch.bfloat16, kind, torch.int64, seed)
        idx.copy_(i2)
        g.copy_(g2)
        with torch.no_grad():
            table.copy_(t2)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, (out, grad) in graphs:
            _check_rows(out, table, idx, 3.0)
            _check_grad(grad, g, idx, 3.0)


def test_capture_beside_an_eager_graph(cuda):
    """A graph of the table that lives on the default stream: a captured backward is refused, an eager one is not."""
    import FasterGSVDACudaBackend as F
    table, idx, g = _inputs(cuda, 30, 16, 100, torch.float32, 'even', torch.int64)
    table.requires_grad_(True)
    eager = F.embedding_lookup(table, idx)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='release it first'):
        with torch.cuda.graph(graph):
            torch.autograd.grad(F.embedding_lookup(table, idx), table, g)
    torch.cuda.synchronize()
    grad, = torch.autograd.grad(eager, table, g)
    _check_grad(grad, g, idx, 1.0)
    del eager, grad
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad, = torch.autograd.grad(F.embedding_lookup(table, idx), table, g)
    graph.replay()
    torch.cuda.synchronize()
    _check_grad(grad, g, idx, 1.0)


def test_saved_indices(cuda):
    """The backward needs the indices of the forward: a changed or released copy is an error, not another gradient."""
    import FasterGSVDACudaBackend as F
    table = torch.randn(8, 4, device=cuda, requires_grad=True)
    idx = torch.tensor([1, 2, 3], device=cuda)
    out = F.embedding_lookup(table, idx)
    idx += 1
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()
    out = F.embedding_lookup(table, idx)
    out.sum().backward()
    with pytest.raises(RuntimeError, match='second time'):
        out.sum().backward()
    # gradients of several lookups of one table, one of them twice in the graph, add up
    table.grad = None
    a = F.embedding_lookup(table, idx, scale=2.0)
    (a + a * F.embedding_lookup(table, idx[:1])).sum().backward()
    ref = table.detach().double().cpu().requires_grad_(True)
    b = 2.0 * ref[idx.cpu()]
    (b + b * ref[idx[:1].cpu()]).sum().backward()
    # sums and products of a few values: at most 16 roundings of the largest
    assert (table.grad.double().cpu() - ref.grad).abs().max() <= 16 * E32 * ref.grad.abs().max()
    no = F.embedding_lookup(table.detach(), idx)
    assert not no.requires_grad and F.embedding_lookup(table, idx).grad_fn is not None


def test_refusals(cuda):
    import FasterGSVDACudaBackend as F
    table, idx = torch.randn(8, 4, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)
    for bad in (table.t(), table.double(), table.cpu(), torch.tensor(1.0, device=cuda), table.int()):
        with pytest.raises(RuntimeError, match='table'):
            F.embedding_lookup(bad, idx)
    for bad in (idx.cpu(), idx.float(), idx.short(), idx.bool()):
        with pytest.raises(RuntimeError, match='indices'):
            F.embedding_lookup(table, bad)
    for bad in (8, -1):
        with pytest.raises(ValueError, match='padding_index'):
            F.embedding_lookup(table, idx, padding_index=bad)
    table.requires_grad_(True)
    grad, = torch.autograd.grad(F.embedding_lookup(table, idx).sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_forward_mode_is_refused(cuda):
    import FasterGSVDACudaBackend as F
    from torch.autograd import forward_ad
    table, idx = torch.randn(8, 4, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(table, torch.ones_like(table))
        with pytest.raises(RuntimeError, match='forward-mode'):
            F.embedding_lookup(dual, idx)
        assert torch.equal(F.embedding_lookup(table, idx), table[idx])
    with pytest.raises(RuntimeError):  # tensors of a function transform have no memory of their own
        torch.func.vmap(lambda t: F.embedding_lookup(t, idx))(table[None].expand(2, 8, 4).contiguous())


def test_tracers_are_refused(cuda):
    """What a tracer would record, run on other inputs, would give the memory of an allocation: refused in both directions. A
    mode that only watches is none of them."""
    import FasterGSVDACudaBackend as F
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    table, idx, g = _inputs(cuda, 30, 16, 100, torch.float32, 'even', torch.int64)
    for trace in (lambda f: torch.jit.trace(f, (table, idx)), lambda f: make_fx(f)(table, idx), lambda f: make_fx(f, tracing_mode='fake')(table, idx)):
        with pytest.raises(RuntimeError, match='cannot be traced'):
            trace(lambda t, i: F.embedding_lookup(t, i, scale=2.0) + 1.0)
    table.requires_grad_(True)
    out = F.embedding_lookup(table, idx)
    with pytest.raises(RuntimeError, match='cannot be traced'):
        make_fx(lambda x: torch.autograd.grad(out, table, x, retain_graph=True)[0] + 1.0)(g)
    with FlopCounterMode(display=False):
        out = F.embedding_lookup(table, idx, scale=0.5)
        out.backward(g)
    _check_rows(out, table, idx, 0.5)
    _check_grad(table.grad, g, idx, 0.5)


def test_lazily_negated_tensors(cuda):
    """Tensors whose memory holds the negative of their values (torch's views of conjugates' imaginary parts)."""
    import FasterGSVDACudaBackend as F
    table, idx, g = _inputs(cuda, 30, 16, 100, torch.float32, 'even', torch.int64)
    leaf = table.clone().requires_grad_(True)
    out = F.embedding_lookup(torch._neg_view(leaf), torch._neg_view(idx), scale=2.0)
    assert torch._neg_view(idx).is_neg() and torch._neg_view(leaf).is_neg()
    _check_rows(out, -table, -idx, 2.0)
    out.backward(torch._neg_view(g))
    _check_grad(leaf.grad, g, -idx, 2.0)  # negated twice: by the view of the table and by that of the gradient


@pytest.mark.parametrize('index_type', [torch.int64, torch.int32], ids=['int64', 'int32'])
@pytest.mark.parametrize('rows,width', [(200, 4), (4096, 3), (70_001, 1), (300_000, 2)], ids=['one pass', 'two passes', 'three passes', 'three passes, sparse'])
@pytest.mark.parametrize('tokens', [454_656, 454_657, 1_300_001, 2_000_003])
def test_gradients_of_long_lists(cuda, tokens, rows, width, index_type):
    """Lists sorted in tiles of 4, 10, 16 and again 10 keys per thread, by one to three digits, in an even and in a skewed
    order."""
    import FasterGSVDACudaBackend as F
    for kind in ('even', 'skewed'):
        table, idx, g = _inputs(cuda, rows, width, tokens, torch.float32, kind, index_type)
        table.requires_grad_(True)
        out = F.embedding_lookup(table, idx, scale=0.5)
        _check_rows(out, table, idx, 0.5)
        out.backward(g)
        _check_grad(table.grad, g, idx, 0.5)


def test_errors_keep_their_kind(cuda):
    """Out of memory is torch's error for it, and what a hook raises comes through (activation checkpoints stop their second
    forward that way)."""
    import FasterGSVDACudaBackend as F
    table, idx, g = _inputs(cuda, 30, 16, 100, torch.float32, 'even', torch.int64)
    wide = torch.zeros(1, 2 ** 28, device=cuda)
    with pytest.raises(torch.OutOfMemoryError):
        F.embedding_lookup(wide, torch.zeros(4096, dtype=torch.int32, device=cuda))
    table.requires_grad_(True)

    class Stop(Exception):
        pass

    def stop(x):
        raise Stop

    with torch.autograd.graph.saved_tensors_hooks(stop, lambda x: x):
        with pytest.raises(Stop):
            F.embedding_lookup(table, idx)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, stop):
        out = F.embedding_lookup(table, idx)
    with pytest.raises(Stop):
        torch.autograd.grad(out, table, g)
    for reentrant in (False, True):
        out = torch.utils.checkpoint.checkpoint(lambda t: F.embedding_lookup(t, idx, scale=2.0), table, use_reentrant=reentrant)
        table.grad = None
        out.backward(g)
        _check_grad(table.grad, g, idx, 2.0)


def test_hooks_on_the_node_and_on_saved_indices(cuda):
    """What hooks and direct calls hand to the backward is checked before a kernel reads it: sizes, types, devices, orders."""
    import FasterGSVDACudaBackend as F
    table, idx, g = _inputs(cuda, 30, 16, 100, torch.float32, 'even', torch.int64)
    table.requires_grad_(True)
    for spoil in (lambda x: x[:50], lambda x: x[:, :8], lambda x: x.cpu(), lambda x: x.new_empty(0), lambda x: x.to_sparse()):
        out = F.embedding_lookup(table, idx)
        with pytest.raises(RuntimeError, match='gradient of another size or device'):  # torch checks nothing of a direct call
            out.grad_fn(spoil(g))
        out.grad_fn.register_prehook(lambda grads: (spoil(grads[0]),))  # noqa: B023
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, table, g)
    for spoil in (lambda x: x[:50], lambda x: x.short(), lambda x: x.cpu(), lambda x: torch.stack([x, x], 1)[:, 0], lambda x: x.float()):
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, spoil):
            out = F.embedding_lookup(table, idx)
        with pytest.raises(RuntimeError, match='saved indices of embedding_lookup'):
            torch.autograd.grad(out, table, g)
    # and what stays within bounds goes through
    _check_grad(F.embedding_lookup(table, idx).grad_fn(g), g, idx, 1.0)
    out = F.embedding_lookup(table, idx, scale=2.0)
    out.grad_fn.register_prehook(lambda grads: (2.0 * grads[0],))
    _check_grad(torch.autograd.grad(out, table, g)[0], g, idx, 4.0)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x.int(), lambda x: x):
        out = F.embedding_lookup(table, idx)
    _check_grad(torch.autograd.grad(out, table, g)[0], g, idx, 1.0)
    with torch.autograd.graph.save_on_cpu():
        out = F.embedding_lookup(table, idx)
    _check_grad(torch.autograd.grad(out, table, g)[0], g, idx, 1.0)


def test_freed_storages_are_refused(cuda):
    """Tensors whose storage was resized beneath them keep an address and a place within nothing."""
    import FasterGSVDACudaBackend as F
    table, idx, g = _inputs(cuda, 30, 16, 100, torch.float32, 'even', torch.int64)
    table.requires_grad_(True)

    def freed(x, of=lambda x: x):
        flat = torch.cat([x.detach().reshape(-1)] * 2)
        view = of(flat[x.numel():].view(x.shape))
        flat.untyped_storage().resize_((flat.numel() - 1) * x.element_size())
        return view

    with pytest.raises(RuntimeError, match='table has less memory'):
        F.embedding_lookup(freed(table), idx)
    with pytest.raises(RuntimeError, match='indices has less memory'):
        F.embedding_lookup(table, freed(idx))
    with pytest.raises(RuntimeError, match='indices has less memory'):
        F.embedding_lookup(table, freed(torch.stack([idx, idx], 1), lambda x: x[:, 1]))
    out = F.embedding_lookup(table, idx)
    for bad in (freed(g), freed(g.t().contiguous(), torch.t)):
        with pytest.raises(RuntimeError, match='gradient of a lookup has less memory'):
            torch.autograd.grad(out, table, bad, retain_graph=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, freed):
        out = F.embedding_lookup(table, idx)
    with pytest.raises(RuntimeError, match='saved indices has less memory'):
        torch.autograd.grad(out, table, g)
    p = torch.nn.Parameter(torch.ones(8, device=cuda))
    for name in ('grad', 'exp_avg', 'exp_avg_sq'):
        opt = F.FusedAdamW([p])
        p.grad = torch.ones(8, device=cuda)
        opt.step()
        if name == 'grad':
            p.grad = freed(p.grad)
        else:
            opt.state[p][name] = freed(opt.state[p][name])
        with pytest.raises(RuntimeError, match='has less memory'):
            opt.step()
