"""Rows sorted by expert and back against plain 64-bit implementations."""
import pytest
import torch

from flashoverlap_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):                               # half the distance of the numbers around zero
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def order_ref(ids, experts):
    flat = ids.reshape(-1).tolist()
    rows = [[i for i, e in enumerate(flat) if e == x] for x in range(experts)] if experts <= 16 else None
    if rows is None:
        rows = [[] for _ in range(experts)]
        for i, e in enumerate(flat):
            if 0 <= e < experts:
                rows[e].append(i)
    source = [i for r in rows for i in r]
    slot = [-1] * len(flat)
    for s, i in enumerate(source):
        slot[i] = s
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + len(r))
    return (torch.tensor(slot, dtype=torch.int32).view(ids.shape), torch.tensor(source + [-1] * (len(flat) - len(source)), dtype=torch.int32),
            torch.tensor(offsets, dtype=torch.int32))


# one choice, one warp's step and the next, one CTA's and a cluster's, one expert, as many as there may be, more choices than experts
SHAPES = [(1, 1, 1), (1, 8, 64), (5, 3, 7), (32, 1, 3), (33, 1, 1024), (512, 8, 64), (513, 8, 5), (1000, 5, 1), (9973, 6, 100), (700, 64, 1000),
          (40000, 8, 256)]


@pytest.mark.parametrize("tokens,top_k,experts", SHAPES)
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_sort(cuda, tokens, top_k, experts, kind):
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts + 2, (tokens, top_k), generator=g, dtype=kind)     # some are served elsewhere
    if kind == torch.int64:
        ids[ids == experts] = 1 << 32                                                  # 0 if it lost its upper half
    got = ops.moe_sort(ids.to(cuda), experts)
    for a, b in zip(got, order_ref(ids, experts)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("tokens,top_k,experts", [(33, 1, 1024), (513, 8, 5), (700, 64, 1000), (40000, 8, 256)])
def test_sort_in_smaller_clusters(cuda, tokens, top_k, experts):
    """As on a device, or a part of one, without a place for a cluster of sixteen, or of eight."""
    ids = torch.randint(-1, experts + 2, (tokens, top_k), device=cuda)
    ref = ops.moe_sort(ids, experts)
    for most in (15, 8, 7, 1):
        for a, b in zip(torch.ops.flashoverlap_op.moe_sort(ids, experts, most), ref):
            assert torch.equal(a, b)
    for bad in (0, 17):
        with pytest.raises(RuntimeError):
            torch.ops.flashoverlap_op.moe_sort(ids, experts, bad)


def test_sort_extremes(cuda):
    none = ops.moe_sort(torch.full((50, 4), -1, device=cuda), 9)
    assert (none.slot == -1).all() and (none.source == -1).all() and (none.offsets == 0).all()
    one = ops.moe_sort(torch.full((3000, 4), 8, device=cuda), 9)                       # the same expert, twice a token too
    assert torch.equal(one.slot.view(-1), torch.arange(12000, device=cuda, dtype=torch.int32))
    assert one.offsets.tolist() == [0] * 9 + [12000]
    empty = ops.moe_sort(torch.empty(0, 4, dtype=torch.int32, device=cuda), 9)
    assert empty.slot.shape == (0, 4) and empty.source.numel() == 0 and (empty.offsets == 0).all()
    wide = torch.randint(0, 9, (300, 8), device=cuda)
    for a, b in zip(ops.moe_sort(wide[:, 1::3], 9), ops.moe_sort(wide[:, 1::3].contiguous(), 9)):
        assert torch.equal(a, b)


def _problem(cuda, dt, tokens, top_k, experts, dim, wt=torch.float32, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    ids = torch.randint(0, experts + experts // 3 + 1, (tokens, top_k), device=cuda, generator=g)
    ids[0] = -1                                                                        # a token that nobody here serves
    x = torch.randn(tokens, dim, device=cuda, generator=g).to(dt)
    y = torch.randn(tokens * top_k, dim, device=cuda, generator=g).to(dt)
    w = torch.rand(tokens, top_k, device=cuda, generator=g).to(wt)
    return ops.moe_sort(ids, experts), x, y, w


CASES = [(1, 1, 1, 8), (2, 8, 4, 64), (17, 3, 5, 1032), (300, 10, 16, 264), (65, 64, 300, 72), (1000, 2, 8, 4096), (129, 9, 33, 2056)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("tokens,top_k,experts,dim", CASES)
def test_dispatch(cuda, dt, tokens, top_k, experts, dim):
    order, x, _, _ = _problem(cuda, dt, tokens, top_k, experts, dim)
    rows = int(order.offsets[-1])
    torch.full((tokens * top_k, dim), float("nan"), device=cuda, dtype=dt)             # what the allocator hands out next
    got = ops.moe_dispatch(x, order)
    assert torch.equal(got[:rows], x[order.source[:rows].long() // top_k]) and (got[rows:] == 0).all()


def _combine_ref(y, w, order):
    slot = order.slot.long()
    there = (slot >= 0)[..., None]
    rows = torch.where(there, y.double()[slot.clamp(min=0)], 0.0)
    terms = rows * w.double()[..., None]
    return terms.sum(1), terms.abs().sum(1)


@pytest.mark.parametrize("wt", [torch.float32, None])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("tokens,top_k,experts,dim", CASES)
def test_combine(cuda, dt, wt, tokens, top_k, experts, dim):
    order, _, y, w = _problem(cuda, dt, tokens, top_k, experts, dim, wt or dt)
    y[int(order.offsets[-1]):] = float("nan")                                          # rows without a choice are not looked at
    for weights in (w, None):
        ref, mag = _combine_ref(y, w if weights is not None else torch.ones_like(w), order)
        got = ops.moe_combine(y, weights, order)
        # top_k products and sums in 32 bits, one rounding
        assert ((got.double() - ref).abs() <= half_step(dt) * ref.abs() + (top_k + 1) * 2.0 ** -23 * mag + smallest(dt)).all()
        assert (got[0] == 0).all()


@pytest.mark.parametrize("wt", [torch.float32, None])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("tokens,top_k,experts,dim", CASES)
def test_gradients(cuda, dt, wt, tokens, top_k, experts, dim):
    order, x, y, w = _problem(cuda, dt, tokens, top_k, experts, dim, wt or dt)
    rows = int(order.offsets[-1])
    g_rows, g_out = torch.randn_like(y), torch.randn_like(x)
    g_rows[rows:] = float("nan")                                                       # nobody's: they reach no token
    x, y, w = (v.requires_grad_() for v in (x, y, w))
    gx, = torch.autograd.grad(ops.moe_dispatch(x, order), x, g_rows)
    ref, mag = _combine_ref(g_rows, torch.ones_like(w), order)
    assert gx.dtype == dt and ((gx.double() - ref).abs() <= half_step(dt) * ref.abs() + (top_k + 1) * 2.0 ** -23 * mag + smallest(dt)).all()

    gy, gw = torch.autograd.grad(ops.moe_combine(y, w, order), (y, w), g_out)
    slot = order.slot.long()
    ref = torch.zeros(tokens * top_k, dim, dtype=torch.float64, device=cuda)
    ref[slot[slot >= 0]] = (g_out.double()[:, None] * w.detach().double()[..., None])[slot >= 0]
    # one 32-bit product, one rounding
    assert ((gy.double() - ref).abs() <= (half_step(dt) + 2.0 ** -23) * ref.abs() + smallest(dt)).all() and (gy[rows:] == 0).all()
    terms = g_out.double()[:, None] * y.detach().double()[slot.clamp(min=0)] * (slot >= 0)[..., None]
    ref, mag = terms.sum(-1), terms.abs().sum(-1)
    # at most dim sums in 32 bits, and a rounding where the weights have 16
    own = half_step(w.dtype) if w.dtype != torch.float32 else 0.0
    assert gw.dtype == w.dtype and ((gw.double() - ref).abs() <= own * ref.abs() + (dim + 1) * 2.0 ** -24 * mag + smallest(w.dtype)).all()
    assert (gw[order.slot < 0] == 0).all()
    # one of the two alone
    only, = torch.autograd.grad(ops.moe_combine(y, w.detach(), order), y, g_out)
    assert torch.equal(only, gy)
    only, = torch.autograd.grad(ops.moe_combine(y.detach(), w, order), w, g_out)
    assert torch.equal(only, gw)


def test_gradients_against_differences(cuda):
    """The sum is linear in the rows and in the weights: its change along a direction is the gradient's product with it."""
    order, x, y, w = _problem(cuda, torch.float16, 40, 4, 6, 128)
    leaves = [y.requires_grad_(), w.requires_grad_()]
    g = torch.randn(40, 128, device=cuda).half()
    grads = torch.autograd.grad(ops.moe_combine(y, w, order), leaves, g)
    with torch.no_grad():
        base = ops.moe_combine(y, w, order).double()
        for i, (v, grad) in enumerate(zip(leaves, grads)):
            moved = v + torch.randn_like(v)
            after = (ops.moe_combine(moved, w, order) if i == 0 else ops.moe_combine(y, moved, order)).double()
            step = moved.double() - v.double()
            # outputs and gradients are off by 2^-11 of their values each, their 32-bit sums by far less
            bound = 2.0 ** -10.9 * (((after.abs() + base.abs()) * g.double().abs()).sum() + (grad.double() * step).abs().sum())
            assert (((after - base) * g.double()).sum() - (grad.double() * step).sum()).abs() <= bound


def test_strided_unaligned_and_expanded(cuda):
    order, x, y, w = _problem(cuda, torch.bfloat16, 33, 4, 6, 136)
    mem = torch.empty(33 * 136 + 8, device=cuda, dtype=x.dtype)
    odd = mem[3:3 + 33 * 136].view(33, 136).copy_(x)                                   # 6 bytes past a boundary
    wide = torch.cat([x, x], 1)
    for v in (odd, wide[:, :136], x.t().contiguous().t()):
        assert torch.equal(ops.moe_dispatch(v, order), ops.moe_dispatch(x, order))
    assert torch.equal(ops.moe_combine(y.t().contiguous().t(), w.t().contiguous().t(), order), ops.moe_combine(y, w, order))
    y.requires_grad_()
    g, = torch.autograd.grad(ops.moe_combine(y, w, order).sum(), y)                    # an expanded gradient
    ones, = torch.autograd.grad(ops.moe_combine(y, w, order), y, torch.ones_like(x))
    assert torch.equal(g, ones)


def test_nothing_to_do(cuda):
    order = ops.moe_sort(torch.empty(0, 3, dtype=torch.int64, device=cuda), 4)
    x = torch.empty(0, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    y = torch.empty(0, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    w = torch.empty(0, 3, device=cuda, requires_grad=True)
    rows, out = ops.moe_dispatch(x, order), ops.moe_combine(y, w, order)
    assert rows.shape == (0, 64) and out.shape == (0, 64)
    for g, v in zip(torch.autograd.grad((rows.sum() + out.sum()), (x, y, w)), (x, y, w)):
        assert g.shape == v.shape


def test_an_order_of_something_else_stays_inside_the_matrix(cuda):
    """Rows that are not there are taken as not served: nothing is read or written beyond the rows."""
    order, x, y, w = _problem(cuda, torch.bfloat16, 20, 2, 4, 64)
    bad = order._replace(slot=torch.where(order.slot == 3, 1 << 30, torch.where(order.slot == 5, -7, order.slot)),
                         offsets=order.offsets - 1000)
    kept = (bad.slot >= 0) & (bad.slot < 40)
    ref, _ = _combine_ref(y, w * kept, bad._replace(slot=torch.where(kept, bad.slot, -1)))
    got = ops.moe_combine(y, w, bad)
    assert ((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -20).all()


def _poison(shape, dt, cuda):
    """What the allocator hands out next holds NaN (a row number that is none, read as one)."""
    kept = [torch.full(shape, float("nan"), device=cuda, dtype=dt) for _ in range(4)]
    torch.cuda.synchronize()
    del kept


def _rows_ref(values, order, rows):
    """[rows, dim]: ``values`` [tokens, top_k, dim] at the slots that lie in [0, offsets[-1]), zeros elsewhere."""
    slot, last = order.slot.long(), min(max(int(order.offsets[-1]), 0), rows)
    there = (slot >= 0) & (slot < last)
    ref = torch.zeros(rows, values.shape[-1], dtype=values.dtype, device=values.device)
    ref[slot[there]] = values[there]
    return ref


# one row, a part of what a warp looks after, every size on both sides of 65536 choices, rows of one vector (few warps for many rows)
EDITED = [(1, 1, 1, 8), (3, 2, 2, 64), (128, 8, 16, 264), (205, 5, 7, 1032), (1100, 64, 300, 8), (8192, 8, 64, 72), (8193, 8, 64, 72), (700, 64, 1000, 2056),
          (20000, 9, 33, 8)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("tokens,top_k,experts,dim", EDITED)
@pytest.mark.parametrize("edit", ["dropped", "one", "all", "moved"])
def test_rows_that_an_edited_order_leaves_out_are_zeros(cuda, dt, tokens, top_k, experts, dim, edit):
    """Choices dropped from a sorted order by a -1 in their slots, or rows dealt out anew: a row that no slot names is zeros in the
    dispatch's result and in the gradient of the combine's rows."""
    order, x, y, w = _problem(cuda, dt, tokens, top_k, experts, dim)
    g = torch.Generator(device=cuda).manual_seed(1)
    rows, last = tokens * top_k, int(order.offsets[-1])
    slot = order.slot.clone()
    if edit == "dropped":
        slot[torch.rand(slot.shape, device=cuda, generator=g) < 0.3] = -1
    elif edit == "one":
        slot[slot == last // 2] = -1
    elif edit == "all":
        slot[:] = -1
    else:                                          # other rows than the sort's, whose sources are then others too
        to = torch.cat([torch.randperm(last, device=cuda, generator=g), torch.full((1,), -1, device=cuda)])
        slot = to[slot.long()].to(torch.int32)
        slot[::2, 0] = -1
    order = order._replace(slot=slot)
    # the sort's sources, which tell most, none, some that cannot be taken
    for order in (order, order._replace(source=None), order._replace(source=order.source.long())):
        _poison((rows, dim), dt, cuda)
        assert torch.equal(ops.moe_dispatch(x, order), _rows_ref(x[:, None].expand(-1, top_k, -1), order, rows))
        go = torch.randn(tokens, dim, device=cuda, generator=g).to(dt)
        y.requires_grad_()
        _poison((rows, dim), dt, cuda)
        gy, = torch.autograd.grad(ops.moe_combine(y, w, order), y, go)
        assert torch.equal(gy, _rows_ref((go.float()[:, None] * w[..., None]).to(dt), order, rows))
        y.requires_grad_(False)
        _poison((rows, dim), dt, cuda)
        dr, dw = torch.ops.flashoverlap_op.moe_combine_backward(go, y, w, order.slot, order.offsets, True, True)
        assert torch.equal(dr, gy) and (dw[order.slot < 0] == 0).all()


@pytest.mark.parametrize("tokens,top_k", [(20, 2), (9000, 8)])
def test_an_order_of_something_else_in_both_directions(cuda, tokens, top_k):
    """Slots outside the matrix and offsets outside it: rows with a choice have its token, all others are zeros."""
    order, x, y, w = _problem(cuda, torch.bfloat16, tokens, top_k, 4, 64)
    n = tokens * top_k
    slot = torch.where(order.slot == 3, 1 << 30, torch.where(order.slot == 5, -7, order.slot))
    slot = torch.where(order.slot == 8, n, slot).to(torch.int32)
    kept = (slot >= 0) & (slot < n)
    go = torch.randn(tokens, 64, device=cuda).bfloat16()
    for shift in (0, -3, -(1 << 20), 1 << 30):     # the last ones' rows are not the experts', nobody's are, all are
        bad = order._replace(slot=slot, offsets=order.offsets + shift)
        _poison((n, 64), torch.bfloat16, cuda)
        assert torch.equal(ops.moe_dispatch(x, bad), _rows_ref(x[:, None].expand(-1, top_k, -1), bad, n))
        _poison((n, 64), torch.bfloat16, cuda)
        dr, dw = torch.ops.flashoverlap_op.moe_combine_backward(go, y, w, bad.slot, bad.offsets, True, True)
        assert torch.equal(dr, _rows_ref((go.float()[:, None] * w[..., None]).bfloat16(), bad, n))
        terms = go.double()[:, None] * y.double()[torch.where(kept, slot, 0).long()] * kept[..., None]
        assert ((dw.double() - terms.sum(-1)).abs() <= 65 * 2.0 ** -24 * terms.abs().sum(-1)).all() and (dw[~kept] == 0).all()


def test_rows_beyond_32_bit_offsets(cuda):
    """2.6e9 elements: byte and element offsets pass 32 bits."""
    tokens, top_k, dim = 40000, 8, 8192
    ids = torch.arange(tokens * top_k, device=cuda).view(tokens, top_k) % 64
    order = ops.moe_sort(ids, 64)
    x = torch.randn(tokens, dim, device=cuda).to(torch.bfloat16)
    rows = ops.moe_dispatch(x, order)
    for s in (0, tokens * top_k // 2, tokens * top_k - 1):
        assert torch.equal(rows[s], x[int(order.source[s]) // top_k])
    assert torch.equal(ops.moe_combine(rows, torch.full((tokens, top_k), 0.125, device=cuda), order), x)


def test_replayed_graph_and_another_stream(cuda):
    order, x, y, w = _problem(cuda, torch.bfloat16, 700, 8, 16, 512)
    ids = torch.randint(0, 16, (700, 8), device=cuda)

    def step():
        o = ops.moe_sort(ids, 16)
        rows = ops.moe_dispatch(x, o)
        out = ops.moe_combine(rows, w, o)
        return (*o, rows, out, *torch.ops.flashoverlap_op.moe_combine_backward(out, rows, w, o.slot, o.offsets, True, True))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    side = torch.cuda.Stream()
    for seed in range(3):
        ids.copy_(torch.randint(0, 16, ids.shape, device=cuda))
        x.normal_()
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("tokens", [300, 9000])
def test_choices_dropped_between_replays(cuda, tokens):
    """Two graphs of an order whose slots are edited in place, replayed on two streams at once: every replay goes by the slots as they are."""
    dt, top_k, dim = torch.bfloat16, 8, 128
    order, x, y, w = _problem(cuda, dt, tokens, top_k, 16, dim)
    order = order._replace(slot=order.slot.clone())
    go = torch.randn(tokens, dim, device=cuda).to(dt)

    def step(source):
        return (torch.ops.flashoverlap_op.moe_dispatch(x, order.slot, order.offsets, source),
                *torch.ops.flashoverlap_op.moe_combine_backward(go, y, w, order.slot, order.offsets, True, True, source))

    graphs = []
    for source in (order.source, None):
        step(source)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(source)
        graphs.append((graph, out, torch.cuda.Stream()))
    for _ in range(3):
        order.slot[torch.rand(order.slot.shape, device=cuda) < 0.2] = -1
        torch.cuda.synchronize()
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        rows = _rows_ref(x[:, None].expand(-1, top_k, -1), order, tokens * top_k)
        grad = _rows_ref((go.float()[:, None] * w[..., None]).to(dt), order, tokens * top_k)
        for _, (r, dr, dw), _ in graphs:
            assert torch.equal(r, rows) and torch.equal(dr, grad) and (dw[order.slot < 0] == 0).all()


def test_refuses(cuda):
    order, x, y, w = _problem(cuda, torch.bfloat16, 20, 2, 4, 64)
    ids = torch.zeros(20, 2, dtype=torch.int32, device=cuda)
    for bad, experts in ((ids.cpu(), 4), (ids.float(), 4), (ids.view(-1), 4), (ids, 0), (ids, 1025), (ids[:, :0], 4), (ids.repeat(1, 33), 4)):
        with pytest.raises(RuntimeError):
            ops.moe_sort(bad, experts)
    for bad in (x.cpu(), x.float(), x[:19], x[:, :60], x.view(-1), x.view(20, 8, 8)):
        with pytest.raises(RuntimeError):
            ops.moe_dispatch(bad, order)
    for bad in (y.cpu(), y.float(), y[:39], y[:, :60], y.view(-1)):
        with pytest.raises(RuntimeError):
            ops.moe_combine(bad, w, order)
    for bad in (w.cpu(), w.half(), w.double(), w[:19], w[:, :1], w.view(-1)):
        with pytest.raises(RuntimeError):
            ops.moe_combine(y, bad, order)
    for bad in (order._replace(slot=order.slot.long()), order._replace(slot=order.slot.cpu()), order._replace(slot=order.slot.view(-1)),
                order._replace(slot=order.slot.t())):
        with pytest.raises(RuntimeError):
            ops.moe_combine(y, w, bad)
    for bad in (order.offsets.long(), order.offsets.cpu(), order.offsets[:1], order.offsets[::2]):
        with pytest.raises(RuntimeError):
            ops.moe_dispatch(x, order._replace(offsets=bad))
