"""The operators around a mixture-of-experts block as they are used together: one forward pass in 8 bits, a training step,
and what recording a gradient asks of them."""
import pytest
import torch
import torch.nn.functional as F

from flashoverlap_b200 import ops

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def impl(cuda):
    i = ops.OverlapImpl()
    i.nccl_init(0, 1, [0] * 16)
    return i


def _weights(cuda, experts, n, k):
    q = torch.randint(-127, 128, (experts, n, k), device=cuda, dtype=torch.int8)
    return q, (0.5 + torch.rand(experts, n, device=cuda)) * (1.5 / (73 * k ** 0.5))


def _norm(v):
    return v / (v.square().mean(-1, keepdim=True) + EPS).sqrt()


def _off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


# a decode batch, a ragged chunk, experts without a token, a token without an expert here
@pytest.mark.parametrize("tokens,top_k,experts,here", [(1, 2, 8, 8), (16, 8, 64, 64), (517, 3, 20, 7)])
def test_block_in_8_bits(cuda, impl, tokens, top_k, experts, here):
    """norm, rows by expert, SwiGLU experts in 8 bits, back with the router's weights, norm, gate, residual, next norm."""
    dt, hidden, ffn = torch.bfloat16, 1024, 512
    torch.manual_seed(tokens)
    x = torch.randn(tokens, hidden, device=cuda).to(dt)
    pre, post, nxt = ((1 + 0.1 * torch.randn(hidden, device=cuda)).to(dt) for _ in range(3))
    gate = (0.5 + 0.1 * torch.randn(hidden, device=cuda)).to(dt)
    w1, s1 = _weights(cuda, here, 2 * ffn, hidden)
    w2, s2 = _weights(cuda, here, hidden, ffn)
    router = torch.randn(experts, hidden, device=cuda).to(dt) * 0.05

    z = ops.rmsnorm(x, pre, EPS)
    best, ids = (z @ router.t()).float().topk(top_k, dim=1)
    weights = best.softmax(1)
    order = ops.moe_sort(ids, here)
    rows = ops.moe_dispatch(z, order)
    gu = ops.linear_i8(impl, rows, w1, s1, order.offsets)
    act = torch.empty(tokens * top_k, ffn, device=cuda, dtype=dt)
    torch.ops.flashoverlap_op.swiglu(gu, act)
    y = ops.linear_i8(impl, act, w2, s2, order.offsets)
    t = ops.moe_combine(y, weights, order)
    h, out = ops.rmsnorm_add_rmsnorm(x, t, post, nxt, gate, 1.0, EPS)
    impl.check_status()

    # the same in 64 bits from the same normed tokens and choices, weights as they are stored
    zd, ref_t = z.double(), torch.zeros(tokens, hidden, dtype=torch.float64, device=cuda)
    for e in range(here):
        token, k = (ids == e).nonzero(as_tuple=True)
        if len(token):
            g, u = (zd[token] @ (w1[e].double() * s1[e].double()[:, None]).t()).split(ffn, 1)
            ref_t.index_add_(0, token, weights.double()[token, k][:, None] * ((F.silu(g) * u) @ (w2[e].double() * s2[e].double()[:, None]).t()))
    # activations in 8 bits are off by up to half of 1 / 127 of a row's largest (about 4 of its root mean square), uniformly:
    # 4 / 254 / sqrt(3) = 0.9 % for each of three products that they pass through, roundings to bf16 beside that
    assert _off(t, ref_t) <= 3 * 4 / 254 / 3 ** 0.5 + 2 ** -7
    ref_h = x.double() + gate.double() * _norm(t.double()) * post.double()
    assert _off(h, ref_h) <= 2 ** -8 and _off(out, _norm(ref_h) * nxt.double()) <= 2 ** -8


def _step(x, ids, experts, leaves):
    """A block with 16-bit experts: dispatch, one product for every expert, combine, norms."""
    weights, post, nxt, gate, logits = leaves
    order = ops.moe_sort(ids, experts)
    rows = ops.moe_dispatch(x, order)
    y = torch.bmm(rows.view(experts, -1, rows.shape[1]), weights).view(rows.shape)
    t = ops.moe_combine(y, logits.softmax(1), order)
    return ops.rmsnorm_add_rmsnorm(x, t, post, nxt, gate, 0.8, EPS)


def _problem(cuda, tokens=96, top_k=2, experts=4, hidden=256):
    """Every expert gets the same number of rows, so that the products are one batched one."""
    torch.manual_seed(5)
    ids = torch.arange(tokens * top_k).view(tokens, top_k) % experts
    dt = torch.bfloat16
    r = lambda *s: torch.randn(*s, device=cuda)
    x = r(tokens, hidden).to(dt)
    leaves = [(r(experts, hidden, hidden) / hidden ** 0.5).to(dt), (1 + 0.1 * r(hidden)).to(dt), (1 + 0.1 * r(hidden)).to(dt),
              (0.5 + 0.1 * r(hidden)).to(dt), r(tokens, top_k)]
    return x, ids.to(cuda), experts, leaves, (r(tokens, hidden).to(dt), r(tokens, hidden).to(dt))


def _reference(x, ids, experts, leaves, gs):
    x, leaves = x.double().requires_grad_(), [v.double().requires_grad_() for v in leaves]
    weights, post, nxt, gate, logits = leaves
    p = logits.softmax(1)
    t = torch.zeros_like(x)
    for e in range(experts):
        token, k = (ids == e).nonzero(as_tuple=True)
        t = t.index_add(0, token, p[token, k][:, None] * (x[token] @ weights[e]))
    h = 0.8 * x + gate * _norm(t) * post
    return torch.autograd.grad((h, _norm(h) * nxt), [x, *leaves], [g.double() for g in gs])


def test_training_step(cuda):
    x, ids, experts, leaves, gs = _problem(cuda)
    ref = _reference(x, ids, experts, leaves, gs)
    x, leaves = x.requires_grad_(), [v.requires_grad_() for v in leaves]
    got = torch.autograd.grad(_step(x, ids, experts, leaves), [x, *leaves], gs)
    for a, b, v in zip(got, ref, [x, *leaves]):
        assert a.dtype == v.dtype
        # five roundings to bf16 follow one another (rows, products, their sum, and back), each 2^-9 of the value at most,
        # and the norm behind small sums raises them by a factor of two or so
        assert _off(a, b) <= 2 * 5 * 2 ** -8


def test_training_step_captured(cuda):
    x, ids, experts, leaves, gs = _problem(cuda)
    x, leaves = x.requires_grad_(), [v.requires_grad_() for v in leaves]

    def step():
        return torch.autograd.grad(_step(x, ids, experts, leaves), [x, *leaves], gs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(2):
        with torch.no_grad():
            x.normal_()
            ids.copy_(ids.flip(0))
        graph.replay()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_capture_refuses_leaves_of_a_live_graph(cuda):
    """With a graph of the same leaf alive elsewhere, a captured backward pass would end the process; the call says so."""
    x = torch.randn(8, 64, device=cuda).to(torch.bfloat16).requires_grad_()
    w = torch.ones(64, device=cuda, dtype=torch.bfloat16)
    order = ops.moe_sort(torch.zeros(8, 1, dtype=torch.int32, device=cuda), 1)
    alive = ops.moe_dispatch(x, order)
    logits = torch.ones(8, 1, device=cuda)
    for call in (lambda: ops.moe_dispatch(x, order), lambda: ops.moe_combine(x, logits, order), lambda: ops.rmsnorm_add_rmsnorm(x, x, w, w)):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="live graph"):
            with torch.cuda.graph(graph):
                call()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g, = torch.autograd.grad(ops.moe_dispatch(x, order), x, torch.ones_like(x))
    graph.replay()
    assert (g == 1).all()


def test_no_second_derivative(cuda):
    x = torch.randn(8, 64, device=cuda).to(torch.bfloat16).requires_grad_()
    w = torch.ones(64, device=cuda, dtype=torch.bfloat16)
    order = ops.moe_sort(torch.zeros(8, 1, dtype=torch.int32, device=cuda), 1)
    for out in (ops.moe_dispatch(x, order), ops.moe_combine(x, torch.ones(8, 1, device=cuda), order), ops.rmsnorm_add_rmsnorm(x, x, w, w)[1]):
        g, = torch.autograd.grad(out.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            g.sum().backward()


def test_inputs_changed_before_the_backward_pass(cuda):
    x = torch.randn(8, 64, device=cuda).to(torch.bfloat16)
    w = torch.ones(64, device=cuda, dtype=torch.bfloat16).requires_grad_()
    h, y = ops.rmsnorm_add_rmsnorm(x, x, w, w)
    x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_8_bit_objects_are_made_before_a_capture(cuda):
    fresh = ops.OverlapImpl()
    a, s = torch.zeros(8, 64, device=cuda, dtype=torch.int8), torch.ones(8, device=cuda)
    c = torch.empty(8, 8, device=cuda, dtype=torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(graph):
            fresh.gemm_i8(a, a, s, s, c, None)
    fresh.gemm_i8(a, a, s, s, c, None)
    fresh.check_status()
    assert (c == 0).all()


def test_other_derivatives_are_refused_not_lost(cuda):
    """Forward-mode derivatives raise, and what torch.func makes of the operators is right or raises; nothing comes back without
    its derivative."""
    import torch.autograd.forward_ad as fwd
    impl = ops.OverlapImpl()
    impl.nccl_init(0, 1, [0] * 16)
    x, t = (torch.randn(8, 64, device=cuda).bfloat16() for _ in range(2))
    w, sb = torch.ones(64, device=cuda).bfloat16(), torch.ones(64, device=cuda)
    b = torch.ones(64, 64, device=cuda, dtype=torch.int8)
    order = ops.moe_sort(torch.zeros(8, 2, dtype=torch.int32, device=cuda), 4)
    calls = (lambda a: ops.rmsnorm_add_rmsnorm(a, t, w, w)[1], lambda a: ops.rmsnorm_add_rmsnorm(x, a, w, w, w)[0],
             lambda a: ops.moe_dispatch(a, order), lambda a: ops.moe_combine(torch.cat([a, a]), None, order),
             lambda a: ops.quantize_rows(a)[1], lambda a: ops.linear_i8(impl, a, b, sb))
    for f in calls:
        with fwd.dual_level():
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    f(fwd.make_dual(x, x))
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (x,))
        try:
            each = torch.func.vmap(f)(torch.stack([x, t]))
        except RuntimeError:
            pass
        else:
            assert torch.equal(each, torch.stack([f(x), f(t)]))
        try:
            grad = torch.func.grad(lambda v: f(v).float().sum())(x)
        except RuntimeError:
            pass
        else:
            v = x.detach().requires_grad_()
            f(v).float().sum().backward()
            assert torch.equal(grad, v.grad)
    weights = torch.rand(8, 2, device=cuda)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ops.moe_combine(torch.cat([x, x]), fwd.make_dual(weights, weights), order)
