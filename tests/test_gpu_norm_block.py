"""The norms around a block and their gradients against a plain 64-bit implementation."""
import pytest
import torch

from flashoverlap_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
EPS = 1e-5


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def reference(x, t, pw, w, gate, alpha, gh=None, gy=None):
    """{name: (value, magnitude of what is added up to it)} in 64 bits."""
    x, t, pw, w = (v.double() for v in (x, t, pw, w))
    rows, dim = x.shape
    lines = 1 if gate is None else gate.numel() // dim
    g = torch.ones(1, dim, dtype=torch.float64, device=x.device) if gate is None else gate.double().view(lines, dim)
    g = g.repeat_interleave(rows // lines, 0)
    mean = lambda v: v.mean(1, keepdim=True)
    n1 = t / (mean(t * t) + EPS).sqrt()
    r1 = 1 / (mean(t * t) + EPS).sqrt()
    h = alpha * x + g * n1 * pw
    hm = (alpha * x).abs() + (g * n1 * pw).abs()
    r2 = 1 / (mean(h * h) + EPS).sqrt()
    n2, n2m = h * r2, hm * r2
    out = {"h": (h, hm), "y": (n2 * w, n2m * w.abs())}
    if gh is None and gy is None:
        return out
    zero = torch.zeros_like(x)
    gh, gy = (zero if v is None else v.double() for v in (gh, gy))
    a = gy * w
    dh = gh + r2 * (a - n2 * mean(a * n2))
    dhm = gh.abs() + r2 * (a.abs() + n2m * mean(a.abs() * n2m))
    b, bm = dh * g * pw, dhm * (g * pw).abs()
    out["x"] = (alpha * dh, abs(alpha) * dhm)
    out["t"] = (r1 * (b - n1 * mean(b * n1)), r1 * (bm + n1.abs() * mean(bm * n1.abs())))
    out["pw"] = ((dh * g * n1).sum(0), (dhm * (g * n1).abs()).sum(0))
    out["w"] = ((gy * n2).sum(0), (gy.abs() * n2m).sum(0))
    if gate is not None:
        part = lambda v: v.view(lines, rows // lines, dim).sum(1).view(gate.shape)
        out["gate"] = (part(dh * n1 * pw), part(dhm * (n1 * pw).abs()))
    return out


def check(name, got, ref, dt, rows):
    value, mag = ref
    # a row's sums have at most dim / threads + 16 <= 48 terms one after the other, 1 / sqrt is within 2 units, and about
    # twenty more 32-bit operations follow one another: 2^-16 of what is added up; a column's sum has up to `rows` terms more
    loose = 2.0 ** -16 + (rows * 2.0 ** -24 if name in ("pw", "w", "gate") else 0.0)
    bound = half_step(dt) * value.abs() * (1 + loose) + loose * mag + smallest(dt)
    assert got.dtype == dt and got.shape == value.shape
    off = (got.double() - value).abs() - bound
    assert (off <= 0).all(), (name, float(off.max()), float(value.abs().max()))


def problem(cuda, dt, rows, dim, gate, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=cuda, generator=g)
    lines = {None: 0, "channel": 1, "row": rows}.get(gate, gate)
    gate = (0.5 + r(lines, dim)).to(dt) if lines else None
    return [(2 * r(rows, dim)).to(dt), (0.3 * r(rows, dim)).to(dt), (1 + 0.2 * r(dim)).to(dt), (1 + 0.2 * r(dim)).to(dt), gate,
            r(rows, dim).to(dt), r(rows, dim).to(dt)]


# one vector, a part of a warp, every number of vectors a thread, its first and last sizes; one row, fewer and more than CTAs
SHAPES = [(1, 8, None), (3, 8, 3), (130, 72, "channel"), (7, 2048, 7), (200, 2056, 2), (5000, 264, 8), (3000, 1024, 1500), (1200, 4104, "channel"),
          (33, 8192, None), (600, 8200, 3), (12, 16384, "row"), (301, 16384, "channel"), (2, 4096, 2), (20000, 16, 4), (1, 16384, "channel"),
          # lines that CTAs share: fewer lines than CTAs, more, and both for rows that a cluster shares; lines that are one CTA's
          (1024, 8192, 64), (1600, 8192, 200), (9000, 1032, 900), (600, 9000, 30), (1000, 16384, 125), (2072, 8192, 148)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,dim,gate", SHAPES)
def test_forward(cuda, dt, rows, dim, gate):
    x, t, pw, w, gv, _, _ = problem(cuda, dt, rows, dim, gate)
    for alpha in (1.0, 0.3):
        ref = reference(x, t, pw, w, gv, alpha)
        for name, got in zip("hy", ops.rmsnorm_add_rmsnorm(x, t, pw, w, gv, alpha, EPS)):
            check(name, got, ref[name], dt, rows)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,dim,gate", SHAPES)
def test_gradients(cuda, dt, rows, dim, gate):
    x, t, pw, w, gv, gh, gy = problem(cuda, dt, rows, dim, gate)
    names = ["x", "t", "pw", "w"] + (["gate"] if gv is not None else [])
    leaves = [v.requires_grad_() for v in (x, t, pw, w, gv) if v is not None]
    h, y = ops.rmsnorm_add_rmsnorm(x, t, pw, w, gv, 0.7, EPS)
    plain = ops.rmsnorm_add_rmsnorm(*[None if v is None else v.detach() for v in (x, t, pw, w, gv)], 0.7, EPS)
    assert torch.equal(h, plain[0]) and torch.equal(y, plain[1])
    detached = [None if v is None else v.detach() for v in (x, t, pw, w, gv)]
    for a, b in ((gh, gy), (None, gy), (gh, None)):
        outs, grads = zip(*[(o, g) for o, g in ((h, a), (y, b)) if g is not None])
        got = torch.autograd.grad(outs, leaves, grads, retain_graph=True)
        ref = reference(*detached, 0.7, a, b)
        for name, v in zip(names, got):
            check(name, v, ref[name], dt, rows)


def test_gradients_against_differences(cuda):
    """Along random directions, in steps that 11 bits resolve: the change of <gh, h> + <gy, y> against the gradients."""
    dt = torch.float16
    x, t, pw, w, gv, gh, gy = problem(cuda, dt, 24, 512, 6)
    leaves = [v.requires_grad_() for v in (x, t, pw, w, gv)]
    grads = torch.autograd.grad(ops.rmsnorm_add_rmsnorm(*leaves, 1.0, EPS), leaves, (gh, gy))

    def f(*v):
        r = reference(*v, 1.0)
        return float((r["h"][0] * gh.double()).sum() + (r["y"][0] * gy.double()).sum())

    for i, (v, g) in enumerate(zip(leaves, grads)):
        d = torch.randn(v.shape, device=cuda, dtype=torch.float64)
        # central differences of the 64-bit function: truncation of the order of the step's square
        at = lambda s: f(*[u.detach().double() + s * d if j == i else u.detach().double() for j, u in enumerate(leaves)])
        slope = (at(1e-4) - at(-1e-4)) / 2e-4
        # the gradient's roundings, half a step of 2^-11 each, in the direction's sum
        bound = 2.0 ** -11 * float((g.double().abs() * d.abs()).sum()) + 1e-5 * abs(slope) + 1e-4
        assert abs(float((g.double() * d).sum()) - slope) <= bound, i


def test_some_gradients_only(cuda):
    x, t, pw, w, gv, gh, gy = problem(cuda, torch.bfloat16, 64, 256, 4)
    every = [v.detach().clone().requires_grad_() for v in (x, t, pw, w, gv)]
    full = torch.autograd.grad(ops.rmsnorm_add_rmsnorm(*every), every, (gh, gy))
    for i in range(5):
        vs = [v.detach() for v in (x, t, pw, w, gv)]
        vs[i] = vs[i].clone().requires_grad_()
        only, = torch.autograd.grad(ops.rmsnorm_add_rmsnorm(*vs), vs[i], (gh, gy))
        assert torch.equal(only, full[i])


def test_a_gate_line_for_all_rows_is_a_channel_gate(cuda):
    x, t, pw, w, gv, _, _ = problem(cuda, torch.bfloat16, 40, 128, "channel")
    for a, b in zip(ops.rmsnorm_add_rmsnorm(x, t, pw, w, gv.view(-1)), ops.rmsnorm_add_rmsnorm(x, t, pw, w, gv)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_of_zeros_and_of_what_is_no_number(cuda, dt):
    x, t, pw, w, gv, _, _ = problem(cuda, dt, 6, 64, None)
    x[0], t[0] = 0, 0
    t[1, 5] = float("nan")
    x[2, 7] = float("inf")
    h, y = ops.rmsnorm_add_rmsnorm(x, t, pw, w)
    assert (h[0] == 0).all() and (y[0] == 0).all()
    assert h[1].isnan().all() and y[1].isnan().all()
    assert h[2, 7].isinf() and y[2, 7].isnan() and (y[2, :7] == 0).all()
    ref = reference(x[3:], t[3:], pw, w, None, 1.0)
    for name, got in (("h", h[3:]), ("y", y[3:])):
        check(name, got, ref[name], dt, 3)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 64), (40, 1032), (20, 8192), (5, 9000)])
def test_rows_whose_parts_cancel(cuda, dt, rows, dim):
    """The residual stream undoes the block's output up to what is left of roundings, in every second row."""
    x, t, pw, w, gv, gh, gy = problem(cuda, dt, rows, dim, "channel")
    u = reference(torch.zeros_like(x), t, pw, w, gv, 1.0)["h"][0]
    x[::2] = (-u / 0.7).to(dt)[::2]
    leaves = [v.requires_grad_() for v in (x, t, pw, w, gv)]
    h, y = ops.rmsnorm_add_rmsnorm(*leaves, 0.7, EPS)
    detached = [v.detach() for v in leaves]
    ref = reference(*detached, 0.7, gh, gy)
    check("h", h, ref["h"], dt, rows)
    # 2^-16 of the parts are off in H, and so in its mean square: up to that over H's root mean square, relative, in Y
    value, (_, hm) = ref["y"][0], ref["h"]
    rms = ref["h"][0].square().mean(1, keepdim=True).add(EPS).sqrt()
    off = 2.0 ** -16 * (hm / rms * w.double().abs() + value.abs() * (hm.square().mean(1, keepdim=True).sqrt() / rms))
    assert ((y.double() - value).abs() <= half_step(dt) * value.abs() + off + smallest(dt)).all()
    for g in torch.autograd.grad((h, y), leaves, (gh, gy)):
        assert g.isfinite().all()


def test_values_that_only_their_norm_brings_into_range(cuda):
    """Squares of T fit 32 bits, squares of T with the weights do not."""
    dt = torch.bfloat16
    x, t, pw, w, gv, gh, gy = problem(cuda, dt, 12, 2048, "channel")
    t, gv = t * 1e16, gv * 3e3
    t[3], t[4] = t[3] * 1e20, 0                     # beyond 32 bits when squared: no part of the block is left, as in 32 bits throughout
    ref = reference(x, t, pw, w, gv, 1.0)
    h, y = ops.rmsnorm_add_rmsnorm(x, t, pw, w, gv, 1.0, EPS)
    rows = [r for r in range(12) if r != 3]
    for name, got in (("h", h), ("y", y)):
        check(name, got[rows], tuple(v[rows] for v in ref[name]), dt, 12)
    assert torch.equal(h[3], x[3])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,dim,gate", [(1, 64, "channel"), (40, 1032, "channel"), (20, 8192, "channel"), (5, 9000, "channel"), (40, 1032, "row"),
                                           (64, 256, 4), (40, 1032, None), (12, 9000, "row")])
def test_gradients_of_rows_whose_parts_cancel(cuda, dt, rows, dim, gate):
    """H is what is left of roundings in every second row, and 1 / rms of it large: gradients within what 32 bits leave of H."""
    x, t, pw, w, gv, gh, gy = problem(cuda, dt, rows, dim, gate)
    u = reference(torch.zeros_like(x), t, pw, w, gv, 1.0)["h"][0]
    x[::2] = (-u / 0.7).to(dt)[::2]
    inputs = (x, t, pw, w, gv)
    names = ["x", "t", "pw", "w"] + (["gate"] if gv is not None else [])
    leaves = [v.requires_grad_() for v in inputs if v is not None]
    h, y = ops.rmsnorm_add_rmsnorm(*inputs, 0.7, EPS)
    detached = [None if v is None else v.detach() for v in inputs]
    xd, td, pwd, wd = (v.double() for v in detached[:4])
    lines = 1 if gv is None else gv.numel() // dim
    g = torch.ones(1, dim, dtype=torch.float64, device=cuda) if gv is None else detached[4].double().view(lines, dim)
    g = g.repeat_interleave(rows // lines, 0)
    mean = lambda v: v.mean(1, keepdim=True)
    r1 = 1 / (mean(td * td) + EPS).sqrt()
    n1, pg = td * r1, pwd * g
    hd, hm = 0.7 * xd + n1 * pg, (0.7 * xd).abs() + (n1 * pg).abs()
    r2 = 1 / (mean(hd * hd) + EPS).sqrt()
    n2 = hd * r2
    few = 2.0 ** -16                               # of what is added up, as in check()
    for a_gh, a_gy in ((gh, gy), (None, gy), (gh, None)):
        outs, grads = zip(*[(o, v) for o, v in ((h, a_gh), (y, a_gy)) if v is not None])
        got = dict(zip(names, torch.autograd.grad(outs, leaves, grads, retain_graph=True)))
        ref = reference(*detached, 0.7, a_gh, a_gy)
        zero = torch.zeros_like(xd)
        ghd, gyd = (zero if v is None else v.double() for v in (a_gh, a_gy))
        a = (gyd * wd).abs()
        # H is off by `few` of its parts, its mean square by twice the mean of |H| times that, so 1 / rms relatively by
        # few * rms(parts) / rms(H), and n2 = H / rms by both
        off_r2 = few * mean(hm * hm).sqrt() * r2
        off_n2 = few * hm * r2 + n2.abs() * off_r2
        # dH = gh + r2 (a - n2 mean(a n2)): every factor's error times the others
        c2 = mean(a * n2.abs())
        off_c2 = mean(a * off_n2) + few * c2
        off_dh = few * ghd.abs() + (few + off_r2) * r2 * (a + n2.abs() * c2) + r2 * (off_n2 * c2 + n2.abs() * off_c2)
        dh = ref["x"][0] / 0.7
        # the second mean, of dH G PW n1, is made of sums of dH's parts: those errors once for dH and once for the sums
        off_c1 = 2 * mean(off_dh * (n1 * pg).abs())
        b = (dh * pg).abs()
        off_t = r1 * (off_dh * pg.abs() + n1.abs() * off_c1 + few * (b + n1.abs() * mean(b * n1.abs())))
        column = few + rows * 2.0 ** -24           # and a column's sum has up to `rows` terms
        off = {"x": 0.7 * off_dh, "t": off_t, "w": (gyd.abs() * off_n2 + column * (gyd * n2).abs()).sum(0),
               "pw": ((off_dh + column * dh.abs()) * (g * n1).abs()).sum(0)}
        if gv is not None:
            off["gate"] = ((off_dh + column * dh.abs()) * (pwd * n1).abs()).view(lines, rows // lines, dim).sum(1).view(gv.shape)
        for name, v in got.items():
            value = ref[name][0]
            assert ((v.double() - value).abs() <= half_step(dt) * value.abs() + 1.01 * off[name] + smallest(dt)).all(), (
                name, float(((v.double() - value).abs() - half_step(dt) * value.abs()).max()), float(off[name].max()))
            # The bound would see a term that is missing or has the wrong sign.  (What is left in H is about 2^-9 (bf16) or 2^-12 (fp16) of
            # its parts, of which 2^-16 are 2^-7 or 2^-4 of H; each gradient has that in from two to four factors.)
            assert float(off[name].norm()) <= 0.5 * float(value.norm())


@pytest.mark.parametrize("gate", ["channel", "row"])
def test_gradients_of_values_that_only_their_norm_brings_into_range(cuda, gate):
    dt = torch.bfloat16
    x, t, pw, w, gv, gh, gy = problem(cuda, dt, 12, 2048, gate)
    t, gv = t * 1e16, gv * 3e3
    t[3], t[4] = t[3] * 1e20, 0
    leaves = [v.requires_grad_() for v in (x, t, pw, w, gv)]
    got = torch.autograd.grad(ops.rmsnorm_add_rmsnorm(*leaves, 1.0, EPS), leaves, (gh, gy))
    detached = [v.detach().clone() for v in leaves]
    detached[1][3] = 0                             # squares beyond 32 bits: as in the forward pass, nothing is left of the row's block
    ref = reference(*detached, 1.0, gh, gy)
    rows = [r for r in range(12) if r != 3]
    for name, v in zip(("x", "t", "pw", "w", "gate"), got):
        if name == "t":
            assert (v[3] == 0).all()
            check(name, v[rows], tuple(u[rows] for u in ref[name]), dt, 12)
        else:
            check(name, v, ref[name], dt, 12)


def test_nothing_to_do(cuda):
    x, t, pw, w, gv, _, _ = problem(cuda, torch.bfloat16, 0, 64, "channel")
    leaves = [v.requires_grad_() for v in (x, t, pw, w, gv)]
    h, y = ops.rmsnorm_add_rmsnorm(*leaves)
    grads = torch.autograd.grad(h.sum() + y.sum(), leaves)
    assert h.shape == y.shape == (0, 64) and all((g == 0).all() and g.shape == v.shape for g, v in zip(grads, leaves))


def test_strided_unaligned_and_expanded(cuda):
    x, t, pw, w, gv, gh, gy = problem(cuda, torch.float16, 24, 136, 4)
    ref = ops.rmsnorm_add_rmsnorm(x, t, pw, w, gv)
    mem = torch.empty(24 * 136 + 8, device=cuda, dtype=x.dtype)
    odd = mem[1:1 + 24 * 136].view(24, 136).copy_(t)
    for got in (ops.rmsnorm_add_rmsnorm(x.t().contiguous().t(), odd, pw, w, gv),
                ops.rmsnorm_add_rmsnorm(torch.cat([x, x], 1)[:, 136:], t, torch.stack([pw, pw], 1)[:, 0], w, gv)):
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    x.requires_grad_()
    a, = torch.autograd.grad(ops.rmsnorm_add_rmsnorm(x, t, pw, w, gv)[1].sum(), x)
    b, = torch.autograd.grad(ops.rmsnorm_add_rmsnorm(x, t, pw, w, gv)[1], x, torch.ones_like(t))
    assert torch.equal(a, b)


def test_replayed_graph_and_another_stream(cuda):
    x, t, pw, w, gv, gh, gy = problem(cuda, torch.bfloat16, 1000, 1024, 10)
    op = torch.ops.flashoverlap_op

    def step():
        h, y, stats = op.rmsnorm_add_rmsnorm(x, t, pw, w, gv, 0.5, EPS, True)
        return (h, y, *op.rmsnorm_add_rmsnorm_backward(gh, gy, x, t, pw, w, gv, stats, 0.5))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    side = torch.cuda.Stream()
    for _ in range(3):
        x.normal_()
        gh.normal_()
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_rows_beyond_32_bit_offsets(cuda):
    """2.2e9 elements, each row as by itself; the weights' gradients of rows that are alike add up."""
    dt, rows, dim = torch.bfloat16, 270000, 8192
    x, t, pw, w, gv, gh, gy = problem(cuda, dt, 1000, dim, None)
    far = [v.repeat(rows // 1000, 1) for v in (x, t, gh, gy)]
    op = torch.ops.flashoverlap_op
    h, y, stats = op.rmsnorm_add_rmsnorm(far[0], far[1], pw, w, None, 0.5, EPS, True)
    h1, y1, stats1 = op.rmsnorm_add_rmsnorm(x, t, pw, w, None, 0.5, EPS, True)
    assert torch.equal(h[-1000:], h1) and torch.equal(y[-1000:], y1) and torch.equal(h[:1000], h1)
    grads = op.rmsnorm_add_rmsnorm_backward(far[2], far[3], far[0], far[1], pw, w, None, stats, 0.5)
    alone = op.rmsnorm_add_rmsnorm_backward(gh, gy, x, t, pw, w, None, stats1, 0.5)
    for a, b in zip(grads[:2], alone[:2]):
        assert torch.equal(a[-1000:], b) and torch.equal(a[134000:135000], b)
    for a, b in zip(grads[2:4], alone[2:4]):           # two roundings to bf16, and 32-bit sums of 270000 terms
        assert ((a.double() - 270 * b.double()).norm() <= 2 * 2.0 ** -8 * (270 * b.double()).norm())


def test_refuses(cuda):
    x, t, pw, w, gv, gh, gy = problem(cuda, torch.bfloat16, 24, 64, 4)
    for bad in ((x.cpu(), t, pw, w, gv), (x, t.cpu(), pw, w, gv), (x.float(), t.float(), pw.float(), w.float(), None), (x, t.half(), pw, w, gv),
                (x, t[:12], pw, w, gv), (x, t, pw[:32], w, gv), (x, t, pw, w.view(1, 64), gv), (x, t, pw, w.half(), gv), (x, t, pw, w, gv.half()),
                (x, t, pw, w, gv[:, :32]), (x, t, pw, w, gv.repeat(2, 1)[:5]), (x, t, pw, w, gv[:0]), (x, t, pw, w, gv.cpu()), (x, t, pw, w, gv[0, 0]),
                (x[0], t[0], pw, w, None), (x[:, :60], t[:, :60], pw[:60], w[:60], None), (x[:, :0], t[:, :0], pw[:0], w[:0], None)):
        with pytest.raises(RuntimeError):
            ops.rmsnorm_add_rmsnorm(*bad)
    wide = torch.zeros(2, 16392, device=cuda, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.rmsnorm_add_rmsnorm(wide, wide, wide[0], wide[0])
    op = torch.ops.flashoverlap_op
    _, _, stats = op.rmsnorm_add_rmsnorm(x, t, pw, w, gv, 1.0, EPS, True)
    for a, b, s in ((gh.half(), gy, stats), (gh[:12], gy, stats), (gh, gy.cpu(), stats), (gh, gy, stats[:12]), (gh, gy, stats.double()), (gh, gy, stats.cpu())):
        with pytest.raises(RuntimeError):
            op.rmsnorm_add_rmsnorm_backward(a, b, x, t, pw, w, gv, s, 1.0)


def test_refuses_stats_between_words(cuda):
    x, t, pw, w, gv, gh, gy = problem(cuda, torch.bfloat16, 24, 64, 4)
    odd = torch.zeros(49, device=cuda)[1:].view(24, 2)   # pairs that do not lie on 8 bytes
    with pytest.raises(RuntimeError, match="stats"):
        torch.ops.flashoverlap_op.rmsnorm_add_rmsnorm_backward(gh, gy, x, t, pw, w, gv, odd, 1.0)


def test_refuses_rows_whose_numbers_do_not_fit(cuda):
    x, w = torch.zeros(1, 8, device=cuda, dtype=torch.bfloat16), torch.ones(8, device=cuda, dtype=torch.bfloat16)
    for rows in (2 ** 31 - 3, 2 ** 31 - 1, 2 ** 31):
        many = x.expand(rows, 8)
        with pytest.raises(RuntimeError, match="too many rows"):
            ops.rmsnorm_add_rmsnorm(many, many, w, w)
