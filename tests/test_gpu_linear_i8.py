"""8-bit linear layers, dense and by expert, against exact integer sums."""
import pytest
import torch

from flashoverlap_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def impl(cuda):
    i = ops.OverlapImpl()
    i.nccl_init(0, 1, [0] * 16)
    return i


def quantized(x):
    """The definition, one 32-bit operation at a time, on the host."""
    f = x.detach().cpu().float()
    top = f.abs().amax(1).clamp(min=2.0 ** -100)
    q = (f * (torch.tensor(127.0) / top)[:, None]).round()
    return q.to(torch.int8), top / torch.tensor(127.0)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 8), (3, 256), (5, 264), (100, 2048), (7, 2056), (33, 4104), (4, 8200), (2, 16392), (3, 32768), (1000, 72)])
def test_quantize(cuda, dt, rows, dim):
    x = (torch.randn(rows, dim, device=cuda) * torch.logspace(-3, 2, rows, device=cuda)[:, None]).to(dt)
    x[0, 0] = -300.0                               # the largest in magnitude is negative
    q, s = ops.quantize_rows(x)
    rq, rs = quantized(x)
    assert q.dtype == torch.int8 and torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)
    assert int(q[0, 0]) == -127


@pytest.mark.parametrize("dt", DTYPES)
def test_quantize_special_rows(cuda, dt):
    x = torch.randn(8, 64, device=cuda).to(dt)
    x[0] = 0
    x[1, 3], x[2, 5], x[3, 63] = float("nan"), float("inf"), float("-inf")
    x[4] = torch.finfo(dt).max * torch.randn(64, device=cuda).sign()
    x[5] = torch.finfo(dt).smallest_normal * torch.randn(64, device=cuda).sign()
    x[6] = torch.arange(64, device=cuda) - 0.0
    x[6, 0] = 127                                  # step one: integers stay
    x[7] = torch.arange(64, device=cuda) / 2
    x[7, 0] = 127                                  # ties go to even
    q, s = ops.quantize_rows(x)
    for r in (1, 2, 3):
        assert (q[r] == 0).all() and s[r].isnan()
    keep = [0, 4, 5, 6, 7]
    rq, rs = quantized(x[keep])
    assert torch.equal(q[keep].cpu(), rq) and torch.equal(s[keep].cpu(), rs)
    assert (q[0] == 0).all() and q[6, 1:].tolist() == list(range(1, 64)) and q[7, 1:6].tolist() == [0, 1, 2, 2, 2]
    assert ops.quantize_rows(x[:0])[0].shape == (0, 64)


def _operands(cuda, M, N, K, experts=0, seed=0, extreme=False):
    g = torch.Generator(device=cuda).manual_seed(seed)
    e = max(1, experts)
    if extreme:                                    # the largest sums there are
        a = torch.full((M, K), -128, device=cuda, dtype=torch.int8)
        b = torch.full((e, N, K), -128, device=cuda, dtype=torch.int8)
    else:
        a = torch.randint(-128, 128, (M, K), device=cuda, generator=g, dtype=torch.int8)
        b = torch.randint(-128, 128, (e, N, K), device=cuda, generator=g, dtype=torch.int8)
    sa, sb = torch.rand(M, device=cuda, generator=g) * 1e-3, torch.rand(e, N, device=cuda, generator=g) * 1e-2
    return (a, b, sa, sb) if experts else (a, b[0], sa, sb[0])


def _ref(a, b, sa, sb):
    return (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()


def _close(got, ref, dt):
    # the sum's conversion to 32 bits and two products, one rounding
    return ((got.double() - ref).abs() <= half_step(dt) * ref.abs() + 4 * 2.0 ** -24 * ref.abs() + smallest(dt)).all()


# one token; both sides of every tile width and split; N and K that end inside a tile; more tiles than CTAs; a second wave
DENSE = [(1, 8, 16), (1, 4096, 4096), (3, 136, 272), (16, 256, 1024), (17, 3584, 512), (32, 1000, 2048), (33, 512, 8192), (64, 520, 144), (65, 4096, 1024),
         (128, 264, 4096), (129, 264, 160), (200, 8192, 512), (255, 1032, 1040), (257, 512, 128), (1000, 2056, 400), (4096, 2560, 256), (300, 24, 28672),
         (5000, 4104, 80), (2048, 8192, 1024)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N,K", DENSE)
def test_gemm(cuda, impl, dt, M, N, K):
    a, b, sa, sb = _operands(cuda, M, N, K)
    mem = torch.full((M + 2, N), float("nan"), device=cuda, dtype=dt)
    impl.gemm_i8(a, b, sa, sb, mem[1:M + 1] if N % 8 == 0 and N * 2 % 16 == 0 else mem[:M], None)
    impl.check_status()
    assert _close(mem[1:M + 1], _ref(a, b, sa, sb), dt)
    assert mem[0].isnan().all() and mem[-1].isnan().all()          # nothing beyond the matrix


# a problem for everything that may run: tokens of a tile and split (0, 1: 256-row tiles; 0, 2: 512), M, N, K, experts (0: dense)
PLANS = [(0, 1, 9929, 40, 48, 0), (0, 1, 9825, 40, 48, 2), (0, 2, 14245, 272, 18032, 0), (16, 1, 1, 40, 48, 0), (16, 1, 2, 40, 48, 1),
         (16, 2, 2, 4264, 656, 0), (16, 2, 43, 40, 736, 40), (16, 4, 1, 40, 512, 0), (16, 4, 1, 40, 528, 1), (32, 1, 4924, 40, 48, 0), (32, 1, 4777, 40, 48, 1),
         (32, 2, 2646, 40, 1264, 0), (32, 2, 2454, 48, 1168, 1), (32, 4, 1234, 40, 896, 0), (32, 4, 1333, 40, 848, 6), (32, 8, 1, 40, 1552, 0),
         (32, 8, 1, 40, 1568, 1), (64, 1, 62, 13168, 16736, 0), (64, 1, 13468, 40, 144, 54), (64, 2, 4910, 40, 1600, 0), (64, 2, 4731, 40, 1616, 7),
         (64, 4, 2399, 40, 1584, 0), (64, 4, 2648, 40, 1296, 2), (64, 8, 1252, 40, 2992, 0), (64, 8, 1225, 40, 2880, 1), (128, 1, 11218, 40, 3936, 0),
         (128, 1, 9694, 40, 4320, 44), (128, 2, 4922, 40, 4432, 0), (128, 2, 5020, 40, 4976, 2), (128, 4, 2421, 48, 7280, 0), (128, 4, 2320, 40, 7920, 6),
         (128, 8, 1247, 40, 15472, 0), (128, 8, 1150, 48, 12928, 5)]


@pytest.mark.parametrize("tokens,split,M,N,K,experts", PLANS)
def test_every_kernel(cuda, impl, tokens, split, M, N, K, experts):
    a, b, sa, sb = _operands(cuda, M, N, K, experts)
    mem = torch.full((M + 2, N), float("nan"), device=cuda, dtype=torch.bfloat16)
    c = mem[1:M + 1]
    if experts:                                    # uneven, the first one's none if there are others, two rows nobody's
        cuts = (torch.linspace(0, 1, experts)[1:] ** 2 * max(M - 2, 1)).int().tolist() if experts > 1 else [max(M - 2, 1)]
        offsets = torch.tensor([0, *([0] if experts > 1 else []), *cuts], device=cuda, dtype=torch.int32)
        ref = torch.zeros(M, N, dtype=torch.float64, device=cuda)
        for e, lo, hi in _segments(offsets, M):
            ref[lo:hi] = _ref(a[lo:hi], b[e], sa[lo:hi], sb[e])
    else:
        offsets, ref = None, _ref(a, b, sa, sb)
    impl.gemm_i8(a, b, sa, sb, c, offsets)
    impl.check_status()
    assert (impl.get_option("last_i8_tokens"), impl.get_option("last_i8_split")) == (tokens, split)
    assert _close(c, ref, torch.bfloat16) and mem[0].isnan().all() and mem[-1].isnan().all()


@pytest.mark.parametrize("M", [1, 40, 500])
def test_gemm_largest_sums(cuda, impl, M):
    a, b, sa, sb = _operands(cuda, M, 256, 131056, extreme=True)
    c = torch.empty(M, 256, device=cuda, dtype=torch.bfloat16)
    impl.gemm_i8(a, b, sa, sb, c, None)
    impl.check_status()
    assert _close(c, torch.full((M, 256), 128.0 * 128 * 131056, device=cuda, dtype=torch.float64) * sa.double()[:, None] * sb.double(), torch.bfloat16)


def _segments(offsets, M):
    o = offsets.tolist()
    return [(e, a, b) for e, (a, b) in enumerate(zip(o, o[1:]))]


# rows of the experts; the rest are nobody's
GROUPED = [([1], 0, 64, 64), ([0, 0, 5, 0], 3, 136, 272), ([16, 17, 1, 0, 33], 0, 512, 1024), ([3] * 40, 7, 264, 512), ([100, 0, 300, 128], 20, 1032, 160),
           ([256, 512, 1, 255, 257], 0, 520, 400), ([0, 2000, 30], 1, 2560, 256), ([700] + [1] * 50, 0, 256, 144), ([0, 0], 9, 64, 64),
           ([2, 0, 1] * 341, 5, 72, 32), ([300, 299, 301, 400, 350, 280, 333, 260], 100, 4096, 512)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("counts,rest,N,K", GROUPED)
def test_gemm_by_expert(cuda, impl, dt, counts, rest, N, K):
    M = sum(counts) + rest
    a, b, sa, sb = _operands(cuda, M, N, K, len(counts))
    offsets = torch.tensor([0] + counts, device=cuda).cumsum(0).to(torch.int32)
    mem = torch.full((M + 2, N), float("nan"), device=cuda, dtype=dt)
    c = mem[1:M + 1]
    impl.gemm_i8(a, b, sa, sb, c, offsets)
    impl.check_status()
    ref = torch.zeros(M, N, dtype=torch.float64, device=cuda)
    for e, lo, hi in _segments(offsets, M):
        ref[lo:hi] = _ref(a[lo:hi], b[e], sa[lo:hi], sb[e])
    assert _close(c, ref, dt) and (c[M - rest:] == 0).all()
    assert mem[0].isnan().all() and mem[-1].isnan().all()


@pytest.mark.parametrize("M,experts", [(600, 2), (30, 3)])
def test_offsets_that_are_none(cuda, impl, M, experts):
    """Offsets out of order or out of range are reported and nothing beyond the matrices is touched; rows that lie outside
    the first and the last offset are zero."""
    a, b, sa, sb = _operands(cuda, M, 64, 64, experts)
    c = torch.empty(M, 64, device=cuda, dtype=torch.bfloat16)
    for bad in ([0, M + 1], [0, -5], [5, 2], [0, 1 << 30]):
        offsets = torch.tensor(bad + [M] * (experts - 1), dtype=torch.int32, device=cuda)
        impl.gemm_i8(a, b, sa, sb, c, offsets)
        with pytest.raises(RuntimeError, match="bad argument"):
            impl.check_status()
        impl.reset_status()
    offsets = torch.tensor([4, 10] + [M - 3] * (experts - 1), dtype=torch.int32, device=cuda)
    impl.gemm_i8(a, b, sa, sb, c, offsets)
    impl.check_status()
    assert (c[:4] == 0).all() and (c[-3:] == 0).all() and _close(c[4:10], _ref(a[4:10], b[0], sa[4:10], sb[0]), torch.bfloat16)


@pytest.mark.parametrize("M,experts,at", [(1, 40, 33), (2, 40, 39), (2, 1000, 999), (15, 200, 100), (40, 100, 99), (2000, 100, 99)])
def test_offsets_that_are_none_behind_all_rows(cuda, impl, M, experts, at):
    """Every row has its expert before the offset that is out of range: that is reported all the same, and the rows are right."""
    a, b, sa, sb = _operands(cuda, M, 64, 64, experts)
    offsets = torch.arange(experts + 1, dtype=torch.int32, device=cuda).clamp(max=M)
    offsets[min(32, experts):] = M
    c = torch.empty(M, 64, device=cuda, dtype=torch.bfloat16)
    impl.gemm_i8(a, b, sa, sb, c, offsets)
    impl.check_status()
    right = c.clone()
    offsets[at] = M + 5
    impl.gemm_i8(a, b, sa, sb, c, offsets)
    with pytest.raises(RuntimeError, match="bad argument"):
        impl.check_status()
    impl.reset_status()
    assert torch.equal(c, right)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape,N", [((1, 64), 64), ((2, 3, 512), 136), ((512,), 64), ((300, 272), 264)])
def test_linear(cuda, impl, dt, shape, N):
    x = torch.randn(*shape, device=cuda).to(dt)
    K = shape[-1]
    _, b, _, sb = _operands(cuda, 1, N, K)
    y = ops.linear_i8(impl, x, b, sb)
    impl.check_status()
    q, s = quantized(x.reshape(-1, K))
    assert y.shape == (*shape[:-1], N) and y.dtype == dt
    assert _close(y.reshape(-1, N), _ref(q.to(cuda), b, s.to(cuda), sb), dt)


# a token or a few, every split; K that ends inside a block or a 16-byte piece of it; one row more, and longer rows
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,K", [(8, 16), (40, 48), (136, 144), (4096, 528), (1024, 1040), (28672, 1024), (136, 2064), (8192, 3584), (4096, 4112), (40, 8192), (40, 8208)])
def test_linear_of_a_few_tokens_is_its_two_steps(cuda, impl, dt, N, K):
    _, b, _, sb = _operands(cuda, 1, N, K)
    for M in (1, 2, 3, 4, 5):
        x = (torch.randn(M, K, device=cuda) * torch.logspace(-2, 2, M, device=cuda)[:, None]).to(dt)
        x[0, -1] = 100.0                           # the largest lies in the last CTA's part
        if M == 3:
            x[1, 0] = float("inf")
            x[2] = 0
        mem = torch.full((M, N), float("nan"), device=cuda, dtype=dt)
        q, s = ops.quantize_rows(x)
        impl.gemm_i8(q, b, s, sb, mem, None)
        y = ops.linear_i8(impl, x, b, sb)
        impl.check_status()
        assert torch.equal(y.view(torch.int16), mem.view(torch.int16)) or (M == 3 and torch.equal(y[[0, 2]], mem[[0, 2]]) and y[1].isnan().all())
        if M == 1:                                 # in a graph, behind a kernel that lets it start early
            graph, w = torch.cuda.CUDAGraph(), torch.ones(K, device=cuda, dtype=dt)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                n = ops.rmsnorm(x, w)
                captured = ops.linear_i8(impl, n, b, sb)
            for _ in range(3):
                x.normal_()
                graph.replay()
                assert torch.equal(captured, ops.linear_i8(impl, ops.rmsnorm(x, w), b, sb))


def test_linear_special_rows_stay_in_their_rows(cuda, impl):
    x = torch.randn(20, 64, device=cuda).to(torch.bfloat16)
    x[3, 1], x[7, 5], x[11] = float("nan"), float("inf"), 0
    _, b, _, sb = _operands(cuda, 1, 64, 64)
    y = ops.linear_i8(impl, x, b, sb)
    assert y[3].isnan().all() and y[7].isnan().all() and (y[11] == 0).all()
    rest = [r for r in range(20) if r not in (3, 7)]
    assert torch.equal(y[rest], ops.linear_i8(impl, x[rest], b, sb))


def test_linear_strided_and_unaligned(cuda, impl):
    x = torch.randn(24, 144, device=cuda).to(torch.float16)
    _, b, _, sb = _operands(cuda, 1, 64, 144)
    ref = ops.linear_i8(impl, x, b, sb)
    mem = torch.empty(24 * 144 + 8, device=cuda, dtype=x.dtype)
    for v in (mem[1:1 + 24 * 144].view(24, 144).copy_(x), torch.cat([x, x], 1)[:, :144], x.t().contiguous().t()):
        assert torch.equal(ops.linear_i8(impl, v, b, sb), ref)
    assert ops.linear_i8(impl, x[:0], b, sb).shape == (0, 64)


def test_replayed_graph_and_another_stream(cuda, impl):
    for M, experts in ((20, 0), (700, 0), (60, 5), (900, 3)):
        a, b, sa, sb = _operands(cuda, M, 512, 256, experts)
        x = torch.randn(M, 256, device=cuda).to(torch.bfloat16)
        offsets = torch.linspace(0, M, experts + 1, device=cuda).int() if experts else None
        ops.linear_i8(impl, x, b, sb, offsets)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = ops.linear_i8(impl, x, b, sb, offsets)
        side = torch.cuda.Stream()
        for i in range(3):
            x.normal_()
            if experts:
                offsets[1] = 10 * i
            graph.replay()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                eager = ops.linear_i8(impl, x, b, sb, offsets)
            torch.cuda.synchronize()
            assert torch.equal(captured, eager)
    impl.check_status()


def test_beyond_32_bit_offsets(cuda, impl):
    """C and the activations pass 2^31 elements, then the weights do."""
    M, N, K = 270000, 8192, 64
    x = torch.randn(M, K, device=cuda).to(torch.bfloat16)
    _, b, _, sb = _operands(cuda, 1, N, K)
    y = ops.linear_i8(impl, x, b, sb)
    for lo in (0, M // 2, M - 700):
        assert torch.equal(y[lo:lo + 700], ops.linear_i8(impl, x[lo:lo + 700], b, sb))
    del x, y
    experts, N, K = 40, 8192, 8192
    b = torch.randint(-128, 128, (experts, N, K), device=cuda, dtype=torch.int8)
    sb = torch.rand(experts, N, device=cuda) * 1e-2
    for rows in (3, 300):                      # either kernel
        x = torch.randn(2 * rows, K, device=cuda).to(torch.bfloat16)
        offsets = torch.tensor([0] + [rows] * (experts - 1) + [2 * rows], device=cuda, dtype=torch.int32)
        y = ops.linear_i8(impl, x, b, sb, offsets)
        for e, part in ((0, slice(0, rows)), (experts - 1, slice(rows, 2 * rows))):
            assert torch.equal(y[part], ops.linear_i8(impl, x[part], b[e], sb[e]))
    impl.check_status()


def test_refuses(cuda, impl):
    a, b, sa, sb = _operands(cuda, 32, 64, 128)
    c = torch.empty(32, 64, device=cuda, dtype=torch.bfloat16)
    impl.gemm_i8(a, b, sa, sb, c, None)
    mem = torch.zeros(1 << 16, device=cuda, dtype=torch.int8)
    off = torch.zeros(2, dtype=torch.int32, device=cuda)
    for bad in ((a.cpu(), b, sa, sb, c), (a.float(), b, sa, sb, c), (a[:, :64], b, sa, sb, c), (a, b.cpu(), sa, sb, c), (a, b.half(), sa, sb, c),
                (a, b.view(1, 64, 128), sa, sb, c), (a, b[:60], sa, sb[:60], c[:, :60].contiguous()), (a[:, :120].contiguous(), b[:, :120].contiguous(), sa, sb, c),
                (a, b, sa[:31], sb, c), (a, b, sa.double(), sb, c), (a, b, sa.cpu(), sb, c), (a, b, sa, sb[:63], c), (a, b, sa, sb.half(), c),
                (a, b, sa, sb, c[:31]), (a, b, sa, sb, c.float()), (a, b, sa, sb, c.cpu()), (a, b, sa, sb, c.t()), (a.view(-1), b, sa, sb, c),
                (mem[8:8 + 32 * 128].view(32, 128), b, sa, sb, c), (a, b, sa, sb, a.view(torch.bfloat16)), (a, b, sa, sb, mem[2:2 + 4096].view(torch.bfloat16).view(32, 64)),
                (a, b, sa, mem.view(torch.float32)[1:65], c)):
        with pytest.raises(RuntimeError):
            impl.gemm_i8(*bad, None)
    for o, w, s in ((off, b, sb), (off.long(), b[None], sb[None]), (off.cpu(), b[None], sb[None]), (off[:1], b[None], sb[None]), (off, b[None], sb), (off, b[None, :0], sb[None, :0])):
        with pytest.raises(RuntimeError):
            impl.gemm_i8(a, w, sa, s, c, o)
    x = torch.randn(4, 128, device=cuda).to(torch.bfloat16)
    for bad, w in ((x.float(), b), (x.cpu(), b), (x[:, :64], b), (x[:, :0], b[:, :0])):
        with pytest.raises(RuntimeError):
            ops.linear_i8(impl, bad, w, sb)
    for bad in (x.float(), x.cpu(), x[0], x[:, :4], torch.zeros(1, 32776, device=cuda, dtype=x.dtype), x.clone().requires_grad_()):
        with pytest.raises(RuntimeError):
            ops.quantize_rows(bad)
    with pytest.raises(RuntimeError):
        ops.linear_i8(impl, x.clone().requires_grad_(), b, sb)
    impl.check_status()
