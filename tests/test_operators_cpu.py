"""What the new-tensor operators refuse without a GPU: host tensors, before anything is launched."""
import pytest
import torch

from flashoverlap_b200 import ops


def test_host_tensors_are_refused(lib):
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    order = ops.ExpertOrder(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    y = torch.zeros(8, 64, dtype=torch.bfloat16)
    impl = ops.OverlapImpl()
    q, s = torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8)
    for call in (lambda: ops.moe_sort(order.slot, 2), lambda: ops.moe_dispatch(x, order), lambda: ops.moe_combine(y, None, order),
                 lambda: ops.moe_combine(y, torch.ones(4, 2), order), lambda: ops.rmsnorm_add_rmsnorm(x, x, w, w),
                 lambda: ops.rmsnorm_add_rmsnorm(x, x, w, w, w, 0.5), lambda: ops.quantize_rows(x), lambda: ops.linear_i8(impl, x, q, s),
                 lambda: impl.gemm_i8(q, q, s, s, torch.zeros(8, 8, dtype=torch.bfloat16), None)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_no_gradient_is_left_out_silently(lib):
    impl = ops.OverlapImpl()
    x = torch.zeros(4, 64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.quantize_rows(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.linear_i8(impl, x, torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8))


def test_sorts_where_large_clusters_have_no_place(lib):
    """Sixteen CTAs for many choices, but never a cluster that the device cannot place."""
    ctas = torch.ops.flashoverlap_op.moe_sort_ctas
    for most in range(1, 17):
        for choices in (0, 1, 2048, 2049, 8192, 8193, 2 ** 31 - 1):
            wanted = 1 if choices <= 2048 else 8 if choices <= 8192 else 16
            assert ctas(choices, most) == max(c for c in (1, 8, 16) if c <= min(most, wanted))


def test_backward_passes_as_operators_have_no_gradient_to_lose(lib):
    op = torch.ops.flashoverlap_op
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    order = (torch.zeros(4, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    y, p, stats = torch.zeros(8, 64, dtype=torch.bfloat16), torch.ones(4, 2), torch.zeros(4, 2)
    for grad in (x, y, p):
        grad.requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            op.moe_combine_backward(x, y, p, *order, True, True)
        grad.requires_grad_(False)
    for grad in (x, w, stats):
        grad.requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            op.rmsnorm_add_rmsnorm_backward(x, None, x, x, w, w, None, stats, 1.0)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):
            op.rmsnorm_add_rmsnorm_backward(x, None, x, x, w, w, None, stats, 1.0)
        grad.requires_grad_(False)
