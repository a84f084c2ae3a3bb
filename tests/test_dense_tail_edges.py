"""Calls of ops.dropout, ops.layer_norm and ops.linear_cross_entropy at the ends of what their documentation allows: masks that leave
nothing, values that are not finite, sizes that no launch fits, forms and tiles that a rule on sizes chooses. Tolerances as in
test_dense_tail.py: one rounding of the result, plus the fp32 roundings on the way, counted."""
import pytest
import torch

from test_dense_tail import BF16, F16, F32, gen, gpu, head

TYPES = pytest.mark.parametrize("t", [F32, BF16, F16])


# ---- rows do not meet --------------------------------------------------------------------------------------------------------
@gpu
@TYPES
@pytest.mark.parametrize("n,K,C", [(700, 64, 5000), (700, 128, 5000), (700, 190, 5000), (700, 250, 5000)])
def test_rows_in_another_order_give_the_same_values(dev, hiplib, n, K, C, t):
    """a row's loss and gradient do not depend on which lane or workgroup has it, nor on the tiles its workgroup walks beside others:
    to the bit, in any order of the rows and each time (K up to 128, 192, 256: the narrow form)"""
    from pagraph_amd import ops
    g = gen(61 + K, dev)
    lin = head(dev, K, C, t, g)
    h = torch.randn(n, K, generator=g, device=dev).to(t)
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    up = torch.randn(n, generator=g, device=dev)

    def values(order):
        x = h[order].requires_grad_()
        loss = ops.linear_cross_entropy(x, lin, lab[order], reduction="none")
        return [loss.detach()] + list(torch.autograd.grad(loss, [x], up[order]))
    want = values(torch.arange(n, device=dev))
    for k in range(4):
        order = torch.randperm(n, generator=g, device=dev)
        assert all(torch.equal(a, b[order]) for a, b in zip(values(order), want)), k
