"""The gate, the token placement and the rows' ways on host tensors, against plain 64-bit statements; the gradient of
those statements against differences; and what the public calls refuse."""
import pytest
import torch

from tests import routing_reference as ref

KINDS = [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)]


@pytest.mark.parametrize("score,normalize", KINDS)
def test_reference_gradient_of_the_gate_agrees_with_differences(score, normalize):
    """Central differences of step 1e-5 in 64 bits: the error is step^2 * third derivative + 1e-16 / step, 1e-9 or so."""
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(3, 9, generator=g, dtype=torch.float64, requires_grad=True)
    flow = torch.randn(3, 4, generator=g, dtype=torch.float64)
    weights, _ = ref.gate(logits, 4, score, normalize)
    grad, = torch.autograd.grad(weights, logits, flow)
    for t in range(3):
        for e in range(9):
            step = torch.zeros_like(logits)
            step[t, e] = 1e-5
            up, down = (ref.gate((logits + s * step).detach(), 4, score, normalize)[0] for s in (1, -1))
            assert abs(float(((up - down) * flow).sum() / 2e-5) - float(grad[t, e])) < 1e-8


@pytest.mark.parametrize("score,normalize", KINDS)
def test_host_gate_matches_the_reference(score, normalize):
    from stk_b200 import dmoe
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(20, 11, generator=g)
    logits[3, :] = -torch.inf
    logits[4, 2:] = -torch.inf
    logits[5, :] = 1.0
    mask = torch.ones(20, dtype=torch.bool)
    mask[7] = False
    logits.requires_grad_()
    weights, ids = dmoe.top_k_gate(logits, 3, score=score, normalize=normalize, token_mask=mask)
    exact = logits.detach().double().requires_grad_()
    expect, expect_ids = ref.gate(exact, 3, score, normalize, mask)
    assert torch.equal(ids, expect_ids) and weights.dtype == torch.float32
    torch.testing.assert_close(weights.double(), expect, rtol=128 * ref.U32, atol=0)
    flow = torch.randn(20, 3, generator=g)
    grad, = torch.autograd.grad(weights, logits, flow)
    expect_grad, = torch.autograd.grad(expect, exact, flow.double())
    expect_grad = torch.nan_to_num(expect_grad)          # rows without a choice: 0 (the reference softmax of them is NaN)
    torch.testing.assert_close(grad.double(), expect_grad, rtol=0, atol=256 * ref.U32 * float(flow.abs().sum(1).max()))


@pytest.mark.parametrize("tokens,top_k,experts,block", [(0, 2, 3, 128), (1, 1, 1, 128), (5, 2, 4, 128), (300, 3, 7, 128),
                                                        (129, 1, 2, 128), (70, 2, 5, 16), (40, 1, 9, 1)])
@pytest.mark.parametrize("fixed", [False, True])
def test_host_plan_and_rows(tokens, top_k, experts, block, fixed):
    from stk_b200 import dmoe
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=g)
    rows = dmoe.plan_rows(tokens * top_k, experts, block) + block if fixed else None
    plan = dmoe.plan_tokens(ids, experts, block=block, rows=rows)
    index, position, bins = ref.placement(ids, experts, block, rows)
    assert torch.equal(plan.index, index) and torch.equal(plan.position, position) and torch.equal(plan.bin_rows, bins)
    assert plan.rows == index.numel() and plan.block_rows * block == plan.rows
    x = torch.randn(tokens, 6, generator=g, requires_grad=True)
    weights = torch.rand(tokens, top_k, generator=g, requires_grad=True)
    moved = dmoe.sort_tokens(x, plan)
    assert torch.equal(moved.detach(), ref.sort_rows(x.detach(), position, top_k, plan.rows))
    out = dmoe.unsort_tokens(2 * moved, weights, plan)
    live = (ids >= 0).float()
    torch.testing.assert_close(out, 2 * x * (weights * live).sum(1, keepdim=True), rtol=16 * ref.U32, atol=16 * ref.U32)
    dx, dw = torch.autograd.grad(out.sum(), (x, weights))
    torch.testing.assert_close(dw, 2 * x.detach().sum(1, keepdim=True) * live, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(dx, 2 * (weights.detach() * live).sum(1, keepdim=True).expand_as(dx), rtol=1e-5, atol=1e-5)


def test_plan_rows_is_enough_and_reached():
    from stk_b200 import dmoe
    # the worst batch: one slot in each of all experts but one, which gets the rest
    for slots, experts, block in [(10, 4, 128), (1000, 4, 128), (3, 8, 16), (1, 1, 128)]:
        used = min(slots, experts)
        ids = torch.arange(slots).clamp(max=used - 1)
        assert dmoe.plan_tokens(ids, experts, block=block).rows <= dmoe.plan_rows(slots, experts, block)
    assert dmoe.plan_rows(4, 4) == 512 and dmoe.plan_rows(0, 4) == 0 and dmoe.plan_rows(129, 1) == 256


def test_refusals():
    from stk_b200 import dmoe
    x = torch.randn(4, 8)
    for bad in (lambda: dmoe.top_k_gate(x[0], 2), lambda: dmoe.top_k_gate(x, 0), lambda: dmoe.top_k_gate(x, 9),
                lambda: dmoe.top_k_gate(x, 2, score="relu"), lambda: dmoe.top_k_gate(x.double(), 2),
                lambda: dmoe.top_k_gate(torch.randn(2, 1025), 2), lambda: dmoe.top_k_gate(torch.randn(2, 64), 33),
                lambda: dmoe.top_k_gate(x, 2, token_mask=torch.ones(4)),
                lambda: dmoe.top_k_gate(x, 2, token_mask=torch.ones(3, dtype=torch.bool)),
                lambda: dmoe.plan_tokens(x, 4), lambda: dmoe.plan_tokens(torch.zeros(2, 2, 2, dtype=torch.int32), 4),
                lambda: dmoe.plan_tokens(torch.zeros(4, dtype=torch.int32), 0),
                lambda: dmoe.plan_tokens(torch.zeros(4, dtype=torch.int32), 1025),
                lambda: dmoe.plan_tokens(torch.zeros(4, dtype=torch.int32), 4, block=0),
                lambda: dmoe.plan_tokens(torch.zeros((4, 0), dtype=torch.int32), 4),
                lambda: dmoe.plan_tokens(torch.full((4,), 4), 4),
                lambda: dmoe.plan_tokens(torch.zeros(4, dtype=torch.int32), 4, rows=384),
                lambda: dmoe.plan_tokens(torch.zeros(4, dtype=torch.int32), 4, rows=513)):
        with pytest.raises(ValueError):
            bad()
    plan = dmoe.plan_tokens(torch.tensor([[0, 1], [1, 2]]), 3)
    rows = torch.zeros(plan.rows, 8)
    for bad in (lambda: dmoe.sort_tokens(x, plan), lambda: dmoe.sort_tokens(x[0], plan),
                lambda: dmoe.sort_tokens(x[:2].double(), plan), lambda: dmoe.unsort_tokens(rows[1:], None, plan),
                lambda: dmoe.unsort_tokens(rows, torch.ones(2, 3), plan), lambda: dmoe.unsort_tokens(rows, torch.ones(4), plan),
                lambda: dmoe.unsort_tokens(rows, torch.ones(2, 2, dtype=torch.float64), plan)):
        with pytest.raises(ValueError):
            bad()


def test_entry_points_check_before_any_launch():
    """Without a device: every call returns its code before a kernel is launched."""
    from stk_b200.backend import lib
    L = lib.load()
    p = 4096                                              # an aligned address that is never read
    gate = lambda tokens=1, experts=4, k=2, ld=4, dtype=3, logits=p: L.stk_b200_top_k_gate(
        logits, ld, tokens, experts, k, 0, 1, None, p, p, None, dtype, None)
    assert gate(tokens=0) == 0 and gate(tokens=-1) == -2 and gate(k=5) == -2 and gate(k=0) == -2 and gate(ld=-1) == -2
    assert gate(experts=1025, ld=1025) == -9 and gate(experts=64, ld=64, k=33) == -9 and gate(dtype=2) == -3
    assert gate(logits=None) == -1
    assert L.stk_b200_top_k_gate_backward(p, 4, 1, 4, 2, 0, 0, p, p, None, p, p, 3, None) == -1    # no statistics
    place = lambda slots=4, experts=4, block=128, rows=512, ids=p: L.stk_b200_place_tokens(
        ids, slots, experts, block, rows, 0, p, p, p, None, None, 0, None)
    assert place(rows=384) == -2 and place(rows=513) == -2 and place(block=0) == -2 and place(experts=0) == -2
    assert place(experts=1025, rows=1025 * 128) == -9 and place(ids=None) == -1
    assert place(slots=8192, rows=128 * 128) == -7        # more than one CTA's slots need a workspace
    assert L.stk_b200_place_workspace_bytes(4096, 64) == 0 and L.stk_b200_place_workspace_bytes(4097, 64) == 512
    assert L.stk_b200_sort_rows(None, 8, p, p, p, 4, 2, 128, 8, 1, None) == -1
    assert L.stk_b200_sort_rows(p, 8, p, p, p, 4, 0, 128, 8, 1, None) == -2
    assert L.stk_b200_sort_rows(p, 8, p, p, p, 4, 2, 128, 8, 2, None) == -3
    assert L.stk_b200_sort_rows(p + 1, 8, p, p, p, 4, 2, 128, 8, 1, None) == -4
    assert L.stk_b200_sum_rows(p, 8, p, None, None, 4, 2, 8, 1, None) == -1
    assert L.stk_b200_sum_rows(p, 8, p, None, p, 4, 2, 0, 1, None) == 0
    assert L.stk_b200_unsort_backward(p, 8, p, 8, p, None, p, p, None, 4, 2, 128, 8, 1, None) == -1
    assert L.stk_b200_unsort_backward(p, 8, p, 8, p, p, p, None, None, 4, 2, 128, 8, 1, None) == 0


def test_tangents_go_through_the_host_path():
    """Host tensors take torch operations, which have forward-mode derivatives: they agree with the reverse mode's."""
    from torch.autograd import forward_ad
    from stk_b200 import dmoe
    g = torch.Generator().manual_seed(4)
    plan = dmoe.plan_tokens(torch.tensor([[0, 2], [1, -1], [2, 1], [0, 1]]), 3)
    x, dx = torch.randn(4, 5, generator=g), torch.randn(4, 5, generator=g)
    logits, dlogits = torch.randn(4, 6, generator=g), torch.randn(4, 6, generator=g)

    def value(x, logits):
        weights, _ = dmoe.top_k_gate(logits, 2, normalize=False)
        return dmoe.unsort_tokens(dmoe.sort_tokens(x, plan), weights, plan).square().sum()

    leaves = [x.clone().requires_grad_(), logits.clone().requires_grad_()]
    grads = torch.autograd.grad(value(*leaves), leaves)
    with forward_ad.dual_level():
        out = value(forward_ad.make_dual(x, dx), forward_ad.make_dual(logits, dlogits))
        slope = forward_ad.unpack_dual(out).tangent
    torch.testing.assert_close(slope, (grads[0] * dx).sum() + (grads[1] * dlogits).sum(), rtol=1e-4, atol=1e-5)


def test_counts_are_whole_numbers():
    """1.5 choices are not one choice."""
    from stk_b200 import dmoe
    x, ids = torch.randn(4, 8), torch.zeros(4, dtype=torch.int32)
    for bad in (lambda: dmoe.top_k_gate(x, 1.5), lambda: dmoe.plan_tokens(ids, 4.5), lambda: dmoe.plan_tokens(ids, 4, block=16.5),
                lambda: dmoe.plan_tokens(ids, 4, rows=512.5)):
        with pytest.raises(ValueError, match="whole number"):
            bad()
    assert all(torch.equal(a, b) for a, b in zip(dmoe.top_k_gate(x, 2.0), dmoe.top_k_gate(x, 2)))
    assert dmoe.plan_tokens(ids, 4.0, block=128.0, rows=512.0).rows == 512
