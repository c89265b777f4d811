"""The token rows, the gate and the 4-bit records past 2^31 elements or bytes, every row looked at.  All values are small
whole numbers, so that every sum is exact and results are equal, not close: products of values up to 3 over 4096 columns
stay below 2^16, sums of halves and quarters of them need 5 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOKENS, HIDDEN, TOP_K, EXPERTS = 290000, 4096, 2, 8
CHUNK = 20000


def whole(rows, cols, seed):
    """bfloat16 whole numbers -3..3, every row and column another."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    for r in range(0, rows, CHUNK):
        out[r:r + CHUNK] = torch.randint(-3, 4, (min(CHUNK, rows - r), cols), generator=g, device="cuda", dtype=torch.int8)
    return out


def plan_of(seed=0):
    from stk_b200 import dmoe
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, EXPERTS, (TOKENS, TOP_K), generator=g, device="cuda")
    ids[5::1000, 1] = -1
    return dmoe.plan_tokens(ids, EXPERTS)


def rows_by_token(rows, plan, t0, t1, j):
    """The rows of choice j of tokens [t0, t1), zeros where there is none, in 32 bits."""
    at = plan.position.view(TOKENS, TOP_K)[t0:t1, j].long()
    return rows[at.clamp(min=0)].float() * (at >= 0)[:, None]


def test_sorted_rows_and_their_gradient():
    from stk_b200 import dmoe
    plan = plan_of()
    assert plan.rows * HIDDEN > 2 ** 31
    x = whole(TOKENS, HIDDEN, 1).requires_grad_()
    rows = dmoe.sort_tokens(x, plan)
    for r in range(0, plan.rows, CHUNK):
        slot = plan.index[r:r + CHUNK].long()
        expect = x.detach()[slot.clamp(min=0) // TOP_K] * (slot >= 0)[:, None]
        assert torch.equal(rows.detach()[r:r + CHUNK], expect)
    drows = whole(plan.rows, HIDDEN, 2)
    dx, = torch.autograd.grad(rows, x, drows)
    for t in range(0, TOKENS, CHUNK):
        end = min(TOKENS, t + CHUNK)
        expect = rows_by_token(drows, plan, t, end, 0) + rows_by_token(drows, plan, t, end, 1)
        assert torch.equal(dx[t:end].float(), expect)


def test_weighted_return_and_both_gradients():
    from stk_b200 import dmoe
    plan = plan_of(3)
    rows = whole(plan.rows, HIDDEN, 4).requires_grad_()
    weights = torch.tensor([0.5, 0.25], device="cuda").expand(TOKENS, TOP_K).clone()
    weights[::3] = -0.5
    weights.requires_grad_()
    out = dmoe.unsort_tokens(rows, weights, plan)
    dout = whole(TOKENS, HIDDEN, 5)
    drows, dweights = torch.autograd.grad(out, (rows, weights), dout)
    w = weights.detach()
    for t in range(0, TOKENS, CHUNK):
        end = min(TOKENS, t + CHUNK)
        parts = [rows_by_token(rows.detach(), plan, t, end, j) for j in range(TOP_K)]
        assert torch.equal(out.detach()[t:end].float(), w[t:end, :1] * parts[0] + w[t:end, 1:] * parts[1])
        for j in range(TOP_K):
            assert torch.equal(dweights[t:end, j], (parts[j].double() * dout[t:end].double()).sum(1).float())
    for r in range(0, plan.rows, CHUNK):
        slot = plan.index[r:r + CHUNK].long()
        scale = w.view(-1)[slot.clamp(min=0)] * (slot >= 0)
        expect = scale[:, None] * dout[slot.clamp(min=0) // TOP_K].float()
        assert torch.equal(drows[r:r + CHUNK].float(), expect)


@pytest.mark.parametrize("normalize", [False, True])
def test_gate(normalize):
    """Every row as a call on the rows around it alone gives it."""
    from stk_b200 import dmoe
    tokens, experts = 2200000, 1000
    g = torch.Generator(device="cuda").manual_seed(6)
    logits = torch.empty((tokens, experts), dtype=torch.float16, device="cuda")
    for r in range(0, tokens, 100000):
        logits[r:r + 100000] = torch.randn(100000, experts, generator=g, device="cuda")
    assert logits.numel() > 2 ** 31
    logits.requires_grad_()
    weights, ids = dmoe.top_k_gate(logits, 2, normalize=normalize)
    flow = torch.randn(tokens, 2, generator=g, device="cuda")
    dlogits, = torch.autograd.grad(weights, logits, flow)
    for r in range(0, tokens, 100000):
        some = logits.detach()[r:r + 100000].clone().requires_grad_()
        expect, expect_ids = dmoe.top_k_gate(some, 2, normalize=normalize)
        assert torch.equal(weights.detach()[r:r + 100000], expect.detach()) and torch.equal(ids[r:r + 100000], expect_ids)
        assert torch.equal(dlogits[r:r + 100000], torch.autograd.grad(expect, some, flow[r:r + 100000])[0])


def test_gradient_of_an_empty_gate():
    from stk_b200 import dmoe
    for normalize in (False, True):
        leaf = torch.empty(0, 8, device="cuda", requires_grad=True)
        weights, ids = dmoe.top_k_gate(leaf, 2, normalize=normalize)
        assert weights.shape == (0, 2) and ids.shape == (0, 2) and weights.requires_grad
        grad, = torch.autograd.grad(weights.sum(), leaf)
        assert grad.shape == (0, 8) and grad.dtype == leaf.dtype


def test_4_bit_records():
    """The experts behind the first 2^31 bytes of records: as each alone."""
    from stk_b200 import dmoe
    experts, outputs, inputs = 300, 4096, 4096
    g = torch.Generator(device="cuda").manual_seed(7)
    codes = torch.empty((experts, outputs, inputs // 2), dtype=torch.uint8, device="cuda")
    for e in range(experts):
        codes[e] = torch.randint(0, 256, (outputs, inputs // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 + 0.02 * torch.rand(experts, outputs, inputs // 128, generator=g, device="cuda")).bfloat16()
    w = dmoe.pack_int4(codes, scales)
    assert w.records.numel() > 2 ** 31
    x = torch.randn(3, inputs, generator=g, device="cuda").bfloat16()
    ids = torch.tensor([[299, 0], [250, 298], [1, 299]], device="cuda")
    y = dmoe.int4_matvec(x, w, ids)
    for t in range(3):
        for j in range(2):
            e = int(ids[t, j])
            alone = dmoe.pack_int4(codes[e:e + 1], scales[e:e + 1])
            # the number of rows of a call decides how many warps share a row, and so the order of its sums: on either side
            # half a step of the type (2^-8) and (K / 32 + 16) 2^-24 + 2^-22 of the sum of magnitudes
            expect = dmoe.int4_matvec(x[t:t + 1], alone)[0].double()
            size = alone.dequantize(torch.float32)[0].double().abs() @ x[t].double().abs()
            tol = 2 * ((inputs / 32 + 16) * 2.0 ** -24 + 2.0 ** -22) * size + 2.0 ** -7 * expect.abs()
            assert bool(((y[t, j].double() - expect).abs() <= tol).all())
