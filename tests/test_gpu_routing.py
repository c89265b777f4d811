"""The gate, the token placement and the rows' ways on the GPU, against plain 64-bit statements (tests/routing_reference.py).

Tolerances, with u = 2^-24 (one rounding to 32 bits) and h = half a step of the output's type:
* gate weights: relative 128 u.  The exponent's argument l - max and its product with log2(e) are rounded once each, errors
  of |l - max| u of the exponential (|l - max| < 40 for the logits here); the power of two is 4 u off, the sum over a
  row adds at most 32 + 5, the division 2.
* gate gradient: h |d| for its type, and 256 u w_i (|g_i| + sum |g_j| w_j): the same errors in every term of a difference.
* sums over choices: h |out| and (k + 1) u times the sum of the terms' magnitudes.
* dot products: (h / 32 + 16) u times the sum of the magnitudes: a lane adds at most hidden / 32 terms, then come
  5 steps over the lanes and 8 over the warps."""
import threading

import pytest
import torch

from tests import routing_reference as ref
from tests.test_routing_host import KINDS

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def gate_logits(tokens, experts, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, experts, generator=g) * 3).to(dtype)


def check_gate(logits, top_k, score, normalize, mask=None, weights_and_ids=None):
    from stk_b200 import dmoe
    dev = logits.cuda().requires_grad_()
    weights, ids = dmoe.top_k_gate(dev, top_k, score=score, normalize=normalize,
                                   token_mask=None if mask is None else mask.cuda())
    exact = logits.double().requires_grad_()
    expect, expect_ids = ref.gate(exact, top_k, score, normalize, mask)
    assert weights.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu(), expect_ids)
    torch.testing.assert_close(weights.detach().cpu().double(), expect.detach(), rtol=128 * ref.U32, atol=0)
    g = torch.Generator().manual_seed(7)
    flow = torch.randn(logits.shape[0], top_k, generator=g)
    grad, = torch.autograd.grad(weights, dev, flow.cuda())
    expect_grad, = torch.autograd.grad(expect, exact, flow.double())
    # w_i of every logit: the weight that it has or (not chosen, plain softmax) would have
    w = torch.zeros_like(exact)
    if score == "softmax" and not normalize:
        w = torch.softmax(exact.detach(), 1).nan_to_num()
    rows = torch.arange(len(logits))[:, None].expand_as(expect_ids)
    valid = expect_ids >= 0
    w[rows[valid], expect_ids[valid].long()] = expect.detach()[valid]
    size = torch.zeros_like(exact)
    size[rows[valid], expect_ids[valid].long()] = flow.double().abs()[valid]
    inner = (flow.double().abs() * expect.detach()).sum(1, keepdim=True)
    expect_grad = expect_grad.nan_to_num()                # (rows without a choice)
    tol = ref.half_step(logits.dtype) * expect_grad.abs() + 256 * ref.U32 * w * (size + inner) + ref.TINY[logits.dtype]
    assert grad.dtype == logits.dtype
    assert bool(((grad.cpu().double() - expect_grad).abs() <= tol).all())


@pytest.mark.parametrize("score,normalize", KINDS)
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 2, 2), (5, 7, 3), (33, 8, 8), (70, 16, 1), (40, 31, 5),
                                                  (33, 64, 2), (30, 160, 6), (17, 257, 8), (9, 513, 32), (3, 1024, 32)])
def test_gate(tokens, experts, top_k, score, normalize):
    for dtype in DTYPES:
        check_gate(gate_logits(tokens, experts, dtype), top_k, score, normalize)


@pytest.mark.parametrize("score,normalize", KINDS)
def test_gate_masks_and_ties(score, normalize):
    for dtype in DTYPES:
        logits = gate_logits(24, 37, dtype, 1)
        logits[0] = -torch.inf                            # no expert left
        logits[1, 2:] = -torch.inf                        # fewer than k
        logits[2] = 0.5                                   # all equal: the lowest experts
        logits[3, ::2], logits[3, 1::2] = 0.0, -0.0       # the two zeros are equal
        logits[4, 5] = logits[4, 30] = 9.0
        logits[5] = torch.finfo(dtype).min                # the type's lowest value is a value like any other
        logits[6, 3:] = torch.finfo(dtype).min
        mask = torch.ones(24, dtype=torch.bool)
        mask[20:] = False
        check_gate(logits, 4, score, normalize, mask)


@pytest.mark.parametrize("score,normalize", KINDS)
def test_gate_nan_and_infinity(score, normalize):
    """A NaN shows in its own row, with ids that name experts, and nowhere else; behind the token mask it does not show."""
    from stk_b200 import dmoe
    logits = gate_logits(6, 40, torch.float32, 2)
    clean = logits.clone()
    logits[1, 17] = torch.nan
    logits[3] = torch.nan
    logits[4, 2] = torch.inf
    mask = torch.tensor([True, True, True, False, True, True]).cuda()
    dev = logits.cuda().requires_grad_()
    weights, ids = dmoe.top_k_gate(dev, 3, score=score, normalize=normalize, token_mask=mask)
    grad, = torch.autograd.grad(weights.sum(), dev)
    expect, expect_ids = dmoe.top_k_gate(clean.cuda(), 3, score=score, normalize=normalize)
    for t in (0, 2, 5):
        assert torch.equal(weights[t], expect[t]) and torch.equal(ids[t], expect_ids[t])
        assert bool(torch.isfinite(grad[t]).all())
    assert bool(weights[1].isnan().any()) and int(ids[1, 0]) == 17 and bool(((ids[1] >= 0) & (ids[1] < 40)).all())
    assert int(ids[4, 0]) == 2
    assert ids[3].tolist() == [-1] * 3 and weights[3].tolist() == [0.0] * 3 and not bool(grad[3].any())


def test_gate_strides_streams_and_partial_use():
    from stk_b200 import dmoe
    wide = gate_logits(50, 130, torch.bfloat16, 3).cuda()
    for view in (wide[:, 1:65], wide[::2, :64], wide.t()[:50], wide[0:1].expand(50, 130)):
        got = dmoe.top_k_gate(view, 3)
        expect = dmoe.top_k_gate(view.contiguous(), 3)
        assert all(torch.equal(a, b) for a, b in zip(got, expect))
    # the gradient goes through a view, and a call whose weights nobody asks about passes none
    base = gate_logits(50, 130, torch.float32, 4).cuda().requires_grad_()
    weights, ids = dmoe.top_k_gate(base[:, 1:65], 2, normalize=False)
    weights[:, 0].sum().backward()
    assert not bool(base.grad[:, 65:].any()) and bool(base.grad[:, 1:65].any())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = dmoe.top_k_gate(base[:, 1:65], 2, normalize=False)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again[0], weights) and torch.equal(again[1], ids)
    empty = dmoe.top_k_gate(torch.empty(0, 8, device="cuda", requires_grad=True), 2)
    assert empty[0].shape == (0, 2)
    torch.autograd.grad(empty[0].sum(), base, allow_unused=True) if empty[0].requires_grad else None


# ------------------------------------------------------------------------------ placement
@pytest.mark.parametrize("tokens,top_k,experts,block", [(0, 2, 3, 128), (1, 1, 1, 128), (5, 2, 4, 128), (300, 3, 7, 128),
                                                        (4096, 1, 64, 128), (4097, 1, 64, 128), (3000, 3, 1024, 16),
                                                        (20000, 2, 33, 128), (513, 8, 5, 1)])
@pytest.mark.parametrize("fixed", [False, True])
def test_plan(tokens, top_k, experts, block, fixed):
    from stk_b200 import dmoe
    g = torch.Generator().manual_seed(tokens + experts)
    low = -1 if tokens % 2 else 0
    for kind in ("even", "one", "none"):
        ids = torch.randint(low, experts, (tokens, top_k), generator=g)
        if kind == "one":
            ids[:] = experts - 1
        if kind == "none":
            ids[:] = -3
        rows = dmoe.plan_rows(tokens * top_k, experts, block) + 3 * block if fixed else None
        expect = dmoe.plan_tokens(ids, experts, block=block, rows=rows)      # the host's, tested there
        for dtype in (torch.int16, torch.int32, torch.int64):
            plan = dmoe.plan_tokens(ids.cuda().to(dtype), experts, block=block, rows=rows)
            assert plan.rows == expect.rows and plan.block_rows == expect.block_rows
            for name in ("index", "position", "bin_rows"):
                assert torch.equal(getattr(plan, name).cpu(), getattr(expect, name)), name


def test_plan_reports_experts_that_do_not_exist():
    from stk_b200 import dmoe
    from stk_b200.backend import lib
    assert lib.device_status() == 0
    plan = dmoe.plan_tokens(torch.tensor([0, 5, 1, 99, 4], device="cuda"), 5)
    assert lib.device_status() == -2 and lib.device_status() == 0
    assert plan.position.tolist() == [0, -1, 128, -1, 256]       # as if they had none
    plan = dmoe.plan_tokens(torch.tensor([2 ** 32, 1, 2 ** 33 + 2, -2 ** 33], device="cuda"), 5)  # 0, 1, 2, 0 in 32 bits
    assert lib.device_status() == -2 and plan.position.tolist() == [-1, 0, -1, -1]


def test_plans_of_two_threads_at_once():
    from stk_b200 import dmoe
    batches = [torch.randint(0, 12, (997 + 640 * i, 2), generator=torch.Generator().manual_seed(i)) for i in range(8)]
    expect = [dmoe.plan_tokens(b, 12) for b in batches]
    wrong = []

    def work(mine):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    for i in mine:
                        plan = dmoe.plan_tokens(batches[i].cuda(), 12)
                        if plan.rows != expect[i].rows or not torch.equal(plan.index.cpu(), expect[i].index):
                            wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(range(n, 8, 2),)) for n in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


# ------------------------------------------------------------------------------ rows
def rows_case(tokens, hidden, experts, top_k, dtype, fixed=False, seed=0):
    from stk_b200 import dmoe
    g = torch.Generator().manual_seed(seed + tokens + hidden)
    ids = torch.randint(-1 if tokens > 3 else 0, experts, (tokens, top_k), generator=g)
    rows = dmoe.plan_rows(tokens * top_k, experts) if fixed else None
    plan = dmoe.plan_tokens(ids.cuda(), experts, rows=rows)
    return plan, g


CASES = [(0, 8, 3, 2), (1, 1, 1, 1), (3, 64, 2, 2), (130, 8, 3, 2), (257, 1001, 5, 3), (65, 514, 9, 1), (64, 1024, 8, 2), (33, 4100, 4, 4),
         (40, 130, 24, 20), (200, 2052, 16, 2)]


@pytest.mark.parametrize("tokens,hidden,experts,top_k", CASES)
@pytest.mark.parametrize("fixed", [False, True])
def test_sort_rows_and_gradient(tokens, hidden, experts, top_k, fixed):
    from stk_b200 import dmoe
    for dtype in DTYPES:
        plan, g = rows_case(tokens, hidden, experts, top_k, dtype, fixed)
        x = torch.randn(tokens, hidden, generator=g).to(dtype)
        dev = x.cuda().requires_grad_()
        rows = dmoe.sort_tokens(dev, plan)
        position = plan.position.cpu()
        assert torch.equal(rows.detach().cpu(), ref.sort_rows(x, position, top_k, plan.rows))
        drows = torch.randn(plan.rows, hidden, generator=g).to(dtype)
        dx, = torch.autograd.grad(rows, dev, drows.cuda())
        expect, size = ref.sum_rows(drows, position, None, tokens, top_k)
        tol = ref.half_step(dtype) * expect.abs() + (top_k + 1) * ref.U32 * size + ref.TINY[dtype]
        assert dx.dtype == dtype and bool(((dx.cpu().double() - expect).abs() <= tol).all())
        again, = torch.autograd.grad(dmoe.sort_tokens(dev, plan), dev, drows.cuda())
        assert torch.equal(dx, again)                    # the same bits from run to run


@pytest.mark.parametrize("tokens,hidden,experts,top_k", CASES)
@pytest.mark.parametrize("fixed", [False, True])
def test_unsort_rows_and_gradients(tokens, hidden, experts, top_k, fixed):
    from stk_b200 import dmoe
    for dtype in DTYPES:
        plan, g = rows_case(tokens, hidden, experts, top_k, dtype, fixed, 1)
        rows = torch.randn(plan.rows, hidden, generator=g).to(dtype)
        rows[plan.index.cpu() < 0] = torch.nan           # what is in padding rows does not matter
        weights = torch.randn(tokens, top_k, generator=g)
        dev, dev_w = rows.cuda().requires_grad_(), weights.cuda().requires_grad_()
        out = dmoe.unsort_tokens(dev, dev_w, plan)
        position, index = plan.position.cpu(), plan.index.cpu()
        expect, size = ref.sum_rows(rows, position, weights, tokens, top_k)
        tol = ref.half_step(dtype) * expect.abs() + (top_k + 1) * ref.U32 * size + ref.TINY[dtype]
        assert out.dtype == dtype and bool(((out.detach().cpu().double() - expect).abs() <= tol).all())
        dout = torch.randn(tokens, hidden, generator=g).to(dtype)
        drows, dweights = torch.autograd.grad(out, (dev, dev_w), dout.cuda())
        for s, r in enumerate(position.tolist()):
            if r < 0:
                assert float(dweights.reshape(-1)[s]) == 0.0
        live = index >= 0
        slot = index[live].long()
        expect_rows = torch.zeros(plan.rows, hidden, dtype=torch.float64)
        expect_rows[live] = weights.reshape(-1)[slot].double()[:, None] * dout[slot // top_k].double()
        tol = (ref.half_step(dtype) + 2 * ref.U32) * expect_rows.abs() + ref.TINY[dtype]
        assert bool(((drows.cpu().double() - expect_rows).abs() <= tol).all())
        terms = rows[live].double() * dout[slot // top_k].double()
        expect_w, size_w = torch.zeros(tokens * top_k, dtype=torch.float64), torch.zeros(tokens * top_k, dtype=torch.float64)
        expect_w[slot], size_w[slot] = terms.sum(1), terms.abs().sum(1)
        got = dweights.cpu().double().reshape(-1)
        assert bool(((got - expect_w).abs() <= (hidden / 32 + 16) * ref.U32 * size_w).all())
        # one gradient alone is the same gradient
        out = dmoe.unsort_tokens(dev, dev_w, plan)
        assert torch.equal(torch.autograd.grad(out, dev, dout.cuda(), retain_graph=True)[0], drows)
        assert torch.equal(torch.autograd.grad(out, dev_w, dout.cuda())[0], dweights)


def test_gradients_of_the_rows_against_differences():
    """In fp32 with inputs of a few bits, steps of 2^-4 and a function that is bilinear: differences are exact up to the
    roundings of the sums (about 300 terms of magnitude 1, so 300 * 2^-24 * 2^4 * 8 < 3e-3)."""
    from stk_b200 import dmoe
    g = torch.Generator().manual_seed(5)
    ids = torch.tensor([[0, 2], [1, -1], [2, 2], [0, 1]])
    plan = dmoe.plan_tokens(ids.cuda(), 3)
    x = (torch.randint(-8, 8, (4, 19), generator=g) / 8).cuda()
    w = (torch.randint(-8, 8, (4, 2), generator=g) / 8).cuda()
    scale = (torch.randint(-8, 8, (plan.rows, 19), generator=g) / 8).cuda()
    probe = (torch.randint(-8, 8, (4, 19), generator=g) / 8).cuda()

    def value(x, w):
        return (dmoe.unsort_tokens(dmoe.sort_tokens(x, plan) * scale, w, plan) * probe).sum()

    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    grads = torch.autograd.grad(value(xg, wg), (xg, wg))
    for which, t in enumerate((x, w)):
        for i in range(t.numel()):
            step = torch.zeros_like(t).view(-1)
            step[i] = 2.0 ** -4
            step = step.view_as(t)
            up = value(x + step, w) if which == 0 else value(x, w + step)
            down = value(x - step, w) if which == 0 else value(x, w - step)
            assert abs(float((up - down) * 8) - float(grads[which].view(-1)[i])) < 3e-3


def test_rows_take_views_and_weights_of_other_kinds():
    from stk_b200 import dmoe
    plan, g = rows_case(90, 64, 4, 2, torch.bfloat16)
    wide = torch.randn(90, 200, generator=g).to(torch.bfloat16).cuda()
    for view in (wide[:, :64], wide[:, 3:67], wide.t()[:90, :64], wide[:1, :64].expand(90, 64), wide[:, :0]):
        assert torch.equal(dmoe.sort_tokens(view, plan), dmoe.sort_tokens(view.contiguous(), plan))
    rows = torch.randn(plan.rows, 80, generator=g).to(torch.bfloat16).cuda()
    weights = torch.rand(90, 2, generator=g).cuda()
    expect = dmoe.unsort_tokens(rows[:, 8:72].contiguous(), weights, plan)
    assert torch.equal(dmoe.unsort_tokens(rows[:, 8:72], weights, plan), expect)
    assert torch.equal(dmoe.unsort_tokens(rows[:, 8:72], torch.stack((weights, weights), 2)[:, :, 0], plan), expect)
    # 16-bit weights: used as they are, gradient in their type
    w16 = weights.to(torch.bfloat16).requires_grad_()
    out = dmoe.unsort_tokens(rows, w16, plan)
    assert torch.equal(out, dmoe.unsort_tokens(rows, w16.detach().float(), plan))
    assert torch.autograd.grad(out.sum(), w16)[0].dtype == torch.bfloat16    # (a broadcast gradient, too)
    # no weights: ones
    leaf = rows.clone().requires_grad_()
    out = dmoe.unsort_tokens(leaf, None, plan)
    assert torch.equal(out, dmoe.unsort_tokens(rows, torch.ones(90, 2, device="cuda"), plan))
    grad, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert torch.equal(grad, (plan.index >= 0)[:, None].expand_as(grad).to(grad.dtype))
    # one choice a token: ids and weights may be flat
    flat = dmoe.plan_tokens(torch.randint(0, 3, (90,), generator=g).cuda(), 3)
    x = torch.randn(90, 33, generator=g).cuda()
    assert torch.equal(dmoe.unsort_tokens(dmoe.sort_tokens(x, flat), torch.ones(90, device="cuda"), flat), x)


def test_rows_of_plans_without_slots():
    """No slot has an expert: no row at all, or only padding."""
    from stk_b200 import dmoe
    none = torch.full((5, 2), -1, device="cuda")
    for ids, rows in ((none, None), (none, 1024), (none[:0], None), (none[:0], 256)):
        plan = dmoe.plan_tokens(ids, 4, rows=rows)
        assert plan.rows == (rows or 0) and bool((plan.index == -1).all()) and bool((plan.position == -1).all())
        assert plan.bin_rows.tolist() == [0, 0, 0, plan.block_rows]
        x = torch.randn(len(ids), 40, device="cuda", requires_grad=True)
        w = torch.rand(len(ids), 2, device="cuda", requires_grad=True)
        moved = dmoe.sort_tokens(x, plan)
        assert moved.shape == (plan.rows, 40) and not bool(moved.any())
        leaf = torch.full((plan.rows, 40), torch.nan, device="cuda", requires_grad=True)
        out = dmoe.unsort_tokens(leaf, w, plan)
        assert out.shape == x.shape and not bool(out.any())
        grads = torch.autograd.grad(out, (leaf, w), torch.ones_like(out))
        assert not bool(grads[0].any()) and not bool(grads[1].any())
        assert not bool(torch.autograd.grad(moved, x, torch.ones_like(moved))[0].any())


def test_backward_accumulates_and_takes_shared_use():
    """The same rows and weights used twice, and .backward() into leaves that hold gradients already."""
    from stk_b200 import dmoe
    plan, g = rows_case(50, 24, 3, 2, torch.float32)
    x = torch.randn(50, 24, generator=g).cuda().requires_grad_()
    w = torch.rand(50, 2, generator=g).cuda().requires_grad_()
    moved = dmoe.sort_tokens(x, plan)
    once = torch.autograd.grad(dmoe.unsort_tokens(moved, w, plan).sum(), (x, w), retain_graph=True)
    for _ in range(2):
        (dmoe.unsort_tokens(moved, w, plan).sum() + dmoe.unsort_tokens(moved, w, plan).sum()).backward(retain_graph=True)
    torch.testing.assert_close(x.grad, 4 * once[0], rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(w.grad, 4 * once[1], rtol=1e-6, atol=1e-6)


def test_rows_beyond_32_bit_offsets():
    from stk_b200 import dmoe
    tokens, hidden, top_k = 290000, 4096, 2               # 580000 rows and padding: 2.4e9 elements
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(0, 8, (tokens, top_k), generator=g, device="cuda")
    plan = dmoe.plan_tokens(ids, 8)
    x = torch.arange(tokens, device="cuda", dtype=torch.float32)[:, None].expand(tokens, hidden).to(torch.bfloat16)
    rows = dmoe.sort_tokens(x, plan)
    assert rows.numel() > 2 ** 31
    for r in (0, 1, plan.rows // 2, plan.rows - 130, plan.rows - 129):
        s = int(plan.index[r])
        assert torch.equal(rows[r], x[s // top_k] if s >= 0 else torch.zeros_like(rows[r]))
    weights = torch.full((tokens, top_k), 0.5, device="cuda")
    assert torch.equal(dmoe.unsort_tokens(rows, weights, plan), x)


# ------------------------------------------------------------------------------ together
def layer(x, router, w1, w2, top_k, fixed):
    """A dMoE layer as a training program writes it."""
    from stk_b200 import dmoe
    experts = router.shape[1]
    weights, ids = dmoe.top_k_gate(x @ router, top_k)
    rows = dmoe.plan_rows(ids.numel(), experts) if fixed else None
    plan = dmoe.plan_tokens(ids, experts, rows=rows)
    topo = dmoe.topology_from_bins(plan.bin_rows, plan.block_rows, w1.shape[1] // experts, x.dtype, x.device,
                                   materialize=False)
    y = dmoe.expert_mlp(dmoe.sort_tokens(x, plan), w1, w2, topo)
    return dmoe.unsort_tokens(y, weights, plan), ids


def layer_inputs(tokens, hidden, ffn, experts, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *shape, scale: (torch.randn(*shape, generator=g) * scale).to(dtype)
    return (make(tokens, hidden, scale=1.0), make(hidden, experts, scale=0.1), make(hidden, experts * ffn, scale=0.08),
            make(experts * ffn, hidden, scale=0.08))


@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("tokens,experts,top_k", [(300, 4, 2), (7, 4, 1), (513, 6, 3)])
def test_training_step_of_a_whole_layer(tokens, experts, top_k, fixed):
    """Against 64 bits, choices taken from the GPU's logits.  Every result went through at most eight roundings to the
    type on its way (logits, pre-activation, activation, experts' row, output, and the same back), each of half a step
    relative to the norm."""
    hidden, ffn, dtype = 128, 256, torch.float16
    inputs = layer_inputs(tokens, hidden, ffn, experts, dtype)
    dev = [t.cuda().requires_grad_() for t in inputs]
    out, ids = layer(*dev, top_k, fixed)
    dout = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(9)).to(dtype)
    grads = torch.autograd.grad(out, dev, dout.cuda())
    exact = [t.double().requires_grad_() for t in inputs]
    x, router, w1, w2 = exact
    logits = x @ router
    weights = torch.softmax(torch.gather(logits, 1, ids.cpu().long()), 1)
    expect = torch.zeros(tokens, hidden, dtype=torch.float64)
    for e in range(experts):
        y = torch.nn.functional.gelu(x @ w1[:, e * ffn:(e + 1) * ffn]) @ w2[e * ffn:(e + 1) * ffn]
        expect = expect + (weights * (ids.cpu() == e)).sum(1, keepdim=True) * y
    expect_grads = torch.autograd.grad(expect, exact, dout.double())
    for name, a, b in zip(("out", "x", "router", "w1", "w2"), (out.detach(), *grads), (expect.detach(), *expect_grads)):
        # (one choice with normalized weights: the router's gradient is zero, and has to be)
        assert float((a.cpu().double() - b).norm()) <= 8 * ref.half_step(dtype) * float(b.norm()), name


def test_training_step_captured_in_a_graph_equals_the_eager_one():
    """With the number of rows fixed in advance nothing waits for the device: forward and backward are captured once and
    replayed on other inputs.  (The gradients are asked for by torch.autograd.grad, which touches no leaf's accumulator.)"""
    tokens, hidden, ffn, experts, top_k, dtype = 200, 128, 256, 4, 2, torch.bfloat16
    inputs = [t.cuda() for t in layer_inputs(tokens, hidden, ffn, experts, dtype)]
    others = [t.cuda() for t in layer_inputs(tokens, hidden, ffn, experts, dtype, seed=1)]
    dout = torch.randn(tokens, hidden, device="cuda").to(dtype)

    def step(leaves):
        out, _ = layer(*leaves, top_k, True)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    eager = [[t.clone() for t in step([t.clone().requires_grad_() for t in some])] for some in (inputs, others)]
    static = [t.clone().requires_grad_() for t in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for some, expect in ((others, eager[1]), (inputs, eager[0]), (others, eager[1])):
        with torch.no_grad():
            for a, b in zip(static, some):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, expect):
            assert torch.equal(a, b)


def test_reading_the_rows_back_is_refused_while_capturing():
    from stk_b200 import dmoe
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    scratch = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scratch.add_(1)
        with pytest.raises(RuntimeError, match="plan_rows"):
            dmoe.plan_tokens(ids, 4)


def test_second_derivatives_are_refused():
    from stk_b200 import dmoe
    plan = dmoe.plan_tokens(torch.tensor([0, 1], device="cuda"), 2)
    x = torch.randn(2, 8, device="cuda", requires_grad=True)
    grad, = torch.autograd.grad((dmoe.sort_tokens(x, plan) ** 2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize("score,normalize", KINDS)
def test_gate_choices_without_an_expert_weigh_nothing_beside_nan_and_infinity(score, normalize):
    """Fewer than k logits above -inf, and one of them NaN or +inf: the choices that are left over have id -1 and weight 0, as
    on the host, and every choice of a row with a NaN has weight NaN."""
    from stk_b200 import dmoe
    for dtype in DTYPES:
        for experts in (3, 16, 40, 300):
            logits = torch.full((6, experts), -torch.inf, dtype=dtype)
            logits[0, 2], logits[1, 1] = torch.nan, torch.inf
            logits[2, 0], logits[2, 2] = torch.nan, 1.0
            logits[3, 0], logits[3, 2] = torch.inf, 1.0
            logits[4, 2], logits[4, 1] = 2.0, 1.0
            logits[5] = torch.nan
            weights, ids = dmoe.top_k_gate(logits.cuda(), 3, score=score, normalize=normalize)
            expect, expect_ids = dmoe.top_k_gate(logits, 3, score=score, normalize=normalize)
            assert torch.equal(ids.cpu(), expect_ids)
            torch.testing.assert_close(weights.cpu(), expect, rtol=128 * ref.U32, atol=0, equal_nan=True)
            assert not bool(weights[ids < 0].any())
            assert bool(weights[[0, 2, 5]][ids[[0, 2, 5]] >= 0].isnan().all())


def test_tangents_are_refused():
    """Forward-mode differentiation: the kernels refuse a dual tensor, with and without a graph, instead of dropping its
    tangent, and take the same tensors without one inside a dual level."""
    from torch.autograd import forward_ad
    from stk_b200 import dmoe
    plan = dmoe.plan_tokens(torch.tensor([[0, 1], [1, 2]], device="cuda"), 3)
    x, logits = torch.randn(2, 8, device="cuda"), torch.randn(2, 3, device="cuda")
    rows, weights = torch.randn(plan.rows, 8, device="cuda"), torch.rand(2, 2, device="cuda")
    w = dmoe.quantize_int4(torch.randn(3, 32, 32, device="cuda").half(), group=32)
    h, ids = torch.randn(2, 32, device="cuda").half(), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    calls = [lambda d: dmoe.top_k_gate(d(logits), 2), lambda d: dmoe.sort_tokens(d(x), plan),
             lambda d: dmoe.unsort_tokens(d(rows), weights, plan), lambda d: dmoe.unsort_tokens(rows, d(weights), plan),
             lambda d: dmoe.int4_matvec(d(h), w, ids), lambda d: dmoe.expert_mlp_int4(d(h), ids, weights, w, w),
             lambda d: dmoe.expert_mlp_int4(h, ids, d(weights), w, w)]
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in calls:
            call(lambda t: t)
            for context in (torch.enable_grad, torch.no_grad):
                with context(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(dual)
        leaf = x.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="forward-mode"):
            dmoe.sort_tokens(dual(leaf), plan)


def test_plan_with_bins_that_end_at_the_32_bit_limit():
    """One bin whose last row is 2^31 - 2: neither slots + block - 1 nor the walk over the padding fits 32 bits."""
    from stk_b200 import dmoe
    for block, ids in ((2 ** 31 - 1, [0, 0]), (2 ** 31 - 16, [0, -1, 0])):
        assert dmoe.plan_rows(len(ids), 1, block) == block
        for rows in (None, block):
            plan = dmoe.plan_tokens(torch.tensor(ids, device="cuda"), 1, block=block, rows=rows)
            assert plan.rows == block and plan.block_rows == 1 and plan.bin_rows.tolist() == [1]
            assert plan.position.tolist() == [i - (i > 0 and ids[1] < 0) if e >= 0 else -1 for i, e in enumerate(ids)]
            assert plan.index[:4].tolist() == [s for s, e in enumerate(ids) if e >= 0] + [-1, -1]
            assert bool((plan.index[2:] == -1).all())
            del plan


@pytest.mark.parametrize("tokens", [0, 6])
@pytest.mark.parametrize("fixed", [False, True])
def test_a_layer_on_a_batch_without_live_tokens(tokens, fixed):
    """No tokens, or padding alone: the step runs, its output and its gradients are zeros of their shapes."""
    from stk_b200 import dmoe
    hidden, ffn, experts = 128, 256, 4
    x, router, w1, w2 = (t.cuda().requires_grad_() for t in layer_inputs(tokens, hidden, ffn, experts, torch.float16))
    mask = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    weights, ids = dmoe.top_k_gate(x @ router, 2, token_mask=mask)
    plan = dmoe.plan_tokens(ids, experts, rows=512 if fixed else None)
    assert plan.rows == (512 if fixed else 0)
    topo = dmoe.topology_from_bins(plan.bin_rows, plan.block_rows, ffn, x.dtype, x.device, materialize=False)
    y = dmoe.expert_mlp(dmoe.sort_tokens(x, plan), w1, w2, topo)
    out = dmoe.unsort_tokens(y, weights, plan)
    assert out.shape == (tokens, hidden) and not bool(out.any())
    for leaf, grad in zip((x, router, w1, w2), torch.autograd.grad(out.float().sum(), (x, router, w1, w2))):
        assert grad.shape == leaf.shape and not bool(grad.any())
