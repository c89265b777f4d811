"""Products with 4-bit expert weights on the GPU against 64 bits.

Tolerance of a product of K inputs, with S = sum |w x|: half a step of the result's type, and (K / 32 + 16) 2^-24 S for the
32-bit sum over groups and parts (at most K / 32 group sums and 8 parts are added), and 2^-22 S for the sums inside the
products of 16 inputs (two to a group of 32, whose terms the tensor cores align to the largest before they add them)."""
import pytest
import torch

from tests.routing_reference import TINY, U32, half_step
from tests.test_int4_host import bits, values

pytestmark = pytest.mark.gpu


def check_matvec(tokens, top_k, experts, outputs, inputs, group, dtype, zeros, gelu=False, ids=None, seed=0):
    from stk_b200 import dmoe
    codes, packed, scales, zero = bits(experts, outputs, inputs, group, dtype, zeros, seed)
    move = lambda t: None if t is None else t.cuda()
    w = dmoe.pack_int4(move(packed), move(scales), move(zero))
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(tokens, inputs, generator=g).to(dtype)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=g) if ids is None else ids
    y = dmoe.int4_matvec(x.cuda(), w, ids.cuda(), gelu=gelu)
    assert y.shape == (tokens, top_k, outputs) and y.dtype == dtype
    full = values(codes, scales, zero, group)
    for t in range(tokens):
        for j in range(top_k):
            e = int(ids[t, j])
            got = y[t, j].cpu().double()
            if e < 0:
                assert not bool(got.any())
                continue
            expect, size = full[e] @ x[t].double(), full[e].abs() @ x[t].double().abs()
            error = ((inputs / 32 + 16) * U32 + 2.0 ** -22) * size
            if gelu:                                      # its slope is at most 1.13; its own roundings are a few 2^-24 of it
                expect = torch.nn.functional.gelu(expect)
                error = 1.13 * error + 1e-5 * expect.abs()
            tol = half_step(dtype) * expect.abs() + error + TINY[dtype]
            assert bool(((got - expect).abs() <= tol).all()), (t, j)


@pytest.mark.parametrize("tokens,top_k,experts,outputs,inputs,group", [
    (1, 1, 1, 1, 32, 32), (1, 2, 8, 64, 128, 128), (3, 2, 4, 17, 96, 32), (8, 1, 2, 130, 320, 64), (9, 2, 3, 48, 64, 64),
    (17, 3, 2, 100, 1024, 128), (40, 2, 5, 33, 160, 32), (300, 2, 3, 16, 128, 64), (2, 2, 300, 32, 64, 32)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_matvec(tokens, top_k, experts, outputs, inputs, group, zeros, dtype):
    check_matvec(tokens, top_k, experts, outputs, inputs, group, dtype, zeros)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_matvec_of_long_rows_and_gelu(dtype):
    check_matvec(2, 2, 4, 64, 14336, 128, dtype, False)
    check_matvec(5, 2, 2, 2064, 256, 64, dtype, True, gelu=True)
    check_matvec(12, 1, 1, 4096, 64, 64, dtype, False)


def test_the_same_expert_for_every_choice_and_for_none():
    check_matvec(70, 4, 3, 40, 128, 64, torch.bfloat16, False, ids=torch.full((70, 4), 1))
    check_matvec(4, 2, 30, 40, 128, 64, torch.float16, True, ids=torch.full((4, 2), 29))
    check_matvec(4, 2, 30, 40, 128, 64, torch.float16, True, ids=torch.full((4, 2), -1))
    check_matvec(40, 2, 3, 40, 128, 64, torch.float16, True, ids=torch.full((40, 2), -1))


@pytest.mark.parametrize("tokens,experts,outputs,inputs,group,zeros", [
    (6, 8, 14336, 2176, 128, False), (20, 4, 9000, 4096, 64, True), (24, 3, 5000, 1120, 32, True), (160, 2, 2000, 640, 64, False)])
def test_shares_of_many_rows(tokens, experts, outputs, inputs, group, zeros):
    """Enough rows that a block takes them in groups of every size, and changes experts on its way; more slots than one
    launch takes.  Against 64 bits on the GPU."""
    from stk_b200 import dmoe
    dtype = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(outputs)
    packed = torch.randint(0, 256, (experts, outputs, inputs // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 + 0.02 * torch.rand(experts, outputs, inputs // group, generator=g, device="cuda")).to(dtype)
    zero = torch.randint(0, 16, scales.shape, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    w = dmoe.pack_int4(packed, scales, zero)
    x = torch.randn(tokens, inputs, generator=g, device="cuda").to(dtype)
    ids = torch.randint(0, experts, (tokens, 2), generator=g, device="cuda")
    y = dmoe.int4_matvec(x, w, ids)
    for e in range(experts):
        full = w.dequantize(torch.float32)[e].double()
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        expect, size = x[token].double() @ full.t(), x[token].double().abs() @ full.abs().t()
        tol = half_step(dtype) * expect.abs() + ((inputs / 32 + 16) * U32 + 2.0 ** -22) * size
        assert bool(((y[token, choice].double() - expect).abs() <= tol).all())
    assert torch.equal(y, dmoe.int4_matvec(x, w, ids))


def test_one_matrix_views_and_streams():
    from stk_b200 import dmoe
    codes, packed, scales, zero = bits(1, 50, 128, 64, torch.bfloat16, True)
    w = dmoe.pack_int4(packed, scales, zero).to("cuda")
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(6, 300, generator=g).bfloat16().cuda()
    x = wide[:, 1:129]                                    # neither contiguous nor on a 16-byte boundary
    y = dmoe.int4_matvec(x, w)
    assert y.shape == (6, 50)
    assert torch.equal(y, dmoe.int4_matvec(x.contiguous(), w, torch.zeros(6, 1, dtype=torch.int64, device="cuda"))[:, 0])
    flat = torch.empty(1 + 128, dtype=torch.bfloat16, device="cuda")[1:].view(1, 128)
    flat.copy_(x[:1])
    assert torch.equal(dmoe.int4_matvec(flat, w), y[:1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = dmoe.int4_matvec(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, y)
    assert dmoe.int4_matvec(x[:0], w).shape == (0, 50)
    with pytest.raises(ValueError, match="forward only"):
        dmoe.int4_matvec(x.detach().requires_grad_(), w)


def test_non_finite_inputs_stay_in_their_own_results():
    """The products take eight slots at a time: a NaN of one does not reach the others, nor a slot without an expert."""
    from stk_b200 import dmoe
    _, packed, scales, zero = bits(2, 32, 128, 64, torch.float16, False)
    w = dmoe.pack_int4(packed, scales, zero).to("cuda")
    x = torch.randn(5, 128, generator=torch.Generator().manual_seed(3)).half().cuda()
    ids = torch.tensor([[0], [0], [-1], [1], [0]], device="cuda")
    clean = dmoe.int4_matvec(x, w, ids)
    x[1, 7], x[2, 3] = torch.nan, torch.nan
    got = dmoe.int4_matvec(x, w, ids)
    assert bool(got[1].isnan().all())
    for t in (0, 2, 3, 4):
        assert torch.equal(got[t], clean[t])
    weights = torch.ones(5, 1, device="cuda")
    _, packed, scales, zero = bits(2, 128, 32, 32, torch.float16, False)
    w2 = dmoe.pack_int4(packed, scales, zero).to("cuda")
    out = dmoe.expert_mlp_int4(x, ids, weights, w, w2)
    assert not bool(out[2].any()) and bool(out[1].isnan().all()) and bool(out[[0, 3, 4]].isfinite().all())


def test_experts_that_do_not_exist_are_reported():
    from stk_b200 import dmoe
    from stk_b200.backend import lib
    _, packed, scales, zero = bits(3, 32, 64, 64, torch.float16, False)
    w = dmoe.pack_int4(packed, scales, zero).to("cuda")
    x = torch.randn(4, 64, device="cuda").half()
    assert lib.device_status() == 0
    y = dmoe.int4_matvec(x, w, torch.tensor([[0], [3], [1], [-1]], device="cuda"))
    assert lib.device_status() == -2 and lib.device_status() == 0
    assert not bool(y[1].any()) and not bool(y[3].any()) and bool(y[0].any())
    for far in (77, 2 ** 32, 2 ** 33 + 1):
        y = dmoe.int4_matvec(x[:1], w, torch.tensor([[far]], device="cuda"))
        assert lib.device_status() == -2 and not bool(y.any())


def mlp64(x, ids, weights, first, second):
    """(out, sums of magnitudes over both products) in 64 bits."""
    out = torch.zeros(x.shape[0], second.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if e >= 0:
                h = torch.nn.functional.gelu(first[e] @ x[t].double())
                out[t] += weights[t, j].double() * (second[e] @ h)
                size[t] += weights[t, j].double().abs() * (second[e].abs() @ h.abs())
    return out, size


@pytest.mark.parametrize("tokens,top_k,experts,hidden,ffn,group,zeros,dtype", [
    (1, 2, 8, 128, 512, 128, False, torch.float16), (5, 2, 4, 96, 320, 32, True, torch.bfloat16),
    (16, 2, 8, 256, 1024, 128, False, torch.bfloat16), (64, 2, 16, 128, 192, 64, True, torch.bfloat16),
    (33, 4, 4, 64, 128, 64, False, torch.float16)])
def test_mlp(tokens, top_k, experts, hidden, ffn, group, zeros, dtype):
    """The hidden activations are rounded once to the type: half a step of it times sum |w2 h| at the very most; in the
    2-norm the roundings of thousands of activations do not line up, and the result is within two roundings."""
    from stk_b200 import dmoe
    one, two = bits(experts, ffn, hidden, group, dtype, zeros, 1), bits(experts, hidden, ffn, group, dtype, zeros, 2)
    move = lambda t: None if t is None else t.cuda()
    w1, w2 = (dmoe.pack_int4(*map(move, b[1:])) for b in (one, two))
    g = torch.Generator().manual_seed(4)
    x = torch.randn(tokens, hidden, generator=g).to(dtype)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=g)
    weights = torch.rand(tokens, top_k, generator=g)
    out = dmoe.expert_mlp_int4(x.cuda(), ids.cuda(), weights.cuda(), w1, w2)
    expect, size = mlp64(x, ids, weights, values(one[0], one[2], one[3], group), values(two[0], two[2], two[3], group))
    assert out.dtype == dtype
    off = out.cpu().double() - expect
    tol = half_step(dtype) * (expect.abs() + 1.1 * size) + 2e-4 * size + TINY[dtype]
    assert bool((off.abs() <= tol).all())
    assert float(off.norm() / expect.norm()) <= 2 * half_step(dtype)
    again = dmoe.expert_mlp_int4(x.cuda(), ids.cuda(), weights.cuda(), w1, w2)
    assert torch.equal(out, again)


def test_decoding_step_with_the_gate_and_captured():
    """gate -> 4-bit experts as a serving program runs it, eager and replayed from a graph on other tokens; two graphs
    replayed at once on two streams do not disturb each other."""
    from stk_b200 import dmoe
    experts, hidden, ffn, top_k = 8, 256, 512, 2
    g = torch.Generator().manual_seed(5)
    router = (torch.randn(hidden, experts, generator=g) * 0.1).half().cuda()
    w1 = dmoe.quantize_int4((torch.randn(experts, hidden, ffn, generator=g) * 0.08).half().cuda(), group=64)
    w2 = dmoe.quantize_int4((torch.randn(experts, ffn, hidden, generator=g) * 0.08).half().cuda(), group=64, zero_points=True)
    batches = [torch.randn(6, hidden, generator=g).half().cuda() for _ in range(4)]

    def step(x):
        weights, ids = dmoe.top_k_gate(x @ router, top_k)
        return dmoe.expert_mlp_int4(x, ids, weights, w1, w2), ids

    eager = [step(x) for x in batches]
    first, second = (w.dequantize(torch.float64).cpu() for w in (w1, w2))
    for x, (out, ids) in zip(batches, eager):
        logits = (x @ router).double().cpu()
        weights = torch.softmax(torch.gather(logits, 1, ids.cpu().long()), 1)
        expect, _ = mlp64(x.cpu(), ids.cpu(), weights, first, second)
        assert float((out.cpu().double() - expect).norm() / expect.norm()) <= 2 * half_step(torch.float16)
    graphs, inputs, outputs, streams = [], [], [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        inputs.append(batches[0].clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append(step(inputs[i])[0])
        graphs.append(graph)
    for turn in range(20):
        a, b = turn % 4, (turn * 3 + 1) % 4
        torch.cuda.synchronize()
        for i, which in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                inputs[i].copy_(batches[which])
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outputs[0], eager[a][0]) and torch.equal(outputs[1], eager[b][0])


def test_calls_in_a_row_between_other_kernels():
    """Launches that begin while the one before them runs out: many short calls back to back, between products and gates of
    the same stream, give what each gives alone."""
    import stk_b200 as stk
    from stk_b200 import dmoe
    experts, hidden, ffn = 4, 128, 256
    g = torch.Generator().manual_seed(8)
    make = lambda *shape: (torch.randn(*shape, generator=g) * 0.1).half().cuda()
    w1, w2 = dmoe.quantize_int4(make(experts, hidden, ffn)), dmoe.quantize_int4(make(experts, ffn, hidden))
    topo = dmoe.topology_from_bins(torch.ones(experts, dtype=torch.int32, device="cuda"), experts, ffn, torch.float16, "cuda")
    a, b = make(experts * 128, hidden), make(hidden, experts * ffn)
    batches = [(make(t, hidden) * 10, torch.randint(-1, experts, (t, 2), generator=g).cuda(), torch.rand(t, 2, generator=g).cuda())
               for t in (1, 3, 150, 17)]

    def step(x, ids, weights):
        out = dmoe.expert_mlp_int4(x, ids, weights, w1, w2)
        product = stk.ops.sdd(a, b, topo).data
        plan = dmoe.plan_tokens(ids.repeat(30, 1), experts, rows=dmoe.plan_rows(60 * len(ids), experts))
        return out, dmoe.int4_matvec(x, w1, ids), product, plan.position

    alone = []
    for batch in batches:
        torch.cuda.synchronize()
        alone.append(step(*batch))
        torch.cuda.synchronize()
    for _ in range(50):
        for batch, expect in zip(batches, alone):
            assert all(torch.equal(p, q) for p, q in zip(step(*batch), expect))


def test_quantized_experts_stay_near_the_16_bit_ones():
    """quantize_int4 takes dmoe.expert_mlp's weights in the documented views: the two forms of the layer agree up to what
    4 bits lose.  Every weight is off by half a scale at most, a scale being a seventh of the group's largest
    magnitude (about 3 standard deviations for 128 normal values): 0.29 * 3 / 7 = 0.12 of a standard deviation, so each
    product by 0.12 of its own norm, and the two in a row by 0.12 * 2 and the second order; 0.3 in all."""
    from stk_b200 import dmoe
    experts, hidden, ffn, tokens = 4, 256, 512, 9
    g = torch.Generator().manual_seed(6)
    w1 = (torch.randn(hidden, experts * ffn, generator=g) * 0.08).bfloat16().cuda()
    w2 = (torch.randn(experts * ffn, hidden, generator=g) * 0.08).bfloat16().cuda()
    x = torch.randn(tokens, hidden, generator=g).bfloat16().cuda()
    weights, ids = dmoe.top_k_gate(torch.randn(tokens, experts, generator=g).cuda(), 2)
    plan = dmoe.plan_tokens(ids, experts)
    topo = dmoe.topology_from_bins(plan.bin_rows, plan.block_rows, ffn, x.dtype, x.device, materialize=False)
    full = dmoe.unsort_tokens(dmoe.expert_mlp(dmoe.sort_tokens(x, plan), w1, w2, topo), weights, plan).float()
    small = dmoe.expert_mlp_int4(x, ids, weights, dmoe.quantize_int4(w1.view(hidden, experts, ffn).transpose(0, 1)),
                                 dmoe.quantize_int4(w2.view(experts, ffn, hidden))).float()
    assert float((small - full).norm() / full.norm()) <= 0.3


@pytest.mark.parametrize("tokens,inputs,group", [(3, 256, 128), (12, 192, 64), (16, 1024, 32), (1, 96, 32)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_inputs_under_zero_weights_add_nothing(tokens, inputs, group, zeros, dtype):
    """Codes at the zero point stand for weights of 0: inputs of 3e4 under them leave a result within the tolerance above,
    whose S does not know them, and a row of such codes gives exactly 0, whatever its scales are.  (0 times a finite
    number is 0 in the products and aligns no other term.)  Inputs with a large mean have a large S and are within it."""
    from stk_b200 import dmoe
    outputs = 50
    codes, _, scales, zero = bits(1, outputs, inputs, group, dtype, zeros, 11)
    point = torch.full_like(codes, 8) if zero is None else zero.repeat_interleave(group, 2)
    codes[:, :, ::7] = point[:, :, ::7]
    nothing = [0, 3, 9, 21, 49]
    codes[:, nothing] = point[:, nothing]
    w = dmoe.pack_int4((codes[..., 0::2] | (codes[..., 1::2] << 4)).cuda(), scales.cuda(), None if zero is None else zero.cuda())
    full = values(codes, scales, zero, group)[0]
    g = torch.Generator().manual_seed(12)
    x = torch.randn(tokens, inputs, generator=g)
    outliers = x.clone()
    outliers[:, ::7] = 3e4 * torch.sign(x[:, ::7])
    for some in (outliers.to(dtype), (x + 200).to(dtype)):
        y = dmoe.int4_matvec(some.cuda(), w).cpu().double()
        assert not bool(y[:, nothing].any())
        expect, size = some.double() @ full.t(), some.double().abs() @ full.abs().t()
        tol = half_step(dtype) * expect.abs() + ((inputs / 32 + 16) * U32 + 2.0 ** -22) * size + TINY[dtype]
        assert bool(((y - expect).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gelu_of_exact_products(dtype):
    """One input under a weight of 1: the product is exact, and what remains is the GeLU's own error: (x^2 + 8) 2^-23 of it (its
    argument is rounded twice, by 2^-24 each, which x^2 multiplies in the negative tail; erfc and two products add a few 2^-24), half a
    step of the type, and half the type's smallest step."""
    from stk_b200 import dmoe
    v = torch.tensor([0.0, 1e-6, -1e-6, 1e-3, -1e-3, 0.05, -0.05, 0.5, -0.5, 1.0, -1.0, 2.5, -2.5, 4.0, -4.0, 5.8, -5.8, -6.5, -7.9, 8.0,
                      -8.0, -8.1, -8.5, -9.0, -10.0, -12.0, -13.0, -14.0, -17.0, -100.0, -3e4, 12.0, 3e4]).to(dtype)
    codes = torch.full((1, 32, 32), 8, dtype=torch.uint8)
    codes[0, :, 5] = 9
    w = dmoe.pack_int4((codes[..., 0::2] | (codes[..., 1::2] << 4)).cuda(), torch.ones(1, 32, 1, dtype=dtype, device="cuda"))
    x = torch.zeros(len(v), 32, dtype=dtype)
    x[:, 5] = v
    y = dmoe.int4_matvec(x.cuda(), w, gelu=True).cpu().double()
    exact = v.double()
    expect = (0.5 * exact * torch.special.erfc(-exact * 0.5 ** 0.5))[:, None]
    tol = (half_step(dtype) + (exact.clamp(max=0) ** 2 + 8)[:, None] * 2 * U32) * expect.abs() + TINY[dtype]
    assert bool(((y - expect).abs() <= tol).all())


@pytest.mark.parametrize("inputs,group", [(32, 32), (64, 64), (160, 32), (192, 64), (128, 128)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinite_inputs(inputs, group, zeros, dtype):
    """An infinity goes into its results as the formula has it, also where a record of 128 inputs is not full."""
    from stk_b200 import dmoe
    codes = torch.full((1, 32, inputs // 2), 0x99, dtype=torch.uint8, device="cuda")
    scales = torch.ones(1, 32, inputs // group, dtype=dtype, device="cuda")
    w = dmoe.pack_int4(codes, scales, torch.full_like(scales, 8, dtype=torch.uint8) if zeros else None)
    for at in (5, inputs - 32, inputs - 1):
        x = torch.ones(4, inputs, dtype=dtype, device="cuda")
        x[0, at], x[1, at], x[2, at] = torch.inf, -torch.inf, torch.nan
        y = dmoe.int4_matvec(x, w)
        assert bool((y[0] == torch.inf).all()) and bool((y[1] == -torch.inf).all()) and bool(y[2].isnan().all())
        assert bool((y[3] == inputs).all())
        y = dmoe.int4_matvec(x, w, gelu=True)
        assert bool((y[0] == torch.inf).all()) and bool((y[1] == 0).all()) and bool(y[2].isnan().all())


def test_first_calls_of_two_threads_at_once():
    """Each kernel's first launch looks its device up; two threads may do so at the same time."""
    import threading
    from stk_b200 import dmoe
    cases, wrong = [], []
    for seed, (group, zeros, dtype) in enumerate([(32, True, torch.float16), (64, False, torch.bfloat16), (128, True, torch.bfloat16)]):
        _, packed, scales, zero = bits(3, 96, 256, group, dtype, zeros, seed)
        w = dmoe.pack_int4(packed, scales, zero).to("cuda")
        g = torch.Generator().manual_seed(seed)
        cases.append((torch.randn(5, 256, generator=g).to(dtype).cuda(), w, torch.randint(-1, 3, (5, 2), generator=g).cuda()))
    start = threading.Barrier(2)

    def work(out):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(20):
                    out.append([dmoe.int4_matvec(*c) for c in cases])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    torch.cuda.synchronize()
    results = [[], []]
    threads = [threading.Thread(target=work, args=(r,)) for r in results]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong
    alone = [dmoe.int4_matvec(*c) for c in cases]
    assert all(torch.equal(a, b) for r in results for turn in r for a, b in zip(turn, alone))
