"""4-bit expert weights on the host: the layout and back, the quantiser, and what the calls refuse."""
import pytest
import torch


def bits(experts, outputs, inputs, group, dtype, zeros, seed=0):
    """(codes [E, N, K] 0..15, packed two a byte, scales, zeros)"""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (experts, outputs, inputs), generator=g, dtype=torch.uint8)
    packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
    scales = (0.01 + 0.02 * torch.rand(experts, outputs, inputs // group, generator=g)).to(dtype)
    zero = torch.randint(0, 16, scales.shape, generator=g, dtype=torch.uint8) if zeros else None
    return codes, packed, scales, zero


def values(codes, scales, zero, group):
    """What the codes stand for, [E, N, K] in 64 bits."""
    spread = lambda t: t.double().repeat_interleave(group, 2)
    return (codes.double() - (8 if zero is None else spread(zero))) * spread(scales)


@pytest.mark.parametrize("experts,outputs,inputs,group", [(1, 1, 32, 32), (2, 16, 64, 64), (3, 17, 96, 32), (2, 40, 128, 128),
                                                          (1, 130, 320, 64), (2, 33, 384, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_pack_and_back(experts, outputs, inputs, group, zeros):
    from stk_b200 import dmoe
    codes, packed, scales, zero = bits(experts, outputs, inputs, group, torch.float16, zeros)
    w = dmoe.pack_int4(packed, scales, zero)
    assert (w.num_experts, w.outputs, w.inputs, w.group, w.dtype) == (experts, outputs, inputs, group, torch.float16)
    assert torch.equal(w.dequantize(torch.float64), values(codes, scales, zero, group))


def test_layout_of_one_record():
    """The documented place of a weight: strip, half, lane (g, t), word 2h + s, nibble 4b + 2p + r; and of its scale and
    zero point: group, strip, g, r."""
    from stk_b200 import dmoe
    for row, col in ((0, 0), (5, 1), (8, 2), (23, 63), (31, 127), (17, 100), (40, 190)):
        codes = torch.zeros(1, 64, 256, dtype=torch.uint8)
        codes[0, row, col] = 15
        scales, zeros = torch.zeros(1, 64, 4, dtype=torch.float16), torch.zeros(1, 64, 4, dtype=torch.uint8)
        scales[0, row, col // 64], zeros[0, row, col // 64] = 1.0, 7
        w = dmoe.pack_int4(codes[..., 0::2] | (codes[..., 1::2] << 4), scales, zeros)
        assert w.records.shape == (1, 2, 2, 2048 + 128 + 64) and int((w.records != 0).sum()) in (3, 4)
        record = w.records[0, row // 32, col // 128].clone()
        strip, r, g, half = row % 32 // 16, row % 16 // 8, row % 8, col % 128 // 64
        h, t, s, p, b = col % 64 // 32, col % 32 // 8, col % 8 // 4, col % 4 // 2, col % 2
        expect = 15 << 4 * (4 * b + 2 * p + r)            # turned left by 6 bits for float16
        expect = (expect << 6 | expect >> 26) & 0xffffffff
        words = record[:2048].view(torch.int32).view(2, 2, 32, 4)
        assert int(words[strip, half, 4 * g + t, 2 * h + s]) & 0xffffffff == expect
        assert float(record[2048:2176].view(torch.float16).view(2, 2, 8, 2)[half, strip, g, r]) == 1.0
        assert int(record[2176:].view(2, 2, 8, 2)[half, strip, g, r]) == 7


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantize_is_within_half_a_step(zero_points, dtype):
    """A value is off by half a scale, and by what the scale's own rounding (half a step of its type, times a code of
    at most 15) and the clamp to 0..15 that it can cause take: 0.5 + 16 * half a step of the type, in scales.  With zero
    points, rounding the zero point moves the ends of the range by half a scale more."""
    from stk_b200 import dmoe
    g = torch.Generator().manual_seed(3)
    w = (torch.randn(2, 256, 48, generator=g) * 0.05).to(dtype)
    w[0, :64, 5] = 0.0                                    # a group of zeros stays one
    q = dmoe.quantize_int4(w, group=64, zero_points=zero_points)
    back = q.dequantize(torch.float64)
    v = w.double().transpose(1, 2).reshape(2, 48, 4, 64)
    step = (v.amax(3).clamp(min=0) - v.amin(3).clamp(max=0)) / 15 if zero_points else v.abs().amax(3) / 7
    scales = step.to(dtype).double().repeat_interleave(64, 2)
    bound = (0.5 + (0.5 if zero_points else 0) + 16 * torch.finfo(dtype).eps / 2) * scales
    assert bool(((back - w.double().transpose(1, 2)).abs() <= bound).all())
    assert not bool(back[0, 5, :64].any())


def test_refusals():
    from stk_b200 import dmoe
    _, packed, scales, zero = bits(2, 16, 128, 64, torch.float16, True)
    for bad in (lambda: dmoe.pack_int4(packed[0], scales), lambda: dmoe.pack_int4(packed.int(), scales),
                lambda: dmoe.pack_int4(packed, scales.float()), lambda: dmoe.pack_int4(packed, scales[:, :8]),
                lambda: dmoe.pack_int4(packed, scales[:, :, :0]), lambda: dmoe.pack_int4(packed, scales.repeat(1, 1, 4)),
                lambda: dmoe.pack_int4(packed, scales, zero.int()), lambda: dmoe.pack_int4(packed, scales, zero[:1]),
                lambda: dmoe.pack_int4(packed, scales, zero + 16),
                lambda: dmoe.pack_int4(torch.zeros(1, 1, 513 * 16, dtype=torch.uint8), torch.ones(1, 1, 513).half()),
                lambda: dmoe.pack_int4(packed[:0], scales[:0]),
                lambda: dmoe.quantize_int4(torch.randn(2, 64, 8)), lambda: dmoe.quantize_int4(torch.randn(64, 8).half()),
                lambda: dmoe.quantize_int4(torch.randn(2, 96, 8).half()),
                lambda: dmoe.quantize_int4(torch.randn(2, 64, 8).half(), group=16)):
        with pytest.raises(ValueError):
            bad()
    w = dmoe.pack_int4(packed, scales, zero)
    x, ids = torch.randn(3, 128).half(), torch.zeros(3, 2, dtype=torch.int32)
    for bad in (lambda: dmoe.int4_matvec(x, packed, ids), lambda: dmoe.int4_matvec(x[:, :64], w, ids),
                lambda: dmoe.int4_matvec(x.bfloat16(), w, ids), lambda: dmoe.int4_matvec(x, w, ids[:2]),
                lambda: dmoe.int4_matvec(x, w, ids.float()), lambda: dmoe.int4_matvec(x, w, ids[:, 0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        dmoe.int4_matvec(x, w, ids)


def test_entry_points_check_before_any_launch():
    from stk_b200.backend import lib
    L = lib.load()
    p = 4096                                              # an aligned address that is never read
    call = lambda slots=4, div=2, experts=2, n=16, k=128, group=64, dtype=1, x=p, words=p: L.stk_b200_int4_matvec(
        words, x, p, p, slots, div, experts, n, k, group, 0, 0, 0, dtype, None)
    assert [L.stk_b200_int4_record_bytes(g, z) for g in (16, 32, 64, 128) for z in (0, 1)] == [
        0, 0, 2304, 2432, 2176, 2240, 2112, 2144]
    assert call(slots=0) == 0 and call(slots=-1) == -2 and call(div=0) == -2 and call(experts=0) == -2 and call(n=0) == -2
    assert call(k=96) == -2 and call(group=16) == -2 and call(dtype=3) == -3 and call(dtype=2) == -3
    assert call(k=513 * 64) == -9 and call(experts=70000) == -9 and call(x=None) == -1 and call(x=p + 2) == -4 and call(words=p + 8) == -4
    mlp = lambda tokens=4, k=2, outputs=128, group=64, weights=p, ws=p, size=1 << 20, dtype=1: L.stk_b200_int4_mlp(
        p, p, p, p, weights, p, tokens, k, 2, 128, 256, outputs, group, 0, 64, 0, dtype, ws, size, None)
    assert mlp(tokens=0) == 0 and mlp(tokens=-1) == -2 and mlp(k=0) == -2 and mlp(outputs=0) == -2 and mlp(group=48) == -2
    assert mlp(weights=None) == -1 and mlp(ws=None) == -7 and mlp(ws=p + 4) == -7 and mlp(size=8191) == -7
    assert mlp(dtype=3) == -3 and mlp(tokens=1 << 31) == -9
    assert L.stk_b200_int4_mlp_workspace_bytes(8, 256, 128) == 8192 and L.stk_b200_int4_mlp_workspace_bytes(0, 256, 128) == 0


def test_tangents_are_refused_before_any_launch():
    """A dual tensor of forward-mode differentiation requires no gradient; its tangent must not be dropped without a word."""
    from torch.autograd import forward_ad
    from stk_b200 import dmoe
    w = dmoe.quantize_int4(torch.randn(2, 64, 64).half(), group=64)
    x, ids, weights = torch.randn(3, 64).half(), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, 2)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: dmoe.int4_matvec(dual, w, ids), lambda: dmoe.expert_mlp_int4(dual, ids, weights, w, w)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            dmoe.int4_matvec(x, w, ids)                   # (no tangent: the next check's)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        dmoe.int4_matvec(x, w, ids)


def test_the_mlp_checks_its_second_product_before_the_first_one_runs():
    """Without a device a launch fails with another code than these."""
    from stk_b200.backend import lib
    L = lib.load()
    p = 4096                                              # an aligned address that is never read
    mlp = lambda second=p, outputs=128, ffn=256, group=64: L.stk_b200_int4_mlp(
        p, second, p, p, p, p, 4, 2, 2, 128, ffn, outputs, 64, 0, group, 0, 1, p, 1 << 40, None)
    assert mlp(group=48) == -2 and mlp(group=64, ffn=96) == -2 and mlp(second=None) == -1 and mlp(second=p + 8) == -4
    assert mlp(outputs=(1 << 20) + 32) == -9 and mlp(ffn=513 * 64) == -9
