"""Experts with 4-bit weights for decoding: few tokens, whose products are bound by the bytes of the chosen experts'
weights.  Public as stk_b200.dmoe.pack_int4 / quantize_int4 / int4_matvec / expert_mlp_int4.

A weight stands for (code - zero) * scale, code 0..15, with a scale and a zero point (8 unless given) for each output
row and group of 32, 64 or 128 inputs.  Beside dmoe.expert_mlp, which wants the tokens in bins of 128 rows, the
products here take tokens and expert choices as they are.  Forward only; CUDA only, like the block-sparse products.
The reference has no counterpart.
"""
import torch

from stk_b200.backend import lib as _lib
from stk_b200.routing import ids32, refuse_tangents

GROUPS = (32, 64, 128)
MAX_EXPERTS = 1024
MAX_GROUPS = 512       # of the inputs
# Where in a 16-bit float with the exponent of 16 the step is 1: the first bit of a code (int4_sm100.cuh).
_BITS = {torch.float16: 6, torch.bfloat16: 3}


def _turn(words, bits):
    """The int32 words turned left by `bits`."""
    return (words << bits) | ((words >> (32 - bits)) & ((1 << bits) - 1))


class Int4Experts:
    """The 4-bit weights [num_experts, outputs, inputs] of a set of experts in the kernels' layout (pack_int4): records of
    32 outputs x 128 inputs, each with its codes, scales and zero points."""

    __slots__ = ("records", "num_experts", "outputs", "inputs", "group", "zero_points", "dtype")

    def __init__(self, records, num_experts, outputs, inputs, group, zero_points, dtype):
        self.records, self.dtype, self.zero_points = records, dtype, zero_points
        self.num_experts, self.outputs, self.inputs, self.group = num_experts, outputs, inputs, group

    @property
    def device(self):
        return self.records.device

    def to(self, device):
        return Int4Experts(self.records.to(device), self.num_experts, self.outputs, self.inputs, self.group,
                           self.zero_points, self.dtype)

    def dequantize(self, dtype=torch.float32):
        """The weights as numbers, [num_experts, outputs, inputs]."""
        records = self.records
        e, blocks, units, _ = records.shape
        n = 128 // self.group                           # groups of a record
        words = _turn(records[..., :2048].contiguous().view(torch.int32), 32 - _BITS[self.dtype])
        b = words.view(torch.uint8).view(e, blocks, units, 2, 2, 8, 4, 2, 2, 2, 2)  # strip, half, g, t, h, s, b, p
        codes = torch.stack((b & 15, b >> 4), dim=-1)                               # ..., r
        codes = codes.permute(0, 1, 3, 11, 5, 2, 4, 7, 6, 8, 10, 9)                 # strip r g, unit half h t s p b
        codes = codes.reshape(e, blocks * 32, units * n, self.group).to(dtype)
        per_row = lambda t: t.view(e, blocks, units, n, 2, 8, 2).permute(0, 1, 4, 6, 5, 2, 3).reshape(
            e, blocks * 32, units * n, 1).to(dtype)    # strip r g, unit group
        zero = per_row(records[..., 2048 + 64 * n:].contiguous()) if self.zero_points else 8
        scales = per_row(records[..., 2048:2048 + 64 * n].contiguous().view(self.dtype))
        whole = ((codes - zero) * scales).view(e, blocks * 32, units * 128)
        return whole[:, :self.outputs, :self.inputs].contiguous()


def pack_int4(codes, scales, zeros=None):
    """Int4Experts from weights as checkpoints hold them.

    codes: uint8 [E, N, K / 2], two codes a byte along the inputs, the lower four bits first; scales: [E, N, K / group]
    float16 or bfloat16 (the type of the activations); zeros: uint8 [E, N, K / group] with values 0..15, or None for 8
    everywhere.  One matrix without experts is E = 1.  Done once, when weights are loaded."""
    if codes.dim() != 3 or codes.dtype != torch.uint8:
        raise ValueError(f"pack_int4: codes must be uint8 [experts, outputs, inputs / 2], got {codes.dtype} "
                         f"{tuple(codes.shape)}")
    experts, outputs, inputs = codes.shape[0], codes.shape[1], 2 * codes.shape[2]
    if min(experts, outputs, inputs) < 1 or experts > MAX_EXPERTS:
        raise ValueError(f"pack_int4: 1 to {MAX_EXPERTS} experts with weights, got {tuple(codes.shape)}")
    if scales.dim() != 3 or tuple(scales.shape[:2]) != (experts, outputs) or scales.shape[2] < 1 \
            or inputs % scales.shape[2] or inputs // scales.shape[2] not in GROUPS:
        raise ValueError(f"pack_int4: scales must be [{experts}, {outputs}, {inputs} / group] with a group of "
                         f"{', '.join(map(str, GROUPS))} inputs, got {tuple(scales.shape)}")
    if scales.shape[2] > MAX_GROUPS:
        raise ValueError(f"pack_int4: at most {MAX_GROUPS} groups of inputs, got {scales.shape[2]}")
    if scales.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"pack_int4: scales are float16 or bfloat16, got {scales.dtype}")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError(f"pack_int4: zeros must be uint8 {tuple(scales.shape)}, got {zeros.dtype} {tuple(zeros.shape)}")
    if len({t.device for t in (codes, scales, zeros) if t is not None}) > 1:
        raise ValueError("pack_int4: codes, scales and zeros must be on one device")
    if zeros is not None and bool((zeros > 15).any()):
        raise ValueError("pack_int4: zero points are 0..15")
    group, blocks, units = inputs // scales.shape[2], (outputs + 31) // 32, (inputs + 127) // 128
    n = 128 // group                                    # groups of a record
    size = _lib.load().stk_b200_int4_record_bytes(group, int(zeros is not None))
    records = torch.empty((experts, blocks, units, size), dtype=torch.uint8, device=codes.device)
    pad = torch.nn.functional.pad
    more = 32 * blocks - outputs
    for e in range(experts):                           # (one at a time: no second copy of all weights)
        v = pad(codes[e], (0, 64 * units - inputs // 2, 0, more)).view(blocks, 2, 2, 8, units, 2, 2, 4, 2, 2)
        lo, hi = v[:, :, 0], v[:, :, 1]                 # rows g and g + 8: strip, g, unit, half, h, t, s, p
        b = torch.stack(((lo & 15) | (hi << 4), (lo >> 4) | (hi & 0xF0)), dim=-2)          # ..., s, b, p
        b = b.permute(0, 3, 1, 4, 2, 6, 5, 7, 8, 9).reshape(blocks, units, 2048)           # unit, strip, half, g, t, h, s, b, p
        one = records[e]
        one[..., :2048] = _turn(b.view(torch.int32), _BITS[scales.dtype]).view(torch.uint8)
        per_row = lambda t: pad(t[e], (0, n * units - t.shape[2], 0, more)).view(blocks, 2, 2, 8, units, n).permute(
            0, 4, 5, 1, 3, 2).reshape(blocks, units, 32 * n)  # unit, group, strip, g, r
        one[..., 2048:2048 + 64 * n] = per_row(scales).view(torch.uint8)
        if zeros is not None:
            one[..., 2048 + 64 * n:] = per_row(zeros)
    return Int4Experts(records, experts, outputs, inputs, group, zeros is not None, scales.dtype)


def quantize_int4(w, group=128, zero_points=False):
    """Int4Experts nearest to the float16 or bfloat16 weights w [E, K, N] (any strides): expert e computes x @ w[e].
    dmoe.expert_mlp's w1 [h, E * f] is w1.view(h, E, f).transpose(0, 1), its w2 [E * f, h] is w2.view(E, f, h).

    Without zero points a group's scale is its largest magnitude / 7 (codes 1..15); with them, its codes span the range
    of the group's values and 0.  Done once, when weights are loaded."""
    if w.dim() != 3 or w.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"quantize_int4: expected float16 or bfloat16 [experts, inputs, outputs], got {w.dtype} "
                         f"{tuple(w.shape)}")
    if group not in GROUPS or w.shape[1] % group or w.numel() == 0:
        raise ValueError(f"quantize_int4: the inputs must be whole groups of {', '.join(map(str, GROUPS))}, got "
                         f"{w.shape[1]} inputs, group {group}")
    experts, inputs, outputs = w.shape
    codes, scales, zeros = [], [], []
    for e in range(experts):                           # (one at a time: 32-bit copies of one expert only)
        v = w[e].t().reshape(outputs, inputs // group, group).float()
        if zero_points:
            low, high = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
            scale = ((high - low) / 15).to(w.dtype)
        else:
            scale = (v.abs().amax(2) / 7).to(w.dtype)
        # (a group of zeros, or one below the type's smallest number, keeps scale 0 and stands for zeros)
        step = torch.where(scale > 0, scale.float(), torch.ones_like(scale, dtype=torch.float32))
        zero = torch.round(-low / step).clamp(0, 15) if zero_points else torch.full_like(step, 8)
        q = (torch.round(v / step[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8).view(outputs, inputs)
        codes.append(q[:, 0::2] | (q[:, 1::2] << 4))
        scales.append(scale)
        zeros.append(zero.to(torch.uint8))
    return pack_int4(torch.stack(codes), torch.stack(scales), torch.stack(zeros) if zero_points else None)


def _check_call(what, x, w, expert_ids):
    if not isinstance(w, Int4Experts):
        raise ValueError(f"{what}: weights come from pack_int4 or quantize_int4, got {type(w).__name__}")
    if x.dim() != 2 or x.shape[1] != w.inputs:
        raise ValueError(f"{what}: x must be [tokens, {w.inputs}], got {tuple(x.shape)}")
    if x.dtype != w.dtype:
        raise ValueError(f"{what}: x is {x.dtype}, the weights' scales are {w.dtype}")
    if expert_ids is not None and (expert_ids.dim() != 2 or expert_ids.shape[0] != x.shape[0] or
                                   expert_ids.shape[1] < 1 or
                                   expert_ids.dtype not in (torch.int16, torch.int32, torch.int64)):
        raise ValueError(f"{what}: expert_ids must be integers [{x.shape[0]}, k], got {expert_ids.dtype} "
                         f"{tuple(expert_ids.shape)}")
    refuse_tangents(what, x)
    if not x.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA tensors only (there is no CPU path); got a tensor on {x.device}")
    if w.device != x.device or (expert_ids is not None and expert_ids.device != x.device):
        raise ValueError(f"{what}: all tensors must be on one device")
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError(f"{what} is forward only: x requires a gradient (call it under torch.no_grad())")


def _matvec(x, w, ids, x_div, gelu, out):
    _lib.launch("stk_b200_int4_matvec", x.device, w.records.data_ptr(), x.data_ptr(), ids.data_ptr(), out.data_ptr(),
                ids.numel(), x_div, w.num_experts, w.outputs, w.inputs, w.group, int(w.zero_points), int(gelu),
                int(out.dtype == torch.float32), _lib.dtype_code(w.dtype))
    return out


def _operand(x):
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def int4_matvec(x, w, expert_ids=None, gelu=False):
    """y[t, j] = W_e x[t] for e = expert_ids[t, j]: [T, k, N] in x's type (sums in 32 bits, rounded once), zeros where
    the id is negative; without expert_ids (weights of one expert) [T, N].  gelu: the GeLU (erf form) of the products.
    x [T, K] float16 or bfloat16, the type of the weights' scales.  Weights are exact (code - zero) times their scale: what
    lies under a code at its zero point adds nothing.  An infinity in a row of x makes its results infinite, or NaN where its weight
    is 0, and so may finite values above 1e35 (a group's sum is taken before its scale).
    Made for few tokens: an expert's weights are read once for every 16 slots that chose it, and anew for every 256
    slots of the call."""
    _check_call("int4_matvec", x, w, expert_ids)
    if expert_ids is None and w.num_experts != 1:
        raise ValueError(f"int4_matvec: {w.num_experts} experts need expert_ids")
    tokens = x.shape[0]
    ids = (torch.zeros((tokens, 1), dtype=torch.int32, device=x.device) if expert_ids is None
           else ids32(expert_ids))
    out = x.new_empty((tokens, ids.shape[1], w.outputs))
    _matvec(_operand(x), w, ids, ids.shape[1], gelu, out)
    return out[:, 0] if expert_ids is None else out


def expert_mlp_int4(x, expert_ids, weights, w1, w2):
    """The experts' MLP of a dMoE layer on few tokens (decoding), from 4-bit weights:
    out[t] = sum_j weights[t, j] * W2_e GeLU(W1_e x[t]), e = expert_ids[t, j], [T, h_out] in x's type.

    x [T, h] float16 or bfloat16 (forward only: a gradient or a tangent is refused); expert_ids [T, k] and weights [T, k] as top_k_gate gives them (a negative id
    contributes nothing); w1, w2: Int4Experts with f outputs and f inputs.  The hidden activations are rounded to x's
    type, as in dmoe.expert_mlp (a tenth more error in the result at most); the sums over inputs and over choices are in 32
    bits and rounded once."""
    _check_call("expert_mlp_int4", x, w1, expert_ids)
    refuse_tangents("expert_mlp_int4", weights)
    if not isinstance(w2, Int4Experts) or w2.num_experts != w1.num_experts or w2.inputs != w1.outputs \
            or w2.dtype != w1.dtype or w2.device != w1.device:
        raise ValueError("expert_mlp_int4: w2 must hold the same experts, in the same type and on the same device, with "
                         f"{w1.outputs} inputs")
    if tuple(weights.shape) != tuple(expert_ids.shape) or weights.device != x.device:
        raise ValueError(f"expert_mlp_int4: weights must be {tuple(expert_ids.shape)} on {x.device}, got "
                         f"{tuple(weights.shape)} on {weights.device}")
    _lib.row_dtype_code(weights.dtype)
    if torch.is_grad_enabled() and weights.requires_grad:
        raise ValueError("expert_mlp_int4 is forward only: weights require a gradient (call it under torch.no_grad())")
    tokens, top_k = expert_ids.shape
    ids, weights, x = ids32(expert_ids), weights.float().contiguous(), _operand(x)
    out = x.new_empty((tokens, w2.outputs))
    ws_bytes = _lib.load().stk_b200_int4_mlp_workspace_bytes(tokens * top_k, w1.outputs, w2.outputs)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    _lib.launch("stk_b200_int4_mlp", x.device, w1.records.data_ptr(), w2.records.data_ptr(), x.data_ptr(), ids.data_ptr(),
                weights.data_ptr(), out.data_ptr(), tokens, top_k, w1.num_experts, w1.inputs, w1.outputs, w2.outputs,
                w1.group, int(w1.zero_points), w2.group, int(w2.zero_points), _lib.dtype_code(x.dtype), ws.data_ptr(),
                ws_bytes)
    return out
