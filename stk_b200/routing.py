"""The trainable way of the tokens through a dMoE layer: the router's gate, the placement of the chosen (token, choice)
slots in padded expert bins, the copy of the token rows there and the weighted sum of the experts' rows back, each
with its gradient.  Public as stk_b200.dmoe.top_k_gate / plan_rows / plan_tokens / sort_tokens / unsort_tokens:

    weights, ids = dmoe.top_k_gate(x @ w_router, top_k)
    plan = dmoe.plan_tokens(ids, num_experts)
    topo = dmoe.topology_from_bins(plan.bin_rows, plan.block_rows, ffn, x.dtype, x.device, materialize=False)
    y = dmoe.expert_mlp(dmoe.sort_tokens(x, plan), w1, w2, topo)
    out = dmoe.unsort_tokens(y, weights, plan)             # differentiable in x, w_router, w1 and w2

A step with its backward pass can be captured in a CUDA graph (plan_tokens with rows=...) as long as no eager graph of the
same leaves is alive that was made on the default stream: torch's engine waits for the stream of a leaf's accumulator,
in torch.autograd.grad too, and raises an error where that is not the capturing one.

On CUDA tensors everything runs as kernels of libstk_b200.so, with first derivatives in reverse mode; second ones and those
in forward mode are refused.  Host tensors take plain torch operations (as in
stk_b200.dmoe: for tests, not for production use).  The reference is a matmul library and has no counterpart.
"""
import threading

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from stk_b200.backend import lib as _lib

BLOCK = 128
MAX_EXPERTS = 1024     # of the gate and of a plan
MAX_TOP_K = 32         # of the gate
_SCORES = {"softmax": 0, "sigmoid": 1}


def _rows(t):
    """`t`, or a copy, as rows that are contiguous in themselves.  (Rows that are one row repeated, with a stride of 0,
    are fine: they are only read.)"""
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _whole(what, name, value):
    n = int(value)
    if n != value:
        raise ValueError(f"{what}: {name} must be a whole number, got {value}")
    return n


def ids32(ids):
    """Expert ids as contiguous int32; 64-bit ones beyond it stay beyond every expert."""
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, 2 ** 31 - 1)
    return ids.to(torch.int32).contiguous()


def refuse_tangents(what, *tensors):
    """The kernels have no forward-mode derivatives, and a tangent that they dropped would count as zero."""
    if forward_ad._current_level < 0:                  # outside every dual level nothing has one (0.8 us of 10 to ask a call's)
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


def _once(backward):
    """once_differentiable for a backward pass made of kernels, at no cost where no graph of it is wanted."""
    recorded = once_differentiable(backward)
    return lambda ctx, *grads: (recorded if torch.is_grad_enabled() else backward)(ctx, *grads)


# ------------------------------------------------------------------------------ gate
def _gate(logits, mask, top_k, score, normalize, stats):
    tokens, experts = logits.shape
    weights = logits.new_empty((tokens, top_k), dtype=torch.float32)
    ids = logits.new_empty((tokens, top_k), dtype=torch.int32)
    rows = _rows(logits)
    _lib.launch("stk_b200_top_k_gate", logits.device, rows.data_ptr(), _ld(rows), tokens, experts, top_k, score,
                normalize, _lib.ptr(mask), weights.data_ptr(), ids.data_ptr(), _lib.ptr(stats),
                _lib.row_dtype_code(logits.dtype))
    return weights, ids


class _TopKGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, top_k, score, normalize):
        # (the gradient of the plain softmax reaches every logit; the normalized softmax weights alone give theirs)
        dense = score == 0 and not normalize
        stats = logits.new_empty((logits.shape[0], 2), dtype=torch.float32) if dense else None
        weights, ids = _gate(logits, mask, top_k, score, normalize, stats)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits if dense or score == 1 else None, weights, ids, stats)
        ctx.like = (logits.shape, logits.dtype, score, normalize)
        return weights, ids

    @staticmethod
    @_once
    def backward(ctx, dweights, _):
        if dweights is None:
            return None, None, None, None, None
        logits, weights, ids, stats = ctx.saved_tensors
        (tokens, experts), dtype, score, normalize = ctx.like
        dweights = dweights.contiguous()
        dlogits = weights.new_empty((tokens, experts), dtype=dtype)
        rows = dlogits if logits is None else _rows(logits)
        _lib.launch("stk_b200_top_k_gate_backward", weights.device, rows.data_ptr(), _ld(rows), tokens, experts,
                    weights.shape[1], score, normalize, weights.data_ptr(), ids.data_ptr(), _lib.ptr(stats),
                    dweights.data_ptr(), dlogits.data_ptr(), _lib.row_dtype_code(dtype))
        return dlogits, None, None, None, None


def _host_gate(logits, mask, top_k, score, normalize):
    values = logits.float()
    nan = values.detach().isnan()
    ids = torch.sort(values.detach().masked_fill(nan, torch.inf), dim=1, descending=True, stable=True).indices[:, :top_k]
    top = torch.gather(values, 1, ids)
    valid = top.detach() != -torch.inf
    if mask is not None:
        valid = valid & mask[:, None]
    top = top.masked_fill(~valid, -torch.inf)
    if score == 0:
        some = valid.any(1, keepdim=True)
        if normalize:
            weights = torch.softmax(top.masked_fill(~some, 0.0), 1)
        else:
            whole = values.masked_fill(~some, 0.0)
            weights = torch.gather(torch.softmax(whole, 1), 1, ids)
    elif normalize:
        some = valid.any(1, keepdim=True)
        logs = torch.nn.functional.logsigmoid(top.masked_fill(~valid, 0.0)).masked_fill(~valid & some, -torch.inf)
        weights = torch.softmax(logs, 1)
    else:
        weights = torch.sigmoid(top)
    weights = weights + torch.zeros(()).masked_fill(nan.any(1, keepdim=True), torch.nan)
    return weights.masked_fill(~valid, 0.0), ids.masked_fill(~valid, -1).to(torch.int32)


def top_k_gate(logits, top_k, score="softmax", normalize=True, token_mask=None):
    """The router's choice: (weights float32 [T, k], expert_ids int32 [T, k]) of the k largest logits of every token,
    the largest first, differentiable in `logits` through the weights.

    logits: [T, E] float16, bfloat16 or float32, E <= 1024; k <= min(E, 32).  score: "softmax" (over all E logits) or
    "sigmoid"; normalize: the k weights of a token are scaled to add up to 1.  Equal logits go to the lower expert, and
    an expert whose logit is -inf is never chosen.  A choice that is left without an expert (fewer than k logits above
    -inf, or token_mask[t] False: bool [T], padding tokens) has id -1 and weight 0 and passes no gradient; plan_tokens
    gives it no row.  A NaN counts as +inf among the logits and makes the token's weights NaN."""
    if logits.dim() != 2:
        raise ValueError(f"top_k_gate: logits must be [tokens, experts], got {tuple(logits.shape)}")
    if score not in _SCORES:
        raise ValueError(f"top_k_gate: score must be one of {sorted(_SCORES)}, got {score!r}")
    tokens, experts = logits.shape
    _lib.row_dtype_code(logits.dtype)
    top_k = _whole("top_k_gate", "top_k", top_k)
    if not 1 <= experts <= MAX_EXPERTS or not 1 <= top_k <= min(experts, MAX_TOP_K):
        raise ValueError(f"top_k_gate: 1 <= top_k <= min(experts, {MAX_TOP_K}) and experts <= {MAX_EXPERTS}, got "
                         f"top_k = {top_k}, {experts} experts")
    if token_mask is not None:
        if token_mask.dtype != torch.bool or tuple(token_mask.shape) != (tokens,):
            raise ValueError(f"top_k_gate: token_mask must be bool [{tokens}], got {token_mask.dtype} "
                             f"{tuple(token_mask.shape)}")
        if token_mask.device != logits.device:
            raise ValueError(f"top_k_gate: the logits are on {logits.device}, the token mask on {token_mask.device}")
        token_mask = token_mask.contiguous()
    if not logits.is_cuda:
        return _host_gate(logits, token_mask, top_k, _SCORES[score], normalize)
    refuse_tangents("top_k_gate", logits)
    args = (logits, token_mask, top_k, _SCORES[score], int(bool(normalize)))
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TopKGate.apply(*args)
    return _gate(*args, None)


# ------------------------------------------------------------------------------ placement
class TokenPlan:
    """Where the slots of one routed batch (slot = token * top_k + choice) sit in padded expert bins; made by
    plan_tokens and not to be changed.

    index     int32 [rows]       slot in the row, -1: padding
    position  int32 [T * top_k]  row of the slot, -1: a slot without an expert
    bin_rows  int32 [E]          blocks of every expert's bin, as topology_from_bins takes them
    rows, block_rows             rows of all bins, and the same in blocks (host ints)"""

    __slots__ = ("index", "position", "bin_rows", "rows", "block_rows", "tokens", "top_k", "num_experts", "block")

    def __init__(self, index, position, bin_rows, rows, tokens, top_k, num_experts, block):
        self.index, self.position, self.bin_rows = index, position, bin_rows
        self.rows, self.block_rows = rows, rows // block
        self.tokens, self.top_k, self.num_experts, self.block = tokens, top_k, num_experts, block


def plan_rows(slots, num_experts, block=BLOCK):
    """Most rows that `slots` choices can take in bins padded to a multiple of `block`, whatever the choices are."""
    return (slots + min(slots, num_experts) * (block - 1)) // block * block


_pinned = threading.local()


def _host_word():
    """Pinned int64 of this thread, which a kernel writes and the thread waits for: never in two uses at once."""
    word = getattr(_pinned, "word", None)
    if word is None:
        word = _pinned.word = torch.zeros(1, dtype=torch.int64).pin_memory()
    return word


def plan_tokens(expert_ids, num_experts, block=BLOCK, rows=None):
    """TokenPlan of expert_ids ([T] or [T, k], integers; a negative id: no expert): every expert's slots in order, its
    bin padded to a multiple of `block` rows.

    rows None: as many rows as this batch needs, none for a batch without a live token - the one read-back of the step (the
    call waits for the stream).
    rows = plan_rows(slots, num_experts) or more, a multiple of `block`: that many, the surplus as padding at the end
    of the last expert's bin; nothing waits for the device, and the step can be captured in a CUDA graph."""
    if expert_ids.dim() not in (1, 2) or expert_ids.dtype not in (torch.int16, torch.int32, torch.int64):
        raise ValueError(f"plan_tokens: expert_ids must be integers [T] or [T, k], got {expert_ids.dtype} "
                         f"{tuple(expert_ids.shape)}")
    num_experts, block = _whole("plan_tokens", "num_experts", num_experts), _whole("plan_tokens", "block", block)
    rows = None if rows is None else _whole("plan_tokens", "rows", rows)
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"plan_tokens: 1 to {MAX_EXPERTS} experts, got {num_experts}")
    if block < 1:
        raise ValueError(f"plan_tokens: block must be positive, got {block}")
    tokens = expert_ids.shape[0]
    top_k = 1 if expert_ids.dim() == 1 else expert_ids.shape[1]
    if top_k < 1:
        raise ValueError("plan_tokens: no choices")
    flat = expert_ids.reshape(-1)
    slots, need = flat.numel(), plan_rows(flat.numel(), num_experts, block)
    if need > 2 ** 31 - 1:
        raise ValueError(f"plan_tokens: {slots} slots are beyond what 32-bit row numbers name")
    if rows is not None and (rows < need or rows % block or rows > 2 ** 31 - 1):
        raise ValueError(f"plan_tokens: rows must be a multiple of {block} and at least plan_rows(...) = {need}, got {rows}")
    if not flat.is_cuda:
        index, position, bin_rows = _host_plan(flat.long(), num_experts, block, rows)
        return TokenPlan(index, position, bin_rows, index.numel(), tokens, top_k, num_experts, block)
    dev = flat.device
    if rows is None and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("plan_tokens: reading the number of rows back cannot be captured; pass rows=plan_rows(...)")
    flat = ids32(flat)
    length = need if rows is None else rows
    index, position, bin_rows = flat.new_empty(length), flat.new_empty(slots), flat.new_empty(num_experts)
    ws_bytes = _lib.load().stk_b200_place_workspace_bytes(slots, num_experts)
    ws = flat.new_empty(ws_bytes // 4) if ws_bytes else None
    word = _host_word() if rows is None else None
    _lib.launch("stk_b200_place_tokens", dev, flat.data_ptr(), slots, num_experts, block, length, int(rows is not None),
                index.data_ptr(), position.data_ptr(), bin_rows.data_ptr(), _lib.ptr(word), _lib.ptr(ws), ws_bytes)
    if rows is None:
        torch.cuda.current_stream(dev).synchronize()
        length = int(word)
        index = index[:length]
    return TokenPlan(index, position, bin_rows, length, tokens, top_k, num_experts, block)


def _host_plan(flat, num_experts, block, rows):
    if bool((flat >= num_experts).any()):
        raise ValueError(f"plan_tokens: expert ids reach {int(flat.max())}, there are {num_experts} experts")
    live = torch.nonzero(flat >= 0).view(-1)
    order = live[torch.argsort(flat[live], stable=True)]
    counts = torch.bincount(flat[live], minlength=num_experts)
    blocks = (counts + block - 1) // block
    used = int(blocks.sum()) * block
    starts = (torch.cumsum(blocks, 0) - blocks) * block
    first = torch.cumsum(counts, 0) - counts
    experts = flat[order]
    place = starts[experts] + torch.arange(order.numel()) - first[experts]
    position = torch.full((flat.numel(),), -1, dtype=torch.int32)
    position[order] = place.to(torch.int32)
    index = torch.full((used if rows is None else rows,), -1, dtype=torch.int32)
    index[place] = order.to(torch.int32)
    if rows is not None:
        blocks[-1] += (rows - used) // block
    return index, position, blocks.to(torch.int32)


# ------------------------------------------------------------------------------ rows there and back
def _sum_rows(rows, weights, plan):
    rows = _rows(rows)
    hidden = rows.shape[1]
    out = rows.new_empty((plan.tokens, hidden))
    _lib.launch("stk_b200_sum_rows", rows.device, rows.data_ptr(), _ld(rows), plan.position.data_ptr(),
                _lib.ptr(weights), out.data_ptr(), plan.tokens, plan.top_k, hidden, _lib.row_dtype_code(rows.dtype))
    return out


def _sort_rows(x, plan):
    x = _rows(x)
    hidden = x.shape[1]
    rows = x.new_empty((plan.rows, hidden))
    _lib.launch("stk_b200_sort_rows", x.device, x.data_ptr(), _ld(x), rows.data_ptr(), plan.index.data_ptr(),
                plan.position.data_ptr(), plan.tokens, plan.top_k, plan.rows, hidden, _lib.row_dtype_code(x.dtype))
    return rows


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return _sort_rows(x, plan)

    @staticmethod
    @_once
    def backward(ctx, drows):
        return _sum_rows(drows, None, ctx.plan), None


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan):
        ctx.plan = plan
        need_weights = weights is not None and ctx.needs_input_grad[1]
        ctx.save_for_backward(rows if need_weights else None, weights)
        ctx.like = (rows.shape, rows.dtype)
        return _sum_rows(rows, weights, plan)

    @staticmethod
    @_once
    def backward(ctx, dout):
        rows, weights = ctx.saved_tensors
        plan, (shape, dtype) = ctx.plan, ctx.like
        dout = _rows(dout)
        drows = dweights = None
        if ctx.needs_input_grad[0]:
            drows = dout.new_empty(shape, dtype=dtype)
        if rows is not None:
            rows = _rows(rows)
            dweights = torch.empty_like(weights)
        _lib.launch("stk_b200_unsort_backward", dout.device, dout.data_ptr(), _ld(dout), _lib.ptr(rows),
                    0 if rows is None else _ld(rows), _lib.ptr(weights), plan.index.data_ptr(),
                    plan.position.data_ptr(), _lib.ptr(drows), _lib.ptr(dweights), plan.tokens, plan.top_k, plan.rows,
                    shape[1], _lib.row_dtype_code(dtype))
        return drows, dweights, None


def _check_rows(what, t, n, name, plan):
    if t.dim() != 2 or t.shape[0] != n:
        raise ValueError(f"{what}: expected {n} rows ({name}), got {tuple(t.shape)}")
    _lib.row_dtype_code(t.dtype)
    if t.device != plan.position.device:
        raise ValueError(f"{what}: the rows are on {t.device}, the plan on {plan.position.device}")


def sort_tokens(x, plan):
    """The token rows x [T, h] (float16, bfloat16 or float32) in the padded expert order of `plan`: [plan.rows, h],
    zeros in padding rows.  Differentiable: the gradient of a token is the sum of those of its rows, added up in
    32 bits."""
    _check_rows("sort_tokens", x, plan.tokens, "tokens of the plan", plan)
    if x.is_cuda:
        refuse_tangents("sort_tokens", x)
        return _SortTokens.apply(x, plan) if torch.is_grad_enabled() and x.requires_grad else _sort_rows(x, plan)
    valid = plan.index >= 0
    out = x.new_zeros((plan.rows, x.shape[1]))
    return out.index_put((torch.nonzero(valid).view(-1),),
                         x[torch.div(plan.index[valid].long(), plan.top_k, rounding_mode="floor")])


def unsort_tokens(rows, weights, plan):
    """The way back: out[t] = sum_j weights[t, j] * rows[row of slot t * k + j], [T, h], added up in 32 bits and rounded
    once.  rows [plan.rows, h]; weights [T, k] (or [T] for k = 1) float32 or a 16-bit float, None: all ones.  Slots
    without an expert contribute nothing.  Differentiable in `rows` (padding rows get zeros) and in `weights` (a slot
    without an expert gets 0)."""
    _check_rows("unsort_tokens", rows, plan.rows, "rows of the plan", plan)
    if weights is not None:
        if weights.shape != (plan.tokens, plan.top_k) and (plan.top_k != 1 or weights.shape != (plan.tokens,)):
            raise ValueError(f"unsort_tokens: weights must be [{plan.tokens}, {plan.top_k}], got {tuple(weights.shape)}")
        _lib.row_dtype_code(weights.dtype)
        if weights.device != rows.device:
            raise ValueError(f"unsort_tokens: the rows are on {rows.device}, the weights on {weights.device}")
        if weights.dim() == 1:
            weights = weights[:, None]
        weights = weights.float().contiguous()
    if rows.is_cuda:
        refuse_tangents("unsort_tokens", rows, weights)
        if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)):
            return _UnsortTokens.apply(rows, weights, plan)
        return _sum_rows(rows, weights, plan)
    position = plan.position.long()
    # (a gather of at least one row, so that an empty plan needs no case of its own)
    padded = torch.cat([rows.float(), torch.zeros((1, rows.shape[1]))])
    y = padded[torch.where(position >= 0, position, torch.full_like(position, plan.rows))]
    y = y.view(plan.tokens, plan.top_k, rows.shape[1])
    if weights is not None:
        y = y * weights[:, :, None]
    return y.sum(1).to(rows.dtype)
